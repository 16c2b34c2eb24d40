// Shared-prefix attention for few query rows per KV head (decode), the merge of
// partial results and the accumulated key weights.  Formulas and the row and
// partial-result conventions: prefix_attention.cuh.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "pdl.cuh"
#include "prefix_attention.cuh"
#include "tile_math.cuh"

namespace nb200 {
namespace {

using namespace tile;

// ---- matrix fragments ------------------------------------------------------

template <bool BF>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}

// 16-byte copy to shared memory, zeros where the source does not exist
__device__ __forceinline__ void cp16z(uint32_t dst, const void *src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void cp4z(uint32_t dst, const void *src, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}

// ---- the streaming kernel --------------------------------------------------
//
// A unit attends one tile of rows to one key range: 16 rows of a 16-bit cache
// (an m16n8k16 A operand), or 8 rows of an INT8 cache, whose FP32 queries and
// softmax weights fill the 16 rows of A as FP16 pairs hi + lo (the codes
// themselves are exact in FP16), so that INT8 costs no further products and
// keeps FP32 accuracy.  Each warp of a unit walks its own blocks of keys (one
// pass, running maximum and sum), fed by its own ring of asynchronous copies;
// the states of a unit's warps meet in shared memory at the end.
//
// Bound by HBM where keys are long and many: 256 sessions of 3712 INT8 keys and 4
// KV heads behind 384 shared ones (518 MB) 106 us, 4.9 TB/s, of the 79 us that a
// copy of the bytes would take.  What is left is instructions: 64 % of the issue
// slots, half of them on the integer pipe, which turns the codes into FP16 (three
// of its instructions for four codes of K, eight for eight of V).  Two stages a
// ring: three were slower (121 against 113 us), fewer CTAs fit.

constexpr int kWarps = 4;
// Keys of a range that one warp takes by itself (1024 sessions of 64 INT8 slots: 36 us
// against 48 with four warps a unit; two sequences of 200 keys: 11 against 5.3), and
// four times as many where the units are 16 a multiprocessor or more (1019 sessions
// of 135 slots and 8 KV heads: 94 against 125 us).
constexpr int kShortRange = 64;
constexpr int kManyUnits = 2368;

template <int TYPE, int HD>
struct StreamGeom {
    static constexpr bool I8 = TYPE == kCacheI8;
    static constexpr int kSize = I8 ? 1 : 2;
    static constexpr int kRows = I8 ? 8 : 16;                             // query rows of a tile
    static constexpr int kKeys = I8 ? 32 : (HD == 64 ? 32 : 16);          // keys of a block
    static constexpr int kStages = 2;
    static constexpr int kKRow = HD * kSize;                              // bytes of a K row in shared memory
    // INT8 V rows are read a word per (key, four dimensions), keys of one
    // access two rows apart: 16 bytes of padding spread them over the banks
    static constexpr int kVRow = I8 ? HD + 16 : HD * 2;
    static constexpr int kVOff = kKeys * kKRow;
    static constexpr int kSOff = kVOff + kKeys * kVRow;
    static constexpr int kStage = kSOff + (I8 ? 2 * kKeys * 4 : 0);
    static constexpr int kMerge = 16 * HD * 4 + 64 * 4;                   // one warp's state at the end
    static constexpr int kRing = kStages * kStage;
    static constexpr int kWarpBytes = (kRing > kMerge ? kRing : kMerge);
    static constexpr int kSmem = kWarps * kWarpBytes;
    static_assert(kStage % 16 == 0 && kVOff % 16 == 0 && kWarpBytes % 16 == 0, "alignment of the copies");
};

struct KeySet {
    const char *k, *v;
    const float *ks, *vs;
    long long k_step, v_step, ks_step, vs_step;   // bytes (K, V), elements (scales) per key
};

struct StreamGrid {
    int own_units, own_tiles, prefix_units, prefix_tiles;
    int own_slots, prefix_slots;
    int joint;                                    // own units take the prefix too
};

// One lane's part of the copies of a warp's blocks: 16-byte pieces of K and V
// rows, a scale of each; advances by a fixed number of keys.
template <int TYPE, int HD>
struct BlockCopy {
    using G = StreamGeom<TYPE, HD>;
    static constexpr int kChunks = HD * G::kSize / 16;      // 16-byte pieces of a row
    static constexpr int kPer = 32 / kChunks;               // rows of one warp-wide copy
    const char *k, *v;
    const float *ks, *vs;
    long long k_per, v_per, k_next, v_next, ks_next, vs_next;

    __device__ __forceinline__ void set(const KeySet &s, int j0, int keys, int lane) {
        const long long r = j0 + lane / kChunks, piece = lane % kChunks * 16;
        k = s.k + r * s.k_step + piece;
        v = s.v + r * s.v_step + piece;
        k_per = kPer * s.k_step;
        v_per = kPer * s.v_step;
        k_next = keys * s.k_step;
        v_next = keys * s.v_step;
        if constexpr (G::I8) {
            static_assert(G::kKeys == 32, "one scale a lane");
            ks = s.ks + (long long)(j0 + lane) * s.ks_step;
            vs = s.vs + (long long)(j0 + lane) * s.vs_step;
            ks_next = keys * s.ks_step;
            vs_next = keys * s.vs_step;
        }
    }

    // `left` keys exist; rows behind them become zeros
    __device__ __forceinline__ void block(char *stage, int left, int lane) {
        const uint32_t base = smem_addr(stage);
        const int c = lane % kChunks, r0 = lane / kChunks;
        const char *kp = k, *vp = v;
#pragma unroll
        for (int i = 0; i < G::kKeys / kPer; ++i) {
            const int r = r0 + i * kPer;
            int kc = c, vc = c;
            if constexpr (TYPE != kCacheI8) {
                kc = vc = c ^ (r & 7);                       // rows of an 8x8 matrix on different banks
            } else if constexpr (HD == 128) {
                kc = c ^ ((r & 1) << 2);
            }
            const bool valid = r < left;
            cp16z(base + r * G::kKRow + kc * 16, valid ? kp : k, valid);
            cp16z(base + G::kVOff + r * G::kVRow + vc * 16, valid ? vp : v, valid);
            kp += k_per;
            vp += v_per;
        }
        k += k_next;
        v += v_next;
        if constexpr (G::I8) {
            const bool valid = lane < left;
            cp4z(base + G::kSOff + lane * 4, ks, valid);
            cp4z(base + G::kSOff + 128 + lane * 4, vs, valid);
            ks += ks_next;
            vs += vs_next;
        }
    }
};

template <int TYPE, int HD>
__device__ __forceinline__ KeySet prefix_set(const PrefixAttn &p, int g) {
    constexpr int kSize = StreamGeom<TYPE, HD>::kSize;
    KeySet s;
    s.k = (const char *)p.pk + g * p.pks[0] * kSize;
    s.v = (const char *)p.pv + g * p.pvs[0] * kSize;
    s.k_step = p.pks[1] * kSize;
    s.v_step = p.pvs[1] * kSize;
    if constexpr (TYPE == kCacheI8) {
        s.ks = p.pkscale + g * p.pkss[0];
        s.vs = p.pvscale + g * p.pvss[0];
        s.ks_step = p.pkss[1];
        s.vs_step = p.pvss[1];
    }
    return s;
}

// W warps share a unit's keys: four where the ranges are long, one (and four
// units a CTA, no merge between warps) where they are short.
template <int TYPE, int HD, int W>
__device__ __forceinline__ void stream_unit(const PrefixAttn &p, const StreamGrid &grid) {
    using G = StreamGeom<TYPE, HD>;
    constexpr bool I8 = G::I8, BF = TYPE == kCacheBF16;
    constexpr int NT = G::kKeys / 8;                 // 8-key columns of a block
    constexpr int KS = HD / 16;                      // k steps of Q K^T
    extern __shared__ __align__(16) char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g8 = lane >> 2, c = lane & 3;
    char *ring = smem + warp * G::kWarpBytes;
    const int part = warp % W;                       // of the unit's warps

    // the unit: rows [m0, m0 + rows) of KV head g, keys [lo, hi)
    const int R = p.group, TR = p.tokens * R;
    int unit = blockIdx.x * (kWarps / W) + warp / W, g, m0, rows, lo, hi, slot, seq = -1, len = 0, nq = 0;
    if (unit >= grid.own_units + grid.prefix_units) return;
    KeySet s;
    if (unit < grid.own_units) {
        slot = unit % grid.own_slots;
        unit /= grid.own_slots;
        const int tile = unit % grid.own_tiles;
        unit /= grid.own_tiles;
        g = unit % p.kvheads;
        seq = unit / p.kvheads;
        m0 = seq * TR + tile * G::kRows;
        rows = min(G::kRows, TR - tile * G::kRows);
        len = own_length(p, seq);
        nq = own_tokens(p, seq);
        const int t0 = tile * G::kRows / R, t1 = min((tile * G::kRows + rows - 1) / R, nq - 1);
        hi = max(0, min(len, len - nq + t1 + 1));    // behind the last visible key of the tile
        lo = p.window ? max(0, len - nq + t0 - p.window + 1) : 0;
        if (t0 >= nq) rows = 0;                      // padding rows only
        const long long row = p.cache_row ? p.cache_row[seq] : seq;
        s.k = (const char *)p.k + (row * p.ks[0] + g * p.ks[1]) * G::kSize;
        s.v = (const char *)p.v + (row * p.vs[0] + g * p.vs[1]) * G::kSize;
        s.k_step = p.ks[2] * G::kSize;
        s.v_step = p.vs[2] * G::kSize;
        if constexpr (I8) {
            s.ks = p.kscale + row * p.kss[0] + g * p.kss[1];
            s.vs = p.vscale + row * p.vss[0] + g * p.vss[1];
            s.ks_step = p.kss[2];
            s.vs_step = p.vss[2];
        }
        const int n = max(0, hi - lo), each = (ceil_div(n, grid.own_slots) + G::kKeys - 1) / G::kKeys * G::kKeys;
        const int a = min(hi, lo + slot * each);
        hi = min(hi, a + each);
        lo = a;
        slot += p.prefix_slots;
    } else {
        unit -= grid.own_units;
        slot = unit % grid.prefix_slots;
        unit /= grid.prefix_slots;
        const int tile = unit % grid.prefix_tiles;
        g = unit / grid.prefix_tiles;
        m0 = tile * G::kRows;
        rows = min(G::kRows, p.batch * TR - m0);
        s = prefix_set<TYPE, HD>(p, g);
        const int each = (ceil_div(p.prefix, grid.prefix_slots) + G::kKeys - 1) / G::kKeys * G::kKeys;
        lo = min(p.prefix, slot * each);
        hi = min(p.prefix, lo + each);
    }
    if (rows <= 0) return;

    // first copies, then the queries
    int mine, left;                                  // this warp's blocks; keys from the next one to be copied on
    BlockCopy<TYPE, HD> copy;
    auto begin = [&] {
        const int blocks = ceil_div(max(0, hi - lo), G::kKeys);
        mine = blocks > part ? (blocks - part + W - 1) / W : 0;
        left = hi - lo - part * G::kKeys;
        copy.set(s, lo + part * G::kKeys, W * G::kKeys, lane);
#pragma unroll
        for (int i = 0; i < G::kStages - 1; ++i) {
            if (i < mine) copy.block(ring + i * G::kStage, left, lane);
            left -= W * G::kKeys;
            cp_async_commit();
        }
    };
    begin();

    // this lane's rows (g8 and, 16-bit, g8 + 8), their visible own keys [first, last]
    constexpr int kMine = I8 ? 1 : 2;
    int first[kMine], last[kMine];
    const char *qrow[kMine];
#pragma unroll
    for (int e = 0; e < kMine; ++e) {
        const int m = m0 + min(g8 + 8 * e, rows - 1);
        const int b = m / TR, t = (m - b * TR) / R, h = g * R + m % R;
        qrow[e] = (const char *)p.q + (b * p.qs[0] + t * p.qs[1] + h * p.qs[2]) * (I8 ? 4 : 2);
        first[e] = 0;
        last[e] = 0x7fffffff;
        if (seq >= 0) {
            last[e] = t < nq ? len - nq + t : -1;
            first[e] = p.window ? len - nq + t - p.window + 1 : 0;
        }
        last[e] = min(last[e], hi - 1);
    }
    int all_from = max(first[0], first[kMine - 1]), all_to = min(last[0], last[kMine - 1]);
    uint32_t qa[KS][4];
    float qscale = p.scale2;
    if constexpr (I8) {
        // dimension order of the K words below: k step s of lane column c holds
        // dimensions 64 (s / 4) + 16 c + 4 (s % 4) + 0..3
        const float *q = (const float *)qrow[0];
        float x[KS][4], most = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const float4 f = *(const float4 *)(q + 64 * (k / 4) + 16 * c + 4 * (k % 4));
            x[k][0] = f.x; x[k][1] = f.y; x[k][2] = f.z; x[k][3] = f.w;
            most = fmaxf(fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y))), fmaxf(fabsf(f.z), fabsf(f.w)));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        float up, down;
        row_scale(most, up, down);
        qscale *= down;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            split2(x[k][0] * up, x[k][1] * up, qa[k][0], qa[k][1]);
            split2(x[k][2] * up, x[k][3] * up, qa[k][2], qa[k][3]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            qa[k][0] = *(const uint32_t *)(qrow[0] + (16 * k + 2 * c) * 2);
            qa[k][1] = *(const uint32_t *)(qrow[1] + (16 * k + 2 * c) * 2);
            qa[k][2] = *(const uint32_t *)(qrow[0] + (16 * k + 2 * c + 8) * 2);
            qa[k][3] = *(const uint32_t *)(qrow[1] + (16 * k + 2 * c + 8) * 2);
        }
    }

    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float top[kMine], sum[kMine], vnorm = 0.f;
#pragma unroll
    for (int e = 0; e < kMine; ++e) top[e] = kNegInf, sum[e] = 0.f;
    float *logits = nullptr;
    if (p.logits && seq >= 0)
        logits = p.logits + ((long long)(seq * p.kvheads + g) * TR + (m0 - seq * TR)) * p.capacity;

    bool then_prefix = seq >= 0 && grid.joint;
    for (int i = 0;; ++i) {
        if (i == mine) {
            if (!then_prefix) break;
            // then the prefix, on the same state; every query sees all of it
            then_prefix = false;
            asm volatile("cp.async.wait_all;" ::: "memory");
            __syncwarp();
            s = prefix_set<TYPE, HD>(p, g);
            lo = all_from = 0;
            hi = p.prefix;
            all_to = hi - 1;
#pragma unroll
            for (int e = 0; e < kMine; ++e) first[e] = 0, last[e] = hi - 1;
            logits = nullptr;
            begin();
            i = -1;
            continue;
        }
        cp_async_wait<G::kStages - 2>();
        __syncwarp();
        {   // the stage that was read last takes the copy two blocks ahead
            const int n = i + G::kStages - 1;
            if (n < mine) copy.block(ring + (n % G::kStages) * G::kStage, left, lane);
            left -= W * G::kKeys;
            cp_async_commit();
        }
        const char *stage = ring + (i % G::kStages) * G::kStage;
        const uint32_t base = smem_addr(stage);
        const int j0 = lo + (part + i * W) * G::kKeys;

        // z = Q K^T
        float z[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) z[n][0] = z[n][1] = z[n][2] = z[n][3] = 0.f;
        if constexpr (I8) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int r = 8 * n + g8;
#pragma unroll
                for (int x = 0; x < HD / 64; ++x) {
                    const int chunk = HD == 128 ? (4 * x + c) ^ ((r & 1) << 2) : c;
                    const uint4 w = *(const uint4 *)(stage + r * G::kKRow + chunk * 16);
                    const uint32_t u[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u,
                                           w.w ^ 0x80808080u};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        mma16816<false>(z[n], qa[4 * x + e], i8x2_to_f16<0x4140>(u[e]), i8x2_to_f16<0x4342>(u[e]));
                }
            }
        } else {
            const int r = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
#pragma unroll
            for (int n = 0; n < NT; n += 2)
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    uint32_t b[4];
                    const int row = 8 * n + r;
                    ldsm4(b, base + row * G::kKRow + (((2 * k + half) ^ (row & 7)) << 4));
                    mma16816<BF>(z[n], qa[k], b[0], b[1]);
                    mma16816<BF>(z[n + 1], qa[k], b[2], b[3]);
                }
        }

        // scale, mask, running maximum
        float best[kMine];
#pragma unroll
        for (int e = 0; e < kMine; ++e) best[e] = kNegInf;
        float vs[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if constexpr (I8) {
                const float2 ks = *(const float2 *)(stage + G::kSOff + (8 * n + 2 * c) * 4);
                const float2 v2 = *(const float2 *)(stage + G::kSOff + 128 + (8 * n + 2 * c) * 4);
                vs[n][0] = v2.x;
                vs[n][1] = v2.y;
                z[n][0] = (z[n][0] + z[n][2]) * (ks.x * qscale);
                z[n][1] = (z[n][1] + z[n][3]) * (ks.y * qscale);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) z[n][e] *= qscale;
            }
        }
        if (j0 < all_from || j0 + G::kKeys - 1 > all_to) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2 * kMine; ++e) {
                    const int key = j0 + 8 * n + 2 * c + (e & 1);
                    if (key > last[e >> 1] || key < first[e >> 1]) z[n][e] = kNegInf;
                }
        }
        if (logits) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2 * kMine; ++e) {
                    const int row = g8 + 8 * (e >> 1), key = j0 + 8 * n + 2 * c + (e & 1);
                    if (row < rows && key < hi) logits[(long long)row * p.capacity + key] = z[n][e];
                }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2 * kMine; ++e) best[e >> 1] = fmaxf(best[e >> 1], z[n][e]);
        float keep[kMine];
        bool moved = false;
#pragma unroll
        for (int e = 0; e < kMine; ++e) {
            best[e] = fmaxf(best[e], __shfl_xor_sync(0xffffffffu, best[e], 1));
            best[e] = fmaxf(best[e], __shfl_xor_sync(0xffffffffu, best[e], 2));
            const float t = fmaxf(top[e], best[e]);
            keep[e] = t == top[e] ? 1.f : ex2(top[e] - t);   // top = -inf: 0
            moved |= t != top[e];
            top[e] = t;
            sum[e] *= keep[e];
        }
        // INT8: V's scales go into the softmax weights, relative to the largest
        // scale so far (a power of two), with 2^12 above FP16's small numbers
        float vinv = 1.f;
        if constexpr (I8) {
            // (a scale a lane; sizes of floats order as their bits)
            const uint32_t size = *(const uint32_t *)(stage + G::kSOff + 128 + lane * 4) & 0x7fffffffu;
            const uint32_t most = __reduce_max_sync(0xffffffffu, size);
            const float vmax = __uint_as_float(max(most, 0x0da24260u) & 0x7f800000u);   // at least 1e-30
            if (vmax > vnorm) {                              // the same in every lane
                const float f = vnorm / vmax;
#pragma unroll
                for (int e = 0; e < kMine; ++e) keep[e] *= f;
                moved = true;
                vnorm = vmax;
            }
            vinv = 4096.f / vnorm;
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int d = 0; d < HD / 8; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[d][e] *= keep[I8 ? 0 : e >> 1];
        }

        // weights, then out += P V
        float base2[kMine];
#pragma unroll
        for (int e = 0; e < kMine; ++e) base2[e] = top[e] == kNegInf ? 0.f : top[e];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2 * kMine; ++e) {
                z[n][e] = ex2(z[n][e] - base2[e >> 1]);
                sum[e >> 1] += z[n][e];
            }
#pragma unroll
        for (int k = 0; k < G::kKeys / 16; ++k) {
            uint32_t a[4];
            if constexpr (I8) {
                split2(z[2 * k][0] * (vs[2 * k][0] * vinv), z[2 * k][1] * (vs[2 * k][1] * vinv), a[0], a[1]);
                split2(z[2 * k + 1][0] * (vs[2 * k + 1][0] * vinv), z[2 * k + 1][1] * (vs[2 * k + 1][1] * vinv), a[2],
                       a[3]);
                const char *v0 = stage + G::kVOff + (16 * k + 2 * c) * G::kVRow + 4 * g8;
#pragma unroll
                for (int x = 0; x < HD / 32; ++x) {
                    // dimensions 32 x + 4 n + 0..3 of column n, as four column tiles
                    const uint32_t w0 = *(const uint32_t *)(v0 + 32 * x) ^ 0x80808080u;
                    const uint32_t w1 = *(const uint32_t *)(v0 + G::kVRow + 32 * x) ^ 0x80808080u;
                    const uint32_t w2 = *(const uint32_t *)(v0 + 8 * G::kVRow + 32 * x) ^ 0x80808080u;
                    const uint32_t w3 = *(const uint32_t *)(v0 + 9 * G::kVRow + 32 * x) ^ 0x80808080u;
                    const uint32_t l01 = __byte_perm(w0, w1, 0x5140), h01 = __byte_perm(w0, w1, 0x7362);
                    const uint32_t l23 = __byte_perm(w2, w3, 0x5140), h23 = __byte_perm(w2, w3, 0x7362);
                    mma16816<false>(o[4 * x], a, i8x2_to_f16<0x4140>(l01), i8x2_to_f16<0x4140>(l23));
                    mma16816<false>(o[4 * x + 1], a, i8x2_to_f16<0x4342>(l01), i8x2_to_f16<0x4342>(l23));
                    mma16816<false>(o[4 * x + 2], a, i8x2_to_f16<0x4140>(h01), i8x2_to_f16<0x4140>(h23));
                    mma16816<false>(o[4 * x + 3], a, i8x2_to_f16<0x4342>(h01), i8x2_to_f16<0x4342>(h23));
                }
            } else {
                // the softmax weights are rounded to the cache's type for the product, off by
                // half a step of each at most; their sum keeps 32 bits (two sequences of 200
                // keys in bf16: 1.7e-3 from the definition, 1.6e-3 with 32-bit weights, the
                // output's rounding the most of it)
                a[0] = pack2<BF>(z[2 * k][0], z[2 * k][1]);
                a[1] = pack2<BF>(z[2 * k][2], z[2 * k][3]);
                a[2] = pack2<BF>(z[2 * k + 1][0], z[2 * k + 1][1]);
                a[3] = pack2<BF>(z[2 * k + 1][2], z[2 * k + 1][3]);
                const int row = 16 * k + (lane & 15), half = lane >> 4;
#pragma unroll
                for (int d = 0; d < HD / 16; ++d) {
                    uint32_t b[4];
                    ldsm4t(b, base + G::kVOff + row * G::kVRow + (((2 * d + half) ^ (row & 7)) << 4));
                    mma16816<BF>(o[2 * d], a, b[0], b[1]);
                    mma16816<BF>(o[2 * d + 1], a, b[2], b[3]);
                }
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();

    // each warp's state to shared memory: o[row][d] from kMerge's start, then (top, sum)
    float *mo = (float *)ring, *ms = mo + 16 * HD;
#pragma unroll
    for (int e = 0; e < kMine; ++e) {
        sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 1);
        sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 2);
        if (c == 0) {
            ms[2 * (g8 + 8 * e)] = top[e];
            ms[2 * (g8 + 8 * e) + 1] = sum[e];
        }
    }
    if constexpr (I8) {
        const float f = vnorm * (1.f / 4096.f);
#pragma unroll
        for (int x = 0; x < HD / 32; ++x)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                // columns 2c + e of the four column tiles: dimensions 32 x + 4 (2c + e) + 0..3
                float4 v;
                v.x = (o[4 * x][e] + o[4 * x][e + 2]) * f;
                v.y = (o[4 * x + 1][e] + o[4 * x + 1][e + 2]) * f;
                v.z = (o[4 * x + 2][e] + o[4 * x + 2][e + 2]) * f;
                v.w = (o[4 * x + 3][e] + o[4 * x + 3][e + 2]) * f;
                *(float4 *)(mo + g8 * HD + 32 * x + 8 * c + 4 * e) = v;
            }
    } else {
#pragma unroll
        for (int d = 0; d < HD / 8; ++d) {
            *(float2 *)(mo + g8 * HD + 8 * d + 2 * c) = make_float2(o[d][0], o[d][1]);
            *(float2 *)(mo + (g8 + 8) * HD + 8 * d + 2 * c) = make_float2(o[d][2], o[d][3]);
        }
    }
    if constexpr (W == 1)
        __syncwarp();
    else
        __syncthreads();

    const long long nrows = (long long)p.batch * p.tokens * p.heads;
    const bool direct = p.prefix_slots + p.own_slots == 1;
    const char *states = ring - part * G::kWarpBytes;
    for (int i = threadIdx.x % (32 * W); i < rows * (HD / 4); i += 32 * W) {
        const int r = i / (HD / 4), d = 4 * (i % (HD / 4));
        float tops[W], t = kNegInf, total = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            tops[w] = ((const float *)(states + w * G::kWarpBytes) + 16 * HD)[2 * r];
            t = fmaxf(t, tops[w]);
        }
        const float t0 = t == kNegInf ? 0.f : t;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float *q = (const float *)(states + w * G::kWarpBytes);
            const float f = ex2(tops[w] - t0);
            total += f * q[16 * HD + 2 * r + 1];
            const float4 v = *(const float4 *)(q + r * HD + d);
            acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
        }
        const float inv = total > 0.f ? 1.f / total : total == 0.f ? 0.f : total;
        acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
        const float lse = total == 0.f ? kNegInf : t0 + log2f(total);
        const int m = m0 + r, b = m / TR, tt = (m - b * TR) / R, h = g * R + m % R;
        const long long row = ((long long)b * p.tokens + tt) * p.heads + h;
        if (direct) {
            if (tt < own_tokens(p, b)) {
                char *dst = (char *)p.out + (b * p.os[0] + tt * p.os[1] + h * p.os[2] + d) * (I8 ? 4 : 2);
                if constexpr (I8)
                    *(float4 *)dst = acc;
                else
                    *(uint2 *)dst = make_uint2(pack2<BF>(acc.x, acc.y), pack2<BF>(acc.z, acc.w));
                if (d == 0 && p.lse) p.lse[row] = lse * kLn2;
            }
            if (d == 0 && p.neg_lse) p.neg_lse[neg_lse_at(p, b, tt, h)] = -lse;
        } else {
            *(float4 *)(p.part_o + (slot * nrows + row) * HD + d) = acc;
            if (d == 0) p.part_lse[slot * nrows + row] = lse;
        }
    }
}

template <int TYPE, int HD, int W>
__global__ __launch_bounds__(kWarps * 32, HD == 64 ? 4 : 3) void prefix_stream_kernel(
    const __grid_constant__ PrefixAttn p, const __grid_constant__ StreamGrid grid) {
    stream_unit<TYPE, HD, W>(p, grid);
    pdl_enter();   // (at the end: what follows this kernel follows the tile kernel beside it too)
}

// ---- merge -----------------------------------------------------------------

// HD / 4 threads a row: the weighted sum of the row's partial results.  Bound by
// their bytes, mostly out of L2: 4096 rows of 128 dimensions with 10 each (21 MB)
// 5.8 us.
template <int TYPE, int HD>
__device__ __forceinline__ void merge_row(const PrefixAttn &p, long long row, int part) {
    constexpr bool I8 = TYPE == kCacheI8, BF = TYPE == kCacheBF16;
    const long long nrows = (long long)p.batch * p.tokens * p.heads;
    const int slots = p.prefix_slots + p.own_slots;
    const int h = (int)(row % p.heads);
    const long long bt = row / p.heads;
    const int t = (int)(bt % p.tokens), b = (int)(bt / p.tokens);
    if (t >= own_tokens(p, b)) return;
    // four partial results in flight at a time, merged as they come (o of an empty
    // range was not written: it is read and not used)
    float top = kNegInf, total = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < slots; i += 4) {
        float l[4];
        float4 v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            l[e] = i + e < slots ? p.part_lse[(i + e) * nrows + row] : kNegInf;
            v[e] = *(const float4 *)(p.part_o + (min(i + e, slots - 1) * nrows + row) * HD + part);
        }
        const float now = fmaxf(max3(top, l[0], l[1]), fmaxf(l[2], l[3]));
        const float base = now == kNegInf ? 0.f : now, keep = ex2(top - base);
        total *= keep;
        acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
        top = now;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (l[e] == kNegInf) continue;
            const float f = ex2(l[e] - base);
            total += f;
            acc.x += f * v[e].x; acc.y += f * v[e].y; acc.z += f * v[e].z; acc.w += f * v[e].w;
        }
    }
    const float t0 = top == kNegInf ? 0.f : top;
    const float inv = total == 0.f ? 0.f : 1.f / total;
    acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
    char *dst = (char *)p.out + (b * p.os[0] + t * p.os[1] + h * p.os[2] + part) * (I8 ? 4 : 2);
    if constexpr (I8)
        *(float4 *)dst = acc;
    else
        *(uint2 *)dst = make_uint2(pack2<BF>(acc.x, acc.y), pack2<BF>(acc.z, acc.w));
    if (part == 0) {
        const float lse = total == 0.f ? kNegInf : t0 + log2f(total);
        if (p.lse) p.lse[row] = lse * kLn2;
        if (p.neg_lse) p.neg_lse[neg_lse_at(p, b, t, h)] = -lse;
    }
}

constexpr int kWeightKeys = 512;   // keys of one CTA of the weights from kept logits

template <int TYPE, int HD>
__global__ __launch_bounds__(128) void prefix_finish_kernel(const PrefixAttn p, int merge_blocks) {
    pdl_enter();
    const long long nrows = (long long)p.batch * p.tokens * p.heads;
    constexpr int kPer = 128 / (HD / 4);
    if ((int)blockIdx.x < merge_blocks) {
        const long long row = (long long)blockIdx.x * kPer + threadIdx.x / (HD / 4);
        if (row < nrows) merge_row<TYPE, HD>(p, row, 4 * (threadIdx.x % (HD / 4)));
        return;
    }
    // weights of sequence b, KV head g, from the kept logits of its rows
    const int chunks = ceil_div(p.capacity, kWeightKeys);
    int unit = blockIdx.x - merge_blocks;
    const int chunk = unit % chunks;
    unit /= chunks;
    const int g = unit % p.kvheads, b = unit / p.kvheads, TR = p.tokens * p.group;
    __shared__ float lse[kMaxLogitRows];
    const int len = own_length(p, b), nq = own_tokens(p, b);
    if ((int)threadIdx.x < TR) {
        const int t = threadIdx.x / p.group, h = g * p.group + threadIdx.x % p.group;
        const long long row = ((long long)b * p.tokens + t) * p.heads + h;
        const int slots = p.prefix_slots + p.own_slots;
        float l = 0.f;
        if (t < nq) {
            if (slots == 1) {
                l = -p.neg_lse[neg_lse_at(p, b, t, h)];
            } else {
                float top = kNegInf, total = 0.f;
                for (int i = 0; i < slots; i += 4) {       // four in flight at a time
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = i + e < slots ? p.part_lse[(i + e) * nrows + row] : kNegInf;
                    const float now = fmaxf(max3(top, x[0], x[1]), fmaxf(x[2], x[3]));
                    const float base = now == kNegInf ? 0.f : now;
                    total *= ex2(top - base);
                    top = now;
#pragma unroll
                    for (int e = 0; e < 4; ++e) total += ex2(x[e] - base);
                }
                l = total == 0.f ? 0.f : (top == kNegInf ? 0.f : top) + log2f(total);
            }
            if (l == kNegInf) l = 0.f;
        }
        lse[threadIdx.x] = l;
    }
    __syncthreads();
    const float *z = p.logits + (long long)(b * p.kvheads + g) * TR * p.capacity;
    const float *win = p.weights + b * p.ws[0] + g * p.ws[1];
    float *wout = p.weights_out + b * p.wos[0] + g * p.wos[1];
    // kWeightKeys / 128 keys of a thread, their loads in flight together
    constexpr int kMine = kWeightKeys / 128;
    const int j0 = chunk * kWeightKeys + threadIdx.x, past = len - nq;
    float w[kMine], old[kMine];
#pragma unroll
    for (int e = 0; e < kMine; ++e) {
        const int j = j0 + e * 128;
        old[e] = j < p.capacity ? win[j * p.ws[2]] : 0.f;
        w[e] = 0.f;
    }
#pragma unroll 2
    for (int r = 0; r < nq * p.group; ++r) {
        const int i = past + r / p.group;             // own index of the row's query
        const int from = p.window ? i - p.window + 1 : 0;
        float x[kMine];
#pragma unroll
        for (int e = 0; e < kMine; ++e) {
            const int j = j0 + e * 128;
            x[e] = j <= i && j >= from ? z[(long long)r * p.capacity + j] : kNegInf;
        }
#pragma unroll
        for (int e = 0; e < kMine; ++e) w[e] += ex2(x[e] - lse[r]);
    }
#pragma unroll
    for (int e = 0; e < kMine; ++e) {
        const int j = j0 + e * 128;
        if (j < p.capacity) wout[j * p.wos[2]] = old[e] + w[e];
    }
}

// ---- weights of any number of rows -----------------------------------------
//
// Keys are the rows of the product K Q^T: a warp holds 16 keys as the A operand
// and walks the sequence's query rows, eight columns at a time, adding
// 2^(z - L_row) of the rows that see the key.  Only for more query heads a KV head
// than a tile of the tensor-core kernel has rows (it took 3200 us for two prompts
// of 4096 tokens, the tiles take 182), for 16-bit queries of strides that the copy
// engine does not take (expanded ones), and to copy the weights of calls without
// tokens.

template <int TYPE, int HD>
__global__ __launch_bounds__(128) void key_weights_kernel(const PrefixAttn p) {
    pdl_enter();
    constexpr bool I8 = TYPE == kCacheI8, BF = TYPE == kCacheBF16;
    constexpr int KS = HD / 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, c = lane & 3;
    const int chunks = ceil_div(p.capacity, 64), unit = blockIdx.x / chunks;
    const int g = unit % p.kvheads, b = unit / p.kvheads;
    const int key0 = (blockIdx.x % chunks * 4 + warp) * 16, TR = p.tokens * p.group;
    if (key0 >= p.capacity) return;
    const int len = own_length(p, b), nq = own_tokens(p, b);
    const long long crow = p.cache_row ? p.cache_row[b] : b;
    float sum[2] = {0.f, 0.f};
    if (key0 < len && nq > 0) {
        uint32_t ka[KS][4];
        float ks[2] = {p.scale2, p.scale2};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const long long j = min(key0 + g8 + 8 * e, len - 1);
            const char *row = (const char *)p.k + (crow * p.ks[0] + g * p.ks[1] + j * p.ks[2]) * (I8 ? 1 : 2);
            if constexpr (I8) {
                ks[e] *= p.kscale[crow * p.kss[0] + g * p.kss[1] + j * p.kss[2]];
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    const uint32_t u = *(const uint32_t *)(row + 64 * (k / 4) + 16 * c + 4 * (k % 4)) ^ 0x80808080u;
                    ka[k][e] = i8x2_to_f16<0x4140>(u);
                    ka[k][e + 2] = i8x2_to_f16<0x4342>(u);
                }
            } else {
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    ka[k][e] = *(const uint32_t *)(row + (16 * k + 2 * c) * 2);
                    ka[k][e + 2] = *(const uint32_t *)(row + (16 * k + 2 * c + 8) * 2);
                }
            }
        }
        // the first query that sees key0, the last that sees key0 + 15
        const int t0 = max(0, key0 - (len - nq));
        const int t1 = p.window ? min((long long)nq, (long long)key0 + 15 + p.window - (len - nq)) : nq;
        for (int m = t0 * p.group / 8 * 8; m < t1 * p.group; m += 8) {
            const int r = min(m + g8, TR - 1), t = r / p.group, h = g * p.group + r % p.group;
            const char *q = (const char *)p.q + (b * p.qs[0] + t * p.qs[1] + h * p.qs[2]) * (I8 ? 4 : 2);
            float z[4] = {0.f, 0.f, 0.f, 0.f};
            float down = 1.f;
            if constexpr (I8) {
                float x[KS][4], most = 0.f;
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[k][e] = ((const float *)q)[64 * (k / 4) + 16 * c + 4 * (k % 4) + e];
                        most = fmaxf(most, fabsf(x[k][e]));
                    }
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                float up;
                row_scale(most, up, down);
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    uint32_t h0, l0, h1, l1;
                    split2(x[k][0] * up, x[k][1] * up, h0, l0);
                    split2(x[k][2] * up, x[k][3] * up, h1, l1);
                    mma16816<false>(z, ka[k], h0, h1);
                    mma16816<false>(z, ka[k], l0, l1);
                }
            } else {
#pragma unroll
                for (int k = 0; k < KS; ++k)
                    mma16816<BF>(z, ka[k], *(const uint32_t *)(q + (16 * k + 2 * c) * 2),
                                 *(const uint32_t *)(q + (16 * k + 2 * c + 8) * 2));
            }
            // columns 2c, 2c + 1: rows m + 2c + x
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const float dn = __shfl_sync(0xffffffffu, down, 4 * (2 * c + x));
                const int r2 = m + 2 * c + x, t2 = r2 / p.group;
                if (r2 < nq * p.group) {
                    const float l = p.neg_lse[((long long)b * p.kvheads + g) * TR + r2];
                    const int i = len - nq + t2;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int j = key0 + g8 + 8 * e;
                        if (j <= i && (!p.window || j > i - p.window))
                            sum[e] += ex2(z[2 * e + x] * (ks[e] * dn) + l);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 1);
        sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 2);
        const long long j = key0 + g8 + 8 * e;
        if (c == 0 && j < p.capacity)
            p.weights_out[b * p.wos[0] + g * p.wos[1] + j * p.wos[2]] =
                p.weights[b * p.ws[0] + g * p.ws[1] + j * p.ws[2]] + sum[e];
    }
}

}  // namespace

bool launch_prefix_stream(const PrefixAttn &p, bool prefix, bool own, bool joint, bool after_tiles, cudaStream_t st) {
    return by_geometry(p, [&](auto type, auto hd) -> bool {
        using G = StreamGeom<type(), hd()>;
        StreamGrid grid{};
        const int rows = p.tokens * p.group;
        grid.own_slots = std::max(1, p.own_slots);
        grid.prefix_slots = std::max(1, p.prefix_slots);
        grid.own_tiles = ceil_div(rows, G::kRows);
        grid.prefix_tiles = ceil_div(p.batch * rows, G::kRows);
        grid.joint = joint;
        grid.own_units = own ? p.batch * p.kvheads * grid.own_tiles * grid.own_slots : 0;
        grid.prefix_units = prefix ? p.kvheads * grid.prefix_tiles * grid.prefix_slots : 0;
        const int units = grid.own_units + grid.prefix_units;
        if (units == 0) return true;
        auto launch = [&](auto warps) -> bool {
            auto kernel = prefix_stream_kernel<type(), hd(), warps()>;
            static bool configured[64] = {};
            int dev = 0;
            NB_CUDA_TRY(cudaGetDevice(&dev));
            if (dev < 0 || dev >= 64 || !configured[dev]) {
                NB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmem));
                if (dev >= 0 && dev < 64) configured[dev] = true;
            }
            const int blocks = ceil_div(units, kWarps / warps());
            if (after_tiles) {
                NB_CUDA_TRY(launch_pdl(kernel, dim3(blocks), dim3(kWarps * 32), (size_t)G::kSmem, st, p, grid));
            } else {
                kernel<<<blocks, kWarps * 32, G::kSmem, st>>>(p, grid);
                NB_CUDA_TRY(cudaGetLastError());
            }
            return true;
        };
        const int span = p.window ? std::min<long long>(p.capacity, (long long)p.window + p.tokens) : p.capacity;
        const int longest = std::max(own ? ceil_div(span, grid.own_slots) + (joint ? p.prefix : 0) : 0,
                                     prefix ? ceil_div(p.prefix, grid.prefix_slots) : 0);
        // one warp a unit on short ranges, and on longer ones where the units are many
        const bool alone = longest <= kShortRange || (longest <= 4 * kShortRange && units >= kManyUnits);
        return alone ? launch(std::integral_constant<int, 1>()) : launch(std::integral_constant<int, kWarps>());
    });
}

bool launch_prefix_finish(const PrefixAttn &p, cudaStream_t st) {
    return by_geometry(p, [&](auto type, auto hd) -> bool {
        const long long rows = (long long)p.batch * p.tokens * p.heads;
        const int merge = p.prefix_slots + p.own_slots > 1 ? (int)((rows + 512 / hd() - 1) / (512 / hd())) : 0;
        const int weights = p.logits ? p.batch * p.kvheads * ceil_div(p.capacity, kWeightKeys) : 0;
        if (merge + weights == 0) return true;
        NB_CUDA_TRY(launch_pdl(prefix_finish_kernel<type(), hd()>, dim3(merge + weights), dim3(128), 0, st, p, merge));
        return true;
    });
}

bool launch_key_weights(const PrefixAttn &p, cudaStream_t st) {
    return by_geometry(p, [&](auto type, auto hd) -> bool {
        const dim3 grid(ceil_div(p.capacity, 64) * p.batch * p.kvheads);
        if (grid.x == 0) return true;
        NB_CUDA_TRY(launch_pdl(key_weights_kernel<type(), hd()>, grid, dim3(128), 0, st, p));
        return true;
    });
}

}  // namespace nb200
