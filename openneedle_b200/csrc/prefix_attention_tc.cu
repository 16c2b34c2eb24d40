// Shared-prefix attention on the sm_100a tensor cores, for many query rows per
// KV head: the whole batch's rows against the prefix, a sequence's rows of a
// chunk or prompt against its own keys.  Formulas and the row and
// partial-result conventions: prefix_attention.cuh.
//
// One CTA attends up to 256 rows (two tiles of 128) to one key range, 128 keys at
// a time.  A warp feeds K and V by TMA, one thread issues the products S = Q K^T
// (into TMEM) and O += P V (P from TMEM, V from shared memory), and each tile has
// a warpgroup whose thread i owns row i: it reads its 128 logits back, keeps the
// row's maximum and sum in registers, writes the weights over the logits (the
// first half's product starts while the second is computed) and, where the
// maximum grew by more than 2^8, rescales its row of O.  While one tile is in its
// softmax the tensor core works for the other.  TMEM holds the two tiles' O and
// two (128 dimensions) or three (64) buffers of logits; with three, a tile's next
// logits are computed during its softmax.  Up to 128 rows run with both tiles on
// the same rows and alternate key steps, as two key ranges.
//
// Two prompts of 4096 tokens, 32 heads, 128 dimensions, causal: 340 us, 810 TFLOP/s
// (bf16).  A step of 128 keys takes about 3500 cycles: the products 2200 (a product
// S of 128 columns 80 cycles an instruction rather than 64, as both operands come
// from shared memory), a tile's softmax 1700, of which the exponentials 1000, and the
// chain softmax - O - next logits leaves the tensor core idle in between, as TMEM has
// no room for another buffer beside two O of 128 columns.  Steps of 64 keys with four
// buffers took 480 us (a product of 64 columns takes nearly the time of one of 128),
// four warpgroups of softmax 345, a part of the exponentials as polynomials on the
// FP32 pipe 347 to 362.  Short calls pay about 9 us a CTA beside its steps: queries,
// first copies, and the output (a 16k document asked about by 128 users: 47 us for
// 15 steps).
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "pdl.cuh"
#include "prefix_attention.cuh"
#include "tile_math.cuh"

namespace nb200 {
namespace {

using namespace tile;

__device__ int g_tile_fault = 0;                 // a bounded wait ran out

constexpr float kGrow = 8.f;                     // log2 growth of a maximum that is left to the weights

constexpr int kStep = 128;                       // keys of a step
constexpr int kTileThreads = 384;                // two warpgroups of rows, one of products, copies, conversions
constexpr int kMathWarps = 8, kProductWarp = 8, kCopyWarp = 9, kConvertWarp = 10;
// 2 * 128 * 208 + 128 * 88 = 384 * 168
constexpr int kMathRegisters = 208, kOtherRegisters = 88;

template <int TYPE, int HD>
struct TileGeom {
    static constexpr bool I8 = TYPE == kCacheI8;
    static constexpr int kPieces = I8 ? 2 : 1;                    // FP32 queries and weights as FP16 pairs
    static constexpr int kQBytes = kTile * HD * 2;                // a piece of a tile of queries
    static constexpr int kKVBytes = kStep * HD * 2;               // a step's K or V in 16 bits
    // the FP32 queries' pairs of two 128-dimension tiles would fill the shared memory
    static constexpr int kQTiles = I8 && HD == 128 ? 1 : 2;
    static constexpr int kStages = HD == 64 ? (I8 ? 4 : 6) : (I8 ? 3 : 4);
    static constexpr int kBuffers = HD == 64 ? 3 : 2;             // of logits
    // whether a step's K can be there before the weights of kBuffers items earlier
    static constexpr bool kEarly = kStages >= (kBuffers == 3 ? 6 : 4);
    static constexpr int kRaw = I8 ? (HD == 64 ? 4 : 2) : 0;      // INT8 steps on their way
    static constexpr int kRawBytes = kStep * HD;
    static constexpr int kScaleRing = 8;                          // steps whose scales are held
    static constexpr int kRing = kQTiles * kPieces * kQBytes;
    static constexpr int kRawAt = kRing + kStages * kKVBytes;
    static constexpr int kScaleAt = kRawAt + kRaw * kRawBytes;
    static constexpr int kSmem = kScaleAt + (I8 ? kScaleRing * 2 * kStep * 4 : 0) + 1024;
    static constexpr int kConverters = I8 ? 2 : 0;                // warps
    // A product's sums are cut to 24 bits towards zero, 16 times a step for the pairs: O
    // shrinks by up to 2^-19 a step. So after every kHold steps it is added to sums that the
    // row's thread holds (in local memory), and starts at zero. 16000 shared keys, 1200
    // tokens, 64 / 128 dimensions: 9e-6 / 14e-6 off in 183 / 459 us without, 0.8e-6 / 1.0e-6
    // in 174 / 452 so (elementary operations in 32 bits: 2.4e-6); 2 steps for 128
    // dimensions: 0.8e-6 in 471. 16-bit outputs need it only after many more keys: ranges.
    static constexpr int kHold = HD == 64 ? 2 : 3;
    static_assert(kSmem <= 232448 - 4096, "shared memory of a CTA");
    // a step's scales are written when the stage of the K kStages / 2 steps before is
    // free, at which time softmaxes of the kBuffers - 1 steps before that may be running
    static_assert(kScaleRing >= kStages / 2 + kBuffers, "scales in use");
};

// The buffers of logits in turn, and the phase of their barriers.
struct Turn {
    int buffer = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void on(int items, int buffers) {
        for (buffer += items; buffer >= buffers; buffer -= buffers) phase ^= 1;
    }
};

// Units of work: (range, row tiles, KV head[, sequence]).
struct TileGrid {
    int own_units, own_tiles, own_ranges, own_alt, own_rows;          // rows of a unit
    int prefix_units, prefix_tiles, prefix_ranges, prefix_alt, prefix_rows;
    int stream_next, prefix_first;
    int joint;                                                        // own units take the prefix first
    // whether the cache's head and sequence axes advance in the tensor maps
    int k_head, k_seq, v_head, v_seq, pk_head, pv_head;
};

template <int TYPE, int HD>
__global__ __launch_bounds__(kTileThreads, 1) void prefix_tile_kernel(
    const PrefixAttn p, const TileGrid grid, const __grid_constant__ CUtensorMap mk,
    const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mpk,
    const __grid_constant__ CUtensorMap mpv) {
    using G = TileGeom<TYPE, HD>;
    constexpr bool I8 = G::I8, BF = TYPE == kCacheBF16;
    constexpr int kStages = G::kStages;
    extern __shared__ __align__(16) char smem_raw[];
    char *smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    char *ring = smem + G::kRing;
    float *scales = (float *)(smem + G::kScaleAt);               // [kScaleRing][K, V][kStep]
    __shared__ __align__(8) uint64_t full[kStages], empty[kStages], raw_full[4], raw_empty[4];
    __shared__ __align__(8) uint64_t s_full[3], p_full[3][2], o_done[2], o_full[2], q_full, drained;
    __shared__ float qscale[I8 ? 256 : 1];
    __shared__ float vmost[G::kScaleRing][2];
    __shared__ const char *qrow[256];
    __shared__ uint32_t tmem_at;
    __shared__ int abort_at;
    volatile int *abort_flag = &abort_at;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // the unit
    const int R = p.group, TR = p.tokens * R;
    // the units with more steps come first, so that the last wave holds the short ones
    int unit = grid.prefix_first ? (int)blockIdx.x - grid.prefix_units : blockIdx.x;
    if (unit < 0) unit += grid.own_units + grid.prefix_units;
    int g, m0, rows, lo, hi, slot, seq = -1, len = 0, nq = 0, alt;
    const float *ksc = nullptr, *vsc = nullptr;
    long long ksc_step = 0, vsc_step = 0;
    int kz, kw, vz, vw, before = 0;                              // before: steps of the prefix ahead of [lo, hi)
    const CUtensorMap *km, *vm;
    if (unit < grid.own_units) {
        alt = grid.own_alt;
        slot = unit % grid.own_ranges;
        unit /= grid.own_ranges;
        // later tokens see more keys: their units first
        const int tile = grid.own_tiles - 1 - unit % grid.own_tiles;
        unit /= grid.own_tiles;
        g = unit % p.kvheads;
        seq = unit / p.kvheads;
        m0 = seq * TR + tile * grid.own_rows;
        rows = min(grid.own_rows, TR - tile * grid.own_rows);
        len = own_length(p, seq);
        nq = own_tokens(p, seq);
        const int t0 = tile * grid.own_rows / R, t1 = min((tile * grid.own_rows + rows - 1) / R, nq - 1);
        hi = max(0, min(len, len - nq + t1 + 1));
        lo = p.window ? max(0, len - nq + t0 - p.window + 1) : 0;
        if (t0 >= nq) rows = 0;
        const int n = max(0, hi - lo), each = (ceil_div(n, grid.own_ranges) + kStep - 1) / kStep * kStep;
        const int a = min(hi, lo + slot * each);
        hi = min(hi, a + each);
        lo = a;
        slot = p.prefix_slots + (alt ? 2 * slot : slot);
        const int row = p.cache_row ? p.cache_row[seq] : seq;
        km = &mk;
        vm = &mv;
        kz = g * grid.k_head; kw = row * grid.k_seq; vz = g * grid.v_head; vw = row * grid.v_seq;
        if constexpr (I8) {
            ksc = p.kscale + (long long)row * p.kss[0] + g * p.kss[1];
            vsc = p.vscale + (long long)row * p.vss[0] + g * p.vss[1];
            ksc_step = p.kss[2];
            vsc_step = p.vss[2];
        }
        if (grid.joint) before = ceil_div(p.prefix, kStep);
    } else {
        alt = grid.prefix_alt;
        unit -= grid.own_units;
        slot = unit % grid.prefix_ranges;
        unit /= grid.prefix_ranges;
        const int tile = unit % grid.prefix_tiles;
        g = unit / grid.prefix_tiles;
        m0 = tile * grid.prefix_rows;
        rows = min(grid.prefix_rows, p.batch * TR - m0);
        const int each = (ceil_div(p.prefix, grid.prefix_ranges) + kStep - 1) / kStep * kStep;
        lo = min(p.prefix, slot * each);
        hi = min(p.prefix, lo + each);
        slot = alt ? 2 * slot : slot;
        km = &mpk;
        vm = &mpv;
        kz = g * grid.pk_head; kw = 0; vz = g * grid.pv_head; vw = 0;
        if constexpr (I8) {
            ksc = p.pkscale + g * p.pkss[0];
            vsc = p.pvscale + g * p.pvss[0];
            ksc_step = p.pkss[1];
            vsc_step = p.pvss[1];
        }
    }
    // the streaming kernel of the same call works on other keys: it may start on the
    // multiprocessors that have no tile CTA, or none left (a tile CTA has 64512 of one's 65536
    // registers: the two never share one)
    if (grid.stream_next) pdl_launch_dependents();
    if (rows <= 0) return;                        // the whole CTA
    const int n = before + ceil_div(max(0, hi - lo), kStep);     // steps of keys
    const int tiles = alt ? 1 : (rows > kTile ? 2 : 1);          // row tiles
    // item k: step and tile; its logits in buffer k % ahead, so that they follow the
    // output product of the item `ahead` before: one of its tile's last two, and the
    // products of its tile's items before that have ended when they are there
    const int each = alt ? 1 : tiles, items = n * each, ahead = alt || tiles == 2 ? G::kBuffers : 2;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&full[i], I8 ? 32 * G::kConverters : 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < G::kRaw; ++i) {
            mbar_init(&raw_full[i], 1);
            mbar_init(&raw_empty[i], 32 * G::kConverters);
        }
        for (int i = 0; i < 3; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i][0], kTile);
            mbar_init(&p_full[i][1], kTile);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&o_done[i], 1);
            mbar_init(&o_full[i], 1);
        }
        mbar_init(&q_full, 32 * kMathWarps);
        mbar_init(&drained, 1);
        abort_at = 0;
        fence_barrier_init();
    }
    if (warp == kProductWarp) tc::alloc(&tmem_at, 512);

    for (int r = threadIdx.x; r < tiles * kTile; r += kTileThreads) {
        const int m = m0 + r, b = m / TR, t = (m - b * TR) / R, h = g * R + m % R;
        qrow[r] = r < rows ? (const char *)p.q + (b * p.qs[0] + t * p.qs[1] + h * p.qs[2]) * (I8 ? 4 : 2) : nullptr;
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_at;

    if (warp >= kMathWarps) {
        fewer_registers<kOtherRegisters>();
        if (warp == kCopyWarp) {
            // ---- copies: tile j's K, then its V
            if (lane == 0) {
                int issued = 0;
                for (int i = 0; i < 2 * n; ++i) {
                    const bool shared = (i >> 1) < before, v = i & 1;
                    const CUtensorMap *map = shared ? (v ? &mpv : &mpk) : (v ? vm : km);
                    const int key = shared ? (i >> 1) * kStep : lo + ((i >> 1) - before) * kStep;
                    const int z = shared ? g * (v ? grid.pv_head : grid.pk_head) : (v ? vz : kz);
                    const int w = shared ? 0 : (v ? vw : kw);
                    if constexpr (I8) {
                        const int s = i % G::kRaw;
                        if (i >= G::kRaw && !wait_phase(&raw_empty[s], (uint32_t)(i / G::kRaw - 1) & 1, abort_flag))
                            break;
                        mbar_arrive_expect_tx(&raw_full[s], G::kRawBytes);
                        tma_load_4d(smem + G::kRawAt + s * G::kRawBytes, map, 0, key, z, w, &raw_full[s]);
                    } else {
                        const int s = i % kStages;
                        if (i >= kStages && !wait_phase(&empty[s], (uint32_t)(i / kStages - 1) & 1, abort_flag)) break;
                        mbar_arrive_expect_tx(&full[s], G::kKVBytes);
    #pragma unroll
                        for (int c = 0; c < HD / 64; ++c)
                            tma_load_4d(ring + s * G::kKVBytes + c * (kStep * 128), map, 64 * c, key, z, w, &full[s]);
                    }
                    ++issued;
                }
                // no copy is in flight when the CTA ends, whatever became of its consumers
                constexpr int kDepth = I8 ? G::kRaw : kStages;
                for (int i = max(0, issued - kDepth); i < issued; ++i)
                    mbar_wait(I8 ? &raw_full[i % kDepth] : &full[i % kDepth], (uint32_t)(i / kDepth) & 1);
            }
            __syncwarp();
        } else if (warp == kProductWarp) {
            // ---- products
            const uint32_t q0 = smem_addr(smem), r0 = smem_addr(ring), s0 = tmem + 2 * HD;
            constexpr uint32_t ids = idesc(BF, false, kStep), ido = idesc(BF, true, HD);
            auto step_of = [&](int k) { return each == 2 ? k >> 1 : k; };
            auto tile_of = [&](int k) { return alt || each == 2 ? k & 1 : 0; };
            auto have = [&](int i) { wait_phase(&full[i % kStages], (uint32_t)(i / kStages) & 1, abort_flag); };
            auto logits = [&](int k, int buffer) {        // S_k = Q K^T
                const int i = 2 * step_of(k), w = tile_of(k);
                const uint32_t kt = r0 + (i % kStages) * G::kKVBytes;
                const uint32_t q = q0 + (alt ? 0 : w) * (G::kPieces * G::kQBytes);
                __syncwarp();
                if (elect_one()) {
                    tc::fence_after();
#pragma unroll
                    for (int x = 0; x < G::kPieces; ++x)
#pragma unroll
                        for (int c = 0; c < HD / 16; ++c)
                            // (INT8: the small lo pieces first, the sum grows last)
                            tc::mma_bf16_ss(s0 + buffer * kStep,
                                            desc_k(q + (G::kPieces - 1 - x) * G::kQBytes + (c / 4) * (kTile * 128) +
                                                   (c % 4) * 32),
                                            desc_k(kt + (c / 4) * (kStep * 128) + (c % 4) * 32), ids, x + c > 0);
                    tc::commit(&s_full[buffer]);
                    if (each == 1 || w == 1) tc::commit(&empty[i % kStages]);
                }
                __syncwarp();
            };
            auto values = [&](int k, int buffer, int half) {   // O += P_k V, half of the keys
                const int i = 2 * step_of(k) + 1, w = tile_of(k);
                const uint32_t v = r0 + (i % kStages) * G::kKVBytes, pk = s0 + buffer * kStep;
                const bool first = k < (alt ? 2 : each) && half == 0;
                __syncwarp();
                if (elect_one()) {
                    tc::fence_after();
#pragma unroll
                    for (int x = 0; x < G::kPieces; ++x)
#pragma unroll
                        for (int e = 0; e < kStep / 32; ++e) {
                            const int c = half * (kStep / 32) + e;
                            // 32 keys take 32 columns: 16 of their weights (hi), 16 of lo
                            mma_ts(tmem + w * HD, pk + 32 * (c >> 1) + 8 * (c & 1) + 16 * x,
                                   desc_mn<kStep>(v + c * 2048), ido, !first || x + e > 0);
                        }
                    if (half) {
                        tc::commit(&o_done[w]);
                        if (k + (alt ? 2 : each) >= items) tc::commit(&o_full[w]);
                        if (each == 1 || w == 1) tc::commit(&empty[i % kStages]);
                    }
                }
                __syncwarp();
            };
            auto have_v = [&](int j) {
                have(2 * j + 1);
                const int valid = j < before ? p.prefix - j * kStep : hi - lo - (j - before) * kStep;
                if (!I8 && valid < kStep) {               // rows behind the range: whatever they hold, zeros
                    char *v = ring + ((2 * j + 1) % kStages) * G::kKVBytes;
                    for (int i = valid * 8 + lane; i < kStep * 8; i += 32)
#pragma unroll
                        for (int c = 0; c < HD / 64; ++c)
                            *(uint4 *)(v + c * (kStep * 128) + i * 16) = make_uint4(0, 0, 0, 0);
                    fence_proxy_async();
                }
                __syncwarp();
            };
            if (n > 0) wait_phase(&q_full, 0, abort_flag);
            for (int k = 0; k < min(items, ahead); ++k) {
                have(2 * step_of(k));
                logits(k, k);
            }
            Turn turn;
            for (int k = 0; k < items; ++k) {
                const bool more = k + ahead < items;
                if (each == 1 || !(k & 1)) have_v(step_of(k));
                if (G::kEarly && more) have(2 * step_of(k + ahead));
                wait_phase(&p_full[turn.buffer][0], turn.phase, abort_flag);
                values(k, turn.buffer, 0);
                wait_phase(&p_full[turn.buffer][1], turn.phase, abort_flag);
                values(k, turn.buffer, 1);
                if (more) {
                    if (!G::kEarly) have(2 * step_of(k + ahead));
                    logits(k + ahead, turn.buffer);
                }
                turn.on(1, ahead);
            }
            __syncwarp();
            if (__any_sync(0xffffffffu, *abort_flag)) {   // no product is in flight when TMEM is freed
                if (elect_one()) tc::commit(&drained);
                mbar_wait(&drained, 0);
                __syncwarp();
            }
        } else if (warp >= kConvertWarp) {
            // ---- INT8 tiles to FP16, exactly
            if constexpr (I8) {
                const int me = threadIdx.x - 32 * kConvertWarp;
                constexpr int kN = 32 * G::kConverters, kChunks = HD / 16;
                for (int i = 0; i < 2 * n; ++i) {
                    const int s = i % kStages, rs = i % G::kRaw, j = i >> 1;
                    if (!(i & 1)) {
                        // both scales of the step's keys (V's zero behind the range), and V's largest
                        float *sk = scales + (j % G::kScaleRing) * 2 * kStep, most = 0.f;
                        float kx[kStep / kN], vx[kStep / kN];
    #pragma unroll
                        for (int e = 0; e < kStep / kN; ++e) {
                            const int x = me + e * kN;
                            if (j < before) {
                                const int key = j * kStep + x;
                                kx[e] = key < p.prefix ? p.pkscale[g * p.pkss[0] + key * p.pkss[1]] : 0.f;
                                vx[e] = key < p.prefix ? p.pvscale[g * p.pvss[0] + key * p.pvss[1]] : 0.f;
                            } else {
                                const int key = lo + (j - before) * kStep + x;
                                kx[e] = key < hi ? ksc[key * ksc_step] : 0.f;
                                vx[e] = key < hi ? vsc[key * vsc_step] : 0.f;
                            }
                            most = fmaxf(most, fabsf(vx[e]));
                        }
#pragma unroll
                        for (int d = 16; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
                        if (i >= kStages) wait_phase(&empty[s], (uint32_t)(i / kStages - 1) & 1, abort_flag);
    #pragma unroll
                        for (int e = 0; e < kStep / kN; ++e) {
                            sk[me + e * kN] = kx[e];
                            sk[kStep + me + e * kN] = vx[e];
                        }
                        if (lane == 0) vmost[j % G::kScaleRing][warp - kConvertWarp] = most;
                    } else if (i >= kStages) {
                        wait_phase(&empty[s], (uint32_t)(i / kStages - 1) & 1, abort_flag);
                    }
                    wait_phase(&raw_full[rs], (uint32_t)(i / G::kRaw) & 1, abort_flag);
                    const char *src = smem + G::kRawAt + rs * G::kRawBytes;
                    char *dst = ring + s * G::kKVBytes;
    #pragma unroll 4
                    for (int x = me; x < kStep * kChunks; x += kN) {
                        const int r = x / kChunks, c = x % kChunks;
                        uint4 a, b;
                        i8x16_to_f16(*(const uint4 *)(src + x * 16), a, b);
                        *(uint4 *)(dst + piece_at<kStep>(r, 2 * c)) = a;
                        *(uint4 *)(dst + piece_at<kStep>(r, 2 * c + 1)) = b;
                    }
                    fence_proxy_async();
                    mbar_arrive(&raw_empty[rs]);
                    mbar_arrive(&full[s]);
                }
            }
        }
    } else {
        more_registers<kMathRegisters>();
        // the queries, in the products' layout; rows that do not exist are zeros
        constexpr int kN = 32 * kMathWarps;
        if constexpr (I8) {
            // HD / 4 lanes a row, four rows of each lane in flight
            constexpr int kLanes = HD / 4, kPer = kN / kLanes;
            const int l = threadIdx.x % kLanes;
            for (int r0 = threadIdx.x / kLanes; r0 < tiles * kTile; r0 += 4 * kPer) {
                float4 x[4];
    #pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = r0 + e * kPer;
                    const char *q = r < tiles * kTile ? qrow[r] : nullptr;
                    x[e] = q ? *(const float4 *)(q + l * 16) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
    #pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = r0 + e * kPer;
                    float most = fmaxf(fmaxf(fabsf(x[e].x), fabsf(x[e].y)), fmaxf(fabsf(x[e].z), fabsf(x[e].w)));
    #pragma unroll
                    for (int d = kLanes / 2; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
                    float up, down;
                    row_scale(most, up, down);
                    uint2 h, lo2;
                    split2(x[e].x * up, x[e].y * up, h.x, lo2.x);
                    split2(x[e].z * up, x[e].w * up, h.y, lo2.y);
                    if (r < tiles * kTile) {
                        if (l == 0) qscale[r] = p.scale2 * down;
                        char *q = smem + (r / kTile) * 2 * G::kQBytes + piece_at<kTile>(r % kTile, l / 2) + (l & 1) * 8;
                        *(uint2 *)q = h;
                        *(uint2 *)(q + G::kQBytes) = lo2;
                    }
                }
            }
        } else {
            constexpr int kChunks = HD / 8, kPer = kN / kChunks;
            const int c = threadIdx.x % kChunks;
            for (int r0 = threadIdx.x / kChunks; r0 < tiles * kTile; r0 += 6 * kPer) {
                uint4 x[6];
    #pragma unroll
                for (int e = 0; e < 6; ++e) {
                    const int r = r0 + e * kPer;
                    const char *q = r < tiles * kTile ? qrow[r] : nullptr;
                    x[e] = q ? *(const uint4 *)(q + c * 16) : make_uint4(0, 0, 0, 0);
                }
    #pragma unroll
                for (int e = 0; e < 6; ++e) {
                    const int r = r0 + e * kPer;
                    if (r < tiles * kTile)
                        *(uint4 *)(smem + (r / kTile) * G::kQBytes + piece_at<kTile>(r % kTile, c)) = x[e];
                }
            }
        }
        fence_proxy_async();
        mbar_arrive(&q_full);

        // ---- softmax: thread = row
        const int w = warp >> 2, r = threadIdx.x & (kTile - 1);
        const int mine = alt ? (n - w + 1) >> 1 : (w < tiles ? n : 0);   // steps of this tile
        const int m = m0 + (alt ? r : w * kTile + r);
        const bool row_ok = (alt ? r : w * kTile + r) < rows;
        const int b = m / TR, t = (m - b * TR) / R, h = g * R + m % R;
        int first = 0, last = hi - 1;
        if (seq >= 0) {
            last = t < nq ? min(hi - 1, len - nq + t) : -1;
            if (p.window) first = len - nq + t - p.window + 1;
        }
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t s0 = tmem + 2 * HD + lanes, ot = tmem + w * HD + lanes;
        float zs = p.scale2;
        if constexpr (I8) {
            wait_phase(&q_full, 0, abort_flag);
            zs = qscale[alt ? r : w * kTile + r];
        }
        // columns of logits in registers: all of a step; INT8, whose weights take three
        // times the instructions, reads them twice (for the maximum and for the weights),
        // 32 at a time in loops: its code does not fit the instruction cache otherwise
        // (20 against 26 us for a prefix of 384 keys)
        constexpr int kRead = I8 ? 32 : kStep;
        float top = kNegInf, sum = 0.f, vnorm = 0.f;
        // INT8: O leaves for these sums every kHold steps, held * hold + O is the whole
        // (see kHold)
        float held[HD], hold = 0.f;
        Turn turn;
        turn.on(w, ahead);
        for (int i = 0; i < mine; ++i, turn.on(each == 2 || alt ? 2 : 1, ahead)) {
            const int j = alt ? 2 * i + w : i;
            const int j0 = j < before ? j * kStep : lo + (j - before) * kStep;
            const int from = j < before ? 0 : first, to = j < before ? p.prefix - 1 : last;   // keys the row sees
            wait_phase(&s_full[turn.buffer], turn.phase, abort_flag);
            if (I8) {
                const int v = 2 * j + 1;                  // (and the step's scales)
                wait_phase(&full[v % kStages], (uint32_t)(v / kStages) & 1, abort_flag);
            }
            tc::fence_after();
            const uint32_t ts = s0 + turn.buffer * kStep;
            const float *sk = scales + (j % G::kScaleRing) * 2 * kStep;
            // kRead logits of the row from column c on, INT8: times K's scales; -inf where not seen
            const bool edge = j0 < from || j0 + kStep - 1 > to;
            float2 z[kRead / 2];
            auto read = [&](int c) {
                uint32_t raw[kRead / 32][32];
#pragma unroll
                for (int x = 0; x < kRead / 32; ++x) tc::ld32(ts + c + 32 * x, raw[x]);
                tc::wait_ld();
#pragma unroll
                for (int e = 0; e < kRead / 2; ++e)
                    z[e] = make_float2(__uint_as_float(raw[e / 16][2 * (e % 16)]),
                                       __uint_as_float(raw[e / 16][2 * (e % 16) + 1]));
                if constexpr (I8) {
#pragma unroll
                    for (int e = 0; e < kRead / 2; e += 2) {
                        const float4 s4 = *(const float4 *)(sk + c + 2 * e);
                        z[e] = mul2(z[e], make_float2(s4.x, s4.y));
                        z[e + 1] = mul2(z[e + 1], make_float2(s4.z, s4.w));
                    }
                }
                if (edge) {
                    const int x0 = from - j0 - c, x1 = to - j0 - c;
#pragma unroll
                    for (int e = 0; e < kRead / 2; ++e) {
                        if (2 * e < x0 || 2 * e > x1) z[e].x = kNegInf;
                        if (2 * e + 1 < x0 || 2 * e + 1 > x1) z[e].y = kNegInf;
                    }
                }
            };
            float best[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
#pragma unroll 1
            for (int c = 0; c < kStep; c += kRead) {
                read(c);
#pragma unroll
                for (int e = 0; e < kRead / 2; ++e) best[e & 3] = max3(best[e & 3], z[e].x, z[e].y);
            }
            const float now = max3(fmaxf(best[0], best[1]), best[2], best[3]) * zs;
            float keep = 1.f;
            if (now > top + kGrow || (top == kNegInf && now > kNegInf)) {
                keep = ex2(top - now);                // top = -inf: 0
                top = now;
            }
            sum *= keep;
            float vinv = 1.f;
            if constexpr (I8) {
                // V's scales relative to the largest so far (a power of two), times 2^6:
                // weights up to 2^kGrow then stay within FP16's 2^16, and what its small
                // numbers lose is below 2^-31 of the largest; the same in all threads
                const float most = fmaxf(fmaxf(vmost[j % G::kScaleRing][0], vmost[j % G::kScaleRing][1]), 1e-30f);
                const float norm = __uint_as_float(__float_as_uint(most) & 0x7f800000u);
                if (norm > vnorm) {
                    keep *= vnorm / norm;
                    vnorm = norm;
                }
                vinv = 64.f / vnorm;
            }
            const bool leave = I8 && i > 0 && i % G::kHold == 0;
            if (leave || (i > 0 && __any_sync(0xffffffffu, keep != 1.f))) {
                // O holds the steps before: the last one's product has to end first (the
                // ones before that had ended when these logits were computed)
                wait_phase(&o_done[w], (uint32_t)(i - 1) & 1, abort_flag);
                tc::fence_after();
                hold *= keep;
                if (leave) {
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        uint32_t o[32];
                        tc::ld32(ot + c, o);
                        tc::wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const float x = __uint_as_float(o[e]) * keep;
                            held[c + e] = hold == 0.f ? x : fmaf(held[c + e], hold, x);
                            o[e] = 0;
                        }
                        tc::st32(ot + c, o);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < HD; c += 32) {
                        uint32_t o[32];
                        tc::ld32(ot + c, o);
                        tc::wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                        tc::st32(ot + c, o);
                    }
                }
                if (I8 && leave) hold = 1.f;
            }
            const float base = top == kNegInf ? 0.f : -top;
            const float2 zs2 = make_float2(zs, zs), base2 = make_float2(base, base), vinv2 = make_float2(vinv, vinv);
            float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
            for (int c0 = 0; c0 < kStep; c0 += kRead) {
                if (kRead < kStep) read(c0);
#pragma unroll
                for (int x = 0; x < kRead; x += 32) {
                    const int c = c0 + x;
                    uint32_t hi16[16], lo16[I8 ? 16 : 1];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float2 y = fma2(z[x / 2 + e], zs2, base2);
                        y.x = ex2(y.x);
                        y.y = ex2(y.y);
                        part[e & 1] = add2(part[e & 1], y);
                        if constexpr (I8) {
                            const float2 v2 = *(const float2 *)(sk + kStep + c + 2 * e);
                            y = mul2(y, mul2(v2, vinv2));
                            split2(y.x, y.y, hi16[e], lo16[e]);
                        } else {
                            // the softmax weights are rounded to the cache's type for the
                            // product, off by half a step of each at most, as V and the output
                            // are; their sum keeps 32 bits.  (Pairs as INT8's would double the
                            // output product; two prompts of 4096 tokens in bf16 end 2.1e-3 from
                            // the definition, 1.7e-3 with 32-bit weights.)
                            hi16[e] = pack2<BF>(y.x, y.y);
                        }
                    }
                    tc::st16(ts + c, hi16);                // over the logits of these keys
                    if constexpr (I8) tc::st16(ts + c + 16, lo16);
                    if (c & 32) {                          // half of the keys
                        tc::wait_st();
                        tc::fence_before();
                        mbar_arrive(&p_full[turn.buffer][c >> 6]);
                    }
                }
            }
            part[0] = add2(part[0], part[1]);
            sum += part[0].x + part[0].y;
        }
        if (mine > 0) wait_phase(&o_full[w], 0, abort_flag);
        tc::fence_after();
        if (*abort_flag) sum = __int_as_float(0x7fffffff);   // NaN in out, lse and the weights that follow from it
        if (alt || w < tiles) {
            const float inv = sum == 0.f ? 0.f : (I8 ? vnorm * (1.f / 64.f) : 1.f) / sum;
            const float lse = sum == 0.f ? kNegInf : (top == kNegInf ? 0.f : top) + log2f(sum);
            const long long nrows = (long long)p.batch * p.tokens * p.heads;
            const long long row = ((long long)b * p.tokens + t) * p.heads + h;
            const bool direct = p.prefix_slots + p.own_slots == 1;
            const long long part = (slot + (alt ? w : 0)) * nrows + row;
            const bool write = row_ok && (!direct || t < own_tokens(p, b));
            if (row_ok) {
                if (!direct) {
                    p.part_lse[part] = lse;
                } else {
                    if (p.neg_lse) p.neg_lse[neg_lse_at(p, b, t, h)] = -lse;
                    if (p.lse && write) p.lse[row] = lse * kLn2;
                }
            }
#pragma unroll
            for (int c = 0; c < HD; c += 32) {
                uint32_t o[32];
                if (mine > 0) {
                    tc::ld32(ot + c, o);
                    tc::wait_ld();
                }
                float v[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    float x = __uint_as_float(o[e]);
                    if constexpr (I8)
                        if (hold != 0.f) x = fmaf(held[c + e], hold, x);
                    v[e] = sum == 0.f ? 0.f : x * inv;
                }
                if (!write) continue;
                if (!direct) {
                    float *dst = p.part_o + part * HD + c;
#pragma unroll
                    for (int e = 0; e < 32; e += 8)       // lanes hold rows apart: whole sectors each
                        asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst + e), "f"(v[e]),
                                     "f"(v[e + 1]), "f"(v[e + 2]), "f"(v[e + 3]), "f"(v[e + 4]), "f"(v[e + 5]),
                                     "f"(v[e + 6]), "f"(v[e + 7])
                                     : "memory");
                } else {
                    char *dst = (char *)p.out + (b * p.os[0] + t * p.os[1] + h * p.os[2] + c) * (I8 ? 4 : 2);
                    if constexpr (I8) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            ((float4 *)dst)[e] = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            ((uint4 *)dst)[e] = make_uint4(
                                pack2<BF>(v[8 * e], v[8 * e + 1]), pack2<BF>(v[8 * e + 2], v[8 * e + 3]),
                                pack2<BF>(v[8 * e + 4], v[8 * e + 5]), pack2<BF>(v[8 * e + 6], v[8 * e + 7]));
                    }
                }
            }
        }
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (warp == kProductWarp) tc::dealloc(tmem, 512);
    if (threadIdx.x == 0 && *abort_flag) atomicExch(&g_tile_fault, 1);
}

// ---- accumulated key weights ------------------------------------------------
//
// The logits once more, keys as the rows: S^T = K Q^T for two tiles of 128 keys
// against 128 query rows at a time, and sum over the rows of 2^(z - lse_row).
// Thread = key and half of the rows: the sum runs along the thread's TMEM lane in
// a fixed order.  K stays in shared memory
// for the whole CTA; the rows come by TMA, their lse beside them; two TMEM
// buffers a tile let the next product run during the exponentials, which bound
// the kernel (one a logit).  Powers of two by a polynomial on the FP32 pipe, for a
// part of them, did not pay: the more the slower (180 us for none or one of eight,
// 217 for five of eight, two prompts of 4096 tokens).

// four warpgroups of keys, two a tile, and one of products and copies:
// 4 * 128 * 104 + 128 * 64 = 640 * 96
constexpr int kWeightThreads = 640, kWeightWarps = 16;
constexpr int kWeightRegisters = 104, kWeightOthers = 64;

template <int TYPE, int HD>
struct WeightGeom {
    static constexpr bool I8 = TYPE == kCacheI8;
    static constexpr int kPieces = I8 ? 2 : 1;
    static constexpr int kTileBytes = kTile * HD * 2;
    static constexpr int kStageBytes = kPieces * kTileBytes;      // 128 query rows
    static constexpr int kStages = HD == 64 ? 4 : (I8 ? 2 : 4);
    static constexpr int kRing = 2 * kTileBytes;                  // behind the two key tiles
    static constexpr int kSmem = kRing + kStages * kStageBytes + 1024;
    static_assert(kSmem <= 232448 - 6144, "shared memory of a CTA");
};

// FP32 queries as FP16 pairs: hi and lo rows [B][kvheads][tokens * R][hd] each
// and the factor of every row, for the weights kernel's loads.
template <int HD>
__global__ __launch_bounds__(256) void split_queries_kernel(const PrefixAttn p) {
    constexpr int kLanes = HD / 4, kPer = 256 / kLanes;
    const long long rows = (long long)p.batch * p.tokens * p.heads;
    const long long row = (long long)blockIdx.x * kPer + threadIdx.x / kLanes;
    const int l = threadIdx.x % kLanes, TR = p.tokens * p.group;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < rows) {
        const long long bg = row / TR;
        const int m = (int)(row % TR), b = (int)(bg / p.kvheads), g = (int)(bg % p.kvheads);
        x = *(const float4 *)((const float *)p.q + b * p.qs[0] + m / p.group * p.qs[1] +
                              (g * p.group + m % p.group) * p.qs[2] + 4 * l);
    }
    float most = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
#pragma unroll
    for (int d = kLanes / 2; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
    float up, down;
    row_scale(most, up, down);
    pdl_enter();      // the next kernel waits for this one only: so this one ends after its predecessor
    if (row >= rows) return;
    uint2 h, lo;
    split2(x.x * up, x.y * up, h.x, lo.x);
    split2(x.z * up, x.w * up, h.y, lo.y);
    *(uint2 *)((char *)p.q16 + (row * HD + 4 * l) * 2) = h;
    *(uint2 *)((char *)p.q16 + ((rows + row) * HD + 4 * l) * 2) = lo;
    if (l == 0) p.q16_scale[row] = p.scale2 * down;
}

template <int TYPE, int HD>
__global__ __launch_bounds__(kWeightThreads, 1) void weight_tile_kernel(const PrefixAttn p, int tile_rows,
                                                                      const __grid_constant__ CUtensorMap mq) {
    using G = WeightGeom<TYPE, HD>;
    constexpr bool I8 = G::I8, BF = TYPE == kCacheBF16;
    constexpr int kStages = G::kStages;
    extern __shared__ __align__(16) char smem_raw[];
    char *smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    __shared__ __align__(8) uint64_t full[kStages], empty[kStages], s_full[2][2], s_free[2][2], drained;
    __shared__ __align__(16) float lse[kStages][I8 ? 2 : 1][kTile];   // minus the rows' lse, INT8: their factors
    __shared__ uint32_t tmem_at;
    __shared__ int abort_at;
    volatile int *abort_flag = &abort_at;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int R = p.group, TR = p.tokens * R;
    const int pairs = p.batch * p.kvheads, unit = blockIdx.x % pairs;
    const int g = unit % p.kvheads, b = unit / p.kvheads, key0 = blockIdx.x / pairs * 2 * kTile;
    const int len = own_length(p, b), nq = own_tokens(p, b), past = len - nq;   // own index of query 0
    // the rows that see a key of this CTA: queries [t0, t1)
    const int t0 = max(0, key0 - past);
    const long long behind = p.window ? (long long)min(key0 + 2 * kTile, len) - 1 + p.window - past : nq;
    const int t1 = (int)min((long long)nq, behind);
    const int m0 = t0 * R, rows = key0 < len ? max(0, (t1 - t0) * R) : 0;
    const int n = ceil_div(rows, tile_rows);

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&full[i], 1 + 32);
            mbar_init(&empty[i], 1 + 4 * kTile);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&s_full[i >> 1][i & 1], 1);
            mbar_init(&s_free[i >> 1][i & 1], 2 * kTile);
        }
        mbar_init(&drained, 1);
        abort_at = 0;
        fence_barrier_init();
    }
    if (warp == kWeightWarps) tc::alloc(&tmem_at, 512);
    pdl_enter();
    if (n > 0) {
        // two tiles of keys (zeros where there are none)
        constexpr int kChunks = HD * (I8 ? 1 : 2) / 16, kPer = kWeightThreads / kChunks;
        const long long crow = p.cache_row ? p.cache_row[b] : b;
        const char *k = (const char *)p.k + (crow * p.ks[0] + g * p.ks[1]) * (I8 ? 1 : 2);
        const long long step = p.ks[2] * (I8 ? 1 : 2);
        const int c = threadIdx.x % kChunks;
        for (int r0 = threadIdx.x / kChunks; r0 < 2 * kTile; r0 += 4 * kPer) {
            uint4 x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = r0 + e * kPer;
                x[e] = r < 2 * kTile && key0 + r < len ? *(const uint4 *)(k + (key0 + r) * step + c * 16)
                                                       : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = r0 + e * kPer;
                if (r >= 2 * kTile) continue;
                char *t = smem + (r / kTile) * G::kTileBytes;
                if constexpr (I8) {
                    uint4 a, d;
                    i8x16_to_f16(x[e], a, d);
                    *(uint4 *)(t + piece_at<kTile>(r % kTile, 2 * c)) = a;
                    *(uint4 *)(t + piece_at<kTile>(r % kTile, 2 * c + 1)) = d;
                } else {
                    *(uint4 *)(t + piece_at<kTile>(r % kTile, c)) = x[e];
                }
            }
        }
        // rows behind a short tile stay what they are here: zeros, and weightless
        for (int i = threadIdx.x; i < kStages * kTile; i += kWeightThreads) {
            lse[i / kTile][0][i % kTile] = kNegInf;
            if constexpr (I8) lse[i / kTile][1][i % kTile] = 0.f;
        }
        if (tile_rows < kTile) {
            char *q = smem + G::kRing;
            for (int i = threadIdx.x; i < kStages * G::kStageBytes / 16; i += kWeightThreads)
                *(uint4 *)(q + i * 16) = make_uint4(0, 0, 0, 0);
        }
    }
    fence_proxy_async();
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_at;

    if (warp >= kWeightWarps) {
        fewer_registers<kWeightOthers>();
        if (warp == kWeightWarps + 1) {
            // ---- query rows
            if (lane == 0) {
                int issued = 0;
                for (int i = 0; i < n; ++i) {
                    const int s = i % kStages, mi = m0 + i * tile_rows;
                    if (i >= kStages && !wait_phase(&empty[s], (uint32_t)(i / kStages - 1) & 1, abort_flag)) break;
                    char *dst = smem + G::kRing + s * G::kStageBytes;
                    mbar_arrive_expect_tx(&full[s], G::kPieces * HD * 2 * tile_rows);
                    for (int x = 0; x < G::kPieces; ++x)
                        for (int c = 0; c < HD / 64; ++c) {
                            char *d = dst + x * G::kTileBytes + c * (kTile * 128);
                            // rows (t, r): INT8 from the split copy [pieces][B * kvheads][tokens * R][hd]
                            if constexpr (I8)
                                tma_load_4d(d, &mq, 64 * c, mi, unit, x, &full[s]);
                            else
                                tma_load_4d(d, &mq, 64 * c, g * R, mi / R, b, &full[s]);
                        }
                    ++issued;
                }
                for (int i = max(0, issued - kStages); i < issued; ++i)
                    mbar_wait(&full[i % kStages], (uint32_t)(i / kStages) & 1);
            }
            __syncwarp();
        } else if (warp == kWeightWarps + 2) {
            // ---- their lse (and INT8 factors)
            const float *src = p.neg_lse + (long long)unit * TR + m0, *fac = nullptr;
            if constexpr (I8) fac = p.q16_scale + (long long)unit * TR + m0;
            for (int i = 0; i < n; ++i) {
                const int s = i % kStages, at = i * tile_rows;
                if (i >= kStages && !wait_phase(&empty[s], (uint32_t)(i / kStages - 1) & 1, abort_flag)) break;
#pragma unroll
                for (int e = 0; e < kTile / 32; ++e) {
                    const int x = lane + 32 * e, m = min(at + x, rows - 1);   // (rows behind the last: not counted)
                    if (x < tile_rows) {
                        cp_async<4>(&lse[s][0][x], src + m);
                        if constexpr (I8) cp_async<4>(&lse[s][1][x], fac + m);
                    }
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(&full[s]))
                             : "memory");
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            __syncwarp();
        } else if (warp == kWeightWarps) {
            // ---- products
            constexpr uint32_t ids = idesc(BF, false, kTile);
            const uint32_t k0 = smem_addr(smem), q0 = smem_addr(smem) + G::kRing;
            for (int i = 0; i < n; ++i) {
                const int s = i % kStages;
                wait_phase(&full[s], (uint32_t)(i / kStages) & 1, abort_flag);
                for (int w = 0; w < 2; ++w) {
                    if (i >= 2) wait_phase(&s_free[w][i & 1], (uint32_t)(i / 2 - 1) & 1, abort_flag);
                    __syncwarp();
                    if (elect_one()) {
                        tc::fence_after();
#pragma unroll
                        for (int x = G::kPieces - 1; x >= 0; --x)      // the small pieces first
#pragma unroll
                            for (int c = 0; c < HD / 16; ++c) {
                                const uint32_t at = (c / 4) * (kTile * 128) + (c % 4) * 32;
                                tc::mma_bf16_ss(tmem + (2 * w + (i & 1)) * kTile, desc_k(k0 + w * G::kTileBytes + at),
                                                desc_k(q0 + s * G::kStageBytes + x * G::kTileBytes + at), ids,
                                                x < G::kPieces - 1 || c > 0);
                            }
                        tc::commit(&s_full[w][i & 1]);
                        if (w == 1) tc::commit(&empty[s]);
                    }
                    __syncwarp();
                }
            }
            if (__any_sync(0xffffffffu, *abort_flag)) {   // no product is in flight when TMEM is freed
                if (elect_one()) tc::commit(&drained);
                mbar_wait(&drained, 0);
                __syncwarp();
            }
        }
        __syncwarp();
    } else {
        more_registers<kWeightRegisters>();
        // ---- thread = key and half of the rows
        constexpr int kCols = kTile / 2;
        const int w = warp >> 3, half = (warp >> 2) & 1, j = key0 + w * kTile + (threadIdx.x & (kTile - 1));
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        float ks = p.scale2;
        if constexpr (I8) {
            const long long crow = p.cache_row ? p.cache_row[b] : b;
            ks = j < len ? p.kscale[crow * p.kss[0] + g * p.kss[1] + j * p.kss[2]] : 0.f;
        }
        // the rows that see the key: [from, to) of the CTA's
        long long from = max(0LL, ((long long)j - past - t0) * R), to = rows;
        if (p.window) to = min(to, ((long long)j + p.window - past - t0) * R);
        if (j >= len) to = 0;
        float total = 0.f;
        const float2 k2 = make_float2(ks, ks);
        for (int i = 0; i < n; ++i) {
            const int s = i % kStages;
            wait_phase(&s_full[w][i & 1], (uint32_t)(i / 2) & 1, abort_flag);
            // (the rows' lse: written before the products' wait for the same phase)
            wait_phase(&full[s], (uint32_t)(i / kStages) & 1, abort_flag);
            tc::fence_after();
            const uint32_t ts = tmem + (2 * w + (i & 1)) * kTile + half * kCols + lanes;
            uint32_t raw[2][32];
            tc::ld32(ts, raw[0]);
            tc::ld32(ts + 32, raw[1]);
            tc::wait_ld();
            tc::fence_before();
            mbar_arrive(&s_free[w][i & 1]);
            const long long at = (long long)i * tile_rows + half * kCols;
            const int x0 = (int)max(0LL, min((long long)kCols, from - at));
            const int x1 = (int)max(0LL, min((long long)kCols, to - at));
            const float *ls = &lse[s][0][half * kCols], *fs = &lse[s][I8 ? 1 : 0][half * kCols];
            float2 part[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) part[c] = make_float2(0.f, 0.f);
            if (__all_sync(0xffffffffu, x0 == 0 && x1 == kCols)) {
#pragma unroll
                for (int c = 0; c < kCols; c += 4) {
                    const float4 l4 = *(const float4 *)(ls + c);
                    float2 a = make_float2(__uint_as_float(raw[c / 32][c % 32]),
                                           __uint_as_float(raw[c / 32][c % 32 + 1]));
                    float2 d = make_float2(__uint_as_float(raw[c / 32][c % 32 + 2]),
                                           __uint_as_float(raw[c / 32][c % 32 + 3]));
                    if constexpr (I8) {
                        const float4 f4 = *(const float4 *)(fs + c);
                        a = fma2(a, mul2(k2, make_float2(f4.x, f4.y)), make_float2(l4.x, l4.y));
                        d = fma2(d, mul2(k2, make_float2(f4.z, f4.w)), make_float2(l4.z, l4.w));
                    } else {
                        a = fma2(a, k2, make_float2(l4.x, l4.y));
                        d = fma2(d, k2, make_float2(l4.z, l4.w));
                    }
                    a = make_float2(ex2(a.x), ex2(a.y));
                    d = make_float2(ex2(d.x), ex2(d.y));
                    part[(c / 4) & 1] = add2(part[(c / 4) & 1], a);
                    part[2 + ((c / 4) & 1)] = add2(part[2 + ((c / 4) & 1)], d);
                }
            } else if (x0 < x1) {
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
                    float f = ks;
                    if constexpr (I8) f *= fs[c];
                    const float y = ex2(fmaf(__uint_as_float(raw[c / 32][c % 32]), f, ls[c]));
                    if (c >= x0 && c < x1) part[c & 3].x += y;
                }
            }
            mbar_arrive(&empty[s]);
            part[0] = add2(add2(part[0], part[1]), add2(part[2], part[3]));
            total += part[0].x + part[0].y;
        }
        if (*abort_flag) total = __int_as_float(0x7fffffff);   // (NaN)
        float *halves = &lse[0][0][0];                 // (free once every thread is past its rows)
        static_assert(kStages >= 2, "room for the sums");
        asm volatile("bar.sync 1, 512;" ::: "memory");
        if (half) halves[w * kTile + (threadIdx.x & (kTile - 1))] = total;
        tile_sync(2 + w);
        if (!half && j < p.capacity)
            p.weights_out[b * p.wos[0] + g * p.wos[1] + j * p.wos[2]] =
                p.weights[b * p.ws[0] + g * p.ws[1] + j * p.ws[2]] +
                (total + halves[w * kTile + (threadIdx.x & (kTile - 1))]);
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (warp == kWeightWarps) tc::dealloc(tmem, 512);
    if (threadIdx.x == 0 && *abort_flag) atomicExch(&g_tile_fault, 1);
}

// ---- host ------------------------------------------------------------------

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    });
    return fn;
}

// Map of a cache [seqs][heads][keys][hd] in steps of kStep keys: 128-byte
// swizzled chunks of 64 16-bit values, or whole INT8 rows.  Axes of stride 0
// (or one element) get extent 1 and their flag 0: the kernel's coordinate stays 0.
bool cache_map(CUtensorMap *map, const void *base, int type, int hd, long long keys, long long heads, long long seqs,
               long long key_stride, long long head_stride, long long seq_stride, int *head_flag, int *seq_flag) {
    auto fn = encoder();
    if (!fn) {
        set_error("cuTensorMapEncodeTiled is unavailable");
        return false;
    }
    const bool i8 = type == kCacheI8;
    const long long size = i8 ? 1 : 2, row = hd * size;
    *head_flag = head_stride != 0 && heads > 1;
    *seq_flag = seq_stride != 0 && seqs > 1;
    if (!*head_flag) heads = 1;
    if (!*seq_flag) seqs = 1;
    const long long ks = keys > 1 ? key_stride * size : row;     // (above zero: keys of stride 0 are streamed)
    const cuuint64_t dims[4] = {(cuuint64_t)hd, (cuuint64_t)keys, (cuuint64_t)heads, (cuuint64_t)seqs};
    const cuuint64_t strides[3] = {(cuuint64_t)ks, (cuuint64_t)(*head_flag ? head_stride * size : row),
                                   (cuuint64_t)(*seq_flag ? seq_stride * size : row)};
    const cuuint32_t box[4] = {(cuuint32_t)(i8 ? hd : 64), (cuuint32_t)kStep, 1, 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult r =
        fn(map, i8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void *>(base), dims,
           strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
           i8 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("prefix attention: the cache's strides cannot be described to the copy engine");
        return false;
    }
    return true;
}

}  // namespace

int read_and_clear_tile_fault() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_tile_fault, sizeof(int)) != cudaSuccess) return -1;
    if (v) cudaMemcpyToSymbol(g_tile_fault, &zero, sizeof(int));
    return v ? 1 : 0;
}

bool launch_prefix_tiles(const PrefixAttn &p, const PrefixSplit &prefix, const PrefixSplit &own, bool joint,
                         long long cache_rows, bool stream_next, cudaStream_t st) {
    auto run = [&](auto type, auto hd) -> bool {
        using G = TileGeom<type(), hd()>;
        TileGrid grid{};
        grid.stream_next = stream_next;
        grid.joint = joint;
        const int rows = p.tokens * p.group;
        CUtensorMap mk{}, mv{}, mpk{}, mpv{};
        int unused;
        if (own.tiles) {
            grid.own_alt = own.alt;
            grid.own_rows = own.alt ? kTile : 2 * kTile;
            grid.own_tiles = ceil_div(rows, grid.own_rows);
            grid.own_ranges = own.ranges;
            grid.own_units = p.batch * p.kvheads * grid.own_tiles * own.ranges;
            if (!cache_map(&mk, p.k, type(), hd(), p.capacity, p.kvheads, cache_rows, p.ks[2], p.ks[1], p.ks[0],
                           &grid.k_head, &grid.k_seq) ||
                !cache_map(&mv, p.v, type(), hd(), p.capacity, p.kvheads, cache_rows, p.vs[2], p.vs[1], p.vs[0],
                           &grid.v_head, &grid.v_seq))
                return false;
        }
        if (prefix.tiles) {
            grid.prefix_alt = prefix.alt;
            grid.prefix_rows = prefix.alt ? kTile : 2 * kTile;
            grid.prefix_tiles = ceil_div(p.batch * rows, grid.prefix_rows);
            grid.prefix_ranges = prefix.ranges;
            grid.prefix_units = p.kvheads * grid.prefix_tiles * prefix.ranges;
        }
        if (prefix.tiles || joint) {
            if (!cache_map(&mpk, p.pk, type(), hd(), p.prefix, p.kvheads, 1, p.pks[1], p.pks[0], 0, &grid.pk_head,
                           &unused) ||
                !cache_map(&mpv, p.pv, type(), hd(), p.prefix, p.kvheads, 1, p.pvs[1], p.pvs[0], 0, &grid.pv_head,
                           &unused))
                return false;
        }
        // the prefix's units before the own keys' where theirs are the longer ranges: 37 tokens
        // of 16 sequences over 4096 shared and 509 own keys in f16 take 32.8 us so, 39.7 otherwise
        const int span = p.window ? std::min<long long>(p.capacity, (long long)p.window + p.tokens) : p.capacity;
        grid.prefix_first = prefix.tiles && own.tiles && p.prefix / prefix.ranges > span / own.ranges;
        const int blocks = grid.own_units + grid.prefix_units;
        if (blocks == 0) return true;
        auto kernel = prefix_tile_kernel<type(), hd()>;
        static bool configured[64] = {};
        int dev = 0;
        NB_CUDA_TRY(cudaGetDevice(&dev));
        if (dev < 0 || dev >= 64 || !configured[dev]) {
            NB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmem));
            if (dev >= 0 && dev < 64) configured[dev] = true;
        }
        kernel<<<blocks, kTileThreads, G::kSmem, st>>>(p, grid, mk, mv, mpk, mpv);
        NB_CUDA_TRY(cudaGetLastError());
        return true;
    };
    return by_geometry(p, run);
}

bool launch_weight_tiles(const PrefixAttn &p, cudaStream_t st) {
    auto run = [&](auto type, auto hd) -> bool {
        using G = WeightGeom<type(), hd()>;
        auto fn = encoder();
        if (!fn) {
            set_error("cuTensorMapEncodeTiled is unavailable");
            return false;
        }
        const int R = p.group, tile_rows = kTile / R * R;
        const long long rows = (long long)p.batch * p.tokens * p.heads;
        CUtensorMap mq{};
        CUresult r;
        const cuuint32_t estr[4] = {1, 1, 1, 1};
        if constexpr (G::I8) {
            // [2][B * kvheads][tokens * R][hd], the split copy
            const long long TR = (long long)p.tokens * R, units = (long long)p.batch * p.kvheads;
            const cuuint64_t dims[4] = {(cuuint64_t)hd(), (cuuint64_t)TR, (cuuint64_t)units, 2};
            const cuuint64_t strides[3] = {(cuuint64_t)hd() * 2, (cuuint64_t)(TR * hd() * 2),
                                           (cuuint64_t)(rows * hd() * 2)};
            const cuuint32_t box[4] = {64, (cuuint32_t)tile_rows, 1, 1};
            r = fn(&mq, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, p.q16, dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        } else {
            // [B][tokens][heads][hd]: R heads of tile_rows / R tokens a box
            auto stride = [&](long long s, int n) { return (cuuint64_t)(n > 1 ? s * 2 : hd() * 2); };
            const cuuint64_t dims[4] = {(cuuint64_t)hd(), (cuuint64_t)p.heads, (cuuint64_t)p.tokens,
                                        (cuuint64_t)p.batch};
            const cuuint64_t strides[3] = {stride(p.qs[2], p.heads), stride(p.qs[1], p.tokens),
                                           stride(p.qs[0], p.batch)};
            const cuuint32_t box[4] = {64, (cuuint32_t)R, (cuuint32_t)(tile_rows / R), 1};
            r = fn(&mq, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void *>(p.q), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        }
        if (r != CUDA_SUCCESS) {
            set_error("prefix attention: the queries' strides cannot be described to the copy engine");
            return false;
        }
        if constexpr (G::I8) {
            const int per = 256 / (hd() / 4);
            NB_CUDA_TRY(launch_pdl(split_queries_kernel<hd()>, dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0,
                                   st, p));
        }
        auto kernel = weight_tile_kernel<type(), hd()>;
        static bool configured[64] = {};
        int dev = 0;
        NB_CUDA_TRY(cudaGetDevice(&dev));
        if (dev < 0 || dev >= 64 || !configured[dev]) {
            NB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmem));
            if (dev >= 0 && dev < 64) configured[dev] = true;
        }
        const int blocks = p.batch * p.kvheads * ceil_div(p.capacity, 2 * kTile);
        if (blocks == 0) return true;
        NB_CUDA_TRY(launch_pdl(kernel, dim3(blocks), dim3(kWeightThreads), (size_t)G::kSmem, st, p, tile_rows, mq));
        return true;
    };
    return by_geometry(p, run);
}

}  // namespace nb200
