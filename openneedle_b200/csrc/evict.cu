// Eviction from a KV cache by accumulated attention weight.
//
// Of a sequence's n own keys, `keep` stay per KV head where n is larger: the
// first `first`, the last `recent`, and of those between them the keep - first -
// recent of the largest weight (ties: the lower index; NaN counts as -inf).
// They are packed in their order into the front of the output.
//
// Bound by the bytes of the kept rows for large caches: 1024 rows of 3712 INT8 keys
// thinned to 1024 (260 MB) 65 us, 4.0 TB/s, of which the copies alone take 50; two
// documents of 65536 bf16 keys and 8 KV heads thinned to 8192 (139 MB) 21 us for the
// selection and 23 for the copies (5.7 TB/s).
#include <algorithm>

#include "common.cuh"
#include "evict.cuh"
#include "pdl.cuh"
#include "sm100_async.cuh"

namespace nb200 {
namespace {

constexpr int kThreads = 1024;
constexpr int kCopyRows = 296;   // rows (two a multiprocessor) from which the selecting CTAs copy

// Order-preserving unsigned key of a weight; both zeros are one value.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (isnan(w)) w = -__builtin_huge_valf();
    const uint32_t u = __float_as_uint(w + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// kRowsOf kept rows, `step` apart from row i0 on, to the output, all in flight at
// once: the thread's 16-byte piece of K and of V (a row has 1 << shift pieces).
constexpr int kRowsOf = 2;

__device__ __forceinline__ void copy_rows(const Evict &e, int unit, int i0, int step, int kept, int shift) {
    const int g = unit % e.kvheads, b = unit / e.kvheads, piece = threadIdx.x & ((1 << shift) - 1);
    const int *idx = e.indices + (long long)unit * e.keep;
    long long j[kRowsOf];
#pragma unroll
    for (int r = 0; r < kRowsOf; ++r) j[r] = i0 + r * step < kept ? idx[i0 + r * step] : -1;
    const char *k = e.k + b * e.ks[0] + g * e.ks[1] + piece * 16, *v = e.v + b * e.vs[0] + g * e.vs[1] + piece * 16;
    uint4 x[kRowsOf], y[kRowsOf];
#pragma unroll
    for (int r = 0; r < kRowsOf; ++r)
        if (j[r] >= 0) {
            x[r] = __ldcs((const uint4 *)(k + j[r] * e.ks[2]));
            y[r] = __ldcs((const uint4 *)(v + j[r] * e.vs[2]));
        }
    float s[kRowsOf];
    const bool scales = e.kscale && piece < 2;       // piece 0 moves K's, piece 1 V's
    if (scales) {
        const float *sc = piece == 0 ? e.kscale + b * e.kss[0] + g * e.kss[1] : e.vscale + b * e.vss[0] + g * e.vss[1];
        const long long next = piece == 0 ? e.kss[2] : e.vss[2];
#pragma unroll
        for (int r = 0; r < kRowsOf; ++r)
            if (j[r] >= 0) s[r] = sc[j[r] * next];
    }
    char *ko = e.ko + b * e.kos[0] + g * e.kos[1] + piece * 16, *vo = e.vo + b * e.vos[0] + g * e.vos[1] + piece * 16;
#pragma unroll
    for (int r = 0; r < kRowsOf; ++r)
        if (j[r] >= 0) {
            const long long i = i0 + r * step;
            *(uint4 *)(ko + i * e.kos[2]) = x[r];
            *(uint4 *)(vo + i * e.vos[2]) = y[r];
            if (scales) {
                if (piece == 0)
                    e.kscale_o[b * e.ksos[0] + g * e.ksos[1] + i * e.ksos[2]] = s[r];
                else
                    e.vscale_o[b * e.vsos[0] + g * e.vsos[1] + i * e.vsos[2]] = s[r];
            }
        }
}

// Selection with a row's weights in registers: a cluster of C CTAs per
// (sequence, KV head), each thread up to kMine weights of its CTA's contiguous
// segment.  The key of the last weight that stays is found eight bits at a time
// from the top: the keys that still match are counted by digit in shared memory
// (few of them after the first round), the counts of a cluster's CTAs meet by
// distributed shared memory, and the search ends where a digit's keys are just as
// many as stay.  Then ties (where some of them stay and others not) and kept
// positions are ranked in index order, and everything is written.  The weights
// are read once; bound by the latency of the rounds.
constexpr int kMine = 16;

template <int C, int T, bool COPY>
__global__ __launch_bounds__(T, T == 256 ? 4 : 1) void evict_rank_kernel(const Evict e, int shift) {
    constexpr int kWarpsIn = T / 32;
    const int row = blockIdx.x / C, rank = blockIdx.x % C;
    const int g = row % e.kvheads, b = row / e.kvheads;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n = max(0, min(e.lengths[b], e.capacity)), kept = min(n, e.keep);
    const float *w = e.weights + b * e.ws[0] + g * e.ws[1];
    float *wo = e.weights_o + b * e.wos[0] + g * e.wos[1];
    int *idx = e.indices + (long long)row * e.keep;
    __shared__ int counts[4][256];
    __shared__ int sums[8], found[3];
    __shared__ int ranks[2][kMine * kWarpsIn + 1];   // ties, kept: of (i, warp), then exclusive sums; last: their total
    for (int i = tid; i < 1024; i += T) (&counts[0][0])[i] = 0;

    const int lo = e.first, hi = n - e.recent, seg = ceil_div(ceil_div(e.capacity, C), T) * T, j0 = rank * seg;
    const int mine = min(kMine, ceil_div(max(0, min(seg, n - j0)), T));
    float x[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int j = j0 + i * T + tid;
        x[i] = i < mine && j < n ? w[j * e.ws[2]] : 0.f;
    }
    auto all_sync = [&] {
        if constexpr (C > 1) {
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
            asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        } else {
            __syncthreads();
        }
    };
    // the value of another CTA's copy of a shared variable
    auto of_cta = [&](const int *v, int cta) -> int {
        if constexpr (C == 1) return *v;
        uint32_t a = smem_addr(v), r;
        int y;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(cta));
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(y) : "r"(r) : "memory");
        return y;
    };
    all_sync();                                      // counts are zero; no weight is read after this

    const bool choose = n > e.keep;
    int need = e.keep - e.first - e.recent;          // of the keys equal to `prefix` so far
    const bool none = need == 0;
    uint32_t prefix = 0;
    bool exact = false;                              // all keys from `prefix` on stay
    if (choose && !none) {                           // the same in every CTA of the row
        for (int it = 0; it < 4 && !exact; ++it) {
            const int shift = 24 - 8 * it;
            const uint32_t mask = it == 0 ? 0u : ~0u << (shift + 8);
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                if (i >= mine) break;
                const int j = j0 + i * T + tid;
                const uint32_t u = weight_key(x[i]);
                if (j >= lo && j < hi && (u & mask) == prefix) atomicAdd(&counts[it][(u >> shift) & 255], 1);
            }
            all_sync();
            // thread d has the digit 255 - d: the one in which the need-th largest key lies
            int total = 0, above = 0;
            if (tid < 256) {
                for (int r = 0; r < C; ++r) total += of_cta(&counts[it][255 - tid], r);
                above = total;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, above, d);
                    if (lane >= d) above += y;
                }
                if (lane == 31) sums[warp] = above;
            }
            __syncthreads();
            if (tid < 256) {
                for (int k = 0; k < warp; ++k) above += sums[k];
                if (above >= need && above - total < need) {
                    found[0] = 255 - tid;
                    found[1] = need - (above - total);
                    found[2] = total;
                }
            }
            __syncthreads();
            prefix |= (uint32_t)found[0] << shift;
            need = found[1];
            exact = need == found[2];
        }
    }

    // ranks of the ties: exclusive sums over (i, warp), then over the CTAs
    auto exclusive = [&](int which) -> int {         // the CTA's own offset
        int *v = ranks[which];
        __syncthreads();
        if (warp == 0) {
            int carry = 0;
            for (int k = 0; k < mine * kWarpsIn; k += 32) {
                const int y = k + lane < mine * kWarpsIn ? v[k + lane] : 0;
                int s = y;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int z = __shfl_up_sync(0xffffffffu, s, d);
                    if (lane >= d) s += z;
                }
                if (k + lane < mine * kWarpsIn) v[k + lane] = carry + s - y;
                carry += __shfl_sync(0xffffffffu, s, 31);
            }
            if (lane == 0) v[kMine * kWarpsIn] = carry;
        }
        all_sync();
        int before = 0;
        for (int r = 0; r < rank; ++r) before += of_cta(&v[kMine * kWarpsIn], r);
        return before;
    };
    int tie_base = 0;
    if (choose && !none && !exact) {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            if (i >= mine) break;
            const int j = j0 + i * T + tid;
            const unsigned m = __ballot_sync(0xffffffffu, j >= lo && j < hi && weight_key(x[i]) == prefix);
            if (lane == 0) ranks[0][i * kWarpsIn + warp] = __popc(m);
        }
        tie_base = exclusive(0);
    }
    uint32_t stays = 0;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        if (i >= mine) break;
        const int j = j0 + i * T + tid;
        const uint32_t u = weight_key(x[i]);
        const bool middle = choose && j >= lo && j < hi;
        bool s = j < n && (!middle || (!none && u >= prefix));
        if (!exact) {                                // the first `need` of the ties stay
            const bool tie = middle && !none && u == prefix;
            const unsigned m = __ballot_sync(0xffffffffu, tie);
            if (tie) s = tie_base + ranks[0][i * kWarpsIn + warp] + __popc(m & ((1u << lane) - 1)) < need;
        }
        const unsigned k = __ballot_sync(0xffffffffu, s);
        if (lane == 0) ranks[1][i * kWarpsIn + warp] = __popc(k);
        stays |= (uint32_t)s << i;
    }
    const int base = exclusive(1);
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        if (i >= mine) break;
        const bool s = stays >> i & 1;
        const unsigned k = __ballot_sync(0xffffffffu, s);
        if (s) {
            const int at = base + ranks[1][i * kWarpsIn + warp] + __popc(k & ((1u << lane) - 1));
            idx[at] = j0 + i * T + tid;
            wo[at * e.wos[2]] = x[i];
        }
    }
    for (int i = kept + rank * T + tid; i < e.keep; i += C * T) idx[i] = -1;
    for (int i = kept + rank * T + tid; i < e.out_capacity; i += C * T) wo[i * e.wos[2]] = 0.f;
    if (g == 0 && rank == 0 && tid == 0) e.lengths_o[b] = kept;
    if constexpr (C > 1) all_sync();                 // no CTA ends while another reads its counts
    if constexpr (COPY) {
        __syncthreads();                             // (the indexes)
        const int step = T >> shift;
        for (int i = tid >> shift; i < kept; i += kRowsOf * step) copy_rows(e, row, i, step, kept, shift);
    }
}

// Selection of rows too long for that: one CTA per (sequence, KV head) reads the
// weights in four passes over the keys' bytes, then ranks them in chunks.
__global__ __launch_bounds__(kThreads) void evict_select_kernel(const Evict e) {
    const int g = blockIdx.x % e.kvheads, b = blockIdx.x / e.kvheads;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n = max(0, min(e.lengths[b], e.capacity)), kept = min(n, e.keep);
    const float *w = e.weights + b * e.ws[0] + g * e.ws[1];
    float *wo = e.weights_o + b * e.wos[0] + g * e.wos[1];
    int *idx = e.indices + (long long)blockIdx.x * e.keep;
    __shared__ int hist[256];
    __shared__ int sums[32];
    __shared__ int pick, left;

    const int lo = e.first, hi = n - e.recent;       // candidates where n > keep
    uint32_t prefix = 0;
    int need = e.keep - e.first - e.recent;          // still to find among the keys equal to `prefix` so far
    if (n > e.keep) {
        for (int shift = 24; shift >= 0 && need > 0; shift -= 8) {
            for (int i = tid; i < 256; i += kThreads) hist[i] = 0;
            __syncthreads();
            const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
            for (int j = lo + tid; j < hi; j += kThreads) {
                const uint32_t u = weight_key(w[j * e.ws[2]]);
                if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift) & 255], 1);
            }
            __syncthreads();
            if (warp == 0) {
                // the bin, from above, in which the `need`-th key lies
                int mine = 0;
                for (int i = 0; i < 8; ++i) mine += hist[255 - 8 * lane - i];
                int above = mine;
                for (int d = 1; d < 32; d <<= 1) {
                    const int x = __shfl_up_sync(0xffffffffu, above, d);
                    if (lane >= d) above += x;
                }
                above -= mine;
                if (above < need && above + mine >= need) {
                    int bin = 255 - 8 * lane;
                    while (above + hist[bin] < need) above += hist[bin--];
                    pick = bin;
                    left = need - above;
                }
            }
            __syncthreads();
            prefix |= (uint32_t)pick << shift;
            need = left;
            __syncthreads();
        }
    }
    // `need` of the keys equal to `prefix` stay, the lowest indexes first (none
    // stays of candidates that need nothing: no key is above ~0)
    const bool none = e.keep - e.first - e.recent == 0;
    int out = 0, equal = 0;                          // of all chunks before
    for (int j0 = 0; j0 < n; j0 += kThreads) {
        const int j = j0 + tid;
        const float x = j < n ? w[j * e.ws[2]] : 0.f;
        const uint32_t u = weight_key(x);
        const bool middle = n > e.keep && j >= lo && j < hi;
        const bool tie = middle && !none && u == prefix;
        // ties before this one: in this chunk and in earlier ones
        const unsigned tb = __ballot_sync(0xffffffffu, tie);
        if (lane == 0) sums[warp] = __popc(tb);
        __syncthreads();
        int before = 0, all = 0;
        for (int i = 0; i < 32; ++i) {
            before += i < warp ? sums[i] : 0;
            all += sums[i];
        }
        before += __popc(tb & ((1u << lane) - 1));
        const bool stays = j < n && (!middle || (!none && (u > prefix || (tie && equal + before < need))));
        equal += all;
        __syncthreads();
        const unsigned sb = __ballot_sync(0xffffffffu, stays);
        if (lane == 0) sums[warp] = __popc(sb);
        __syncthreads();
        before = 0, all = 0;
        for (int i = 0; i < 32; ++i) {
            before += i < warp ? sums[i] : 0;
            all += sums[i];
        }
        before += __popc(sb & ((1u << lane) - 1));
        // in place: a write goes to out + before <= j, read by all threads above
        if (stays) {
            idx[out + before] = j;
            wo[(long long)(out + before) * e.wos[2]] = x;
        }
        out += all;
        __syncthreads();
    }
    for (int i = kept + tid; i < e.keep; i += kThreads) idx[i] = -1;
    for (int i = kept + tid; i < e.out_capacity; i += kThreads) wo[i * e.wos[2]] = 0.f;
    if (g == 0 && tid == 0) e.lengths_o[b] = kept;
}

// Kept rows to other memory by a grid of their own.
__global__ __launch_bounds__(256) void evict_gather_kernel(const Evict e, int chunks, int shift) {
    const int unit = blockIdx.x / chunks;
    pdl_enter();
    const int kept = min(max(0, min(e.lengths[unit / e.kvheads], e.capacity)), e.keep);
    copy_rows(e, unit, blockIdx.x % chunks * (kRowsOf * (256 >> shift)) + (threadIdx.x >> shift), 256 >> shift, kept,
              shift);
}

// The same in place: one CTA moves a (sequence, KV head) front to back, a
// chunk's rows read by all threads before any is written (row i moves to i from
// an index >= i, so a chunk's writes reach rows of this and earlier chunks only).
__global__ __launch_bounds__(kThreads) void evict_move_kernel(const Evict e) {
    pdl_enter();
    const int g = blockIdx.x % e.kvheads, b = blockIdx.x / e.kvheads;
    const int pieces = e.row_bytes / 16, rows = kThreads / pieces, piece = threadIdx.x % pieces;
    const int n = max(0, min(e.lengths[b], e.capacity)), kept = min(n, e.keep);
    if (n <= e.keep) return;
    const int *idx = e.indices + (long long)blockIdx.x * e.keep;
    for (int i0 = e.first; i0 < kept; i0 += rows) {
        const int i = i0 + threadIdx.x / pieces;
        const bool valid = threadIdx.x / pieces < rows && i < kept;
        uint4 k, v;
        float ks = 0.f, vs = 0.f;
        long long j = i;
        if (valid) {
            j = idx[i];
            k = *(const uint4 *)(e.k + b * e.ks[0] + g * e.ks[1] + j * e.ks[2] + piece * 16);
            v = *(const uint4 *)(e.v + b * e.vs[0] + g * e.vs[1] + j * e.vs[2] + piece * 16);
            if (piece == 0 && e.kscale) {
                ks = e.kscale[b * e.kss[0] + g * e.kss[1] + j * e.kss[2]];
                vs = e.vscale[b * e.vss[0] + g * e.vss[1] + j * e.vss[2]];
            }
        }
        __syncthreads();
        if (valid && j != i) {
            *(uint4 *)(e.ko + b * e.kos[0] + g * e.kos[1] + i * e.kos[2] + piece * 16) = k;
            *(uint4 *)(e.vo + b * e.vos[0] + g * e.vos[1] + i * e.vos[2] + piece * 16) = v;
            if (piece == 0 && e.kscale) {
                e.kscale_o[b * e.ksos[0] + g * e.ksos[1] + i * e.ksos[2]] = ks;
                e.vscale_o[b * e.vsos[0] + g * e.vsos[1] + i * e.vsos[2]] = vs;
            }
        }
        __syncthreads();
    }
}

}  // namespace

namespace {

template <int C, int T, bool COPY = false>
bool launch_rank(const Evict &e, int rows, int shift, cudaStream_t st) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(rows * C);
    cfg.blockDim = dim3(T);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    NB_CUDA_TRY(cudaLaunchKernelEx(&cfg, evict_rank_kernel<C, T, COPY>, e, shift));
    return true;
}

}  // namespace

bool launch_evict(const Evict &e, cudaStream_t st) {
    const int units = e.batch * e.kvheads;
    if (units == 0) return true;
    const int pieces = e.row_bytes / 16, shift = pieces == 4 ? 2 : pieces == 8 ? 3 : 4;
    const int n = e.capacity;
    // where the rows fill the machine, each CTA copies its own (one's selection runs
    // beside another's copies: 69 -> 65 us for 1024 rows of 3712 INT8 keys)
    if (!e.in_place && n <= 256 * kMine && units >= kCopyRows) return launch_rank<1, 256, true>(e, units, shift, st);
    // a row's weights in registers: as few CTAs as hold them
    bool ok;
    if (n <= 256 * kMine)
        ok = launch_rank<1, 256>(e, units, shift, st);
    else if (n <= 1024 * kMine)
        ok = launch_rank<1, 1024>(e, units, shift, st);
    else if (n <= 4 * 1024 * kMine)
        ok = launch_rank<4, 1024>(e, units, shift, st);
    else if (n <= 8 * 1024 * kMine)
        ok = launch_rank<8, 1024>(e, units, shift, st);
    else {
        evict_select_kernel<<<units, kThreads, 0, st>>>(e);
        NB_CUDA_TRY(cudaGetLastError());
        ok = true;
    }
    if (!ok) return false;
    if (e.in_place) {
        NB_CUDA_TRY(launch_pdl(evict_move_kernel, dim3(units), dim3(kThreads), 0, st, e));
        return true;
    }
    const int chunks = ceil_div(e.keep, kRowsOf * (256 >> shift));
    if (chunks == 0) return true;
    NB_CUDA_TRY(launch_pdl(evict_gather_kernel, dim3(units * chunks), dim3(256), 0, st, e, chunks, shift));
    return true;
}

}  // namespace nb200
