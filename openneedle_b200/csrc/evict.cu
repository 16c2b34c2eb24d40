// Eviction from a KV cache by accumulated attention weight.
//
// Of a sequence's n own keys, `keep` stay per KV head where n is larger: the
// first `first`, the last `recent`, and of those between them the keep - first -
// recent of the largest weight (ties: the lower index; NaN counts as -inf).
// They are packed in their order into the front of the output.
#include <algorithm>

#include "common.cuh"
#include "evict.cuh"
#include "pdl.cuh"

namespace nb200 {
namespace {

constexpr int kThreads = 1024;

// Order-preserving unsigned key of a weight; both zeros are one value.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (isnan(w)) w = -__builtin_huge_valf();
    const uint32_t u = __float_as_uint(w + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One CTA per (sequence, KV head): the key of the last weight that stays by
// four passes over its bytes, then the positions in order.
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

// Kept rows to other memory: a 16-byte piece of K and of V a thread.
__global__ __launch_bounds__(256) void evict_gather_kernel(const Evict e, int chunks) {
    pdl_enter();
    const int unit = blockIdx.x / chunks, g = unit % e.kvheads, b = unit / e.kvheads;
    const int pieces = e.row_bytes / 16, rows = 256 / pieces;
    const int piece = threadIdx.x % pieces;
    const int kept = min(max(0, min(e.lengths[b], e.capacity)), e.keep);
    const int i = blockIdx.x % chunks * rows + threadIdx.x / pieces;
    if (i >= kept) return;
    const long long j = e.indices[(long long)unit * e.keep + i];
    const uint4 k = *(const uint4 *)(e.k + b * e.ks[0] + g * e.ks[1] + j * e.ks[2] + piece * 16);
    const uint4 v = *(const uint4 *)(e.v + b * e.vs[0] + g * e.vs[1] + j * e.vs[2] + piece * 16);
    *(uint4 *)(e.ko + b * e.kos[0] + g * e.kos[1] + i * e.kos[2] + piece * 16) = k;
    *(uint4 *)(e.vo + b * e.vos[0] + g * e.vos[1] + i * e.vos[2] + piece * 16) = v;
    if (piece == 0 && e.kscale) {
        e.kscale_o[b * e.ksos[0] + g * e.ksos[1] + i * e.ksos[2]] = e.kscale[b * e.kss[0] + g * e.kss[1] + j * e.kss[2]];
        e.vscale_o[b * e.vsos[0] + g * e.vsos[1] + i * e.vsos[2]] = e.vscale[b * e.vss[0] + g * e.vss[1] + j * e.vss[2]];
    }
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

bool launch_evict(const Evict &e, cudaStream_t st) {
    const int units = e.batch * e.kvheads;
    if (units == 0) return true;
    evict_select_kernel<<<units, kThreads, 0, st>>>(e);
    NB_CUDA_TRY(cudaGetLastError());
    if (e.in_place) {
        NB_CUDA_TRY(launch_pdl(evict_move_kernel, dim3(units), dim3(kThreads), 0, st, e));
        return true;
    }
    const int chunks = ceil_div(e.keep, 256 / (e.row_bytes / 16));
    if (chunks == 0) return true;
    NB_CUDA_TRY(launch_pdl(evict_gather_kernel, dim3(units * chunks), dim3(256), 0, st, e, chunks));
    return true;
}

}  // namespace nb200
