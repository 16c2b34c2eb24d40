// Attention of a batch that shares a prefix, over caches of INT8 rows with FP32
// scales or of 16-bit values, and the softmax weights its own keys receive:
// parameters and launches shared by prefix_attention.cu (streaming kernel for
// few rows, the merge of partial results, key weights), prefix_attention_tc.cu
// (tcgen05 tiles for many rows) and the C ABI.
//
// Rows.  For one KV head, row m = (b * tokens + t) * R + r stands for query
// token t of sequence b and query head g * R + r (R = heads / kvheads).  The
// prefix takes all B * tokens * R rows as one matrix; a sequence's own keys
// take its tokens * R consecutive rows.
//
// Partial results.  Disjoint key ranges of one row are attended separately;
// each yields o = sum_j e^(z_j - lse) v_j and lse = log2 sum_j 2^(z_j) over its
// range (z in log2 units; -inf and unwritten o for an empty range), and
// out = sum_i 2^(lse_i - L) o_i with L = log2 sum_i 2^(lse_i).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace nb200 {

constexpr int kMaxLogitRows = 64;   // query rows of a KV head up to which the weights may come from kept logits

enum CacheType { kCacheI8 = 0, kCacheBF16 = 1, kCacheF16 = 2 };

struct PrefixAttn {
    int batch, tokens, heads, kvheads, group, hd;   // group = heads / kvheads
    int prefix, capacity, window, type;
    float scale2;                                    // softmax scale * log2(e)
    const void *q;                                   // f32 (INT8 cache) or the cache's type
    long long qs[3];                                 // strides in elements: batch, token, head
    void *out;
    long long os[3];
    const void *k, *v;
    long long ks[3], vs[3];                          // batch, KV head, key
    const float *kscale, *vscale;
    long long kss[3], vss[3];
    const void *pk, *pv;
    long long pks[2], pvs[2];                        // KV head, key
    const float *pkscale, *pvscale;
    long long pkss[2], pvss[2];
    const int *lengths;                              // own keys of each sequence, the new tokens' among them
    const int *ntokens;                              // queries of each sequence (null: `tokens`)
    const int *cache_row;                            // row of k, v and scales of each sequence (null: its own index)
    float *lse;                                      // [B][tokens][heads], natural log (null: not written)
    const float *weights;
    long long ws[3];
    float *weights_out;
    long long wos[3];
    // partial results, in the caller's workspace
    int prefix_slots, own_slots;                     // key ranges of the prefix and of the own keys
    float *part_o;                                   // [slots][rows][hd], rows = B * tokens * heads as out's
    float *part_lse;                                 // [slots][rows]
    float *neg_lse;                                  // [B][kvheads][tokens * R], minus log2's lse (null: not needed)
    void *q16;                                       // weights of an INT8 cache's many rows: split queries
    float *q16_scale;                                // and their factors
    float *logits;                                   // [B * kvheads][tokens * R][capacity], log2 (null: not kept)
};

__device__ __forceinline__ int own_length(const PrefixAttn &p, int b) {
    return max(0, min(p.lengths[b], p.capacity));
}
// The place of token t, head h of sequence b in neg_lse.
__device__ __forceinline__ long long neg_lse_at(const PrefixAttn &p, int b, int t, int h) {
    return (((long long)b * p.kvheads + h / p.group) * p.tokens + t) * p.group + h % p.group;
}
__device__ __forceinline__ int own_tokens(const PrefixAttn &p, int b) {
    return p.ntokens ? max(0, min(p.ntokens[b], p.tokens)) : p.tokens;
}

// f of the cache type and the head dimension as compile-time constants.
template <typename F>
bool by_geometry(const PrefixAttn &p, F f) {
    using I8 = std::integral_constant<int, kCacheI8>;
    using BF = std::integral_constant<int, kCacheBF16>;
    using F16 = std::integral_constant<int, kCacheF16>;
    using D64 = std::integral_constant<int, 64>;
    using D128 = std::integral_constant<int, 128>;
    if (p.hd == 64)
        return p.type == kCacheI8 ? f(I8(), D64()) : p.type == kCacheBF16 ? f(BF(), D64()) : f(F16(), D64());
    return p.type == kCacheI8 ? f(I8(), D128()) : p.type == kCacheBF16 ? f(BF(), D128()) : f(F16(), D128());
}

// How one set of keys is attended: by the streaming kernel or by tiles, in how
// many key ranges; `alt`: both row tiles of a CTA on the same rows and alternate
// key tiles, each with its partial result.
struct PrefixSplit {
    bool tiles = false, alt = false;
    int ranges = 0;
    int slots() const { return alt ? 2 * ranges : ranges; }
};

// The merge of the partial results, weights of few rows from kept logits, and
// weights of any number of rows from neg_lse.
bool launch_prefix_finish(const PrefixAttn &p, cudaStream_t st);
bool launch_key_weights(const PrefixAttn &p, cudaStream_t st);
// Streaming kernel: `prefix` / `own` say which key sets it takes; after_tiles:
// the tile kernel of the same call was launched before it with stream_next, may
// still run, and has ended when it ends; joint: the own keys' units take the
// prefix too (prefix_slots 0).
bool launch_prefix_stream(const PrefixAttn &p, bool prefix, bool own, bool joint, bool after_tiles, cudaStream_t st);
// Tile kernel for the sets whose split says `tiles`; joint: the own keys' units
// take the prefix too (prefix_slots 0); cache_rows: extent of the first axis of k
// and v; stream_next: the streaming kernel of the same call follows.
bool launch_prefix_tiles(const PrefixAttn &p, const PrefixSplit &prefix, const PrefixSplit &own, bool joint,
                         long long cache_rows, bool stream_next, cudaStream_t st);
// Weights of many rows from neg_lse (and, INT8, q16): group up to 128.
bool launch_weight_tiles(const PrefixAttn &p, cudaStream_t st);
// 1 if a bounded wait of the tile kernels ran out since the last call, -1 if
// the flag could not be read.
int read_and_clear_tile_fault();

}  // namespace nb200
