// C ABI of the stateless cache operators: attention behind a shared prefix,
// accumulated key weights, eviction.  Argument checks, the split of the work
// into key ranges, and the workspace.
#include <algorithm>
#include <cmath>
#include <exception>
#include <initializer_list>
#include <string>

#include "../../include/needle2_b200.h"
#include "cache_ops.cuh"
#include "common.cuh"
#include "evict.cuh"
#include "prefix_attention.cuh"

namespace nb200 {
namespace {

constexpr long long kMaxUnits = 0x7fffffff;
// Slots of a cache or prefix: indexes of keys are 32-bit, and the ends of key ranges (up to
// 2^19, of a multiple of 32 keys each, or 2^16 of 128) and loops by a CTA's threads go
// beyond the last one.
constexpr long long kMaxKeys = 0x7e000000;

bool refuse(const char *msg) {
    set_error(msg);
    return false;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Pointer and strides (of axes longer than one) of rows read 16 bytes at a time.
bool rows_ok(const void *p, const long long *stride, std::initializer_list<int> extent, int size, const char *what) {
    if (!p) return refuse((std::string(what) + " is null").c_str());
    bool ok = aligned16(p);
    for (int n : extent) ok = ok && (n <= 1 || (*stride * size) % 16 == 0), ++stride;
    return ok || refuse((std::string(what) + ": the pointer and the strides must be multiples of 16 bytes").c_str());
}

bool sizes_ok(const needle2_prefix_attention_args &a) {
    if (a.batch < 0 || a.tokens < 0 || a.heads < 1 || a.kvheads < 1 || a.prefix < 0 || a.capacity < 0 || a.window < 0)
        return refuse("prefix attention: negative size");
    if (a.heads % a.kvheads) return refuse("prefix attention: heads must be a multiple of kvheads");
    if (a.head_dim != 64 && a.head_dim != 128) return refuse("prefix attention: head_dim must be 64 or 128");
    if (a.cache_type < 0 || a.cache_type > 2) return refuse("prefix attention: unknown cache type");
    if (!(a.scale > 0.f) || !std::isfinite(a.scale))
        return refuse("prefix attention: scale must be positive and finite");
    const long long rows = (long long)a.batch * a.tokens;
    // units of work, row numbers and the first key of a window (before a sequence's, where it is
    // shorter) are 32-bit
    if (a.capacity > kMaxKeys || a.prefix > kMaxKeys || rows * a.heads > kMaxUnits / 4 ||
        (a.window < a.capacity && (long long)a.window + a.tokens > kMaxKeys) ||
        (long long)a.batch * a.kvheads > kMaxUnits / 64 ||
        (long long)a.batch * a.kvheads * (((long long)a.capacity + 63) / 64) > kMaxUnits)
        return refuse("prefix attention: the call is too large");
    return true;
}

constexpr int kJointKeys = 512;
constexpr long long kMaxLogits = 1LL << 27;   // kept for the weights

struct Plan {
    PrefixSplit prefix, own;
    bool joint, joint_tiles, logits, neg_lse, weight_tiles, fits;
    long long part_o, part_lse, neg_lse_at, logits_at, q16_at, q16_scale_at, bytes;
};

// Whether the weights may come from the logits that the streaming kernel keeps.
bool keeps_logits(const needle2_prefix_attention_args &a) {
    return a.tokens > 0 && (long long)a.tokens * (a.heads / a.kvheads) <= kMaxLogitRows &&
           (long long)a.batch * a.tokens * a.heads * a.capacity <= kMaxLogits;
}

// The copy engine's maps take strides above zero and below 2^40 bytes; an axis of heads
// or sequences may also stand still (the maps leave it out). Keys of other strides (one
// row expanded along the axis) are streamed, whose loads take any address.
bool can_map(long long stride, long long n, int size) {
    return n <= 1 || (stride > 0 && stride < (1LL << 40) / size);
}
bool can_map_cache(long long key, long long keys, long long head, long long heads, long long seq, long long seqs,
                   int size) {
    return can_map(key, keys, size) && (head == 0 || can_map(head, heads, size)) &&
           (seq == 0 || can_map(seq, seqs, size));
}

int sm_count() {
    static int count[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    if (dev < 0 || dev >= 64) return 148;
    if (!count[dev] && cudaDeviceGetAttribute(&count[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        count[dev] = 148;
    return count[dev];
}

// Keys of a range: products cut their sums to 24 bits towards zero, 16-bit caches' eight
// times 128 keys, INT8's 16 times, by 2^-25 of the end's on the average. So many keys
// stay well within half a step of FP16, and INT8's streaming within 2^-16 (65536 keys
// of one sign in a range: 2^-13.6); its tiles' sums leave the accumulator long before.
constexpr long long kTileKeysI8 = 1LL << 40, kTileKeys16 = 32768, kStreamKeysI8 = 4096, kStreamKeys16 = 1 << 18;

// Query rows of a streaming unit.
int stream_rows(const needle2_prefix_attention_args &a) { return a.cache_type == kCacheI8 ? 8 : 16; }

// `group_rows` query rows in each of `groups` row groups, against up to `keys` keys: in how
// many key ranges streaming (s) and tiles (t) take them. More for more keys.
void ranges_of(const needle2_prefix_attention_args &a, int sms, long long groups, long long group_rows, long long keys,
               PrefixSplit &s, PrefixSplit &t) {
    const bool i8 = a.cache_type == kCacheI8;
    const long long tile_keys = i8 ? kTileKeysI8 : kTileKeys16, stream_keys = i8 ? kStreamKeysI8 : kStreamKeys16;
    t.tiles = true;
    t.alt = group_rows <= 128 || (i8 && a.head_dim == 128);
    const long long tiles = groups * ((group_rows + (t.alt ? 127 : 255)) / (t.alt ? 128 : 256));
    const long long most = (keys + (t.alt ? 511 : 255)) / (t.alt ? 512 : 256);
    t.ranges = (int)std::max((keys + tile_keys - 1) / tile_keys,
                             std::max(1LL, std::min({sms / std::max(1LL, tiles), most, 32LL})));
    const long long units = groups * ((group_rows + stream_rows(a) - 1) / stream_rows(a));
    const long long want = (4LL * sms + units - 1) / std::max(1LL, units);
    s.ranges = (int)std::max((keys + stream_keys - 1) / stream_keys,
                             std::max(1LL, std::min({want, (keys + 255) / 256, 64LL})));
}

long long padded(long long bytes) { return (bytes + 255) / 256 * 256; }

Plan plan_of(const needle2_prefix_attention_args &a) {
    Plan p{};
    const int sms = sm_count();
    const bool i8 = a.cache_type == kCacheI8;
    const int R = a.heads / a.kvheads, tile = stream_rows(a);
    const long long rows = (long long)a.batch * a.tokens * a.heads;
    // Tiles or streaming by their times, fitted to measurements (us): a tile CTA has its
    // multiprocessor to itself and takes 9 beside its keys, whose conversion INT8 waits for,
    // a streaming unit 1.2 beside its keys, of which the 16-bit caches' 128 dimensions take
    // longest.  (358 sequences of 16 rows and 88 INT8 keys: 500 by tiles, 100 streaming; 600
    // KV heads x 24 FP16 rows x 3436 keys: 212, 174; 800 x 10 INT8 rows x 2000: 404, 197;
    // two prompts of 4096 tokens: 340, 5100.)
    // Weights of the own keys: behind tiles a CTA of 256 keys takes the product again;
    // streaming keeps the logits of few rows.  (600 x 24 rows x 3436: 319 and 58.)
    const double key = (i8 ? 4.3e-3 : 6e-3) * (a.head_dim == 128 ? 1.7 : 1.0);
    auto split = [&](long long groups, long long group_rows, long long keys, bool weights, bool mapped) {
        PrefixSplit s, t;
        ranges_of(a, sms, groups, group_rows, keys, s, t);
        if (group_rows <= tile || !mapped) return s;
        const long long tiles = groups * ((group_rows + (t.alt ? 127 : 255)) / (t.alt ? 128 : 256));
        const long long units = groups * ((group_rows + tile - 1) / tile);
        const double waves = std::max(1.0, (double)tiles * t.ranges / sms);
        const double tile_key =
            i8 ? (a.head_dim == 128 ? 33e-3 : 29e-3) : (t.alt ? 11e-3 : 14.5e-3) * (a.head_dim == 128 ? 1.3 : 1.0);
        double by_tiles = waves * (9.0 + tile_key * (double)keys / t.ranges);
        double streaming = 4.0 + units * (1.2 + key * (double)keys) / sms;
        if (weights) {
            const double ctas = std::max(1.0, (double)groups * ((a.capacity + 255) / 256) / sms);
            const double again = 5.0 + ctas * (a.head_dim == 128 ? 7.5 : 5.7);
            by_tiles += again;
            streaming += keeps_logits(a) ? 3.0 + std::max(0.3 * group_rows, groups * group_rows * 1.1e-6 * a.capacity)
                                         : again;
        }
        return by_tiles < streaming ? t : s;
    };
    const int span = a.window ? (int)std::min<long long>(a.capacity, (long long)a.window + a.tokens) : a.capacity;
    const int size = i8 ? 1 : 2;
    const long long seqs = a.cache_rows ? 2 : a.batch;      // (of the cache: known to the caller only)
    auto own_mapped = [&](const long long (&s)[3]) {
        return can_map_cache(s[2], a.capacity, s[1], a.kvheads, s[0], seqs, size);
    };
    auto prefix_mapped = [&](const long long (&s)[2]) {
        return can_map_cache(s[1], a.prefix, s[0], a.kvheads, 0, 1, size);
    };
    if (a.capacity || !a.prefix)
        p.own = split((long long)a.batch * a.kvheads, (long long)a.tokens * R, span, a.weights != nullptr,
                      own_mapped(a.k_stride) && own_mapped(a.v_stride));
    if (a.prefix)
        p.prefix = split(a.kvheads, (long long)a.batch * a.tokens * R, a.prefix, false,
                         prefix_mapped(a.prefix_k_stride) && prefix_mapped(a.prefix_v_stride));
    // few rows and keys: one kernel whose units take both key sets one after the other
    p.joint = a.prefix && a.capacity && !p.own.tiles && !p.prefix.tiles && a.prefix + (long long)span <= kJointKeys;
    if (p.joint) {
        p.prefix.ranges = 0;
        p.own.ranges = 1;
    }
    // tiles of the sequences' own rows that fill the machine take the prefix first, in
    // the same accumulators: no partial results
    p.joint_tiles = a.prefix && p.own.tiles && p.prefix.tiles && p.own.ranges == 1 &&
                    (i8 || a.prefix + (long long)span <= kTileKeys16) &&
                    (long long)a.batch * a.kvheads * ((a.tokens * R + 255) / 256) * 5 >= 4LL * sms;
    if (p.joint_tiles) p.prefix = PrefixSplit{};
    if (!a.capacity && p.own.ranges) {               // no key at all: the streaming kernel writes the zeros
        p.own = PrefixSplit{};
        p.own.ranges = 1;
    }
    p.logits = a.weights && !p.own.tiles && keeps_logits(a);
    p.neg_lse = a.weights != nullptr;
    // (INT8's queries are split into the workspace first, whatever their strides)
    const bool q_mapped = i8 || (can_map(a.q_stride[0], a.batch, 2) && can_map(a.q_stride[1], a.tokens, 2) &&
                                 can_map(a.q_stride[2], a.heads, 2));
    p.weight_tiles = a.weights && !p.logits && a.tokens > 0 && R <= 128 && q_mapped;
    long long at = 0;
    auto take = [&](long long bytes) {
        const long long r = at;
        at += padded(bytes);
        return r;
    };
    const int n = p.own.slots() + p.prefix.slots();
    if (n > 1) {
        p.part_o = take(rows * n * a.head_dim * 4);
        p.part_lse = take(rows * n * 4);
    }
    if (p.neg_lse) p.neg_lse_at = take(rows * 4);
    if (p.logits) p.logits_at = take((long long)a.batch * a.kvheads * a.tokens * R * a.capacity * 4);
    if (p.weight_tiles && a.cache_type == kCacheI8) {
        p.q16_at = take(rows * a.head_dim * 4);
        p.q16_scale_at = take(rows * 4);
    }
    p.bytes = n > 1 ? at + 16 : at;              // partial rows lie on 32 bytes, the workspace on 16
    // (more rows than a tile against keys that cannot be mapped, in many ranges)
    auto units = [&](const PrefixSplit &s, long long groups, long long group_rows) {
        const int unit_rows = s.tiles ? 128 : tile;
        return groups * ((group_rows + unit_rows - 1) / unit_rows) * s.ranges;
    };
    p.fits = units(p.own, (long long)a.batch * a.kvheads, (long long)a.tokens * R) +
                 units(p.prefix, a.kvheads, (long long)a.batch * a.tokens * R) <= kMaxUnits;
    return p;
}

bool plan_call(const needle2_prefix_attention_args &a, Plan &p) {
    if (!sizes_ok(a)) return false;
    p = plan_of(a);
    return p.fits || refuse("prefix attention: the call is too large");
}

template <int N>
void copy(long long (&to)[N], const long long (&from)[N]) {
    for (int i = 0; i < N; ++i) to[i] = from[i];
}

bool attention(const needle2_prefix_attention_args &a, void *workspace, long long bytes, cudaStream_t st) {
    if (!sizes_ok(a)) return false;
    if (a.batch == 0) return true;
    const int size = a.cache_type == kCacheI8 ? 1 : 2, qsize = a.cache_type == kCacheI8 ? 4 : 2;
    const bool i8 = a.cache_type == kCacheI8;
    if (a.tokens > 0) {
        if (!rows_ok(a.q, a.q_stride, {a.batch, a.tokens, a.heads}, qsize, "q") ||
            !rows_ok(a.out, a.out_stride, {a.batch, a.tokens, a.heads}, qsize, "out"))
            return false;
    }
    if (a.capacity) {
        // (with cache_rows the first axis is the cache's, which this call does not know)
        const int lead = a.cache_rows ? 2 : a.batch;
        if (!rows_ok(a.k, a.k_stride, {lead, a.kvheads, a.capacity}, size, "k") ||
            !rows_ok(a.v, a.v_stride, {lead, a.kvheads, a.capacity}, size, "v"))
            return false;
        if (i8 && (!a.k_scales || !a.v_scales)) return refuse("an INT8 cache needs its scales");
    }
    if (a.prefix) {
        if (!rows_ok(a.prefix_k, a.prefix_k_stride, {a.kvheads, a.prefix}, size, "prefix_k") ||
            !rows_ok(a.prefix_v, a.prefix_v_stride, {a.kvheads, a.prefix}, size, "prefix_v"))
            return false;
        if (i8 && (!a.prefix_k_scales || !a.prefix_v_scales)) return refuse("an INT8 prefix needs its scales");
    }
    if (!a.lengths) return refuse("lengths is null");
    if ((a.weights != nullptr) != (a.weights_out != nullptr))
        return refuse("weights and weights_out go together");
    Plan plan;
    if (!plan_call(a, plan)) return false;
    if (bytes < plan.bytes || (plan.bytes && (!workspace || !aligned16(workspace))))
        return refuse("prefix attention: the workspace is too small or not 16-byte aligned");
    PrefixAttn p{};
    p.batch = a.batch; p.tokens = a.tokens; p.heads = a.heads; p.kvheads = a.kvheads;
    p.group = a.heads / a.kvheads; p.hd = a.head_dim;
    p.prefix = a.prefix; p.capacity = a.capacity; p.type = a.cache_type;
    p.window = a.window >= a.capacity ? 0 : a.window;   // own indexes are below the capacity
    p.scale2 = a.scale * 1.4426950408889634f;
    p.q = a.q; p.out = a.out; p.k = a.k; p.v = a.v; p.pk = a.prefix_k; p.pv = a.prefix_v;
    p.kscale = a.k_scales; p.vscale = a.v_scales; p.pkscale = a.prefix_k_scales; p.pvscale = a.prefix_v_scales;
    copy(p.qs, a.q_stride); copy(p.os, a.out_stride); copy(p.ks, a.k_stride); copy(p.vs, a.v_stride);
    copy(p.kss, a.k_scale_stride); copy(p.vss, a.v_scale_stride);
    copy(p.pks, a.prefix_k_stride); copy(p.pvs, a.prefix_v_stride);
    copy(p.pkss, a.prefix_k_scale_stride); copy(p.pvss, a.prefix_v_scale_stride);
    p.lengths = a.lengths; p.ntokens = a.token_counts; p.cache_row = a.cache_rows;
    p.lse = a.lse;
    p.weights = a.weights; p.weights_out = a.weights_out;
    copy(p.ws, a.weights_stride); copy(p.wos, a.weights_out_stride);
    p.prefix_slots = plan.prefix.slots();
    p.own_slots = plan.own.slots();
    char *base = static_cast<char *>(workspace);
    const int n = p.own_slots + p.prefix_slots;
    if (n > 1) {
        base += reinterpret_cast<uintptr_t>(base) % 32;
        p.part_o = reinterpret_cast<float *>(base + plan.part_o);
        p.part_lse = reinterpret_cast<float *>(base + plan.part_lse);
    }
    if (plan.neg_lse) p.neg_lse = reinterpret_cast<float *>(base + plan.neg_lse_at);
    if (plan.logits) p.logits = reinterpret_cast<float *>(base + plan.logits_at);
    if (a.tokens > 0) {
        const bool stream_prefix = plan.prefix.ranges && !plan.prefix.tiles;
        const bool stream_own = plan.own.ranges && !plan.own.tiles;
        const bool tiles = plan.prefix.tiles || plan.own.tiles, stream = stream_prefix || stream_own;
        // the first axis of a cache addressed by cache_rows has an extent that only the caller knows
        if (tiles &&
            !launch_prefix_tiles(p, plan.prefix, plan.own, plan.joint_tiles, a.cache_rows ? 1LL << 30 : a.batch, stream,
                                 st))
            return false;
        if (stream && !launch_prefix_stream(p, stream_prefix, stream_own, plan.joint, tiles, st)) return false;
    }
    if (!launch_prefix_finish(p, st)) return false;
    if (!a.weights || plan.logits) return true;
    if (!plan.weight_tiles) return launch_key_weights(p, st);
    if (a.cache_type == kCacheI8) {
        p.q16 = base + plan.q16_at;
        p.q16_scale = reinterpret_cast<float *>(base + plan.q16_scale_at);
    }
    return launch_weight_tiles(p, st);
}

bool evict(const needle2_evict_args &a, cudaStream_t st) {
    if (a.batch < 0 || a.kvheads < 1 || a.capacity < 0 || a.keep < 0 || a.first < 0 || a.recent < 0)
        return refuse("evict: negative size");
    if (a.head_dim != 64 && a.head_dim != 128) return refuse("evict: head_dim must be 64 or 128");
    if (a.cache_type < 0 || a.cache_type > 2) return refuse("evict: unknown cache type");
    if ((long long)a.first + a.recent > a.keep) return refuse("evict: first + recent must not exceed keep");
    if (a.out_capacity < a.keep) return refuse("evict: the output holds fewer than keep slots");
    if ((long long)a.batch * a.kvheads > kMaxUnits / 64 ||
        (long long)a.batch * a.kvheads * (((long long)a.keep + 15) / 16) > kMaxUnits || a.capacity > kMaxKeys ||
        a.out_capacity > kMaxKeys)
        return refuse("evict: the call is too large");
    if (a.batch == 0) return true;
    const int size = a.cache_type == kCacheI8 ? 1 : 2;
    if (!a.lengths || !a.lengths_out || (a.keep && !a.indices)) return refuse("evict: null pointer");
    if (a.lengths == a.lengths_out) return refuse("evict: lengths_out must not be lengths");
    if (a.capacity) {
        if (!rows_ok(a.k, a.k_stride, {a.batch, a.kvheads, a.capacity}, size, "k") ||
            !rows_ok(a.v, a.v_stride, {a.batch, a.kvheads, a.capacity}, size, "v"))
            return false;
        if (!a.weights) return refuse("evict: weights is null");
    }
    if (a.out_capacity) {
        if (!rows_ok(a.k_out, a.k_out_stride, {a.batch, a.kvheads, a.out_capacity}, size, "k_out") ||
            !rows_ok(a.v_out, a.v_out_stride, {a.batch, a.kvheads, a.out_capacity}, size, "v_out"))
            return false;
        if (!a.weights_out) return refuse("evict: weights_out is null");
    }
    const bool i8 = a.cache_type == kCacheI8;
    if (i8 && ((a.capacity && (!a.k_scales || !a.v_scales)) ||
               (a.out_capacity && (!a.k_scales_out || !a.v_scales_out))))
        return refuse("evict: an INT8 cache needs its scales");
    auto same = [](const long long *x, const long long *y) { return x[0] == y[0] && x[1] == y[1] && x[2] == y[2]; };
    const bool in_place = a.k == a.k_out;
    if (in_place && a.capacity) {
        bool ok = a.v == a.v_out && a.weights == a.weights_out && a.out_capacity == a.capacity &&
                  same(a.k_stride, a.k_out_stride) && same(a.v_stride, a.v_out_stride) &&
                  same(a.weights_stride, a.weights_out_stride);
        if (i8)
            ok = ok && a.k_scales == a.k_scales_out && a.v_scales == a.v_scales_out &&
                 same(a.k_scale_stride, a.k_scale_out_stride) && same(a.v_scale_stride, a.v_scale_out_stride);
        if (!ok) return refuse("evict: in place, every output must be its input");
    }
    Evict e{};
    e.batch = a.batch; e.kvheads = a.kvheads; e.capacity = a.capacity; e.out_capacity = a.out_capacity;
    e.keep = a.keep; e.first = a.first; e.recent = a.recent;
    e.row_bytes = a.head_dim * size;
    e.k = (const char *)a.k; e.v = (const char *)a.v; e.ko = (char *)a.k_out; e.vo = (char *)a.v_out;
    for (int i = 0; i < 3; ++i) {
        e.ks[i] = a.k_stride[i] * size; e.vs[i] = a.v_stride[i] * size;
        e.kos[i] = a.k_out_stride[i] * size; e.vos[i] = a.v_out_stride[i] * size;
    }
    if (i8) {
        e.kscale = a.k_scales; e.vscale = a.v_scales; e.kscale_o = a.k_scales_out; e.vscale_o = a.v_scales_out;
    }
    copy(e.kss, a.k_scale_stride); copy(e.vss, a.v_scale_stride);
    copy(e.ksos, a.k_scale_out_stride); copy(e.vsos, a.v_scale_out_stride);
    e.weights = a.weights; e.weights_o = a.weights_out;
    copy(e.ws, a.weights_stride); copy(e.wos, a.weights_out_stride);
    e.lengths = a.lengths; e.lengths_o = a.lengths_out; e.indices = a.indices;
    e.in_place = in_place;
    return launch_evict(e, st);
}

}  // namespace

long long prefix_attention_workspace(const needle2_prefix_attention_args &a) {
    Plan plan;
    return plan_call(a, plan) ? plan.bytes : -1;
}
long long prefix_attention_workspace_most(const needle2_prefix_attention_args &a) {
    if (!sizes_ok(a)) return -1;
    const int sms = sm_count();
    const int R = a.heads / a.kvheads;
    long long most = 0;
    for (long long batch = 1; batch <= a.batch; ++batch) {
        auto slots = [&](long long groups, long long group_rows, long long keys) {
            PrefixSplit s, t;
            ranges_of(a, sms, groups, group_rows, keys, s, t);
            return (long long)(group_rows <= stream_rows(a) ? s.slots() : std::max(s.slots(), t.slots()));
        };
        const long long rows = batch * a.heads, n = slots(batch * a.kvheads, R, a.capacity) +
                                                    (a.prefix ? slots(a.kvheads, batch * R, a.prefix) : 0);
        if (n > 1) most = std::max(most, padded(rows * n * a.head_dim * 4) + padded(rows * n * 4) + 16);
    }
    return most;
}
bool prefix_attention(const needle2_prefix_attention_args &a, void *workspace, long long bytes, cudaStream_t st) {
    return attention(a, workspace, bytes, st);
}

}  // namespace nb200

namespace {

// No exception leaves a C entry.
template <typename F>
long long entry(const void *args, F f) {
    nb200::clear_error();
    if (!args) {
        nb200::set_error("null arguments");
        return -1;
    }
    try {
        return f();
    } catch (const std::exception &e) {
        nb200::set_error(e.what());
    }
    return -1;
}

}  // namespace

extern "C" {

long long needle2_prefix_attention_workspace(const needle2_prefix_attention_args *args) {
    return entry(args, [&] { return nb200::prefix_attention_workspace(*args); });
}

int needle2_prefix_attention_device(const needle2_prefix_attention_args *args, void *workspace,
                                    long long workspace_bytes, void *stream) {
    return (int)entry(args, [&]() -> long long {
        return nb200::prefix_attention(*args, workspace, workspace_bytes, static_cast<cudaStream_t>(stream)) ? 0 : -1;
    });
}

int needle2_evict_device(const needle2_evict_args *args, void *stream) {
    return (int)entry(args, [&]() -> long long {
        return nb200::evict(*args, static_cast<cudaStream_t>(stream)) ? 0 : -1;
    });
}

}  // extern "C"
