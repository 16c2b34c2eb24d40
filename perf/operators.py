"""Measured cases of the cache operators in openneedle_b200.attention:

* prefix   -- ``prefix_attention``: every sequence of a batch attends to one
  shared prefix and to its own cached keys (one new token per sequence while
  decoding, several while a chunk is prefilled or drafted tokens are checked);
* weigh    -- ``accumulate_attention``: the same attention, which also adds to
  each of a sequence's own keys the softmax weight that the call gave it;
* evict    -- ``evict``: keeps, per sequence and KV head, the first and the
  most recent keys and those of the largest accumulated weight, and packs the
  cache.

With z[t, j] = scale * q_t . k_j over the P prefix keys and the own keys
j in (i - window, i] of query t at own index i = length - tokens + t:
  out_t = sum_j softmax(z_t)_j v_j,  weights_j += sum over t and the KV head's
query heads of softmax(z_t)_j.  An INT8 cache holds k = k8 * k_scale with one
FP32 scale per key and KV head, and the same for v.

``run`` computes the plain form with elementary torch operations in 32 bits, or
(``own``) calls the library.  Layouts: q, out [B, T, H, D]; k, v [B, KV, S, D];
prefix k, v [KV, P, D]; scales and weights without the last axis.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _attend(name, op, cache, b, t, heads, kv, d, p, s, lens, window=0, lse=False):
    return {"name": name, "op": op, "cache": cache, "b": b, "t": t, "heads": heads, "kv": kv, "d": d, "p": p, "s": s,
            "lens": lens, "window": window, "lse": lse}


def _evict(name, cache, b, kv, d, s, keep, first, recent, lens):
    return {"name": name, "op": "evict", "cache": cache, "b": b, "kv": kv, "d": d, "s": s, "keep": keep,
            "first": first, "recent": recent, "lens": lens}


def listed():
    return [
        # one session of the 12-layer, 512-wide model's geometry, a few tokens after a short prompt: latency
        _attend("prefix one session", "prefix", "int8", 1, 1, 8, 4, 64, 48, 64, "ragged"),
        # 256 sessions behind a 384-token tool prefix at context 4096: the own keys' bytes decide
        _attend("prefix decode 4096 int8", "prefix", "int8", 256, 1, 8, 4, 64, 384, 3712, "full"),
        # 1024 sessions early in their answers behind a long shared prompt
        _attend("prefix 1024 sessions int8", "prefix", "int8", 1024, 1, 8, 4, 64, 2048, 64, "ragged"),
        # a 16k document asked about by 128 users, 16-bit cache
        _attend("prefix document bf16", "prefix", "bf16", 128, 1, 32, 8, 128, 16384, 256, "ragged"),
        # a chunk of 37 new tokens per sequence (prefill of a query, or drafted tokens), own keys in a window
        _attend("prefix chunk f16", "prefix", "f16", 16, 37, 16, 2, 64, 4096, 509, "ragged", 128, True),
        # decode of two short sequences that keep their weights: latency
        _attend("weigh two sequences", "weigh", "bf16", 2, 1, 8, 4, 64, 0, 200, "ragged"),
        # decode of 64 sessions whose caches are to be thinned out, behind the tool prefix
        _attend("weigh decode int8", "weigh", "int8", 64, 1, 8, 4, 64, 384, 4001, "ragged"),
        # a chunk after a shared prefix, one KV head per query head
        _attend("weigh chunk f16", "weigh", "f16", 8, 257, 8, 8, 128, 1000, 700, "ragged"),
        # two prompts of 4096 tokens, prefilled whole before their caches are thinned out
        _attend("weigh prefill bf16", "weigh", "bf16", 2, 4096, 32, 8, 128, 0, 4096, "full"),
        # one sequence: latency
        _evict("evict one sequence", "int8", 1, 4, 64, 509, 128, 4, 32, "full"),
        # 256 sessions at context 4096, thinned to a quarter
        _evict("evict 256 sessions int8", "int8", 256, 4, 64, 3712, 1024, 4, 128, "ragged"),
        # two long documents
        _evict("evict document bf16", "bf16", 2, 8, 128, 65536, 8192, 16, 1024, "full"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = max(_cost(c) for c in listed() if c["op"] != "evict")
    most_evict = max(_cost(c) for c in listed() if c["op"] == "evict")
    while True:
        op = rng.choice(("prefix", "prefix", "weigh", "weigh", "evict"))
        cache = rng.choice(("int8", "bf16", "f16"))
        d = rng.choice((64, 128))
        heads, kv = rng.choice(((8, 4), (8, 8), (16, 2), (32, 8), (4, 1), (6, 2), (12, 4)))
        lens = rng.choice(("full", "ragged", "ragged"))
        if op == "evict":
            s = _log(rng, 32, 65536)
            keep = max(1, min(s, _log(rng, max(1, s // 16), s)))
            first = min(keep, rng.choice((0, 1, 4, 16)))
            c = _evict("", cache, _log(rng, 1, 256), kv, d, s, keep, first, rng.randint(0, (keep - first) // 2), lens)
            fits = _cost(c) <= most_evict
        else:
            t = 1 if rng.random() < 0.5 else _log(rng, 2, 2048)
            p = 0 if rng.random() < 0.2 else _log(rng, 16, 16384)
            s = max(t, _log(rng, 8, 4096))
            c = _attend("", op, cache, _log(rng, 1, 1024), t, heads, kv, d, p, s, lens,
                        rng.choice((0, 0, _log(rng, 8, 2048))), op == "prefix" and rng.random() < 0.3)
            fits = _cost(c) <= most
        if fits:
            del c["name"]
            return c


def _lengths(case):
    """Own keys of each sequence: all of the capacity, or spread over it (a new session that has none or one among
    them); at least the call's own tokens."""
    b, s, t = case["b"], case["s"], case.get("t", 1)
    if case["lens"] == "full":
        return [s] * b
    lens = [t + int((s - t) * ((0.37 + 0.6180339887 * i) % 1.0)) for i in range(b)]
    if t == 1 and b >= 8:
        lens[1], lens[5] = 0, 1
    return lens


def _pairs(case):
    """(query, own key) pairs of one query head over the batch, and own keys that any query reads."""
    pairs = keys = 0
    t, w = case["t"], case["window"]
    for n in _lengths(case):
        m = min(n, t)                                   # queries that see own keys
        if w:
            full = max(0, min(m, n - w + 1))            # queries whose window is full
            rest = m - full
            pairs += full * w + rest * (n - m) + rest * (rest + 1) // 2
            keys += min(n, w + t - 1)
        else:
            pairs += m * (n - m) + m * (m + 1) // 2
            keys += n
    return pairs, keys


def work(case):
    lens = _lengths(case)
    row = case["d"] + 4 if case["cache"] == "int8" else 2 * case["d"]      # bytes of one key of one KV head
    kv = case["kv"]
    if case["op"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lens)
        # weights and kept rows read; kept rows, weights and indices of every output slot written
        moved = kv * (4 * sum(lens) + 4 * kept * row + 8 * case["b"] * case["keep"])
        return {"bytes": moved + 8 * case["b"], "flops": 0}
    pairs, keys = _pairs(case)
    rows = case["b"] * case["t"] * case["heads"]
    size = 4 if case["cache"] == "int8" else 2
    moved = 2 * rows * case["d"] * size + 2 * kv * (keys + case["p"]) * row + 4 * case["b"]
    if case["lse"]:
        moved += 4 * rows
    if case["op"] == "weigh":
        moved += 8 * kv * case["b"] * case["s"]
    return {"bytes": moved, "flops": 4 * case["d"] * (case["heads"] * pairs + rows * case["p"])}


def _cost(case):
    """What draw() compares: the plain form's traffic grows with the pairs, the weights' and sorts' with the slots."""
    w = work(case)
    if case["op"] == "evict":
        return max(w["bytes"], 4 * case["b"] * case["kv"] * case["s"] * case["d"])
    slots = case["b"] * case["t"] * case["heads"] * (case["p"] + case["s"])
    return max(w["flops"] / 2e5, w["bytes"] / 4e3, slots / 5e2, case["b"] * case["kv"] * case["s"] * case["d"] / 1e3)


def _cache(g, case, lead, keys):
    """K or V of `keys` keys: codes and scales (INT8: code 127 at each row's largest), or values."""
    x = torch.randn(*lead, keys, case["d"], generator=g, device="cuda", dtype=torch.float32)
    # keys differ in size, as the positions and tokens of a text do
    x *= torch.exp(0.3 * torch.randn(*lead, keys, 1, generator=g, device="cuda"))
    if case["cache"] != "int8":
        return x.to(TYPES[case["cache"]]), None
    most = x.abs().amax(-1, keepdim=True)
    return torch.round(x * (127.0 / most)).clamp_(-127, 127).to(torch.int8), (most / 127.0)[..., 0].contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    b, kv, s, d = case["b"], case["kv"], case["s"], case["d"]
    st = {"case": case}
    st["k"], st["ks"] = _cache(g, case, (b, kv), s)
    st["v"], st["vs"] = _cache(g, case, (b, kv), s)
    order = np.random.RandomState(seed % (1 << 31)).permutation(b)
    st["lengths"] = torch.tensor([_lengths(case)[i] for i in order], dtype=torch.int32, device="cuda")
    if case["op"] != "prefix":
        # what earlier calls accumulated, each query a total of one: heavy-tailed, and keys that no query ever gave a
        # weight above zero
        w = torch.exp(2.0 * torch.randn(b, kv, s, generator=g, device="cuda")) / s
        st["weights"] = torch.where(torch.rand(b, kv, s, generator=g, device="cuda") < 0.25, torch.zeros_like(w), w)
    if case["op"] == "evict":
        keep = case["keep"]
        st["out"] = {"k": torch.zeros_like(st["k"][:, :, :keep]), "v": torch.zeros_like(st["v"][:, :, :keep]),
                     "weights": torch.zeros(b, kv, keep, device="cuda"),
                     "indices": torch.zeros(b, kv, keep, dtype=torch.int32, device="cuda"),
                     "lengths": torch.zeros(b, dtype=torch.int32, device="cuda")}
        if st["ks"] is not None:
            st["out"]["k_scales"] = torch.zeros(b, kv, keep, device="cuda")
            st["out"]["v_scales"] = torch.zeros(b, kv, keep, device="cuda")
        return st
    q = 1.5 * torch.randn(b, case["t"], case["heads"], d, generator=g, device="cuda")
    st["q"] = q if case["cache"] == "int8" else q.to(TYPES[case["cache"]])
    if case["p"]:
        st["pk"], st["pks"] = _cache(g, case, (kv,), case["p"])
        st["pv"], st["pvs"] = _cache(g, case, (kv,), case["p"])
    return st


# ---- the plain forms -------------------------------------------------------

def _float(x, scales):
    return x.float() if scales is None else x.float() * scales.unsqueeze(-1)


def _plain_attention(st):
    c = st["case"]
    b, t, h, kv, d, p, s = (c[n] for n in ("b", "t", "heads", "kv", "d", "p", "s"))
    r, scale = h // kv, d ** -0.5
    # queries by KV head: [B, KV, T * R, D]
    q = st["q"].float().reshape(b, t, kv, r, d).permute(0, 2, 1, 3, 4).reshape(b, kv, t * r, d)
    k, v = _float(st["k"], st["ks"]), _float(st["v"], st["vs"])
    # own index of each query, and the own keys that it sees
    i = (st["lengths"].view(b, 1) - t + torch.arange(t, device="cuda")).repeat_interleave(r, 1).view(b, 1, t * r, 1)
    j = torch.arange(s, device="cuda")
    seen = j <= i
    if c["window"]:
        seen = seen & (j > i - c["window"])
    z = torch.matmul(q, k.transpose(2, 3)) * scale
    z = z.masked_fill(~seen, -math.inf)
    top = z.amax(-1, keepdim=True)
    if p:
        pk, pv = _float(st["pk"], st["pks"]), _float(st["pv"], st["pvs"])
        qp = q.permute(1, 0, 2, 3).reshape(kv, b * t * r, d)
        zp = torch.matmul(qp, pk.transpose(1, 2)) * scale
        top = torch.maximum(top, zp.amax(-1).view(kv, b, t * r, 1).permute(1, 0, 2, 3))
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(z.sub_(top))
    total = e.sum(-1, keepdim=True)
    # keys behind a sequence's length hold nothing
    v = v.masked_fill(j.view(1, 1, s, 1) >= st["lengths"].view(b, 1, 1, 1), 0.0)
    o = torch.matmul(e, v)
    if p:
        ep = torch.exp(zp.sub_(top.permute(1, 0, 2, 3).reshape(kv, b * t * r, 1)))
        total = total + ep.sum(-1).view(kv, b, t * r, 1).permute(1, 0, 2, 3)
        o = o + torch.matmul(ep, pv).view(kv, b, t * r, d).permute(1, 0, 2, 3)
    some = torch.where(total > 0, total, torch.ones_like(total))
    o = (o / some).view(b, kv, t, r, d).permute(0, 2, 1, 3, 4).reshape(b, t, h, d).to(st["q"].dtype)
    if c["op"] == "weigh":
        return {"out": o, "weights": st["weights"] + (e / some).sum(2)}
    if c["lse"]:
        lse = (top + torch.log(total)).view(b, kv, t, r).permute(0, 2, 1, 3).reshape(b, t, h)
        return {"out": o, "lse": lse}
    return {"out": o}


def _plain_evict(st):
    c, out = st["case"], st["out"]
    s, keep, first, recent = (c[n] for n in ("s", "keep", "first", "recent"))
    b, kv = c["b"], c["kv"]
    n = st["lengths"].view(b, 1, 1)
    j = torch.arange(s, device="cuda")
    # kept in any case before all others, keys behind the length after all others, ties to the lowest index
    w = st["weights"].masked_fill((j < first) | (j >= n - recent), math.inf)
    w = w.masked_fill(j >= n, -math.inf)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.clamp(n, max=keep)
    slot = torch.arange(keep, device="cuda")
    valid = (slot < kept).expand(b, kv, keep)
    order = torch.sort(order.masked_fill(~valid, s), dim=-1).values
    at = order.clamp(max=s - 1)
    rows = at.unsqueeze(-1).expand(b, kv, keep, c["d"])
    out["k"].copy_(torch.where(valid.unsqueeze(-1), torch.gather(st["k"], 2, rows), out["k"]))
    out["v"].copy_(torch.where(valid.unsqueeze(-1), torch.gather(st["v"], 2, rows), out["v"]))
    if st["ks"] is not None:
        out["k_scales"].copy_(torch.where(valid, torch.gather(st["ks"], 2, at), out["k_scales"]))
        out["v_scales"].copy_(torch.where(valid, torch.gather(st["vs"], 2, at), out["v_scales"]))
    out["weights"].copy_(torch.gather(st["weights"], 2, at).masked_fill(~valid, 0.0))
    out["indices"].copy_(at.masked_fill(~valid, -1))
    out["lengths"].copy_(kept.view(b))
    return out


# ---- one pass ----------------------------------------------------------------

def run(state):
    c = state["case"]
    if not own:
        return _plain_evict(state) if c["op"] == "evict" else _plain_attention(state)
    from openneedle_b200 import attention
    if c["op"] == "evict":
        attention.evict(state["k"], state["v"], state["weights"], state["lengths"], c["keep"], first=c["first"],
                        recent=c["recent"], k_scales=state["ks"], v_scales=state["vs"],
                        out=attention.Evicted(**state["out"]))
        return state["out"]
    args = {"window": c["window"]}
    if c["p"]:
        args.update(prefix_k=state["pk"], prefix_v=state["pv"])
    if c["cache"] == "int8":
        args.update(k_scales=state["ks"], v_scales=state["vs"])
        if c["p"]:
            args.update(prefix_k_scales=state["pks"], prefix_v_scales=state["pvs"])
    if c["op"] == "weigh":
        out, weights = attention.accumulate_attention(state["q"], state["k"], state["v"], state["lengths"],
                                                      state["weights"], **args)
        return {"out": out, "weights": weights}
    if c["lse"]:
        out, lse = attention.prefix_attention(state["q"], state["k"], state["v"], state["lengths"], return_lse=True,
                                              **args)
        return {"out": out, "lse": lse}
    return {"out": attention.prefix_attention(state["q"], state["k"], state["v"], state["lengths"], **args)}


# ---- the definitions in 64 bits ------------------------------------------------

def _exact_attention(st):
    """Sequence by sequence and KV head by KV head: the keys that exist, the definition on them."""
    c = st["case"]
    t, h, kv, d, p, w = (c[n] for n in ("t", "heads", "kv", "d", "p", "window"))
    r = h // kv
    lens = st["lengths"].tolist()
    out = torch.zeros(c["b"], t, h, d, dtype=torch.float64, device="cuda")
    lse = torch.full((c["b"], t, h), -math.inf, dtype=torch.float64, device="cuda")
    weights = st["weights"].double() if c["op"] == "weigh" else None

    def wide(name, scales, at, n):
        x = st[name][at][:n].double()
        return x if st[scales] is None else x * st[scales][at][:n].double()[:, None]

    for g in range(kv):
        pk = wide("pk", "pks", g, p) if p else None
        pv = wide("pv", "pvs", g, p) if p else None
        for b, n in enumerate(lens):
            k, v = wide("k", "ks", (b, g), n), wide("v", "vs", (b, g), n)
            if p:
                k, v = torch.cat((pk, k)), torch.cat((pv, v))
            if not len(k):
                continue
            own_at = torch.arange(-p, n, device="cuda")              # own index of each key, the prefix below zero
            query_at = torch.arange(n - t, n, device="cuda")
            visible = own_at[None] <= torch.clamp(query_at, min=-1)[:, None]
            if w:
                visible = visible & ((own_at[None] < 0) | (own_at[None] > query_at[:, None] - w))
            z = torch.einsum("trd,kd->trk", st["q"][b, :, g * r:(g + 1) * r].double(), k) / math.sqrt(d)
            z = torch.where(visible[:, None, :], z, torch.full_like(z, -math.inf))
            rows = torch.logsumexp(z, -1)
            soft = torch.exp(z - torch.where(rows == -math.inf, torch.zeros_like(rows), rows)[..., None])
            out[b, :, g * r:(g + 1) * r] = torch.einsum("trk,kd->trd", soft, v)
            lse[b, :, g * r:(g + 1) * r] = rows
            if weights is not None:
                weights[b, g, :n] += soft[..., p:].sum((0, 1))
    if weights is not None:
        return {"out": out, "weights": weights}
    return {"out": out, "lse": lse} if c["lse"] else {"out": out}


def _exact_evict(st):
    """On the host: the order by (weight, index) of the keys between the first and the recent ones."""
    c = st["case"]
    keep, first, recent = c["keep"], c["first"], c["recent"]
    w = st["weights"].double().cpu().numpy()
    lens = st["lengths"].tolist()
    out = {n: np.zeros(tuple(x.shape), np.int64 if n in ("indices", "lengths") else np.float64)
           for n, x in st["out"].items()}
    out["indices"][:] = -1
    at_all = {n: st[m].double().cpu().numpy() for n, m in (("k", "k"), ("v", "v"), ("k_scales", "ks"),
                                                           ("v_scales", "vs")) if st[m] is not None}
    at_all["weights"] = w
    for b, n in enumerate(lens):
        out["lengths"][b] = min(n, keep)
        for g in range(c["kv"]):
            if n <= keep:
                at = np.arange(n)
            else:
                middle = np.arange(first, n - recent)
                best = middle[np.lexsort((middle, -w[b, g, middle]))][:keep - first - recent]
                at = np.concatenate((np.arange(first), np.sort(best), np.arange(n - recent, n)))
            out["indices"][b, g, :len(at)] = at
            for name, x in at_all.items():
                out[name][b, g, :len(at)] = x[b, g, at]
    return out


def exact(case, seed):
    # about 20 us a small operation: leave out what would take too long sequence by sequence
    w = work(case)
    if case["op"] != "evict" and (case["b"] * case["kv"] > 12000 or w["flops"] > 2e13):
        return None
    st = prepare(case, seed)
    return _exact_evict(st) if case["op"] == "evict" else _exact_attention(st)
