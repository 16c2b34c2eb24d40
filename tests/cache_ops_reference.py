"""The cache operators' definitions in 64 bits, sequence by sequence on the host,
and inputs and error bounds for their tests."""
import math

import torch

TYPES = {"int8": torch.int8, "bf16": torch.bfloat16, "f16": torch.float16}


def make_cache(g, cache, shape, spread=0.3):
    """Random K or V rows [*shape]: (stored, scales or None)."""
    x = torch.randn(*shape, generator=g) * torch.exp(spread * torch.randn(*shape[:-1], 1, generator=g))
    if cache != "int8":
        return x.to(TYPES[cache]), None
    most = x.abs().amax(-1, keepdim=True) if x.numel() else x.sum(-1, keepdim=True)
    return torch.round(x * (127.0 / most)).clamp(-127, 127).to(torch.int8), (most / 127.0)[..., 0].contiguous()


def make_inputs(cache, b, t, heads, kv, d, p, s, lengths, seed=0, sharp=1.5):
    g = torch.Generator().manual_seed(seed)
    q = sharp * torch.randn(b, t, heads, d, generator=g)
    c = {"q": q if cache == "int8" else q.to(TYPES[cache])}
    c["k"], c["k_scales"] = make_cache(g, cache, (b, kv, s, d))
    c["v"], c["v_scales"] = make_cache(g, cache, (b, kv, s, d))
    if p:
        c["prefix_k"], c["prefix_k_scales"] = make_cache(g, cache, (kv, p, d))
        c["prefix_v"], c["prefix_v_scales"] = make_cache(g, cache, (kv, p, d))
    c["lengths"] = torch.tensor(lengths, dtype=torch.int32)
    c["weights"] = torch.rand(b, kv, s, generator=g) / max(s, 1)
    return c


def wide(x, scales):
    return x.double() if scales is None else x.double() * scales.double().unsqueeze(-1)


def attention(c, window=0, tokens=None, scale=None):
    """out, lse, weights in 64 bits, and bounds on their errors (None rows: not written)."""
    q = c["q"].double()
    b, t, heads, d = q.shape
    kv, s = c["k"].shape[1:3]
    r = heads // kv
    scale = d ** -0.5 if scale is None else scale
    p = c["prefix_k"].shape[1] if c.get("prefix_k") is not None else 0
    out = torch.zeros(b, t, heads, d, dtype=torch.float64)
    lse = torch.full((b, t, heads), -math.inf, dtype=torch.float64)
    weights = c["weights"].double().clone()
    gained = torch.zeros_like(weights)
    mix = torch.zeros_like(out)          # sum of p |v|, what an output's rounding errors are relative to
    dz = torch.zeros(b, t, heads, dtype=torch.float64)   # sum |q k| of the largest
    total_v = torch.zeros_like(out)      # sum of |v| over the visible keys
    most_v = torch.zeros(b, t, heads, dtype=torch.float64)   # their number times the largest |v| scale times 127
    for i in range(b):
        n = max(0, min(int(c["lengths"][i]), s))
        m = t if tokens is None else max(0, min(int(tokens[i]), t))
        for g in range(kv):
            k = wide(c["k"][i, g, :n], None if c["k_scales"] is None else c["k_scales"][i, g, :n])
            v = wide(c["v"][i, g, :n], None if c["v_scales"] is None else c["v_scales"][i, g, :n])
            if p:
                pk = wide(c["prefix_k"][g], None if c["prefix_k_scales"] is None else c["prefix_k_scales"][g])
                pv = wide(c["prefix_v"][g], None if c["prefix_v_scales"] is None else c["prefix_v_scales"][g])
                k, v = torch.cat((pk, k)), torch.cat((pv, v))
            for x in range(m):
                at = n - m + x
                seen = list(range(p)) + [p + j for j in range(max(0, at - window + 1) if window else 0, at + 1)]
                if not seen:
                    continue
                for h in range(g * r, (g + 1) * r):
                    z = scale * (k[seen] @ q[i, x, h])
                    soft = torch.softmax(z, 0)
                    out[i, x, h] = soft @ v[seen]
                    lse[i, x, h] = torch.logsumexp(z, 0)
                    mix[i, x, h] = soft @ v[seen].abs()
                    total_v[i, x, h] = v[seen].abs().sum(0)
                    dz[i, x, h] = scale * (k[seen].abs() @ q[i, x, h].abs()).max()
                    if c["v_scales"] is not None:
                        vs = c["v_scales"][i, g, :n]
                        vs = (torch.cat((c["prefix_v_scales"][g], vs)) if p else vs)[seen].double()
                        most_v[i, x, h] = len(seen) * 127 * vs.abs().max()
                    own = torch.tensor([j - p for j in seen if j >= p], dtype=torch.long)
                    gained[i, g, own] += soft[len(seen) - len(own):]
    weights += gained
    return {"out": out, "lse": lse, "weights": weights, "gained": gained, "mix": mix, "dz": dz, "total_v": total_v,
            "most_v": most_v}


def bounds(c, ref):
    """Elementwise error bounds of out, lse and weights.

    A logit is a sum of D products in 32-bit accumulation (at most D/4 + 8
    roundings of 2^-24, each relative to the sum of the products' sizes; the INT8
    queries' FP16 pairs carry 22 bits, 2^-23 more) and a few scalings; its error
    e enters a softmax weight as the factor 1 + 2 e.  The exponential and the
    sums add 2^-20.  16-bit caches round each softmax weight (half a step, and
    half of the smallest FP16 number, 2^-25, where they fall below its normal
    range) and the output (half a step).  INT8 caches multiply the softmax weights
    by V's scales over the power of two at or below the largest, times at least
    2^6, and round the product to an FP16 pair: 2^-22 of it, or half of the
    smallest FP16 number, 2^-25 / 2^6, of the largest scale for each key."""
    d = c["q"].shape[-1]
    e = ref["dz"] * (d / 4 + 12) * 2.0 ** -24 + 2.0 ** -22 * ref["lse"].abs().nan_to_num(posinf=0.0)
    rel = 2 * e + 2.0 ** -20
    out = ref["mix"] * rel.unsqueeze(-1)
    kind = c["k"].dtype
    if kind == torch.int8:
        out = out + 2.0 ** -24 * ref["out"].abs() + 2.0 ** -31 * ref["most_v"].unsqueeze(-1)
    else:
        half = torch.finfo(kind).eps / 2
        out = (out + half * ref["mix"]) * (1 + half) + half * ref["out"].abs()
        if kind == torch.float16:
            out = out + 2.0 ** -25 * ref["total_v"] + 2.0 ** -25
    lse = e + 2.0 ** -20 + 2.0 ** -22 * ref["lse"].abs().nan_to_num(posinf=0.0)
    weights = ref["gained"] * (rel.max() + 2.0 ** -24 * c["q"].shape[1] * c["q"].shape[2]) + \
        2.0 ** -23 * ref["weights"].abs()
    return {"out": out, "lse": lse, "weights": weights}


def check(got, ref, bound, name):
    got = got.detach().cpu().double()
    same = (got == ref) | (got.isnan() & ref.isnan())
    off = torch.where(same, torch.zeros_like(ref), (got - ref).abs())
    bad = ~(off <= bound)
    if bad.any():
        at = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} values outside their bound, first at {at}: "
                             f"{float(got[at])} for {float(ref[at])}, bound {float(bound[at]):.3g}")


def evict(c, keep, first, recent):
    """The kept indexes of each sequence and KV head."""
    b, kv, s = c["weights"].shape
    kept = []
    for i in range(b):
        n = max(0, min(int(c["lengths"][i]), s))
        row = []
        for g in range(kv):
            if n <= keep:
                row.append(list(range(n)))
                continue
            w = [-math.inf if math.isnan(x) else x for x in c["weights"][i, g].tolist()]
            middle = sorted(range(first, n - recent), key=lambda j: (-w[j], j))[:keep - first - recent]
            row.append(list(range(first)) + sorted(middle) + list(range(n - recent, n)))
        kept.append(row)
    return kept
