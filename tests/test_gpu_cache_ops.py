"""Attention behind a shared prefix, accumulated key weights and eviction on the
GPU against their definitions in 64 bits (cache_ops_reference.py, whose bounds
follow from the roundings of each step)."""
import math

import pytest
import torch

import cache_ops_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from openneedle_b200 import attention, build
    build.build()
    return attention


def cuda(c):
    return {n: None if x is None else x.cuda() for n, x in c.items()}


def call(ops, c, weigh=False, **more):
    d = cuda(c)
    args = {n: d.get(n) for n in ("prefix_k", "prefix_v", "k_scales", "v_scales", "prefix_k_scales",
                                  "prefix_v_scales")}
    if weigh:
        return ops.accumulate_attention(d["q"], d["k"], d["v"], d["lengths"], d["weights"], **args, **more)
    return ops.prefix_attention(d["q"], d["k"], d["v"], d["lengths"], return_lse=True, **args, **more)


def both(ops, c, **more):
    """out and lse of prefix_attention and out and weights of accumulate_attention within their bounds."""
    ref = R.attention(c, **{n: x for n, x in more.items() if n in ("window", "scale")})
    bound = R.bounds(c, ref)
    out, lse = call(ops, c, **more)
    R.check(out, ref["out"], bound["out"], "out")
    R.check(lse, ref["lse"], bound["lse"], "lse")
    out2, weights = call(ops, c, weigh=True, **more)
    R.check(out2, ref["out"], bound["out"], "out of accumulate_attention")
    R.check(weights, ref["weights"], bound["weights"], "weights")
    return out, lse, weights


CACHES = ("int8", "bf16", "f16")


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("d", (64, 128))
@pytest.mark.parametrize("b,heads,kv,p,s,lengths", [
    (1, 8, 4, 0, 1, [1]),                                   # one key
    (1, 8, 4, 1, 1, [0]),                                   # one prefix key, no own
    (3, 8, 4, 48, 64, [17, 0, 64]),
    (2, 4, 1, 33, 97, [97, 50]),                            # one KV head
    (2, 16, 2, 130, 31, [31, 1]),                           # eight query heads a KV head
    (5, 6, 6, 257, 200, [200, 33, 0, 1, 129]),              # one query head a KV head
    (40, 8, 4, 300, 40, [(7 * i) % 41 for i in range(40)]),  # more prefix rows than one tile
    (1, 32, 1, 70, 90, [90])])                              # more query heads than a tile's rows
def test_one_token(ops, cache, d, b, heads, kv, p, s, lengths):
    both(ops, R.make_inputs(cache, b, 1, heads, kv, d, p, s, lengths, seed=b + p))


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("d", (64, 128))
@pytest.mark.parametrize("b,t,heads,kv,p,s,lengths,window", [
    (2, 2, 8, 4, 5, 20, [20, 2], 0),
    (2, 7, 4, 2, 0, 40, [40, 9], 0),
    (1, 33, 8, 4, 65, 150, [150], 0),
    (2, 33, 8, 4, 65, 150, [150, 33], 16),
    (2, 5, 4, 4, 3, 50, [50, 3], 4),                        # fewer own keys than tokens: the first see the prefix only
    (2, 5, 4, 4, 0, 50, [50, 3], 4),                        # ... or nothing
    (1, 150, 2, 1, 0, 150, [150], 0),
    (1, 140, 3, 1, 129, 300, [300], 37),
    (2, 1, 8, 4, 17, 70, [70, 20], 16),                     # decode in a window
    (2, 1, 8, 4, 17, 70, [70, 20], 1)])
def test_several_tokens(ops, cache, d, b, t, heads, kv, p, s, lengths, window):
    both(ops, R.make_inputs(cache, b, t, heads, kv, d, p, s, lengths, seed=t + p), window=window)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("d", (64, 128))
@pytest.mark.parametrize("b,t,heads,kv,p,s,window", [
    (20, 130, 8, 8, 200, 140, 0),                           # own row tiles that fill the machine take the prefix
    (20, 130, 8, 8, 129, 300, 70),
    (170, 90, 1, 1, 260, 100, 0),                           # ... both tiles of a CTA on the same rows
    (3, 12, 40, 8, 30, 40, 0),                              # 60 rows: weights from kept logits
    (2, 3, 130, 1, 20, 50, 0)])                             # more query heads a KV head than a tile has rows
def test_many_rows(ops, cache, d, b, t, heads, kv, p, s, window):
    """Larger calls, against the definition on the GPU in 64 bits with the bounds of cache_ops_reference."""
    lengths = [t + (7 * i) % (s - t + 1) for i in range(b)]
    c = R.make_inputs(cache, b, t, heads, kv, d, p, s, lengths, seed=t)
    g = cuda(c)
    r = heads // kv
    wide = lambda x, sc: x.double() if sc is None else x.double() * sc.double().unsqueeze(-1)   # noqa: E731
    k, v = wide(g["k"], g["k_scales"]), wide(g["v"], g["v_scales"])
    pk = wide(g["prefix_k"], g["prefix_k_scales"]).expand(b, -1, -1, -1)
    pv = wide(g["prefix_v"], g["prefix_v_scales"]).expand(b, -1, -1, -1)
    k, v = torch.cat((pk, k), 2), torch.cat((pv, v), 2)
    q = g["q"].double().view(b, t, kv, r, d).permute(0, 2, 1, 3, 4)                 # [B, KV, T, R, D]
    at = (g["lengths"].view(b, 1) - t + torch.arange(t, device="cuda")).view(b, 1, t, 1, 1)
    j = torch.arange(-p, s, device="cuda")
    seen = (j < 0) | ((j <= at) & (j > at - window if window else j >= 0))
    z = torch.einsum("bgtrd,bgkd->bgtrk", q, k) * d ** -0.5
    z = z.masked_fill(~seen, -math.inf)
    soft = torch.softmax(z, -1)
    back = lambda x: x.permute(0, 2, 1, 3, *range(4, x.dim())).reshape(b, t, heads, *x.shape[4:]).cpu()   # noqa: E731
    gained = soft[..., p:].sum((2, 3)).cpu()
    count = seen.expand_as(z).sum(-1)
    most = (127 * count * torch.cat((g["prefix_v_scales"].expand(b, -1, -1), g["v_scales"]), 2).abs().amax(-1)
            .view(b, kv, 1, 1)).double() if cache == "int8" else torch.zeros_like(z[..., 0])
    ref = {"out": back(torch.einsum("bgtrk,bgkd->bgtrd", soft, v)), "lse": back(torch.logsumexp(z, -1)),
           "weights": c["weights"].double() + gained, "gained": gained,
           "mix": back(torch.einsum("bgtrk,bgkd->bgtrd", soft, v.abs())), "most_v": back(most),
           "total_v": back(torch.einsum("bgtrk,bgkd->bgtrd", seen.expand_as(z).double(), v.abs())),
           "dz": back(torch.where(seen, torch.einsum("bgtrd,bgkd->bgtrk", q.abs(), k.abs()) * d ** -0.5,
                                  torch.zeros_like(z)).amax(-1))}
    bound = R.bounds(c, ref)
    out, lse = call(ops, c, window=window)
    R.check(out, ref["out"], bound["out"], "out")
    R.check(lse, ref["lse"], bound["lse"], "lse")
    out, weights = call(ops, c, weigh=True, window=window)
    R.check(out, ref["out"], bound["out"], "out of accumulate_attention")
    R.check(weights, ref["weights"], bound["weights"], "weights")


@pytest.mark.parametrize("t", (1, 100))
def test_offsets_beyond_32_bits(ops, t):
    """The last keys of a cache of 34 million INT8 rows (2.2 GB), in a window."""
    s, n = 34_000_000, 34_000_000 - 3
    g = torch.Generator("cuda").manual_seed(1)
    k = torch.zeros(1, 1, s, 64, dtype=torch.int8, device="cuda")
    k[:, :, -400:] = torch.randint(-127, 128, (1, 1, 400, 64), generator=g, device="cuda", dtype=torch.int8)
    scales = torch.full((1, 1, s), 0.01, device="cuda")
    q = torch.randn(1, t, 2, 64, generator=g, device="cuda")
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    out, lse = ops.prefix_attention(q, k, k, lengths, k_scales=scales, v_scales=scales, window=64, return_lse=True)
    tail = slice(s - 400, s)
    near = {"k_scales": scales[:, :, tail].clone(), "v_scales": scales[:, :, tail].clone(), "window": 64,
            "return_lse": True}
    out2, lse2 = ops.prefix_attention(q, k[:, :, tail].clone(), k[:, :, tail].clone(), lengths - (s - 400), **near)
    # the same keys from the front of a small cache: only the order of the sums may differ
    assert (out - out2).abs().max() <= 1e-5 * out2.abs().max() and (lse - lse2).abs().max() <= 1e-5


def test_lengths_are_clamped(ops):
    c = R.make_inputs("bf16", 3, 1, 8, 4, 64, 20, 60, [60, 0, 60], seed=3)
    want = call(ops, c) + call(ops, c, weigh=True)
    c["lengths"] = torch.tensor([2 ** 31 - 1, -5, 61], dtype=torch.int32)
    for x, y in zip(want, call(ops, c) + call(ops, c, weigh=True)):
        assert torch.equal(x, y)
    c = R.make_inputs("bf16", 2, 40, 8, 4, 64, 20, 60, [60, 60], seed=3)
    want = call(ops, c)
    got = call(ops, c, tokens=torch.tensor([1000, 40], dtype=torch.int32).cuda())
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    e = evict_inputs("bf16", 2, 2, 64, 50, [50, 0], seed=4)
    first, _ = evicted(ops, e, 20, 1, 2)
    e["lengths"] = torch.tensor([5000, -3], dtype=torch.int32)
    for x, y in zip(first, evicted(ops, e, 20, 1, 2)[0]):
        assert x is y is None or torch.equal(x, y)


@pytest.mark.parametrize("cache", CACHES)
def test_rows_that_see_nothing(ops, cache):
    c = R.make_inputs(cache, 3, 1, 8, 4, 64, 0, 16, [0, 5, 0])
    out, lse, weights = both(ops, c)
    assert (out[0] == 0).all() and torch.isneginf(lse[0]).all() and (out[2] == 0).all()
    assert torch.equal(weights[0].cpu(), c["weights"][0])


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("t", (1, 40))
def test_padded_tokens_are_left_alone(ops, cache, t):
    c = R.make_inputs(cache, 4, t, 8, 4, 64, 20, 80, [80, 70, 60, 50], seed=9)
    tokens = torch.tensor([t, 0, t // 2, 1], dtype=torch.int32)
    c["q"][3, 1:] = math.nan
    ref = R.attention(c, tokens=tokens)
    bound = R.bounds(c, {n: x.nan_to_num() for n, x in ref.items()})
    out = torch.full_like(c["q"].nan_to_num(), 7.0).cuda()
    call(ops, c, tokens=tokens.cuda(), out=out)
    for i in range(4):
        n = int(tokens[i])
        R.check(out[i, :n], ref["out"][i, :n], bound["out"][i, :n], "out")
        assert (out[i, n:] == 7.0).all()
    out2 = torch.full_like(out, 7.0)
    _, weights = call(ops, c, weigh=True, tokens=tokens.cuda(), out=out2)
    assert torch.equal(out2, out)
    R.check(weights, ref["weights"], bound["weights"].nan_to_num(), "weights")


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("t", (1, 40))
def test_what_lies_behind_the_length_is_not_used(ops, cache, t):
    lengths = [t + 3, t, 90]
    c = R.make_inputs(cache, 3, t, 8, 4, 128, 50, 100, lengths, seed=3)
    clean = call(ops, c)
    clean_w = call(ops, c, weigh=True)
    for i, n in enumerate(lengths):
        if cache == "int8":
            c["k_scales"][i, :, n:] = math.nan
            c["v_scales"][i, :, n:] = math.inf
        else:
            c["k"][i, :, n:] = math.nan
            c["v"][i, :, n:] = math.inf
    for x, y in zip(clean + clean_w, call(ops, c) + call(ops, c, weigh=True)):
        assert torch.equal(x, y)
    # ... nor before every query's window
    c = R.make_inputs(cache, 1, t, 8, 4, 128, 50, 100, [95], seed=4)
    clean = call(ops, c, window=6) + call(ops, c, weigh=True, window=6)
    n = 95 - t - 5
    if cache == "int8":
        c["v_scales"][0, :, :n] = math.nan
    else:
        c["v"][0, :, :n] = math.nan
    for x, y in zip(clean, call(ops, c, window=6) + call(ops, c, weigh=True, window=6)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("t", (1, 40))
def test_a_row_of_nan_stays_alone(ops, cache, t):
    c = R.make_inputs(cache, 3, t, 8, 4, 64, 50, 100, [100, 80, 60], seed=5)
    clean = call(ops, c)
    c["q"][1, 0, 3, 5] = math.nan
    out, lse = call(ops, c)
    assert out[1, 0, 3].isnan().all() and lse[1, 0, 3].isnan()
    hit = torch.zeros(3, t, 8, dtype=torch.bool, device="cuda")
    hit[1, 0, 3] = True
    assert torch.equal(out[~hit], clean[0][~hit]) and torch.equal(lse[~hit], clean[1][~hit])


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("t", (1, 24))
def test_large_and_small_logits(ops, cache, t):
    """Softmax weights from one key to all keys alike, scales over many powers of two."""
    for sharp, scale in ((30.0, None), (0.0, None), (1.0, 1e-3)):
        both(ops, R.make_inputs(cache, 2, t, 8, 4, 64, 37, 60, [60, 24], seed=6, sharp=sharp), scale=scale)
    c = R.make_inputs(cache, 2, t, 8, 4, 64, 37, 60, [60, 24], seed=7)
    if cache == "int8":                                     # V scales from row to row, rising and falling
        c["v_scales"] *= 2.0 ** (torch.arange(60) % 23 - 11.0)
        c["prefix_v_scales"] *= 2.0 ** torch.arange(37).flip(0)
        c["v_scales"][:, :, 3] = 0.0
        c["q"][:, :, 1] *= 1e-20
        c["q"][:, :, 2] = 0.0
    both(ops, c)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("t", (1, 40))
def test_strides(ops, cache, t):
    """Caches laid out [B, S, KV, D], a slice of a longer cache, queries inside a fused projection."""
    c = R.make_inputs(cache, 3, t, 8, 4, 64, 50, 100, [100, 80, 60], seed=8)
    plain = call(ops, c) + call(ops, c, weigh=True)
    d = cuda(c)
    fused = torch.zeros(3, t, 16, 64, dtype=d["q"].dtype, device="cuda")
    fused[:, :, 4:12] = d["q"]
    d["q"] = fused[:, :, 4:12]
    for n in ("k", "v"):
        d[n] = d[n].transpose(1, 2).contiguous().transpose(1, 2)
        longer = torch.zeros(4, 60, 64, dtype=d[n].dtype, device="cuda")
        longer[:, 7:57] = d["prefix_" + n]
        d["prefix_" + n] = longer[:, 7:57]
        if cache == "int8":
            s = n + "_scales"
            d[s] = d[s].permute(2, 0, 1).contiguous().permute(1, 2, 0)
            d["prefix_" + s] = d["prefix_" + s].t().contiguous().t()
    d["weights"] = d["weights"].transpose(1, 2).contiguous().transpose(1, 2)
    args = {n: d.get(n) for n in ("prefix_k", "prefix_v", "k_scales", "v_scales", "prefix_k_scales",
                                  "prefix_v_scales")}
    wide = torch.zeros(3, t, 10, 64, dtype=plain[0].dtype, device="cuda")
    got = ops.prefix_attention(d["q"], d["k"], d["v"], d["lengths"], out=wide[:, :, 1:9], return_lse=True, **args)
    assert got[0].data_ptr() == wide[:, :, 1:9].data_ptr()
    assert (wide[:, :, 0] == 0).all() and (wide[:, :, 9] == 0).all()
    more = ops.accumulate_attention(d["q"], d["k"], d["v"], d["lengths"], d["weights"], weights_out=d["weights"],
                                    **args)
    assert more[1] is d["weights"]
    for x, y in zip(plain, got + more):
        assert torch.equal(x, y)


def test_one_token_without_its_axis(ops):
    c = R.make_inputs("bf16", 3, 1, 8, 4, 64, 50, 100, [100, 80, 60], seed=8)
    out, lse = call(ops, c)
    c["q"] = c["q"][:, 0]
    out2, lse2 = call(ops, c)
    assert torch.equal(out[:, 0], out2) and torch.equal(lse[:, 0], lse2)


def test_empty_calls(ops):
    c = R.make_inputs("f16", 2, 1, 8, 4, 64, 50, 100, [100, 80], seed=8)
    d = cuda(c)
    out = ops.prefix_attention(d["q"][:0], d["k"][:0], d["v"][:0], d["lengths"][:0])
    assert out.shape == (0, 1, 8, 64)
    out, w = ops.accumulate_attention(d["q"][:, :0], d["k"], d["v"], d["lengths"], d["weights"])
    assert out.shape == (2, 0, 8, 64) and torch.equal(w, d["weights"])
    # no own slots: the prefix alone
    ref = R.attention({**c, "lengths": torch.zeros(2, dtype=torch.int32)})
    out = ops.prefix_attention(d["q"], d["k"][:, :, :0], d["v"][:, :, :0], d["lengths"], d["prefix_k"], d["prefix_v"])
    R.check(out, ref["out"], R.bounds(c, ref)["out"], "out")


# ---- eviction -----------------------------------------------------------------

def evicted(ops, c, keep, first, recent, **more):
    d = cuda(c)
    return ops.evict(d["k"], d["v"], d["weights"], d["lengths"], keep, first=first, recent=recent,
                     k_scales=d["k_scales"], v_scales=d["v_scales"], **more), d


def check_evicted(e, c, keep, first, recent, behind=None):
    for i, row in enumerate(R.evict(c, keep, first, recent)):
        for g, at in enumerate(row):
            n = len(at)
            assert int(e.lengths[i]) == n
            assert e.indices[i, g].tolist() == at + [-1] * (keep - n)
            for name in ("k", "v", "k_scales", "v_scales"):
                if c[name] is not None:
                    got = getattr(e, name)[i, g].cpu()
                    assert torch.equal(got[:n], c[name][i, g][at]), name
                    if behind is not None:
                        assert torch.equal(got[n:], behind[name][i, g, n:got.shape[0]]), name
            w = e.weights[i, g].cpu()
            assert torch.equal(w[:n].nan_to_num(nan=-5.0), c["weights"][i, g][at].nan_to_num(nan=-5.0))
            assert (w[n:] == 0).all()


def evict_inputs(cache, b, kv, d, s, lengths, seed=0):
    c = R.make_inputs(cache, b, 1, kv, kv, d, 0, s, lengths, seed)
    g = torch.Generator().manual_seed(seed)
    # ties, among them zeros of both signs, and weights over many powers of two
    c["weights"] = torch.exp(4 * torch.randn(b, kv, s, generator=g))
    c["weights"] = torch.where(torch.rand(b, kv, s, generator=g) < 0.3, torch.zeros(()), c["weights"])
    c["weights"] = torch.where(torch.rand(b, kv, s, generator=g) < 0.1, -torch.zeros(()), c["weights"])
    c["weights"] = torch.where(torch.rand(b, kv, s, generator=g) < 0.2, c["weights"].round(), c["weights"])
    return c


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("b,kv,d,s,lengths,keep,first,recent", [
    (1, 1, 64, 1, [1], 1, 0, 0),
    (2, 4, 64, 50, [50, 20], 20, 4, 8),
    (3, 2, 128, 1500, [1500, 0, 1025], 333, 0, 0),
    (2, 2, 64, 2100, [2100, 1024], 1024, 1000, 24),         # nothing to choose
    (2, 2, 128, 700, [700, 699], 699, 1, 1),
    (2, 1, 64, 30, [30, 9], 64, 4, 4),                      # keep above the capacity
    (2, 2, 64, 300, [300, 150], 0, 0, 0),                   # nothing stays
    (2, 3, 64, 9000, [9000, 8999], 1, 0, 1)])
def test_evict(ops, cache, b, kv, d, s, lengths, keep, first, recent):
    c = evict_inputs(cache, b, kv, d, s, lengths, seed=s)
    e, _ = evicted(ops, c, keep, first, recent)
    check_evicted(e, c, keep, first, recent)
    if keep <= s:
        before = {n: None if c[n] is None else c[n].clone() for n in c}
        e, d = evicted(ops, c, keep, first, recent, in_place=True)
        assert e.k is d["k"] and e.weights is d["weights"]
        # rows behind the kept ones may hold what was there or nothing else: unchanged
        check_evicted(e, c, keep, first, recent, behind=before)


@pytest.mark.parametrize("value", (0.0, -0.0, math.nan, -math.inf, math.inf, -3.0))
def test_evict_equal_weights(ops, value):
    c = evict_inputs("bf16", 2, 2, 64, 5000, [5000, 4097], seed=1)
    c["weights"][0] = value
    c["weights"][1, :, ::3] = value
    for keep, first, recent in ((100, 0, 0), (4096, 3, 1000)):
        e, _ = evicted(ops, c, keep, first, recent)
        check_evicted(e, c, keep, first, recent)


def test_evict_into_strided_outputs(ops):
    c = evict_inputs("int8", 2, 4, 64, 600, [600, 77], seed=2)
    d = cuda(c)
    whole = torch.full((2, 200, 4, 64), 9, dtype=torch.int8, device="cuda")
    f = lambda: torch.full((2, 200, 4), 9.0, device="cuda")      # noqa: E731
    w, ks, vs = f(), f(), f()
    other = whole.clone()
    out = ops.Evicted(whole.transpose(1, 2), other.transpose(1, 2), w.transpose(1, 2),
                      torch.zeros(2, dtype=torch.int32, device="cuda"),
                      torch.zeros(2, 4, 150, dtype=torch.int32, device="cuda"), ks.transpose(1, 2), vs.transpose(1, 2))
    e = ops.evict(d["k"], d["v"], d["weights"], d["lengths"], 150, first=5, recent=10, k_scales=d["k_scales"],
                  v_scales=d["v_scales"], out=out)
    nines = torch.full((2, 4, 200, 64), 9, dtype=torch.int8)
    behind = {"k": nines, "v": nines,
              "k_scales": torch.full((2, 4, 200), 9.0), "v_scales": torch.full((2, 4, 200), 9.0)}
    check_evicted(e, c, 150, 5, 10, behind=behind)


@pytest.mark.parametrize("cache,d,s", [("int8", 64, 40), ("bf16", 128, 33), ("int8", 64, 4100)])
def test_evict_many_rows(ops, cache, d, s):
    """More rows than the machine has places for: selection and copies in one kernel, and (4100) in two."""
    b, kv = 75, 4
    c = evict_inputs(cache, b, kv, d, s, [s - (i * 7) % s for i in range(b)], seed=s)
    e, _ = evicted(ops, c, s // 3, 2, 5)
    check_evicted(e, c, s // 3, 2, 5)


@pytest.mark.parametrize("s,lengths", [(20000, [20000, 70]), (70000, [70000, 66000]), (140000, [140000, 139999])])
def test_evict_long_rows(ops, s, lengths):
    """One CTA, four, eight a row, and rows beyond their registers; against a stable sort."""
    g = torch.Generator("cuda").manual_seed(s)
    b, kv, d, keep, first, recent = 2, 2, 64, 5000, 16, 700
    k = torch.randint(-127, 128, (b, kv, s, d), generator=g, device="cuda", dtype=torch.int8)
    v = torch.randint(-127, 128, (b, kv, s, d), generator=g, device="cuda", dtype=torch.int8)
    ks, vs = (torch.rand(b, kv, s, generator=g, device="cuda") for _ in range(2))
    w = torch.exp(4 * torch.randn(b, kv, s, generator=g, device="cuda"))
    w[torch.rand(b, kv, s, generator=g, device="cuda") < 0.4] = 0.0
    w = torch.where(torch.rand(b, kv, s, generator=g, device="cuda") < 0.3, w.round(), w)
    e = ops.evict(k, v, w, torch.tensor(lengths, dtype=torch.int32, device="cuda"), keep, first=first, recent=recent,
                  k_scales=ks, v_scales=vs)
    for i, n in enumerate(lengths):
        assert int(e.lengths[i]) == min(n, keep)
        for h in range(kv):
            if n <= keep:
                at = torch.arange(n, device="cuda")
            else:
                x = w[i, h, :n].clone()
                x[:first] = math.inf
                x[n - recent:] = math.inf
                at = torch.sort(x, descending=True, stable=True).indices[:keep].sort().values
            m = len(at)
            assert torch.equal(e.indices[i, h, :m], at.int()) and (e.indices[i, h, m:] == -1).all()
            for x, y in ((e.k, k), (e.v, v), (e.k_scales, ks), (e.v_scales, vs), (e.weights, w)):
                assert torch.equal(x[i, h, :m], y[i, h][at])
            assert (e.weights[i, h, m:] == 0).all()


# ---- the KV pool's shared-prefix query -------------------------------------------

@pytest.mark.parametrize("heads,kvheads,hd,window,prefix,sessions", [
    (8, 4, 64, 0, 24, 3), (8, 4, 64, 16, 7, 5), (8, 8, 64, 0, 5, 4), (4, 1, 128, 9, 33, 40), (4, 2, 128, 0, 0, 3),
    (16, 2, 64, 0, 300, 70), (8, 4, 64, 24, 700, 33)])
def test_pool_query_shared(ops, heads, kvheads, hd, window, prefix, sessions):
    """KVCache.query_shared against KVCache.query on the same pool (whose outputs the oracle pins): ring windows
    before and after they are full, sessions in another order and left out."""
    import numpy as np
    from util import FP32_REL_TOL, rel_err
    rng = np.random.default_rng(prefix + sessions)
    kv = ops.KVCache(sessions, heads, kvheads, hd, prefix + 64, window, prefix)
    if prefix:
        kv.set_prefix(*(rng.normal(size=(prefix, kvheads * hd)).astype(np.float32) for _ in range(2)))
    for step in range(40):
        ids = rng.permutation(sessions)
        k, v = (rng.normal(size=(sessions, kvheads * hd)).astype(np.float32) for _ in range(2))
        kv.store(ids, [prefix + step] * sessions, k, v)
        if step in (0, 10, 39):
            some = rng.permutation(sessions)[:max(1, sessions - 2)]
            q = rng.normal(size=(len(some), heads * hd)).astype(np.float32)
            got = kv.query_shared(some, [prefix + step] * len(some), q)
            assert rel_err(got, kv.query(some, [prefix + step] * len(some), q)) <= FP32_REL_TOL
            qd = torch.from_numpy(q).cuda()
            out = torch.empty_like(qd)
            kv.query_shared_device(some, [prefix + step] * len(some), qd, out)
            torch.cuda.synchronize()
            np.testing.assert_array_equal(out.cpu().numpy(), got)
    with pytest.raises(RuntimeError, match="appears twice"):
        kv.query_shared([0, 0], [prefix] * 2, np.zeros((2, heads * hd), np.float32))
    if prefix:
        with pytest.raises(RuntimeError, match="inside the shared prefix"):
            kv.query_shared([0], [prefix - 1], np.zeros((1, heads * hd), np.float32))


# ---- a run of them together, streams and graphs -------------------------------------

@pytest.mark.parametrize("cache", CACHES)
def test_prefill_evict_decode(ops, cache):
    """A prompt behind a shared prefix, its cache thinned out in place, then decoded on: the operators as a
    generation loop uses them, against the same steps on the definitions."""
    b, kv, heads, d, p, s, t, keep = 3, 2, 4, 64, 40, 128, 60, 48
    lengths = [60, 90, 75]
    c = R.make_inputs(cache, b, t, heads, kv, d, p, s, lengths, seed=12)
    c["weights"] = torch.zeros(b, kv, s)
    dev = cuda(c)
    args = {n: dev.get(n) for n in ("prefix_k", "prefix_v", "k_scales", "v_scales", "prefix_k_scales",
                                    "prefix_v_scales")}
    scales = {n: dev[n] for n in ("k_scales", "v_scales")}
    ref = R.attention(c)
    out, w = ops.accumulate_attention(dev["q"], dev["k"], dev["v"], dev["lengths"], dev["weights"],
                                      weights_out=dev["weights"], **args)
    R.check(out, ref["out"], R.bounds(c, ref)["out"], "prefill")
    c["weights"] = w.cpu()                                      # the same weights decide on both sides
    kept = R.evict(c, keep, 2, 8)
    e = ops.evict(dev["k"], dev["v"], w, dev["lengths"], keep, first=2, recent=8, in_place=True, **scales)
    check_evicted(e, c, keep, 2, 8)
    for i in range(b):
        for g in range(kv):
            n = len(kept[i][g])
            for name in ("k", "v", "weights", "k_scales", "v_scales"):
                if c[name] is not None:
                    c[name][i, g, :n] = c[name][i, g][kept[i][g]].clone()
            c["weights"][i, g, n:] = 0
    lengths = e.lengths.clone()
    for step in range(3):
        new = R.make_inputs(cache, b, 1, heads, kv, d, 0, 1, [1] * b, seed=20 + step)
        c["lengths"] = lengths.cpu() + 1
        for i in range(b):
            at = int(lengths[i])
            for name in ("k", "v", "k_scales", "v_scales"):
                if c[name] is not None:
                    c[name][i, :, at] = new[name][i, :, 0]
                    dev[name][i, :, at] = new[name][i, :, 0].cuda()
        lengths += 1
        c["q"] = new["q"]
        ref = R.attention(c)
        bound = R.bounds(c, ref)
        out, w = ops.accumulate_attention(new["q"].cuda(), dev["k"], dev["v"], lengths, dev["weights"],
                                          weights_out=dev["weights"], **args)
        R.check(out, ref["out"], bound["out"], f"step {step}")
        R.check(w, ref["weights"], bound["weights"], f"weights of step {step}")
        c["weights"] = w.cpu()


@pytest.mark.parametrize("cache", CACHES)
def test_workspace_on_sixteen_bytes(ops, monkeypatch, cache):
    """A workspace that starts on an odd multiple of 16 bytes: nothing outside it is written."""
    c = R.make_inputs(cache, 40, 1, 8, 4, 64, 600, 300, [(11 * i) % 301 for i in range(40)], seed=51)
    plain = call(ops, c) + call(ops, c, weigh=True)
    empty, around = torch.empty, []

    def shifted(*size, **more):
        if more.get("dtype") != torch.uint8:
            return empty(*size, **more)
        around.append(torch.full((size[0] + 64,), 77, **more))
        return around[-1][16:16 + size[0]]

    monkeypatch.setattr(torch, "empty", shifted)
    got = call(ops, c) + call(ops, c, weigh=True)
    assert len(around) == 2
    for x, y in zip(got, plain):
        assert torch.equal(x, y)
    for x in around:
        assert x.data_ptr() % 32 == 0 and bool((x[:16] == 77).all()) and bool((x[-48:] == 77).all())


@pytest.mark.parametrize("d", (64, 128))
def test_long_sums_keep_their_bits(ops, d):
    """Equal weights over 16000 INT8 keys of one sign: the means, where each sum that is cut and not rounded
    shows. Products: 3 steps of 16 sums, 2^-23 each; weights as pairs: 2^-21; the sums of the steps, of the
    weights and the rest: 150 roundings of 2^-24. Together 2^-16."""
    g = torch.Generator().manual_seed(d)
    b, t, heads, kv, keys = 4, 600, 16, 4, 16000
    v = torch.randint(1, 128, (kv, keys, d), generator=g, dtype=torch.int8)
    scales = torch.rand(kv, keys, generator=g) + 0.5
    mean = (v.double() * scales.double()[..., None]).mean(1)
    none = torch.zeros(b, kv, 8, d, dtype=torch.int8, device="cuda")
    out = ops.prefix_attention(torch.zeros(b, t, heads, d, device="cuda"), none, none,
                               torch.zeros(b, dtype=torch.int32, device="cuda"), prefix_k=v.cuda(), prefix_v=v.cuda(),
                               k_scales=none[..., 0].float(), v_scales=none[..., 0].float(),
                               prefix_k_scales=scales.cuda(), prefix_v_scales=scales.cuda())
    want = mean.repeat_interleave(heads // kv, 0)
    off = (out.double().cpu() - want).abs() / want
    assert float(off.max()) <= 2.0 ** -16, float(off.max())


@pytest.mark.parametrize("d", (64, 128))
def test_long_sums_of_single_tokens(ops, d):
    """The same for single tokens of sequences that fill the machine: 512 cut sums of pairs in 4096 keys, 2^-25
    each on the average (2^-16), and as much again for the merge and the rest."""
    b, kv, keys = 150, 4, 40000
    g = torch.Generator(device="cuda").manual_seed(d)
    v = torch.randint(1, 128, (b, kv, keys, d), generator=g, dtype=torch.int8, device="cuda")
    scales = torch.rand(b, kv, keys, generator=g, device="cuda") + 0.5
    out = ops.prefix_attention(torch.zeros(b, kv, d, device="cuda"), v, v,
                               torch.full((b,), keys, dtype=torch.int32, device="cuda"), k_scales=scales,
                               v_scales=scales)
    for i in (0, 70, 149):
        want = (v[i].double() * scales[i].double()[..., None]).mean(1)
        off = (out[i].double() - want).abs() / want
        assert float(off.max()) <= 2.0 ** -15, float(off.max())


@pytest.mark.parametrize("d", (64, 128))
@pytest.mark.parametrize("shared", (True, False))
def test_long_sums_in_sixteen_bits(ops, d, shared):
    """The same with 100000 FP16 keys, shared or own: cut sums 8 for 128 keys, 2^-25 each on the average, over at
    most 32768 keys: 2^-14; the output's rounding: 2^-11. Together 2^-10.8."""
    g = torch.Generator().manual_seed(d)
    b, t, heads, kv, keys = 2, 1200, 16, 4, 100000
    v = (torch.rand(b, kv, keys, d, generator=g) + 0.5).half()
    mean = v.double().mean(2)
    v = v.cuda()
    none = torch.zeros(b, kv, 8, d, dtype=torch.float16, device="cuda")
    q = torch.zeros(b, t, heads, d, dtype=torch.float16, device="cuda")
    lengths = torch.zeros(b, dtype=torch.int32, device="cuda")
    if shared:
        out = ops.prefix_attention(q, none, none, lengths, prefix_k=v[0], prefix_v=v[0])
        want = mean[:1].expand(b, kv, d)
    else:
        out = ops.prefix_attention(q, v, v, lengths + keys)[:, -1:]
        want = mean
    want = want.repeat_interleave(heads // kv, 1)[:, None]
    off = (out.double().cpu() - want).abs() / want
    assert float(off.max()) <= 2.0 ** -10.8, float(off.max())


@pytest.mark.parametrize("t", (1, 40))
def test_streams_and_graphs(ops, t):
    """Calls on a side stream, and two captured graphs replayed in turn with new inputs: each keeps its own
    workspace."""
    cs = [R.make_inputs("int8", 3, t, 8, 4, 64, 300, 100, [100, 80, 60], seed=30 + i) for i in range(3)]
    plain = [call(ops, c, weigh=True) for c in cs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    ds = [cuda(c) for c in cs]
    names = ("prefix_k", "prefix_v", "k_scales", "v_scales", "prefix_k_scales", "prefix_v_scales")

    def run(d, **more):
        out, w = ops.accumulate_attention(d["q"], d["k"], d["v"], d["lengths"], d["weights"],
                                          **{n: d[n] for n in names}, **more)
        e = ops.evict(d["k"], d["v"], w, d["lengths"], 50, recent=5, k_scales=d["k_scales"], v_scales=d["v_scales"],
                      **more)
        return out, w, e

    torch.cuda.synchronize()
    for given in (side, side.cuda_stream):
        out, w, _ = run(ds[0], stream=given)
        side.synchronize()
        assert torch.equal(out, plain[0][0]) and torch.equal(w, plain[0][1])
    eager = [run(d)[2] for d in ds]
    live = [{n: None if x is None else x.clone() for n, x in ds[i].items()} for i in range(2)]
    graphs, results = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(run(live[i]))
        graphs.append(graph)
    for a, b in ((0, 1), (2, 0), (1, 2)):
        for i, j in ((0, a), (1, b)):
            for n, x in ds[j].items():
                if x is not None:
                    live[i][n].copy_(x)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for i, j in ((0, a), (1, b)):
            assert torch.equal(results[i][0], plain[j][0]) and torch.equal(results[i][1], plain[j][1])
            for x, y in zip(results[i][2], eager[j]):
                assert torch.equal(x, y)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("t,s", [(1, 30), (1, 64), (3, 300), (40, 64)])
def test_prefix_that_is_a_view_of_the_cache(ops, cache, t, s):
    """The shared prompt kept in the first slots of sequence 0: its prefix and its own keys start at one address.
    Prefixes in a pass with the own keys (one and four warps a unit) and apart; the same as with copies."""
    c = R.make_inputs(cache, 3, t, 8, 4, 64, 0, s, [0 if t == 1 else s, s // 2 + 1, s], seed=60 + t)
    d = cuda(c)
    scales = {n: d[n] for n in ("k_scales", "v_scales")}

    def run(change):
        prefix = {"prefix_" + n: None if d[n] is None else change(d[n][0, :, :20]) for n in ("k", "v", *scales)}
        out, lse = ops.prefix_attention(d["q"], d["k"], d["v"], d["lengths"], return_lse=True, **scales, **prefix)
        return (out, lse) + ops.accumulate_attention(d["q"], d["k"], d["v"], d["lengths"], d["weights"], **scales,
                                                     **prefix)

    for x, y in zip(run(lambda x: x), run(lambda x: x.clone())):
        assert torch.equal(x, y)


def dense_reference(c):
    """cache_ops_reference.attention on the GPU, all sequences at once (a prefix, lengths of at least the tokens)."""
    g = cuda(c)
    b, t, heads, d = c["q"].shape
    kv, s = c["k"].shape[1:3]
    p, r = c["prefix_k"].shape[1], heads // kv
    wide = lambda x, sc: x.double() if sc is None else x.double() * sc.double().unsqueeze(-1)   # noqa: E731
    k, v = (torch.cat((wide(g["prefix_" + n], g[f"prefix_{n}_scales"]).expand(b, -1, -1, -1),
                       wide(g[n], g[n + "_scales"])), 2) for n in ("k", "v"))
    q = g["q"].double().view(b, t, kv, r, d).permute(0, 2, 1, 3, 4)                 # [B, KV, T, R, D]
    at = (g["lengths"].view(b, 1) - t + torch.arange(t, device="cuda")).view(b, 1, t, 1, 1)
    seen = torch.arange(-p, s, device="cuda") <= at
    z = (torch.einsum("bgtrd,bgkd->bgtrk", q, k) * d ** -0.5).masked_fill(~seen, -math.inf)
    size = (torch.einsum("bgtrd,bgkd->bgtrk", q.abs(), k.abs()) * d ** -0.5).masked_fill(~seen, 0)
    soft = torch.softmax(z, -1)
    back = lambda x: x.permute(0, 2, 1, 3, *range(4, x.dim())).reshape(b, t, heads, *x.shape[4:]).cpu()   # noqa: E731
    gained = soft[..., p:].sum((2, 3)).cpu()
    most = torch.zeros_like(z[..., 0])
    if g["v_scales"] is not None:
        scales = torch.cat((g["prefix_v_scales"].expand(b, -1, -1), g["v_scales"]), 2).double()
        most = 127 * seen.expand_as(z).sum(-1) * scales.abs().amax(-1).view(b, kv, 1, 1)
    return {"out": back(torch.einsum("bgtrk,bgkd->bgtrd", soft, v)), "lse": back(torch.logsumexp(z, -1)),
            "weights": c["weights"].double() + gained, "gained": gained, "most_v": back(most),
            "mix": back(torch.einsum("bgtrk,bgkd->bgtrd", soft, v.abs())), "dz": back(size.amax(-1)),
            "total_v": back(torch.einsum("bgtrk,bgkd->bgtrd", seen.expand_as(z).double(), v.abs()))}


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("b,t", [(1, 1), (24, 1), (6, 200)])
@pytest.mark.parametrize("expanded", [("k", "v"), ("prefix_k", "prefix_v"), ("k",), ("prefix_v",)])
def test_keys_expanded_along_their_axis(ops, cache, b, t, expanded):
    """One key's row standing for all of them (a stride of 0), at sizes that stream and that would take tiles."""
    heads, kv, p, s = 16, 4, 450, 210
    c = R.make_inputs(cache, b, t, heads, kv, 64, p, s, [s - 3 - i % 5 for i in range(b)], seed=70 + t)
    for n in expanded:
        c[n] = c[n][..., :1, :].expand_as(c[n])
    ref = dense_reference(c)
    bound = R.bounds(c, ref)
    d = {n: None if x is None else x.cuda() for n, x in c.items()}
    for n in expanded:
        d[n] = d[n][..., :1, :].contiguous().expand_as(d[n])
        assert d[n].stride(-2) == 0
    args = {n: d[n] for n in ("prefix_k", "prefix_v", "k_scales", "v_scales", "prefix_k_scales", "prefix_v_scales")
            if n in d}
    out, lse = ops.prefix_attention(d["q"], d["k"], d["v"], d["lengths"], return_lse=True, **args)
    R.check(out, ref["out"], bound["out"], "out")
    R.check(lse, ref["lse"], bound["lse"], "lse")
    out, weights = ops.accumulate_attention(d["q"], d["k"], d["v"], d["lengths"], d["weights"], **args)
    R.check(out, ref["out"], bound["out"], "out of accumulate_attention")
    R.check(weights, ref["weights"], bound["weights"], "weights")


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("b,t,axis", [(6, 200, 0), (6, 200, 1), (6, 200, 2), (3, 1, 0), (3, 1, 2)])
def test_queries_expanded_along_an_axis(ops, cache, b, t, axis):
    """The same query for every sequence, token or head, as a stride of 0."""
    c = R.make_inputs(cache, b, t, 16, 4, 64, 450, 210, [207 - i for i in range(b)], seed=80 + t)
    c["q"] = c["q"].narrow(axis, 0, 1).expand_as(c["q"])
    ref = dense_reference(c)
    bound = R.bounds(c, ref)
    d = cuda(c)
    d["q"] = d["q"].narrow(axis, 0, 1).contiguous().expand_as(d["q"])
    args = {n: d[n] for n in ("prefix_k", "prefix_v", "k_scales", "v_scales", "prefix_k_scales", "prefix_v_scales")}
    out, lse = ops.prefix_attention(d["q"], d["k"], d["v"], d["lengths"], return_lse=True, **args)
    R.check(out, ref["out"], bound["out"], "out")
    R.check(lse, ref["lse"], bound["lse"], "lse")
    out, weights = ops.accumulate_attention(d["q"], d["k"], d["v"], d["lengths"], d["weights"], **args)
    R.check(out, ref["out"], bound["out"], "out of accumulate_attention")
    R.check(weights, ref["weights"], bound["weights"], "weights")


def test_pool_query_shared_allocates_once(ops):
    """The pool's workspace does not grow with the positions."""
    import numpy as np
    kv = ops.KVCache(64, 8, 1, 128, 8192, 0, 0)
    ids = list(range(64))
    q = np.ones((64, 8 * 128), np.float32)
    kv.store(ids, [0] * 64, *(np.ones((64, 128), np.float32) for _ in range(2)))
    free = []
    for at in (0, 700, 8191):
        kv.query_shared(ids, [at] * 64, q)
        free.append(torch.cuda.mem_get_info()[0])
    assert free[0] == free[1] == free[2]


def test_pool_query_shared_in_a_graph(ops):
    """A captured call stays good when later calls are longer and of more sessions."""
    import numpy as np
    rng = np.random.default_rng(3)
    kv = ops.KVCache(64, 8, 1, 128, 4000, 0, 500)
    kv.set_prefix(*(rng.normal(size=(500, 128)).astype(np.float32) for _ in range(2)))
    for at in range(500, 4000):
        kv.store(list(range(64)), [at] * 64, *(rng.normal(size=(64, 128)).astype(np.float32) for _ in range(2)))
    q = torch.from_numpy(rng.normal(size=(64, 1024)).astype(np.float32)).cuda()
    out, want = torch.zeros(3, 1024, device="cuda"), torch.zeros(3, 1024, device="cuda")
    few = ([5, 0, 9], [610, 619, 604])
    kv.query_shared_device(*few, q, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv.query_shared_device(*few, q, out, stream=torch.cuda.current_stream())
    every = torch.zeros(64, 1024, device="cuda")
    kv.query_shared_device(list(range(64)), [3999] * 64, q, every)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    again = torch.zeros(64, 1024, device="cuda")
    kv.query_shared_device(list(range(64)), [3999] * 64, q, again)
    assert torch.equal(again, every)


@pytest.mark.parametrize("cache", ("bf16", "f16"))
@pytest.mark.parametrize("d", (64, 128))
def test_long_sums_of_single_tokens_in_sixteen_bits(ops, cache, d):
    """Single tokens of sequences that fill the machine over 262144 keys of one sign, the longest range that streams:
    a warp takes a quarter of it, 4096 cut sums of 16 keys, 2^-25 each on the average: 2^-13; the output's rounding:
    2^-11 or 2^-8; and a twentieth for the weights' sums and the merge."""
    b, kv, keys = 150, 4, 1 << 18
    g = torch.Generator(device="cuda").manual_seed(d)
    v = (torch.rand(1, kv, keys, d, generator=g, device="cuda") + 0.5).to(R.TYPES[cache])
    own = v.expand(b, -1, -1, -1)                            # the sequences' own keys: one cache for all
    q = torch.zeros(b, kv, d, dtype=v.dtype, device="cuda")
    out = ops.prefix_attention(q, own, own, torch.full((b,), keys, dtype=torch.int32, device="cuda"))
    want = v[0].double().mean(1)
    off = ((out.double() - want) / want).abs()
    assert float(off.max()) <= 1.05 * (2.0 ** -13 + torch.finfo(v.dtype).eps / 2), float(off.max())


@pytest.mark.parametrize("cache", CACHES)
def test_calls_repeat_themselves(ops, cache):
    """Bit for bit: no atomics and no order of arrival in out, lse, weights or an eviction."""
    for t, s in ((1, 900), (70, 300)):
        c = R.make_inputs(cache, 20, t, 8, 4, 64, 700, s, [t + (37 * i) % (s - t) for i in range(20)], seed=90 + t)
        first = call(ops, c) + call(ops, c, weigh=True)
        e = evicted(ops, {**c, "weights": first[3].cpu()}, 60, 2, 5)[0]
        for _ in range(5):
            got = call(ops, c) + call(ops, c, weigh=True)
            again = evicted(ops, {**c, "weights": got[3].cpu()}, 60, 2, 5)[0]
            for x, y in zip(first + tuple(e), got + tuple(again)):
                assert x is y is None or torch.equal(x, y)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("layout", ("key", "sequence"))
def test_keys_and_values_of_one_tensor(ops, cache, layout):
    """K and V rows side by side, or a sequence's behind one another: attended and thinned out in place."""
    b, kv, s, d = 3, 4, 300, 64
    c = R.make_inputs(cache, b, 1, 8, kv, d, 0, s, [300, 120, 77], seed=95)
    plain = call(ops, c, weigh=True)
    e, _ = evicted(ops, c, 90, 3, 10)
    dev = cuda(c)
    shape = (b, kv, s, 2, d) if layout == "key" else (b, 2, kv, s, d)
    whole = torch.zeros(shape, dtype=c["k"].dtype, device="cuda")
    k, v = (whole[:, :, :, i] if layout == "key" else whole[:, i] for i in (0, 1))
    k.copy_(dev["k"])
    v.copy_(dev["v"])
    scales = {n: dev[n] for n in ("k_scales", "v_scales")}
    got = ops.accumulate_attention(dev["q"], k, v, dev["lengths"], dev["weights"], **scales)
    assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])
    i = ops.evict(k, v, dev["weights"], dev["lengths"], 90, first=3, recent=10, in_place=True, **scales)
    assert torch.equal(i.indices, e.indices) and torch.equal(i.lengths, e.lengths)
    for j, n in enumerate(e.lengths.tolist()):
        for x, y in ((k, e.k), (v, e.v), (dev["weights"], e.weights)):
            assert torch.equal(x[j, :, :n], y[j, :, :n])
        assert torch.equal(k[j, :, n:], c["k"][j, :, n:].cuda()) and torch.equal(v[j, :, n:], c["v"][j, :, n:].cuda())


@pytest.mark.parametrize("in_place", (False, True))
def test_evict_beyond_32_bit_offsets(ops, in_place):
    """The last keys of a cache of 34 million INT8 rows (2.2 GB) have the weights."""
    s, n, keep, first, recent = 34_000_000, 34_000_000 - 3, 700, 10, 20
    g = torch.Generator("cuda").manual_seed(2)
    k = torch.zeros(1, 1, s, 64, dtype=torch.int8, device="cuda")
    k[:, :, -2000:] = torch.randint(-127, 128, (1, 1, 2000, 64), generator=g, device="cuda", dtype=torch.int8)
    k[:, :, :first] = 7
    v = -k
    scales = torch.rand(1, 1, s, generator=g, device="cuda")
    w = torch.zeros(1, 1, s, device="cuda")
    w[:, :, -1500:] = torch.rand(1, 1, 1500, generator=g, device="cuda") + 0.5
    x = w[0, 0, :n].clone()
    x[:first] = x[n - recent:] = 2.0
    at = torch.sort(x, descending=True, stable=True).indices[:keep].sort().values
    want = [y[0, 0][at] for y in (k, v, w, scales)]
    e = ops.evict(k, v, w, torch.tensor([n], dtype=torch.int32, device="cuda"), keep, first=first, recent=recent,
                  k_scales=scales, v_scales=scales.clone(), in_place=in_place)
    assert torch.equal(e.indices[0, 0], at.int()) and int(e.lengths) == keep
    for x, y in zip((e.k, e.v, e.weights, e.k_scales), want):
        assert torch.equal(x[0, 0, :keep], y)
    assert not e.weights[0, 0, keep:].any()


@pytest.mark.parametrize("t", (1, 100))
def test_weights_beyond_32_bit_offsets(ops, t):
    """The weights of the last keys of the same cache, and the others' as they were."""
    s, n = 34_000_000, 34_000_000 - 3
    g = torch.Generator("cuda").manual_seed(3)
    k = torch.zeros(1, 1, s, 64, dtype=torch.int8, device="cuda")
    k[:, :, -400:] = torch.randint(-127, 128, (1, 1, 400, 64), generator=g, device="cuda", dtype=torch.int8)
    scales = torch.full((1, 1, s), 0.01, device="cuda")
    q = torch.randn(1, t, 2, 64, generator=g, device="cuda")
    w = torch.rand(1, 1, s, generator=g, device="cuda")
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    _, got = ops.accumulate_attention(q, k, k, lengths, w, k_scales=scales, v_scales=scales, window=64)
    tail = slice(s - 400, s)
    _, want = ops.accumulate_attention(q, k[:, :, tail].clone(), k[:, :, tail].clone(), lengths - (s - 400),
                                       w[:, :, tail].clone(), k_scales=scales[:, :, tail].clone(),
                                       v_scales=scales[:, :, tail].clone(), window=64)
    # the same keys from the front of a small cache: only the order of the sums may differ
    assert (got[:, :, tail] - want).abs().max() <= 1e-5 * want.max()
    assert torch.equal(got[:, :, :s - 400], w[:, :, :s - 400])


def test_no_wait_ran_out(ops):
    """None of the calls above has raised the flag that a bounded wait of the tiles sets on its end."""
    from openneedle_b200 import native
    torch.cuda.synchronize()
    assert native.device_fault() == 0
