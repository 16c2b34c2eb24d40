"""The cache operators' argument checks (CPU only): what the Python entry points
refuse before they touch a GPU, and the C ABI's own refusals."""
import ctypes as ct

import pytest
import torch

import cache_ops_reference as R
from openneedle_b200 import attention, build


@pytest.fixture(scope="module", autouse=True)
def library():
    build.build()


def inputs(cache="int8", t=1):
    return R.make_inputs(cache, 2, t, 8, 4, 64, 20, 30, [30, 10])


def attend(c, weigh=False, **more):
    args = {n: c.get(n) for n in ("prefix_k", "prefix_v", "k_scales", "v_scales", "prefix_k_scales",
                                  "prefix_v_scales")}
    args.update(more)
    if weigh:
        return attention.accumulate_attention(c["q"], c["k"], c["v"], c["lengths"], c["weights"], **args)
    return attention.prefix_attention(c["q"], c["k"], c["v"], c["lengths"], **args)


def evict(c, keep=8, **more):
    return attention.evict(c["k"], c["v"], c["weights"], c["lengths"], keep,
                           **{"k_scales": c["k_scales"], "v_scales": c["v_scales"], **more})


@pytest.mark.parametrize("change,message", [
    ({"q": lambda x: x.half()}, "q must be"),
    ({"q": lambda x: x[:1]}, "q must be"),
    ({"q": lambda x: x[0, 0]}, "q must be"),
    ({"q": lambda x: x.transpose(2, 3).contiguous().transpose(2, 3)}, "last axis"),
    ({"k": lambda x: x.int()}, "int8, bfloat16 or float16"),
    ({"k": lambda x: x[0]}, "int8, bfloat16 or float16"),
    ({"v": lambda x: x[:, :, :-1]}, "v must be"),
    ({"k_scales": lambda x: None}, "needs k_scales"),
    ({"v_scales": lambda x: x.double()}, "v_scales must be"),
    ({"prefix_k": lambda x: None}, "go together"),
    ({"prefix_k": lambda x: x.half()}, "prefix_k and prefix_v must be"),
    ({"prefix_v": lambda x: x[:, :5]}, "prefix_v must be"),
    ({"prefix_v_scales": lambda x: None}, "needs prefix_k_scales"),
    ({"lengths": lambda x: x.long()}, "lengths must be"),
    ({"weights": lambda x: x[:, :, :3]}, "weights must be"),
    ({"weights": lambda x: None}, "needs weights"),
    ({"q": lambda x: x.requires_grad_()}, "no gradients"),
    ({}, "CUDA tensors")])
def test_attention_refuses(change, message):
    c = inputs()
    for n, f in change.items():
        c[n] = f(c[n])
    with pytest.raises(ValueError, match=message):
        attend(c, weigh=True)


@pytest.mark.parametrize("more,message", [
    ({"window": -1}, "window"),
    ({"tokens": torch.zeros(3, dtype=torch.int32)}, "tokens must be"),
    ({"out": torch.zeros(2, 1, 8, 64, dtype=torch.bfloat16)}, "out must be"),
    ({"out": torch.zeros(2, 1, 1, 64).expand(2, 1, 8, 64)}, "expanded"),
    ({"weights_out": torch.zeros(2, 4, 29)}, "weights_out must be")])
def test_attention_refuses_options(more, message):
    with pytest.raises(ValueError, match=message):
        attend(inputs(), weigh=True, **more)


def test_outputs_must_not_overlap_inputs():
    c = inputs()
    with pytest.raises(ValueError, match="out overlaps"):
        attend(c, out=c["q"])
    with pytest.raises(ValueError, match="weights_out overlaps"):
        whole = torch.zeros(2, 5, 30)
        c["weights"] = whole[:, :4]
        attend(c, weigh=True, weights_out=whole[:, 1:])
    c = inputs("bf16")
    with pytest.raises(ValueError, match="scales belong to INT8"):
        attend(c, k_scales=torch.zeros(2, 4, 30), v_scales=torch.zeros(2, 4, 30))
    c = inputs()
    e = attention.Evicted(c["k"][:, :, :8], c["v"], c["weights"], c["lengths"], None)
    with pytest.raises(ValueError):
        evict(c, out=e)


@pytest.mark.parametrize("more,message", [
    ({"keep": -1}, "must not"), ({"first": 5, "recent": 4}, "exceed keep"), ({"first": -1}, "must not"),
    ({"in_place": True, "out": ()}, "exclude"), ({"in_place": True, "keep": 31}, "capacity"),
    ({"k_scales": None}, "needs k_scales"), ({}, "CUDA tensors")])
def test_evict_refuses(more, message):
    with pytest.raises(ValueError, match=message):
        evict(inputs(), **{"keep": 8, **more})


# ---- the C ABI ------------------------------------------------------------------

def pack(**change):
    """A valid call of two sequences on an INT8 cache; addresses that nothing reads."""
    a = dict(batch=2, tokens=1, heads=8, kvheads=4, head_dim=64, prefix=600, capacity=32, window=0, cache_type=0,
             scale=0.125, q=4096, out=8192, k=4096, v=4096, ks=4096, vs=4096, pk=4096, pv=4096, pks=4096, pvs=4096,
             lengths=4096, counts=0, rows=0, lse=0, weights=0, weights_out=0, kstride=64)
    a.update(change)
    three, flat, flat2 = (8192, 2048, a["kstride"]), (128, 32, 1), (16, 1)
    return attention._ATTENTION_SIZES.pack(
        a["batch"], a["tokens"], a["heads"], a["kvheads"], a["head_dim"], a["prefix"], a["capacity"], a["window"],
        a["cache_type"], a["scale"], 512, 512, 64, 512, 512, 64, *three, 8192, 2048, 64, *flat, *flat, 38400, 64, 38400,
        64, *flat2, *flat2, *flat, *flat) + attention._ATTENTION_POINTERS.pack(
        a["q"], a["out"], a["k"], a["v"], a["ks"], a["vs"], a["pk"], a["pv"], a["pks"], a["pvs"], a["lengths"],
        a["counts"], a["rows"], a["lse"], a["weights"], a["weights_out"])


def test_workspace_grows_with_what_is_asked():
    lib = attention._bind_operators()[0]
    plain = lib.needle2_prefix_attention_workspace(pack())
    assert 0 < plain < lib.needle2_prefix_attention_workspace(pack(weights=4096, weights_out=4096))
    assert lib.needle2_prefix_attention_workspace(pack(batch=0)) >= 0
    assert lib.needle2_prefix_attention_workspace(None) == -1


@pytest.mark.parametrize("change,message", [
    ({"batch": -1}, "negative size"), ({"tokens": -1}, "negative size"), ({"prefix": -1}, "negative size"),
    ({"capacity": -1}, "negative size"), ({"window": -2}, "negative size"), ({"kvheads": 0}, "negative size"),
    ({"heads": 6}, "multiple of kvheads"), ({"head_dim": 96}, "head_dim"), ({"cache_type": 3}, "cache type"),
    ({"scale": 0.0}, "scale"), ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"),
    ({"batch": 1 << 30}, "too large"), ({"tokens": 1 << 28}, "too large"),
    ({"q": 0}, "q is null"), ({"q": 4104}, "q: the pointer"), ({"out": 4100}, "out: the pointer"),
    ({"k": 4097}, "k: the pointer"), ({"kstride": 72}, "k: the pointer"), ({"v": 0}, "v is null"),
    ({"ks": 0}, "needs its scales"), ({"pks": 0}, "needs its scales"), ({"pv": 0}, "prefix_v is null"),
    ({"lengths": 0}, "lengths is null"), ({"weights": 4096}, "go together"), ({}, "workspace")])
def test_c_abi_refuses(change, message):
    lib = attention._bind_operators()[0]
    assert lib.needle2_prefix_attention_device(pack(**change), None, 0, None) == -1
    assert message in attention.last_error()


@pytest.mark.parametrize("change,message", [
    ({"batch": -1}, "negative size"), ({"head_dim": 80}, "head_dim"), ({"cache_type": 7}, "cache type"),
    ({"keep": 3}, "exceed keep"), ({"out_capacity": 7}, "fewer than keep"), ({"batch": 1 << 29}, "too large"),
    ({"k": 0}, "k is null"), ({"k": 4100}, "multiples of 16"), ({"kstride": 72}, "multiples of 16"),
    ({"v_out": 4104}, "v_out"), ({"k_scales": 0}, "needs its scales"), ({"weights": 0}, "weights is null"),
    ({"weights_out": 0}, "weights_out is null"), ({"lengths": 0}, "null pointer"),
    ({"lengths": 65536}, "must not be lengths"), ({"k_out": 4096}, "in place")])
def test_c_abi_refuses_evictions(change, message):
    lib = attention._bind_operators()[0]
    a = dict(batch=2, kvheads=4, head_dim=64, capacity=32, out_capacity=32, keep=8, first=2, recent=2, cache_type=0)
    p = dict(k=4096, v=4096, k_scales=4096, v_scales=4096, weights=4096, lengths=4096, k_out=16384, v_out=16384,
             k_scales_out=16384, v_scales_out=16384, weights_out=16384, indices=16384, lengths_out=65536)
    three, flat = (8192, 2048, change.pop("kstride", 64)), (128, 32, 1)
    for n, x in change.items():
        (a if n in a else p)[n] = x
    sizes = attention._EVICT_SIZES.pack(*a.values(), *three, *three, *flat, *flat, *flat, *three, *three, *flat, *flat,
                                        *flat)
    assert lib.needle2_evict_device(sizes + attention._EVICT_POINTERS.pack(*p.values()), None) == -1
    assert message in attention.last_error()
    assert lib.needle2_evict_device(None, None) == -1


def test_keys_that_the_copy_engine_cannot_walk_are_streamed():
    """200 tokens of 8 sequences against 4096 shared keys: tiles split the prefix into few ranges, streaming into
    others, which the workspace shows; a stride of 0 along the keys is planned as streaming."""
    lib = attention._bind_operators()[0]
    sizes = {}
    for stride in (64, 0):
        args = bytearray(pack(batch=8, tokens=200, prefix=4096))
        at = attention._ATTENTION_SIZES.size - 8 * (32 - 18 - 1)       # prefix_k_stride[1]
        assert int.from_bytes(args[at:at + 8], "little") == 64
        args[at:at + 8] = stride.to_bytes(8, "little")
        sizes[stride] = lib.needle2_prefix_attention_workspace(bytes(args))
    assert 0 < sizes[64] != sizes[0] > 0


@pytest.mark.parametrize("name", ("q", "weights", "k_scales", "v_scales", "prefix_k_scales", "prefix_v_scales", "out",
                                  "weights_out"))
@pytest.mark.parametrize("forward", (False, True))
def test_attention_drops_no_gradient(name, forward):
    """Of whatever floating tensor, backward or forward mode."""
    from torch.autograd import forward_ad
    c = inputs()
    c.update(out=torch.zeros_like(c["q"]), weights_out=torch.zeros_like(c["weights"]))
    more = {n: c[n] for n in ("out", "weights_out")}
    with pytest.raises(ValueError, match="CUDA tensors"):
        attend(c, weigh=True, **more)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="CUDA tensors"):
            attend(c, weigh=True, **more)
        x = forward_ad.make_dual(c[name], torch.ones_like(c[name])) if forward else c[name].requires_grad_()
        c[name] = x
        if name in more:
            more[name] = x
        with pytest.raises(ValueError, match="no gradients"):
            attend(c, weigh=True, **more)
        with torch.no_grad(), pytest.raises(ValueError, match="no gradients" if forward else "CUDA tensors"):
            attend(c, weigh=True, **more)


@pytest.mark.parametrize("name", ("weights", "k_scales", "v_scales", "out"))
@pytest.mark.parametrize("forward", (False, True))
def test_evict_drops_no_gradient(name, forward):
    from torch.autograd import forward_ad
    c = inputs()
    out = attention.Evicted(*(torch.zeros_like(c[n][:, :, :8]) for n in ("k", "v", "weights")),
                            torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, 8, dtype=torch.int32),
                            *(torch.zeros_like(c[n][:, :, :8]) for n in ("k_scales", "v_scales")))
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="CUDA tensors"):
            evict(c, out=out)
        x = out.v_scales if name == "out" else c[name]
        x = forward_ad.make_dual(x, torch.ones_like(x)) if forward else x.requires_grad_()
        if name == "out":
            out = out._replace(v_scales=x)
        else:
            c[name] = x
        with pytest.raises(ValueError, match="no gradients"):
            evict(c, out=out)


def test_options_in_tensors_are_taken_by_value(monkeypatch):
    """A scale, a window or a count that is held in a tensor and changes in place: no plan of its earlier value."""
    scale, window, keep = torch.tensor(0.125), torch.tensor(4), torch.tensor(8)
    plans = {}
    monkeypatch.setattr(attention, "_plans", plans)
    for i in range(2):
        with pytest.raises(ValueError, match="CUDA tensors"):
            attend(inputs(), scale=scale, window=window)
        with pytest.raises(ValueError, match="CUDA tensors"):
            evict(inputs(), keep=keep, first=torch.tensor(1), recent=torch.tensor(2))
        assert len(plans) == 2 * (i + 1)
        scale *= 2
        window += 1
        keep += 1
    packed = [p[0] for p in plans.values()]
    at = attention.struct.calcsize("@9i")
    assert [attention.struct.unpack_from("@f", x, at)[0] for x in packed[::2]] == [0.125, 0.25]
    assert [attention.struct.unpack_from("@9i", x)[7] for x in packed[::2]] == [4, 5]
    assert [attention.struct.unpack_from("@9i", x)[5] for x in packed[1::2]] == [8, 9]
    with pytest.raises(ValueError, match="scale"):
        attend(inputs(), scale=torch.tensor(0.0))


def test_workspaces_are_sized_on_the_tensors_device(monkeypatch):
    """The plan of tensors of device 1, made while another device is current: the library is asked under device 1."""
    import contextlib
    from torch._subclasses.fake_tensor import FakeTensorMode
    current, asked = [0], []

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], d.index
        yield
        current[0] = before

    class Library:
        def needle2_prefix_attention_workspace(self, args):
            asked.append(current[0])
            return 0

    monkeypatch.setattr(torch.cuda, "device", device)
    types = attention._bind_operators()[2]
    with FakeTensorMode():
        q, k = (torch.empty(2, n, 5, 64, dtype=torch.bfloat16, device="cuda:1") for n in (8, 4))
        lengths = torch.empty(2, dtype=torch.int32, device="cuda:1")
        attention._plan_attention(Library(), torch, types, q.transpose(1, 2), k, k, lengths, None, None, None, None,
                                  None, None, None, None, None, 0, None, None)
    assert asked == [1] and current == [0]


def expanded(**change):
    """`pack` with keys of stride 0, which take no memory, whatever their number."""
    args = bytearray(pack(kstride=0, **change))
    at = attention.struct.calcsize("@9if") + (-attention.struct.calcsize("@9if") % 8)
    for i in (11, 18, 19, 20, 21):                          # v's, and those of the prefix
        args[at + 8 * i:at + 8 * i + 8] = bytes(8)
    return bytes(args)


@pytest.mark.parametrize("change", [
    {"capacity": 0x7f000000}, {"prefix": 0x7f000000},        # ends of key ranges
    {"capacity": 0x7d800000, "window": 0x7d700000, "tokens": 1 << 24},       # the start of a window
    {"batch": 1, "kvheads": 1, "heads": 1, "capacity": 1 << 27, "tokens": 1 << 20}])     # units of streamed keys
def test_calls_beyond_32_bit_numbers_are_refused(change):
    lib = attention._bind_operators()[0]
    assert lib.needle2_prefix_attention_workspace(expanded(**change)) == -1
    assert "too large" in attention.last_error()
    args = expanded(**change, weights=4096, weights_out=4096)
    assert lib.needle2_prefix_attention_device(args, 4096, 1 << 60, None) == -1
    assert "too large" in attention.last_error()


@pytest.mark.parametrize("change", [{"capacity": 0x7f000000}, {"out_capacity": 0x7f000000}])
def test_evictions_beyond_32_bit_indexes_are_refused(change):
    """Loops in steps of a CTA's threads would pass the largest index and never end."""
    lib = attention._bind_operators()[0]
    sizes = dict(batch=1, kvheads=1, head_dim=64, capacity=64, out_capacity=64, keep=8, first=2, recent=2,
                 cache_type=0)
    sizes.update(change)
    args = attention._EVICT_SIZES.pack(*sizes.values(), *[0] * 30) + attention._EVICT_POINTERS.pack(
        *[4096] * 5, 8192, *[16384] * 6, 65536)
    assert lib.needle2_evict_device(args, None) == -1
    assert "too large" in attention.last_error()


def test_interleaved_tensors_share_nothing():
    """Rows between one another's: K and V of one tensor, an output in a fused projection beside its queries."""
    c = inputs("bf16")
    both = torch.zeros(2, 4, 30, 2, 64, dtype=torch.bfloat16)
    per = torch.zeros(2, 2, 4, 30, 64, dtype=torch.bfloat16)
    for k, v in ((both[:, :, :, 0], both[:, :, :, 1]), (per[:, 0], per[:, 1])):
        c["k"], c["v"] = k, v
        with pytest.raises(ValueError, match="CUDA tensors"):
            evict(c, in_place=True)
        with pytest.raises(ValueError, match="CUDA tensors"):
            attend(c, out=torch.zeros(2, 1, 8, 64, dtype=torch.bfloat16))
    c["v"] = both.flatten(3)[:, :, :, 63:127]                # one value of each row is K's
    c["k"] = both[:, :, :, 0]
    with pytest.raises(ValueError, match="overlaps"):
        evict(c, in_place=True)
    fused = torch.zeros(2, 1, 24, 64, dtype=torch.bfloat16)
    c["q"] = fused[:, :, :8]
    with pytest.raises(ValueError, match="CUDA tensors"):
        attend(c, out=fused[:, :, 16:])
    with pytest.raises(ValueError, match="out overlaps"):
        attend(c, out=fused[:, :, 7:15])


def test_shared_bytes_against_a_count():
    """Whether two strided tensors share memory, against the bytes themselves."""
    import random
    rng = random.Random(5)
    seen = {True: 0, False: 0}
    for _ in range(3000):
        flat = torch.zeros(4000, dtype=torch.uint8)
        pair = []
        for size in rng.choices((1, 2, 4), k=2):
            shape = [rng.randint(1, 4) for _ in range(rng.randint(0, 3))] + [rng.choice((1, 4, 6))]
            strides = [rng.choice((0, 1, 2, 4, 6, 8, 12, 24, 40, 7, 13)) for _ in shape[:-1]] + [1]
            start = rng.randint(0, 30) * 4
            base = flat if size == 1 else flat.view(torch.int16 if size == 2 else torch.int32)
            x = base.as_strided(shape, strides, start // size)
            points = [start]
            for n, s in zip(shape, strides):
                points = [p + i * s * size for p in points for i in range(n)]
            pair.append((x, {p + i for p in points for i in range(size)}))
        (x, a), (y, b) = pair
        got = attention._share(x, y)
        seen[got] += 1
        assert got == bool(a & b), (x.shape, x.stride(), y.shape, y.stride())
    assert min(seen.values()) > 300


def test_sizes_beyond_the_librarys_numbers():
    c = inputs("bf16")
    with pytest.raises(ValueError, match="too large"):
        evict(c, keep=1 << 31)
    for scale in (1e39, 1e-50):                              # infinity and zero in 32 bits
        with pytest.raises(ValueError, match="scale must be positive and finite"):
            attend(c, scale=scale)
    for n in ("k", "v"):
        c[n] = c[n][:, :, :1].expand(2, 4, 1 << 31, 64)
    with pytest.raises(ValueError, match="too large"):
        attend(c)
    c["weights"] = c["weights"][:, :, :1].expand(2, 4, 1 << 31)
    with pytest.raises(ValueError, match="too large"):
        evict(c)
