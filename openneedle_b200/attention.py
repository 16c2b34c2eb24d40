"""Batched INT8 KV cache and attention on the GPU (ctypes over libneedle2_b200.so).

``KVCache`` holds ``sessions`` sequences of one attention layer that share one
read-only prefix (stored once on the device).  Its slot map, INT8 rule and
attention follow OpenNeedle's Engine (needle2/csrc/engine.cpp:500, 898-967,
1005-1021); ``export`` returns a session's cache in the reference's own
layout.  Host-array methods copy in and out; ``*_device`` methods take torch
CUDA tensors and do not synchronise.
"""
from __future__ import annotations

import contextlib
import ctypes as ct
import functools
import struct
from typing import NamedTuple

import numpy as np

from .native import _check, _library, _stream_ptr, last_error

_p = ct.c_void_p
_i = ct.c_int


def _bind():
    lib = _library()
    if getattr(lib, "_kv_bound", False):
        return lib
    lib.needle2_kv_create.argtypes = [_i, _i, _i, _i, _i, _i, _i]
    lib.needle2_kv_create.restype = _p
    lib.needle2_kv_destroy.argtypes = [_p]
    lib.needle2_kv_destroy.restype = None
    lib.needle2_kv_storage_bytes.argtypes = [_p]
    lib.needle2_kv_storage_bytes.restype = ct.c_size_t
    lib.needle2_kv_set_prefix.argtypes = [_p, _p, _p]
    lib.needle2_kv_set_prefix_device.argtypes = [_p, _p, _p, _p]
    lib.needle2_kv_store.argtypes = [_p, _p, _p, _p, _p, _i]
    lib.needle2_kv_store_device.argtypes = [_p, _p, _p, _p, _p, _i, _p]
    lib.needle2_attention_query.argtypes = [_p, _p, _p, _p, _p, _i]
    lib.needle2_attention_query_device.argtypes = [_p, _p, _p, _p, _p, _i, _p]
    lib.needle2_attention_query_shared.argtypes = [_p, _p, _p, _p, _p, _i]
    lib.needle2_attention_query_shared_device.argtypes = [_p, _p, _p, _p, _p, _i, _p]
    lib.needle2_attention_decode.argtypes = [_p, _p, _p, _p, _p, _p, _p, _i]
    lib.needle2_attention_decode_device.argtypes = [_p, _p, _p, _p, _p, _p, _p, _i, _p]
    lib.needle2_attention_prefill.argtypes = [_p, _p, _p, _i, _p, _p, _p, _p, _i]
    lib.needle2_attention_prefill_device.argtypes = [_p, _p, _p, _i, _p, _p, _p, _p, _i, _p]
    lib.needle2_kv_export.argtypes = [_p, _i, _p, _p, _p, _p]
    for name in ("needle2_kv_set_prefix", "needle2_kv_set_prefix_device", "needle2_kv_store",
                 "needle2_kv_store_device", "needle2_attention_query", "needle2_attention_query_device",
                 "needle2_attention_query_shared", "needle2_attention_query_shared_device",
                 "needle2_attention_decode", "needle2_attention_decode_device", "needle2_attention_prefill",
                 "needle2_attention_prefill_device", "needle2_kv_export"):
        getattr(lib, name).restype = _i
    lib._kv_bound = True
    return lib


def _f32(a):
    return np.ascontiguousarray(a, dtype=np.float32)


def _i32(a):
    return np.ascontiguousarray(a, dtype=np.int32).reshape(-1)


class KVCache:
    """INT8 KV cache of one layer for ``sessions`` sequences sharing a prefix."""

    def __init__(self, sessions, heads, kvheads, head_dim, max_seq, window=0, prefix_len=0):
        self.sessions, self.heads, self.kvheads, self.head_dim = int(sessions), int(heads), int(kvheads), int(head_dim)
        self.max_seq, self.window, self.prefix_len = int(max_seq), int(window), int(prefix_len)
        if not 0 <= self.prefix_len <= self.max_seq:
            raise ValueError("prefix_len must lie between 0 and max_seq")
        if self.heads % self.kvheads:
            raise ValueError("heads must be a multiple of kvheads")
        self._lib = _bind()
        self._handle = self._lib.needle2_kv_create(self.sessions, self.heads, self.kvheads, self.head_dim,
                                                   self.max_seq, self.window, self.prefix_len)
        if not self._handle:
            raise MemoryError(f"could not create the KV cache: {last_error()}")

    def __del__(self):
        if getattr(self, "_handle", None):
            self._lib.needle2_kv_destroy(self._handle)
            self._handle = None

    @property
    def capacity(self) -> int:
        return self.window + self.prefix_len if self.window else self.max_seq

    @property
    def storage_bytes(self) -> int:
        return int(self._lib.needle2_kv_storage_bytes(self._handle))

    def _kv_width(self):
        return self.kvheads * self.head_dim

    def set_prefix(self, k, v) -> None:
        k, v = _f32(k), _f32(v)
        if k.shape != (self.prefix_len, self._kv_width()) or v.shape != k.shape:
            raise ValueError("prefix K/V must be [prefix_len, kvheads*head_dim]")
        _check(self._lib.needle2_kv_set_prefix(self._handle, k.ctypes.data, v.ctypes.data), "kv_set_prefix")

    def store(self, session_ids, positions, k, v) -> None:
        ids, pos = _i32(session_ids), _i32(positions)
        k, v = _f32(k), _f32(v)
        if k.shape != (ids.size, self._kv_width()) or v.shape != k.shape or pos.size != ids.size:
            raise ValueError("store: k, v must be [count, kvheads*head_dim]")
        _check(self._lib.needle2_kv_store(self._handle, ids.ctypes.data, pos.ctypes.data, k.ctypes.data,
                                          v.ctypes.data, ids.size), "kv_store")

    def query(self, session_ids, positions, q):
        return self._query(self._lib.needle2_attention_query, session_ids, positions, q)

    def query_shared(self, session_ids, positions, q):
        """``query`` with the shared prefix attended once for all the sessions of
        the call (head_dim 64 or 128, positions behind the prefix): for long
        prefixes and many sessions."""
        return self._query(self._lib.needle2_attention_query_shared, session_ids, positions, q)

    def _query(self, call, session_ids, positions, q):
        ids, pos, q = _i32(session_ids), _i32(positions), _f32(q)
        if q.shape != (ids.size, self.heads * self.head_dim) or pos.size != ids.size:
            raise ValueError("query: q must be [count, heads*head_dim]")
        out = np.empty_like(q)
        _check(call(self._handle, ids.ctypes.data, pos.ctypes.data, q.ctypes.data, out.ctypes.data, ids.size),
               "attention_query")
        return out

    def decode(self, session_ids, positions, q, k, v):
        ids, pos, q, k, v = _i32(session_ids), _i32(positions), _f32(q), _f32(k), _f32(v)
        n = ids.size
        if q.shape != (n, self.heads * self.head_dim) or k.shape != (n, self._kv_width()) or v.shape != k.shape:
            raise ValueError("decode: q [count, heads*hd], k/v [count, kvheads*hd]")
        out = np.empty_like(q)
        _check(self._lib.needle2_attention_decode(self._handle, ids.ctypes.data, pos.ctypes.data, q.ctypes.data,
                                                  k.ctypes.data, v.ctypes.data, out.ctypes.data, n),
               "attention_decode")
        return out

    def prefill(self, session_ids, start_positions, q, k, v):
        """q [count, tokens, heads*hd], k/v [count, tokens, kvheads*hd] -> out like q."""
        ids, pos, q, k, v = _i32(session_ids), _i32(start_positions), _f32(q), _f32(k), _f32(v)
        n = ids.size
        if q.ndim != 3 or q.shape[0] != n or q.shape[2] != self.heads * self.head_dim:
            raise ValueError("prefill: q must be [count, tokens, heads*head_dim]")
        t = q.shape[1]
        if k.shape != (n, t, self._kv_width()) or v.shape != k.shape:
            raise ValueError("prefill: k/v must be [count, tokens, kvheads*head_dim]")
        out = np.empty_like(q)
        _check(self._lib.needle2_attention_prefill(self._handle, ids.ctypes.data, pos.ctypes.data, t, q.ctypes.data,
                                                   k.ctypes.data, v.ctypes.data, out.ctypes.data, n),
               "attention_prefill")
        return out

    def export(self, session: int) -> dict:
        cap, w = self.capacity, self._kv_width()
        r = {"keys_i8": np.zeros((cap, w), np.int8), "values_i8": np.zeros((cap, w), np.int8),
             "k_scales": np.zeros((cap, self.kvheads), np.float32),
             "v_scales": np.zeros((cap, self.kvheads), np.float32)}
        _check(self._lib.needle2_kv_export(self._handle, int(session), r["keys_i8"].ctypes.data,
                                           r["values_i8"].ctypes.data, r["k_scales"].ctypes.data,
                                           r["v_scales"].ctypes.data), "kv_export")
        return r

    # ---- device tensors (torch CUDA, contiguous float32); ids/positions are host arrays
    def set_prefix_device(self, k, v, stream=None) -> None:
        _check(self._lib.needle2_kv_set_prefix_device(self._handle, k.data_ptr(), v.data_ptr(), _stream_ptr(stream)),
               "kv_set_prefix_device")

    def decode_device(self, session_ids, positions, q, k, v, out, stream=None) -> None:
        ids, pos = _i32(session_ids), _i32(positions)
        _check(self._lib.needle2_attention_decode_device(self._handle, ids.ctypes.data, pos.ctypes.data, q.data_ptr(),
                                                         k.data_ptr(), v.data_ptr(), out.data_ptr(), ids.size,
                                                         _stream_ptr(stream)), "attention_decode_device")

    def store_device(self, session_ids, positions, k, v, stream=None) -> None:
        ids, pos = _i32(session_ids), _i32(positions)
        _check(self._lib.needle2_kv_store_device(self._handle, ids.ctypes.data, pos.ctypes.data, k.data_ptr(),
                                                 v.data_ptr(), ids.size, _stream_ptr(stream)), "kv_store_device")

    def query_device(self, session_ids, positions, q, out, stream=None) -> None:
        ids, pos = _i32(session_ids), _i32(positions)
        _check(self._lib.needle2_attention_query_device(self._handle, ids.ctypes.data, pos.ctypes.data, q.data_ptr(),
                                                        out.data_ptr(), ids.size, _stream_ptr(stream)),
               "attention_query_device")

    def query_shared_device(self, session_ids, positions, q, out, stream=None) -> None:
        ids, pos = _i32(session_ids), _i32(positions)
        _check(self._lib.needle2_attention_query_shared_device(self._handle, ids.ctypes.data, pos.ctypes.data,
                                                               q.data_ptr(), out.data_ptr(), ids.size,
                                                               _stream_ptr(stream)), "attention_query_shared_device")

    def prefill_device(self, session_ids, start_positions, tokens, q, k, v, out, stream=None) -> None:
        ids, pos = _i32(session_ids), _i32(start_positions)
        _check(self._lib.needle2_attention_prefill_device(self._handle, ids.ctypes.data, pos.ctypes.data, int(tokens),
                                                          q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                                          ids.size, _stream_ptr(stream)), "attention_prefill_device")


# ---- stateless operators on caches that the caller owns ---------------------------
#
# These take torch CUDA tensors with any strides whose last axis is contiguous
# (rows on 16-byte boundaries), run on torch's current stream or on `stream`
# without synchronising, allocate through torch (results and workspace belong to
# that stream, so captured graphs each keep their own) and have no gradients.
# Inputs may be views of one another; outputs share no byte with them unless a call
# says so. A bounded wait of a kernel that ran out, which no working order brings
# about, leaves NaN in the call's outputs and sets native.device_fault().

# needle2_prefix_attention_args and needle2_evict_args: sizes and strides, then the pointers
_ATTENTION_SIZES = struct.Struct("@9if32q")
_ATTENTION_POINTERS = struct.Struct("@16P")
_EVICT_SIZES = struct.Struct("@9i0q30q")
_EVICT_POINTERS = struct.Struct("@13P")


class Evicted(NamedTuple):
    """What ``evict`` leaves: the packed cache, and which keys stayed."""
    k: object
    v: object
    weights: object
    lengths: object
    indices: object
    k_scales: object = None
    v_scales: object = None


@functools.lru_cache(maxsize=1)
def _bind_operators():
    lib = _library()
    lib.needle2_prefix_attention_workspace.argtypes = [ct.c_char_p]
    lib.needle2_prefix_attention_workspace.restype = ct.c_longlong
    lib.needle2_prefix_attention_device.argtypes = [ct.c_char_p, _p, ct.c_longlong, _p]
    lib.needle2_prefix_attention_device.restype = _i
    lib.needle2_evict_device.argtypes = [ct.c_char_p, _p]
    lib.needle2_evict_device.restype = _i
    import torch
    types = {torch.int8: (0, torch.float32), torch.bfloat16: (1, torch.bfloat16), torch.float16: (2, torch.float16)}

    def current_stream(index):
        return torch.cuda.current_stream(index).cuda_stream

    return (lib, torch, types, getattr(torch._C, "_cuda_getCurrentRawStream", current_stream),
            torch.autograd.forward_ad)


def _on_stream(torch, device, stream):
    """The context in which torch allocates and launches for `device` and `stream` (None: the current one); None
    where that is the present one."""
    if device.type != "cuda":
        raise ValueError("the operators run on CUDA tensors")
    if stream is None:
        return None if torch.cuda.current_device() == device.index else torch.cuda.device(device)
    if not isinstance(stream, torch.cuda.Stream):
        handle = _stream_ptr(stream)
        stream = torch.cuda.ExternalStream(handle, device=device) if handle else torch.cuda.default_stream(device)
    if stream.device != device:
        raise ValueError("the stream belongs to another device than the tensors")
    return torch.cuda.stream(stream)


def _want(x, name, shape, dtype, device, last=True):
    if x.dtype != dtype or x.shape != shape or x.device != device:
        raise ValueError(f"{name} must be a {dtype} tensor of shape {tuple(shape)} on {device}, got {x.dtype} "
                         f"{tuple(x.shape)} on {x.device}")
    if last and x.stride(-1) != 1 and x.shape[-1] > 1:
        raise ValueError(f"{name}: the last axis must be contiguous")


def _extent(x, name=None):
    """The bytes from a tensor's first element to behind its last (0 for None); outputs, which are named, must not
    be expanded."""
    if x is None or not x.numel():
        return 0
    if x.is_contiguous():
        return x.nbytes
    if name and any(s == 0 and n > 1 for n, s in zip(x.shape, x.stride())):
        raise ValueError(f"{name} must not be expanded")
    return (1 + sum((n - 1) * s for n, s in zip(x.shape, x.stride()))) * x.element_size()


def _apart(outs, ins):
    """Refuse outputs that share memory with an input or with one another; (tensor, bytes, name) and (tensor, bytes)."""
    ins = list(ins)
    spans = sorted([(x.data_ptr(), n, name) for x, n, name in outs if n] + [(x.data_ptr(), n, "") for x, n in ins if n])
    end = end_out = 0                                      # of all spans, of the outputs' so far
    for start, n, name in spans:
        if start < (end if name else end_out):
            break
        end = max(end, start + n)
        if name:
            end_out = max(end_out, start + n)
    else:
        return
    # address ranges meet: those of rows that lie between one another's (K and V of one tensor) may share nothing
    for i, (x, n, name) in enumerate(outs):
        for y, m in [o[:2] for o in outs[i + 1:]] + ins:
            if n and m and x.data_ptr() < y.data_ptr() + m and y.data_ptr() < x.data_ptr() + n and _share(x, y):
                raise ValueError(f"{name} overlaps an input or another output")


def _axes(x):
    """A tensor's axes as [(stride, elements)] in bytes, and the bytes that are contiguous at each of their points."""
    width = x.element_size()
    axes = sorted((s * width, n) for n, s in zip(x.shape, x.stride()) if n > 1)
    while axes and axes[0][0] <= width:                    # (0: expanded)
        s, n = axes.pop(0)
        width += (n - 1) * s
    return axes, width


def _share(x, y):
    """Whether any byte belongs to both tensors (or may, where their strides are too involved to tell)."""
    (xa, xw), (ya, yw) = _axes(x), _axes(y)
    steps = {}                                             # stride: the range of the difference of x's and y's index
    for s, n in xa:
        lo, hi = steps.get(s, (0, 0))
        steps[s] = lo, hi + n - 1
    for s, n in ya:
        lo, hi = steps.get(s, (0, 0))
        steps[s] = lo - n + 1, hi
    steps = sorted(steps.items(), reverse=True)
    budget = 1000

    def meets(i, low, high):                               # a sum of the steps from i on in [low, high]
        nonlocal budget
        budget -= 1
        if budget < 0:
            return True
        if i == len(steps):
            return low <= 0 <= high
        s, (lo, hi) = steps[i]
        least, most = (sum(r[e] * t for t, r in steps[i + 1:]) for e in (0, 1))
        first, last = max(lo, -((most - low) // s)), min(hi, (high - least) // s)
        return any(meets(i + 1, low - d * s, high - d * s) for d in range(first, last + 1))

    # x's byte minus y's: x.ptr + steps - y.ptr, within (-xw, yw)
    offset = x.data_ptr() - y.data_ptr()
    return meets(0, 1 - xw - offset, yw - 1 - offset)


def _require(*tensors):
    """Whether any of the tensors requires gradients (a plan's answer: it is kept by their layouts, see _layout)."""
    return any(x is not None and x.requires_grad for x in tensors)


def _no_gradients(torch, forward, require, *tensors):
    """Refuse tensors whose gradients or forward-mode tangents the call would drop (INT8 codes have none, their scales
    may)."""
    if require and torch.is_grad_enabled():
        raise ValueError("these operators have no gradients: detach the inputs or call them under torch.no_grad()")
    if any(x is not None and forward.unpack_dual(x).tangent is not None for x in tensors):
        raise ValueError("these operators have no gradients: detach the inputs of their tangents")


def _want_cache(torch, k, v, k_scales, v_scales, shape, name):
    """Check K, V and their scales of a cache of the given shape."""
    _want(k, name + "k", shape, k.dtype, k.device)
    _want(v, name + "v", shape, k.dtype, k.device)
    if k.dtype == torch.int8:
        if k_scales is None or v_scales is None:
            raise ValueError(f"an INT8 cache needs {name}k_scales and {name}v_scales")
        _want(k_scales, name + "k_scales", shape[:-1], torch.float32, k.device, last=False)
        _want(v_scales, name + "v_scales", shape[:-1], torch.float32, k.device, last=False)
    elif k_scales is not None or v_scales is not None:
        raise ValueError(f"{name}k_scales and {name}v_scales belong to INT8 caches only")


def _strides(axes, *tensors):
    """The first `axes` strides of each tensor, zeros for None."""
    return [n for x in tensors for n in ((0,) * axes if x is None else x.stride()[:axes])]


def _pack(sizes, *numbers):
    try:
        return sizes.pack(*numbers)
    except struct.error:
        raise ValueError("the call is too large: its sizes do not fit the library's numbers") from None


def _layout(x):
    return None if x is None else (x.shape, x.stride(), x.dtype, x.get_device(), x.requires_grad)


def _pointer(x):
    return 0 if x is None else x.data_ptr()


# What the checks of a call's shapes, strides, types and options came to: its
# packed sizes and workspace, by those alone.
_plans = {}
_MOST_PLANS = 512


def _remember(key, plan):
    if len(_plans) >= _MOST_PLANS:
        _plans.clear()
    _plans[key] = plan
    return plan


def _plan_attention(lib, torch, types, q, k, v, lengths, weights, weights_out, prefix_k, prefix_v, k_scales, v_scales,
                    prefix_k_scales, prefix_v_scales, tokens, window, scale, out):
    """Check a call; its packed sizes, its workspace's bytes and what follows from its shapes."""
    if k.dim() != 4 or k.dtype not in types:
        raise ValueError("k and v must be [batch, kvheads, capacity, head_dim] of int8, bfloat16 or float16")
    batch, kvheads, capacity, head_dim = k.shape
    device = k.device
    cache_type, qtype = types[k.dtype]
    if q.dim() not in (3, 4):
        raise ValueError("q must be [batch, tokens, heads, head_dim], or [batch, heads, head_dim] for one token")
    single = q.dim() == 3
    count, heads = (1, q.shape[1]) if single else q.shape[1:3]
    _want(q, "q", (batch, heads, head_dim) if single else (batch, count, heads, head_dim), qtype, device)
    _want_cache(torch, k, v, k_scales, v_scales, (batch, kvheads, capacity, head_dim), "")
    prefix = 0
    if (prefix_k is None) != (prefix_v is None):
        raise ValueError("prefix_k and prefix_v go together")
    if prefix_k is not None:
        if prefix_k.dim() != 3 or prefix_k.dtype != k.dtype or prefix_k.device != device:
            raise ValueError("prefix_k and prefix_v must be [kvheads, prefix, head_dim] of the cache's type and device")
        prefix = prefix_k.shape[1]
        _want_cache(torch, prefix_k, prefix_v, prefix_k_scales, prefix_v_scales, (kvheads, prefix, head_dim),
                    "prefix_")
    elif prefix_k_scales is not None or prefix_v_scales is not None:
        raise ValueError("prefix scales without a prefix")
    _want(lengths, "lengths", (batch,), torch.int32, device)
    if tokens is not None:
        _want(tokens, "tokens", (batch,), torch.int32, device)
        if not tokens.is_contiguous():
            raise ValueError("tokens must be contiguous")
    if not lengths.is_contiguous():
        raise ValueError("lengths must be contiguous")
    if window < 0:
        raise ValueError("window must not be negative")
    window = 0 if window >= capacity else window
    scale = head_dim ** -0.5 if scale is None else scale
    if weights is not None:
        _want(weights, "weights", (batch, kvheads, capacity), torch.float32, device, last=False)
    if out is not None:
        _want(out, "out", q.shape, qtype, device)
    if weights_out is not None:
        _want(weights_out, "weights_out", (batch, kvheads, capacity), torch.float32, device, last=False)
    weigh = weights is not None and capacity > 0

    def rows(x):                                           # batch, token, head
        if x is None:                                      # a new tensor
            return [count * heads * head_dim, heads * head_dim, head_dim]
        return [x.stride(0), 0, x.stride(1)] if single else list(x.stride()[:3])

    wide = [kvheads * capacity, capacity, 1] if weights_out is None else list(weights_out.stride())
    sizes = _pack(
        _ATTENTION_SIZES, batch, count, heads, kvheads, head_dim, prefix, capacity, window, cache_type, scale, *rows(q),
        *rows(out), *_strides(3, k, v, k_scales, v_scales), *_strides(2, prefix_k, prefix_v, prefix_k_scales, prefix_v_scales),
        *_strides(3, weights), *wide)
    one = 4096 if weigh else 0                             # (given or not: the pointers are not read)
    # the split goes by the multiprocessors of the current device, which has to be the tensors' then as in the call
    with torch.cuda.device(device) if device.type == "cuda" else contextlib.nullcontext():
        size = lib.needle2_prefix_attention_workspace(sizes + _ATTENTION_POINTERS.pack(*[4096] * 14, one, one))
    if size < 0:
        raise ValueError(last_error())
    extents = None
    if out is not None or weights_out is not None:
        extents = ([_extent(out, "out"), _extent(weights_out, "weights_out")],
                   [_extent(x) for x in (q, k, v, prefix_k, prefix_v, lengths, tokens, k_scales, v_scales,
                                         prefix_k_scales, prefix_v_scales, weights)])
    require = _require(q, k, v, prefix_k, prefix_v, weights, k_scales, v_scales, prefix_k_scales, prefix_v_scales, out,
                       weights_out)
    return sizes, size, (batch, count, heads), weigh, extents, require


def _attend(q, k, v, lengths, weights, weights_out, prefix_k, prefix_v, k_scales, v_scales, prefix_k_scales,
            prefix_v_scales, tokens, window, scale, out, return_lse, stream):
    lib, torch, types, raw_stream, forward = _bind_operators()
    # (numbers from here on: a plan is kept by its options' values, not by the objects that held them)
    window, scale = int(window), None if scale is None else float(scale)
    key = (_layout(q), _layout(k), _layout(v), _layout(lengths), _layout(weights), _layout(weights_out),
           _layout(prefix_k), _layout(prefix_v), _layout(k_scales), _layout(v_scales), _layout(prefix_k_scales),
           _layout(prefix_v_scales), _layout(tokens), window, scale, _layout(out))
    plan = _plans.get(key)
    if plan is None:
        plan = _remember(key, _plan_attention(lib, torch, types, q, k, v, lengths, weights, weights_out, prefix_k,
                                              prefix_v, k_scales, v_scales, prefix_k_scales, prefix_v_scales, tokens,
                                              window, scale, out))
    sizes, size, rows, weigh, extents, require = plan
    if require or getattr(forward, "_current_level", 0) >= 0:    # (inside of a dual level)
        _no_gradients(torch, forward, require, q, k, v, prefix_k, prefix_v, weights, k_scales, v_scales,
                      prefix_k_scales, prefix_v_scales, out, weights_out)
    device = k.device
    if extents is not None:
        same = weights_out is not None and weights_out.data_ptr() == weights.data_ptr() and \
            weights_out.stride() == weights.stride()
        (n_out, n_weights), n_in = extents
        _apart([(out, n_out, "out"), (weights_out, n_weights, "weights_out")],
               zip((q, k, v, prefix_k, prefix_v, lengths, tokens, k_scales, v_scales, prefix_k_scales, prefix_v_scales,
                    weights), n_in[:-1] if same else n_in))
    context = _on_stream(torch, device, stream)
    if context is not None:
        with context:
            return _attend(q, k, v, lengths, weights, weights_out, prefix_k, prefix_v, k_scales, v_scales,
                           prefix_k_scales, prefix_v_scales, tokens, window, scale, out, return_lse, None)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty(rows, dtype=torch.float32, device=device) if return_lse else None
    if weights is not None and weights_out is None:
        weights_out = torch.empty_like(weights, memory_format=torch.contiguous_format)
    workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    args = sizes + _ATTENTION_POINTERS.pack(
        q.data_ptr(), out.data_ptr(), k.data_ptr(), v.data_ptr(), _pointer(k_scales), _pointer(v_scales),
        _pointer(prefix_k), _pointer(prefix_v), _pointer(prefix_k_scales), _pointer(prefix_v_scales),
        lengths.data_ptr(), _pointer(tokens), 0, _pointer(lse), weights.data_ptr() if weigh else 0,
        weights_out.data_ptr() if weigh else 0)
    if lib.needle2_prefix_attention_device(args, _pointer(workspace), size, raw_stream(device.index)):
        _check(-1, "prefix_attention")
    if return_lse and q.dim() == 3:
        lse = lse.squeeze(1)
    return out, lse, weights_out


def prefix_attention(q, k, v, lengths, prefix_k=None, prefix_v=None, *, k_scales=None, v_scales=None,
                     prefix_k_scales=None, prefix_v_scales=None, tokens=None, window=0, scale=None, out=None,
                     return_lse=False, stream=None):
    """Attention of a batch of sequences that share one prefix, whose part is
    computed once for all of them.

    ``q`` [batch, tokens, heads, head_dim] ([batch, heads, head_dim] for one
    token each); ``k``, ``v`` [batch, kvheads, capacity, head_dim] the
    sequences' own keys, of which sequence b has ``lengths[b]`` (int32), those of
    the new tokens among them; ``prefix_k``, ``prefix_v`` [kvheads, prefix,
    head_dim].  Caches are bfloat16 or float16 (q and the result too), or int8
    with float32 scales [.., capacity] / [kvheads, prefix] (q and the result
    float32).  head_dim is 64 or 128.

    Token t of sequence b stands at own index ``lengths[b] - tokens[b] + t`` and
    sees the whole prefix and its own keys up to there, the last ``window`` of
    them if window > 0.  ``tokens`` (int32 [batch]) says how many of q's tokens a
    sequence has; rows behind them are left as they were in ``out`` (in new
    tensors, as in the returned lse, they hold anything).  A query that sees nothing
    gets zeros.  With ``return_lse`` also the natural logarithm of the softmax's
    denominators, float32 [batch, tokens, heads]."""
    out, lse, _ = _attend(q, k, v, lengths, None, None, prefix_k, prefix_v, k_scales, v_scales, prefix_k_scales,
                          prefix_v_scales, tokens, window, scale, out, return_lse, stream)
    return (out, lse) if return_lse else out


def accumulate_attention(q, k, v, lengths, weights, prefix_k=None, prefix_v=None, *, k_scales=None, v_scales=None,
                         prefix_k_scales=None, prefix_v_scales=None, tokens=None, window=0, scale=None, out=None,
                         weights_out=None, stream=None):
    """``prefix_attention``, which also adds to each own key the softmax weights
    that the call gave it: ``weights_out[b, g, j] = weights[b, g, j] + `` the sum
    over the sequence's queries and the query heads of KV head g.  ``weights`` is
    float32 [batch, kvheads, capacity]; ``weights_out`` may be ``weights``.
    Returns (out, weights_out)."""
    if weights is None:
        raise ValueError("accumulate_attention needs weights")
    out, _, weights_out = _attend(q, k, v, lengths, weights, weights_out, prefix_k, prefix_v, k_scales, v_scales,
                                  prefix_k_scales, prefix_v_scales, tokens, window, scale, out, False, stream)
    return out, weights_out


def evict(k, v, weights, lengths, keep, *, first=0, recent=0, k_scales=None, v_scales=None, out=None, in_place=False,
          stream=None):
    """Thin out a cache by the weights that ``accumulate_attention`` gathered.

    Of a sequence's ``lengths[b]`` keys, ``keep`` stay per KV head where there
    are more: the first ``first``, the last ``recent`` and, of those between
    them, the ones of the largest weight (the lower index of equal ones, NaN as
    -inf).  They are packed in their order into the front of the result, an
    ``Evicted`` of k, v, weights [batch, kvheads, n, ..], lengths, indices
    [batch, kvheads, keep] (-1 behind the kept) and an INT8 cache's scales.
    Slots behind the kept keys have weight 0 and otherwise stay as they were.

    The result goes to ``out`` (an ``Evicted`` of tensors with n >= keep slots),
    to the inputs themselves (``in_place``; lengths and indices are new), or to
    new tensors of ``keep`` slots, zero behind the kept keys."""
    lib, torch, types, raw_stream, forward = _bind_operators()
    keep, first, recent, in_place = int(keep), int(first), int(recent), bool(in_place)   # (by value, as above)
    key = (_layout(k), _layout(v), _layout(weights), _layout(lengths), _layout(k_scales), _layout(v_scales), keep,
           first, recent, in_place, None if out is None else tuple(map(_layout, out)))
    plan = _plans.get(key)
    if plan is None:
        plan = _remember(key, _plan_evict(torch, types, k, v, weights, lengths, keep, first, recent, k_scales, v_scales,
                                          out, in_place))
    sizes, shape, (n_out, n_in), require = plan
    if require or getattr(forward, "_current_level", 0) >= 0:
        _no_gradients(torch, forward, require, k, v, weights, k_scales, v_scales, *(() if out is None else out))
    if in_place:
        _apart([(x, n, "the cache") for x, n in zip((k, v, weights, k_scales, v_scales), n_out)], [(lengths, n_in[0])])
    elif out is not None:
        _apart([(x, n, "out") for x, n in zip(out, n_out)], zip((k, v, weights, lengths, k_scales, v_scales), n_in))
    device = k.device
    context = _on_stream(torch, device, stream)
    if context is not None:
        with context:
            return evict(k, v, weights, lengths, keep, first=first, recent=recent, k_scales=k_scales, v_scales=v_scales,
                         out=out, in_place=in_place)
    if in_place:
        out = Evicted(k, v, weights, torch.empty(shape[:1], dtype=torch.int32, device=device),
                      torch.empty(shape, dtype=torch.int32, device=device), k_scales, v_scales)
    elif out is None:
        f32 = {"dtype": torch.float32, "device": device}
        out = Evicted(torch.zeros((*shape, k.shape[3]), dtype=k.dtype, device=device),
                      torch.zeros((*shape, k.shape[3]), dtype=k.dtype, device=device), torch.empty(shape, **f32),
                      torch.empty(shape[:1], dtype=torch.int32, device=device),
                      torch.empty(shape, dtype=torch.int32, device=device),
                      None if k_scales is None else torch.zeros(shape, **f32),
                      None if v_scales is None else torch.zeros(shape, **f32))
    else:
        out = Evicted(*out)
    args = sizes + _EVICT_POINTERS.pack(
        k.data_ptr(), v.data_ptr(), _pointer(k_scales), _pointer(v_scales), weights.data_ptr(), lengths.data_ptr(),
        out.k.data_ptr(), out.v.data_ptr(), _pointer(out.k_scales), _pointer(out.v_scales), out.weights.data_ptr(),
        out.indices.data_ptr(), out.lengths.data_ptr())
    if lib.needle2_evict_device(args, raw_stream(device.index)):
        _check(-1, "evict")
    return out


def _plan_evict(torch, types, k, v, weights, lengths, keep, first, recent, k_scales, v_scales, out, in_place):
    """Check an eviction; its packed sizes, [batch, kvheads, keep], the tensors' extents in bytes, and whether any of
    them requires gradients."""
    if k.dim() != 4 or k.dtype not in types:
        raise ValueError("k and v must be [batch, kvheads, capacity, head_dim] of int8, bfloat16 or float16")
    batch, kvheads, capacity, head_dim = k.shape
    device = k.device
    if keep < 0 or first < 0 or recent < 0 or first + recent > keep:
        raise ValueError("first and recent must not be negative, nor exceed keep together")
    _want_cache(torch, k, v, k_scales, v_scales, (batch, kvheads, capacity, head_dim), "")
    _want(weights, "weights", (batch, kvheads, capacity), torch.float32, device, last=False)
    _want(lengths, "lengths", (batch,), torch.int32, device)
    if not lengths.is_contiguous():
        raise ValueError("lengths must be contiguous")
    slots = keep
    new = [kvheads * keep, keep, 1]
    to = [keep * kvheads * head_dim, keep * head_dim, head_dim] * 2 + new * 2 + new
    if in_place:
        if out is not None:
            raise ValueError("evict: out and in_place exclude each other")
        if keep > capacity:
            raise ValueError("evict: in place, keep must not exceed the capacity")
        slots, to = capacity, _strides(3, k, v, k_scales, v_scales, weights)
    elif out is not None:
        out = Evicted(*out)
        if out.k.dim() != 4 or out.k.shape[2] < keep or out.k.dtype != k.dtype or out.k.device != device:
            raise ValueError("evict: out.k must be a cache of the input's type with at least keep slots")
        slots = out.k.shape[2]
        _want_cache(torch, out.k, out.v, out.k_scales, out.v_scales, (batch, kvheads, slots, head_dim), "out.")
        _want(out.weights, "out.weights", (batch, kvheads, slots), torch.float32, device, last=False)
        _want(out.lengths, "out.lengths", (batch,), torch.int32, device)
        _want(out.indices, "out.indices", (batch, kvheads, keep), torch.int32, device)
        if not out.indices.is_contiguous() or not out.lengths.is_contiguous():
            raise ValueError("out.indices and out.lengths must be contiguous")
        to = _strides(3, out.k, out.v, out.k_scales, out.v_scales, out.weights)
    extents = [], []
    if in_place:
        extents = [_extent(x, "the cache") for x in (k, v, weights, k_scales, v_scales)], [_extent(lengths)]
    elif out is not None:
        extents = ([_extent(x, "out") for x in out],
                   [_extent(x) for x in (k, v, weights, lengths, k_scales, v_scales)])
    sizes = _pack(_EVICT_SIZES, batch, kvheads, head_dim, capacity, slots, keep, first, recent, types[k.dtype][0],
                  *_strides(3, k, v, k_scales, v_scales, weights), *to)
    require = _require(k, v, weights, k_scales, v_scales, *(() if out is None else out))
    return sizes, (batch, kvheads, keep), extents, require
