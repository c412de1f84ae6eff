"""Attention over a paged key-value cache (include/r9vx_attn.h): rotary positions
and the write into the cache, attention of the next tokens and of prompts.

The cache is two tensors [pages, page_size, kv_heads, head_dim] of bf16 or f16,
whose strides may be any as long as the last axis is dense: a permuted
[pages, kv_heads, page_size, head_dim], or both in one allocation.  `table`
(int32 [sequences, columns]) names a sequence's pages in order, `slots` (int64)
places of the whole cache, page * page_size + place.  Calls check what the host
can see of their operands and raise R9vxError; what only the device sees
(a page, a length or a slot out of range) makes the rows it touches NaN, or
writes nothing, and is or-ed into `status`, a device int32 of one element that
the caller clears.
"""
from __future__ import annotations

import functools
import math
import numbers
import struct

from . import ffi
from .ffi import BF16, F16, F32, R9vxError

HEAD_DIMS = (64, 96, 128, 192, 256)

# RopeKvArgs and AttnArgs as bytes: the pointers of a call, and what its operands' shapes and strides give
_ROPE_POINTERS, _ROPE_REST = struct.Struct("10P"), struct.Struct("14Q2I")
_ATTN_POINTERS, _ATTN_REST = struct.Struct("12P"), struct.Struct("13Q4I")


def rope_freqs(rot, base=10000.0, scaling="none", factor=1.0, original_length=0, factors=None, beta_fast=32.0, beta_slow=1.0,
               device="cuda"):
    """(f64 [rot / 2] radians a position, amplitude) for `rope_kv` and `rope`:
    base^(-2i / rot), with factors (rot / 2 numbers) divided by them, and

    linear  divided by `factor`;
    yarn    divided by `factor` where a pair turns less than beta_slow times over
            original_length positions, kept where it turns more than beta_fast
            times, by a straight ramp over the pairs between; amplitude
            1 + 0.1 ln(factor)."""
    import torch

    if rot <= 0 or rot % 16:
        raise R9vxError(-103, f"rot={rot} must be a positive multiple of 16")
    if not base > 1.0 or not factor >= 1.0:
        raise R9vxError(-103, f"base={base} must exceed 1, factor={factor} be at least 1")
    if scaling not in ("none", "linear", "yarn"):
        raise R9vxError(-103, f"scaling {scaling!r}: none, linear or yarn")
    if factors is not None and len(factors) != rot // 2:
        raise R9vxError(-103, f"{len(factors)} factors: rot={rot} has {rot // 2} pairs")
    freqs = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    amplitude = 1.0
    if scaling == "linear":
        freqs = [f / factor for f in freqs]
    if scaling == "yarn":
        if original_length <= 0:
            raise R9vxError(-103, f"original_length={original_length}: yarn goes by the length a model was trained at")

        def pair(turns):  # the (fractional) pair that turns so often over original_length
            return rot * math.log(original_length / (2.0 * math.pi * turns)) / (2.0 * math.log(base))

        low, high = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), rot - 1)
        ramp = [min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(rot // 2)]
        freqs = [f * (1.0 - r) + f / factor * r for f, r in zip(freqs, ramp)]
        amplitude = 1.0 + 0.1 * math.log(factor)
    if factors is not None:
        freqs = [f / float(d) for f, d in zip(freqs, factors)]
    return torch.tensor(freqs, dtype=torch.float64, device=device), amplitude


class _Types:
    torch = None


def _types():
    T = ffi._fp8()
    if _Types.torch is None:
        _Types.f64, _Types.i32, _Types.i64 = (T.torch.float64,), (T.torch.int32,), (T.torch.int64,)
        _Types.halves = (T.torch.bfloat16, T.torch.float16)
        _Types.rows = (T.torch.bfloat16, T.torch.float16, T.torch.float32)
        _Types.code = {T.torch.float32: F32, T.torch.bfloat16: BF16, T.torch.float16: F16}
        _Types.torch = T.torch
    return _Types


@functools.lru_cache(maxsize=4096)
def _bits(x):
    try:
        return struct.unpack("<I", struct.pack("<f", x))[0]
    except (OverflowError, struct.error):
        raise R9vxError(-103, f"{x!r} is no f32 number") from None


# A decode step makes these calls in every layer and each takes a few microseconds
# on the GPU.  What a call checks and fills in goes by its operands' shapes, strides,
# types and devices and by its numbers alone: it is kept by those, and a further call of
# the same ones packs its pointers.

_plans = {}  # of these calls alone: a server whose every prompt has a new length fills it


def _meta(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


def _plan(key, make, *args):
    got = _plans.get(key)
    if got is None:
        got = make(*args)
        if len(_plans) >= 4096:  # a caller that never repeats a size
            _plans.clear()
        _plans[key] = got
    return got


def _number(name, x):
    if not isinstance(x, numbers.Real) or isinstance(x, bool):
        raise R9vxError(-103, f"{name}={x!r} is no number")
    return _bits(x)


def _strides(name, t, dims):
    """A tensor's strides but for the last axis, which must be dense; 0 along an axis of one."""
    shape, stride = t.shape, t.stride()
    if len(shape) != dims:
        raise R9vxError(-103, f"{name} has {len(shape)} dimensions: it must have {dims}")
    if stride[-1] != 1 and shape[-1] > 1:
        raise R9vxError(-103, f"the last axis of {name} must be dense")
    return [s if n > 1 else 0 for n, s in zip(shape[:-1], stride)]


def _like(name, t, dtypes, shape, device):
    """Checks a strided operand as ffi._fp8_operands checks dense ones."""
    if t.dtype not in dtypes:
        raise R9vxError(-103, f"{name} is {t.dtype}: it must be one of {', '.join(map(str, dtypes))}")
    if t.shape != shape:
        raise R9vxError(-103, f"{name} has shape {tuple(t.shape)}: it must be {tuple(shape)}")
    if t.get_device() != device:
        ffi._need_gpu(t)  # raises for an operand in host memory
        raise R9vxError(-104, f"{name} is on cuda:{t.get_device()}, other operands on cuda:{device}")


def _cache(k_cache, v_cache, dtypes, device):
    """(page_size, kv_heads, head_dim, pages, k's strides, v's strides)."""
    ks = _strides("k_cache", k_cache, 4)
    _like("k_cache", k_cache, dtypes, k_cache.shape, device)
    _like("v_cache", v_cache, (k_cache.dtype,), k_cache.shape, device)
    pages, page, kv, dim = k_cache.shape
    return page, kv, dim, ffi._u32("pages", pages), ks, _strides("v_cache", v_cache, 4)


def _rope_plan(q, k, v, positions, freqs, k_cache, v_cache, slots, interleaved, amplitude, q_out, status):
    """(static, the rest of the arguments, device, shape and type of q_out)."""
    T = _types()
    t, heads, dim = ffi._rows("q" if k is not None else "x", q, 3)
    device = ffi._fp8_operands(("positions", positions, T.i32, (t,)), ("freqs", freqs, T.f64, freqs.shape[:1]), ("slots", slots, T.i64, (t,)),
                               ("status", status, T.i32, (1,)))
    name, out_name = ("x", "out") if k is None else ("q", "q_out")
    _like(name, q, T.rows, (t, heads, dim), device)
    page, kv, pages, out, strides = 0, 0, 0, q.dtype, [0] * 10
    if k is not None:
        page, kv, cdim, pages, ks, vs = _cache(k_cache, v_cache, T.halves, device)
        if cdim != dim:
            raise R9vxError(-103, f"the cache's head_dim is {cdim}, q's {dim}")
        _like("k", k, (q.dtype,), (t, kv, dim), device)
        _like("v", v, (q.dtype,), (t, kv, dim), device)
        strides, out = _strides("k", k, 3) + _strides("v", v, 3) + ks + vs, k_cache.dtype
    if q_out is not None:
        _like(out_name, q_out, (out,), (t, heads, dim), device)
    to = _strides(out_name, q_out, 3) if q_out is not None else [heads * dim if t > 1 else 0, dim if heads > 1 else 0]
    st = ffi.RopeKvStatic(*(ffi._u32(n, x) for n, x in (
        ("heads", heads), ("kv_heads", kv), ("head_dim", dim), ("rot", 2 * freqs.shape[0]), ("interleaved", int(interleaved)), ("page_size", page),
        ("in_dtype", T.code[q.dtype]), ("out_dtype", T.code[out]), ("amplitude", _number("amplitude", amplitude)))))
    rest = _ROPE_REST.pack(*_strides(name, q, 3), *strides[:4], *to, *strides[4:], pages, ffi._u32("t", t))
    return st, ffi.ctypes.byref(st), rest, device, (t, heads, dim), out


def rope_kv(q, k, v, positions, freqs, k_cache, v_cache, slots, interleaved=False, amplitude=1.0, q_out=None, status=None,
            stream=None):
    """Turns q [t, heads, head_dim] and k [t, kv_heads, head_dim] by positions
    (int32 [t]) times freqs (f64 [rot / 2], see rope_freqs) and puts k and v
    [t, kv_heads, head_dim] into the cache at slots [t]; -1: nowhere.  Pairs are
    columns i and i + rot / 2, or with interleaved 2i and 2i + 1; columns from rot
    on are copied.  q, k and v are f32 or of the cache's type, with strides
    of their own (views of one projection's rows).  Returns q_out, of the cache's
    type; q_out may be q where q has that type."""
    key = ("rope_kv", q.shape, q.stride(), q.dtype, q.get_device(), _meta(k), _meta(v), _meta(positions), _meta(freqs), _meta(k_cache),
           _meta(v_cache), _meta(slots), interleaved, amplitude, _meta(q_out), _meta(status), ffi._current())
    _, st, rest, device, shape, out = _plan(key, _rope_plan, q, k, v, positions, freqs, k_cache, v_cache, slots, interleaved, amplitude, q_out, status)
    if q_out is None:
        q_out = ffi._new(q, shape, out, stream)
    args = _ROPE_POINTERS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), positions.data_ptr(), freqs.data_ptr(), q_out.data_ptr(),
                               k_cache.data_ptr(), v_cache.data_ptr(), slots.data_ptr(), 0 if status is None else status.data_ptr())
    ffi._check(ffi.load().r9vx_rope_kv_launch(st, args + rest, ffi._raw_stream(device, stream)))
    return q_out


def rope(x, positions, freqs, interleaved=False, amplitude=1.0, out=None, stream=None):
    """rope_kv's turn alone: x [t, heads, head_dim] of f32, bf16 or f16; out has x's type and may be x."""
    key = ("rope", _meta(x), _meta(positions), _meta(freqs), interleaved, amplitude, _meta(out), ffi._current())
    _, st, rest, device, shape, dtype = _plan(key, _rope_plan, x, None, None, positions, freqs, None, None, None, interleaved, amplitude, out, None)
    if out is None:
        out = ffi._new(x, shape, dtype, stream)
    args = _ROPE_POINTERS.pack(x.data_ptr(), 0, 0, positions.data_ptr(), freqs.data_ptr(), out.data_ptr(), 0, 0, 0, 0)
    ffi._check(ffi.load().r9vx_rope_kv_launch(st, args + rest, ffi._raw_stream(device, stream)))
    return out


def decode_workspace_bytes(st: ffi.AttnStatic) -> int:
    return int(ffi.load().r9vx_attn_decode_workspace_bytes(ffi.ctypes.byref(st)))


def prefill_workspace_bytes(st: ffi.AttnStatic) -> int:
    return int(ffi.load().r9vx_attn_prefill_workspace_bytes(ffi.ctypes.byref(st)))


def _attn_plan(q, k_cache, v_cache, table, lengths, offsets, scale, softcap, slopes, causal, window, starts, prefix, out, workspace, status,
               b_bucket, t_bucket, len_bucket):
    """(static, its workspace bytes, the rest of the arguments, device); offsets None: decode."""
    T = _types()
    F = ffi._Fp8
    shape = ffi._rows("q", q, 4 if offsets is None else 3)
    heads, dim = shape[-2:]
    b = ffi._rows("lengths", lengths, 1)[0]
    t = shape[0]  # prefill: rows; decode: sequences
    device = ffi._fp8_operands(("lengths", lengths, T.i32, (t,) if offsets is None else (b,)), ("offsets", offsets, T.i32, (b + 1,)),
                               ("starts", starts, T.i32, (t,)), ("prefix", prefix, T.i32, (b,)), ("slopes", slopes, F.f32, (heads,)),
                               ("status", status, T.i32, (1,)), ("workspace", workspace, F.bytes, workspace.shape if workspace is not None else ()))
    page, kv, cdim, pages, ks, vs = _cache(k_cache, v_cache, T.halves, device)
    _like("q", q, (k_cache.dtype,), (*shape[:-1], cdim), device)
    _like("table", table, T.i32, table.shape, device)
    columns = _strides("table", table, 2)[0]
    if table.shape[0] != b:
        raise R9vxError(-103, f"table has {table.shape[0]} rows: {b} sequences")
    room = table.shape[1] * page
    if len_bucket is None:
        len_bucket = min(room, 1 << 30)
    elif len_bucket > room:
        raise R9vxError(-103, f"len_bucket={len_bucket}: the table's {table.shape[1]} columns hold {room}")
    if out is not None:
        _like("out", out, (q.dtype,), shape, device)
        to = _strides("out", out, len(shape))
    else:
        to = [math.prod(shape[i + 1:]) if n > 1 else 0 for i, n in enumerate(shape[:-1])]
    pad = [] if offsets is None else [0]
    st = ffi.AttnStatic(*(ffi._u32(n, x) for n, x in (
        ("b_bucket", b_bucket or b), ("t_bucket", shape[1] if offsets is None else t_bucket or t), ("len_bucket", len_bucket), ("heads", heads),
        ("kv_heads", kv), ("head_dim", dim), ("page_size", page), ("dtype", T.code[q.dtype]), ("causal", int(causal)), ("window", window),
        ("scale", _number("scale", dim ** -0.5 if scale is None else scale)), ("softcap", _number("softcap", softcap)))))
    nbytes = (decode_workspace_bytes if offsets is None else prefill_workspace_bytes)(st)
    rest = _ATTN_REST.pack(*pad, *_strides("q", q, len(shape)), *pad, *to, *ks, *vs, columns, pages, ffi._u32("b", b),
                           0 if offsets is None else ffi._u32("t", t), 0)
    return st, ffi.ctypes.byref(st), nbytes, rest, device


def decode(q, k_cache, v_cache, table, lengths, scale=None, softcap=0.0, slopes=None, window=0, starts=None, out=None, workspace=None,
           status=None, stream=None, b_bucket=None, len_bucket=None):
    """Attention of each sequence's last new tokens over its pages: q
    [b, new, heads, head_dim] with new 1 to 8 (the tokens' keys and values are in
    the cache already, rope_kv before it), lengths int32 [b] counting them;
    softmax(scale q . k) v, causal, scale 1 / sqrt(head_dim) by default.  softcap:
    scores softcap * tanh(score / softcap); slopes (f32 [heads]): less slope *
    distance; window: that many last keys; starts (int32 [b]): no key before it.
    A length of 0 gives zeros.  b_bucket and len_bucket (by default b and what the
    table holds) pick the kernels."""
    key = ("decode", q.shape, q.stride(), q.dtype, q.get_device(), _meta(k_cache), _meta(v_cache), _meta(table), _meta(lengths), scale, softcap,
           _meta(slopes), window, _meta(starts), _meta(out), _meta(workspace), _meta(status), b_bucket, len_bucket, ffi._current())
    _, st, nbytes, rest, device = _plan(key, _attn_plan, q, k_cache, v_cache, table, lengths, None, scale, softcap, slopes, True, window, starts,
                                        None, out, workspace, status, b_bucket, None, len_bucket)
    if workspace is not None or nbytes:
        workspace = ffi._workspace(workspace, nbytes, q, stream)
    if out is None:
        out = ffi._new(q, q.shape, q.dtype, stream)
    args = _ATTN_POINTERS.pack(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), table.data_ptr(), lengths.data_ptr(), 0,
                               0 if starts is None else starts.data_ptr(), 0, 0 if slopes is None else slopes.data_ptr(), out.data_ptr(),
                               0 if workspace is None else workspace.data_ptr(), 0 if status is None else status.data_ptr())
    ffi._check(ffi.load().r9vx_attn_decode_launch(st, args + rest, ffi._raw_stream(device, stream)))
    return out


def prefill(q, k_cache, v_cache, table, lengths, offsets, scale=None, softcap=0.0, slopes=None, causal=True, window=0, starts=None,
            prefix=None, out=None, workspace=None, status=None, stream=None, b_bucket=None, t_bucket=None, len_bucket=None):
    """Attention of prompts or prompt chunks, packed in q [t, heads, head_dim]:
    sequence i's rows are offsets[i] .. offsets[i + 1] - 1 (int32 [b + 1]) and the
    last of its lengths[i] tokens, all of which the cache holds.  As decode, and
    causal=False: every key of the sequence; starts (int32 [t]): a row sees no key
    before its own (the document it is in); prefix (int32 [b]): keys before it are
    seen by all of the sequence's rows.  Rows outside every sequence are left as
    they were.  b_bucket, t_bucket and len_bucket pick the kernels."""
    if offsets is None:
        raise R9vxError(-103, "offsets are required")
    key = ("prefill", q.shape, q.stride(), q.dtype, q.get_device(), _meta(k_cache), _meta(v_cache), _meta(table), _meta(lengths), _meta(offsets),
           scale, softcap, _meta(slopes), causal, window, _meta(starts), _meta(prefix), _meta(out), _meta(workspace), _meta(status), b_bucket,
           t_bucket, len_bucket, ffi._current())
    _, st, nbytes, rest, device = _plan(key, _attn_plan, q, k_cache, v_cache, table, lengths, offsets, scale, softcap, slopes, causal, window, starts,
                                        prefix, out, workspace, status, b_bucket, t_bucket, len_bucket)
    if workspace is not None or nbytes:
        workspace = ffi._workspace(workspace, nbytes, q, stream)
    if out is None:
        out = ffi._new(q, q.shape, q.dtype, stream)
    args = _ATTN_POINTERS.pack(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), table.data_ptr(), lengths.data_ptr(), offsets.data_ptr(),
                               0 if starts is None else starts.data_ptr(), 0 if prefix is None else prefix.data_ptr(),
                               0 if slopes is None else slopes.data_ptr(), out.data_ptr(), 0 if workspace is None else workspace.data_ptr(),
                               0 if status is None else status.data_ptr())
    ffi._check(ffi.load().r9vx_attn_prefill_launch(st, args + rest, ffi._raw_stream(device, stream)))
    return out
