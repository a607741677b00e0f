"""Serving operators: a paged 8-bit key/value cache, attention over it, and 4-bit weights.

The reference runs dense attention (examples/attention.py:75-113) and dense layers
(examples/nn_kernels.py:23-74) on whole fp32 operands; a decoder that serves many or long
sequences keeps its keys and values in pages and its weights in few bits.  Three operators make
one step of such a decoder, each one launch of libpiton_b200 on the current torch stream,
asynchronous, on CUDA tensors of float32, float16 or bfloat16:

* :func:`kv_append` rotates new keys (and queries) by their positions and stores keys and values
  into the cache;
* :func:`kv_attention` attends one or a few query tokens per sequence over the cache;
* :func:`matvec_w4` multiplies a few rows by a 4-bit weight matrix.

The cache is a :class:`PagedKV`: e4m3 codes ``[pages, kv_heads, page_size, head_dim]`` for keys and
for values, and one power-of-two scale per page and head for each.  Which pages a sequence owns,
and in which order, is the caller's ``table`` (int32 ``[batch, width]``); token p of a sequence is in
page ``table[b, p // page_size]``, slot ``p % page_size``.  A page that is appended to must belong to
one sequence.  Table entries and positions live on the device, so a bad one cannot raise here: the
kernels do not follow it (the token is neither stored nor attended) and ``piton_b200_device_status``
reports 16 (page) or 17 (position).
"""

from __future__ import annotations

import ctypes as C
import math
import struct
from typing import NamedTuple, Optional

import torch

from .runtime.cuda import _lib
from .runtime.cuda._lib import check, lib

_TYPES = {torch.float32: _lib.TYPE_F32, torch.float16: _lib.TYPE_F16, torch.bfloat16: _lib.TYPE_BF16}
_CODES = (torch.float8_e4m3fn, torch.uint8)


class PagedKV(NamedTuple):
    """The paged cache; any tuple of these four tensors will do where a cache is taken."""

    k: torch.Tensor           # float8_e4m3fn [pages, kv_heads, page_size, head_dim]
    v: torch.Tensor
    k_scale: torch.Tensor     # float32 [pages, kv_heads]
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device=None) -> "PagedKV":
        """A cache whose contents are not set (a page is set by the tokens appended to it)."""
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        shape = (pages, kv_heads, page_size, head_dim)
        codes = [torch.empty(shape, dtype=torch.float8_e4m3fn, device=device) for _ in range(2)]
        scales = [torch.empty(shape[:2], dtype=torch.float32, device=device) for _ in range(2)]
        return cls(*codes, *scales)


# A decode step makes these calls every few microseconds, so the ordinary call evaluates one condition
# over everything it needs and packs the C struct with one format; only where the condition fails are
# the arguments looked at one by one (the _refuse_* functions), to say what is wrong.

_LETTERS = {_lib.u64: "Q", _lib.i64: "q", _lib.i32: "i", _lib.u32: "I", _lib.f64: "d"}


def _packer(struct_type):
    """Packs the fields of a ctypes struct, in order, into bytes."""
    s = struct.Struct("@" + "".join(_LETTERS[t] for _, t in struct_type._fields_))
    assert s.size == C.sizeof(struct_type)
    return s.pack


_pack_append, _pack_attention, _pack_matvec = map(_packer, (_lib.KvAppendArgs, _lib.KvAttentionArgs, _lib.MatvecW4Args))
_ENTRY = {}


def _entry(name: str, restype=C.c_int, *rest):
    """The library's function taking a packed struct."""
    f = lib()[name]
    f.restype, f.argtypes = restype, [C.c_char_p, *rest]
    _ENTRY[name] = f
    return f


def _call(name: str, packed: bytes, index: int) -> None:
    f = _ENTRY.get(name) or _entry(name, C.c_int, C.c_void_p)
    if torch.cuda.current_device() == index:
        rc = f(packed, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = f(packed, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        check(rc, name[len("piton_b200_"):])


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _type_of(name: str, t) -> int:
    if not isinstance(t, torch.Tensor) or t.device.type != "cuda" or t.dtype not in _TYPES:
        raise TypeError(f"{name}: expected a float32, float16 or bfloat16 CUDA tensor, got "
                        f"{f'{t.dtype} on {t.device}' if isinstance(t, torch.Tensor) else type(t).__name__}")
    return _TYPES[t.dtype]


def _refuse_tensor(name: str, t, dtypes, index: int) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes or t.get_device() != index:
        raise TypeError(f"{name}: expected {' or '.join(map(str, dtypes))} on cuda:{index}, got "
                        f"{f'{t.dtype} on {t.device}' if isinstance(t, torch.Tensor) else type(t).__name__}")


def _refuse_rows(name: str, t, dtype, heads, dim: int, index: int) -> None:
    _refuse_tensor(name, t, (dtype,), index)
    _need(t.dim() == 3 and t.shape[2] == dim and (heads is None or t.shape[1] == heads),
          f"{name}: shape {tuple(t.shape)}, expected [tokens, {'heads' if heads is None else heads}, {dim}]")
    _need(t.stride(2) == 1, f"{name}: the last dimension must have unit stride")


def _refuse_cache(cache, index: int) -> None:
    k, v, ks, vs = cache
    for name, t, dtypes in (("k", k, _CODES), ("v", v, _CODES), ("k_scale", ks, (torch.float32,)),
                            ("v_scale", vs, (torch.float32,))):
        _refuse_tensor(f"cache {name}", t, dtypes, index)
        _need(t.is_contiguous(), f"cache {name}: must be contiguous")
    _need(k.dim() == 4 and v.shape == k.shape, "cache: codes must be [pages, kv_heads, page_size, head_dim], k and v alike")
    _need(ks.shape == k.shape[:2] and vs.shape == k.shape[:2], "cache: scales must be [pages, kv_heads]")


def _refuse_indices(table, vectors, cu, batch: int, tokens: int, index: int) -> None:
    for name, t, size in vectors + ((("cu", cu, batch + 1),) if cu is not None else ()):
        _refuse_tensor(name, t, (torch.int32,), index)
        _need(t.dim() == 1 and t.shape[0] == size and t.is_contiguous(), f"{name}: expected {size} contiguous int32, got "
              f"shape {tuple(t.shape)}, strides {t.stride()}")
    _need(cu is not None or (tokens % batch == 0 if batch else tokens == 0),
          f"{tokens} tokens are not the same number for each of {batch} sequences: pass cu")


def _table(table, index: int):
    """(batch, width, row stride) of a page table."""
    if not isinstance(table, torch.Tensor) or table.dtype != torch.int32 or table.get_device() != index:
        _refuse_tensor("table", table, (torch.int32,), index)
    if table.dim() != 2 or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError("table: expected [batch, width], rows contiguous")
    batch, width = table.shape
    return batch, width, table.stride(0)


def _same(t, dtype, index: int) -> bool:
    return t.dtype is dtype and t.get_device() == index


def kv_append(k, v, cache, table, starts, *, cu=None, cos=None, sin=None, interleaved: bool = False, q=None):
    """Append ``k``, ``v`` [tokens, kv_heads, head_dim] to ``cache``, rotating keys by position.

    Sequence b already holds ``starts[b]`` tokens; its new ones are rows ``cu[b]:cu[b + 1]`` (``tokens /
    batch`` each without ``cu``) and take the positions after them.  ``cos`` and ``sin`` (float32
    [positions, r / 2]) rotate the first r elements of every key in pairs (i, i + r / 2), or (2 i, 2 i + 1)
    with ``interleaved``; without them nothing is rotated.  ``q`` [tokens, heads, head_dim] is rotated the
    same way.  Any token and head strides, unit stride along head_dim.  Returns ``(q, lengths)``: the
    rotated queries in a new contiguous tensor of q's type (None without q) and int32 ``starts`` plus the
    new tokens.

    A block (page and head) has one scale: the least power of two that holds its values within e4m3's 448;
    when new values make it grow, the block's older codes are requantised.  Non-finite values are stored
    as NaN and do not move the scale."""
    kind = _type_of("k", k)
    index, dtype = k.get_device(), k.dtype
    kc, vc, ks, vs = cache
    shape = kc.shape
    if len(shape) != 4:
        _refuse_cache(cache, index)
    pages, heads, page, dim = shape
    batch, width, stride = _table(table, index)
    tokens = k.shape[0]
    if not (k.dim() == 3 and k.shape == v.shape and k.shape[1] == heads and k.shape[2] == dim and v.dtype is dtype and
            v.get_device() == index and k.stride(2) == 1 and v.stride(2) == 1 and
            kc.dtype in _CODES and vc.dtype in _CODES and vc.shape == shape and ks.shape == shape[:2] == vs.shape and
            _same(ks, torch.float32, index) and _same(vs, torch.float32, index) and kc.get_device() == index and
            vc.get_device() == index and kc.is_contiguous() and vc.is_contiguous() and ks.is_contiguous() and
            vs.is_contiguous() and _same(starts, torch.int32, index) and starts.shape == (batch,) and
            starts.is_contiguous() and
            ((batch and tokens % batch == 0) if cu is None else
             _same(cu, torch.int32, index) and cu.shape == (batch + 1,) and cu.is_contiguous())):
        _refuse_rows("k", k, dtype, heads, dim, index)
        _refuse_rows("v", v, dtype, heads, dim, index)
        _need(v.shape[0] == tokens, f"k has {tokens} tokens, v {v.shape[0]}")
        _refuse_cache(cache, index)
        _refuse_indices(table, (("starts", starts, batch),), cu, batch, tokens, index)
    rot = rope_len = cos_at = sin_at = 0
    if cos is not None or sin is not None:
        _need(cos is not None and sin is not None, "pass both cos and sin, or neither")
        if not (_same(cos, torch.float32, index) and _same(sin, torch.float32, index) and cos.dim() == 2 and
                cos.shape == sin.shape and 2 * cos.shape[1] <= dim and cos.is_contiguous() and sin.is_contiguous()):
            _refuse_tensor("cos", cos, (torch.float32,), index)
            _refuse_tensor("sin", sin, (torch.float32,), index)
            raise ValueError(f"cos, sin: expected two contiguous [positions, at most {dim // 2}], got {tuple(cos.shape)} and "
                             f"{tuple(sin.shape)}")
        rope_len, rot = cos.shape
        rot *= 2
        cos_at, sin_at = cos.data_ptr(), sin.data_ptr()
    q_heads = q_at = out_at = sqt = sqh = 0
    out = None
    if q is not None:
        if not (_same(q, dtype, index) and q.dim() == 3 and q.shape[2] == dim and q.shape[0] == tokens and q.stride(2) == 1):
            _refuse_rows("q", q, dtype, None, dim, index)
            raise ValueError(f"k has {tokens} tokens, q {q.shape[0]}")
        q_heads = q.shape[1]
        sqt, sqh, _ = q.stride()
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        q_at, out_at = q.data_ptr(), out.data_ptr()
    lengths = torch.empty_like(starts)
    skt, skh, _ = k.stride()
    svt, svh, _ = v.stride()
    _call("piton_b200_kv_append",
          _pack_append(k.data_ptr(), v.data_ptr(), q_at, out_at, kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(),
                       table.data_ptr(), starts.data_ptr(), 0 if cu is None else cu.data_ptr(), lengths.data_ptr(), cos_at,
                       sin_at, batch, tokens, heads, q_heads, dim, page, pages, width, stride, skt, skh, svt, svh, sqt, sqh,
                       q_heads * dim, dim, rot, rope_len, kind, 1 if interleaved else 0, 0, 0), index)
    return out, lengths


def kv_attention(q, cache, table, lengths, *, cu=None, scale: Optional[float] = None, window: int = 0,
                 max_length: int = 0, max_new: int = 0, return_lse: bool = False):
    """Attention of ``q`` [tokens, heads, head_dim] over ``cache``; returns a tensor of q's shape and type.

    Sequence b holds ``lengths[b]`` tokens (appended before), the last of them its query tokens, rows
    ``cu[b]:cu[b + 1]`` of q (``tokens / batch`` each without ``cu``).  The query at position p sees the keys up to
    p, with ``window`` only the last ``window`` of them.  heads is a multiple of the cache's kv_heads; ``scale``
    is 1 / sqrt(head_dim) by default.  Rows that see no key are 0.  ``max_length`` (an upper bound of the
    lengths known to the host) and ``max_new`` (of the query tokens a sequence, with ``cu``) size the launch;
    by default the table's width and the number of tokens bound them.  With ``return_lse`` also the float32
    [tokens, heads] logarithms of the rows' sums of exponentials (-inf for rows that see no key)."""
    kind = _type_of("q", q)
    index = q.get_device()
    kc, vc, ks, vs = cache
    shape = kc.shape
    if len(shape) != 4:
        _refuse_cache(cache, index)
    pages, kv_heads, page, dim = shape
    batch, width, stride = _table(table, index)
    if not (q.dim() == 3 and q.shape[2] == dim and q.stride(2) == 1 and
            kc.dtype in _CODES and vc.dtype in _CODES and vc.shape == shape and ks.shape == shape[:2] == vs.shape and
            _same(ks, torch.float32, index) and _same(vs, torch.float32, index) and kc.get_device() == index and
            vc.get_device() == index and kc.is_contiguous() and vc.is_contiguous() and ks.is_contiguous() and
            vs.is_contiguous() and _same(lengths, torch.int32, index) and lengths.shape == (batch,) and
            lengths.is_contiguous() and window >= 0 and max_length >= 0 and max_new >= 0 and
            ((batch and q.shape[0] % batch == 0) if cu is None else
             _same(cu, torch.int32, index) and cu.shape == (batch + 1,) and cu.is_contiguous())):
        _refuse_rows("q", q, q.dtype, None, dim, index)
        _refuse_cache(cache, index)
        _refuse_indices(table, (("lengths", lengths, batch),), cu, batch, q.shape[0], index)
        _need(window >= 0 and max_length >= 0 and max_new >= 0, "window, max_length and max_new must not be negative")
    tokens, heads, _ = q.shape
    sqt, sqh, _ = q.stride()
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=q.device) if return_lse else None
    args = (q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0, kc.data_ptr(), vc.data_ptr(), ks.data_ptr(),
            vs.data_ptr(), table.data_ptr(), lengths.data_ptr(), 0 if cu is None else cu.data_ptr(),
            dim ** -0.5 if scale is None else scale, batch, tokens, heads, kv_heads, dim, page, pages, width, stride, sqt, sqh,
            heads * dim, dim, window, max_length, max_new)
    packed = _pack_attention(*args, 0, 0, kind, 0)
    need = (_ENTRY.get("piton_b200_kv_attention_workspace_size") or
            _entry("piton_b200_kv_attention_workspace_size", C.c_size_t))(packed)
    if need:
        scratch = torch.empty(need, dtype=torch.uint8, device=q.device)   # of this call's stream, so calls never share it
        packed = _pack_attention(*args, scratch.data_ptr(), need, kind, 0)
    _call("piton_b200_kv_attention", packed, index)
    return (out, lse) if return_lse else out


def matvec_w4(x, codes, scales, *, group: int = 128, zeros=None, bias=None):
    """``x`` [rows, inner] (or [inner]) times the transpose of a 4-bit weight matrix [outer, inner].

    ``codes`` uint8 [outer, ceil(inner / 2)]: two codes per byte along the inner dimension, the even one in
    the low half.  ``scales`` [outer, ceil(inner / group)] (float32, float16 or bfloat16) and ``zeros`` (uint8 of
    the same shape, the low four bits count; zero point 8 without) per group of 32, 64 or 128: W = scale * (code - zero).  ``bias``
    [outer] of x's type.  Rows of every operand may be strided.  Accumulates in 32 bits, returns x's type.
    Meant for few rows: the weights are read again for every 16."""
    kind = _type_of("x", x)
    index, dtype = x.get_device(), x.dtype
    flat = x.dim() == 1
    if x.dim() not in (1, 2):
        raise ValueError(f"x: shape {tuple(x.shape)}, expected [rows, inner] or [inner]")
    inner = x.shape[-1]
    if group not in (32, 64, 128):
        raise NotImplementedError(f"group {group}: 32, 64 or 128")
    if not isinstance(codes, torch.Tensor) or codes.dim() != 2:
        _refuse_tensor("codes", codes, (torch.uint8,), index)
        raise ValueError(f"codes: shape {tuple(codes.shape)}, expected [outer, {(inner + 1) // 2}]")
    outer, groups = codes.shape[0], -(-inner // group)
    shape = (outer, groups)
    if not (_same(codes, torch.uint8, index) and codes.shape[1] == (inner + 1) // 2 and
            (codes.stride(1) == 1 or codes.shape[1] <= 1) and (x.stride(-1) == 1 or inner <= 1) and
            scales.dtype in _TYPES and scales.get_device() == index and scales.shape == shape and
            (groups <= 1 or scales.stride(1) == 1) and
            (zeros is None or (_same(zeros, torch.uint8, index) and zeros.shape == shape and
                               (groups <= 1 or zeros.stride(1) == 1))) and
            (bias is None or (_same(bias, dtype, index) and bias.shape == (outer,) and (outer <= 1 or bias.stride(0) == 1)))):
        _refuse_tensor("codes", codes, (torch.uint8,), index)
        _refuse_tensor("scales", scales, tuple(_TYPES), index)
        if zeros is not None:
            _refuse_tensor("zeros", zeros, (torch.uint8,), index)
        if bias is not None:
            _refuse_tensor("bias", bias, (dtype,), index)
        raise ValueError(f"x {tuple(x.shape)}, codes {tuple(codes.shape)}, scales {tuple(scales.shape)}, zeros "
                         f"{None if zeros is None else tuple(zeros.shape)}, bias {None if bias is None else tuple(bias.shape)}: "
                         f"expected codes [{outer}, {(inner + 1) // 2}], scales and zeros {list(shape)}, bias [{outer}], each with "
                         f"unit stride in its last dimension")
    rows = 1 if flat else x.shape[0]
    y = x.new_empty(outer if flat else (rows, outer))
    _call("piton_b200_matvec_w4",
          _pack_matvec(x.data_ptr(), codes.data_ptr(), scales.data_ptr(), 0 if zeros is None else zeros.data_ptr(),
                       0 if bias is None else bias.data_ptr(), y.data_ptr(), rows, inner, outer, 0 if flat else x.stride(0),
                       codes.stride(0), scales.stride(0), 0 if zeros is None else zeros.stride(0), outer, group, kind,
                       _TYPES[scales.dtype], 0), index)
    return y


def quantize_w4(weight, group: int = 128, zeros: bool = True, dtype=None):
    """Codes, scales and zero points (None if not ``zeros``) of a weight matrix [outer, inner], for
    :func:`matvec_w4`: each group of ``group`` elements spans its own range in 16 steps.  Plain torch, done
    once when weights are loaded; scales are of ``dtype`` (the weight's by default)."""
    if group not in (32, 64, 128):
        raise NotImplementedError(f"group {group}: 32, 64 or 128")
    outer, inner = weight.shape
    groups = -(-inner // group)
    w = torch.zeros((outer, groups * group), dtype=torch.float32, device=weight.device)
    w[:, :inner] = weight
    w = w.view(outer, groups, group)
    if zeros:
        lo, hi = w.amin(-1).clamp(max=0.0), w.amax(-1).clamp(min=0.0)
        step = (hi - lo) / 15.0
    else:
        step = w.abs().amax(-1) / 7.0
    scales = step.to(dtype or weight.dtype)
    step = scales.float()
    inverse = torch.where(step > 0, 1.0 / step, 0.0)
    zero = (-lo * inverse).round().clamp(0, 15) if zeros else torch.full_like(step, 8.0)
    codes = (w * inverse[..., None] + zero[..., None]).round().clamp(0, 15).to(torch.uint8).view(outer, -1)
    packed = codes[:, 0::2] | codes[:, 1::2] << 4
    return packed[:, :(inner + 1) // 2].contiguous(), scales, zero.to(torch.uint8) if zeros else None
