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


def _type_of(name: str, t) -> int:
    try:
        return _TYPES[t.dtype]
    except (KeyError, AttributeError):
        raise TypeError(f"{name}: expected a float32, float16 or bfloat16 CUDA tensor, got "
                        f"{getattr(t, 'dtype', type(t).__name__)}") from None


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _rows(name: str, t, dtype, heads: Optional[int], dim: int, device):
    """Shape and strides of a [tokens, heads, dim] operand with unit stride along dim."""
    if t.dtype != dtype or t.device != device:
        raise TypeError(f"{name}: expected {dtype} on {device}, got {t.dtype} on {t.device}")
    _need(t.dim() == 3 and t.shape[2] == dim and (heads is None or t.shape[1] == heads),
          f"{name}: shape {tuple(t.shape)}, expected [tokens, {'heads' if heads is None else heads}, {dim}]")
    st, sh, sd = t.stride()
    _need(sd == 1, f"{name}: the last dimension must have unit stride")
    return st, sh


def _int32(name: str, t, device, *shape):
    """An int32 index tensor of this shape, unit stride in its last dimension."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != device:
        raise TypeError(f"{name}: expected an int32 tensor on {device}")
    _need(t.shape == shape and (t.numel() <= 1 or t.stride(-1) == 1),
          f"{name}: shape {tuple(t.shape)}, strides {t.stride()}, expected {list(shape)} with unit stride")
    return t.data_ptr()


def _cache(cache, device):
    k, v, ks, vs = cache
    shape = k.shape
    if k.dtype not in _CODES or v.dtype not in _CODES or ks.dtype != torch.float32 or vs.dtype != torch.float32:
        raise TypeError("cache: expected float8_e4m3fn (or uint8) codes and float32 scales")
    if k.device != device or v.device != device or ks.device != device or vs.device != device:
        raise TypeError(f"cache: every tensor must be on {device}")
    _need(len(shape) == 4 and v.shape == shape, "cache: codes must be [pages, kv_heads, page_size, head_dim], k and v alike")
    _need(ks.shape == shape[:2] and vs.shape == shape[:2], "cache: scales must be [pages, kv_heads]")
    _need(k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous(),
          "cache: tensors must be contiguous")
    return shape, (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr())


def _table(table, device):
    if not isinstance(table, torch.Tensor) or table.dtype != torch.int32 or table.device != device:
        raise TypeError(f"table: expected an int32 tensor on {device}")
    _need(table.dim() == 2 and (table.shape[1] <= 1 or table.stride(1) == 1), "table: expected [batch, width], rows contiguous")
    return table.shape[0], table.shape[1], table.stride(0)


def _call(fname: str, args, device, what: str) -> None:
    index = device.index
    if torch.cuda.current_device() == index:
        rc = getattr(lib(), fname)(C.byref(args), torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = getattr(lib(), fname)(C.byref(args), torch._C._cuda_getCurrentRawStream(index))
    if rc:
        check(rc, what)


def _cuda_device(name: str, t):
    if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
        raise TypeError(f"{name}: expected a CUDA tensor")
    return t.device


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
    device = _cuda_device("k", k)
    kind = _type_of("k", k)
    shape, (kc, vc, ks, vs) = _cache(cache, device)
    pages, heads, page, dim = shape
    skt, skh = _rows("k", k, k.dtype, heads, dim, device)
    svt, svh = _rows("v", v, k.dtype, heads, dim, device)
    tokens = k.shape[0]
    _need(v.shape[0] == tokens, f"k has {tokens} tokens, v {v.shape[0]}")
    batch, width, stride = _table(table, device)
    starts_at = _int32("starts", starts, device, batch)
    cu_at = 0 if cu is None else _int32("cu", cu, device, batch + 1)
    _need(cu is not None or (tokens % batch == 0 if batch else tokens == 0),
          f"{tokens} tokens are not the same number for each of {batch} sequences: pass cu")
    rot = rope_len = cos_at = sin_at = 0
    _need((cos is None) == (sin is None), "pass both cos and sin, or neither")
    if cos is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            if t.dtype != torch.float32 or t.device != device:
                raise TypeError(f"{name}: expected float32 on {device}")
            _need(t.dim() == 2 and t.is_contiguous() and 2 * t.shape[1] <= dim and t.shape == cos.shape,
                  f"{name}: expected a contiguous [positions, at most {dim // 2}]")
        rope_len, rot = cos.shape[0], 2 * cos.shape[1]
        cos_at, sin_at = cos.data_ptr(), sin.data_ptr()
    q_heads = q_at = out_at = sqt = sqh = 0
    out = None
    if q is not None:
        sqt, sqh = _rows("q", q, k.dtype, None, dim, device)
        _need(q.shape[0] == tokens, f"k has {tokens} tokens, q {q.shape[0]}")
        q_heads = q.shape[1]
        out = torch.empty((tokens, q_heads, dim), dtype=q.dtype, device=device)
        q_at, out_at = q.data_ptr(), out.data_ptr()
    lengths = torch.empty(batch, dtype=torch.int32, device=device)
    a = _lib.KvAppendArgs(k.data_ptr(), v.data_ptr(), q_at, out_at, kc, vc, ks, vs, table.data_ptr(), starts_at, cu_at,
                          lengths.data_ptr(), cos_at, sin_at, batch, tokens, heads, q_heads, dim, page, pages, width,
                          stride, skt, skh, svt, svh, sqt, sqh, q_heads * dim, dim, rot, rope_len, kind,
                          1 if interleaved else 0, 0, 0)
    _call("piton_b200_kv_append", a, device, "kv_append")
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
    device = _cuda_device("q", q)
    kind = _type_of("q", q)
    shape, (kc, vc, ks, vs) = _cache(cache, device)
    pages, kv_heads, page, dim = shape
    sqt, sqh = _rows("q", q, q.dtype, None, dim, device)
    tokens, heads = q.shape[0], q.shape[1]
    batch, width, stride = _table(table, device)
    lengths_at = _int32("lengths", lengths, device, batch)
    cu_at = 0 if cu is None else _int32("cu", cu, device, batch + 1)
    _need(cu is not None or (tokens % batch == 0 if batch else tokens == 0),
          f"{tokens} tokens are not the same number for each of {batch} sequences: pass cu")
    _need(window >= 0 and max_length >= 0 and max_new >= 0, "window, max_length and max_new must not be negative")
    out = torch.empty((tokens, heads, dim), dtype=q.dtype, device=device)
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=device) if return_lse else None
    a = _lib.KvAttentionArgs(q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0, kc, vc, ks, vs,
                             table.data_ptr(), lengths_at, cu_at, 1.0 / math.sqrt(dim) if scale is None else scale,
                             batch, tokens, heads, kv_heads, dim, page, pages, width, stride, sqt, sqh, heads * dim, dim,
                             window, max_length, max_new, 0, 0, kind, 0)
    need = lib().piton_b200_kv_attention_workspace_size(C.byref(a))
    if need:
        scratch = torch.empty(need, dtype=torch.uint8, device=device)   # of this call's stream, so calls never share it
        a.workspace, a.workspace_bytes = scratch.data_ptr(), need
    _call("piton_b200_kv_attention", a, device, "kv_attention")
    return (out, lse) if return_lse else out


def matvec_w4(x, codes, scales, *, group: int = 128, zeros=None, bias=None):
    """``x`` [rows, inner] (or [inner]) times the transpose of a 4-bit weight matrix [outer, inner].

    ``codes`` uint8 [outer, ceil(inner / 2)]: two codes per byte along the inner dimension, the even one in
    the low half.  ``scales`` [outer, ceil(inner / group)] (float32, float16 or bfloat16) and ``zeros`` (uint8 of
    the same shape, the low four bits count; zero point 8 without) per group of 32, 64 or 128: W = scale * (code - zero).  ``bias``
    [outer] of x's type.  Rows of every operand may be strided.  Accumulates in 32 bits, returns x's type.
    Meant for few rows: the weights are read again for every 16."""
    device = _cuda_device("x", x)
    kind = _type_of("x", x)
    flat = x.dim() == 1
    _need(x.dim() in (1, 2), f"x: shape {tuple(x.shape)}, expected [rows, inner] or [inner]")
    rows, inner = (1, x.shape[0]) if flat else x.shape
    _need(x.shape[-1] <= 1 or x.stride(-1) == 1, "x: the last dimension must have unit stride")
    if codes.dtype != torch.uint8 or codes.device != device:
        raise TypeError(f"codes: expected uint8 on {device}, got {codes.dtype} on {codes.device}")
    _need(codes.dim() == 2 and codes.shape[1] == (inner + 1) // 2 and (codes.shape[1] <= 1 or codes.stride(1) == 1),
          f"codes: shape {tuple(codes.shape)}, expected [outer, {(inner + 1) // 2}] with unit stride")
    outer = codes.shape[0]
    if group not in (32, 64, 128):
        raise NotImplementedError(f"group {group}: 32, 64 or 128")
    groups = -(-inner // group)
    scale_kind = _type_of("scales", scales)
    if scales.device != device:
        raise TypeError(f"scales: expected a tensor on {device}")
    _need(scales.shape == (outer, groups) and (groups <= 1 or scales.stride(1) == 1),
          f"scales: shape {tuple(scales.shape)}, expected {[outer, groups]} with unit stride")
    zeros_at = bias_at = zero_stride = 0
    if zeros is not None:
        if zeros.dtype != torch.uint8 or zeros.device != device:
            raise TypeError(f"zeros: expected uint8 on {device}")
        _need(zeros.shape == (outer, groups) and (groups <= 1 or zeros.stride(1) == 1),
              f"zeros: shape {tuple(zeros.shape)}, expected {[outer, groups]} with unit stride")
        zeros_at, zero_stride = zeros.data_ptr(), zeros.stride(0)
    if bias is not None:
        if bias.dtype != x.dtype or bias.device != device:
            raise TypeError(f"bias: expected {x.dtype} on {device}")
        _need(bias.shape == (outer,) and (outer <= 1 or bias.stride(0) == 1), f"bias: expected [{outer}] with unit stride")
        bias_at = bias.data_ptr()
    y = torch.empty(outer if flat else (rows, outer), dtype=x.dtype, device=device)
    a = _lib.MatvecW4Args(x.data_ptr(), codes.data_ptr(), scales.data_ptr(), zeros_at, bias_at, y.data_ptr(), rows, inner,
                          outer, 0 if flat else x.stride(0), codes.stride(0), scales.stride(0), zero_stride, outer, group,
                          kind, scale_kind, 0)
    _call("piton_b200_matvec_w4", a, device, "matvec_w4")
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
