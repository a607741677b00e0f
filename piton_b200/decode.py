"""Serving operators: a paged 8-bit key/value cache, attention over it, and 4-bit weights.

The reference runs dense attention (examples/attention.py:75-113) and dense layers
(examples/nn_kernels.py:23-74) on whole fp32 operands; a decoder that serves many or long
sequences keeps its keys and values in pages and its weights in few bits.  Three operators make
one step of such a decoder, each one or two launches of libpiton_b200 on the current torch stream,
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
reports 16 (page) or 17 (position or offset).

There is no backward: inputs that require grad are refused unless gradients are off (``torch.no_grad()``).
"""

from __future__ import annotations

import ctypes as C
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


_ENTRIES = ("piton_b200_kv_append", "piton_b200_kv_attention", "piton_b200_kv_attention_workspace_size",
            "piton_b200_matvec_w4_workspace_size", "piton_b200_matvec_w4")
_bound = None


def _calls():
    """The extension module that checks and marshals the calls, bound to the loaded library."""
    global _bound
    if _bound is None:
        try:
            from . import _decode_calls
        except ImportError as e:
            raise ImportError(f"piton_b200/_decode_calls.so: {e}; build it with `python -m piton_b200.build`") from e
        handle = lib()
        _decode_calls.bind(*(C.cast(getattr(handle, name), C.c_void_p).value for name in _ENTRIES), torch.OutOfMemoryError)
        _bound = _decode_calls
    return _bound


def _failed(what: str, result, refuse, *args):
    """Raises for a call that gave a status code, or None for an argument that `refuse` finds."""
    if result is None:
        refuse(*args)
        raise ValueError(f"{what}: unsupported arguments")
    check(result, what)


# What is wrong with a call that was not made: the arguments one by one.

def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _refuse_gradient(*tensors) -> None:
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        raise RuntimeError("the serving operators have no backward and an input requires grad: call them under torch.no_grad(), or "
                           "detach it")


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
    if not isinstance(cache, tuple) or len(cache) != 4:
        raise TypeError("cache: expected a PagedKV or a tuple (k, v, k_scale, v_scale)")
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


def _refuse_table(table, index: int) -> int:
    _refuse_tensor("table", table, (torch.int32,), index)
    _need(table.dim() == 2 and (table.shape[1] <= 1 or table.stride(1) == 1), "table: expected [batch, width], rows contiguous")
    return table.shape[0]


def _refuse_append(k, v, cache, table, starts, cu, cos, sin, interleaved, q) -> None:
    _type_of("k", k)
    _refuse_gradient(k, v, q, cos, sin, *(cache if isinstance(cache, tuple) else ()))
    index, dtype = k.get_device(), k.dtype
    _refuse_cache(cache, index)
    heads, dim = cache[0].shape[1], cache[0].shape[3]
    _refuse_rows("k", k, dtype, heads, dim, index)
    _refuse_rows("v", v, dtype, heads, dim, index)
    tokens = k.shape[0]
    _need(v.shape[0] == tokens, f"k has {tokens} tokens, v {v.shape[0]}")
    batch = _refuse_table(table, index)
    _refuse_indices(table, (("starts", starts, batch),), cu, batch, tokens, index)
    if cos is not None or sin is not None:
        _need(cos is not None and sin is not None, "pass both cos and sin, or neither")
        _refuse_tensor("cos", cos, (torch.float32,), index)
        _refuse_tensor("sin", sin, (torch.float32,), index)
        _need(cos.dim() == 2 and cos.shape == sin.shape and 2 * cos.shape[1] <= dim and cos.is_contiguous() and
              sin.is_contiguous(), f"cos, sin: expected two contiguous [positions, at most {dim // 2}], got {tuple(cos.shape)} and "
              f"{tuple(sin.shape)}")
    if q is not None:
        _refuse_rows("q", q, dtype, None, dim, index)
        _need(q.shape[0] == tokens, f"k has {tokens} tokens, q {q.shape[0]}")


def _refuse_attention(q, cache, table, lengths, cu, scale, window, max_length, max_new, return_lse) -> None:
    _type_of("q", q)
    _refuse_gradient(q, *(cache if isinstance(cache, tuple) else ()))
    index = q.get_device()
    _refuse_cache(cache, index)
    _refuse_rows("q", q, q.dtype, None, cache[0].shape[3], index)
    batch = _refuse_table(table, index)
    _refuse_indices(table, (("lengths", lengths, batch),), cu, batch, q.shape[0], index)
    _need(window >= 0 and max_length >= 0 and max_new >= 0, "window, max_length and max_new must not be negative")


def _refuse_matvec(x, codes, scales, group, zeros, bias) -> None:
    _type_of("x", x)
    _refuse_gradient(x, scales, bias)
    index = x.get_device()
    if group not in (32, 64, 128):
        raise NotImplementedError(f"group {group}: 32, 64 or 128")
    _need(x.dim() in (1, 2), f"x: shape {tuple(x.shape)}, expected [rows, inner] or [inner]")
    _refuse_tensor("codes", codes, (torch.uint8,), index)
    _refuse_tensor("scales", scales, tuple(_TYPES), index)
    if zeros is not None:
        _refuse_tensor("zeros", zeros, (torch.uint8,), index)
    if bias is not None:
        _refuse_tensor("bias", bias, (x.dtype,), index)
    outer, inner = codes.shape[0], x.shape[-1]
    raise ValueError(f"x {tuple(x.shape)}, codes {tuple(codes.shape)}, scales {tuple(scales.shape)}, zeros "
                     f"{None if zeros is None else tuple(zeros.shape)}, bias {None if bias is None else tuple(bias.shape)}: "
                     f"expected codes [{outer}, {(inner + 1) // 2}], scales and zeros [{outer}, {-(-inner // group)}], bias "
                     f"[{outer}], each with unit stride in its last dimension")


def kv_append(k, v, cache, table, starts, *, cu=None, cos=None, sin=None, interleaved: bool = False, q=None):
    """Append ``k``, ``v`` [tokens, kv_heads, head_dim] to ``cache``, rotating keys by position.

    Sequence b already holds ``starts[b]`` tokens; its new ones are rows ``cu[b]:cu[b + 1]`` (``tokens /
    batch`` each without ``cu``) and take the positions after them.  ``cos`` and ``sin`` (float32
    [positions, r / 2]) rotate the first r elements of every key in pairs (i, i + r / 2), or (2 i, 2 i + 1)
    with ``interleaved``; without them nothing is rotated.  ``q`` [tokens, heads, head_dim] is rotated the
    same way.  Any token and head strides, unit stride along head_dim.  Returns ``(q, lengths)``: the
    rotated queries in a new contiguous tensor of q's type (None without q) and int32 ``starts`` plus the
    new tokens.  A token past the rows of ``cos`` and ``sin`` is stored as zeros and its rotated query is 0
    (device status 17); so is the rotated query of a token that no sequence's range names.

    A block (page and head) has one scale: the least power of two that holds its values within e4m3's 448;
    when new values make it grow, the block's older codes are requantised.  Non-finite values are stored
    as NaN and do not move the scale."""
    args = (k, v, cache, table, starts, cu, cos, sin, interleaved, q)
    result = (_bound or _calls()).kv_append(*args)
    if result.__class__ is not tuple:
        _failed("kv_append", result, _refuse_append, *args)
    return result


def kv_attention(q, cache, table, lengths, *, cu=None, scale: Optional[float] = None, window: int = 0,
                 max_length: int = 0, max_new: int = 0, return_lse: bool = False):
    """Attention of ``q`` [tokens, heads, head_dim] over ``cache``; returns a tensor of q's shape and type.

    Sequence b holds ``lengths[b]`` tokens (appended before), the last of them its query tokens, rows
    ``cu[b]:cu[b + 1]`` of q (``tokens / batch`` each without ``cu``).  The query at position p sees the keys up to
    p, with ``window`` only the last ``window`` of them.  heads is a multiple of the cache's kv_heads; ``scale``
    is 1 / sqrt(head_dim) by default.  Rows that see no key are 0, and so are rows of tokens that no sequence's
    range names.  ``max_length`` (an upper bound of the lengths known to the host) and ``max_new`` (of the query
    tokens a sequence, with ``cu``) size the launch and change no result; by default the table's width and the
    number of tokens bound them.  Scores, sums and the softmax are held in 32 bits; inside the products float32
    queries and the softmax's weights have 22 bits, the weights of bfloat16 rows 11.  With ``return_lse`` also the float32
    [tokens, heads] logarithms of the rows' sums of exponentials (-inf for rows that see no key)."""
    args = (q, cache, table, lengths, cu, scale, window, max_length, max_new, return_lse)
    result = (_bound or _calls()).kv_attention(*args)
    if result is None or result.__class__ is int:
        _failed("kv_attention", result, _refuse_attention, *args)
    return result


def matvec_w4(x, codes, scales, *, group: int = 128, zeros=None, bias=None):
    """``x`` [rows, inner] (or [inner]) times the transpose of a 4-bit weight matrix [outer, inner].

    ``codes`` uint8 [outer, ceil(inner / 2)]: two codes per byte along the inner dimension, the even one in
    the low half.  ``scales`` [outer, ceil(inner / group)] (float32, float16 or bfloat16) and ``zeros`` (uint8 of
    the same shape, any value; zero point 8 without) per group of 32, 64 or 128: W = scale * (code - zero).  ``bias``
    [outer] of x's type.  Rows of every operand may be strided.  Accumulates in 32 bits, returns x's type.
    Meant for few rows: the weights are read again for every 16.

    Codes less their zero points and x enter the products as they are (fp32 as three parts that add up to it, down to 2^-133), so only the 32-bit
    sums are rounded.  Infinities and NaN in x and in the scales reach the outputs that the formula says, no other rows."""
    result = (_bound or _calls()).matvec_w4(x, codes, scales, group, zeros, bias)
    if result is None or result.__class__ is int:
        _failed("matvec_w4", result, _refuse_matvec, x, codes, scales, group, zeros, bias)
    return result


@torch.no_grad()
def quantize_w4(weight, group: int = 128, zeros: bool = True, dtype=None):
    """Codes, scales and zero points (None if not ``zeros``) of a weight matrix [outer, inner], for
    :func:`matvec_w4`: each group of ``group`` elements spans its own range in 16 steps.  Plain torch, done
    once when weights are loaded; scales are of ``dtype`` (the weight's by default).  Rows of codes start on
    16 bytes, which :func:`matvec_w4` reads fastest."""
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
    bytes_ = (inner + 1) // 2
    packed = torch.zeros((outer, bytes_ + -bytes_ % 16), dtype=torch.uint8, device=weight.device)
    packed[:, :bytes_] = (codes[:, 0::2] | codes[:, 1::2] << 4)[:, :bytes_]
    return packed[:, :bytes_], scales, zero.to(torch.uint8) if zeros else None
