"""Plain implementations the decode operators are checked against, on the CPU.

Attention and the 4-bit product are computed in float64 from the operators' definitions; the
append, whose outputs are 8-bit codes, follows the definition step by step in float32 (every
product and sum rounded by itself), so codes and scales have to be equal.
"""

import math

import torch

E4M3 = torch.float8_e4m3fn


def rotate(x, cos, sin, interleaved):
    """x [n, heads, dim] float32 or float64, cos / sin [n, r / 2]."""
    r = 2 * cos.shape[1]
    y = x.clone()
    first = range(0, r, 2) if interleaved else range(r // 2)
    for i, a in enumerate(first):
        b = a + 1 if interleaved else a + r // 2
        c, s = cos[:, i, None], sin[:, i, None]
        y[:, :, a] = x[:, :, a] * c - x[:, :, b] * s
        y[:, :, b] = x[:, :, b] * c + x[:, :, a] * s
    return y


def scale_of(a: float) -> float:
    """The least power of two s >= 2^-120 (and <= 2^120) with a <= 448 s."""
    e = -120
    while e < 120 and a > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def append(k, v, cache, table, starts, cu, cos, sin, interleaved, q):
    """Updates the CPU copies in `cache` (uint8 codes) in place; returns (q, lengths)."""
    kc, vc, ks, vs = cache
    page = kc.shape[2]
    lengths = []
    q_out = None if q is None else torch.empty(q.shape, dtype=q.dtype)
    for b, start in enumerate(starts.tolist()):
        t0, t1 = int(cu[b]), int(cu[b + 1])
        n = t1 - t0
        lengths.append(start + n)
        x = k[t0:t1].float()
        if cos is not None:
            c, s = cos[start:start + n], sin[start:start + n]
            x = rotate(x, c, s, interleaved)
            if q is not None:
                q_out[t0:t1] = rotate(q[t0:t1].float(), c, s, interleaved).to(q.dtype)
        elif q is not None:
            q_out[t0:t1] = q[t0:t1]
        for new, codes, scales in ((x, kc, ks), (v[t0:t1].float(), vc, vs)):
            done = 0
            while done < n:
                place, slot = divmod(start + done, page)
                count = min(n - done, page - slot)
                at = int(table[b, place])
                for h in range(codes.shape[1]):
                    block = new[done:done + count, h]
                    a = torch.where(block.isfinite(), block.abs(), 0.0).max().item()
                    s = scale_of(a)
                    if slot:
                        before = scales[at, h].item()
                        if s > before:
                            old = codes[at, h, :slot].view(E4M3).float() * (before / s)
                            codes[at, h, :slot] = old.to(E4M3).view(torch.uint8)
                        s = max(s, before)
                    y = torch.where(block.isfinite(), block * (1.0 / s), math.nan)
                    codes[at, h, slot:slot + count] = y.to(E4M3).view(torch.uint8)
                    scales[at, h] = s
                done += count
    return q_out, torch.tensor(lengths, dtype=torch.int32)


def same_codes(a, b):
    """Equal codes; any NaN equals any NaN."""
    a, b = a.view(torch.uint8).cpu(), b.view(torch.uint8).cpu()
    return bool(((a == b) | (((a & 127) == 127) & ((b & 127) == 127))).all())


def attention(q, cache, table, lengths, cu, scale=None, window=0):
    """(out, lse, spread) in float64; spread [tokens, heads] = scale * max_j sum_d |q_d k_jd|, for tolerances."""
    kc, vc, ks, vs = [t.cpu() for t in cache]
    table, lengths = table.cpu(), lengths.cpu()
    page, d = kc.shape[2], kc.shape[3]
    tokens, heads = q.shape[:2]
    group = heads // kc.shape[1]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    q = q.cpu().double()
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64)
    spread = torch.zeros((tokens, heads), dtype=torch.float64)
    for b in range(table.shape[0]):
        t0, t1 = int(cu[b]), int(cu[b + 1])
        length = int(lengths[b])
        ids = table[b, :-(-length // page)].long() if length > 0 else table[b, :0].long()
        if not len(ids):
            continue
        k = kc.view(torch.uint8)[ids].view(E4M3).double() * ks[ids].double()[..., None, None]
        v = vc.view(torch.uint8)[ids].view(E4M3).double() * vs[ids].double()[..., None, None]
        k, v = (t.transpose(1, 2).reshape(-1, kc.shape[1], d)[:length] for t in (k, v))
        for t in range(t0, t1):
            end = length - (t1 - t0) + (t - t0) + 1
            first = max(0, end - window) if window else 0
            if end <= first:
                continue
            kk, vv = (x[first:end].repeat_interleave(group, 1) for x in (k, v))
            s = torch.einsum("hd,khd->hk", q[t], kk) * scale
            spread[t] = torch.einsum("hd,khd->hk", q[t].abs(), kk.abs()).amax(-1) * abs(scale)
            lse[t] = torch.logsumexp(s, -1)
            out[t] = torch.einsum("hk,khd->hd", torch.softmax(s, -1), vv)
    return out, lse, spread


def matvec_w4(x, codes, scales, zeros, bias, group):
    """(y, magnitude) in float64; magnitude = sum |x w| + |bias|, for tolerances."""
    inner = x.shape[-1]
    codes = codes.cpu()
    w = torch.stack((codes & 15, codes >> 4), -1).flatten(1)[:, :inner].double()
    at = torch.arange(inner) // group
    z = zeros.cpu().double()[:, at] if zeros is not None else 8.0
    w = (w - z) * scales.cpu().double()[:, at]
    x = x.cpu().double()
    y, size = x @ w.T, x.abs() @ w.abs().T
    if bias is not None:
        y, size = y + bias.cpu().double(), size + bias.cpu().double().abs()
    return y, size
