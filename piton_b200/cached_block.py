"""Attention of a decoder layer served from a paged 8-bit cache with 4-bit weights.

:class:`CachedBlock` runs the operators of :mod:`piton_b200.decode` as a decoder uses them: the
projection to queries, keys and values (``matvec_w4``), rotation and storage of the new tokens
(``kv_append``), attention over everything stored (``kv_attention``) and the projection back
(``matvec_w4``).  A call takes any number of new tokens per sequence, a ragged prompt or one token
each; a step of one token each may be recorded in a CUDA graph, since lengths stay on the device.

``python -m piton_b200.cached_block`` appends a batch of ragged prompts, decodes from a graph and
compares a step with the same layer in float64 without quantisation.
"""

from __future__ import annotations

import argparse

import torch

from . import decode


def rotation_tables(dim: int, positions: int, device, base: float = 10000.0):
    """cos and sin, float32 [positions, dim / 2]."""
    inverse = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    angles = torch.arange(positions, dtype=torch.float64)[:, None] * inverse
    return angles.cos().float().to(device), angles.sin().float().to(device)


class PageTable:
    """Pages of a pool handed to sequences in the order they are asked for, and given back (on the host)."""

    def __init__(self, batch: int, pages: int, page_size: int, width: int, device):
        self.page_size = page_size
        self.free = list(range(pages - 1, -1, -1))
        self.owned = [0] * batch
        self.host = torch.full((batch, width), -1, dtype=torch.int32)
        self.table = self.host.to(device)

    def reserve(self, lengths) -> None:
        """Gives sequence b the pages that ``lengths[b]`` tokens need; where one cannot have them (MemoryError) none gets any."""
        needs = list(self.owned)
        for b, length in enumerate(lengths):
            needs[b] = max(needs[b], -(-int(length) // self.page_size))
        for b, need in enumerate(needs):
            if need > self.host.shape[1]:
                raise MemoryError(f"sequence {b}: {need} pages, the table holds {self.host.shape[1]}")
        if sum(needs) - sum(self.owned) > len(self.free):
            raise MemoryError(f"{sum(needs) - sum(self.owned)} pages wanted, {len(self.free)} free")
        for b, need in enumerate(needs):
            for place in range(self.owned[b], need):
                self.host[b, place] = self.free.pop()
            self.owned[b] = need
        self.table.copy_(self.host)

    def release(self, b: int) -> None:
        """Takes sequence b's pages back; calls already made on the current stream still find its tokens in them."""
        self.free += reversed(self.host[b, :self.owned[b]].tolist())
        self.host[b, :self.owned[b]] = -1
        self.owned[b] = 0
        self.table.copy_(self.host)


class CachedBlock:
    """``x + W_o attention(W_qkv x)`` over a paged cache; weights are quantised to 4 bits once, here.

    ``qkv`` [(heads + 2 kv_heads) head_dim, width] and ``out`` [width, heads head_dim] are any float
    tensors on the GPU; activations are of ``dtype``."""

    def __init__(self, qkv, out, heads: int, kv_heads: int, positions: int, group: int = 128, dtype=torch.bfloat16):
        self.heads, self.kv_heads, self.group = heads, kv_heads, group
        self.dim = out.shape[1] // heads
        if qkv.shape != ((heads + 2 * kv_heads) * self.dim, out.shape[0]) or out.shape[1] != heads * self.dim:
            raise ValueError(f"qkv {tuple(qkv.shape)} and out {tuple(out.shape)} do not fit {heads} + 2 x {kv_heads} heads")
        self.qkv = decode.quantize_w4(qkv, group, dtype=dtype)
        self.out = decode.quantize_w4(out, group, dtype=dtype)
        self.cos, self.sin = rotation_tables(self.dim, positions, qkv.device)

    def _product(self, x, weight):
        codes, scales, zeros = weight
        return decode.matvec_w4(x, codes, scales, group=self.group, zeros=zeros)

    def __call__(self, x, cache, table, starts, cu=None, max_length: int = 0, max_new: int = 0):
        """``x`` [tokens, width]: the new tokens of sequences that hold ``starts`` tokens (rows ``cu[b]:cu[b + 1]``, or
        tokens / batch each).  Returns the layer's output and the sequences' new lengths (on the device)."""
        q, k, v = self._product(x, self.qkv).view(len(x), -1, self.dim).split((self.heads, self.kv_heads, self.kv_heads), 1)
        q, lengths = decode.kv_append(k, v, cache, table, starts, cu=cu, cos=self.cos, sin=self.sin, q=q)
        o = decode.kv_attention(q, cache, table, lengths, cu=cu, max_length=max_length, max_new=max_new)
        return x + self._product(o.view(len(x), -1), self.out), lengths


def plain(block_weights, heads, kv_heads, cos, sin, xs):
    """The layer on whole sequences ``xs`` (a list of [tokens, width]) in float64, nothing quantised."""
    qkv_w, out_w = (w.double() for w in block_weights)
    dim, r = out_w.shape[1] // heads, cos.shape[1]
    ys = []
    for x in xs:
        x = x.double()
        q, k, v = (x @ qkv_w.T).view(len(x), -1, dim).split((heads, kv_heads, kv_heads), 1)
        c, s = cos[:len(x), None].double(), sin[:len(x), None].double()
        q, k = (torch.cat((t[..., :r] * c - t[..., r:] * s, t[..., r:] * c + t[..., :r] * s), -1) for t in (q, k))
        k, v = (t.repeat_interleave(heads // kv_heads, 1) for t in (k, v))
        scores = torch.einsum("qhd,khd->hqk", q, k) / dim ** 0.5
        seen = torch.ones(scores.shape[1:], dtype=torch.bool, device=x.device).tril()
        weights = scores.masked_fill(~seen, float("-inf")).softmax(-1)
        ys.append(x + torch.einsum("hqk,khd->qhd", weights, v).flatten(1) @ out_w.T)
    return ys


def main(argv=None) -> float:
    parser = argparse.ArgumentParser(prog="python -m piton_b200.cached_block", description=__doc__.split("\n")[0])
    parser.add_argument("--batch", type=int, default=8)
    parser.add_argument("--prompt", type=int, default=500, help="longest prompt; they differ")
    parser.add_argument("--steps", type=int, default=64)
    parser.add_argument("--width", type=int, default=2048)
    parser.add_argument("--heads", type=int, default=16)
    parser.add_argument("--kv-heads", type=int, default=4)
    parser.add_argument("--head-dim", type=int, default=128)
    parser.add_argument("--page", type=int, default=64)
    args = parser.parse_args(argv)
    g = torch.Generator(device="cuda").manual_seed(0)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    inner = args.heads * args.head_dim
    weights = normal((args.heads + 2 * args.kv_heads) * args.head_dim, args.width) / args.width ** 0.5, \
        normal(args.width, inner) / inner ** 0.5
    longest = args.prompt + args.steps + 1
    block = CachedBlock(*weights, args.heads, args.kv_heads, longest)
    width = -(-longest // args.page)
    pages = PageTable(args.batch, args.batch * width, args.page, width, "cuda")
    cache = decode.PagedKV.empty(args.batch * width, args.kv_heads, args.head_dim, args.page)

    prompts = [max(1, args.prompt * (b + 1) // args.batch) for b in range(args.batch)]
    pages.reserve([n + args.steps + 1 for n in prompts])
    cu = torch.tensor([0, *prompts], dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    x = normal(sum(prompts), args.width).bfloat16()
    y, lengths = block(x, cache, pages.table, torch.zeros(args.batch, dtype=torch.int32, device="cuda"), cu, longest, max(prompts))

    # a step of one token each, checked and then recorded: it reads and writes `token` and `held`
    token, held = normal(args.batch, args.width).bfloat16(), lengths
    want = plain(weights, args.heads, args.kv_heads, block.cos, block.sin, [torch.cat((a, t[None])) for a, t in zip(x.split(prompts), token)])
    step, held_next = block(token, cache, pages.table, held, max_length=longest)
    want = torch.stack([w[-1] for w in want])
    error = float((step.double() - want).norm() / (want - token.double()).norm())
    print(f"a step after prompts of {prompts[0]} to {prompts[-1]} tokens: relative error {error:.4f} (4-bit weights, 8-bit cache)")

    held = held_next.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step, held_next = block(token, cache, pages.table, held, max_length=longest)
        token.copy_(torch.nn.functional.normalize(step.float(), dim=-1) * args.width ** 0.5)
        held.copy_(held_next)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    for _ in range(args.steps):
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    if held.tolist() != [n + 1 + args.steps for n in prompts] or not bool(torch.isfinite(token).all()):
        raise RuntimeError(f"decoding ended at lengths {held.tolist()}")
    print(f"{args.steps} steps of {args.batch} tokens: {start.elapsed_time(end) / max(args.steps, 1) * 1e3:.1f} us a step")
    return error


if __name__ == "__main__":
    main()
