"""The decode operators run together (piton_b200.cached_block) against plain implementations.

Tolerances.  The cache holds each element of the rotated keys and of the values rounded to e4m3:
half a step is 2^-4 of the element, or scale 2^-10 among the subnormals, and an older code may be
rounded to a grown scale's subnormals once more; the fp32 projection before it is off by at most
(inner / 16 + 32) 2^-22 of its sum of magnitudes.  The output is compared with float64 arithmetic on
the cache as it was stored: the projection's error moves the queries by that bound, so scores by its
sum with |k|, and so the weights; what follows is linear, so |W_o| carries the bound on.
"""

import pytest
import torch

import decode_ref as ref
from piton_b200 import cached_block, decode

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -23


def make(seed, width=192, heads=4, kv_heads=2, dim=32, group=64, page=16, positions=200, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn(((heads + 2 * kv_heads) * dim, width), generator=g, device="cuda") / width ** 0.5
    out = torch.randn((width, heads * dim), generator=g, device="cuda") / (heads * dim) ** 0.5
    return cached_block.CachedBlock(qkv, out, heads, kv_heads, positions, group, dtype), g


def run(block, cache, pages, batch, rounds, g, width):
    """Appends rounds of new tokens; returns inputs and outputs per sequence, and the final lengths."""
    starts = torch.zeros(batch, dtype=torch.int32, device="cuda")
    held = [0] * batch
    xs, ys = [[] for _ in range(batch)], [[] for _ in range(batch)]
    for news in rounds:
        held = [h + n for h, n in zip(held, news)]
        pages.reserve(held)
        cu = torch.tensor([0, *news], dtype=torch.int32).cumsum(0, dtype=torch.int32)
        x = torch.randn((sum(news), width), generator=g, device="cuda")
        y, starts = block(x, cache, pages.table, starts, cu.cuda())
        assert starts.tolist() == held
        for b, (a, c) in enumerate(zip(x.split(news), y.split(news))):
            xs[b].append(a)
            ys[b].append(c)
    return [torch.cat(x).cpu() for x in xs], [torch.cat(y).cpu() for y in ys], held


@pytest.mark.parametrize("rounds", [[[5, 40, 1], [1, 1, 1], [1, 1, 1]], [[0, 17, 33], [3, 0, 16], [1, 1, 0]], [[1, 1, 1]]])
def test_block_against_float64(cuda, rounds):
    block, g = make(len(rounds))
    width, dim, heads, kv_heads, page = 192, 32, 4, 2, 16
    pages = cached_block.PageTable(3, 30, page, 10, "cuda")
    cache = decode.PagedKV.empty(30, kv_heads, dim, page)
    xs, ys, held = run(block, cache, pages, 3, rounds, g, width)
    codes, scales, zeros = block.qkv
    group = block.group
    table = pages.host
    first = [[0] for _ in range(3)]
    for news in rounds:
        for b in range(3):
            first[b].append(first[b][-1] + news[b])
    for b, x in enumerate(xs):
        if not len(x):
            continue
        qkv, size = ref.matvec_w4(x, codes, scales, zeros, None, group)
        off = (width / 16 + 32) * 2 * EPS * size
        q, k, v = qkv.view(len(x), -1, dim).split((heads, kv_heads, kv_heads), 1)
        dq, dk, dv = off.view(len(x), -1, dim).split((heads, kv_heads, kv_heads), 1)
        cos, sin = block.cos[:len(x)].cpu().double(), block.sin[:len(x)].cpu().double()
        q, k = ref.rotate(q, cos, sin, False), ref.rotate(k, cos, sin, False)
        spin = lambda d: d + d.roll(dim // 2, -1) + 4 * EPS      # |cos|, |sin| <= 1, and the rotation's own roundings
        dq, dk = spin(dq) + 4 * EPS * q.abs().amax(), spin(dk) + 4 * EPS * k.abs().amax()
        # what is stored
        ids = table[b, :-(-held[b] // page)].long()
        stored = []                                     # the tokens of the sequence: what its last page's other slots hold is not set
        for want, d, c, s in ((k, dk, cache.k, cache.k_scale), (v, dv, cache.v, cache.v_scale)):
            got = c.view(torch.uint8).cpu()[ids].view(ref.E4M3).double() * s.cpu()[ids].double()[..., None, None]
            got = got.transpose(1, 2).reshape(-1, kv_heads, dim)[:held[b]]
            stored.append(got.abs())
            step = s.cpu()[ids].double().repeat_interleave(page, 0)[:held[b], :, None] * 2.0 ** -10
            assert ((got - want).abs() <= (want.abs() + d) * 2.0 ** -4 + d + 2 * step).all()
        # the outputs of the last round, from the cache as it is now
        for t in range(first[b][-2], held[b]):
            cu = [0, 1]
            one = table[b:b + 1]
            row = q[t:t + 1]
            out, _, spread = ref.attention(row, cache, one, torch.tensor([t + 1]), cu)
            top, kmax = stored[1].max(), stored[0].amax(0).repeat_interleave(heads // kv_heads, 0)     # [heads, dim]
            score = (dq[t] * kmax).sum(-1) / dim ** 0.5 + 2 * (dim + 8) * EPS * spread[0]
            moved = (top * (2 * score + 2.0 ** -17))[:, None].expand(heads, dim).reshape(1, -1)
            y, size = ref.matvec_w4(out.reshape(1, -1), *block.out[:2], block.out[2], None, group)
            _, carried = ref.matvec_w4(moved, *block.out[:2], block.out[2], None, group)
            tol = carried + (heads * dim / 16 + 32) * 2 * EPS * (size + carried) + 2 * EPS * (y.abs() + x[t].abs().double())
            assert ((ys[b][t].double() - (x[t].double() + y[0])).abs() <= tol[0]).all()


def test_graph_steps_equal_eager_steps(cuda):
    results = []
    for graphed in (False, True):
        block, g = make(7, dtype=torch.bfloat16)
        pages = cached_block.PageTable(2, 8, 16, 4, "cuda")
        pages.reserve([40, 50])
        cache = decode.PagedKV.empty(8, 2, 32, 16)
        x = torch.randn((2, 192), generator=g, device="cuda").bfloat16()
        held = torch.zeros(2, dtype=torch.int32, device="cuda")

        def step():
            y, lengths = block(x, cache, pages.table, held, max_length=64)
            x.copy_(y)
            held.copy_(lengths)

        step()
        if graphed:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        for _ in range(30):
            graph.replay() if graphed else step()
        torch.cuda.synchronize()
        assert held.tolist() == [31, 31]
        results.append((x, cache.k_scale[pages.host[0, :1].long()]))
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_pages_run_out(cuda):
    pages = cached_block.PageTable(2, 3, 16, 2, "cuda")
    pages.reserve([17, 16])
    with pytest.raises(MemoryError):
        pages.reserve([17, 17])


def test_weights_that_do_not_fit_the_heads(cuda):
    with pytest.raises(ValueError):
        cached_block.CachedBlock(torch.zeros((100, 64), device="cuda"), torch.zeros((64, 64), device="cuda"), 2, 1, 10)


def test_command(cuda, capsys):
    # 4-bit weights in groups of 128 of a normal distribution are off by about a tenth of its deviation
    assert cached_block.main(["--batch", "3", "--prompt", "50", "--steps", "5", "--width", "256", "--heads", "4", "--kv-heads", "2",
                              "--head-dim", "32", "--page", "16"]) < 0.3
    assert "us a step" in capsys.readouterr().out
