"""What the decode operators return for rows that no sequence names, that bounds did not count or that are refused:
never what the memory held before.  Tolerances are those of test_gpu_decode.py.
"""

import math

import pytest
import torch

import decode_ref as ref
from piton_b200 import decode
from test_gpu_decode import TYPES, bound, cpu, gen, page_table, random_cache, status, tables

pytestmark = pytest.mark.gpu


def litter():
    """Leaves blocks of NaN for the allocator to hand out again."""
    blocks = [torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda") for n in (512, 4096, 65536, 1 << 20, 1 << 22, 1 << 24) for _ in range(3)]
    torch.cuda.synchronize()
    del blocks


def check(lengths, cu, tokens, *, dtype, dim=64, page=32, kv_heads=2, group=3, **kw):
    table, pages = page_table([-(-n // page) for n in lengths], -(-max(lengths) // page), 1)
    cache = random_cache(pages, kv_heads, page, dim, 1)
    q = torch.randn((tokens, kv_heads * group, dim), generator=gen(2), device="cuda").to(dtype)
    lens, cu = torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.tensor(cu, dtype=torch.int32, device="cuda")
    table = table.cuda()
    litter()
    out, lse = decode.kv_attention(q, tuple(cache), table, lens, cu=cu, return_lse=True, **kw)
    want, want_lse, spread = ref.attention(q, cache, table, lens, cu)
    top = float((cache[1].float() * cache[3][..., None, None]).abs().max())
    assert ((out.cpu().double() - want).abs() <= bound(dtype, dim, spread, top)).all()
    empty = want_lse == -math.inf
    assert bool((out.cpu()[empty] == 0).all()) and torch.equal(lse.cpu() == -math.inf, empty)
    assert bool(torch.isfinite(lse.cpu()[~empty]).all())
    assert status() == 0
    return empty


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("max_length", [0, 1])                 # with and without splits of the keys
@pytest.mark.parametrize("lengths", [[300, 90, 41], [6000, 700, 2500]])
@pytest.mark.parametrize("dim", [32, 128])
def test_attention_of_more_query_tokens_than_max_new(cuda, dtype, max_length, lengths, dim):
    for max_new in (1, 2, 5):
        empty = check(lengths, [0, 4, 5, 45], 45, dtype=dtype, dim=dim, max_length=max_length, max_new=max_new)
        assert not bool(empty.any())


def test_attention_max_new_past_32_bits(cuda):
    check([300, 90], [0, 4, 5], 5, dtype=torch.float16, max_new=1 << 40)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("max_length", [0, 1])
@pytest.mark.parametrize("lengths", [[300, 90], [6000, 700], [40000, 31]])
@pytest.mark.parametrize("cu,tokens", [([3, 5, 6], 11), ([0, 0, 0], 4), ([0, 2, 2], 3), ([4, 4, 5], 5)])
def test_attention_of_tokens_that_no_sequence_names(cuda, dtype, max_length, lengths, cu, tokens):
    empty = check(lengths, cu, tokens, dtype=dtype, max_length=max_length)
    named = torch.zeros(tokens, dtype=torch.bool)
    named[cu[0]:cu[-1]] = True
    assert torch.equal(empty, ~named[:, None].expand(empty.shape))


# ---- append ----

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,page,rot,interleaved", [(64, 16, 64, False), (128, 128, 64, True), (32, 32, 32, False), (64, 64, 34, False)])
@pytest.mark.parametrize("rows", [1, 37, 40, 80])
def test_append_past_the_rotation_tables(cuda, dtype, dim, page, rot, interleaved, rows):
    # tables end inside a block of new tokens, before one, at one token: the tokens before that are stored as ever, the others are zeros
    starts, news = [30, 0, 39, 200, 36], [45, 70, 1, 2, 3]
    table, pages = page_table([-(-(s + n) // page) for s, n in zip(starts, news)], -(-202 // page), 3)
    cache = random_cache(pages, 2, page, dim, 5)
    cu = torch.tensor([0, *news]).cumsum(0).to(torch.int32)
    tokens = int(cu[-1])
    qkv = torch.randn((tokens, 8, dim), generator=gen(6), device="cuda").to(dtype)
    q, k, v = qkv.split((4, 2, 2), 1)
    cos, sin = tables(rot, 300)
    held = torch.cat([torch.arange(s, s + n) for s, n in zip(starts, news)]) < rows
    starts = torch.tensor(starts, dtype=torch.int32)
    want = cpu(cache)
    cleared = [torch.where(held[:, None, None], t.cpu(), 0) for t in (k, v, q)]
    want_q, want_l = ref.append(*cleared[:2], want, table, starts, cu, cos.cpu(), sin.cpu(), interleaved, cleared[2])
    litter()
    got_q, got_l = decode.kv_append(k, v, tuple(cache), table.cuda(), starts.cuda(), cu=cu.cuda(), cos=cos[:rows].contiguous(),
                                    sin=sin[:rows].contiguous(), interleaved=interleaved, q=q)
    assert status() == (0 if bool(held.all()) else 17)
    assert torch.equal(got_q.cpu(), want_q) and torch.equal(got_l.cpu(), want_l)
    for got, w in zip(cache[:2], want[:2]):                     # (zeros of either sign are the same)
        assert ref.same_codes(got, w) or bool(((got.view(torch.uint8).cpu() == w) | ((got.view(torch.uint8).cpu() | w) & 127 == 0)).all())
    for got, w in zip(cache[2:], want[2:]):
        assert torch.equal(got.cpu(), w)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rot", [0, 34, 64])
@pytest.mark.parametrize("cu,tokens", [([3, 5, 6], 9), ([0, 0, 0], 4), ([0, 40, 40], 43), ([4, 4, 5], 5)])
def test_append_queries_that_no_sequence_names(cuda, dtype, rot, cu, tokens):
    table, pages = page_table([4, 4], 4, 3)
    cache = random_cache(pages, 2, 16, 64, 5)
    before = cpu(cache)
    qkv = torch.randn((tokens, 10, 64), generator=gen(6), device="cuda").to(dtype)
    q, k, v = qkv.split((6, 2, 2), 1)
    cos, sin = tables(rot, 80) if rot else (None, None)
    cu_t = torch.tensor(cu, dtype=torch.int32)
    starts = torch.tensor([9, 5], dtype=torch.int32)
    named = torch.zeros(tokens, dtype=torch.bool)
    named[cu[0]:cu[-1]] = True
    host = [None if t is None else t.cpu() for t in (cos, sin)]
    want_q, want_l = ref.append(k.cpu(), v.cpu(), before, table, starts, cu_t, *host, False, q.cpu())
    litter()
    got_q, got_l = decode.kv_append(k, v, tuple(cache), table.cuda(), starts.cuda(), cu=cu_t.cuda(), cos=cos, sin=sin, q=q)
    assert status() == 0
    assert torch.equal(got_q.cpu()[named], want_q[named]) and bool((got_q.cpu()[~named] == 0).all())
    assert torch.equal(got_l.cpu(), want_l)
    assert all(ref.same_codes(a, b) for a, b in zip(cache[:2], before[:2]))


@pytest.mark.parametrize("rot", [0, 34, 64])
def test_append_below_zero_and_offsets_past_the_tokens(cuda, rot):
    cos, sin = tables(rot, 80) if rot else (None, None)
    k = torch.randn((6, 2, 64), generator=gen(1), device="cuda")
    table, pages = page_table([4, 4, 4], 4, 3)
    cache = random_cache(pages, 2, 16, 64, 5)
    before = cpu(cache)
    litter()
    q, lengths = decode.kv_append(k, k, tuple(cache), table.cuda(), torch.tensor([3, -1, 8], dtype=torch.int32, device="cuda"), cos=cos, sin=sin, q=k)
    assert status() == 17 and lengths.tolist() == [5, 0, 10]
    assert bool((q[2:4] == 0).all()) and bool((q[[0, 1, 4, 5]] != 0).any(-1).all())
    for a, b in zip(cache, before):
        a = a.view(torch.uint8) if a.dtype == ref.E4M3 else a
        assert torch.equal(a.cpu()[table[1].long()], b[table[1].long()])
    litter()
    cu = torch.tensor([0, 60, 70, 80], dtype=torch.int32, device="cuda")
    starts = torch.tensor([3, 7, 8], dtype=torch.int32, device="cuda")
    _, lengths = decode.kv_append(k, k, tuple(cache), table.cuda(), starts, cu=cu, cos=cos, sin=sin, q=k)
    assert status() == 17 and lengths.tolist() == [9, 7, 8]


def test_tokens_of_no_sequence_are_refused(cuda):
    cache = decode.PagedKV.empty(2, 1, 32, 16)
    table, none = torch.zeros((0, 1), dtype=torch.int32, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    k, cu = torch.ones((2, 1, 32), device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        decode.kv_append(k, k, cache, table, none, cu=cu, q=k)
    with pytest.raises(ValueError):
        decode.kv_attention(k, cache, table, none, cu=cu)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("grow", [1e-3, 1.0, 40.0])
def test_append_again_changes_nothing(cuda, dtype, grow):
    # the same tokens at the same places a second time: scales that grew stay, old codes are not requantised again
    starts, news, page = [0, 5, 31, 64], [40, 1, 9, 16], 16
    table, pages = page_table([-(-(s + n) // page) for s, n in zip(starts, news)], 5, 2)
    cache = random_cache(pages, 2, page, 64, 3)
    k, v = (torch.randn((sum(news), 2, 64), generator=gen(i), device="cuda").to(dtype) * grow for i in range(2))
    cu = torch.tensor([0, *news]).cumsum(0).to(torch.int32).cuda()
    cos, sin = tables(64, 100)
    args = tuple(cache), table.cuda(), torch.tensor(starts, dtype=torch.int32, device="cuda")
    decode.kv_append(k, v, *args, cu=cu, cos=cos, sin=sin)
    once = cpu(cache)
    decode.kv_append(k, v, *args, cu=cu, cos=cos, sin=sin)
    assert all(torch.equal(a, b) for a, b in zip(once, cpu(cache)))
    # and the second call does write: other tokens change the codes
    decode.kv_append(v, k, *args, cu=cu, cos=cos, sin=sin)
    assert not any(torch.equal(a, b) for a, b in zip(once[:2], cpu(cache)[:2]))
