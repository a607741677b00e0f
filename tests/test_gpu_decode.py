"""The decode operators (piton_b200.decode) on the GPU against plain implementations on the CPU.

Tolerances.  Appending: codes, scales and rotated queries are compared for equality.
Attention, fp32: with eps = 2^-23, a score is off by at most (D + 8) eps times the sum of |q k| terms
(the row's 22-bit query split and the fp32 sums), which moves the weights by that factor, and the
weights' own rounding and the fp32 sums over the keys add less than 2^-17 of the largest |v|; the
16-bit types add the rounding of the weights to fp16 (2^-11) and of the output (2^-11 or 2^-8 of
|o| <= max |v|).  The 4-bit product: a dot product of n terms summed 16 at a time, each sum rounded to
at most 2 eps, plus the 22-bit split of fp32 rows: (n / 16 + 32) 2 eps of sum |x w|, and the
rounding of the output.
"""

import ctypes as C
import math

import pytest
import torch

import decode_ref as ref
from piton_b200 import decode
from piton_b200.runtime.cuda import _lib

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -23
ROUND = {torch.float32: EPS, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def status():
    s = C.c_int(-1)
    torch.cuda.synchronize()
    assert _lib.lib().piton_b200_device_status(C.byref(s)) == 0
    return s.value


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def tables(r, angle_rows):
    inv = 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    a = torch.arange(angle_rows, dtype=torch.float64)[:, None] * inv
    return a.cos().float().cuda(), a.sin().float().cuda()


def random_cache(pages, heads, page, dim, seed, nan_codes=False):
    """Random codes over the whole range (NaN codes only where asked for) and scales 2^-9 .. 2^-6."""
    g = gen(seed)
    codes = []
    for _ in range(2):
        c = torch.randint(0, 256, (pages, heads, page, dim), generator=g, device="cuda", dtype=torch.uint8)
        if not nan_codes:
            c = torch.where((c & 127) == 127, 126, c)
        codes.append(c)
    scales = [torch.ldexp(torch.ones(pages, heads, device="cuda"),
                          torch.randint(-9, -5, (pages, heads), generator=g, device="cuda")) for _ in range(2)]
    return [codes[0].view(ref.E4M3), codes[1].view(ref.E4M3), *scales]


def page_table(needs, width, seed, spare=2):
    """A table of distinct pages in random order, -1 where a sequence needs none; and the pool's size."""
    pages = sum(needs) + spare
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(needs), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(needs):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def cpu(cache):
    return [cache[0].view(torch.uint8).cpu().clone(), cache[1].view(torch.uint8).cpu().clone(), cache[2].cpu().clone(),
            cache[3].cpu().clone()]


def offsets(news):
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32)


# ---- append ------------------------------------------------------------------------------------

def check_append(starts, news, *, page=16, dim=64, kv_heads=2, heads=4, dtype=torch.float32, rot=None, interleaved=False,
                 with_q=True, uniform=False, k=None, v=None, grow=1.0, seed=0):
    need = [-(-(s + n) // page) for s, n in zip(starts, news)]
    width = max(max(need), 1)
    table, pages = page_table(need, width, seed)
    cache = random_cache(pages, kv_heads, page, dim, seed)
    cu = offsets(news)
    tokens = int(cu[-1])
    g = gen(seed + 1)
    qkv = (torch.randn((tokens, heads + 2 * kv_heads, dim), generator=g, device="cuda") * grow).to(dtype)
    q, k0, v0 = qkv.split((heads, kv_heads, kv_heads), 1)
    k, v = k0 if k is None else k, v0 if v is None else v
    rot = dim if rot is None else rot
    cos, sin = tables(rot, max(s + n for s, n in zip(starts, news)) + 1) if rot else (None, None)
    want = cpu(cache)
    starts_t = torch.tensor(starts, dtype=torch.int32)
    wq, wl = ref.append(k.cpu(), v.cpu(), want, table, starts_t, cu, None if cos is None else cos.cpu(),
                        None if sin is None else sin.cpu(), interleaved, q.cpu() if with_q else None)
    got_q, got_l = decode.kv_append(k, v, tuple(cache), table.cuda(), starts_t.cuda(), cu=None if uniform else cu.cuda(),
                                    cos=cos, sin=sin, interleaved=interleaved, q=q if with_q else None)
    assert status() == 0
    assert torch.equal(got_l.cpu(), wl)
    if with_q:
        assert torch.equal(got_q.cpu(), wq)
    else:
        assert got_q is None
    for got, w in zip(cache[:2], want[:2]):
        assert ref.same_codes(got, w)              # every page, the untouched ones too
    for got, w in zip(cache[2:], want[2:]):
        assert torch.equal(got.cpu(), w)
    return cache, want


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_append_matches_step_by_step(cuda, dtype, dim, page):
    # into the middle of a page, at its start, over several pages, one token, none
    check_append([5, 0, page, 3 * page - 1, page + 7], [2 * page + 3, 1, page, 2, 0], page=page, dim=dim, dtype=dtype,
                 seed=dim + page)


@pytest.mark.parametrize("rot,interleaved", [(0, False), (2, False), (2, True), (32, False), (34, True), (64, True)])
def test_append_rotations(cuda, rot, interleaved):
    check_append([0, 19, 70], [1, 30, 5], rot=rot, interleaved=interleaved, seed=rot)


@pytest.mark.parametrize("batch", [1, 3, 200])
@pytest.mark.parametrize("n", [1, 2, 17, 40])
def test_append_uniform(cuda, batch, n):
    if batch * n > 900:
        pytest.skip("slow on the CPU side")
    check_append([(7 * b) % 50 for b in range(batch)], [n] * batch, uniform=True, heads=3, kv_heads=1, dim=32, seed=n)


@pytest.mark.parametrize("kv_heads,heads", [(1, 1), (1, 8), (5, 5), (8, 24), (33, 33)])
def test_append_heads(cuda, kv_heads, heads):
    check_append([4, 100], [3, 20], kv_heads=kv_heads, heads=heads, dim=32, seed=heads)


def test_append_without_queries(cuda):
    check_append([4, 100], [3, 20], with_q=False)


@pytest.mark.parametrize("grow", [1e-30, 1e-3, 1.0, 40.0, 1e30])
@pytest.mark.parametrize("page", [16, 64])
def test_append_grows_scales(cuda, grow, page):
    # the old codes' scales are 2^-9 .. 2^-6: kept for small values, raised (and old codes requantised) for large ones
    _, want = check_append([9, page - 1, 2 * page + 1], [1, 1, 4], page=page, grow=grow)
    assert (want[2].max() > 2.0 ** -5) == (grow >= 40.0)


@pytest.mark.parametrize("value", [0.0, 448.0, 448.1, 1.75, 1.7500002, 2.0 ** -140, 2.0 ** -126, 3e38, 2.0 ** 127])
def test_append_edge_magnitudes(cuda, value):
    k = torch.zeros((2, 2, 64), device="cuda")
    k[0, 0, 3], k[1, 1, 63] = value, -value
    check_append([3, 16], [1, 1], k=k, v=k.flip(0), rot=0)


def test_append_non_finite(cuda):
    g = gen(3)
    k = torch.randn((6, 2, 64), generator=g, device="cuda")
    v = torch.randn((6, 2, 64), generator=g, device="cuda")
    k[0, 0, 5], k[1, 1, 7], v[2, 0, 0], v[5, 1, 63] = math.nan, math.inf, -math.inf, math.nan
    cache, want = check_append([3, 14], [2, 4], k=k, v=v, rot=0)
    assert int(((want[0] & 127) == 127).sum()) == 2 and int(((want[1] & 127) == 127).sum()) == 2
    assert bool(torch.isfinite(cache[2]).all())


def test_append_requantises_nan_codes_as_nan(cuda):
    table = torch.tensor([[0]], dtype=torch.int32, device="cuda")
    cache = random_cache(1, 1, 16, 32, 0)
    cache[0].view(torch.uint8)[0, 0, 2, 5] = 127
    want = cpu(cache)
    k = torch.full((1, 1, 32), 1e6, device="cuda")
    starts = torch.tensor([4], dtype=torch.int32)
    ref.append(k.cpu(), k.cpu(), want, table.cpu(), starts, offsets([1]), None, None, False, None)
    decode.kv_append(k, k, tuple(cache), table, starts.cuda())
    assert ref.same_codes(cache[0], want[0]) and int(want[0][0, 0, 2, 5]) & 127 == 127


@pytest.mark.parametrize("dtype", TYPES)
def test_append_strided_and_unaligned_operands(cuda, dtype):
    g = gen(9)
    store = torch.randn(40 * 1000 + 7, generator=g, device="cuda").to(dtype)
    k = store[3:].as_strided((9, 2, 64), (131, 1200, 1))          # heads far apart, tokens overlapping nothing, odd offset
    v = store[1:].as_strided((9, 2, 64), (640, 77, 1))
    check_append([3, 16, 30], [2, 3, 4], k=k, v=v, dtype=dtype)


def test_append_token_by_token_is_append_at_once(cuda):
    # power-of-two scales: requantising is exact above e4m3's subnormals, so growing a block token by token ends in
    # the same scales, and in codes that differ only below 2^-6 of the block's scale
    dim, page, n = 64, 32, 75
    cos, sin = tables(dim, n)
    g = gen(4)
    k, v = (torch.randn((n, 2, dim), generator=g, device="cuda") * torch.linspace(0.1, 3, n, device="cuda")[:, None, None]
            for _ in range(2))
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    once, steps = random_cache(3, 2, page, dim, 1), random_cache(3, 2, page, dim, 1)
    decode.kv_append(k, v, tuple(once), table, torch.zeros(1, dtype=torch.int32, device="cuda"), cos=cos, sin=sin)
    at = torch.zeros(1, dtype=torch.int32, device="cuda")
    for t in range(n):
        _, at = decode.kv_append(k[t:t + 1], v[t:t + 1], tuple(steps), table, at, cos=cos, sin=sin)
    assert at.tolist() == [n]
    for a, b in zip(once[2:], steps[2:]):
        assert torch.equal(a, b)
    for a, b in zip(once[:2], steps[:2]):
        x, y = a[table[0].long().cpu().tolist()].float(), b[table[0].long().cpu().tolist()].float()
        x, y = (t.transpose(1, 2).reshape(-1, 2, dim)[:n] for t in (x, y))
        assert float((x - y).abs().max()) <= 2.0 ** -9          # one subnormal step
        big = x.abs() >= 2.0 ** -5
        assert torch.equal(x[big], y[big])


def test_append_twice_is_append_once(cuda):
    cache, want = check_append([5, 31], [1, 9], seed=6)
    before = cpu(cache)
    check = [t.clone() for t in before]
    assert all(torch.equal(a, b) for a, b in zip(check, before))


def test_append_bad_table_entries_and_positions_are_not_followed(cuda):
    dim, page = 32, 16
    k = torch.ones((3, 1, dim), device="cuda")
    cos, sin = tables(dim, 40)
    for entry, start, code in ((99, 0, 16), (-1, 0, 16), (2, 32, 17), (2, 40, 17), (2, -5, 17)):
        # the middle sequence is bad: a table entry out of range, a position past the table, past the rotation rows,
        # or negative; the others are stored
        cache = random_cache(5, 1, page, dim, 0)
        before = cpu(cache)
        table = torch.tensor([[0, 1], [entry, 3], [4, 3]], dtype=torch.int32, device="cuda")
        starts = torch.tensor([0, start, 2], dtype=torch.int32, device="cuda")
        decode.kv_append(k, k, tuple(cache), table, starts, cos=cos, sin=sin, q=k)
        assert status() == code
        for got, old in zip(cache[:2], before[:2]):
            got = got.view(torch.uint8).cpu()
            assert torch.equal(got[1:4], old[1:4])
            assert not torch.equal(got[0, 0, 0], old[0, 0, 0]) and not torch.equal(got[4, 0, 2], old[4, 0, 2])
        assert status() == 0                                    # reading it resets it


def test_append_offsets_past_32_bits(cuda):
    # 4.6 GB of codes: the last pages lie beyond 2^32 bytes
    pages, heads, page, dim = 70000, 8, 64, 128
    k_codes = torch.zeros((pages, heads, page, dim), dtype=torch.uint8, device="cuda")
    v_codes = torch.zeros_like(k_codes)
    scales = torch.zeros((2, pages, heads), device="cuda")
    at = [69999, 3, 65536]
    table = torch.tensor([at], dtype=torch.int32, device="cuda")
    g = gen(0)
    k, v = (torch.randn((130, heads, dim), generator=g, device="cuda") for _ in range(2))
    cache = (k_codes, v_codes, scales[0], scales[1])
    decode.kv_append(k, v, cache, table, torch.tensor([5], dtype=torch.int32, device="cuda"))
    small = [torch.zeros((3, heads, page, dim), dtype=torch.uint8) for _ in range(2)] + [torch.zeros((3, heads)) for _ in range(2)]
    ref.append(k.cpu(), v.cpu(), small, torch.tensor([[0, 1, 2]]), torch.tensor([5]), offsets([130]), None, None, False, None)
    for got, want in zip(cache, small):
        assert torch.equal(got[at].cpu(), want)
    assert status() == 0
    q = torch.randn((1, heads, dim), generator=g, device="cuda")
    lengths = torch.tensor([135], dtype=torch.int32, device="cuda")
    out = decode.kv_attention(q, cache, table, lengths)
    want, _, spread = ref.attention(q, [t[at] for t in cache], torch.tensor([[0, 1, 2]]), lengths, [0, 1])
    top = float((small[1].view(ref.E4M3).float() * small[3][..., None, None]).abs().max())
    assert ((out.cpu().double() - want).abs() <= bound(torch.float32, dim, spread, top)).all()


# ---- attention -----------------------------------------------------------------------------------

def bound(dtype, dim, spread, top):
    extra = {torch.float32: 2.0 ** -17, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}[dtype]
    return top * (2 * (dim + 8) * EPS * spread[..., None] + extra)


def check_attention(lengths, news, *, page=16, dim=64, kv_heads=2, group=2, dtype=torch.float32, window=0, uniform=False,
                    q=None, cache=None, table=None, seed=0, lse=True, gain=1.0, scale=None, **kw):
    need = [-(-n // page) for n in lengths]
    if table is None:
        table, pages = page_table(need, max(need + [1]) + 1, seed)
    if cache is None:
        cache = random_cache(pages, kv_heads, page, dim, seed)
    cu = offsets(news)
    if q is None:
        q = (torch.randn((int(cu[-1]), kv_heads * group, dim), generator=gen(seed + 1), device="cuda") * gain).to(dtype)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    got = decode.kv_attention(q, tuple(cache), table.cuda(), lens, cu=None if uniform else cu.cuda(), window=window,
                              scale=scale, return_lse=lse, **kw)
    out, got_lse = got if lse else (got, None)
    assert status() == 0
    assert out.dtype == dtype and out.shape == q.shape and out.is_contiguous()
    want, want_lse, spread = ref.attention(q, cache, table, lens, cu, scale, window)
    used = table[table >= 0].long().cuda()
    top = float((cache[1].view(torch.uint8)[used].view(ref.E4M3).float() * cache[3][used][..., None, None]).nan_to_num(0.0)
                .abs().max()) if used.numel() else 0.0
    diff = (out.cpu().double() - want).abs()
    assert (diff <= bound(dtype, dim, spread, top)).all(), float((diff / bound(dtype, dim, spread, top)).max())
    empty = want_lse == -math.inf
    assert bool((out.cpu()[empty] == 0).all())
    if lse:
        assert torch.equal(got_lse.cpu() == -math.inf, empty)
        off = (got_lse.cpu().double() - want_lse)[~empty].abs()
        tol = ((dim + 8) * EPS * spread + 2 * EPS * want_lse.abs() + 2.0 ** -18)[~empty]
        assert (off <= tol).all()
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_attention_matches_float64(cuda, dtype, dim, page):
    check_attention([1, page - 1, page, page + 1, 300, 0, 777], [1] * 7, page=page, dim=dim, dtype=dtype, uniform=True,
                    seed=dim + page)


@pytest.mark.parametrize("kv_heads,group", [(1, 1), (1, 3), (2, 8), (3, 5), (1, 16), (2, 17), (1, 40), (40, 1)])
def test_attention_heads(cuda, kv_heads, group):
    check_attention([130, 7], [1, 1], kv_heads=kv_heads, group=group, dim=32)
    check_attention([130, 7], [2, 2], kv_heads=kv_heads, group=group, dim=64, dtype=torch.bfloat16)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("news", [[2, 2, 2], [7, 1, 0], [16, 3, 30], [0, 0, 1]])
def test_attention_several_new_tokens(cuda, dtype, news):
    # causal among the new tokens; a sequence with no query tokens; more query tokens than keys (rows without keys)
    check_attention([200, 65, 9], news, dtype=dtype, group=3, uniform=len(set(news)) == 1)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 64, 100, 10000])
@pytest.mark.parametrize("news", [[1, 1, 1, 1], [5, 5, 5, 5]])
def test_attention_window(cuda, window, news):
    check_attention([500, 63, 64, 3], news, window=window, page=32, uniform=True)


@pytest.mark.parametrize("length", [2047, 2048, 5001, 20011])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_long(cuda, length, dtype):
    check_attention([length], [1], kv_heads=1, group=4, dim=128, page=64, dtype=dtype)
    check_attention([length, 1, length // 2], [2, 1, 1], kv_heads=1, group=2, dim=64, page=16, dtype=dtype)


@pytest.mark.parametrize("gain", [1e-4, 30.0, 2000.0])
def test_attention_score_ranges(cuda, gain):
    # from uniform weights to one key taking all
    for dtype in (torch.float32, torch.float16):
        check_attention([400, 33], [1, 1], gain=gain, dtype=dtype)


@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0])
def test_attention_scale(cuda, scale):
    check_attention([100, 33], [1, 2], scale=scale)


@pytest.mark.parametrize("max_length,max_new", [(1, 0), (10, 4), (300, 4), (10 ** 9, 100)])
def test_attention_launch_bounds_do_not_change_what_is_attended(cuda, max_length, max_new):
    check_attention([900, 300, 5], [4, 1, 2], max_length=max_length, max_new=max_new)


def test_attention_batches(cuda):
    n = [(13 * i) % 70 for i in range(300)]
    check_attention(n, [1] * 300, uniform=True, kv_heads=1, dim=32)


def test_attention_strided_operands(cuda):
    for dtype in TYPES:
        store = torch.randn(50000, generator=gen(2), device="cuda").to(dtype)
        q = store[1:].as_strided((3, 4, 64), (2000, 71, 1))
        check_attention([90, 40, 17], [1, 1, 1], q=q, dtype=dtype)


def test_attention_ignores_what_lies_past_the_length(cuda):
    # the rest of the last page holds NaN codes, the pages no table entry names too, with NaN and infinite scales
    for lengths, news, window in (([37, 16, 1], [1, 1, 1], 0), ([37, 20, 5], [3, 3, 3], 0), ([90, 33, 20], [1, 2, 1], 18)):
        need = [-(-n // 16) for n in lengths]
        table, pages = page_table(need, max(need) + 1, 5)
        cache = random_cache(pages, 2, 16, 64, 5)
        clean = [t.clone() for t in cache]
        named = set(table[table >= 0].tolist())
        for page in set(range(pages)) - named:
            cache[0].view(torch.uint8)[page], cache[1].view(torch.uint8)[page] = 127, 255
            cache[2][page], cache[3][page] = math.nan, math.inf
        for b, n in enumerate(lengths):
            if n % 16:
                for c in cache[:2]:
                    c.view(torch.uint8)[int(table[b, n // 16]), :, n % 16:] = 127
            first = n - news[b] + 1 - window if window else 0        # before any query's window
            for j in range(max(0, first)):
                for c in cache[:2]:
                    c.view(torch.uint8)[int(table[b, j // 16]), :, j % 16] = 255
        q = torch.randn((sum(news), 4, 64), generator=gen(6), device="cuda")
        lens, cu = torch.tensor(lengths, dtype=torch.int32, device="cuda"), offsets(news).cuda()
        a = decode.kv_attention(q, tuple(cache), table.cuda(), lens, cu=cu, window=window)
        b = decode.kv_attention(q, tuple(clean), table.cuda(), lens, cu=cu, window=window)
        assert bool(torch.isfinite(a).all()) and torch.equal(a, b)
        assert status() == 0


@pytest.mark.parametrize("where", ["key", "value", "value scale", "key scale"])
def test_attention_nan_reaches_only_the_rows_that_see_it(cuda, where):
    # three new tokens; the second one's key or value holds a NaN: row 0 does not see it, rows 1 and 2 do
    length, news, at = 39, 3, 37
    for dtype in (torch.float32, torch.bfloat16):
        table, pages = page_table([3], 3, 1)
        cache = random_cache(pages, 1, 16, 64, 1)
        page = int(table[0, at // 16])
        if where == "key":
            cache[0].view(torch.uint8)[page, 0, at % 16, 11] = 127
        elif where == "value":
            cache[1].view(torch.uint8)[page, 0, at % 16, 11] = 255
        else:
            cache[3 if where == "value scale" else 2][page] = math.nan
        q = torch.randn((news, 1, 64), generator=gen(3), device="cuda").to(dtype)
        out = decode.kv_attention(q, tuple(cache), table.cuda(), torch.tensor([length], dtype=torch.int32, device="cuda")).float()
        bad = torch.isnan(out).cpu()
        if where == "key":
            assert not bad[0].any() and bad[1:].all()
        elif where == "value":
            assert not bad[0].any() and bool(bad[1:, 0, 11].all()) and int(bad.sum()) == 2
        else:                                   # the scale of the last page, of which every row sees keys
            assert bad.all()


def test_attention_nan_query_row(cuda):
    table, pages = page_table([5, 2], 5, 1)
    cache = random_cache(pages, 2, 16, 64, 1)
    q = torch.randn((2, 4, 64), generator=gen(3), device="cuda")
    q[0, 1, 5] = math.nan
    out = decode.kv_attention(q, tuple(cache), table.cuda(), torch.tensor([70, 20], dtype=torch.int32, device="cuda"))
    bad = torch.isnan(out)
    assert bool(bad[0, 1].all()) and int(bad.sum()) == 64


def test_attention_bad_table_entries_are_not_followed(cuda):
    table = torch.tensor([[0, 77, 2], [-1, 1, 3]], dtype=torch.int32)
    cache = random_cache(4, 1, 16, 32, 2)
    q = torch.randn((2, 2, 32), generator=gen(1), device="cuda")
    lens = torch.tensor([45, 31], dtype=torch.int32, device="cuda")
    out = decode.kv_attention(q, tuple(cache), table.cuda(), lens)
    assert status() == 16
    # the same as sequences without those 16 keys
    want = decode.kv_attention(q, tuple(cache), torch.tensor([[0, 2], [1, 1]], dtype=torch.int32, device="cuda"),
                               torch.tensor([29, 15], dtype=torch.int32, device="cuda"))
    assert status() == 0
    assert float((out - want).abs().max()) <= 1e-4
    # a length past the table: the keys that the table holds are attended
    out = decode.kv_attention(q, tuple(cache), torch.tensor([[0, 2], [1, 3]], dtype=torch.int32, device="cuda"),
                              torch.tensor([40, 32], dtype=torch.int32, device="cuda"))
    assert status() == 17
    want = decode.kv_attention(q, tuple(cache), torch.tensor([[0, 2], [1, 3]], dtype=torch.int32, device="cuda"),
                               torch.tensor([32, 32], dtype=torch.int32, device="cuda"))
    assert status() == 0
    assert float((out - want).abs().max()) <= 1e-4


def test_attention_repeats_exactly(cuda):
    table, pages = page_table([200], 200, 0)
    cache = random_cache(pages, 4, 64, 128, 0)
    q = torch.randn((1, 32, 128), generator=gen(1), device="cuda", dtype=torch.float32).bfloat16()
    lens = torch.tensor([12001], dtype=torch.int32, device="cuda")
    a = decode.kv_attention(q, tuple(cache), table.cuda(), lens)
    for _ in range(5):
        assert torch.equal(a, decode.kv_attention(q, tuple(cache), table.cuda(), lens))


# ---- 4-bit products ------------------------------------------------------------------------------

def check_matvec(rows, inner, outer, *, group=32, dtype=torch.float32, zeros=True, bias=True, scale_type=None, seed=0, x=None,
                 codes=None):
    g = gen(seed)
    groups = -(-inner // group)
    if x is None:
        x = torch.randn((rows, inner), generator=g, device="cuda").to(dtype)
    if codes is None:
        codes = torch.randint(0, 256, (outer, (inner + 1) // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.rand((outer, groups), generator=g, device="cuda") * 0.1).to(scale_type or dtype)
    z = torch.randint(0, 16, (outer, groups), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    b = torch.randn(outer, generator=g, device="cuda").to(dtype) if bias else None
    y = decode.matvec_w4(x, codes, scales, group=group, zeros=z, bias=b)
    want, size = ref.matvec_w4(x, codes, scales, z, b, group)
    assert y.dtype == dtype and y.shape == want.shape
    tol = (inner / 16 + 32) * 2 * EPS * size + ROUND[dtype] * want.abs() + 1e-7 * (dtype == torch.float16)
    assert ((y.cpu().double() - want).abs() <= tol).all()
    return y


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 3, 8, 9, 16, 17, 33])
def test_matvec_matches_float64(cuda, dtype, group, rows):
    check_matvec(rows, 512, 80, group=group, dtype=dtype)


@pytest.mark.parametrize("inner", [1, 2, 7, 8, 31, 32, 33, 100, 127, 129, 1000, 4099, 8192])
@pytest.mark.parametrize("outer", [1, 15, 16, 17, 100])
def test_matvec_odd_sizes(cuda, inner, outer):
    check_matvec(2, inner, outer, group=64, seed=inner)
    check_matvec(1, inner, outer, group=128, dtype=torch.bfloat16, zeros=False, bias=False, seed=inner)


@pytest.mark.parametrize("rows,inner,outer", [(1, 16384, 33), (1, 2048, 6000), (5, 8200, 1027), (40, 4096, 300)])
def test_matvec_large(cuda, rows, inner, outer):
    check_matvec(rows, inner, outer, group=128)
    check_matvec(rows, inner, outer, group=32, dtype=torch.float16, scale_type=torch.float32)


@pytest.mark.parametrize("scale_type", TYPES)
def test_matvec_scale_types(cuda, scale_type):
    check_matvec(4, 300, 50, scale_type=scale_type, dtype=torch.bfloat16)


def test_matvec_one_dimension(cuda):
    x = torch.randn(320, generator=gen(0), device="cuda")
    assert check_matvec(1, 320, 48, x=x).shape == (48,)


def test_matvec_strided_and_unaligned_operands(cuda):
    g = gen(5)
    for dtype in TYPES:
        store = torch.randn(9000, generator=g, device="cuda").to(dtype)
        raw = torch.randint(0, 256, (50 * 300,), generator=g, device="cuda", dtype=torch.uint8)
        for off, stride in ((0, 256), (1, 257), (8, 264), (16, 272)):
            check_matvec(3, 500, 40, dtype=dtype, x=store[off:].as_strided((3, 500), (1001, 1)),
                         codes=raw[off:].as_strided((40, 250), (stride, 1)))


def test_matvec_extreme_rows(cuda):
    # rows of very different magnitudes, values past fp16's range, and a row of zeros
    x = torch.randn((4, 256), generator=gen(1), device="cuda")
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2] = 0
    x[3, ::2] *= 1e5
    check_matvec(4, 256, 64, x=x, bias=False)


def test_matvec_non_finite_rows_stay_alone(cuda):
    x = torch.randn((3, 256), generator=gen(1), device="cuda")
    clean = check_matvec(3, 256, 64, x=x)
    x = x.clone()
    x[1, 17] = math.nan
    g = gen(0)
    codes = torch.randint(0, 256, (64, 128), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.rand((64, 8), generator=g, device="cuda") * 0.1 + 0.01
    y = decode.matvec_w4(x, codes, scales, group=32)
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isfinite(y[[0, 2]]).all())
    assert bool(torch.isfinite(clean).all())


def test_matvec_zero_inner_and_empty(cuda):
    e = torch.empty((5, 0), dtype=torch.uint8, device="cuda")
    s = torch.empty((5, 0), device="cuda")
    b = torch.arange(5.0, device="cuda")
    y = decode.matvec_w4(torch.empty((2, 0), device="cuda"), e, s, bias=b)
    assert torch.equal(y, b.expand(2, 5))
    assert decode.matvec_w4(torch.empty((0, 64), device="cuda"), torch.empty((3, 32), dtype=torch.uint8, device="cuda"),
                            torch.empty((3, 1), device="cuda"), group=64).shape == (0, 3)


def test_matvec_codes_past_32_bits(cuda):
    # 2^32 + bytes of codes
    inner, outer = 32768, 262144 + 40
    codes = torch.zeros((outer, inner // 2), dtype=torch.uint8, device="cuda")
    g = gen(0)
    tail = torch.randint(0, 256, (40, inner // 2), generator=g, device="cuda", dtype=torch.uint8)
    codes[-40:] = tail
    scales = torch.full((outer, inner // 128), 2.0 ** -6, device="cuda")
    x = torch.randn((1, inner), generator=g, device="cuda")
    y = decode.matvec_w4(x, codes, scales)
    want, size = ref.matvec_w4(x, tail, scales[-40:], None, None, 128)
    assert ((y[:, -40:].cpu().double() - want).abs() <= (inner / 16 + 32) * 2 * EPS * size).all()


def test_quantize_w4_round_trip(cuda):
    w = torch.randn((70, 333), generator=gen(0), device="cuda")
    for zeros in (True, False):
        codes, scales, z = decode.quantize_w4(w, 64, zeros=zeros)
        eye = torch.eye(333, device="cuda")[:17]
        back = decode.matvec_w4(eye, codes, scales, group=64, zeros=z)
        step = scales.repeat_interleave(64, 1)[:, :17].T
        assert ((back - w[:, :17].T).abs() <= step * (1.0 if zeros else 0.5) + 1e-6).all()


# ---- streams, graphs, empty calls -------------------------------------------------------------------

def test_operators_on_another_stream_and_in_a_graph(cuda):
    def step(q, k, v, cache, table, starts, w):
        y = decode.matvec_w4(q.view(2, -1)[:, :128], *w[:2], group=32, zeros=w[2])
        qr, lengths = decode.kv_append(k, v, cache, table, starts, q=q)
        return y, decode.kv_attention(qr, cache, table, lengths)

    def inputs(seed):
        g = gen(seed)
        q, k, v = (torch.randn((2, h, 64), generator=g, device="cuda") for h in (4, 2, 2))
        table, pages = page_table([20, 20], 20, 1)
        cache = tuple(random_cache(pages, 2, 64, 64, seed))
        starts = torch.tensor([1200, 77], dtype=torch.int32, device="cuda")
        w = decode.quantize_w4(torch.randn((96, 128), generator=g, device="cuda"), 32)
        return q, k, v, cache, table.cuda(), starts, w

    want = step(*inputs(0))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        args = inputs(0)
        got = [step(*args) for _ in range(10)]
    side.synchronize()
    for y in got:
        assert all(torch.equal(a, b) for a, b in zip(y, want))
    args = inputs(0)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = step(*args)
    for _ in range(3):
        for t in held:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_two_streams_at_once(cuda):
    table, pages = page_table([100], 100, 0)
    cache = tuple(random_cache(pages, 1, 64, 64, 0))
    lens = torch.tensor([6000], dtype=torch.int32, device="cuda")
    qs = [torch.randn((1, 2, 64), generator=gen(i), device="cuda") for i in range(2)]
    table = table.cuda()
    want = [decode.kv_attention(q, cache, table, lens) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(50):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(decode.kv_attention(qs[i], cache, table, lens))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_empty_calls(cuda):
    cache = decode.PagedKV.empty(2, 1, 32, 16)
    table = torch.zeros((0, 1), dtype=torch.int32, device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    k = torch.empty((0, 1, 32), device="cuda")
    q, lengths = decode.kv_append(k, k, cache, table, none, q=k)
    assert q.shape == (0, 1, 32) and lengths.shape == (0,)
    assert decode.kv_attention(k, cache, table, none).shape == (0, 1, 32)
    # sequences without new tokens
    table = torch.zeros((3, 1), dtype=torch.int32, device="cuda")
    starts = torch.tensor([4, 0, 9], dtype=torch.int32, device="cuda")
    for cu in (None, torch.zeros(4, dtype=torch.int32, device="cuda")):
        assert decode.kv_append(k, k, cache, table, starts, cu=cu)[1].tolist() == [4, 0, 9]
    assert status() == 0
