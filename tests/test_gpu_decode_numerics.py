"""Numerics of the decode operators where operands are far apart: zero points of any byte, and what a
product or a softmax must not lose beside something much larger.

Tolerances are those of test_gpu_decode.py unless a test derives its own.
"""

import pytest
import torch

import decode_ref as ref
from piton_b200 import decode
from test_gpu_decode import EPS, ROUND, TYPES, bound, gen, offsets, page_table, random_cache, status

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer", [(1, 384, 40), (9, 2304, 72), (2, 1280, 4800)])
@pytest.mark.parametrize("group", [32, 128])
def test_matvec_zero_points_of_any_byte(cuda, dtype, rows, inner, outer, group):
    # 16 is what a checkpoint that stores zero - 1 in four bits gives; the C interface says uint8
    g = gen(group + rows)
    x = torch.randn((rows, inner), generator=g, device="cuda").to(dtype)
    codes = torch.randint(0, 256, (outer, inner // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.rand((outer, inner // group), generator=g, device="cuda") * 0.1).to(dtype)
    for zeros in (torch.full((outer, inner // group), 16, device="cuda"),
                  torch.randint(0, 256, (outer, inner // group), generator=g, device="cuda")):
        zeros = zeros.to(torch.uint8)
        y = decode.matvec_w4(x, codes, scales, group=group, zeros=zeros)
        want, size = ref.matvec_w4(x, codes, scales, zeros, None, group)
        tol = (inner / 16 + 32) * 2 * EPS * size + ROUND[dtype] * want.abs() + 1e-7 * (dtype == torch.float16)
        assert ((y.cpu().double() - want).abs() <= tol).all()


# A product's operands are exact (4-bit codes less their zero points, and x, fp32 in three pieces), so what is left are the fp32 sums
# of test_gpu_decode.py's bound, (n / 16 + 32) 2 eps of sum |x w|: something large that faces a weight of zero adds nothing to it.

def product_bound(dtype, inner, want, size):
    return (inner / 16 + 32) * 2 * EPS * size + ROUND[dtype] * want.abs() + 1e-7 * (dtype == torch.float16)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer", [(1, 256, 40), (3, 4096, 64), (9, 2304, 72), (2, 1280, 4800)])
@pytest.mark.parametrize("times", [1e3, 5e3, 1e9])
def test_matvec_channels_that_face_zero_weights(cuda, dtype, rows, inner, outer, times):
    # one channel of every 128 is `times` the others and its weights sit at the zero point
    if dtype == torch.float16 and times > 1e4:
        pytest.skip("past the type's range")
    g = gen(rows)
    x = torch.randn((rows, inner), generator=g, device="cuda")
    x[:, 4::128] = times * (1 + torch.rand((rows, inner // 128), generator=g, device="cuda"))
    x = x.to(dtype)
    codes = torch.randint(0, 256, (outer, inner // 2), generator=g, device="cuda", dtype=torch.uint8)
    codes[:, 2::64] = codes[:, 2::64] & 0xF0 | 8
    scales = (torch.rand((outer, inner // 64), generator=g, device="cuda") * 0.1).to(dtype)
    y = decode.matvec_w4(x, codes, scales, group=64)
    want, size = ref.matvec_w4(x, codes, scales, None, None, 64)
    assert float(size.max()) < 1e5
    assert ((y.cpu().double() - want).abs() <= product_bound(dtype, inner, want, size)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,inner,outer", [(1, 128, 24), (5, 1280, 48), (16, 4096, 33), (2, 1280, 4800)])
def test_matvec_codes_around_the_zero_point(cuda, dtype, group, rows, inner, outer):
    # x of one sign; groups whose codes all equal the zero point give exactly 0, others lie one step to either side of it
    g = gen(inner + group)
    x = (0.8 + 0.2 * torch.rand((rows, inner), generator=g, device="cuda")).to(dtype)
    scales = (0.5 + torch.rand((outer, inner // group), generator=g, device="cuda")).to(dtype)
    zeros = torch.randint(1, 15, (outer, inner // group), generator=g, device="cuda", dtype=torch.uint8)
    for spread in (0, 1):
        off = torch.randint(-spread, spread + 1, (outer, inner), generator=g, device="cuda")
        off[::3] = 0
        code = zeros.repeat_interleave(group, 1).int() + off
        codes = (code[:, 0::2] | code[:, 1::2] << 4).to(torch.uint8)
        y = decode.matvec_w4(x, codes, scales, group=group, zeros=zeros)
        want, size = ref.matvec_w4(x, codes, scales, zeros, None, group)
        assert bool((y.cpu()[:, ::3] == 0).all()) and bool((size[:, ::3] == 0).all())
        assert ((y.cpu().double() - want).abs() <= product_bound(dtype, inner, want, size)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer", [(4, 256, 40), (8, 4096, 64), (8, 1280, 4800)])
def test_matvec_keeps_every_bit_of_an_element(cuda, dtype, rows, inner, outer):
    # each row of x has one element of its type's full significand, from 2^-100 to 2^100 (fp16: 2^-8 to 2^8), beside larger ones that face
    # weights of zero.  The product is then one term: its pieces' sum and the scale are rounded, 8 eps at most
    g = gen(inner)
    top = 8 if dtype == torch.float16 else 100
    lone = torch.ldexp(1 + torch.rand(rows, generator=g, device="cuda"), torch.randint(-top, top, (rows,), generator=g, device="cuda"))
    x = torch.zeros((rows, inner), device="cuda")
    x[:, 0::2] = torch.ldexp(torch.ones_like(x[:, 0::2]), torch.tensor(min(top + 6, 100), device="cuda"))
    at = 2 * torch.randint(0, inner // 2, (rows,), generator=g, device="cuda") + 1
    x[torch.arange(rows, device="cuda"), at] = lone
    x = x.to(dtype)
    codes = torch.randint(0, 16, (outer, inner // 2), generator=g, device="cuda", dtype=torch.uint8) << 4 | 8     # even elements: zero
    scales = torch.rand((outer, inner // 128), generator=g, device="cuda")
    y = decode.matvec_w4(x, codes, scales)
    want, _ = ref.matvec_w4(x, codes, scales, None, None, 128)
    want = want.clamp(-65504.0, 65504.0) if dtype == torch.float16 else want
    round_ = 0.0 if dtype == torch.float32 else ROUND[dtype]
    small = 2.0 ** -24 if dtype == torch.float16 else 0.0
    assert ((y.cpu().double() - want).abs() <= (8 * EPS + round_) * want.abs() + small).all()


def test_matvec_infinite_elements(cuda):
    # infinity times a weight: of the weight's sign, NaN where the weight is zero; the other rows are as without it
    g = gen(0)
    codes = torch.randint(0, 256, (60, 256), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.rand((60, 4), generator=g, device="cuda") + 0.1
    weight = (codes[:, 100] >> 4).double().cpu() - 8              # of element 201
    for dtype in TYPES:
        x = torch.randn((3, 512), generator=g, device="cuda").to(dtype)
        clean = decode.matvec_w4(x, codes, scales)
        x[1, 201] = float("inf")
        y = decode.matvec_w4(x, codes, scales)
        assert torch.equal(y[[0, 2]], clean[[0, 2]])
        want = weight * float("inf")
        assert torch.equal(y[1].cpu().double().nan_to_num(nan=7.0), want.nan_to_num(nan=7.0))


# ---- attention ----

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,group", [(32, 1), (64, 5), (128, 16)])
def test_attention_scores_of_any_size(cuda, dtype, dim, group):
    # scores from 2^20 to 2^60, where a step of fp32 is more than the weights' whole range: rows stay averages of values
    lengths = [300, 77, 900]
    table, pages = page_table([-(-n // 16) for n in lengths], 60, 3)
    cache = random_cache(pages, 1, 16, dim, 3)
    top = float((cache[1].float() * cache[3][..., None, None]).abs().max())
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for power in range(20, 61):
        q = torch.randn((3, group, dim), generator=gen(power), device="cuda") * 2.0 ** (power - 3)
        out, lse = decode.kv_attention(q.to(dtype), tuple(cache), table.cuda(), lens, return_lse=True)
        assert float(out.float().abs().max()) <= top * (1 + 2.0 ** -6), power      # (also false for NaN)
        assert bool(torch.isfinite(lse).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_score_one_step_above_a_large_one(cuda, dtype):
    # scores of 2^p and the next fp32 number above, 256 keys apart (the same warp's next keys): the reference of the weights may lag
    # the maximum, but by what the weights' fp16 has room for
    for power in range(20, 32):
        cache = [torch.zeros((33, 1, 16, 32), dtype=torch.uint8, device="cuda").view(ref.E4M3) for _ in range(2)]
        scales = [torch.ones((33, 1), device="cuda") for _ in range(2)]
        cache[0][0, 0, 3, 0], cache[0][16, 0, 5, 0], cache[0][16, 0, 5, 1] = 128.0, 128.0, 16.0
        cache[1][0, 0, 3], cache[1][16, 0, 5] = 1.0, 3.0
        step = 2.0 ** (power - 23)
        if step / 16 < 2.0 ** -9 or (dtype == torch.float16 and power > 22):
            continue
        q = torch.zeros((1, 1, 32), device="cuda")
        q[0, 0, 0], q[0, 0, 1] = 2.0 ** (power - 7), step / 16
        table = torch.arange(33, dtype=torch.int32, device="cuda")[None]
        out = decode.kv_attention(q.to(dtype), (*cache, *scales), table, torch.tensor([500], dtype=torch.int32, device="cuda"),
                                  scale=0.6931471805599453, max_length=1).float()
        w = 2.0 ** -step
        want = (w * 1.0 + 3.0) / (w + 1.0)
        assert float((out - want).abs().max()) <= 2.0 ** -7 * want, (power, out.flatten()[0].item(), want)


def attention_tops(q, cache, table, lengths, cu, window):
    """The largest |v| of each output element's row among the keys that the row sees, dimension by dimension, float64 [tokens, heads, dim]."""
    page, kv_heads, dim = cache[0].shape[2], cache[0].shape[1], cache[0].shape[3]
    group = q.shape[1] // kv_heads
    values = (cache[1].view(ref.E4M3).double() * cache[3].double()[..., None, None]).cpu().abs()
    top = torch.zeros(q.shape, dtype=torch.float64)
    for b in range(len(lengths)):
        v = torch.cat([values[int(i)] for i in table[b, :-(-lengths[b] // page)]], 1)      # [kv_heads, keys, dim]
        for t in range(int(cu[b]), int(cu[b + 1])):
            end = lengths[b] - int(cu[b + 1]) + t + 1
            first = max(0, end - window) if window else 0
            if end > first:
                top[t] = v[:, first:end].amax(1).repeat_interleave(group, 0)
    return top


def check_far(q, cache, table, lengths, news, window):
    cu, lens = offsets(news), torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = decode.kv_attention(q, tuple(cache), table.cuda(), lens, cu=cu.cuda(), window=window).cpu().double()
    want, _, spread = ref.attention(q, cache, table, lens, cu, None, window)
    tol = bound(q.dtype, q.shape[2], spread, attention_tops(q, cache, table, lengths, cu, window))
    if q.dtype == torch.float16:                                # below the type's normal numbers, and past its largest
        tol = tol + 2.0 ** -24
        out, want = (x.clamp(-65504.0, 65504.0) for x in (out, want))
    assert ((out - want).abs() <= tol).all(), float(((out - want).abs() / tol).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,page", [(32, 16), (64, 16), (64, 128), (128, 16), (128, 64)])
@pytest.mark.parametrize("window", [0, 50])
def test_attention_scales_far_apart_row_by_row(cuda, dtype, dim, page, window):
    # random scales over 2^60; every row's tolerance is that of the values which it sees
    lengths, news = [400, 333, 17], [1, 2, 1]
    table, pages = page_table([-(-n // page) for n in lengths], -(-400 // page), 3)
    cache = random_cache(pages, 2, page, dim, 3)
    cache[3].copy_(torch.ldexp(torch.ones(pages, 2, device="cuda"), torch.randint(-30, 30, (pages, 2), generator=gen(4), device="cuda")))
    q = torch.randn((4, 8, dim), generator=gen(1), device="cuda").to(dtype)
    check_far(q, cache, table, lengths, news, window)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,page", [(32, 16), (64, 32), (128, 16), (128, 64)])
@pytest.mark.parametrize("where", ["later token", "before the window", "first page", "one dimension"])
@pytest.mark.parametrize("far", [8, 24, 30, 60])
def test_attention_beside_a_page_of_large_values(cuda, dtype, dim, page, where, far):
    # one page's scale is 2^far times the others'.  Its large values belong to a later query token, lie before the window of a page
    # that is partly visible, face a weight that underflows, or lie in one dimension; the other elements keep their own precision
    table, pages = page_table([20], 20, 7)
    cache = random_cache(pages, 1, page, dim, 7)
    raw = cache[1].view(torch.uint8)
    cache[3].fill_(2.0 ** -9)
    length, news, window = 20 * page, [2], 0
    q = torch.randn((2, 4, dim), generator=gen(2), device="cuda")
    if where == "later token":
        length = 19 * page + 1                                  # the last token alone is in the last page
        big = int(table[0, 19])
    elif where == "before the window":
        window, big = 10 * page + page // 2, int(table[0, 9])   # half of that page is seen by token 0, one key fewer by token 1
        raw[big, :, page // 2 - 1:] = 0
    elif where == "first page":                                 # its keys score far below the others
        big = int(table[0, 0])
        cache[0].view(torch.uint8)[big] = 0xFE                  # -448
        q = q.abs()
        for p in range(1, 20):
            codes = cache[0].view(torch.uint8)[int(table[0, p])]
            cache[0].view(torch.uint8)[int(table[0, p])] = codes & 0x3F
        cache[2].fill_(2.0 ** -2)
        raw[big] = 0
    else:
        big = int(table[0, 5])
        raw[big, :, :, 1:] = 0
    cache[3][big] = 2.0 ** (far - 9)
    check_far(q.to(dtype), cache, table, [length], news, window)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,page", [(32, 64), (64, 64), (128, 32), (128, 128)])
def test_attention_small_values_after_pages_that_are_not_followed(cuda, dtype, dim, page):
    # the first 512 keys are on pages that do not exist, the others' values are around 2^-40 (fp16: 2^-12)
    bad, good = 512 // page, 1 + 300 // page
    table, pages = page_table([good], good, 1)
    cache = random_cache(pages, 1, page, dim, 1)
    cache[3].fill_(2.0 ** (-20 if dtype == torch.float16 else -48))
    holes = torch.cat((torch.full((1, bad), -1, dtype=torch.int32), table), 1)
    q = torch.randn((1, 4, dim), generator=gen(2), device="cuda").to(dtype)
    length = good * page - 3
    out = decode.kv_attention(q, tuple(cache), holes.cuda(), torch.tensor([512 + length], dtype=torch.int32, device="cuda"),
                              max_length=1).cpu().double()
    assert status() == 16
    want, _, spread = ref.attention(q, cache, table, torch.tensor([length]), [0, 1])
    tol = bound(dtype, dim, spread, attention_tops(q, cache, table, [length], [0, 1], 0)) + (2.0 ** -24 if dtype == torch.float16 else 0.0)
    assert ((out - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("length,max_length", [(1500, 0), (1500, 1), (20000, 0)])
def test_attention_nan_value_of_a_key_without_weight(cuda, dtype, length, max_length):
    # 0 times NaN is NaN, in whichever split of the keys it is (several, one, many), and in its own dimension alone
    pages = -(-length // 64)
    cache = [torch.zeros((pages, 1, 64, 64), dtype=torch.uint8, device="cuda") for _ in range(2)]
    cache[0].fill_(0x38), cache[1].fill_(0x38)                  # ones
    cache[0][:pages // 2], cache[1][0, 0, 7, 11] = 0xB8, 0x7F   # the first half of the keys: minus one; a NaN in a value of theirs
    scales = [torch.ones((pages, 1), device="cuda") for _ in range(2)]
    q = torch.full((1, 3, 64), 100.0, device="cuda").to(dtype)
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    out = decode.kv_attention(q, (cache[0].view(ref.E4M3), cache[1].view(ref.E4M3), *scales), table,
                              torch.tensor([length], dtype=torch.int32, device="cuda"), max_length=max_length)
    assert bool(torch.isnan(out[:, :, 11]).all()) and int(torch.isnan(out).sum()) == 3


@pytest.mark.parametrize("dim,group,new", [(32, 4, 1), (64, 8, 1), (128, 4, 4), (128, 16, 1)])
def test_attention_fp16_rows_keep_the_weights(cuda, dim, group, new):
    # a few keys whose values nearly cancel: what is left is rounded once, to the output, beside the bound of fp32 rows (2^-17 of the
    # largest |v|, half an ulp of fp16 there is 2^-11)
    lengths = [5, 6, 7, 9, 30]
    table, pages = page_table([2] * 5, 2, 1)
    cache = random_cache(pages, 2, 16, dim, 1)
    raw = cache[1].view(torch.uint8)
    raw[:, :, 1::2] = raw[:, :, 0::2] ^ 0x80                    # every other value is its neighbour's negative
    cache[2].fill_(2.0 ** -12)                                  # nearly equal weights
    q = torch.randn((5 * new, 2 * group, dim), generator=gen(dim), device="cuda").half()
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = decode.kv_attention(q, tuple(cache), table.cuda(), lens).cpu().double()
    want, _, spread = ref.attention(q, cache, table, lens, offsets([new] * 5))
    top = float((cache[1].float() * cache[3][..., None, None]).abs().max())
    tol = bound(torch.float32, dim, spread, top) + 2.0 ** -11 * want.abs() + 2.0 ** -25
    assert ((out - want).abs() <= tol).all(), float(((out - want).abs() / tol).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer,group", [(4800, 96, 1, 32), (5000, 130, 17, 64), (4800, 128, 31, 128), (2500, 256, 32, 128),
                                                    (3000, 300, 33, 32), (24, 2304, 2050, 64), (64, 700, 700, 128)])
def test_matvec_many_rows(cuda, dtype, rows, inner, outer, group):
    # the weight rows of a launch of many rows of x are cut by how many CTAs there are in all; a few outputs stay whole
    g = gen(rows)
    x = torch.randn((rows, inner), generator=g, device="cuda").to(dtype)
    codes = torch.randint(0, 256, (outer, (inner + 1) // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.rand((outer, -(-inner // group)), generator=g, device="cuda") * 0.1).to(dtype)
    y = decode.matvec_w4(x, codes, scales, group=group)
    want, size = ref.matvec_w4(x, codes, scales, None, None, group)
    assert ((y.cpu().double() - want).abs() <= product_bound(dtype, inner, want, size)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,inner,outer,group", [(1, 1024, 40, 128), (4, 4096, 64, 32), (9, 1280, 4800, 128)])
def test_matvec_of_elements_near_the_largest(cuda, dtype, rows, inner, outer, group):
    # |x| up to 3e38, weights below 1e-4: the outputs are far from the type's largest, and so must the sums on the way be
    g = gen(rows)
    x = ((2 * torch.rand((rows, inner), generator=g, device="cuda") - 1) * 3e38).to(dtype)
    x[:, ::2] = x[:, ::2].abs()
    codes = torch.randint(0, 256, (outer, inner // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.rand((outer, inner // group), generator=g, device="cuda") * 1e-5).to(dtype)
    y = decode.matvec_w4(x, codes, scales, group=group)
    want, size = ref.matvec_w4(x, codes, scales, None, None, group)
    assert float(size.max()) < 3e38
    assert ((y.cpu().double() - want).abs() <= product_bound(dtype, inner, want, size)).all()
