"""The decode operators at the sizes where their kernels change how they cut the work.

Tolerances are those of test_gpu_decode.py.  A product's row of x is held, per block of 128 elements, as
fixed-point numbers of the block's largest magnitude: an element is off by at most 2^-16 of it for the
16-bit types and 2^-24 for fp32 (127 2^8 or 127 2^16 steps, half a step off), which
``test_matvec_outliers`` allows times the sum of |w| over the block.
"""

import ctypes as C
import math

import pytest
import torch

import decode_ref as ref
from piton_b200 import decode
from piton_b200.runtime.cuda import _lib
from test_gpu_decode import (EPS, ROUND, TYPES, bound, check_append, check_attention, check_matvec, gen,
                              offsets, page_table, random_cache, status)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer,group", [
    (1, 700, 4736, 128), (3, 700, 4743, 64), (16, 513, 4737, 32),              # warps along the rows, in several parts
    (5, 4100, 4800, 64), (17, 2304, 4751, 128), (2, 8200, 9000, 32),
    (16, 4352, 100, 128), (9, 2816, 600, 32), (1, 2049, 17, 64), (33, 1300, 64, 64)])
def test_matvec_cuts(cuda, dtype, rows, inner, outer, group):
    check_matvec(rows, inner, outer, group=group, dtype=dtype, seed=rows)


@pytest.mark.parametrize("rows,inner", [(1, 2048), (1, 2049), (8, 256), (8, 257), (4, 512), (16, 128), (16, 257)])
def test_matvec_x_laid_out_by_every_block_or_once(cuda, rows, inner):
    for dtype in TYPES:
        check_matvec(rows, inner, 40, group=64, dtype=dtype, seed=inner)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad", [0, 1, 2, 4, 12])
def test_matvec_row_strides(cuda, dtype, pad):
    # rows of codes that start on 1, 2, 4 or 16 bytes, x whose rows are not aligned; warps along either dimension
    g = gen(pad)
    for rows, inner, outer in ((3, 1000, 50), (2, 1536, 4800)):
        raw = torch.randint(0, 256, (outer * (inner // 2 + pad) + 16,), generator=g, device="cuda", dtype=torch.uint8)
        codes = raw[pad:].as_strided((outer, inner // 2), (inner // 2 + pad, 1))
        x = torch.randn(rows * (inner + pad) + 16, generator=g, device="cuda").to(dtype)[pad:].as_strided((rows, inner), (inner + pad, 1))
        check_matvec(rows, inner, outer, group=128, dtype=dtype, codes=codes, x=x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer", [(2, 384, 48), (3, 4096, 64), (2, 1280, 4800)])
def test_matvec_outliers(cuda, dtype, rows, inner, outer):
    # a few elements a thousand times the others, some of them facing weights of zero
    g = gen(rows)
    x = torch.randn((rows, inner), generator=g, device="cuda")
    x[:, 5::97] *= 1000
    x = x.to(dtype)
    codes = torch.randint(0, 256, (outer, inner // 2), generator=g, device="cuda", dtype=torch.uint8)
    codes[:, 2] = 0x88                                          # elements 4 and 5: zero
    scales = (torch.rand((outer, inner // 32), generator=g, device="cuda") * 0.1).to(dtype)
    y = decode.matvec_w4(x, codes, scales, group=32)
    want, size = ref.matvec_w4(x, codes, scales, None, None, 32)
    half = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -16
    tops = x.cpu().double().abs().view(rows, -1, 128).amax(-1).repeat_interleave(128, 1)
    _, fixed = ref.matvec_w4(tops, codes, scales, None, None, 32)
    tol = (inner / 16 + 32) * 2 * EPS * (size + half * fixed) + half * fixed + ROUND[dtype] * (want.abs() + half * fixed)
    assert ((y.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("rows,inner", [(3, 256), (5, 4096), (16, 1024)])
def test_matvec_non_finite_rows_and_scales_stay_alone(cuda, rows, inner):
    # rows of x share instructions two by two and workspaces; weight rows share tiles
    g = gen(rows)
    x = torch.randn((rows, inner), generator=g, device="cuda")
    codes = torch.randint(0, 256, (50, inner // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.rand((50, inner // 64), generator=g, device="cuda") + 0.01
    clean = decode.matvec_w4(x, codes, scales, group=64)
    x[1, inner - 1], x[2, 0] = math.nan, math.inf
    scales[7, 1], scales[20, 0] = math.nan, math.inf
    y = decode.matvec_w4(x, codes, scales, group=64)
    assert not bool(torch.isfinite(y[1:3]).any())
    assert not bool(torch.isfinite(y[:, [7, 20]]).any())
    keep = [i for i in range(50) if i not in (7, 20)]
    for m in [0, *range(3, rows)]:
        assert torch.equal(y[m, keep], clean[m, keep])


def test_matvec_each_row_is_its_own_product(cuda):
    # what a row gives depends on no other row of x
    g = gen(0)
    codes = torch.randint(0, 256, (300, 1024), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.rand((300, 16), generator=g, device="cuda")
    x = torch.randn((16, 2048), generator=g, device="cuda")
    y = decode.matvec_w4(x, codes, scales)
    other = x.flip(0)
    assert torch.equal(decode.matvec_w4(other, codes, scales).flip(0), y)
    assert all(torch.equal(decode.matvec_w4(x, codes, scales), y) for _ in range(5))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("dim", [32, 128])
def test_append_non_finite_in_blocks_of_any_size(cuda, dtype, page, dim):
    g = gen(page)
    news = [1, 2 * page + 5, 3, page]
    k, v = (torch.randn((sum(news), 3, dim), generator=g, device="cuda") for _ in range(2))
    for t in (k, v):
        flat = t.view(-1)
        at = torch.randint(0, flat.numel(), (12,), generator=g, device="cuda")
        flat[at[:4]], flat[at[4:8]], flat[at[8:]] = math.nan, math.inf, -math.inf
    check_append([2, page - 3, 0, 5 * page], news, page=page, dim=dim, kv_heads=3, heads=6, k=k.to(dtype), v=v.to(dtype), dtype=dtype, rot=0)


@pytest.mark.parametrize("kv_heads,heads,n", [(8, 64, 1), (40, 40, 1), (3, 48, 130)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_append_many_heads(cuda, dtype, kv_heads, heads, n):
    check_append([0, 127, 300], [n] * 3, page=128, dim=128, kv_heads=kv_heads, heads=heads, uniform=True, dtype=dtype, seed=n)
    check_append([0, 127, 300], [n, 0, 1], page=64, dim=64, kv_heads=kv_heads, heads=heads, dtype=dtype, seed=n, rot=48)


@pytest.mark.parametrize("batch,n,kv_heads,page,dim,dtype", [(30, 40, 8, 16, 128, torch.float32), (9, 300, 12, 32, 128, torch.bfloat16),
                                                             (40, 33, 7, 16, 128, torch.float16), (3, 1000, 33, 64, 32, torch.float32)])
def test_append_blocks_that_walk_many_heads(cuda, batch, n, kv_heads, page, dim, dtype):
    check_append([(11 * b) % 40 for b in range(batch)], [n] * batch, page=page, dim=dim, kv_heads=kv_heads, heads=kv_heads, uniform=True,
                 dtype=dtype, rot=dim // 2, interleaved=batch % 2 == 0)
    check_append([(11 * b) % 40 for b in range(batch)], [n - b % 5 for b in range(batch)], page=page, dim=dim, kv_heads=kv_heads, heads=2,
                 dtype=dtype, with_q=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,page", [(32, 16), (64, 128), (128, 16), (128, 64)])
def test_attention_scales_far_apart(cuda, dtype, dim, page):
    # pages whose values' scales differ by up to 2^60 within a sequence, pages of zeros, rising and falling
    lengths = [400, 333, 17]
    need = [-(-n // page) for n in lengths]
    table, pages = page_table(need, max(need), 3)
    cache = random_cache(pages, 2, page, dim, 3)
    g = gen(4)
    cache[3].copy_(torch.ldexp(torch.ones(pages, 2, device="cuda"), torch.randint(-30, 30, (pages, 2), generator=g, device="cuda")))
    cache[3][::4] = 0
    cache[2][1::4] = 0
    top = float((cache[1].float() * cache[3][..., None, None]).abs().max())
    cu, lens = offsets([1, 2, 1]), torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q = torch.randn((4, 8, dim), generator=gen(1), device="cuda").to(dtype)
    for window in (0, 50):
        out = decode.kv_attention(q, tuple(cache), table.cuda(), lens, cu=cu.cuda(), window=window).cpu().double()
        want, _, spread = ref.attention(q, cache, table, lens, cu, None, window)
        tol = bound(dtype, dim, spread, top).expand(want.shape)
        limit = 65520.0 if dtype == torch.float16 else math.inf             # from here on fp16 rounds to infinity
        beyond = out.isinf() & (want * out.sign() + tol >= limit)
        assert (beyond | ((out - want).abs() <= tol)).all()
    assert status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,group,new", [(128, 4, 1), (128, 8, 3), (64, 16, 1), (32, 2, 2)])
def test_attention_many_splits(cuda, dtype, dim, group, new):
    check_attention([70001], [new], page=64, dim=dim, kv_heads=1, group=group, dtype=dtype, uniform=True)


@pytest.mark.parametrize("news", [[4, 4], [3, 9]])
@pytest.mark.parametrize("window", [1, 33, 1000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_attention_window_of_several_row_tiles(cuda, dtype, window, news):
    check_attention([5000, 1200], news, page=16, dim=128, kv_heads=2, group=8, dtype=dtype, window=window, uniform=len(set(news)) == 1)
    check_attention([5000, 1200], news, page=16, dim=128, kv_heads=2, group=8, dtype=dtype, window=window, max_length=5000, max_new=9)


def test_matvec_workspace_is_asked_for(cuda):
    g = gen(0)
    handle = _lib.lib()
    for rows, inner, needs in ((1, 2048, False), (9, 4096, True)):
        x = torch.randn((rows, inner), generator=g, device="cuda")
        codes = torch.randint(0, 256, (32, inner // 2), generator=g, device="cuda", dtype=torch.uint8)
        scales = torch.rand((32, inner // 128), generator=g, device="cuda")
        want = decode.matvec_w4(x, codes, scales)
        y = torch.zeros_like(want)
        args = _lib.MatvecW4Args(x=x.data_ptr(), codes=codes.data_ptr(), scales=scales.data_ptr(), y=y.data_ptr(), rows=rows,
                                 inner=inner, outer=32, stride_x=inner, stride_codes=inner // 2, stride_scales=inner // 128, stride_y=32,
                                 group=128, type=_lib.TYPE_F32, scale_type=_lib.TYPE_F32)
        size = handle.piton_b200_matvec_w4_workspace_size(C.byref(args))
        assert (size > 0) == needs
        stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
        if needs:
            scratch = torch.empty(size + 16, dtype=torch.uint8, device="cuda")
            for at, bytes_ in ((0, 0), (scratch.data_ptr(), size - 1)):
                args.workspace, args.workspace_bytes = at, bytes_
                assert handle.piton_b200_matvec_w4(C.byref(args), stream) == -6
            args.workspace, args.workspace_bytes = scratch.data_ptr() + 8, size
            assert handle.piton_b200_matvec_w4(C.byref(args), stream) == -1
            assert not bool(y.any())
            args.workspace = scratch.data_ptr()
        assert handle.piton_b200_matvec_w4(C.byref(args), stream) == 0
        assert torch.equal(y, want)
