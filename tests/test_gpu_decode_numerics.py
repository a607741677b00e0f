"""Numerics of the decode operators where operands are far apart: zero points of any byte, and what a
product or a softmax must not lose beside something much larger.

Tolerances are those of test_gpu_decode.py unless a test derives its own.
"""

import pytest
import torch

import decode_ref as ref
from piton_b200 import decode
from test_gpu_decode import EPS, ROUND, TYPES, gen

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
