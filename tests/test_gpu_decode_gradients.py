"""The serving operators have no backward: an input that requires grad is refused, not silently cut off."""

import pytest
import torch

from piton_b200 import decode
from test_gpu_decode import gen, random_cache, tables

pytestmark = pytest.mark.gpu


def calls(leaf):
    """The operators with one input at a time replaced by leaf(input)."""
    g = gen(0)
    x = torch.randn((2, 64), generator=g, device="cuda")
    codes = torch.randint(0, 256, (8, 32), generator=g, device="cuda", dtype=torch.uint8)
    scales, bias = torch.rand((8, 1), generator=g, device="cuda"), torch.rand(8, generator=g, device="cuda")
    for args in ((leaf(x), scales, bias), (x, leaf(scales), bias), (x, scales, leaf(bias))):
        yield lambda a=args: decode.matvec_w4(a[0], codes, a[1], group=64, bias=a[2])
    q, k, v = (torch.randn((2, 1, 64), generator=g, device="cuda") for _ in range(3))
    cos, sin = tables(64, 40)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    at = torch.tensor([3, 17], dtype=torch.int32, device="cuda")
    inputs = [q, k, v, cos, sin]
    for i in range(5):
        a = [leaf(t) if i == n else t for n, t in enumerate(inputs)]
        yield lambda a=a: decode.kv_append(a[1], a[2], tuple(random_cache(4, 1, 16, 64, 0)), table, at, cos=a[3], sin=a[4], q=a[0])
    yield lambda: decode.kv_attention(leaf(q), tuple(random_cache(4, 1, 16, 64, 0)), table, at)
    for i in (2, 3):
        cache = random_cache(4, 1, 16, 64, 0)
        cache[i] = leaf(cache[i])
        yield lambda c=cache: decode.kv_attention(q, tuple(c), table, at)


def test_inputs_that_require_grad_are_refused(cuda):
    for call in calls(lambda t: t.clone().requires_grad_()):
        with pytest.raises(RuntimeError, match="backward"):
            call()
        with torch.no_grad():
            got = call()
        for t in got if isinstance(got, tuple) else (got,):
            assert not t.requires_grad
    for call in calls(lambda t: t.clone()):
        call()


def test_quantised_parameters_carry_no_gradient(cuda):
    w = torch.nn.Parameter(torch.randn((16, 64), device="cuda"))
    for zeros in (True, False):
        codes, scales, z = decode.quantize_w4(w, 32, zeros=zeros)
        assert not scales.requires_grad
        assert decode.matvec_w4(torch.ones(64, device="cuda"), codes, scales, group=32, zeros=z).shape == (16,)
