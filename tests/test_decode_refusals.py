"""What the decode operators refuse, and their 4-bit packing; no GPU needed."""

import ctypes as C

import pytest
import torch

from piton_b200 import decode
from piton_b200.runtime.cuda import _lib


def append_args(**kw):
    a = _lib.KvAppendArgs()
    fields = dict(k=4096, v=4096, k_codes=4096, v_codes=4096, k_scale=4096, v_scale=4096, table=4096, starts=4096, lengths=8192,
                  batch=2, tokens=0, kv_heads=2, head_dim=64, page_size=16, num_pages=4, table_width=2, table_stride=2)
    for name, value in {**fields, **kw}.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change,code", [
    (dict(flags=1), _lib.EINVAL), (dict(type=3), _lib.EINVAL), (dict(type=-1), _lib.EINVAL), (dict(batch=-1), _lib.EINVAL),
    (dict(tokens=3), _lib.EINVAL), (dict(kv_heads=0), _lib.EINVAL), (dict(head_dim=48), _lib.ENOTSUP),
    (dict(head_dim=256), _lib.ENOTSUP), (dict(page_size=8), _lib.ENOTSUP), (dict(page_size=17), _lib.ENOTSUP),
    (dict(rot_dim=66), _lib.EINVAL), (dict(rot_dim=3), _lib.EINVAL), (dict(lengths=4096), _lib.EINVAL),
    (dict(tokens=2, k_codes=4104), _lib.EINVAL), (dict(tokens=2, rot_dim=32), _lib.EINVAL),
    (dict(tokens=2, q_heads=2), _lib.EINVAL), (dict(tokens=2, table=0), _lib.EINVAL), (dict(starts=0), _lib.EINVAL),
    (dict(tokens=1 << 33, cu=4096), _lib.EINVAL), (dict(num_pages=1 << 33), _lib.EINVAL),
])
def test_append_refuses(change, code):
    lib = _lib.lib()
    assert lib.piton_b200_kv_append(C.byref(append_args(**change)), None) == code
    assert lib.piton_b200_last_error()


def attention_args(**kw):
    a = _lib.KvAttentionArgs()
    fields = dict(q=4096, out=4096, k_codes=4096, v_codes=4096, k_scale=4096, v_scale=4096, table=4096, lengths=4096, batch=2,
                  tokens=2, q_heads=4, kv_heads=2, head_dim=64, page_size=16, num_pages=4, table_width=2, table_stride=2)
    for name, value in {**fields, **kw}.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change,code", [
    (dict(flags=1), _lib.EINVAL), (dict(type=7), _lib.EINVAL), (dict(q_heads=5), _lib.EINVAL), (dict(q_heads=0), _lib.EINVAL),
    (dict(kv_heads=0), _lib.EINVAL), (dict(tokens=3), _lib.EINVAL), (dict(head_dim=16), _lib.ENOTSUP),
    (dict(page_size=256), _lib.ENOTSUP), (dict(window=-1), _lib.EINVAL), (dict(max_length=-1), _lib.EINVAL), (dict(q=0), _lib.EINVAL),
    (dict(lengths=0), _lib.EINVAL), (dict(v_codes=4097), _lib.EINVAL), (dict(batch=1 << 20, tokens=1 << 20), _lib.EINVAL),
])
def test_attention_refuses(change, code):
    lib = _lib.lib()
    a = attention_args(**change)
    assert lib.piton_b200_kv_attention(C.byref(a), None) == code
    assert lib.piton_b200_last_error()


def test_empty_calls_are_ok_without_a_gpu():
    lib = _lib.lib()
    assert lib.piton_b200_kv_append(C.byref(append_args(batch=0)), None) == _lib.OK
    assert lib.piton_b200_kv_attention(C.byref(attention_args(batch=0, tokens=0)), None) == _lib.OK
    assert lib.piton_b200_kv_attention(C.byref(attention_args(tokens=0)), None) == _lib.OK
    m = _lib.MatvecW4Args(group=32)
    assert lib.piton_b200_matvec_w4(C.byref(m), None) == _lib.OK


def test_null_args():
    lib = _lib.lib()
    assert lib.piton_b200_kv_append(None, None) == _lib.EINVAL
    assert lib.piton_b200_kv_attention(None, None) == _lib.EINVAL
    assert lib.piton_b200_kv_attention_workspace_size(None) == 0
    assert lib.piton_b200_matvec_w4(None, None) == _lib.EINVAL


@pytest.mark.parametrize("change,code", [
    (dict(flags=1), _lib.EINVAL), (dict(type=3), _lib.EINVAL), (dict(scale_type=3), _lib.EINVAL), (dict(group=16), _lib.ENOTSUP),
    (dict(group=0), _lib.ENOTSUP), (dict(rows=-1), _lib.EINVAL), (dict(inner=-1), _lib.EINVAL), (dict(y=0), _lib.EINVAL),
    (dict(x=0), _lib.EINVAL), (dict(rows=1 << 20), _lib.EINVAL), (dict(outer=1 << 32), _lib.EINVAL),
])
def test_matvec_refuses(change, code):
    a = _lib.MatvecW4Args()
    fields = dict(x=4096, codes=4096, scales=4096, y=4096, rows=1, inner=64, outer=16, stride_codes=32, stride_scales=2, group=32)
    for name, value in {**fields, **change}.items():
        setattr(a, name, value)
    assert _lib.lib().piton_b200_matvec_w4(C.byref(a), None) == code


def test_tensors_on_the_cpu_are_refused():
    x = torch.zeros((2, 2, 64))
    t = torch.zeros((2, 2), dtype=torch.int32)
    cache = (torch.zeros((4, 2, 16, 64), dtype=torch.float8_e4m3fn),) * 2 + (torch.zeros((4, 2)),) * 2
    for call in (lambda: decode.kv_append(x, x, cache, t, t[0]), lambda: decode.kv_attention(x, cache, t, t[0]),
                 lambda: decode.matvec_w4(x[0], torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((4, 2)), group=32)):
        with pytest.raises(TypeError):
            call()


@pytest.mark.gpu
class TestOnTheGpu:
    def setup_method(self):
        self.cache = decode.PagedKV.empty(4, 2, 64, 16)
        self.table = torch.zeros((2, 2), dtype=torch.int32, device="cuda")
        self.ints = torch.zeros(2, dtype=torch.int32, device="cuda")
        self.x = torch.zeros((2, 2, 64), device="cuda")
        self.w = (torch.zeros((4, 32), dtype=torch.uint8, device="cuda"), torch.zeros((4, 2), device="cuda"))

    def test_append(self):
        c, t, i, x = self.cache, self.table, self.ints, self.x
        half = torch.zeros((5, 16), device="cuda")
        for error, call in [
            (TypeError, lambda: decode.kv_append(x, x.half(), c, t, i)),
            (TypeError, lambda: decode.kv_append(x.double(), x, c, t, i)),
            (TypeError, lambda: decode.kv_append(x, x, c, t.long(), i)),
            (TypeError, lambda: decode.kv_append(x, x, c, t, i.long())),
            (TypeError, lambda: decode.kv_append(x, x, c, t, i.cpu())),
            (TypeError, lambda: decode.kv_append(x, x, (c.k.float(), c.v, c.k_scale, c.v_scale), t, i)),
            (TypeError, lambda: decode.kv_append(x, x, c, t, i, cos=half.half(), sin=half)),
            (TypeError, lambda: decode.kv_append(x, x, c, t, i, q=x.bfloat16())),
            (ValueError, lambda: decode.kv_append(x[:, :1], x, c, t, i)),
            (ValueError, lambda: decode.kv_append(x, x[:1], c, t, i)),
            (ValueError, lambda: decode.kv_append(x[..., ::2], x[..., ::2], c, t, i)),
            (ValueError, lambda: decode.kv_append(x[:1], x[:1], c, t, i)),
            (ValueError, lambda: decode.kv_append(x, x, c, t, i[:1])),
            (ValueError, lambda: decode.kv_append(x, x, c, t, i, cu=i)),
            (ValueError, lambda: decode.kv_append(x, x, c, t[0], i)),
            (ValueError, lambda: decode.kv_append(x, x, c, t, i, cos=half)),
            (ValueError, lambda: decode.kv_append(x, x, c, t, i, cos=half, sin=half[:4])),
            (ValueError, lambda: decode.kv_append(x, x, c, t, i, cos=half.repeat(1, 3), sin=half.repeat(1, 3))),
            (ValueError, lambda: decode.kv_append(x, x, c, t, i, q=x[:1])),
            (ValueError, lambda: decode.kv_append(x, x, (c.k.transpose(0, 2).contiguous().transpose(0, 2), c.v, c.k_scale, c.v_scale),
                                                  t, i)),
            (ValueError, lambda: decode.kv_append(x, x, (c.k, c.v, c.k_scale[:2], c.v_scale), t, i)),
            (NotImplementedError, lambda: decode.kv_append(x, x, decode.PagedKV.empty(4, 2, 64, 8), t, i)),
        ]:
            with pytest.raises(error):
                call()

    def test_attention(self):
        c, t, i, x = self.cache, self.table, self.ints, self.x
        for error, call in [
            (TypeError, lambda: decode.kv_attention(x.double(), c, t, i)),
            (TypeError, lambda: decode.kv_attention(x, c, t, i.float())),
            (ValueError, lambda: decode.kv_attention(x[:, :1].expand(2, 3, 64), c, t, i)),
            (ValueError, lambda: decode.kv_attention(x[..., :32], c, t, i)),
            (ValueError, lambda: decode.kv_attention(x[:1], c, t, i)),
            (ValueError, lambda: decode.kv_attention(x, c, t, i[:1])),
            (ValueError, lambda: decode.kv_attention(x, c, t, i, window=-1)),
            (ValueError, lambda: decode.kv_attention(x, c, t, i, cu=i)),
            (NotImplementedError, lambda: decode.kv_attention(x[..., :16].contiguous(), decode.PagedKV.empty(4, 2, 16, 16), t, i)),
        ]:
            with pytest.raises(error):
                call()

    def test_matvec(self):
        codes, scales = self.w
        x = torch.zeros((3, 64), device="cuda")
        for error, call in [
            (TypeError, lambda: decode.matvec_w4(x.double(), codes, scales, group=32)),
            (TypeError, lambda: decode.matvec_w4(x, codes.int(), scales, group=32)),
            (TypeError, lambda: decode.matvec_w4(x, codes, scales.double(), group=32)),
            (TypeError, lambda: decode.matvec_w4(x, codes, scales, group=32, zeros=scales)),
            (TypeError, lambda: decode.matvec_w4(x, codes, scales, group=32, bias=torch.zeros(4, device="cuda").half())),
            (ValueError, lambda: decode.matvec_w4(x, codes, scales, group=64)),
            (ValueError, lambda: decode.matvec_w4(x[:, :63], codes[:, :31], scales, group=32)),
            (ValueError, lambda: decode.matvec_w4(x[:, ::2], codes[:, :16], scales[:, :1], group=32)),
            (ValueError, lambda: decode.matvec_w4(x, codes, scales, group=32, bias=torch.zeros(3, device="cuda"))),
            (ValueError, lambda: decode.matvec_w4(x[None], codes, scales, group=32)),
            (NotImplementedError, lambda: decode.matvec_w4(x, codes, scales, group=16)),
        ]:
            with pytest.raises(error):
                call()


@pytest.mark.parametrize("zeros", [True, False])
@pytest.mark.parametrize("inner", [1, 31, 64, 100])
def test_quantize_w4(zeros, inner):
    w = torch.randn((5, inner), generator=torch.Generator().manual_seed(inner))
    w[2] = 0
    codes, scales, z = decode.quantize_w4(w, 32, zeros=zeros)
    groups = -(-inner // 32)
    assert codes.shape == (5, (inner + 1) // 2) and scales.shape == (5, groups)
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(1)[:, :inner].float()
    at = torch.arange(inner) // 32
    step = scales[:, at]
    back = (n - (z.float()[:, at] if zeros else 8.0)) * step
    assert ((back - w).abs() <= step * (1.0 if zeros else 0.5) + 1e-6).all()
