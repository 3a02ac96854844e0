"""Refusals of the MX4 and kv8 entry points: argument checks that reach no device (no GPU)."""
import ctypes

import pytest
import torch

from xrgpu_amd import _native as nat
from xrgpu_amd import ops

P16 = (ctypes.c_uint8 * 64)()
PTR = (ctypes.addressof(P16) + 15) // 16 * 16  # a 16-byte aligned address that is never read


def quant(x=PTR, codes=PTR, scales=PTR, rows=0, K=64, dtype=nat.F16):
    return nat.lib().xrmm_mx4_quantize(x, codes, scales, rows, K, dtype, None)


def mx4(A=PTR, As=None, a=nat.F16, B=PTR, S=PTR, bias=None, Y=PTR, o=nat.F16, M=0, K=64, N=8, ws=None, nws=0):
    return nat.lib().xrmm_matmul_mx4(A, As, a, B, S, bias, Y, o, M, K, N, ws, nws, None)


def append(k=PTR, ks=128, dtype=nat.F16, cache=PTR, cd=nat.I8, table=PTR, starts=None, rows=0, max_new=0, B=1, W=1, pages=1,
           page=16, H=1, D=64, scales=PTR):
    return nat.lib().xrmm_kv8_append(k, k, ks, ks, dtype, cache, cache, scales, scales, cd, table, table, starts, None, rows,
                                     max_new, B, W, pages, page, H, D, None)


def attend(q=PTR, qs=128, dtype=nat.F16, cd=nat.I8, rows=0, B=1, W=1, page=16, Hq=2, H=1, D=64, scale=1.0, window=0, ws=None):
    return nat.lib().xrmm_kv8_attention(q, qs, PTR, dtype, PTR, PTR, PTR, PTR, cd, PTR, PTR, None, None, rows, 0, B, W, 1,
                                        page, Hq, H, D, scale, 1, window, ws, 0, None)


@pytest.mark.parametrize("call,kw,msg", [
    (quant, dict(dtype=nat.I32), "x must be"), (quant, dict(K=0), "K must be positive"),
    (quant, dict(K=(1 << 23) + 1), "2^23"), (quant, dict(rows=-1), "rows"), (quant, dict(rows=1, x=None), "null"),
    (quant, dict(codes=PTR + 1), "aligned"),
    (mx4, dict(a=nat.F32), "A must be"), (mx4, dict(o=nat.I8), "output"), (mx4, dict(K=0), "K must be"),
    (mx4, dict(N=0), "N must be"), (mx4, dict(M=-1), "M must be"), (mx4, dict(M=1, As=PTR), "A_scales"),
    (mx4, dict(M=1, a=nat.U8), "A_scales"), (mx4, dict(M=1, B=None), "null"), (mx4, dict(M=1, B=PTR + 8), "16-byte"),
    (mx4, dict(M=1, a=nat.U8, As=PTR, A=PTR + 4), "16-byte"), (mx4, dict(M=1, Y=PTR + 1), "elements"),
    (mx4, dict(M=1, ws=PTR + 16 if PTR % 256 == 0 else PTR // 256 * 256 + 16), "256-byte"),
    (append, dict(dtype=nat.I8), "k and v"), (append, dict(cd=nat.U8), "int8 or float8"), (append, dict(D=80), "head size"),
    (append, dict(page=48), "page size"), (append, dict(page=8), "page size"), (append, dict(page=512), "page size"),
    (append, dict(H=0), "pages and heads"), (append, dict(rows=3, B=2), "need starts"),
    (append, dict(rows=1, B=0), "without sequences"), (append, dict(rows=2, ks=32), "strides"),
    (append, dict(rows=1, cache=None), "null"), (append, dict(rows=1, cache=PTR + 8), "16-byte"),
    (append, dict(rows=1, k=PTR + 1), "elements"), (append, dict(W=1 << 30), "2^31 tokens"),
    (attend, dict(dtype=nat.F32), "q must be"), (attend, dict(Hq=3, H=2), "multiple"), (attend, dict(window=-1), "window"),
    (attend, dict(scale=float("nan")), "scale"), (attend, dict(scale=float("inf")), "scale"),
    (attend, dict(rows=2, qs=64), "stride"), (attend, dict(rows=1, q=PTR + 1), "elements"), (attend, dict(D=32), "head size"),
    (attend, dict(rows=2, B=1, Hq=1 << 30), "query rows"),
])
def test_c_entry_refuses(call, kw, msg):
    assert call(**kw) == nat.XRMM_EINVAL
    assert msg in nat.last_error()


@pytest.mark.parametrize("call", [quant, mx4, append, attend])
def test_empty_calls_are_ok_without_a_device(call):
    assert call() == nat.XRMM_OK and nat.last_error() == ""


def u8(*s):
    return torch.zeros(s, dtype=torch.uint8)


H16 = torch.float16


@pytest.mark.parametrize("f,msg", [
    (lambda: ops.mx4_quantize(torch.zeros(3, 4, dtype=torch.int32)), "float32, float16 or bfloat16"),
    (lambda: ops.mx4_quantize(torch.zeros(3, 0)), "K positive"),
    (lambda: ops.mx4_quantize(torch.zeros(3, 4)), "on the GPU"),
    (lambda: ops.matmul_mx4(torch.zeros(1, 64, dtype=H16), u8(8, 2, 8), u8(8, 2)), "B must be"),
    (lambda: ops.matmul_mx4(torch.zeros(1, 64, dtype=H16), u8(8, 2, 16), u8(8, 3)), "scales must be"),
    (lambda: ops.matmul_mx4(torch.zeros(1, 65, dtype=H16), u8(8, 2, 16), u8(8, 2)), "blocks of 32"),
    (lambda: ops.matmul_mx4(torch.zeros(1, 64), u8(8, 2, 16), u8(8, 2)), "A must be float16"),
    (lambda: ops.matmul_mx4(u8(1, 2, 16), u8(8, 2, 16), u8(8, 2)), "need A_scales"),
    (lambda: ops.matmul_mx4(u8(1, 3, 16), u8(8, 2, 16), u8(8, 2), A_scales=u8(1, 3)), "A must be uint8"),
    (lambda: ops.matmul_mx4(u8(1, 2, 16), u8(8, 2, 16), u8(8, 2), A_scales=u8(1, 3)), "A_scales must be"),
    (lambda: ops.matmul_mx4(u8(1, 2, 16), u8(8, 2, 16), u8(8, 2), A_scales=u8(1, 2), out_dtype=torch.int8), "out_dtype"),
    (lambda: ops.matmul_mx4(torch.zeros(1, 64, dtype=H16), u8(8, 2, 16), u8(8, 2), out_dtype=torch.float32), "A's dtype"),
    (lambda: ops.matmul_mx4(torch.zeros(1, 64, dtype=H16), u8(8, 2, 16), u8(8, 2), torch.zeros(8)), "bias"),
    (lambda: ops.matmul_mx4(torch.zeros(1, 64, dtype=H16), u8(8, 2, 16), u8(8, 2), out=torch.zeros(1, 7, dtype=H16)), "out must"),
    (lambda: ops.matmul_mx4(torch.zeros(1, 64, dtype=H16), u8(8, 2, 16), u8(8, 2)), "on the GPU"),
])
def test_mx4_front_refuses(f, msg):
    with pytest.raises(nat.XrmmInvalid, match=msg):
        f()


def cache(P=2, H=2, page=16, D=64, B=1, W=2, dt=torch.int8):
    c = torch.zeros(P, H, page, D, dtype=torch.int8).view(dt)
    return dict(k_cache=c, v_cache=c.clone(), k_scales=torch.ones(P, H), v_scales=torch.ones(P, H),
                block_table=torch.zeros(B, W, dtype=torch.int32), lengths=torch.ones(B, dtype=torch.int32))


@pytest.mark.parametrize("change,msg", [
    (dict(k_cache=torch.zeros(2, 2, 16, 64)), "int8 or float8"),
    (dict(v_cache=torch.zeros(2, 2, 16, 96, dtype=torch.int8)), "share a shape"),
    (dict(k_scales=torch.ones(2, 3)), "k_scales"), (dict(v_scales=torch.ones(2, 2, dtype=H16)), "v_scales"),
    (dict(lengths=torch.ones(1, dtype=torch.int64)), "lengths"),
    (dict(block_table=torch.zeros(2, 2, dtype=torch.int32)), "block_table"),
    (dict(starts=torch.zeros(3, dtype=torch.int32)), "starts"), (dict(status=torch.zeros(1)), "status"),
])
def test_kv8_front_refuses_caches(change, msg):
    kw = {**cache(), **change}
    x = torch.zeros(1, 2, 64, dtype=H16)
    with pytest.raises(nat.XrmmInvalid, match=msg):
        ops.kv8_append(x, x, **kw)
    with pytest.raises(nat.XrmmInvalid, match=msg):
        ops.kv8_attention(x, **kw)


def test_kv8_front_refuses_tokens():
    x = torch.zeros(2, 2, 64, dtype=H16)
    for k, v, msg in ((x.int(), x.int(), "float32, float16 or bfloat16"), (x, x.float(), "both"), (x, x[:1], "same tokens"),
                      (x[:, :1], x[:, :1], r"\[tokens, 2, 64\]"), (x.transpose(1, 2).contiguous().transpose(1, 2), x, "contiguous"),
                      (x[:1].expand(2, 2, 64), x, "overlap"), (x, x, "on the GPU")):
        with pytest.raises(nat.XrmmInvalid, match=msg):
            ops.kv8_append(k, v, **cache())
    for q, msg in ((x.float(), "q must be"), (torch.zeros(2, 3, 64, dtype=H16), "multiple"),
                   (torch.zeros(2, 2, 96, dtype=H16), r"\[tokens, 2, 64\]"), (x, "on the GPU")):
        with pytest.raises(nat.XrmmInvalid, match=msg):
            ops.kv8_attention(q, **cache())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.int8])
def test_mx4_geometry_calls_refuse_other_types(dtype):
    for f in (ops.matmul_mx4_workspace_bytes, ops.matmul_mx4_kernel):
        with pytest.raises(nat.XrmmInvalid, match="dtype must be"):
            f(40, 4096, 64, dtype)


def test_kv8_attention_kernel_names_and_refuses():
    kw = dict(batch=1, table_width=4, page_size=64)
    assert ops.kv8_attention_kernel(1, 8, 2, 128, **kw) == "kv8_rows"
    assert ops.kv8_attention_kernel(200, 64, 8, 128, **kw) == "kv8_tile"
    with pytest.raises(nat.XrmmInvalid, match="head size"):
        ops.kv8_attention_kernel(1, 8, 2, 80, **kw)
