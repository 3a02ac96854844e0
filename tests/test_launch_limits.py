"""Calls whose launch would have 2^32 threads or more, of which the runtime runs a part without an error: refused before they reach a device (no GPU)."""
import ctypes

import pytest

from xrgpu_amd import _native as nat

MEM = (ctypes.c_uint8 * 4096)()
PTR = (ctypes.addressof(MEM) + 255) // 256 * 256  # never read
B, H, D = (1 << 20) + 1, 32, 64


def append(B):
    return nat.lib().xrmm_kv8_append(PTR, PTR, H * D, H * D, nat.F16, PTR, PTR, PTR, PTR, nat.I8, PTR, PTR, None, None, B, 0, B, 1, 1, 16, H, D, None)


def attention(B, shared=False, Hq=H):
    lib, own = nat.lib(), (PTR, PTR, PTR, PTR, nat.I8)
    tail = (PTR, PTR, None, None, B, 0, B, 1, 1, 16, Hq, H, D, 1.0, 1, 0, None, 0, None)
    if shared:
        return lib.xrmm_kv8_shared_attention(PTR, Hq * D, PTR, nat.F16, *own, PTR, 1, *tail)
    return lib.xrmm_kv8_attention(PTR, Hq * D, PTR, nat.F16, *own, *tail)


@pytest.mark.parametrize("call", [lambda: append(B), lambda: attention(B), lambda: attention(B, Hq=H * 17), lambda: attention(B, True)],
                         ids=["append", "attention", "attention_tile", "shared"])
def test_refused(call):
    assert call() == nat.XRMM_EDEVICE
    assert "invalid argument" in nat.last_error()


def test_a_call_of_just_fewer_is_none_of_them():
    """It gets as far as the launch, which on a machine without a device says so."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("would run on addresses that are no device's")
    assert attention((1 << 20) - 1) == nat.XRMM_EDEVICE and "invalid argument" not in nat.last_error()
