"""How matmul_mx4 tiles a geometry (no GPU; planned for 256 CUs): every tile has columns of its own, and all columns have a tile."""
import ctypes
import random

import pytest

from xrgpu_amd import _native as nat


def plan(M, K, N, a=nat.F16, ws=1):
    v = (ctypes.c_int64 * 6)()
    assert nat.lib().xrmm_matmul_mx4_plan(M, K, N, a, ws, v) == nat.XRMM_OK
    return list(v)


def check(M, K, N, a, ws):
    t, mt, nb, ns, splits, nws = plan(M, K, N, a, ws)
    if t == 0:
        assert M <= 16 or K > 1 << 21
        return t, ns, splits
    where = (M, K, N, a, ws, t, mt, nb, ns, splits)
    assert t in (64, 128, 256) and (mt - 1) * t < M <= mt * t, where
    assert ns == 0 or (t == 256 and splits == 1), where
    wide = nb * t
    if ns:
        assert wide + 192 * (ns - 1) < N <= wide + 192 * ns, where
    else:
        assert wide - t < N <= wide, where
    assert splits >= 1 and (splits == 1) == (nws == 0) and (ws or nws == 0), where
    assert nws == 0 or nws == 4096 + mt * nb * splits * t * t * 4, where
    return t, ns, splits


@pytest.mark.parametrize("a", [nat.F16, nat.BF16, nat.U8])
def test_feed_forward_widths(a):
    mixed = 0
    for M in (256, 512, 1024, 2040, 2048, 4096, 8192):
        for N in (1024, 4096, 5120, 8192, 10240, 11008, 13824, 14336, 18944, 22016, 28672):
            for K in (512, 4096, 14336):
                mixed += check(M, K, N, a, 1)[1] > 0
                check(M, K, N, a, 0)
    assert mixed > 10


@pytest.mark.parametrize("seed", range(4))
def test_any_geometry(seed):
    rng = random.Random(seed)
    seen = set()
    for _ in range(4000):
        M, K, N = (max(1, int(2 ** rng.uniform(0, top))) for top in (14, 15, 15.5))
        if rng.random() < 0.5:  # numbers of row tiles that divide the CUs
            M = 256 * 2 ** rng.randrange(0, 7) - rng.randrange(0, 200)
        t, ns, splits = check(M, K, N, rng.choice((nat.F16, nat.BF16, nat.U8)), rng.randrange(2))
        seen.add((t, ns > 0, splits > 1))
    assert {(64, False, False), (64, False, True), (128, False, False), (128, False, True), (256, False, False), (256, True, False)} <= seen


def test_refuses():
    v = (ctypes.c_int64 * 6)()
    assert nat.lib().xrmm_matmul_mx4_plan(1, 0, 8, nat.F16, 1, v) == nat.XRMM_EINVAL
    assert nat.lib().xrmm_matmul_mx4_plan(1, 64, 8, nat.F16, 1, None) == nat.XRMM_EINVAL
