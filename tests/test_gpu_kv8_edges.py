"""GPU: attention at the edges of windows, tables and lengths; tolerances as in test_gpu_kv8_scales.py."""
import pytest

from tests.test_gpu_kv8 import Cache, ops, starts_of
from tests.test_gpu_kv8_scales import check, queries

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("page,D", [(16, 64), (32, 128), (16, 256), (64, 96)])
@pytest.mark.parametrize("counts", [[1, 1], [9, 2], [70, 40], [200, 129]])
@pytest.mark.parametrize("window", [1, 20, 100])
def test_pages_behind_the_window_may_be_gone(gpu, page, D, counts, window):
    lens = [513, 300]
    c = Cache("int8", lens, 1, D, page, seed=page)
    for b, (x, n) in enumerate(zip(lens, counts)):
        c.table[b, : max(0, x - n - window + 1) // page] = -1
    assert (c.table[:, 0] == -1).all() or counts[0] == 200
    check(c, queries(sum(counts), 2, D, "f16"), counts, window=window)


@pytest.mark.parametrize("counts", [[10, 3], [70, 200]])  # the first rows stand before position 0
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [(1 << 31) - 1, 1 << 31, (1 << 32) + 5, 1 << 62])
def test_windows_without_end(gpu, counts, causal, window):
    lens = [3, 150]
    c = Cache("int8", lens, 1, 64, 16, seed=1)
    q = queries(sum(counts), 2, 64, "f16")
    check(c, q, counts, causal=causal, window=window)
    a = ops().kv8_attention(q, **c.dev(), starts=starts_of(counts), max_new=1 << 40, causal=causal, window=window)
    assert torch.equal(a, ops().kv8_attention(q, **c.dev(), starts=starts_of(counts), causal=causal))


def test_negative_lengths_see_nothing(gpu):
    c = Cache("int8", [20, 40], 1, 64, 16, seed=2)
    q = queries(4, 2, 64, "f16")
    good = ops().kv8_attention(q, **c.dev())
    for bad in (-1, -(1 << 31)):
        d = c.dev()
        d["lengths"][0] = bad
        for kw in ({}, {"window": (1 << 31) - 1}, {"causal": False}):
            o = ops().kv8_attention(q, **d, **kw)
            assert (o[:2] == 0).all()
        assert torch.equal(ops().kv8_attention(q, **d)[2:], good[2:])


@pytest.mark.parametrize("n,D,page", [(1, 64, 256), (6, 128, 256), (150, 64, 256), (150, 256, 128)])
def test_positions_up_to_2_to_the_31(gpu, n, D, page):
    """A window at the end of the longest table gives what it gives at a short one's end, where all pages before it are gone."""
    far, pages = (0x7FFFFF00 // page) * page, 1024 // page
    c = Cache("int8", [1024], 1, D, page, seed=5, extra=0)
    q, kv = queries(n, 2, D, "f16"), queries(n, 1, D, "bf16", seed=1)
    near, there = c.dev(), c.dev()
    table = torch.full((1, far // page), -1, dtype=torch.int32, device="cuda")
    table[:, -pages:] = near["block_table"]
    there["block_table"], there["lengths"] = table, torch.tensor([far], dtype=torch.int32, device="cuda")
    out = []
    for d in (near, there):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        ops().kv8_append(kv, kv, **d, status=status)
        out.append(ops().kv8_attention(q, **d, window=300, status=status))
        assert int(status.item()) == 0
    assert torch.equal(*out)
    for name in ("k_cache", "v_cache", "k_scales", "v_scales"):
        assert torch.equal(near[name].view(torch.uint8), there[name].view(torch.uint8))


@pytest.mark.parametrize("n", [1, 20, 150])
@pytest.mark.parametrize("length", [0x7FFFFFFF, 0x7FFFFF00, 5000])
def test_lengths_past_the_table_behind_a_window(gpu, n, length):
    """Windows that begin past the table's end: nothing is left to see, and the walk ends at once."""
    c = Cache("int8", [100], 1, 64, 16, seed=6)
    d = c.dev()
    d["lengths"][0] = length
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert (ops().kv8_attention(queries(n, 2, 64, "f16"), **d, window=20, status=status) == 0).all()
    assert int(status.item()) == 55


@pytest.mark.parametrize("n", [5, 40])
def test_positions_below_0_raise_the_status_where_tokens_are_written(gpu, n):
    c = Cache("int8", [3], 1, 64, 16, seed=7)
    d = c.dev()
    q, kv = queries(n, 2, 64, "f16"), queries(n, 1, 64, "f16")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    o = ops().kv8_attention(q, **d, status=status)
    assert int(status.item()) == 0 and (o[: n - 3] == 0).all() and (o[n - 3:] != 0).any()
    ops().kv8_append(kv, kv, **d, status=status)
    assert int(status.item()) == 55
