"""GPU: attention at the edges of windows, tables and lengths; tolerances as in test_gpu_kv8_scales.py."""
import pytest

from tests.test_gpu_kv8 import Cache, ops, starts_of
from tests.test_gpu_kv8_scales import check, kernel_of, queries

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("page,D", [(16, 64), (32, 128), (16, 256), (64, 96)])
@pytest.mark.parametrize("counts,Hq,Hkv,kernel", [([1, 1], 2, 1, "kv8_rows"), ([9, 2], 2, 1, "kv8_rows"), ([70, 40], 2, 1, "kv8_rows"),
                                                  ([150, 90], 64, 8, "kv8_tile")])
@pytest.mark.parametrize("window", [1, 20, 100])
def test_pages_behind_the_window_may_be_gone(gpu, page, D, counts, Hq, Hkv, kernel, window):
    lens = [513, 300]
    c = Cache("int8", lens, Hkv, D, page, seed=page)
    for b, (x, n) in enumerate(zip(lens, counts)):
        c.table[b, : max(0, x - n - window + 1) // page] = -1
    assert (c.table[:, 0] == -1).all()
    check(c, queries(sum(counts), Hq, D, "f16"), counts, window=window, kernel=kernel)


@pytest.mark.parametrize("counts,Hq,Hkv,kernel", [([10, 3], 2, 1, "kv8_rows"), ([70, 200], 2, 1, "kv8_rows"), ([70, 200], 32, 8, "kv8_tile")])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [(1 << 31) - 1, 1 << 31, (1 << 32) + 5, 1 << 62])
def test_windows_without_end(gpu, counts, Hq, Hkv, kernel, causal, window):
    """The first rows stand before position 0."""
    lens = [3, 150]
    c = Cache("int8", lens, Hkv, 64, 16, seed=1)
    q = queries(sum(counts), Hq, 64, "f16")
    check(c, q, counts, causal=causal, window=window, kernel=kernel)
    a = ops().kv8_attention(q, **c.dev(), starts=starts_of(counts), max_new=1 << 40, causal=causal, window=window)
    assert torch.equal(a, ops().kv8_attention(q, **c.dev(), starts=starts_of(counts), causal=causal))


@pytest.mark.parametrize("n,Hq,Hkv,kernel", [(2, 2, 1, "kv8_rows"), (200, 32, 8, "kv8_tile")])
def test_negative_lengths_see_nothing(gpu, n, Hq, Hkv, kernel):
    c = Cache("int8", [20, 40], Hkv, 64, 16, seed=2)
    q = queries(2 * n, Hq, 64, "f16")
    assert kernel_of(c, q, [n, n], ragged=False) == kernel
    good = ops().kv8_attention(q, **c.dev())
    for bad in (-1, -(1 << 31)):
        d = c.dev()
        d["lengths"][0] = bad
        for kw in ({}, {"window": (1 << 31) - 1}, {"causal": False}):
            o = ops().kv8_attention(q, **d, **kw)
            assert (o[:n] == 0).all()
        assert torch.equal(ops().kv8_attention(q, **d)[n:], good[n:])


@pytest.mark.parametrize("n,D,page,Hq,Hkv,kernel", [(1, 64, 256, 2, 1, "kv8_rows"), (6, 128, 256, 2, 1, "kv8_rows"), (150, 64, 256, 2, 1, "kv8_rows"),
                                                    (300, 64, 256, 64, 8, "kv8_tile"), (300, 256, 128, 64, 8, "kv8_tile")])
def test_positions_up_to_2_to_the_31(gpu, n, D, page, Hq, Hkv, kernel):
    """A window at the end of the longest table gives what it gives at a short one's end, where all pages before it are gone."""
    far, pages = (0x7FFFFF00 // page) * page, 1024 // page
    c = Cache("int8", [1024], Hkv, D, page, seed=5, extra=0)
    q, kv = queries(n, Hq, D, "f16"), queries(n, Hkv, D, "bf16", seed=1)
    assert kernel_of(c, q, [n], window=300, ragged=False) == kernel
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


@pytest.mark.parametrize("n,Hq,Hkv,kernel", [(1, 2, 1, "kv8_rows"), (20, 2, 1, "kv8_rows"), (150, 2, 1, "kv8_rows"), (400, 64, 8, "kv8_tile")])
@pytest.mark.parametrize("length", [0x7FFFFFFF, 0x7FFFFF00, 5000])
def test_lengths_past_the_table_behind_a_window(gpu, n, Hq, Hkv, kernel, length):
    """Windows that begin past the table's end: nothing is left to see, and the walk ends at once."""
    c = Cache("int8", [100], Hkv, 64, 16, seed=6)
    d = c.dev()
    assert kernel_of(c, queries(n, Hq, 64, "f16"), [n], window=20, ragged=False) == kernel
    d["lengths"][0] = length
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert (ops().kv8_attention(queries(n, Hq, 64, "f16"), **d, window=20, status=status) == 0).all()
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
