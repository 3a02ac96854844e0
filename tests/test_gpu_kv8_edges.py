"""GPU: attention at the edges of windows, tables and lengths; tolerances as in test_gpu_kv8_scales.py."""
import numpy as np
import pytest

from tests.test_gpu_kv8 import Cache
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
