"""GPU: attention over caches whose scales are anything a float32 can be.

The tolerance is that of test_gpu_kv8.py with its absolute term (2^-35 of the largest value for each token: where a weight
times its scale falls below binary16's normal range) taken from the scales that the row sees.
"""
import numpy as np
import pytest

from oracle import lowbit as LB
from tests.test_gpu_kv8 import DT, Cache, ops, starts_of

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def seen_top(c, counts, Hq, causal, window):
    """The largest value that a page visible to each row may hold: [T, Hq]."""
    H = c.vs.shape[1]
    top, first = np.zeros((sum(counts), Hq)), 0
    for b, n in enumerate(counts):
        L = int(c.lengths[b])
        for i in range(n):
            p = L - n + i
            lo, hi = max(0, p - window + 1) if window else 0, min(L, p + 1) if causal else L
            if hi > lo:
                scales = np.abs(c.vs[c.table[b, lo // c.page: (hi - 1) // c.page + 1]].astype(np.float64)).max(0)
                top[first + i] = np.repeat(scales, Hq // H)
        first += n
    return top * LB.QMAX[c.kind]


def check(c, q, counts, *, causal=True, window=0, scale=None):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    o = ops().kv8_attention(q, **c.dev(), starts=starts_of(counts), max_new=max(counts), causal=causal, window=window, scale=scale,
                            status=status)
    T, Hq, D = q.shape
    s = scale if scale is not None else D ** -0.5
    ref, av, aqk = LB.attention(q.double().cpu().numpy(), c.k, c.v, c.ks, c.vs, c.table, c.lengths, counts, c.kind, scale=s,
                                causal=causal, window=window)
    eps, n = torch.finfo(q.dtype).eps, float(max(int(c.lengths.max()), 1))
    rel = 2.0 ** -10 + 2.0 ** -21 + n * 2.0 ** -23 + 2 * (D + 4) * 2.0 ** -24 * aqk[..., None]
    top = seen_top(c, counts, Hq, causal, window)[..., None]
    tol = eps / 2 * np.abs(ref) + (1 + eps) * (rel * av + n * 2.0 ** -35 * top) + torch.finfo(q.dtype).tiny * eps
    out = o.double().cpu().numpy()
    assert np.isfinite(out).all() and int(status.item()) == 0
    worst = (np.abs(out - ref) - tol).max()
    assert worst <= 0, (worst, np.abs(out - ref).max(), np.abs(ref).max())
    return out


def queries(T, Hq, D, dt, seed=0):
    return torch.randn(T, Hq, D, generator=torch.Generator().manual_seed(seed + T)).to(DT[dt]).cuda()


ROWS = pytest.mark.parametrize("counts", [[1, 1], [5, 3], [70, 40]])  # by rows, by rows of several tokens, by tiles
KIND = pytest.mark.parametrize("kind", ["int8", "e4m3"])
HEADS = pytest.mark.parametrize("D,page", [(64, 16), (128, 64), (256, 32)])


@KIND
@HEADS
@ROWS
@pytest.mark.parametrize("e", [-118, -126, -140, 100])
def test_scales_of_any_size(gpu, kind, D, page, counts, e):
    c = Cache(kind, [150, 90], 2, D, page, seed=D + e % 7)
    c.vs[:] = np.ldexp(np.random.default_rng(e % 5).uniform(0.6, 1.9, c.vs.shape), e).astype(np.float32)
    out = check(c, queries(sum(counts), 4, D, "bf16"), counts)
    assert e == -140 or np.abs(out).max() > 0  # at 2^-140 the results vanish in bfloat16


@KIND
@HEADS
@ROWS
@pytest.mark.parametrize("signs", ["negative", "mixed", "a larger negative one", "negative keys"])
def test_scales_of_either_sign(gpu, kind, D, page, counts, signs):
    c = Cache(kind, [150, 90], 2, D, page, seed=D, scales="any")
    g = np.random.default_rng(D)
    if signs == "negative":
        c.vs *= np.float32(-1)
    elif signs == "mixed":
        c.vs *= g.choice(np.float32([-1, 1]), c.vs.shape)
        c.ks *= g.choice(np.float32([-1, 1]), c.ks.shape)
    elif signs == "negative keys":
        c.ks *= np.float32(-1)
    else:
        c.vs[c.table[:, 1]] *= np.float32(-300)
    check(c, queries(sum(counts), 4, D, "f16"), counts)


@KIND
@HEADS
@ROWS
def test_tiny_scales_before_ordinary_ones(gpu, kind, D, page, counts):
    c = Cache(kind, [300, 200], 1, D, page, seed=D)
    c.vs[c.table[:, : 128 // page]] = np.float32(2.0 ** -126)
    check(c, queries(sum(counts), 4, D, "bf16"), counts)


@ROWS
def test_appended_tiny_values(gpu, counts):
    """Values near the end of bfloat16's range, as kv8_append holds them, come back from a prompt and from single tokens."""
    c = Cache("int8", [150, 90], 2, 64, 16, fill=False)
    d = c.dev()
    x = (torch.randn(240, 2, 64, generator=torch.Generator().manual_seed(1)) * 2.0 ** -116).bfloat16().cuda()
    ops().kv8_append(x, x, **d, starts=starts_of([150, 90]))
    for name, t in (("k", "k_cache"), ("v", "v_cache")):
        setattr(c, name, d[t].view(torch.uint8).cpu().numpy())
    c.ks, c.vs = d["k_scales"].cpu().numpy(), d["v_scales"].cpu().numpy()
    assert 0 < c.vs[c.table[0]].max() < 2.0 ** -119
    out = check(c, queries(sum(counts), 4, 64, "bf16"), counts)
    assert np.abs(out).max() > 2.0 ** -124


@KIND
@HEADS
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("counts,Hq", [([1, 1], 4), ([5, 3], 4), ([70, 40], 1), ([200, 120], 4)])
def test_hidden_pages_change_nothing(gpu, kind, D, page, counts, Hq, window):
    """A value scale 2^60 times the others, where the causal mask or the window hides it from some rows or from all."""
    lens = [max(300, counts[0]), max(200, counts[1])]
    c = Cache(kind, lens, 1, D, page, seed=D)
    far = max(0, min(lens) - min(counts) - 100) // page  # behind the windows; with none, every row sees it
    c.vs[c.table[:, far]] *= np.float32(2.0 ** 60 if window else 1.0)
    last = [(x - 1) // page for x in lens]  # hidden from the rows before it
    for b in (0, 1):
        c.vs[c.table[b, last[b]]] *= np.float32(2.0 ** 60)
    check(c, queries(sum(counts), Hq, D, "bf16"), counts, window=window)


@KIND
@ROWS
def test_a_large_scale_after_a_row_changes_no_bit_of_it(gpu, kind, counts):
    c = Cache(kind, [150, 90], 2, 64, 16, seed=3)
    q = queries(sum(counts), 4, 64, "f16")
    a = ops().kv8_attention(q, **c.dev(), starts=starts_of(counts), max_new=max(counts))
    first = 0
    for n, L in zip(counts, (150, 90)):
        page = (L - 1) // 16
        hidden = min(max(0, page * 16 - (L - n)), n)  # rows at positions before the last page
        c2 = Cache(kind, [150, 90], 2, 64, 16, seed=3)
        for b, x in enumerate((150, 90)):
            c2.vs[c2.table[b, (x - 1) // 16]] *= np.float32(2.0 ** 30)
        b = ops().kv8_attention(q, **c2.dev(), starts=starts_of(counts), max_new=max(counts))
        assert torch.equal(a[first:first + hidden], b[first:first + hidden])
        first += n
