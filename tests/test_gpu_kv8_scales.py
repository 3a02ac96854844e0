"""GPU: attention over caches whose scales are anything a float32 can be, on both kernels.

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
                pages = c.table[b, lo // c.page: (hi - 1) // c.page + 1]
                pages = pages[(pages >= 0) & (pages < c.vs.shape[0])]
                scales = np.abs(c.vs[pages].astype(np.float64)).max(0, initial=0)
                top[first + i] = np.repeat(scales, Hq // H)
        first += n
    return top * LB.QMAX[c.kind]


def kernel_of(c, q, counts, *, causal=True, window=0, max_new=None, ragged=True):
    return ops().kv8_attention_kernel(q.shape[0], q.shape[1], c.k.shape[1], q.shape[2], batch=len(counts), table_width=c.table.shape[1],
                                      page_size=c.page, max_new=max(counts) if max_new is None else max_new, ragged=ragged,
                                      causal=causal, window=window)


def check(c, q, counts, *, causal=True, window=0, scale=None, status=0, kernel=None, out=None, d=None, got=None,
          weights=2.0 ** -10, **kw):
    if kernel is not None:
        assert kernel_of(c, q, counts, causal=causal, window=window) == kernel
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    o = got if got is not None else ops().kv8_attention(q, **(d or c.dev()), starts=starts_of(counts), max_new=max(counts), causal=causal,
                                                        window=window, scale=scale, status=word, out=out, **kw)
    T, Hq, D = q.shape
    assert o.dtype == q.dtype and o.shape == q.shape
    s = scale if scale is not None else D ** -0.5
    ref, av, aqk = LB.attention_of_all(q.double().cpu().numpy(), c.k, c.v, c.ks, c.vs, c.table, c.lengths, counts, c.kind, scale=s,
                                       causal=causal, window=window)
    eps, n = torch.finfo(q.dtype).eps, float(max(int(c.lengths.max()), 1))
    rel = weights + 2.0 ** -21 + n * 2.0 ** -23 + 2 * (D + 4) * 2.0 ** -24 * aqk[..., None]
    top = seen_top(c, counts, Hq, causal, window)[..., None]
    tol = eps / 2 * np.abs(ref) + (1 + eps) * (rel * av + n * 2.0 ** -35 * top) + torch.finfo(q.dtype).tiny * eps
    out = o.double().cpu().numpy()
    assert np.isfinite(out).all() and (got is not None or int(word.item()) == status)
    worst = (np.abs(out - ref) - tol).max()
    assert worst <= 0, (worst, np.abs(out - ref).max(), np.abs(ref).max())
    return o


def queries(T, Hq, D, dt, seed=0):
    return torch.randn(T, Hq, D, generator=torch.Generator().manual_seed(seed + T)).to(DT[dt]).cuda()


# rows of two sequences (of 150 and 90 tokens here), query and key heads, the kernel that takes them
SHAPES = [([1, 1], 4, 2, "kv8_rows"), ([5, 3], 4, 2, "kv8_rows"), ([70, 40], 4, 2, "kv8_rows"), ([150, 90], 32, 8, "kv8_tile")]
SHAPE = pytest.mark.parametrize("counts,Hq,Hkv,kernel", SHAPES)
KIND = pytest.mark.parametrize("kind", ["int8", "e4m3"])
HEADS = pytest.mark.parametrize("D,page", [(64, 16), (128, 64), (256, 32), (96, 128)])


@KIND
@HEADS
@SHAPE
@pytest.mark.parametrize("e", [-118, -126, -140, 100])
def test_scales_of_any_size(gpu, kind, D, page, counts, Hq, Hkv, kernel, e):
    c = Cache(kind, [150, 90], Hkv, D, page, seed=D + e % 7)
    c.vs[:] = np.ldexp(np.random.default_rng(e % 5).uniform(0.6, 1.9, c.vs.shape), e).astype(np.float32)
    out = check(c, queries(sum(counts), Hq, D, "bf16"), counts, kernel=kernel)
    assert e == -140 or out.any()  # at 2^-140 the results vanish in bfloat16


@KIND
@HEADS
@SHAPE
@pytest.mark.parametrize("signs", ["negative", "mixed", "a larger negative one", "negative keys"])
def test_scales_of_either_sign(gpu, kind, D, page, counts, Hq, Hkv, kernel, signs):
    c = Cache(kind, [150, 90], Hkv, D, page, seed=D, scales="any")
    g = np.random.default_rng(D)
    if signs == "negative":
        c.vs *= np.float32(-1)
    elif signs == "mixed":
        c.vs *= g.choice(np.float32([-1, 1]), c.vs.shape)
        c.ks *= g.choice(np.float32([-1, 1]), c.ks.shape)
    elif signs == "negative keys":
        c.ks *= np.float32(-1)
    else:
        c.vs[c.table[:, min(1, 90 // page)]] *= np.float32(-300)
    check(c, queries(sum(counts), Hq, D, "f16"), counts, kernel=kernel)


@KIND
@HEADS
@SHAPE
def test_tiny_scales_before_ordinary_ones(gpu, kind, D, page, counts, Hq, Hkv, kernel):
    c = Cache(kind, [300, 200], Hkv, D, page, seed=D)
    c.vs[c.table[:, : 128 // page]] = np.float32(2.0 ** -126)
    if kernel == "kv8_tile":  # rows that see tiny ones alone, too
        counts = [280, 200]
    check(c, queries(sum(counts), Hq, D, "bf16"), counts, kernel=kernel)


@SHAPE
def test_appended_tiny_values(gpu, counts, Hq, Hkv, kernel):
    """Values near the end of bfloat16's range, as kv8_append holds them, come back from a prompt and from single tokens."""
    c = Cache("int8", [150, 90], Hkv, 64, 16, fill=False)
    d = c.dev()
    x = (torch.randn(240, Hkv, 64, generator=torch.Generator().manual_seed(1)) * 2.0 ** -116).bfloat16().cuda()
    ops().kv8_append(x, x, **d, starts=starts_of([150, 90]))
    for name, t in (("k", "k_cache"), ("v", "v_cache")):
        setattr(c, name, d[t].view(torch.uint8).cpu().numpy())
    c.ks, c.vs = d["k_scales"].cpu().numpy(), d["v_scales"].cpu().numpy()
    assert 0 < c.vs[c.table[0]].max() < 2.0 ** -119
    out = check(c, queries(sum(counts), Hq, 64, "bf16"), counts, kernel=kernel)
    assert out.abs().max() > 2.0 ** -124


@KIND
@HEADS
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("counts,Hq,Hkv,kernel", [([1, 1], 4, 1, "kv8_rows"), ([5, 3], 4, 1, "kv8_rows"), ([70, 40], 1, 1, "kv8_rows"),
                                                  ([200, 150], 32, 8, "kv8_tile")])
def test_hidden_pages_change_nothing(gpu, kind, D, page, counts, Hq, Hkv, kernel, window):
    """A value scale 2^60 times the others, where the causal mask or the window hides it from some rows or from all."""
    lens = [300, 200]
    if kernel == "kv8_tile" and window:
        counts, Hq = [300, 200], 64  # a window's few tokens are cheap by rows
    c = Cache(kind, lens, Hkv, D, page, seed=D)
    # behind the windows of the last rows (with none, every row sees it), and the last page, which the rows before do not see
    far = max(0, min(lens) - min(counts) - 100) // page
    c.vs[c.table[:, far]] *= np.float32(2.0 ** 60 if window else 1.0)
    for b in (0, 1):
        c.vs[c.table[b, (lens[b] - 1) // page]] *= np.float32(2.0 ** 60)
    check(c, queries(sum(counts), Hq, D, "bf16"), counts, window=window, kernel=kernel)


@KIND
@pytest.mark.parametrize("counts", [[5, 3], [70, 40]])
def test_a_large_scale_after_a_row_changes_no_bit_of_it(gpu, kind, counts):
    """By rows; tiles choose their arithmetic for 32 rows together, which is within the tolerance above."""
    page = 16
    c = Cache(kind, [150, 90], 2, 64, page, seed=3)
    q = queries(sum(counts), 4, 64, "f16")
    assert kernel_of(c, q, counts) == "kv8_rows"
    kw = dict(starts=starts_of(counts), max_new=max(counts))
    a = ops().kv8_attention(q, **c.dev(), **kw)
    for b, x in enumerate((150, 90)):
        c.vs[c.table[b, (x - 1) // page]] *= np.float32(2.0 ** 30)
    b = ops().kv8_attention(q, **c.dev(), **kw)
    first = 0
    for n, L in zip(counts, (150, 90)):
        hidden = min(max(0, (L - 1) // page * page - (L - n)), n)  # rows at positions before the last page
        assert torch.equal(a[first:first + hidden], b[first:first + hidden])
        first += n


@KIND
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("lens,counts,Hq,Hkv,D,page,window", [
    ([7, 1, 40], [1, 1, 1], 8, 2, 64, 16, 0), ([200], [1], 32, 8, 64, 16, 0), ([3000, 500], [1, 1], 8, 1, 128, 64, 0), ([64], [4], 4, 1, 96, 32, 0),
    ([90, 300], [2, 8], 2, 2, 256, 128, 0), ([900], [3], 10, 2, 128, 64, 12)])
def test_weights_of_single_tiles_keep_22_bits(gpu, kind, dt, lens, counts, Hq, Hkv, D, page, window):
    """Two binary16 terms: 2^-22 of a weight, numerator and denominator together 2^-21; all else as above."""
    assert max(counts) * Hq // Hkv <= 16
    c = Cache(kind, lens, Hkv, D, page, seed=sum(lens), scales="any")
    check(c, queries(sum(counts), Hq, D, dt), counts, window=window, kernel="kv8_rows", weights=2.0 ** -21)
