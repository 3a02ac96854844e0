"""GPU parity of rope against oracle/decode.py.

An output is off by its one rounding (eps / 2 of it, or of the smallest normal number), sine and cosine rounded to float32 and the
product beside the fused one (2^-24 each) of |a| + |b| times the magnitude, the fused one's own (2^-24 of the output), the angle
(a product in 64 bits and its reduction: 2^-51 of it, the oracle's as much) and the series (10^-11).
"""
import itertools

import numpy as np
import pytest

from oracle import decode as DC

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def ops():
    from xrgpu_amd import ops as _ops
    return _ops


def values(T, H, D, dt, seed=0):
    return torch.randn(T, H, D, generator=torch.Generator().manual_seed(seed + T + H)).to(DT[dt]).cuda()


def check(x, y, pos, f, **kw):
    ref, angle, pair = DC.rope(x.double().cpu().numpy(), pos, f.cpu().numpy(), **kw)
    eps, tiny = torch.finfo(x.dtype).eps, torch.finfo(x.dtype).tiny
    m = abs(kw.get("magnitude", 1.0))
    tol = eps / 2 * np.maximum(np.abs(ref), tiny) + 1.01 * (2.0 ** -24 * np.abs(ref) + m * pair * (2 * 2.0 ** -24 + 1e-11 + 2.0 ** -50 * angle[:, None, None]))
    assert y.dtype == x.dtype and y.shape == x.shape
    off = np.abs(y.double().cpu().numpy() - ref)
    assert (off <= np.where(pair > 0, tol, 0.0)).all() if not (pair == 0).all() else not off.any(), (off - tol).max()


def freq(R, theta=10000.0, **kw):
    return ops().rope_frequencies(R, theta, **kw)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,Hq,Hk,D,R", [(1, 1, 1, 64, 64), (1, 32, 8, 128, 128), (7, 3, 1, 96, 64), (5, 2, 2, 80, 20), (33, 5, 1, 256, 256),
                                         (4, 2, 1, 80, 80), (3, 2, 1, 7, 6), (2, 1, 1, 2, 2), (130, 8, 2, 128, 32), (9, 40, 3, 66, 66),
                                         (1, 1, 0, 1024, 1024), (2, 1, 1, 999, 998), (3, 70, 1, 512, 126), (1025, 4, 4, 64, 16)])
def test_rope(gpu, dt, interleaved, T, Hq, Hk, D, R):
    f, _ = freq(R)
    q, k = values(T, Hq, D, dt), values(T, Hk, D, dt, 1) if Hk else None
    pos = torch.randint(0, 9000, (T,), generator=torch.Generator().manual_seed(T)).int()
    got = ops().rope(q, k, frequencies=f, positions=pos.cuda(), interleaved=interleaved)
    for x, y in zip((q, k), got if Hk else (got,)):
        check(x, y, pos.numpy(), f, interleaved=interleaved)


@pytest.mark.parametrize("dt", list(DT))
def test_far_negative_and_wide_positions(gpu, dt):
    f, _ = freq(128, 500000.0)
    q = values(6, 3, 128, dt)
    pos = torch.tensor([0, -1, -70000, 1000003, (1 << 31) - 1, 5])
    for p in (pos, pos.int()):
        check(q, ops().rope(q, frequencies=f, positions=p.cuda()), p.numpy(), f)
    p = torch.tensor([1 << 40, -(1 << 33), 1 << 52, 3, 2, 1])
    near = f * 0 + 2.0 ** -30  # angles that 64 bits still hold
    check(q, ops().rope(q, frequencies=near, positions=p.cuda()), p.numpy(), near)


@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_is_the_gradient_and_turns_back(gpu, interleaved):
    f, m = freq(64, scaling="yarn", factor=4.0, original_length=4096)
    q = values(20, 3, 96, "f32")
    pos = torch.arange(20).cuda() * 977
    kw = dict(frequencies=f, positions=pos, magnitude=m, interleaved=interleaved)
    y = ops().rope(q, **kw)
    g = torch.randn_like(y)
    back = ops().rope(g, inverse=True, **kw)
    check(g, back, pos.cpu().numpy(), f, magnitude=m, interleaved=interleaved, inverse=True)
    # <y, g> = <q, back>, a bilinear form: the difference quotient of the loss <y, g> along any direction d is <d, back>
    for seed in range(3):
        d = torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)).cuda()
        ahead, behind = ((ops().rope(q + s * d, **kw).double() * g.double()).sum() for s in (0.5, -0.5))
        # float32 of outputs and inputs: 4 roundings of 2^-24 of values up to m (|q| + |d|) |g|
        size = float((m * 2 * (q.abs() + d.abs()).double() * g.abs().double()).sum())
        assert abs(float(ahead - behind) - float((d.double() * back.double()).sum())) <= 12 * 2.0 ** -24 * size
    again = ops().rope(y, inverse=True, **kw)
    assert (again[..., :64] / (m * m) - q[..., :64]).abs().max() <= 16 * 2.0 ** -24 * float(q.abs().max()) and torch.equal(again[..., 64:], q[..., 64:])


@pytest.mark.parametrize("counts", [[1, 1, 1], [4, 4, 4], [3, 0, 7, 1], [0, 0], [1] * 70 + [2] * 60])
def test_positions_of_the_cache(gpu, counts):
    """lengths and starts, as kv8_append's calls have them; rows that starts leave out stay as they were."""
    g = np.random.default_rng(len(counts))
    lens = np.array([n + int(g.integers(0, 5000)) for n in counts], np.int32)
    T = sum(counts)
    f, _ = freq(32)
    q, k = values(T + 3, 4, 64, "bf16"), values(T + 3, 2, 64, "bf16")
    starts = torch.tensor(np.concatenate([[0], np.cumsum(counts)]) + 1, dtype=torch.int32, device="cuda")
    L = torch.tensor(lens, device="cuda")
    outs = [torch.full_like(x, 7.0) for x in (q, k)]
    got = ops().rope(q, k, frequencies=f, lengths=L, starts=starts, out=outs[0], k_out=outs[1])
    assert got[0] is outs[0] and got[1] is outs[1]
    pos = DC.positions(lens, counts)
    for x, y in zip((q, k), outs):
        check(x[1:T + 1], y[1:T + 1], pos, f)
        assert (y[0] == 7).all() and (y[T + 1:] == 7).all()
    if len(set(counts)) == 1 and T:
        y = ops().rope(q[:T], frequencies=f, lengths=L)
        check(q[:T], y, pos, f)


def test_starts_that_run_backwards_write_nothing_wild(gpu):
    q = values(6, 2, 64, "f16")
    f, _ = freq(64)
    L = torch.tensor([10, 20], dtype=torch.int32, device="cuda")
    for starts in ([4, 2, 9], [-5, 3, 1 << 30], [7, 8, 9], [0, 0, 0]):
        out = torch.full_like(q, 7.0)
        ops().rope(q, frequencies=f, lengths=L, starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), out=out)
        assert out.isfinite().all()


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("interleaved", [False, True])
def test_strided_unaligned_and_in_place(gpu, dt, interleaved):
    """Heads in the rows of one product at an odd element, outputs in another one's, and in place."""
    f, _ = freq(48)
    wide = torch.randn(50, 6 * 64 + 3, device="cuda").to(DT[dt])
    q, k = wide[:, 1:257].unflatten(1, (4, 64)), wide[:, 257:385].unflatten(1, (2, 64))
    pos = torch.arange(50, device="cuda") + 100
    kw = dict(frequencies=f, positions=pos, interleaved=interleaved)
    want = ops().rope(q, k, **kw)
    for x, y in zip((q, k), want):
        check(x, y, pos.cpu().numpy(), f, interleaved=interleaved)
    other = torch.full((50, 500), 7.0, device="cuda").to(DT[dt])
    ops().rope(q, k, out=other[:, 3:259].unflatten(1, (4, 64)), k_out=other[:, 300:428].unflatten(1, (2, 64)), **kw)
    assert torch.equal(other[:, 3:259].unflatten(1, (4, 64)), want[0]) and torch.equal(other[:, 300:428].unflatten(1, (2, 64)), want[1])
    assert (other[:, :3] == 7).all() and (other[:, 259:300] == 7).all() and (other[:, 428:] == 7).all()
    rest = torch.cat((wide[:, :1], wide[:, 385:]), 1).clone()
    ops().rope(q, k, out=q, k_out=k, **kw)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(torch.cat((wide[:, :1], wide[:, 385:]), 1), rest)


def test_nonfinite_values_stay_in_their_pairs(gpu):
    f, _ = freq(64)
    q = values(3, 2, 64, "f16")
    q[1, 0, 5], q[2, 1, 40] = float("nan"), float("inf")
    y = ops().rope(q, frequencies=f, positions=torch.tensor([1, 2, 3]).cuda())
    bad = torch.zeros(3, 2, 64, dtype=torch.bool, device="cuda")
    bad[1, 0, 5] = bad[1, 0, 37] = bad[2, 1, 40] = bad[2, 1, 8] = True
    assert torch.equal(~y.isfinite(), bad)


def test_streams_graphs_and_empty(gpu):
    f, _ = freq(128)
    q, k = values(96, 8, 128, "bf16"), values(96, 2, 128, "bf16", 3)
    lengths = torch.arange(96, dtype=torch.int32, device="cuda") + 5
    want = ops().rope(q, k, frequencies=f, lengths=lengths)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    got = ops().rope(q, k, frequencies=f, lengths=lengths, stream=st)
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lengths += 1
        got = ops().rope(q, k, frequencies=f, lengths=lengths)
    for _ in range(3):
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = ops().rope(q, k, frequencies=f, positions=lengths - 1)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    none = ops().rope(q[:0], k[:0], frequencies=f, lengths=lengths[:0])
    assert [tuple(x.shape) for x in none] == [(0, 8, 128), (0, 2, 128)]


def test_frequencies(gpu):
    """Each scaling at its ends: pairs that turn often stay, those that hardly turn are divided by the factor."""
    o = ops()
    f, m = o.rope_frequencies(128, 10000.0)
    assert f.dtype == torch.float64 and f.is_cuda and m == 1.0
    want = 10000.0 ** (-np.arange(64) / 64)
    assert np.abs(f.cpu().numpy() / want - 1).max() < 1e-14
    assert torch.allclose(o.rope_frequencies(128, scaling="linear", factor=8.0)[0] * 8, f, rtol=1e-14)
    n = o.rope_frequencies(128, scaling="ntk", factor=8.0)[0]
    assert abs(float(n[0] / f[0]) - 1) < 1e-14 and abs(float(n[-1] * 8 / f[-1]) - 1) < 1e-12
    for s in ("bands", "yarn"):
        g, m = o.rope_frequencies(128, scaling=s, factor=8.0, original_length=4096)
        turns = (4096 * f / (2 * np.pi)).cpu()
        g, r = g.cpu(), (g / f).cpu()
        assert (r[turns > 40] == 1).all() and torch.allclose(r[turns < 0.8], torch.tensor(0.125, dtype=torch.float64), rtol=1e-14)
        assert (r.diff() <= 0).all() and m == (0.1 * np.log(8.0) + 1 if s == "yarn" else 1.0)


def test_more_rows_than_a_grid_has_threads(gpu):
    """A workgroup a row: 2^24 rows are 2^32 threads, of which a launch's count has 32 bits."""
    T = (1 << 24) + 5
    q = torch.arange(T, dtype=torch.int32, device="cuda").remainder_(251).half().view(T, 1, 1).expand(T, 1, 2).contiguous()
    f = torch.tensor([0.37], dtype=torch.float64, device="cuda")
    for kw in (dict(positions=torch.arange(T, dtype=torch.int32, device="cuda").remainder_(997)), dict(lengths=torch.tensor([T], dtype=torch.int32, device="cuda"))):
        got = ops().rope(q, frequencies=f, **kw)
        step = 1 << 21
        for at in range(0, T, step):  # the same rows in calls of their own
            end = min(T, at + step)
            one = dict(positions=kw["positions"][at:end]) if "positions" in kw else dict(lengths=torch.tensor([end], dtype=torch.int32, device="cuda"))
            assert torch.equal(got[at:end], ops().rope(q[at:end], frequencies=f, **one)), at
