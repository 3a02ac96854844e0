"""GPU: sample against oracle/decode.py.

Weights are whole multiples of 2^-F of the largest, F = min(51, 62 - ceil(log2 V)): each is off by half a unit, and by the
exponential's 2^-45 of itself, so a sum over V of them by no more than V (2^-(F+1) + 2^-45) of the largest. A number that falls that near to a border of the
running sum may draw either neighbour; the borders of top_p and min_p are asserted to be farther off in every case here.
"""
import numpy as np
import pytest

from oracle import decode as DC

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def ops():
    from xrgpu_amd import ops as _ops
    return _ops


def logits(B, V, dt, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed + V)
    x = torch.randn(B, V, generator=g) * spread
    x[torch.arange(B), torch.randint(0, V, (B,), generator=g)] += 6.0
    return x.to(DT[dt]).cuda()


def check(x, u, got=None, **kw):
    t, s = got if got is not None else ops().sample(x, u, **kw)
    assert t.dtype == torch.int32 and s.dtype == torch.float32 and t.shape == s.shape == u.shape
    V = x.shape[1]
    slack = V * (2.0 ** -(min(51, 62 - int(np.ceil(np.log2(V)))) + 1) + 2.0 ** -45)
    for b in range(x.shape[0]):
        of = {n: float(v[b]) if torch.is_tensor(v) else v for n, v in kw.items() if n in ("temperature", "top_k", "top_p", "min_p")}
        w, near = DC.kept(x[b].float().cpu().numpy(), of.get("temperature", 1.0), int(of.get("top_k", 0)), of.get("top_p", 1.0), of.get("min_p", 0.0))
        token, share = int(t[b]), float(s[b])
        if not w.any():
            assert token == -1 and share == -np.inf
            continue
        assert near > 2 * slack, "a border lies on a sum: the case cannot be told"
        may = DC.tokens(w, min(max(float(u[b]), 0.0), 1.0 - 2.0 ** -64), slack)
        assert token in may, (b, token, may, of)
        want = np.log(w[token] / w.sum())
        # float32's rounding, and the weight's own half unit
        assert abs(share - want) <= 2.0 ** -23 * (1 + abs(want)) + 2 * slack / w[token]
    return t, s


FILTERS = [dict(), dict(temperature=0.6), dict(top_k=1), dict(top_k=5), dict(top_k=50, temperature=0.8), dict(top_p=0.9), dict(top_p=0.3, temperature=1.5),
           dict(min_p=0.05), dict(top_k=40, top_p=0.8), dict(top_k=300, top_p=0.95, min_p=0.01, temperature=1.3), dict(top_p=0.99, min_p=0.2),
           dict(temperature=0.0), dict(temperature=0), dict(top_k=10 ** 9), dict(top_p=0.0), dict(min_p=1.0)]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (2, 63), (4, 1000), (2, 4099), (1, 50257 - 255), (5, 8192)])
@pytest.mark.parametrize("kw", FILTERS, ids=str)
def test_sample(gpu, dt, B, V, kw):
    check(logits(B, V, dt), torch.rand(B, generator=torch.Generator().manual_seed(B)).cuda(), **kw)


@pytest.mark.parametrize("B,V", [(1, 128000), (2, 262147), (40, 32000), (300, 3000)])
@pytest.mark.parametrize("kw", FILTERS[::3], ids=str)
def test_sample_large(gpu, B, V, kw):
    x, u = logits(B, V, "bf16"), torch.rand(B, generator=torch.Generator().manual_seed(B)).cuda()
    t, s = ops().sample(x, u, **kw)
    rows = list(range(0, B, max(1, B // 6)))
    check(x[rows], u[rows], got=(t[rows], s[rows]), **kw)


def test_settings_by_row(gpu):
    B = 24
    x = logits(B, 5000, "f32")
    g = torch.Generator().manual_seed(5)
    kw = dict(temperature=(torch.rand(B, generator=g) * 1.5).cuda(), top_k=torch.randint(-1, 60, (B,), generator=g).int().cuda(),
              top_p=(0.3 + torch.rand(B, generator=g)).cuda(), min_p=(torch.rand(B, generator=g) * 0.3 - 0.1).cuda())
    kw["temperature"][::5] = 0.0
    u = torch.rand(B, generator=g).cuda()
    t, s = check(x, u, **kw)
    for name in kw:  # a number for some, tensors for others, and rows by themselves
        b = 7
        one = {n: (v[b:b + 1] if n != name else float(v[b]) if n != "top_k" else max(0, int(v[b]))) for n, v in kw.items()}
        if not (name == "min_p" and one["min_p"] < 0):
            t1, s1 = ops().sample(x[b:b + 1], u[b:b + 1], **one)
            assert torch.equal(t1, t[b:b + 1]) and torch.equal(s1, s[b:b + 1])
    nan = torch.full((B,), float("nan"), device="cuda")
    off, _ = ops().sample(x, u, top_p=nan, min_p=nan)
    assert torch.equal(off, ops().sample(x, u)[0])
    greedy, _ = ops().sample(x, u, temperature=nan)
    assert torch.equal(greedy.long(), x.argmax(1))


@pytest.mark.parametrize("V", [10, 1000, 50000, 131072])
def test_equal_logits_go_by_index(gpu, V):
    """Every border is exact here: of n equal tokens, u draws the floor(u n)-th."""
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1.0 - 2.0 ** -24], device="cuda")
    for value in (0.0, -0.0, 3.0):
        x = torch.full((5, V), value, device="cuda")
        x[:, ::2] *= -1.0 if value == 0.0 else 1.0
        floor = lambda n: [int(np.floor(float(f) * n)) for f in u.cpu()]
        for kw, n in ((dict(), V), (dict(top_k=7), min(7, V)), (dict(top_p=0.5), V // 2), (dict(top_k=V // 2, top_p=0.5), max(1, V // 4 + (V // 2) % 2)),
                      (dict(min_p=1.0), V), (dict(top_p=2.0 ** -20), max(1, -(-V // 2 ** 20)))):
            t, s = ops().sample(x, u, **kw)
            assert t.tolist() == floor(n), kw
            assert (s.cpu() - np.log(1.0 / n)).abs().max() <= 2.0 ** -22 * (1 + np.log(n))
        assert ops().sample(x, u, temperature=0)[0].tolist() == [0] * 5


def test_infinities_nan_and_nothing(gpu):
    inf, nan = float("inf"), float("nan")
    x = torch.full((9, 700), -inf, device="cuda")
    x[1, 5] = -3e38
    x[2] = nan
    x[2, 600:] = 1.0
    x[3, ::7], x[3, 350] = 2.0, inf
    x[4, 100], x[4, 300] = inf, inf
    x[5] = nan
    x[6, 699], x[6, 0] = 0.0, -1.0
    x[7], x[7, 9] = -3e38, 3e38
    x[8, :3] = torch.tensor([-3.0, -2.0, -1.0])
    u = torch.full((9,), 0.6, device="cuda")
    for kw in FILTERS:
        check(x, u, **kw)
    assert ops().sample(x, u)[0].tolist()[:8] == [-1, 5, 660, 350, 300, -1, 699, 9]


@pytest.mark.parametrize("t", [1e-45, 1e-30, 1e-3, 1e30, float("inf")])
def test_temperatures_far_from_one(gpu, t):
    x = logits(3, 3000, "f32")
    x[2, 1000:] = -float("inf")
    u = torch.tensor([0.1, 0.9, 0.5], device="cuda")
    for kw in ({}, dict(top_k=20), dict(top_p=0.123), dict(top_k=100, top_p=0.517)):
        if t > 1e20 and "top_p" in kw and "top_k" not in kw:
            continue  # all weights equal: covered where borders are exact
        got = ops().sample(x, u, temperature=t, **kw)
        assert torch.equal(got[0], ops().sample(x, u, temperature=torch.full((3,), t, device="cuda"), **kw)[0]) or t < 1e-40
        if t < 1:
            assert torch.equal(got[0].long(), x.argmax(1)) or t == 1e-3
        if t == 1e-3 or (t > 1 and "top_p" not in kw):
            check(x, u, got=got, temperature=t, **kw)


def test_numbers_outside_their_range(gpu):
    x = logits(5, 2000, "f16")
    x[:] = x[0]
    u = torch.tensor([-1.0, float("nan"), 1.0, 7.0, 0.0], device="cuda")
    t, _ = ops().sample(x, u, top_k=50)
    w, _ = DC.kept(x[0].float().cpu().numpy(), 1.0, 50)
    at = np.nonzero(w)[0]
    assert t.tolist() == [at[0], at[0], at[-1], at[-1], at[0]]


@pytest.mark.parametrize("dt", list(DT))
def test_strides_and_odd_elements(gpu, dt):
    wide = torch.randn(4, 3007, device="cuda").to(DT[dt])
    x = wide[:, 3:2900]
    wide[:, :3], wide[:, 2900:] = 100.0, 100.0
    u = torch.rand(4, generator=torch.Generator().manual_seed(1)).cuda()
    for kw in (dict(), dict(top_k=30), dict(top_p=0.7), dict(temperature=0.0)):
        check(x, u, **kw)
    none = ops().sample(x[:0], u[:0])
    assert [tuple(v.shape) for v in none] == [(0,), (0,)]


@pytest.mark.parametrize("B,V", [(1, 40000), (3, 128000), (30, 9000), (200, 1000)])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=50, top_p=0.9), dict(top_p=0.9999), dict(top_k=20000)], ids=str)
def test_streams_workspaces_graphs_and_repeats_agree(gpu, B, V, kw):
    """A call's result does not depend on how it is spread: with and without a workspace, eager and captured, again and again."""
    o = ops()
    x, u = logits(B, V, "f16"), torch.rand(B, generator=torch.Generator().manual_seed(V)).cuda()
    x[0, : V // 2] = 1.0  # half a row of ties
    want = o.sample(x, u, **kw)
    rows = [0, B - 1]
    check(x[rows], u[rows], got=tuple(v[rows] for v in want), **kw)
    same = lambda got: all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(same(o.sample(x, u, **kw)) for _ in range(3))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    got = o.sample(x, u, stream=st, **kw)
    st.synchronize()
    assert same(got)
    need = o.sample_workspace_bytes(B, V)
    ws = torch.full((max(need, 4096),), 0xFF, dtype=torch.uint8, device="cuda")
    ws[:4096] = 0
    assert same(o.sample(x, u, workspace=ws, **kw)) and not ws[:4096].any()
    if need:
        with pytest.raises(ValueError):
            o.sample(x, u, workspace=ws[: need - 1], **kw)
    for more in ({}, {"workspace": ws}):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = o.sample(x, u, **kw, **more)
        for i in range(3):
            x.copy_(logits(B, V, "f16", i))
            u.uniform_()
            graph.replay()
            torch.cuda.synchronize()
            want = o.sample(x, u, **kw)
            assert same(got)


def test_one_workspace_serves_different_calls_in_turn(gpu):
    o = ops()
    u = torch.rand(8, generator=torch.Generator().manual_seed(3)).cuda()
    calls = [(logits(b, v, "bf16"), u[:b], kw) for b, v, kw in ((1, 100000, dict(top_p=0.9)), (8, 60000, dict(top_k=9)), (1, 300, {}),
                                                               (2, 100000, dict(temperature=0.0)), (3, 50000, dict(min_p=0.1)))]
    want = [o.sample(x, n, workspace=torch.zeros(max(4096, o.sample_workspace_bytes(*x.shape)), dtype=torch.uint8, device="cuda"), **kw) for x, n, kw in calls]
    for _ in range(2):
        for (x, n, kw), w in zip(calls, want):
            assert all(torch.equal(a, b) for a, b in zip(o.sample(x, n, **kw), w))


@pytest.mark.parametrize("B,V", [(260, 5000), (3, 100000)])
def test_more_ties_than_the_list_holds(gpu, B, V):
    """By a workgroup a row and by parts: thousands of equal logits where the thresholds lie."""
    x = torch.zeros(B, V, device="cuda")
    x[:, 7::V // 3] = 2.0  # three or four larger ones
    u = torch.rand(B, generator=torch.Generator().manual_seed(B)).cuda()
    for kw in (dict(top_k=V // 2), dict(top_p=0.5003), dict(top_k=V // 2, top_p=0.7123), dict(top_k=V // 2, top_p=0.7123, min_p=0.01)):
        t, s = ops().sample(x, u, **kw)
        rows = [0, B // 2, B - 1]
        check(x[rows], u[rows], got=(t[rows], s[rows]), **kw)


@pytest.mark.parametrize("dt,B,V", [("f32", 8, 60000), ("bf16", 8, 60000), ("f16", 64, 128000)])
def test_settings_by_row_in_parts(gpu, dt, B, V):
    """Greedy, empty, masked and unfiltered rows beside ones of small and large top_k and of top_p, in one call that is split over the device: rows
    leave its launches at different places."""
    o = ops()
    g = torch.Generator().manual_seed(B + V)
    wide = torch.zeros(B, V + 3, dtype=DT[dt], device="cuda")
    x = wide[:, 1:1 + V]
    x.copy_(logits(B, V, dt, seed=9))
    wide[:, 0], wide[:, 1 + V:] = 100.0, 100.0
    x[3], x[5] = -float("inf"), float("nan")
    x[6, torch.rand(V, generator=g).cuda() > 0.03] = -float("inf")
    of = lambda values, dtype: torch.tensor([values[b % len(values)] for b in range(B)], dtype=dtype, device="cuda")
    kw = dict(temperature=of([0.7, 1.3, 0.0, 1.0, 1.5, 1.0, 0.9, 1.1], torch.float32), top_k=of([0, 5, 0, 20000, 0, 3, 50, 20000, 0, 1], torch.int32),
              top_p=of([1.0, 0.9, 0.95], torch.float32), min_p=of([0.0, 0.0, 0.02, 0.0, 0.0], torch.float32))
    u = torch.rand(B, generator=g).cuda()
    need = o.sample_workspace_bytes(B, V)
    assert need > 4096
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
    ws[:4096] = 0
    t, s = o.sample(x, u, workspace=ws, **kw)
    assert not ws[:4096].any()
    assert t[3] == t[5] == -1 and s[3] == s[5] == -float("inf")
    rows = list(range(0, B, max(1, B // 16)))
    check(x[rows], u[rows], got=(t[rows], s[rows]), **{n: v[rows] for n, v in kw.items()})
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(o.sample(x, u, workspace=ws, **kw), (t, s)))
    many = 320  # a workgroup a row
    assert o.sample_workspace_bytes(many, V) == 0
    again = torch.arange(many, device="cuda") % B
    if V * many <= 320 * 60000:
        other = o.sample(x[again], u[again], **{n: v[again] for n, v in kw.items()})
        assert torch.equal(other[0], t[again]) and torch.equal(other[1], s[again])
    one = {n: v[:1].clone() for n, v in kw.items()}  # a row by itself, all of its launches for kinds that it does not have
    for b in range(0, B, 3):
        for n, v in kw.items():
            one[n].copy_(v[b:b + 1])
        t1, s1 = o.sample(x[b:b + 1], u[b:b + 1], **one)
        assert torch.equal(t1, t[b:b + 1]) and torch.equal(s1, s[b:b + 1])


@pytest.mark.parametrize("V", [3000, 60000])
@pytest.mark.parametrize("t", [1e-45, 1e-38, 1e-31, 1e-30])
def test_small_temperatures_are_not_none(gpu, V, t):
    """They draw among equal largest logits, which temperature 0 does not; as a number and as a tensor, subnormal ones too."""
    n, u = 7, [0.0, 0.35, 0.5, 0.99]
    x = torch.randn(4, V, generator=torch.Generator().manual_seed(V)).clamp(max=5.0).cuda()
    at = torch.arange(n, device="cuda") * (V // n) + 11
    x[:, at] = 9.0
    u = torch.tensor(u, device="cuda")
    want = at[(u.double() * n).floor().long()].int()
    for setting in (t, torch.full((4,), t, dtype=torch.float32, device="cuda")):
        for kw in ({}, dict(top_k=n), dict(top_p=0.9999), dict(top_k=100, top_p=0.9999)):
            tokens, shares = ops().sample(x, u, temperature=setting, **kw)
            assert torch.equal(tokens, want), (setting, kw)
            # the 64-bit logarithm, rounded to float32
            assert (shares.double() + np.log(n)).abs().max() <= 2.0 ** -24 * np.log(n)
    tokens, shares = ops().sample(x, u, temperature=0.0)
    assert (tokens == at[0]).all() and (shares == 0).all()


@pytest.mark.parametrize("V", [3, 8])
def test_more_rows_than_a_grid_has_threads(gpu, V):
    """A workgroup of 1024 a row: 2^22 rows are 2^32 threads, of which a launch's count has 32 bits."""
    B = (1 << 22) + 5
    g = torch.Generator(device="cuda").manual_seed(V)
    x, u = torch.randn(B, V, generator=g, device="cuda").half(), torch.rand(B, generator=g, device="cuda")
    by_row = dict(temperature=torch.rand(B, generator=g, device="cuda"), top_k=torch.randint(0, 3, (B,), generator=g, device="cuda").int(),
                  top_p=0.3 + torch.rand(B, generator=g, device="cuda"), min_p=torch.rand(B, generator=g, device="cuda") * 0.2)
    for kw in (dict(temperature=0.8), by_row):
        t, s = ops().sample(x, u, **kw)
        step = 1 << 20
        for at in range(0, B, step):  # the same rows in calls of their own
            part = slice(at, min(B, at + step))
            t1, s1 = ops().sample(x[part], u[part], **{n: v[part] if torch.is_tensor(v) else v for n, v in kw.items()})
            assert torch.equal(t[part], t1) and torch.equal(s[part], s1), at
