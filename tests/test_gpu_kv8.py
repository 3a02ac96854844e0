"""GPU parity of kv8_append and kv8_attention against oracle/lowbit.py.

Append follows from comparisons and powers of two (and one float32 division for scales of another quantiser): bit
equality of codes and scales. Attention: an output is off by its one rounding (eps / 2), the weights' rounding to
binary16 (2^-11 of sum p |v|, as the numerator and the denominator round apart; below 2^-14 / 1024 of the largest
weight, 2^-35 of the page's largest value for each token), the scores' float32 sums (D + 4 roundings of
2^-24 of sum |q k|, twice: numerator and denominator), the exponentials (2^-22) and the float32 sums over tokens (2^-24 each).
"""
import numpy as np
import pytest

from oracle import lowbit as LB

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CT = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def ops():
    from xrgpu_amd import ops as _ops
    return _ops


class Cache:
    def __init__(self, kind, lens, H, D, page, seed=0, scales="pow2", extra=2, fill=True):
        g = np.random.default_rng(seed)
        self.kind, self.page = kind, page
        B = len(lens)
        W = max(1, max(-(-max(x, 0) // page) for x in lens))
        P = B * W + extra
        order = g.permutation(P)[: B * W].reshape(B, W).astype(np.int32)
        self.table = order
        for b, x in enumerate(lens):
            order[b, -(-max(x, 0) // page):] = -1  # entries past a sequence's pages are not read
        self.lengths = np.array(lens, np.int32)
        mk = lambda: LB.encode8((g.standard_normal((P, H, page, D)) * LB.QMAX[kind] / 4).clip(-LB.QMAX[kind], LB.QMAX[kind]), kind)
        self.k, self.v = (mk(), mk()) if fill else (np.zeros((P, H, page, D), np.uint8),) * 2
        self.k, self.v = self.k.copy(), self.v.copy()
        unit = 4.0 / LB.QMAX[kind]
        if scales == "pow2":
            mks = lambda: (2.0 ** (np.floor(np.log2(unit)) + g.integers(-2, 3, (P, H)))).astype(np.float32)
        else:
            mks = lambda: (unit * g.uniform(0.3, 2.0, (P, H))).astype(np.float32)
        self.ks, self.vs = mks(), mks()

    def dev(self):
        t = lambda a: torch.from_numpy(a.copy()).cuda()
        return dict(k_cache=t(self.k).view(CT[self.kind]), v_cache=t(self.v).view(CT[self.kind]), k_scales=t(self.ks),
                    v_scales=t(self.vs), block_table=t(self.table), lengths=t(self.lengths))


def starts_of(counts):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")


def check_append(c, k, v, counts, ragged, *, bad=False, **kw):
    d = c.dev()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops().kv8_append(k, v, **d, starts=starts_of(counts) if ragged else None, status=status, **kw)
    wrong = False
    for x, codes, scales in ((k, c.k, c.ks), (v, c.v, c.vs)):
        wrong |= LB.append(x.float().cpu().numpy(), codes, scales, c.table, c.lengths, counts, c.kind)
    assert wrong == bad and int(status.item()) == (55 if bad else 0)
    for n, want in (("k_scales", c.ks), ("v_scales", c.vs)):
        assert np.array_equal(d[n].cpu().numpy(), want, equal_nan=True)
    for n, want in (("k_cache", c.k), ("v_cache", c.v)):
        got = d[n].view(torch.uint8).cpu().numpy()
        # an e4m3 zero may carry either sign
        diff = got != want
        if c.kind == "e4m3":
            diff &= ((got | want) & 127) != 0
        assert not diff.any()
    return d


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("lens,counts,H,D,page", [
    ([1], [1], 1, 64, 16), ([17], [1], 2, 64, 16), ([16], [16], 1, 96, 16), ([100, 3, 64], [1, 1, 1], 2, 128, 32),
    ([70, 33], [40, 33], 3, 64, 16), ([300], [257], 2, 128, 64), ([130, 1, 255], [2, 1, 130], 1, 256, 128),
    ([256, 256], [0, 256], 2, 96, 256), ([5, 9], [0, 0], 1, 64, 16)])
def test_append(gpu, kind, dt, lens, counts, H, D, page):
    c = Cache(kind, lens, H, D, page, seed=sum(lens) + D)
    T = sum(counts)
    g = torch.Generator().manual_seed(T + D)
    k, v = ((torch.randn(T, H, D, generator=g) * torch.exp2(torch.randint(-3, 9, (T, H, 1), generator=g).float())).to(DT[dt]).cuda()
            for _ in range(2))
    same = len(set(counts)) == 1
    check_append(c, k, v, counts, ragged=not same, max_new=max(counts) or None)
    if same and T:
        check_append(Cache(kind, lens, H, D, page, seed=1), k, v, counts, ragged=True)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_append_token_by_token_equals_the_oracle(gpu, kind):
    """Growths of a page's scale one after another, zeros first, and a second page."""
    c = Cache(kind, [0], 2, 64, 16, fill=False)
    c.table = np.array([[1, 0]], np.int32)
    rng = np.random.default_rng(4)
    for t in range(20):
        x = rng.standard_normal((1, 2, 64)) * (0.0 if t < 2 else 1.7 ** t * 1e-3)
        c.lengths = np.array([t + 1], np.int32)
        k = torch.tensor(x, dtype=torch.float32).cuda()
        check_append(c, k, -k, [1], False)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_append_foreign_scales_extremes_and_nonfinite(gpu, kind):
    c = Cache(kind, [21, 40, 37, 20, 35, 21], 2, 64, 32, scales="any")
    c.ks[c.table[3, 0]] = 0.0  # a zero scale starts anew
    c.ks[c.table[5, 0]] = np.nan  # and no scale stays none
    k = torch.randn(12, 2, 64)
    k[0, 0, 5], k[2, 1, 6], k[4] = float("inf"), float("nan"), 3e38
    k[6], k[8] = 0.0, 1e-42
    k = k.cuda()
    check_append(c, k, torch.flip(k, (0,)).contiguous(), [2] * 6, False)


def test_append_strided_tokens_and_unaligned(gpu):
    c = Cache("int8", [50], 2, 64, 16)
    wide = torch.randn(20, 3 * 128 + 1, device="cuda").half()
    k, v = wide[:, 1:129].view(20, 2, 64), wide[:, 130:258].view(20, 2, 64)
    check_append(c, k, v, [20], False)


def test_append_leaves_out_what_does_not_exist(gpu):
    k = torch.randn(6, 1, 64, device="cuda").half()
    for change in (lambda c: c.table.__setitem__((0, 1), -1), lambda c: c.table.__setitem__((0, 1), 1 << 30),
                   lambda c: c.lengths.__setitem__(0, 40), lambda c: c.lengths.__setitem__(0, 3), lambda c: c.lengths.__setitem__(0, -7)):
        c = Cache("int8", [20], 1, 64, 16)
        change(c)
        check_append(c, k, k, [6], False, bad=True)
    # starts outside the rows, running backwards, or past max_new
    for starts, most in (([0, 7], None), ([-1, 5], None), ([4, 2], None), ([0, 6], 5)):
        c = Cache("int8", [20], 1, 64, 16)
        d = c.dev()
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        ops().kv8_append(k, k, **d, starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), max_new=most, status=status)
        assert int(status.item()) == 55 and np.array_equal(d["k_cache"].cpu().numpy().view(np.uint8), c.k)


# ---------------------------------------------------------------------------

def check_attention(c, q, counts, ragged, *, d=None, bad=False, got=None, **kw):
    d = d or c.dev()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    o = got if got is not None else ops().kv8_attention(q, **d, starts=starts_of(counts) if ragged else None, status=status, **kw)
    D = q.shape[2]
    scale = kw.get("scale") or D ** -0.5
    ref, av, aqk = LB.attention(q.double().cpu().numpy(), c.k, c.v, c.ks, c.vs, c.table, c.lengths, counts, c.kind, scale=scale,
                                causal=kw.get("causal", True), window=kw.get("window", 0))
    eps = torch.finfo(q.dtype).eps
    n = float(max(int(c.lengths.max()), 1))
    rel = 2.0 ** -10 + 2.0 ** -21 + n * 2.0 ** -23 + 2 * (D + 4) * 2.0 ** -24 * aqk[..., None]
    top = np.nanmax(np.where(np.isfinite(c.vs), np.abs(c.vs), 0)) * LB.QMAX[c.kind]
    tol = eps / 2 * np.abs(ref) + (1 + eps) * (rel * av + n * 2.0 ** -35 * top) + torch.finfo(q.dtype).tiny * eps
    out = o.double().cpu().numpy()
    assert o.dtype == q.dtype and o.shape == q.shape
    assert np.isfinite(out).all()
    worst = (np.abs(out - ref) - tol).max() if ref.size else 0
    assert worst <= 0, (worst, np.abs(out - ref).max())
    if got is None:
        assert int(status.item()) == (55 if bad else 0)
    return o


ATTN = [  # lens, counts, Hq, Hkv, D, page, window
    ([1], [1], 1, 1, 64, 16, 0), ([5], [1], 4, 2, 128, 16, 0), ([33], [1], 8, 1, 64, 32, 0), ([200], [1], 8, 2, 96, 64, 0),
    ([64], [64], 2, 1, 64, 16, 0), ([300], [1], 20, 1, 128, 64, 0), ([257, 16, 99], [1, 1, 1], 6, 2, 256, 128, 0),
    ([700], [1], 4, 4, 128, 256, 100), ([50, 90], [20, 33], 4, 2, 128, 32, 0), ([130], [70], 5, 1, 96, 16, 17),
    ([3, 0, 40], [5, 0, 2], 2, 2, 64, 16, 0), ([2000], [1], 16, 2, 128, 64, 0), ([1500, 3], [3, 3], 8, 1, 64, 128, 0),
    ([400], [200], 8, 2, 128, 64, 0), ([333], [333], 3, 1, 256, 64, 50), ([97], [97], 1, 1, 64, 16, 1), ([0], [1], 2, 1, 128, 16, 0),
    ([270, 515], [130, 257], 4, 1, 96, 32, 0)]


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("lens,counts,Hq,Hkv,D,page,window", ATTN)
def test_attention(gpu, kind, dt, lens, counts, Hq, Hkv, D, page, window):
    c = Cache(kind, lens, Hkv, D, page, seed=sum(lens) + D, scales="any" if sum(lens) % 2 else "pow2")
    q = torch.randn(sum(counts), Hq, D, generator=torch.Generator().manual_seed(D + sum(counts))).to(DT[dt]).cuda()
    ragged = len(set(counts)) > 1
    check_attention(c, q, counts, ragged, window=window, max_new=max(counts))
    if not ragged:
        check_attention(c, q, counts, True, window=window)


@pytest.mark.parametrize("kind,dt,D,L,window", [("int8", "f16", 64, 2000, 0), ("e4m3", "bf16", 128, 2500, 0), ("int8", "bf16", 96, 3000, 1800),
                                                ("e4m3", "f16", 256, 1500, 0)])
def test_attention_many_rows_with_tokens_split(gpu, kind, dt, D, L, window):
    """Rows enough for tiles of 128 and too few of them to fill the card: their tokens are split and joined."""
    n, Hq = 520, 8
    c = Cache(kind, [L], 1, D, 64, seed=D, scales="any")
    c.vs[c.table[0, 3]] *= np.float32(64.0)  # the parts' sums are in units of different value scales
    need = ops().kv8_attention_workspace_bytes(n, Hq, 1, D, batch=1, table_width=c.table.shape[1], page_size=64, window=window)
    assert need > 4096 and (need - 4096) % (128 * (D + 2) * 4) == 0
    q = torch.randn(n, Hq, D, generator=torch.Generator().manual_seed(D)).to(DT[dt]).cuda()
    check_attention(c, q, [n], False, window=window)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("counts", [[1, 1], [40, 25]])
def test_attention_not_causal_and_other_scale(gpu, kind, counts):
    c = Cache(kind, [130, 61], 2, 128, 32, seed=8)
    q = torch.randn(sum(counts), 4, 128).half().cuda()
    check_attention(c, q, counts, True, causal=False)
    check_attention(c, q, counts, True, causal=False, window=20, scale=0.25)


@pytest.mark.parametrize("counts", [[1], [90]])
def test_attention_sharp_and_spread_scales(gpu, counts):
    """Scores that single out tokens, pages whose value scales differ by 2^12, a page of zeros."""
    c = Cache("int8", [200], 1, 64, 16, seed=9)
    c.vs[c.table[0, ::2]] *= np.float32(2.0 ** -12)
    c.vs[c.table[0, 3]] = 0
    c.ks[c.table[0, 5]] = 0
    q = (torch.randn(counts[0], 2, 64) * 6).bfloat16().cuda()
    check_attention(c, q, counts, False)


@pytest.mark.parametrize("dt,big", [("f16", 6e4), ("bf16", 1e30), ("bf16", 1e-30), ("f16", 6e-8)])
def test_attention_extreme_queries(gpu, dt, big):
    c = Cache("e4m3", [70], 1, 64, 16, seed=10)
    for n in (1, 40):
        q = (torch.randn(n, 2, 64).clamp(-1, 1) * big).to(DT[dt]).cuda()
        check_attention(c, q, [n], False, scale=1.0 / (64 * big))


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("counts", [[1, 1], [50, 30]])
def test_attention_reads_nothing_past_the_tokens(gpu, kind, counts):
    """Slots past a length and pages that no token lies in hold NaN codes and scales."""
    c = Cache(kind, [75, 50], 2, 64, 32, seed=11)
    q = torch.randn(sum(counts), 4, 64).half().cuda()
    clean = check_attention(c, q, counts, True)
    used = set()
    for b, L in enumerate(c.lengths):
        for i in range(-(-int(L) // 32)):
            used.add(int(c.table[b, i]))
        last = c.table[b, (int(L) - 1) // 32]
        c.k[last, :, (int(L) - 1) % 32 + 1:] = 0x7F
        c.v[last, :, (int(L) - 1) % 32 + 1:] = 0x7F
    for p in range(c.k.shape[0]):
        if p not in used:
            c.k[p], c.v[p], c.ks[p], c.vs[p] = 0xFF, 0xFF, np.nan, np.inf
    o = ops().kv8_attention(q, **c.dev(), starts=starts_of(counts))
    assert torch.equal(o, clean)


@pytest.mark.parametrize("n", [1, 40])
def test_attention_nonfinite_scales_and_queries_stay_apart(gpu, n):
    """A NaN page is NaN to the rows that see it alone; a NaN query to its own row and head alone."""
    c = Cache("int8", [200, 200], 2, 64, 32, seed=12)
    c.vs[c.table[0, 6], 1] = np.nan  # tokens 192 .. 199 of the first sequence, head 1
    q = torch.randn(2 * n, 4, 64).half().cuda()
    q[n + n // 2, 0, 3] = float("nan")
    o = ops().kv8_attention(q, **c.dev())
    nan = torch.zeros(2 * n, 4, dtype=torch.bool, device="cuda")
    nan[max(0, n - 8):n, 2:] = True
    nan[n + n // 2, 0] = True
    assert torch.equal(o.isnan().any(-1), nan) and torch.equal(o.isnan().all(-1), nan)


@pytest.mark.parametrize("n", [1, 40])
def test_attention_leaves_out_pages_that_do_not_exist(gpu, n):
    for p in (-1, 1 << 30):
        c = Cache("int8", [100], 1, 64, 16, seed=13)
        c.table[0, 2] = p
        q = torch.randn(n, 2, 64).half().cuda()
        check_attention(c, q, [n], False, bad=True)
    c = Cache("int8", [100], 1, 64, 16, seed=13)
    c.lengths[0] = 130  # past the table
    check_attention(c, q, [n], False, bad=True)


def test_attention_strided_queries_out_and_empty(gpu):
    c = Cache("int8", [90], 2, 64, 16, seed=14)
    wide = torch.randn(30, 4 * 64 + 7, device="cuda").half()
    q = wide[:, 3:259].view(30, 4, 64)
    out = torch.full((30, 4, 64), float("nan"), device="cuda", dtype=torch.float16)
    d = c.dev()
    assert ops().kv8_attention(q, **d, out=out) is out
    check_attention(c, q, [30], False, d=d, got=out)
    none = ops().kv8_attention(q[:0], **d)
    assert tuple(none.shape) == (0, 4, 64)


@pytest.mark.parametrize("n", [1, 150])
def test_attention_other_stream_workspace_graph_and_repeats(gpu, n):
    c = Cache("e4m3", [3000, 800], 2, 128, 64, seed=15)
    d = c.dev()
    q = torch.randn(2 * n, 8, 128).bfloat16().cuda()
    eager = check_attention(c, q, [n, n], False, d=d)
    for _ in range(3):
        assert torch.equal(ops().kv8_attention(q, **d), eager)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    y = ops().kv8_attention(q, **d, stream=st)
    st.synchronize()
    assert torch.equal(y, eager)
    need = ops().kv8_attention_workspace_bytes(2 * n, 8, 2, 128, batch=2, table_width=d["block_table"].shape[1], page_size=64)
    ws = torch.zeros(max(need, 4096), dtype=torch.uint8, device="cuda")
    assert torch.equal(ops().kv8_attention(q, **d, workspace=ws), eager)
    assert not ws[:4096].any()
    if need:
        with pytest.raises(ValueError):
            ops().kv8_attention(q, **d, workspace=ws[: need - 1])
    for kw in ({}, {"workspace": ws}):
        new = torch.randn(2 * n, 2, 128, device="cuda").bfloat16()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops().kv8_append(new, new, **d)
            out = ops().kv8_attention(q, **d, **kw)
        for i in range(3):
            new.copy_(torch.randn(2 * n, 2, 128, device="cuda"))
            q.copy_(torch.randn(2 * n, 8, 128, device="cuda"))
            graph.replay()
            torch.cuda.synchronize()
            for x, y in (("k", "k_cache"), ("v", "v_cache")):
                setattr(c, x, d[y].view(torch.uint8).cpu().numpy())
            c.ks, c.vs = d["k_scales"].cpu().numpy(), d["v_scales"].cpu().numpy()
            got = out.clone()
            check_attention(c, q, [n, n], False, d=d, got=got)
            ops().kv8_attention(q, **d)


def test_append_then_attention_is_a_decode_step(gpu):
    """A prompt, then single tokens, each seen by its own query."""
    c = Cache("int8", [0, 0], 2, 64, 16, fill=False)
    c.table = np.arange(8, dtype=np.int32).reshape(2, 4)
    c.k, c.v = np.zeros((8, 2, 16, 64), np.uint8), np.zeros((8, 2, 16, 64), np.uint8)
    c.ks, c.vs = np.zeros((8, 2), np.float32), np.zeros((8, 2), np.float32)
    for step, n in enumerate((37, 1, 1, 1)):
        c.lengths = c.lengths + np.int32(n)
        g = torch.Generator().manual_seed(step)
        q = torch.randn(2 * n, 4, 64, generator=g).half().cuda()
        k, v = (torch.randn(2 * n, 2, 64, generator=g).half().cuda() for _ in range(2))
        d = check_append(c, k, v, [n, n], False)
        check_attention(c, q, [n, n], False, d=d)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,D,n", [(6, 2, 64, 1), (5, 1, 96, 3), (4, 4, 128, 1), (3, 1, 256, 2), (4, 2, 128, 70)])
def test_attention_queries_and_outputs_at_any_element(gpu, dt, Hq, Hkv, D, n):
    """Tokens an odd number of elements apart, from an odd element on; outputs from an odd element on."""
    c = Cache("int8", [150, 90], Hkv, D, 32, seed=D)
    wide = torch.randn(2 * n, Hq * D + 3, device="cuda").to(DT[dt])
    q = wide[:, 1:1 + Hq * D].unflatten(1, (Hq, D))
    store = torch.full((2 * n * Hq * D + 3,), 7.0, device="cuda").to(DT[dt])
    out = store[1:-2].view(2 * n, Hq, D)
    check_attention(c, q, [n, n], False, out=out)
    assert (store[0] == 7) and (store[-2:] == 7).all()
    check_attention(c, q, [n, n], False, got=out, d=c.dev())
