"""GPU: kv8_shared_attention against oracle/lowbit.py's attention over the tables that it stands for; tolerances as in test_gpu_kv8.py."""
import numpy as np
import pytest

from oracle import lowbit as LB
from tests.test_gpu_kv8 import DT, Cache, check_attention, starts_of

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def ops():
    from xrgpu_amd import ops as _ops
    return _ops


@pytest.fixture(params=["", "kv8_walk", "kv8_prefix_rows", "kv8_prefix_tile"], autouse=True)
def way(request, monkeypatch):
    """Every test by each way that a call can go, beside the one that is estimated fastest."""
    if request.param:
        monkeypatch.setenv("XRMM_KV8_SHARED", request.param)
    return request.param


def shared_cache(kind, shared, lens, H, D, page, **kw):
    """A cache whose sequences have ``lens`` tokens, the first ``shared`` pages common to all: the oracle's table names them, the
    device's holds what must not be read there."""
    width = max(shared, max(-(-max(x, 0) // page) for x in lens))
    c = Cache(kind, [max(1, width * page)] + list(lens), H, D, page, **kw)  # the first one's pages are the shared ones
    pages = c.table[0, :shared].copy()
    c.table, c.lengths = c.table[1:].copy(), np.array(lens, np.int32)
    given = c.table.copy()
    c.table[:, :shared] = pages
    given[:, :shared] = np.where(np.arange(shared) % 2, -1, 1 << 30)
    d = c.dev()
    d["block_table"] = torch.from_numpy(given).cuda()
    d["shared_pages"] = torch.from_numpy(pages.astype(np.int32)).cuda()
    return c, d


def check(c, d, q, counts, *, ragged=None, bad=False, want=None, **kw):
    ragged = len(set(counts)) > 1 if ragged is None else ragged
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    o = ops().kv8_shared_attention(q, **d, starts=starts_of(counts) if ragged else None, status=status, **kw)
    kw.pop("workspace", None), kw.pop("max_new", None), kw.pop("out", None)
    check_attention(c, q, counts, ragged, d=d, got=o, **kw)
    assert int(status.item()) == (55 if bad else 0)
    return o


CASES = [  # shared pages, lens, counts, Hq, Hkv, D, page, window
    (1, [17], [1], 1, 1, 64, 16, 0), (2, [40, 33, 64], [1, 1, 1], 8, 2, 128, 16, 0), (4, [300, 256, 270, 257], [1, 1, 1, 1], 4, 1, 96, 64, 0),
    (20, [330, 400, 321], [1, 1, 1], 16, 2, 256, 16, 0), (3, [100, 120], [4, 9], 5, 1, 64, 32, 0), (6, [500, 390, 384], [100, 6, 30], 8, 2, 128, 64, 0),
    (2, [600, 530], [80, 18], 4, 4, 256, 256, 0), (5, [90, 80, 10, 0, 83], [1, 1, 1, 1, 1], 8, 2, 64, 16, 0),      # inside the shared part, and nothing
    (5, [90, 80, 10, 0, 83], [20, 5, 10, 0, 3], 8, 2, 64, 16, 0), (8, [600, 700], [1, 1], 8, 2, 128, 64, 300),     # windows that begin in the shared part
    (8, [600, 700], [40, 3], 8, 2, 96, 64, 100), (8, [900, 700], [1, 1], 8, 2, 128, 64, 33),                       # and behind it
    (0, [50, 20], [1, 1], 4, 2, 64, 16, 0), (64, [2100, 2049, 2300], [1, 1, 1], 32, 4, 128, 32, 0), (3, [49, 70], [1, 1], 40, 1, 64, 16, 0)]


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("shared,lens,counts,Hq,Hkv,D,page,window", CASES)
def test_shared(gpu, kind, dt, shared, lens, counts, Hq, Hkv, D, page, window):
    c, d = shared_cache(kind, shared, lens, Hkv, D, page, seed=sum(lens) + D, scales="any" if sum(lens) % 2 else "pow2")
    q = torch.randn(sum(counts), Hq, D, generator=torch.Generator().manual_seed(D + sum(counts))).to(DT[dt]).cuda()
    check(c, d, q, counts, window=window, max_new=max(counts))
    if len(set(counts)) == 1:
        check(c, d, q, counts, ragged=True, window=window)


@pytest.mark.parametrize("kind,dt,B,shared,D,G", [("int8", "f16", 70, 20, 128, 4), ("e4m3", "bf16", 33, 40, 64, 8), ("int8", "bf16", 40, 17, 256, 5),
                                                  ("e4m3", "f16", 130, 9, 96, 1)])
def test_many_sequences(gpu, kind, dt, B, shared, D, G):
    page = 64
    lens = [shared * page + 1 + (37 * b) % 150 for b in range(B)]
    c, d = shared_cache(kind, shared, lens, 1, D, page, seed=D)
    q = torch.randn(B, G, D, generator=torch.Generator().manual_seed(D)).to(DT[dt]).cuda()
    check(c, d, q, [1] * B)
    check(c, d, q, [1] * B, ragged=True, max_new=1)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("counts", [[1, 1, 1], [40, 25, 3]])
def test_not_causal_and_other_scales(gpu, kind, counts):
    c, d = shared_cache(kind, 3, [130, 161, 96], 2, 128, 32, seed=8)
    q = torch.randn(sum(counts), 8, 128, generator=torch.Generator().manual_seed(1)).half().cuda()
    check(c, d, q, counts, causal=False)
    check(c, d, q, counts, causal=False, window=50, scale=0.25)
    check(c, d, q, counts, scale=-0.1)


@pytest.mark.parametrize("counts", [[1, 1], [70, 30]])
def test_units_of_both_parts_differ(gpu, counts):
    """Value scales of the shared pages far above and far below those of the sequences' own, a page of zeros, sharp scores."""
    for by in (2.0 ** -12, 2.0 ** 12):
        c, d = shared_cache("int8", 8, [230, 190], 2, 64, 16, seed=9)
        pages = d["shared_pages"].cpu().numpy()
        c.vs[pages] *= np.float32(by)
        c.vs[pages[3]] = 0
        c.ks[pages[5]] = 0
        d.update(k_scales=torch.from_numpy(c.ks.copy()).cuda(), v_scales=torch.from_numpy(c.vs.copy()).cuda())
        q = (torch.randn(sum(counts), 4, 64, generator=torch.Generator().manual_seed(2)) * 4).bfloat16().cuda()
        check(c, d, q, counts)


@pytest.mark.parametrize("n", [1, 30])
def test_nonfinite_pages_reach_the_rows_that_see_them(gpu, n):
    c, d = shared_cache("int8", 4, [200, 150], 2, 64, 32, seed=12)
    q = torch.randn(2 * n, 4, 64, generator=torch.Generator().manual_seed(3)).half().cuda()
    d["v_scales"][d["shared_pages"][1].long(), 1] = float("nan")
    o = ops().kv8_shared_attention(q, **d)
    nan = torch.zeros(2 * n, 4, dtype=torch.bool, device="cuda")
    nan[:, 2:] = True
    assert torch.equal(o.isnan().all(-1), nan) and torch.equal(o.isnan().any(-1), nan)
    d["v_scales"].copy_(torch.from_numpy(c.vs))
    d["v_scales"][int(c.table[0, 6]), 1] = float("nan")  # tokens 192 .. 199 of the first sequence alone
    o = ops().kv8_shared_attention(q, **d)
    nan = torch.zeros(2 * n, 4, dtype=torch.bool, device="cuda")
    nan[max(0, n - 8):n, 2:] = True
    assert torch.equal(o.isnan().all(-1), nan) and torch.equal(o.isnan().any(-1), nan)
    q[n, 0, 3] = float("nan")
    d["v_scales"].copy_(torch.from_numpy(c.vs))
    nan[:] = False
    nan[n, 0] = True
    o = ops().kv8_shared_attention(q, **d)
    assert torch.equal(o.isnan().all(-1), nan) and torch.equal(o.isnan().any(-1), nan)


@pytest.mark.parametrize("n", [1, 40])
def test_pages_that_do_not_exist(gpu, n):
    for p in (-1, 1 << 30):
        c, d = shared_cache("int8", 4, [100, 90], 1, 64, 16, seed=13)
        q = torch.randn(2 * n, 2, 64, generator=torch.Generator().manual_seed(4)).half().cuda()
        d["shared_pages"][2] = p
        c.table[:, 2] = p
        check(c, d, q, [n, n], bad=True)
        c, d = shared_cache("int8", 4, [100, 90], 1, 64, 16, seed=13)
        d["block_table"][1, 4] = p
        c.table[1, 4] = p
        check(c, d, q, [n, n], bad=True)
    c, d = shared_cache("int8", 4, [100, 90], 1, 64, 16, seed=13)
    c.lengths[0] = 130  # past the table
    d["lengths"][0] = 130
    check(c, d, q, [n, n], bad=True)


def test_tables_narrower_than_the_shared_part(gpu):
    """Sequences that end inside the shared part need no columns of their own."""
    c, d = shared_cache("int8", 6, [90, 40, 96], 2, 64, 16, seed=14)
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(5)).half().cuda()
    for width in (2, 0):
        d["block_table"] = d["block_table"][:, :width].contiguous()
        check(c, d, q, [1, 1, 1])


@pytest.mark.parametrize("n", [1, 33])
def test_reads_nothing_else(gpu, n):
    """Slots past a length and pages of no sequence hold NaN."""
    c, d = shared_cache("e4m3", 3, [130, 100], 2, 64, 32, seed=15)
    q = torch.randn(2 * n, 4, 64, generator=torch.Generator().manual_seed(6)).half().cuda()
    clean = check(c, d, q, [n, n])
    used = set(int(p) for b, L in enumerate(c.lengths) for p in c.table[b, : -(-int(L) // 32)])
    for b, L in enumerate(c.lengths):
        last = c.table[b, (int(L) - 1) // 32]
        c.k[last, :, (int(L) - 1) % 32 + 1:] = c.v[last, :, (int(L) - 1) % 32 + 1:] = 0x7F
    for p in range(c.k.shape[0]):
        if p not in used:
            c.k[p], c.v[p], c.ks[p], c.vs[p] = 0xFF, 0xFF, np.nan, np.inf
    e = c.dev()
    assert torch.equal(ops().kv8_shared_attention(q, **{**d, **{n: e[n] for n in ("k_cache", "v_cache", "k_scales", "v_scales")}}), clean)


def test_rows_left_out_stay(gpu):
    c, d = shared_cache("int8", 3, [70, 60], 2, 64, 16, seed=16)
    q = torch.randn(9, 4, 64, generator=torch.Generator().manual_seed(7)).half().cuda()
    out = torch.full((9, 4, 64), 7.0, device="cuda").half()
    starts = torch.tensor([1, 4, 6], dtype=torch.int32, device="cuda")
    ops().kv8_shared_attention(q, **d, starts=starts, out=out)
    assert (out[0] == 7).all() and (out[6:] == 7).all()
    check_attention(c, q[1:6], [3, 2], True, d=d, got=out[1:6].contiguous())
    for wild in ([4, 2, 9], [-5, 3, 1 << 30], [0, 30, 2]):  # sequences that starts names wrongly are left out
        out.fill_(7.0)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        ops().kv8_shared_attention(q, **d, starts=torch.tensor(wild, dtype=torch.int32, device="cuda"), out=out, status=status)
        assert out.isfinite().all() and int(status) == 55


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("n", [1, 40])
def test_queries_and_outputs_at_any_element(gpu, dt, n):
    c, d = shared_cache("int8", 3, [150, 190], 2, 96, 32, seed=17)
    wide = torch.randn(2 * n, 4 * 96 + 3, device="cuda").to(DT[dt])
    q = wide[:, 1:1 + 4 * 96].unflatten(1, (4, 96))
    store = torch.full((2 * n * 4 * 96 + 3,), 7.0, device="cuda").to(DT[dt])
    out = store[1:-2].view(2 * n, 4, 96)
    check(c, d, q, [n, n], out=out)
    assert (store[0] == 7) and (store[-2:] == 7).all()
    assert tuple(ops().kv8_shared_attention(q[:0], **d).shape) == (0, 4, 96)


@pytest.mark.parametrize("B,n", [(2, 1), (12, 1), (3, 70), (60, 1)])
def test_streams_workspaces_graphs_and_repeats(gpu, B, n):
    page, S = 64, 30
    lens = [S * page + n + 40 * b for b in range(B)]
    c, d = shared_cache("e4m3", S, lens, 2, 128, page, seed=18)
    q = torch.randn(B * n, 8, 128, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    eager = check(c, d, q, [n] * B)
    for _ in range(3):
        assert torch.equal(ops().kv8_shared_attention(q, **d), eager)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    y = ops().kv8_shared_attention(q, **d, stream=st)
    st.synchronize()
    assert torch.equal(y, eager)
    need = ops().kv8_shared_attention_workspace_bytes(B * n, 8, 2, 128, batch=B, shared_pages=S, table_width=d["block_table"].shape[1], page_size=page)
    ws = torch.full((max(need, 4096),), 0xFF, dtype=torch.uint8, device="cuda")
    ws[:4096] = 0
    assert torch.equal(ops().kv8_shared_attention(q, **d, workspace=ws), eager) and not ws[:4096].any()
    if need:
        with pytest.raises(ValueError):
            ops().kv8_shared_attention(q, **d, workspace=ws[: need - 1])
    cache = {k: v for k, v in d.items() if k != "shared_pages"}
    full = dict(cache, block_table=torch.from_numpy(c.table.copy()).cuda())  # as an append takes it
    for kw in ({}, {"workspace": ws}):
        new = torch.randn(B * n, 2, 128, device="cuda").bfloat16()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops().kv8_append(new, new, **full)
            out = ops().kv8_shared_attention(q, **d, **kw)
        for _ in range(3):
            new.copy_(torch.randn(B * n, 2, 128, device="cuda"))
            q.copy_(torch.randn(B * n, 8, 128, device="cuda"))
            graph.replay()
            torch.cuda.synchronize()
            for x, y in (("k", "k_cache"), ("v", "v_cache")):
                setattr(c, x, d[y].view(torch.uint8).cpu().numpy())
            c.ks, c.vs = d["k_scales"].cpu().numpy(), d["v_scales"].cpu().numpy()
            got = out.clone()
            if B <= 12:
                check_attention(c, q, [n] * B, False, d=d, got=got)
            # another order of the sums, and weights of eleven bits: within their rounding of the eager call's
            e = ops().kv8_shared_attention(q, **d)
            assert (got.float() - e.float()).abs().max() <= 2.0 ** -7 * float(e.float().abs().max())


def test_the_named_way_is_taken(gpu, way):
    kw = dict(batch=40, shared_pages=4, table_width=6, page_size=16)
    name = ops().kv8_shared_attention_kernel(40, 8, 2, 64, **kw)
    assert name == way if way else name in ("kv8_walk", "kv8_prefix_rows", "kv8_prefix_tile")


@pytest.mark.parametrize("D,G,page", [(128, 4, 64), (64, 8, 16), (256, 4, 128), (96, 1, 32)])
def test_sequences_that_end_among_the_shared_tokens_of_many(gpu, D, G, page):
    """Rows of one tile whose sequences see all, some and none of the shared tokens, in no order, with and without windows."""
    S = 600 // page
    lens = [(S * page + 40, 17, S * page, 0, S * page + 1, 300, S * page - 1, 64)[b % 8] for b in range(45)]
    c, d = shared_cache("int8", S, lens, 1, D, page, seed=D, scales="any")
    q = torch.randn(45, G, D, generator=torch.Generator().manual_seed(D)).half().cuda()
    for kw in (dict(), dict(window=100), dict(causal=False), dict(causal=False, window=90)):
        check(c, d, q, [1] * 45, **kw)
    counts = [min(n, (1, 3, 0, 2)[b % 4]) for b, n in enumerate(lens)]
    q = torch.randn(sum(counts), G, D, generator=torch.Generator().manual_seed(D)).half().cuda()
    for kw in (dict(), dict(window=100)):
        check(c, d, q, counts, **kw)


@pytest.mark.parametrize("kind,dt,D,n", [("int8", "f16", 128, 60), ("e4m3", "bf16", 64, 130), ("int8", "bf16", 256, 40)])
def test_long_shared_parts_are_split(gpu, kind, dt, D, n):
    """Shared tokens in several parts, own tokens of many rows; value scales far apart in the parts."""
    c, d = shared_cache(kind, 24, [24 * 64 + n + 7, 24 * 64 + n], 1, D, 64, seed=D)
    pages = d["shared_pages"].cpu().numpy()
    c.vs[pages[5:9]] *= np.float32(64.0)
    d["v_scales"] = torch.from_numpy(c.vs.copy()).cuda()
    q = torch.randn(2 * n, 8, D, generator=torch.Generator().manual_seed(D)).to(DT[dt]).cuda()
    check(c, d, q, [n, n])


def test_sequences_of_more_rows_than_max_new(gpu, way):
    """They count as wrong: their rows stay as they are, the others' are right."""
    B, shared, page, D = 40, 12, 64, 128
    counts = [1 + b % 2 for b in range(B)]
    counts[3] = 5
    c, d = shared_cache("int8", shared, [shared * page + 7 + 3 * b for b in range(B)], 1, D, page, seed=21)
    q = torch.randn(sum(counts), 4, D, generator=torch.Generator().manual_seed(21)).half().cuda()
    want = ops().kv8_shared_attention(q, **d, starts=starts_of(counts), max_new=5)
    out, status = torch.full_like(q, 7.0), torch.zeros(1, dtype=torch.int32, device="cuda")
    ops().kv8_shared_attention(q, **d, starts=starts_of(counts), max_new=2, out=out, status=status)
    first = sum(counts[:3])
    assert int(status.item()) == 55 and (out[first:first + 5] == 7).all()
    # either call: weights rounded to binary16 (half a step, 2^-11) and the outputs too; scores as float32 sums of D products
    keep = torch.ones(len(q), dtype=torch.bool, device="cuda")
    keep[first:first + 5] = False
    top_k, top_v = 128 * float(c.ks.max()), 128 * float(c.vs.max())
    scores = D * 2.0 ** -24 * float(q.float().abs().sum(-1).max()) * top_k / D ** 0.5
    o, w = out[keep].double(), want[keep].double()
    assert ((o - w).abs() <= 2 * top_v * (2.0 ** -11 + 2 * scores) + (o.abs() + w.abs()) * 2.0 ** -11).all()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D,G,n", [(64, 8, 1), (96, 4, 2), (128, 4, 1), (128, 16, 1), (256, 4, 1), (256, 5, 3)])
def test_weights_of_few_rows_have_two_terms_by_every_way(gpu, kind, D, G, n):
    """Up to 16 rows of a sequence and key head keep 22 bits of a weight, of shared tokens too, as kv8_attention's do.

    Queries of eight small integers and key factors that are powers of two: sums of products are exact. In powers of two, of which ln 2 times as much
    is a weight's relative error, a score is off by 2^-24 of the largest five times (log2 e, the product with it, the difference of two), and an exponent
    of up to 16 by three roundings. With the exponentials' 2^-22 that counts in numerator and denominator; then the second terms' own rounding, 2^-22, and
    float32 sums over the tokens, 2^-24 each: all of sum p |v| / sum p. At last an output's own rounding. Weights of eleven bits are off by up to 2^-12 each, some
    2^-16 of that sum in the mean of 64, as many of these outputs would show."""
    B, page, S = 40, 16, 4
    lens = [S * page + n + b % 4 for b in range(B)]
    lens[5], lens[17] = 50, 64  # among the shared tokens, and at their end
    c, d = shared_cache(kind, S, lens, 1, D, page, seed=D + G)
    g = np.random.default_rng(D + G)
    c.ks[:] = 2.0 ** -7 if kind == "int8" else 2.0 ** -8
    d["k_scales"] = torch.from_numpy(c.ks.copy()).cuda()
    q = np.zeros((B * n, G, D))
    for row in q.reshape(-1, D):
        row[g.choice(D, 8, replace=False)] = g.integers(1, 4, 8) * g.choice((-1, 1), 8)
    o = ops().kv8_shared_attention(torch.from_numpy(q).half().cuda(), **d, scale=2.0 ** -2).double().cpu().numpy()
    for b, L in enumerate(lens):
        pages = c.table[b, : -(-L // page)]
        k, v = (LB.decode8(x[pages, 0].reshape(-1, D)[:L], kind) * np.repeat(s[pages, 0].astype(np.float64), page)[:L, None] for x, s in ((c.k, c.ks), (c.v, c.vs)))
        for i in range(n):
            seen = L - n + i + 1
            z = q[b * n + i] @ k[:seen].T / 4
            p = np.exp(z - z.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            want, size = p @ v[:seen], p @ np.abs(v[:seen])
            top = np.abs(z).max() * np.log2(np.e)
            assert top < 64
            off = 2 * (np.log(2) * 2.0 ** -24 * (5 * top + 3 * 16) + 2.0 ** -22) + 2.0 ** -22 + seen * 2.0 ** -24
            assert (np.abs(o[b * n + i] - want) <= size * off + np.abs(want) * 2.0 ** -11 + 2.0 ** -25).all()


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("n,G", [(1, 8), (4, 4), (1, 1)])
def test_the_walk_is_kv8_attention_bit_for_bit(gpu, monkeypatch, D, n, G):
    """The same kernel by another page lookup, split over workgroups and joined: the same roundings, whatever the compiler makes of either."""
    monkeypatch.setenv("XRMM_KV8_SHARED", "kv8_walk")
    c, d = shared_cache("int8", 40, [2700, 2600], 2, D, 64, seed=D, scales="any")
    q = torch.randn(2 * n, 2 * G, D, generator=torch.Generator().manual_seed(D + n)).half().cuda()
    kw = dict(batch=2, table_width=c.table.shape[1], page_size=64)
    assert ops().kv8_attention_workspace_bytes(2 * n, 2 * G, 2, D, **kw) > 4096  # split
    walked = ops().kv8_shared_attention(q, **d)
    assert torch.equal(walked, ops().kv8_attention(q, **c.dev()))
