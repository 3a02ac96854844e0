"""GPU: attention of many rows on its tile kernel, the kernel asserted; tolerances as in test_gpu_kv8_scales.py."""
import numpy as np
import pytest

from tests.test_gpu_kv8 import Cache, ops, starts_of
from tests.test_gpu_kv8_scales import check, kernel_of, queries

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

# lens, counts, Hq, Hkv, D, page, window
TILES = [([300, 280], [300, 200], 32, 8, 64, 16, 0), ([300, 77], [130, 77], 64, 8, 96, 32, 0), ([401, 300], [200, 150], 32, 8, 128, 64, 0),
         ([500, 390, 64], [200, 150, 1], 32, 8, 128, 256, 0), ([257, 256], [257, 256], 40, 8, 256, 128, 0), ([330, 9], [300, 60], 56, 8, 128, 32, 0),
         ([600, 500], [256, 129], 64, 8, 64, 16, 100), ([600, 500], [256, 129], 64, 8, 256, 16, 33), ([390, 200], [390, 200], 48, 6, 96, 64, 1),
         ([257, 130], [257, 130], 24, 24, 128, 16, 0), ([300, 0, 128], [250, 0, 128], 64, 4, 64, 128, 0)]


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("lens,counts,Hq,Hkv,D,page,window", TILES)
def test_tile(gpu, kind, dt, lens, counts, Hq, Hkv, D, page, window):
    c = Cache(kind, lens, Hkv, D, page, seed=sum(lens) + D, scales="any" if D % 128 else "pow2")
    check(c, queries(sum(counts), Hq, D, dt), counts, window=window, kernel="kv8_tile")


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_not_causal_and_other_scales(gpu, kind, D):
    c = Cache(kind, [230, 161], 8, D, 32, seed=8)
    q = queries(300, 64, D, "f16")
    check(c, q, [200, 100], causal=False, kernel="kv8_tile")
    check(c, q, [200, 100], causal=False, window=20, scale=0.25, kernel="kv8_tile")
    check(c, q, [200, 100], scale=-0.1, kernel="kv8_tile")
    check(c, q, [200, 100], scale=0.0, kernel="kv8_tile")


def test_sharp_and_spread_scales(gpu):
    c = Cache("int8", [300], 8, 64, 16, seed=9)
    c.vs[c.table[0, ::2]] *= np.float32(2.0 ** -12)
    c.vs[c.table[0, 3]] = 0
    c.ks[c.table[0, 5]] = 0
    q = (queries(300, 32, 64, "bf16") * 6).bfloat16()
    check(c, q, [300], kernel="kv8_tile")
    c.vs[:] = 0
    assert not check(c, q, [300], kernel="kv8_tile").any()


@pytest.mark.parametrize("dt,big", [("f16", 6e4), ("bf16", 1e30), ("bf16", 1e-30), ("f16", 6e-8)])
def test_extreme_queries(gpu, dt, big):
    c = Cache("e4m3", [300], 8, 64, 16, seed=10)
    q = (torch.randn(300, 32, 64, generator=torch.Generator().manual_seed(1)).clamp(-1, 1).double() * big).to({"f16": torch.float16, "bf16": torch.bfloat16}[dt]).cuda()
    check(c, q, [300], scale=1.0 / (64 * big), kernel="kv8_tile")


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D", [64, 96, 256])
def test_reads_nothing_past_the_tokens(gpu, kind, D):
    """Slots past a length and pages that no token lies in hold NaN codes and scales."""
    c = Cache(kind, [275, 150], 8, D, 32, seed=11)
    q = queries(350, 32, D, "f16")
    clean = check(c, q, [250, 100], kernel="kv8_tile")
    used = set()
    for b, L in enumerate(c.lengths):
        used |= {int(c.table[b, i]) for i in range(-(-int(L) // 32))}
        last = c.table[b, (int(L) - 1) // 32]
        c.k[last, :, (int(L) - 1) % 32 + 1:] = 0x7F
        c.v[last, :, (int(L) - 1) % 32 + 1:] = 0x7F
    for p in set(range(c.k.shape[0])) - used:
        c.k[p], c.v[p], c.ks[p], c.vs[p] = 0xFF, 0xFF, np.nan, np.inf
    assert torch.equal(ops().kv8_attention(q, **c.dev(), starts=starts_of([250, 100]), max_new=250), clean)


def test_nonfinite_scales_and_queries_stay_apart(gpu):
    c = Cache("int8", [300, 300], 8, 64, 32, seed=12)
    c.vs[c.table[0, 8], 1] = np.nan  # tokens 256 .. 287 of the first sequence, head 1
    q = queries(500, 32, 64, "f16")
    q[250 + 125, 0, 3] = float("nan")
    assert kernel_of(c, q, [250, 250], ragged=False) == "kv8_tile"
    o = ops().kv8_attention(q, **c.dev())
    nan = torch.zeros(500, 32, dtype=torch.bool, device="cuda")
    nan[206:250, 4:8] = True  # positions from 256 on
    nan[375, 0] = True
    assert torch.equal(o.isnan().any(-1), nan) and torch.equal(o.isnan().all(-1), nan)


def test_pages_that_do_not_exist_and_lengths_past_the_table(gpu):
    q = queries(280, 64, 64, "f16")
    for p in (-1, 1 << 30):
        c = Cache("int8", [300], 8, 64, 16, seed=13)
        c.table[0, 4] = p
        check(c, q, [280], status=55, kernel="kv8_tile")
    c = Cache("int8", [300], 8, 64, 16, seed=13)
    c.lengths[0] = 330
    check(c, q, [280], status=55, kernel="kv8_tile")


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_queries_and_outputs_at_any_element(gpu, dt, D):
    n, Hq = 210, 32
    c = Cache("int8", [250, 230], 8, D, 32, seed=D)
    wide = torch.randn(2 * n, Hq * D + 3, device="cuda").to({"f16": torch.float16, "bf16": torch.bfloat16}[dt])
    q = wide[:, 1:1 + Hq * D].unflatten(1, (Hq, D))
    store = torch.full((2 * n * Hq * D + 3,), 7.0, device="cuda").to(q.dtype)
    check(c, q, [n, n], out=store[1:-2].view(2 * n, Hq, D), kernel="kv8_tile")
    assert (store[0] == 7) and (store[-2:] == 7).all()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_graph_stream_and_repeats(gpu, kind):
    n, Hq, Hkv, D = 200, 32, 8, 128
    c = Cache(kind, [400, 280], Hkv, D, 64, seed=15)
    d = c.dev()
    q = queries(2 * n, Hq, D, "bf16")
    first = check(c, q, [n, n], d=d, kernel="kv8_tile")
    for _ in range(3):
        assert torch.equal(ops().kv8_attention(q, **d), first)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    y = ops().kv8_attention(q, **d, stream=st)
    st.synchronize()
    assert torch.equal(y, first)
    need = ops().kv8_attention_workspace_bytes(2 * n, Hq, Hkv, D, batch=2, table_width=d["block_table"].shape[1], page_size=64)
    assert need > 0
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    for kw in ({}, {"workspace": ws}):  # without a workspace of its own a captured call runs unsplit
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops().kv8_attention(q, **d, **kw)
        for i in range(3):
            q.copy_(queries(2 * n, Hq, D, "bf16", seed=i + 1))
            graph.replay()
            torch.cuda.synchronize()
            eager = ops().kv8_attention(q, **d)
            if kw:
                same = torch.equal(out, eager)
                assert same
            check(c, q, [n, n], got=out.clone())
    assert not ws[:4096].any()
