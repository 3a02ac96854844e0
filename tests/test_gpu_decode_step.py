"""GPU: rope, kv8_append, kv8_shared_attention, a product and sample, as a step of several answers to one prompt runs them."""
import numpy as np
import pytest

from oracle import decode as DC
from tests.test_gpu_kv8 import check_append, check_attention
from tests.test_gpu_kv8_shared import shared_cache
from tests.test_gpu_mx4_decoder_layer import SMALL, load
from tests.test_gpu_rope import check as check_rope
from tests.test_gpu_sample import check as check_sample

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def ops():
    from xrgpu_amd import ops as _ops
    return _ops


@pytest.mark.parametrize("kind,dt,B,shared", [("int8", torch.float16, 5, 6), ("e4m3", torch.bfloat16, 40, 20)])
def test_a_step_call_by_call(gpu, kind, dt, B, shared):
    """Heads turned in place in the rows of one product, appended from there, attended over a shared prefix, drawn from; three tokens."""
    o, H, Hq, D, page, V = ops(), 2, 8, 64, 32, 1500
    lens = [shared * page + 3 + 5 * b for b in range(B)]
    c, d = shared_cache(kind, shared, [n + 3 for n in lens], H, D, page, seed=B)
    given = d["block_table"]
    pages = d.pop("shared_pages")
    d["block_table"] = torch.from_numpy(c.table.copy()).cuda()
    f, m = o.rope_frequencies(D, scaling="yarn", factor=4.0, original_length=64)
    w = (torch.randn(V, Hq * D, generator=torch.Generator().manual_seed(1)) * 0.2).to(dt).cuda()
    c.lengths = np.array(lens, np.int32)
    for step in range(3):
        g = torch.Generator().manual_seed(step)
        qkv = torch.randn(B, (Hq + 2 * H) * D, generator=g).to(dt).cuda()
        q, k, v = qkv.view(B, -1, D).split((Hq, H, H), 1)
        before = [x.clone() for x in (q, k, v)]
        c.lengths = c.lengths + np.int32(1)
        d["lengths"].copy_(torch.from_numpy(c.lengths))
        o.rope(q, k, frequencies=f, magnitude=m, lengths=d["lengths"], out=q, k_out=k)
        for x, y in zip(before, (q, k)):
            check_rope(x, y.contiguous(), c.lengths - 1, f, magnitude=m)
        assert torch.equal(v, before[2])
        c.dev = lambda: d
        check_append(c, k, v, [1] * B, False)
        y = o.kv8_shared_attention(q, **{**d, "block_table": given}, shared_pages=pages)
        check_attention(c, q, [1] * B, False, d=d, got=y)
        logits = y.view(B, -1) @ w.t()
        check_sample(logits, torch.rand(B, generator=g).cuda(), temperature=0.7, top_k=40, top_p=0.9123)


@pytest.mark.parametrize("cache", ["int8", "e4m3"])
def test_the_steps_from_a_graph_are_the_eager_ones(gpu, cache):
    """The whole step captured, with the lengths' increment: three replays, eager work between them."""
    ex = load("_decoder_layer_for_steps", "examples", "mx4_decoder_layer.py")
    cfg = ex.Config(**SMALL, cache={"int8": torch.int8, "e4m3": torch.float8_e4m3fn}[cache])
    B, n, V = 12, 100, 700
    layer = ex.Layer(cfg, ex.random_weights(cfg))
    head = ex.Head(cfg, torch.randn(V, cfg.hidden, generator=torch.Generator("cuda").manual_seed(2), device="cuda"))
    caches = []
    for _ in range(2):
        c = ex.Cache(cfg, B, n + 40)
        first = ex.Cache.__new__(ex.Cache)
        first.__dict__.update(c.__dict__, table=c.table[:1], lengths=c.lengths[:1])
        y = ex.prompt(layer, first, [torch.randn(n, cfg.hidden, generator=torch.Generator("cuda").manual_seed(3), device="cuda").to(cfg.dtype)])
        c.share()
        assert c.shared.numel() == n // cfg.page and (c.lengths == n).all()
        caches.append(c)
    start = y.expand(B, -1).contiguous()
    u = torch.zeros(B, device="cuda")
    kw = dict(temperature=0.9, top_k=30, top_p=0.95)
    ws, own = head.workspace(B), layer.workspace(caches[0])

    def step(x, cache):
        t, e = head(x, u, ws, **kw)
        cache.lengths += 1
        return t, layer(e, cache, workspace=own)

    x = start.clone()
    state = [t.clone() for t in caches[0].tensors()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, out = step(x, caches[0])
    for t, s in zip(caches[0].tensors(), state):
        t.copy_(s)
    eager = start.clone()
    for i in range(3):
        u.copy_(torch.rand(B, generator=torch.Generator().manual_seed(i)))
        x.copy_(eager)
        graph.replay()
        torch.cuda.synchronize()
        want, eager = step(eager, caches[1])
        assert torch.equal(tokens, want) and torch.equal(out, eager)
        for a, b in zip(caches[0].tensors(), caches[1].tensors()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert caches[0].status.item() == 0 and caches[1].status.item() == 0


def test_answers_run(gpu):
    ex = load("_decoder_layer_for_answers", "examples", "mx4_decoder_layer.py")
    t = ex.answers(ex.Config(**SMALL), batch=6, tokens=70, vocab=500, steps=5, temperature=1.0, top_k=20)
    assert tuple(t.shape) == (5, 6) and t.dtype == torch.int32 and (t >= 0).all() and (t < 500).all()
    same = ex.answers(ex.Config(**SMALL), batch=6, tokens=70, vocab=500, steps=5, temperature=1.0, top_k=20)
    assert torch.equal(t, same)
    greedy = ex.answers(ex.Config(**SMALL), batch=6, tokens=70, vocab=500, steps=5, temperature=0.0)
    assert (greedy[0] == greedy[0, 0]).all()
