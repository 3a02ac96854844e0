"""GPU: the example layer runs the MX4 and 8-bit cache operators together, each call checked against oracle/lowbit.py.

Every operator's call is compared on its own inputs, with the tolerances of test_gpu_mx4.py and test_gpu_kv8.py; the
graph's steps are compared with eager calls of the same kernels bit for bit.
"""
import importlib.util
import os

import numpy as np
import pytest

from oracle import lowbit as LB

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def load(name, *path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    spec = importlib.util.spec_from_file_location(name, os.path.join(root, *path))
    m = importlib.util.module_from_spec(spec)
    import sys
    sys.modules[name] = m
    spec.loader.exec_module(m)
    return m


class Checked:
    """The operators, each call checked; `seen` counts them."""

    def __init__(self):
        from xrgpu_amd import ops
        self.ops = ops
        self.mx4 = load("_mx4_checks", "tests", "test_gpu_mx4.py")
        self.kv8 = load("_kv8_checks", "tests", "test_gpu_kv8.py")
        self.seen = {}

    def _count(self, name):
        self.seen[name] = self.seen.get(name, 0) + 1

    def mx4_quantize(self, x):
        self._count("quantize")
        codes, scales = self.ops.mx4_quantize(x)
        c, s = LB.mx4_quantize(x.double().cpu().numpy())
        assert np.array_equal(codes.cpu().numpy(), c) and np.array_equal(scales.cpu().numpy(), s)
        return codes, scales

    def matmul_mx4(self, A, codes, scales, *, A_scales=None, out_dtype=None, workspace=None):
        self._count("product" if A_scales is None else "product of 4-bit operands")
        y = self.ops.matmul_mx4(A, codes, scales, A_scales=A_scales, out_dtype=out_dtype, workspace=workspace)
        a = A.double().cpu().numpy() if A_scales is None else LB.mx4_decode(A.cpu().numpy(), A_scales.cpu().numpy())
        self.mx4.check_product(a, codes, scales, None, y)
        return y

    def _cache(self, k, v, ks, vs, table, lengths, kind):
        c = type("C", (), {})()
        c.kind, c.k, c.v = kind, k.view(torch.uint8).cpu().numpy(), v.view(torch.uint8).cpu().numpy()
        c.ks, c.vs, c.table, c.lengths = (t.cpu().numpy().copy() for t in (ks, vs, table, lengths))
        c.dev = lambda: dict(k_cache=k, v_cache=v, k_scales=ks, v_scales=vs, block_table=table, lengths=lengths)
        return c

    def _counts(self, T, lengths, starts):
        return [T // len(lengths)] * len(lengths) if starts is None else starts.diff().tolist()

    def kv8_append(self, k, v, *cache, starts=None, max_new=None, status=None):
        self._count("append")
        kind = "int8" if cache[0].dtype == torch.int8 else "e4m3"
        self.kv8.check_append(self._cache(*cache, kind), k, v, self._counts(k.shape[0], cache[5], starts), starts is not None,
                              max_new=max_new)

    def kv8_attention(self, q, *cache, starts=None, max_new=None, workspace=None, status=None):
        self._count("attention")
        kind = "int8" if cache[0].dtype == torch.int8 else "e4m3"
        c = self._cache(*cache, kind)
        got = self.ops.kv8_attention(q, *cache, starts=starts, max_new=max_new, workspace=workspace, status=status)
        self.kv8.check_attention(c, q, self._counts(q.shape[0], cache[5], starts), starts is not None, d=c.dev(), got=got)
        return got


SMALL = dict(hidden=256, q_heads=8, kv_heads=2, head_dim=64, ffn=416, page=16)


def make(ex, **kw):
    cfg = ex.Config(**{**SMALL, **kw})
    return cfg, ex.random_weights(cfg)


@pytest.mark.parametrize("act4", [False, True])
@pytest.mark.parametrize("cache,dt", [("int8", "bf16"), ("e4m3", "f16")])
def test_every_call_of_prompt_and_steps(gpu, cache, dt, act4):
    ex = load("_mx4_decoder_layer", "examples", "mx4_decoder_layer.py")
    dt = {"f16": torch.float16, "bf16": torch.bfloat16}[dt]
    cfg, w = make(ex, act4=act4, dtype=dt, cache={"int8": torch.int8, "e4m3": torch.float8_e4m3fn}[cache])
    ex.ops = checked = Checked()
    layer = ex.Layer(cfg, w)
    kv = ex.Cache(cfg, 3, 64)
    g = torch.Generator().manual_seed(3)
    y = ex.prompt(layer, kv, [torch.randn(n, cfg.hidden, generator=g).to(dt).cuda() for n in (23, 1, 40)])
    for _ in range(3):
        kv.lengths += 1
        y = layer(y, kv)
    assert y.isfinite().all() and kv.lengths.tolist() == [26, 4, 43] and kv.status.item() == 0
    assert checked.seen.pop("quantize") == (8 if act4 else 4)
    assert checked.seen == {"append": 4, "attention": 4, "product": 12 if act4 else 16,
                            **({"product of 4-bit operands": 4} if act4 else {})}


@pytest.mark.parametrize("batch", [3, 20])
def test_graph_steps_equal_eager_ones(gpu, batch):
    ex = load("_mx4_decoder_layer", "examples", "mx4_decoder_layer.py")
    cfg, w = make(ex, hidden=1024, act4=batch > 16)
    layer = ex.Layer(cfg, w)
    caches = [ex.Cache(cfg, batch, 512) for _ in range(2)]
    g = torch.Generator().manual_seed(4)
    xs = [torch.randn(50 + 17 * i, cfg.hidden, generator=g).to(cfg.dtype).cuda() for i in range(batch)]
    y, z = (ex.prompt(layer, c, xs) for c in caches)
    assert torch.equal(y, z)
    decoder = ex.Decoder(layer, caches[1], z)
    assert torch.equal(caches[0].lengths, caches[1].lengths)
    for _ in range(20):
        caches[0].lengths += 1
        y = layer(y, caches[0])
        torch.cuda.synchronize()
        z = decoder.step(z).clone()
        assert torch.equal(y, z)
    for a, b in zip(caches[0].tensors(), caches[1].tensors(), strict=True):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_the_example_runs(gpu, capsys):
    load("_mx4_decoder_layer", "examples", "mx4_decoder_layer.py").main()
    assert "lengths [801, 1101, 165, 434]" in capsys.readouterr().out
