"""One decoder layer with MX4 weights and a paged 8-bit cache: a batch of prompts, then single tokens from a captured graph.

    python examples/mx4_decoder_layer.py

The weights are quantised once (``mx4_quantize``). A call takes its sequences' new tokens, prompts of any lengths or one token each:
projections of queries, keys and values in one product (``matmul_mx4``), keys and values into the cache from where
the product left them (``kv8_append`` takes a token stride), attention (``kv8_attention``), and the feed-forward
products. With ``act4``, the products of more than 16 rows quantise their activations too and run on 4-bit operands.
"""
import os
import sys
from dataclasses import dataclass

import torch

if __name__ == "__main__":
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from xrgpu_amd import ops  # noqa: E402


@dataclass
class Config:
    hidden: int = 4096
    q_heads: int = 32
    kv_heads: int = 8
    head_dim: int = 128
    ffn: int = 14336
    page: int = 64
    eps: float = 1e-5
    theta: float = 500000.0
    dtype: torch.dtype = torch.bfloat16
    cache: torch.dtype = torch.int8
    act4: bool = False

    def products(self):
        """name -> (N, K)"""
        heads = self.q_heads + 2 * self.kv_heads
        return {"qkv": (heads * self.head_dim, self.hidden), "out": (self.hidden, self.q_heads * self.head_dim),
                "up": (2 * self.ffn, self.hidden), "down": (self.hidden, self.ffn)}


class Cache:
    """Pages of the 8-bit cache, handed out to sequences in order; ``table`` names each sequence's."""

    def __init__(self, cfg, batch, tokens, device="cuda"):
        width = -(-tokens // cfg.page)
        pages = batch * width
        shape = (pages, cfg.kv_heads, cfg.page, cfg.head_dim)
        self.k, self.v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(cfg.cache) for _ in range(2))
        self.ks, self.vs = (torch.zeros(pages, cfg.kv_heads, device=device) for _ in range(2))
        self.table = torch.arange(pages, dtype=torch.int32, device=device).view(batch, width)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)  # 55 once a token had no page

    def tensors(self):
        return self.k, self.v, self.ks, self.vs, self.table, self.lengths


def rms_norm(x, gamma, eps):
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + eps) * gamma).to(x.dtype)


def rotate(x, positions, theta):
    """Each head's halves as the two parts of complex numbers, turned by position * theta^(-2 i / D)."""
    half = x.shape[-1] // 2
    freq = theta ** (-torch.arange(half, device=x.device, dtype=torch.float64) / half)
    angle = positions[:, None, None].double() * freq  # far positions lose their angle in 32 bits
    c, s = angle.cos().float(), angle.sin().float()
    a, b = x[..., :half].float(), x[..., half:].float()
    return torch.cat((a * c - b * s, b * c + a * s), -1).to(x.dtype)


class Layer:
    def __init__(self, cfg, weights):
        """weights: float tensors ``[N, K]`` of ``cfg.products()``."""
        self.cfg = cfg
        self.w = {n: ops.mx4_quantize(weights[n]) for n in cfg.products()}
        self.gamma = [torch.ones(cfg.hidden, device="cuda") for _ in range(2)]

    def workspace(self, cache):
        """A workspace for captured calls of one token a sequence; eager calls use the library's own, by stream."""
        c = self.cfg
        batch, width = cache.table.shape
        at = torch.uint8 if c.act4 and batch > 16 else c.dtype
        need = [ops.matmul_mx4_workspace_bytes(batch, K, N, at) for N, K in c.products().values()]
        need.append(ops.kv8_attention_workspace_bytes(batch, c.q_heads, c.kv_heads, c.head_dim, batch=batch, table_width=width,
                                                      page_size=c.page))
        return torch.zeros(max(need), dtype=torch.uint8, device="cuda") if max(need) else None

    def product(self, x, name, workspace):
        codes, scales = self.w[name]
        if self.cfg.act4 and x.shape[0] > 16:
            a, s = ops.mx4_quantize(x)
            return ops.matmul_mx4(a, codes, scales, A_scales=s, out_dtype=x.dtype, workspace=workspace)
        return ops.matmul_mx4(x, codes, scales, workspace=workspace)

    def __call__(self, x, cache, starts=None, max_new=None, workspace=None):
        """x ``[T, hidden]``: the new tokens, one a sequence without ``starts``; ``cache.lengths`` counts them already."""
        c = self.cfg
        T = x.shape[0]
        if starts is None:
            positions = cache.lengths - 1
        else:
            t = torch.arange(T, dtype=torch.int32, device=x.device)
            b = torch.searchsorted(starts[1:], t, right=True)
            positions = cache.lengths[b] - starts[1:][b] + t
        qkv = self.product(rms_norm(x, self.gamma[0], c.eps), "qkv", workspace).view(T, -1, c.head_dim)
        q, k, v = qkv.split((c.q_heads, c.kv_heads, c.kv_heads), 1)
        q, k = rotate(q, positions, c.theta), rotate(k, positions, c.theta)
        ops.kv8_append(k, v, *cache.tensors(), starts=starts, max_new=max_new, status=cache.status)
        o = ops.kv8_attention(q, *cache.tensors(), starts=starts, max_new=max_new, workspace=workspace, status=cache.status)
        x = x + self.product(o.view(T, -1), "out", workspace)
        gate, up = self.product(rms_norm(x, self.gamma[1], c.eps), "up", workspace).split(c.ffn, 1)
        return x + self.product((torch.nn.functional.silu(gate.float()) * up.float()).to(x.dtype), "down", workspace)


def prompt(layer, cache, xs):
    """The prompts ``xs`` (one ``[n, hidden]`` a sequence) in one call; each sequence's last row of the result."""
    counts = [x.shape[0] for x in xs]
    starts = torch.tensor([0, *torch.tensor(counts).cumsum(0)], dtype=torch.int32, device="cuda")
    cache.lengths += starts[1:] - starts[:-1]
    y = layer(torch.cat(xs), cache, starts, max(counts))
    return y[starts[1:].long() - 1]


class Decoder:
    """Steps of one token a sequence from a graph. The graph holds the lengths' increment too, so a replay is a step."""

    def __init__(self, layer, cache, x):
        self.x = x.clone()
        self.cache = cache
        self.workspace = layer.workspace(cache)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            cache.lengths += 1
            self.y = layer(self.x, cache, workspace=self.workspace)

    def step(self, x):
        self.x.copy_(x)
        self.graph.replay()
        return self.y


def random_weights(cfg, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    return {n: torch.randn(N, K, generator=g, device="cuda") * K ** -0.5 for n, (N, K) in cfg.products().items()}


def main():
    for act4 in (False, True):
        cfg = Config(act4=act4)
        lens = (700, 1000, 64, 333)
        layer = Layer(cfg, random_weights(cfg))
        cache = Cache(cfg, len(lens), 2048)
        xs = [torch.randn(n, cfg.hidden, device="cuda").to(cfg.dtype) for n in lens]
        y = prompt(layer, cache, xs)
        decoder = Decoder(layer, cache, y)
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        y = decoder.step(y)
        a.record()
        for _ in range(100):
            y = decoder.step(y)
        b.record()
        torch.cuda.synchronize()
        assert cache.status.item() == 0 and y.isfinite().all()
        print(f"{'4-bit' if act4 else '16-bit'} activations: lengths {cache.lengths.tolist()}, "
              f"{a.elapsed_time(b) * 10:.1f} us a step of {len(lens)} tokens", flush=True)


if __name__ == "__main__":
    main()
