"""Microscaled 4-bit products and attention over an 8-bit paged cache, as a
serving program calls them: what is timed, their plain forms and their exact
values.

MX4 is the 4-bit microscaling format: blocks of 32 values along the last axis,
E2M1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) and one E8M0 scale byte
(2^(byte - 127)) a block; codes are uint8 ``[..., kb, 16]``, low nibble first,
scales uint8 ``[..., kb]``. The cache holds pages ``[P, Hkv, page, D]`` of int8 or
float8_e4m3fn with one float32 scale for each page and head.

Four operators ("op"): "quantize" (mx4_quantize), "matmul" (matmul_mx4; with
act "mx4" the activations are quantised first, as such a layer does),
"append" (kv8_append) and "attention" (kv8_attention). Codes and scales that
an operator writes follow from comparisons and powers of two alone, so they
are whole numbers with one right value and are returned as they are held.
"""
import math

import torch

own = False


def listed():
    return [
        # one token's hidden state, quantised for a product of MX4 operands: the smallest call
        dict(name="quantize_token", op="quantize", dtype="bf16", M=1, K=4096),
        # a weight matrix as a model is loaded, in full precision, with a last block that is not whole
        dict(name="quantize_weight_f32", op="quantize", dtype="f32", M=14336, K=4090),
        # one token through an FFN up-projection
        dict(name="matmul_decode_m1", op="matmul", act="float", dtype="f16", M=1, K=4096, N=14336, bias=False),
        # a ragged continuous batch through the FFN down-projection
        dict(name="matmul_batch_m37", op="matmul", act="float", dtype="bf16", M=37, K=14336, N=4096, bias=False),
        # a long prompt through the up-projection, activations kept in 16 bits
        dict(name="matmul_prefill_m2048", op="matmul", act="float", dtype="f16", M=2048, K=4096, N=14336, bias=True),
        # prompts of several requests through the up-projection with both operands in MX4
        dict(name="matmul_mx4_prefill_m4096", op="matmul", act="mx4", dtype="bf16", M=4096, K=4096, N=14336,
             bias=False),
        # a decode batch of 64 sequences writes one token each
        dict(name="append_decode_b64", op="append", dtype="f16", cache="int8", B=64, new=1, ragged=False, Hkv=8, D=128,
             page=64, length=2048),
        # a prompt's keys and values enter the cache behind an earlier turn of the same conversation
        dict(name="append_prompt_4100", op="append", dtype="bf16", cache="e4m3", B=1, new=4100, ragged=False, Hkv=8,
             D=128, page=64, length=5000),
        # a short chat, one token: the smallest attention call
        dict(name="attention_decode_short", op="attention", dtype="f16", cache="int8", B=1, new=1, ragged=False, Hq=32,
             Hkv=8, D=64, page=16, length=200, window=0),
        # one sequence with a long context, one token
        dict(name="attention_decode_long", op="attention", dtype="f16", cache="int8", B=1, new=1, ragged=False, Hq=32,
             Hkv=8, D=128, page=64, length=65000, window=0),
        # a continuous batch of unequal contexts, one token each
        dict(name="attention_decode_b48", op="attention", dtype="bf16", cache="e4m3", B=48, new=1, ragged=True, Hq=32,
             Hkv=8, D=128, page=64, length=8000, window=0),
        # two prompts' chunks attend to themselves and to what their caches already hold
        dict(name="attention_prefill_2x2000", op="attention", dtype="f16", cache="int8", B=2, new=2000, ragged=True,
             Hq=32, Hkv=8, D=128, page=64, length=4000, window=0),
    ]


# The most work a drawn case of an operator has: the largest listed one's.
_MOST_MACS = {"float": 2048 * 4096 * 14336, "mx4": 4096 * 4096 * 14336}
_MOST_VALUES = 14336 * 4096        # quantize
_MOST_CACHE = 48 * 8000 * 8 * 128  # cached values of K in an attention or append call
_MOST_PAIRS = 2 * 2000 * 4000 * 32 * 128  # query tokens x context x heads x D


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("quantize", "matmul", "matmul", "matmul", "append", "attention", "attention", "attention"))
    dtype = rng.choice(("f16", "bf16"))
    if op == "quantize":
        K = _log(rng, 64, 14336)
        K = K if rng.random() < 0.3 else max(32, K // 32 * 32)
        return dict(op=op, dtype=rng.choice(("f16", "bf16", "f32")), M=_log(rng, 1, min(16384, _MOST_VALUES // K)), K=K)
    if op == "matmul":
        act = rng.choice(("float", "float", "mx4"))
        N, K = _log(rng, 256, 14336), _log(rng, 512, 14336)
        if rng.random() < 0.7:
            N, K = (N + 63) // 64 * 64, (K + 31) // 32 * 32
        M = max(1, min(_log(rng, 1, 4096), _MOST_MACS[act] // (K * N)))
        return dict(op=op, act=act, dtype=rng.choice((dtype, "f32")) if act == "mx4" else dtype, M=M, K=K, N=N,
                    bias=rng.random() < 0.4)
    D, page = rng.choice((64, 128, 128, 256, 96)), rng.choice((16, 32, 64, 64, 128, 256))
    Hkv, cache = rng.choice((1, 2, 4, 8, 8)), rng.choice(("int8", "e4m3"))
    B = _log(rng, 1, 64)
    length = _log(rng, 1, max(1, min(70000, _MOST_CACHE // (B * Hkv * D))))
    new = 1 if rng.random() < 0.5 else min(length, _log(rng, 2, 4100))
    ragged = rng.random() < 0.5
    if op == "append":
        return dict(op=op, dtype=rng.choice((dtype, "f32")), cache=cache, B=B, new=new, ragged=ragged, Hkv=Hkv, D=D,
                    page=page, length=length)
    Hq = Hkv * rng.choice((1, 2, 4, 5, 8))
    new = max(1, min(new, _MOST_PAIRS // (B * length * Hq * D)))
    return dict(op=op, dtype=dtype, cache=cache, B=B, new=new, ragged=ragged, Hq=Hq, Hkv=Hkv, D=D, page=page,
                length=length, window=_log(rng, 16, 4096) if rng.random() < 0.25 else 0)


# ---------------------------------------------------------------------------
# inputs

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_CT = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_QMAX = {"int8": 127.0, "e4m3": 448.0}


def _lengths(case):
    """Context lengths and new tokens of each sequence: plain arithmetic on the sizes, so that work() needs no tensor."""
    B, n, L = case["B"], case["new"], case["length"]
    if not case["ragged"]:
        return [L] * B, [n] * B
    lens = [max(1, L - (L * 3 * b) // (4 * B)) for b in range(B)]  # the whole length down to about a quarter
    return lens, [max(1, min(x, n - (n * b) // (2 * B))) for b, x in enumerate(lens)]


def _activations(case, g):
    """Normal values as after a normalisation, a few channels far larger, as hidden states have them."""
    x = torch.randn(case["M"], case["K"], device="cuda", generator=g)
    x[:, :: 509] *= 12.0
    return x.to(_DT[case["dtype"]])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "quantize":
        s["x"] = _activations(case, g)
        return s
    if case["op"] == "matmul":
        M, K, N = case["M"], case["K"], case["N"]
        out = _DT[case["dtype"]]
        s["A"] = _activations({**case, "dtype": "bf16"} if out == torch.float32 else case, g)
        w = torch.randn(N, K, device="cuda", generator=g) * 0.03
        s["B"], s["S"] = _quantize(w)  # as a model file holds it
        s["bias"] = (torch.randn(N, device="cuda", generator=g) * 0.1).to(out) if case["bias"] else None
        s["out"] = out
        return s
    lens, news = _lengths(case)
    B, Hkv, D, page = case["B"], case["Hkv"], case["D"], case["page"]
    width = max(-(-x // page) for x in lens)
    pages = B * width + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)[: B * width].view(B, width)
    used = torch.tensor([-(-x // page) for x in lens], device="cuda")
    s["table"] = torch.where(torch.arange(width, device="cuda") < used[:, None], order, -1)
    s["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda") if case["ragged"] else None
    s["counts"] = torch.tensor(news, device="cuda")
    s["max_new"] = max(news)
    shape = (pages, Hkv, page, D)
    for w in ("k", "v"):
        if case["cache"] == "int8":
            c = torch.randn(shape, device="cuda", generator=g).mul_(35).round_().clamp_(-127, 127).to(torch.int8)
        else:
            c = torch.randn(shape, device="cuda", generator=g).mul_(110).clamp_(-448, 448).to(torch.float8_e4m3fn)
        s[w + "_cache"] = c
        # powers of two, as kv8_append leaves them; in an attention case also those of another quantiser, max / qmax
        unit = 4.0 / _QMAX[case["cache"]] if case["op"] == "attention" else 2.0 ** (-5 if case["cache"] == "int8" else -7)
        s[w + "_scales"] = unit * 2.0 ** torch.randint(-1, 2, (pages, Hkv), device="cuda", generator=g).float()
    if case["op"] == "append":
        for w in ("k", "v"):
            s[w] = torch.randn(starts[-1], Hkv, D, device="cuda", generator=g).to(_DT[case["dtype"]])
    else:
        s["q"] = torch.randn(starts[-1], case["Hq"], D, device="cuda", generator=g).to(_DT[case["dtype"]])
    return s


# ---------------------------------------------------------------------------
# one pass

def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        from xrgpu_amd import ops
        if op == "quantize":
            return ops.mx4_quantize(s["x"])
        if op == "matmul":
            if c["act"] == "float":
                return ops.matmul_mx4(s["A"], s["B"], s["S"], s["bias"])
            codes, scales = ops.mx4_quantize(s["A"])
            return ops.matmul_mx4(codes, s["B"], s["S"], s["bias"], A_scales=scales, out_dtype=s["out"])
        cache = (s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["table"], s["lengths"])
        if op == "append":
            ops.kv8_append(s["k"], s["v"], *cache, starts=s["starts"], max_new=s["max_new"])
            return cache[:4]
        return ops.kv8_attention(s["q"], *cache, starts=s["starts"], max_new=s["max_new"], window=c["window"])
    if op == "quantize":
        return _quantize(s["x"])
    if op == "matmul":
        a = s["A"].float()
        if c["act"] == "mx4":
            a = _values(*_quantize(s["A"]))[:, : c["K"]]
        y = a @ _values(s["B"], s["S"])[:, : c["K"]].t()
        if s["bias"] is not None:
            y = y + s["bias"].float()
        return y.to(s["out"])
    if op == "append":
        for w in ("k", "v"):
            _append(s[w], s[w + "_cache"], s[w + "_scales"], s, _QMAX[c["cache"]])
        return s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"]
    return _attention(s)


# The plain forms: elementary torch operations in 32 bits.

def _quantize(x):
    K = x.shape[-1]
    kb = -(-K // 32)
    x = torch.nn.functional.pad(x.float(), (0, kb * 32 - K)).view(-1, kb, 32)
    bits = x.view(torch.int32)
    exponent = ((bits >> 23) & 255).amax(-1)  # the largest magnitude's: its floor(log2) + 127
    scale = (exponent - 2).clamp_min(0)
    inverse = ((254 - scale) << 23).view(torch.float32)
    y = (x * inverse[..., None]).abs()
    code = ((y > 0.25).int() + (y >= 0.75).int() + (y > 1.25).int() + (y >= 1.75).int() + (y > 2.5).int()
            + (y >= 3.5).int() + (y > 5.0).int()) | ((bits < 0).int() << 3)
    bad = exponent == 255
    code = torch.where(bad[..., None], 0, code)
    scale = torch.where(bad, 255, scale)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8), scale.to(torch.uint8)


def _values(codes, scales):
    """MX4 codes [n, kb, 16] and scales [n, kb] -> float32 [n, kb * 32]."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                         device=codes.device)
    nibbles = torch.stack((codes & 15, codes >> 4), -1).int().flatten(-2)
    s = scales.int()
    bits = torch.where(s == 0, 0x00400000, s << 23)  # 2^-127 is below the normal range
    scale = torch.where(s == 255, float("nan"), bits.view(torch.float32))
    return (table[nibbles] * scale[..., None]).flatten(-2)


def _power(r, qmax):
    """The smallest e >= -126 with r <= qmax 2^e, for finite r > 0."""
    e = (((r.view(torch.int32) >> 23) & 255) - 127 - int(math.floor(math.log2(qmax)))).clamp_min(-126)
    return torch.where(r > qmax * _two(e), e + 1, e)


def _two(e):
    return ((e + 127) << 23).view(torch.float32)  # 2^e, -126 <= e <= 127


def _append(x, cache, scales, s, qmax):
    page = cache.shape[2]
    B = s["lengths"].numel()
    seq = torch.repeat_interleave(torch.arange(B, device=x.device), s["counts"], output_size=x.shape[0])
    first = torch.cumsum(s["counts"], 0) - s["counts"]
    pos = s["lengths"].long()[seq] - s["counts"][seq] + torch.arange(x.shape[0], device=x.device) - first[seq]
    where, slot = s["table"][seq, pos // page].long(), pos % page
    x = x.float()
    top = x.abs().amax(-1)  # [T, Hkv]
    pages = torch.unique(where)
    at = torch.searchsorted(pages, where)
    amax = torch.zeros(pages.numel(), x.shape[1], device=x.device)
    amax.scatter_reduce_(0, at[:, None].expand_as(top), top, "amax")
    begin = torch.full((pages.numel(),), page, device=x.device).scatter_reduce_(0, at, slot, "amin")
    old = torch.where(begin[:, None] == 0, 0.0, scales[pages])
    fresh = old == 0
    some = amax.clamp_min(1e-45)
    grow = _power(torch.where(fresh, some, some / torch.where(fresh, 1.0, old)), qmax).clamp(-126, 120)
    grow = torch.where(fresh, grow, grow.clamp_min(0))
    new = torch.where(fresh, torch.where(amax > 0, _two(grow), 0.0), old * _two(torch.where(fresh, 0, grow)))
    shrink = torch.where(fresh, 1.0, _two(-torch.where(fresh, 0, grow)))
    held = cache[pages]
    kept = _round(held.float() * shrink[..., None, None], cache.dtype)
    there = torch.arange(page, device=x.device)[None, None, :, None] < begin[:, None, None, None]
    cache[pages] = torch.where(there, kept.view(torch.int8), held.view(torch.int8)).view(cache.dtype)
    scales[pages] = new
    div = new[at]
    y = torch.where(div[..., None] > 0, x / torch.where(div > 0, div, 1.0)[..., None], 0.0)
    cache.view(torch.int8)[where, :, slot] = _round(y.clamp(-qmax, qmax), cache.dtype).view(torch.int8)


def _round(x, dtype):
    return x.round().to(torch.int8) if dtype == torch.int8 else x.to(dtype)


def _attention(s):
    c = s["case"]
    B, Hq, Hkv, D = c["B"], c["Hq"], c["Hkv"], c["D"]
    n, q = s["max_new"], s["q"]
    table = s["table"].long().clamp_min(0)
    # the cache of each sequence, side by side: [B, Hkv, width * page, D]
    k, v = ((s[w + "_cache"][table].float() * s[w + "_scales"][table][..., None, None]).transpose(1, 2).flatten(2, 3)
            for w in ("k", "v"))
    row = torch.arange(n, device=q.device)
    first = torch.cumsum(s["counts"], 0) - s["counts"]
    have = row < s["counts"][:, None]  # [B, n]: ragged queries, padded
    take = (first[:, None] + row).clamp_max(q.shape[0] - 1)
    qp = q[take].float().transpose(1, 2).reshape(B, Hkv, (Hq // Hkv) * n, D)
    pos = s["lengths"].long()[:, None] - s["counts"][:, None] + row
    t = torch.arange(k.shape[2], device=q.device)
    seen = t <= pos[..., None]  # [B, n, L]
    if c["window"]:
        seen &= t > pos[..., None] - c["window"]
    p = (qp @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(D)).view(B, Hkv, Hq // Hkv, n, -1)
    p = p.masked_fill_(~seen[:, None, None], float("-inf"))
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = (p.flatten(2, 3) @ v).view(B, Hq, n, D).transpose(1, 2)  # [B, n, Hq, D]
    return o[have].to(q.dtype)


# ---------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    op = case["op"]
    size = {"f16": 2, "bf16": 2, "f32": 4}[case["dtype"]]
    if op == "quantize":
        M, K = case["M"], case["K"]
        return {"bytes": M * K * size + M * -(-K // 32) * 17, "flops": 0}
    if op == "matmul":
        M, K, N = case["M"], case["K"], case["N"]
        kb = -(-K // 32)
        return {"bytes": M * K * 2 + N * kb * 17 + M * N * size + (N * size if case["bias"] else 0),
                "flops": 2 * M * N * K}
    lens, news = _lengths(case)
    Hkv, D, page = case["Hkv"], case["D"], case["page"]
    if op == "append":
        return {"bytes": sum(news) * 2 * Hkv * D * (size + 1), "flops": 0}
    pairs = held = 0
    for L, n in zip(lens, news):
        w = case["window"] or L
        seen = [min(w, L - n + i + 1) for i in range(n)]
        pairs += sum(seen)
        held += min(L, w + n - 1)
    table = sum(-(-x // page) for x in lens)
    return {"bytes": 2 * Hkv * (held * D + 4 * table) + 4 * table + 2 * sum(news) * case["Hq"] * D * size,
            "flops": 4 * D * case["Hq"] * pairs}


# ---------------------------------------------------------------------------
# the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_quantize(s["x"].double())
    if op == "matmul":
        a = s["A"].double()
        if case["act"] == "mx4":
            a = _exact_decode(*_exact_quantize(a))[:, : case["K"]]
        y = torch.matmul(a, _exact_decode(s["B"], s["S"])[:, : case["K"]].T)
        return y if s["bias"] is None else y + s["bias"].double()
    lens, news = _lengths(case)
    page, D, Hkv = case["page"], case["D"], case["Hkv"]
    table = s["table"].tolist()
    at = 0
    if op == "append":
        if sum(-(-n // page) + 1 for n in news) * Hkv > 6000:
            return None  # a loop over pages and heads would take too long
        held = {w: [s[w + "_cache"].float().double(), s[w + "_scales"].double()] for w in ("k", "v")}
        for b, (L, n) in enumerate(zip(lens, news)):
            p = L - n
            while p < L:
                stop = min(L, (p // page + 1) * page)
                for w in ("k", "v"):
                    x = s[w][at + p - (L - n): at + stop - (L - n)].double()
                    _exact_page(x, held[w], table[b][p // page], p % page, case["cache"])
                p = stop
            at += n
        (k, ks), (v, vs) = held["k"], held["v"]
        dt = _CT[case["cache"]]
        return k.to(torch.float32).to(dt), v.to(torch.float32).to(dt), ks, vs
    out = torch.empty(sum(news), case["Hq"], D, dtype=torch.float64, device="cuda")
    G = case["Hq"] // Hkv
    for b, (L, n) in enumerate(zip(lens, news)):
        used = torch.tensor(table[b][: -(-L // page)], device="cuda")
        i = torch.arange(L - n, L, device="cuda")[:, None]
        j = torch.arange(L, device="cuda")[None]
        gone = j > i
        if case["window"]:
            gone = gone | (i - j >= case["window"])
        for h in range(Hkv):
            k, v = ((s[w + "_cache"][used, h].float().double() * s[w + "_scales"][used, h].double()[:, None, None])
                    .reshape(-1, D)[:L] for w in ("k", "v"))
            for g in range(G):
                z = torch.matmul(s["q"][at: at + n, h * G + g].double(), k.T) / math.sqrt(D)
                out[at: at + n, h * G + g] = torch.matmul(torch.softmax(z.masked_fill(gone, -math.inf), -1), v)
        at += n
    return out


_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _two64(e):
    """2^e in 64 bits, from its bits: a device pow need not be exact."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_quantize(x):
    n, K = x.shape
    kb = (K + 31) // 32
    z = torch.zeros(n, kb * 32, dtype=torch.float64, device=x.device)
    z[:, :K] = x
    z = z.reshape(n, kb, 32)
    most = z.abs().amax(-1)
    _, e = torch.frexp(most)  # most = m 2^e, 0.5 <= m < 1
    e = torch.where(most > 0, e - 3, -127).clamp(-127, 127)
    u = z.abs() / _two64(e)[..., None]
    # the nearest grid value; of two equally near, the one with an even code
    code = torch.zeros_like(u, dtype=torch.int64)
    for i in range(7):
        mid = (_GRID[i] + _GRID[i + 1]) / 2
        code += ((u >= mid) if i % 2 else (u > mid)).long()
    code += 8 * torch.signbit(z).long()
    return (code[..., ::2] + 16 * code[..., 1::2]).to(torch.uint8), (e + 127).to(torch.uint8)


def _exact_decode(codes, scales):
    c = codes.long()
    c = torch.stack((c % 16, c // 16), -1).reshape(*scales.shape, 32)
    v = torch.tensor(_GRID, dtype=torch.float64, device=codes.device)[c % 8] * (1.0 - 2.0 * (c >= 8).double())
    return (v * _two64(scales.long() - 127)[..., None]).reshape(scales.shape[0], -1)


def _exact_page(x, held, p, slot, kind):
    """New tokens x [n, Hkv, D] enter page p from `slot` on; held: [codes, scales] as float64."""
    codes, scales = held
    for h in range(x.shape[1]):
        most, old = float(x[:, h].abs().max()), 0.0 if slot == 0 else float(scales[p, h])
        base = old if old else 1.0
        e = -126
        if most:
            e = max(-126, math.frexp(most / base)[1] - 1 - (6 if kind == "int8" else 8))
            while most / base > _QMAX[kind] * 2.0 ** e:
                e += 1
        if old:
            e = max(e, 0)
            codes[p, h, :slot] = _exact_round(codes[p, h, :slot] / 2.0 ** e, kind)
        scales[p, h] = base * 2.0 ** e if old or most else 0.0
        now = float(scales[p, h])
        codes[p, h, slot: slot + x.shape[0]] = _exact_round(x[:, h] / now, kind) if now else 0.0


def _exact_round(y, kind):
    if kind == "int8":
        return torch.round(y)
    step = _two64((torch.frexp(y.abs())[1] - 1).clamp_min(-6) - 3)  # e4m3: 3 bits behind the first
    return torch.round(y / step) * step
