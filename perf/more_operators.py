"""What a decode step calls around its products and its cache: rotary positions, attention of a batch that shares
a long prefix, and the draw of the next tokens: what is timed, the plain forms and the exact values.

Three operators ("op"):

"rope" (rope): value pairs (a, b) of each head, turned by the angle position * frequency of their pair:
(a cos - b sin, b cos + a sin), times a magnitude that some scalings for long contexts have; pair i is (i, i + R / 2) of a head's
first R values, or (2 i, 2 i + 1) ("interleaved"); the values behind R pass. "inverse" turns back: the gradient's direction.

"shared" (kv8_shared_attention): attention over the paged 8-bit cache where the first tokens of every sequence of the batch lie in
the same pages.

"sample" (sample): a token for each row of logits, by a given number u in [0, 1): weights exp((x - max) / temperature), of
the top_k largest logits (of equal ones those of the lowest index), of those the shortest prefix in descending order
that holds top_p of their weight, of those the ones of at least min_p of the largest weight; then the first token, by index, at which the
running sum of the kept weights passes u of their total. Temperature 0 takes the largest. Also the logarithm of the drawn
token's share. NaN counts as -infinity.
"""
import math

import torch

own = False


def listed():
    return [
        # one token of a chat: the smallest call
        dict(name="rope_token", op="rope", dtype="bf16", B=1, new=1, ragged=False, given=True, Hq=32, Hk=8, D=128, R=128,
             interleaved=False, inverse=False, length=1500),
        # a decode batch, its queries and keys in the rows of one product, positions from the cache's lengths; part of a head turns
        dict(name="rope_decode_b96", op="rope", dtype="f16", B=96, new=1, ragged=False, given=False, Hq=24, Hk=8, D=96, R=64,
             interleaved=True, inverse=False, length=30000),
        # prompts of several requests in one call, far into a long context
        dict(name="rope_prompts_4100", op="rope", dtype="bf16", B=5, new=1025, ragged=True, given=False, Hq=32, Hk=8, D=128, R=128,
             interleaved=False, inverse=False, length=900000),
        # the gradient of a long prompt's heads, in full precision
        dict(name="rope_inverse_f32", op="rope", dtype="f32", B=1, new=8192, ragged=False, given=True, Hq=32, Hk=8, D=128, R=128,
             interleaved=True, inverse=True, length=8192),
        # eight chats on one system prompt, one token each
        dict(name="shared_chats_b8", op="shared", dtype="f16", cache="int8", B=8, new=1, ragged=True, Hq=32, Hkv=8, D=128,
             page=64, shared=1024, length=200, window=0),
        # a serving batch on long instructions
        dict(name="shared_decode_b64", op="shared", dtype="bf16", cache="e4m3", B=64, new=1, ragged=True, Hq=32, Hkv=8, D=128,
             page=64, shared=8192, length=600, window=0),
        # many questions about one long document
        dict(name="shared_document_b128", op="shared", dtype="f16", cache="int8", B=128, new=1, ragged=False, Hq=32, Hkv=8,
             D=128, page=64, shared=32768, length=301, window=0),
        # the questions' own prompts as they arrive
        dict(name="shared_prompts_8x200", op="shared", dtype="bf16", cache="int8", B=8, new=200, ragged=True, Hq=32, Hkv=8,
             D=128, page=64, shared=6016, length=333, window=0),
        # one sequence, temperature alone: the smallest draw
        dict(name="sample_one", op="sample", dtype="f16", B=1, V=32000, pad=0, temperature=0.8, top_k=0, top_p=1.0, min_p=0.0,
             mixed=False, masked=False),
        # one sequence of a large vocabulary with the usual filters, logits in full precision
        dict(name="sample_one_filtered", op="sample", dtype="f32", B=1, V=128000, pad=0, temperature=0.7, top_k=50, top_p=0.9,
             min_p=0.0, mixed=False, masked=False),
        # a serving batch, every request with settings of its own, some with a grammar that forbids most tokens
        dict(name="sample_mixed_b64", op="sample", dtype="bf16", B=64, V=128000, pad=64, temperature=0.9, top_k=40, top_p=0.95,
             min_p=0.05, mixed=True, masked=True),
        # many answers to one question, drawn from wide distributions
        dict(name="sample_top_p_b256", op="sample", dtype="f32", B=256, V=50001, pad=0, temperature=1.2, top_k=0, top_p=0.95,
             min_p=0.0, mixed=False, masked=False),
    ]


# The most work of a drawn case: the largest listed one's.
_MOST_TURNED = 8192 * 40 * 128 * 4              # bytes that a rope call reads
_MOST_PAIRS = 8 * 200 * 32 * (6016 + 333)       # query heads x tokens seen
_MOST_OWN = 128 * 301 * 8 * 128                 # cached values of K that are no shared ones
_MOST_LOGITS = 256 * 50001


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rope", "shared", "shared", "sample", "sample"))
    if op == "rope":
        dtype = rng.choice(("f16", "bf16", "bf16", "f32"))
        D = rng.choice((64, 80, 96, 128, 128, 256))
        R = rng.choice((D, D, D // 2, max(2, D // 8 * 2)))
        Hk = rng.choice((1, 2, 4, 8, 8))
        Hq = Hk * rng.choice((1, 2, 3, 4, 4, 8))
        B = _log(rng, 1, 256)
        most = max(1, _MOST_TURNED // ((Hq + Hk) * D * (4 if dtype == "f32" else 2)))
        new = 1 if rng.random() < 0.4 else _log(rng, 1, 9000)
        new = max(1, min(new, most // B))
        return dict(op=op, dtype=dtype, B=B, new=new, ragged=new > 1 and rng.random() < 0.5, given=rng.random() < 0.5, Hq=Hq,
                    Hk=Hk, D=D, R=R, interleaved=rng.random() < 0.4, inverse=rng.random() < 0.25,
                    length=new + _log(rng, 1, 1000000))
    if op == "sample":
        V = _log(rng, 100, 260000)
        B = max(1, min(_log(rng, 1, 512), _MOST_LOGITS // V))
        return dict(op=op, dtype=rng.choice(("f16", "bf16", "f32")), B=B, V=V, pad=rng.choice((0, 0, 1, 64)),
                    temperature=round(rng.uniform(0.3, 1.6), 2), top_k=rng.choice((0, 0, 1, 20, 50, 1000, V // 2)),
                    top_p=rng.choice((1.0, 1.0, 0.5, 0.9, 0.99)), min_p=rng.choice((0.0, 0.0, 0.02, 0.2)),
                    mixed=rng.random() < 0.4, masked=rng.random() < 0.3)
    D, page = rng.choice((64, 128, 128, 256, 96)), rng.choice((16, 32, 64, 64, 128, 256))
    Hkv, cache = rng.choice((1, 2, 4, 8, 8)), rng.choice(("int8", "e4m3"))
    Hq = Hkv * rng.choice((1, 2, 4, 4, 5, 8))
    B = _log(rng, 2, 128)
    shared = max(page, min(_log(rng, 100, 40000), _MOST_PAIRS // (B * Hq) // 2) // page * page)
    length = max(1, min(_log(rng, 1, 4000), _MOST_OWN // (B * Hkv * D), _MOST_PAIRS // (B * Hq) // 2))
    new = 1 if rng.random() < 0.6 else min(length, _log(rng, 2, 300))
    new = max(1, min(new, _MOST_PAIRS // (B * Hq * (shared + length))))
    return dict(op=op, dtype=rng.choice(("f16", "bf16")), cache=cache, B=B, new=new, ragged=rng.random() < 0.5, Hq=Hq, Hkv=Hkv,
                D=D, page=page, shared=shared, length=length, window=_log(rng, 16, 8000) if rng.random() < 0.15 else 0)


# ---------------------------------------------------------------------------
# inputs

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_QMAX = {"int8": 127.0, "e4m3": 448.0}


def _lengths(case):
    """Tokens of each sequence behind the shared ones, and its new ones: plain arithmetic on the sizes."""
    B, n, L = case["B"], case["new"], case["length"]
    if not case["ragged"]:
        return [L] * B, [n] * B
    news = [max(1, n - (n * b) // (2 * B)) for b in range(B)]
    return [max(x, L - (L * 3 * b) // (4 * B)) for b, x in enumerate(news)], news


def _starts(news):
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    return starts


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"case": case, **{"rope": _prepare_rope, "shared": _prepare_shared, "sample": _prepare_sample}[case["op"]](case, g)}


def _prepare_rope(case, g):
    lens, news = _lengths(case)
    starts = _starts(news)
    T, Hq, Hk, D = starts[-1], case["Hq"], case["Hk"], case["D"]
    # queries, keys and values as the one product of a layer leaves them
    qkv = torch.randn(T, (Hq + 2 * Hk) * D, device="cuda", generator=g).to(_DT[case["dtype"]])
    s = {"q": qkv[:, : Hq * D].view(T, Hq, D), "k": qkv[:, Hq * D: (Hq + Hk) * D].view(T, Hk, D)}
    # a base of 500000 whose slow pairs are stretched by 8, as for contexts longer than those trained on, and their magnitude
    f = 500000.0 ** (-torch.arange(case["R"] // 2, dtype=torch.float64, device="cuda") / (case["R"] // 2))
    slow = ((2 * math.pi / f - 2048.0) / 6144.0).clamp(0, 1)
    s["frequencies"] = f * (1 - slow) + f / 8 * slow
    s["magnitude"] = 0.1 * math.log(8.0) + 1.0
    ends = torch.tensor(lens, dtype=torch.int32, device="cuda")
    begins = torch.randint(0, max(1, min(lens) // 64), (case["B"],), device="cuda", generator=g).int()
    s["lengths"] = ends - torch.minimum(begins, ends - torch.tensor(news, dtype=torch.int32, device="cuda"))
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda") if case["ragged"] else None
    s["counts"] = torch.tensor(news, device="cuda")
    s["positions"] = _positions(s, T).int() if case["given"] else None
    return s


def _positions(s, T):
    seq = torch.repeat_interleave(torch.arange(s["counts"].numel(), device="cuda"), s["counts"], output_size=T)
    after = torch.cumsum(s["counts"], 0)
    return s["lengths"].long()[seq] - after[seq] + torch.arange(T, device="cuda")


def _prepare_shared(case, g):
    lens, news = _lengths(case)
    B, Hkv, D, page = case["B"], case["Hkv"], case["D"], case["page"]
    S = case["shared"] // page
    width = S + max(-(-x // page) for x in lens)
    pages = S + B * (width - S) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    s = {"shared": order[:S].contiguous()}
    used = torch.tensor([-(-x // page) for x in lens], device="cuda")
    mine = order[S: S + B * (width - S)].view(B, width - S)
    mine = torch.where(torch.arange(width - S, device="cuda") < used[:, None], mine, -1)
    s["table"] = torch.cat((s["shared"].expand(B, S), mine), 1).contiguous()  # the shared pages too, as an append reads it
    s["lengths"] = torch.tensor([case["shared"] + x for x in lens], dtype=torch.int32, device="cuda")
    starts = _starts(news)
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
        s[w + "_scales"] = 4.0 / _QMAX[case["cache"]] * 2.0 ** torch.randint(-1, 2, (pages, Hkv), device="cuda", generator=g).float()
    s["q"] = torch.randn(starts[-1], case["Hq"], D, device="cuda", generator=g).to(_DT[case["dtype"]])
    return s


def _prepare_sample(case, g):
    B, V = case["B"], case["V"]
    rand = lambda *n: torch.rand(*n, device="cuda", generator=g)
    # a few likely tokens above a wide field, as a model's last product leaves them
    x = torch.randn(B, V + case["pad"], device="cuda", generator=g) * 2.2
    likely = torch.randint(0, V, (B, 24), device="cuda", generator=g)
    x.scatter_(1, likely, 6.0 + 4.0 * torch.randn(B, 24, device="cuda", generator=g))
    if case["masked"]:  # every fourth row allows one token in thirty
        gone = (rand(B, V + case["pad"]) > 0.03) & (torch.arange(B, device="cuda") % 4 == 1)[:, None]
        x.masked_fill_(gone, -math.inf)
    s = {"logits": x.to(_DT[case["dtype"]])[:, :V], "u": rand(B)}
    for name in ("temperature", "top_k", "top_p", "min_p"):
        s[name] = case[name]
    if case["mixed"]:  # settings by request: temperatures around the case's, some of them greedy, filters on or off
        on = lambda: rand(B) < 0.5
        s["temperature"] = torch.where(rand(B) < 0.15, 0.0, case["temperature"] * (0.5 + rand(B)))
        s["top_k"] = torch.where(on(), case["top_k"], 0).int()
        s["top_p"] = torch.where(on(), case["top_p"], 1.0).float()
        s["min_p"] = torch.where(on(), case["min_p"], 0.0).float()
    return s


# ---------------------------------------------------------------------------
# one pass

def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        from xrgpu_amd import ops
        if op == "rope":
            where = dict(positions=s["positions"]) if c["given"] else dict(lengths=s["lengths"], starts=s["starts"])
            return ops.rope(s["q"], s["k"], frequencies=s["frequencies"], magnitude=s["magnitude"],
                            interleaved=c["interleaved"], inverse=c["inverse"], **where)
        if op == "shared":
            return ops.kv8_shared_attention(s["q"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["shared"],
                                            s["table"], s["lengths"], starts=s["starts"], max_new=s["max_new"],
                                            window=c["window"])
        return ops.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                          min_p=s["min_p"])
    return {"rope": _rope, "shared": _shared, "sample": _sample}[op](s)


# The plain forms: elementary torch operations.

def _rope(s):
    c = s["case"]
    pos = s["positions"].long() if c["given"] else _positions(s, s["q"].shape[0])
    angle = pos[:, None].double() * s["frequencies"]  # 64 bits: far positions lose their angle in 32
    cos, sin = (f.float()[:, None] * s["magnitude"] for f in (angle.cos(), angle.sin()))
    if c["inverse"]:
        sin = -sin
    R, out = c["R"], []
    for x in (s["q"], s["k"]):
        f = x.float()
        if c["interleaved"]:
            a, b = f[..., 0:R:2], f[..., 1:R:2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = f[..., : R // 2], f[..., R // 2: R]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        out.append(torch.cat((turned, f[..., R:]), -1).to(x.dtype))
    return tuple(out)


def _shared(s):
    c = s["case"]
    B, Hq, Hkv, D, S = c["B"], c["Hq"], c["Hkv"], c["D"], c["shared"]
    G, n, q = Hq // Hkv, s["max_new"], s["q"]
    tail = s["table"][:, S // c["page"]:].long().clamp_min(0)
    # the shared tokens once, [Hkv, S, D], and each sequence's own, [B, Hkv, W, D]
    k0, v0 = ((s[w + "_cache"][s["shared"]].float() * s[w + "_scales"][s["shared"]][..., None, None]).transpose(0, 1).flatten(1, 2)
              for w in ("k", "v"))
    k1, v1 = ((s[w + "_cache"][tail].float() * s[w + "_scales"][tail][..., None, None]).transpose(1, 2).flatten(2, 3)
              for w in ("k", "v"))
    row = torch.arange(n, device=q.device)
    first = torch.cumsum(s["counts"], 0) - s["counts"]
    have = row < s["counts"][:, None]  # [B, n]: ragged queries, padded
    take = (first[:, None] + row).clamp_max(q.shape[0] - 1)
    qp = q[take].float().view(B, n, Hkv, G, D).permute(2, 0, 3, 1, 4)  # [Hkv, B, G, n, D]
    z0 = torch.bmm(qp.reshape(Hkv, B * G * n, D), k0.transpose(1, 2)).view(Hkv, B, G, n, S)
    z1 = torch.matmul(qp.transpose(0, 1).reshape(B, Hkv, G * n, D), k1.transpose(2, 3)).view(B, Hkv, G, n, -1)
    z = torch.cat((z0.transpose(0, 1), z1), -1).mul_(1.0 / math.sqrt(D))
    pos = s["lengths"].long()[:, None] - s["counts"][:, None] + row
    t = torch.arange(z.shape[-1], device=q.device)
    gone = t > pos[..., None]  # [B, n, S + W]
    if c["window"]:
        gone |= t <= pos[..., None] - c["window"]
    z.masked_fill_(gone[:, None, None], float("-inf"))
    z = z.sub_(z.amax(-1, keepdim=True)).exp_()
    total = z.sum(-1, keepdim=True)
    o = torch.bmm(z[..., :S].transpose(0, 1).reshape(Hkv, B * G * n, S), v0).view(Hkv, B, G, n, D).transpose(0, 1)
    o = (o + torch.matmul(z[..., S:].reshape(B, Hkv, G * n, -1), v1).view(B, Hkv, G, n, D)) / total
    return o.permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D)[have].to(q.dtype)


def _sample(s):
    x = s["logits"].float()
    B, V = x.shape
    x = torch.where(x.isnan(), -math.inf, x)
    col = lambda v: v.double()[:, None] if torch.is_tensor(v) else torch.full((B, 1), float(v), dtype=torch.float64, device=x.device)
    temperature, k, p, least = (col(s[name]) for name in ("temperature", "top_k", "top_p", "min_p"))
    greedy = ~(temperature > 0)
    k = torch.where(greedy, 1, torch.where(k > 0, k, V))
    x, order = x.sort(dim=1, descending=True, stable=True)  # of equal logits the lowest index first
    rank = torch.arange(V, device=x.device)
    # 64 bits: the sums' borders decide which token it is
    w = ((x.double() - x[:, :1].double()) / torch.where(greedy, 1.0, temperature)).exp()
    w = torch.where(rank < k, w, 0.0)
    run_ = w.cumsum(1)
    kept = (run_ - w < torch.where(p < 1, p, math.inf) * run_[:, -1:]) | (rank == 0)
    kept &= (w >= least.clamp_max(1.0)) | ~(least > 0)
    w = torch.zeros_like(w).scatter_(1, order, torch.where(kept, w, 0.0))
    run_ = w.cumsum(1)
    total = run_[:, -1:]
    token = (run_ <= s["u"].double()[:, None] * total).sum(1, keepdim=True)
    return token[:, 0].int(), (w.gather(1, token) / total).log()[:, 0].float()


# ---------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    op = case["op"]
    size = {"f16": 2, "bf16": 2, "f32": 4}[case["dtype"]]
    if op == "sample":
        return {"bytes": case["B"] * (case["V"] * size + 12), "flops": 0}
    lens, news = _lengths(case)
    D = case["D"]
    if op == "rope":
        T = sum(news)
        return {"bytes": 2 * T * (case["Hq"] + case["Hk"]) * D * size + 4 * T + 4 * case["R"], "flops": 0}
    S, w = case["shared"], case["window"]
    seen = first = 0  # tokens that the rows see; shared tokens that a row sees
    held = 0
    for L, n in zip(lens, news):
        for i in range(n):
            p = S + L - n + i + 1
            seen += min(w or p, p)
        lo = max(0, S + L - n + 1 - w) if w else 0
        first = max(first, S - lo)
        held += L - max(0, lo - S)
    tables = -(-first // case["page"]) + sum(-(-x // case["page"]) for x in lens)
    return {"bytes": 2 * case["Hkv"] * ((max(0, first) + held) * D + 4 * tables) + 4 * tables + 2 * sum(news) * case["Hq"] * D * size,
            "flops": 4 * D * case["Hq"] * seen}


# ---------------------------------------------------------------------------
# the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "shared": _exact_shared, "sample": _exact_sample}[case["op"]](case, s)


def _exact_rope(case, s):
    lens = s["lengths"].tolist()
    _, news = _lengths(case)
    pos = [p for L, n in zip(lens, news) for p in range(L - n, L)]
    turn = torch.polar(torch.full((1,), s["magnitude"], dtype=torch.float64, device="cuda"),
                       torch.tensor(pos, dtype=torch.float64, device="cuda")[:, None] * s["frequencies"][None])
    if case["inverse"]:
        turn = turn.conj()
    h = case["R"] // 2
    out = []
    for x in (s["q"], s["k"]):
        y = x.double().contiguous()
        a, b = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if case["interleaved"] else (slice(0, h), slice(h, 2 * h))
        z = torch.complex(y[..., a].contiguous(), y[..., b].contiguous()) * turn[:, None, :]
        y[..., a], y[..., b] = z.real, z.imag
        out.append(y)
    return tuple(out)


def _exact_shared(case, s):
    lens, news = _lengths(case)
    S, D, G = case["shared"], case["D"], case["Hq"] // case["Hkv"]
    out = torch.empty(sum(news), case["Hq"], D, dtype=torch.float64, device="cuda")
    for h in range(case["Hkv"]):
        def values(w, pages):
            return (s[w + "_cache"][pages, h].float().double() * s[w + "_scales"][pages, h].double()[:, None, None]).reshape(-1, D)
        k0, v0 = values("k", s["shared"].long()), values("v", s["shared"].long())
        at = 0
        for b, (L, n) in enumerate(zip(lens, news)):
            mine = s["table"][b, S // case["page"]:][: -(-L // case["page"])].long()
            k, v = (torch.cat((x, values(w, mine)[:L])) for w, x in (("k", k0), ("v", v0)))
            p = torch.arange(S + L - n, S + L, device="cuda").repeat_interleave(G)[:, None]
            t = torch.arange(S + L, device="cuda")[None]
            see = t <= p
            if case["window"]:
                see = see & (p - t < case["window"])
            z = torch.matmul(s["q"][at: at + n, h * G: h * G + G].double().reshape(n * G, D), k.T) / math.sqrt(D)
            z = torch.softmax(torch.where(see, z, -math.inf), -1)
            out[at: at + n, h * G: h * G + G] = torch.matmul(z, v).view(n, G, D)
            at += n
    return out


def _exact_sample(case, s):
    x = s["logits"].double()
    tokens, shares = [], []
    for b in range(case["B"]):
        of = lambda name: float(s[name][b] if torch.is_tensor(s[name]) else s[name])
        temperature, k, p, least = of("temperature"), int(of("top_k")), of("top_p"), of("min_p")
        row = torch.nan_to_num(x[b], nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        top = row.max()
        if not temperature > 0:
            tokens.append(int((row == top).nonzero()[0, 0]))
            shares.append(0.0)
            continue
        up, index = torch.sort(-row, stable=True)
        if k > 0:
            up, index = up[:k], index[:k]
        w = torch.exp((-up - top) / temperature)
        if p < 1:
            below = torch.cumsum(w, 0) - w < p * w.sum()  # the weight before a token is short of top_p
            below[0] = True
            w, index = w[below], index[below]
        if least > 0:
            enough = w >= min(least, 1.0)
            w, index = w[enough], index[enough]
        index, by = index.sort()
        w = w[by]
        sums = torch.cumsum(w, 0)
        at = int((sums > float(s["u"][b]) * sums[-1]).nonzero()[0, 0])
        tokens.append(int(index[at]))
        shares.append(float(torch.log(w[at] / sums[-1])))
    return torch.tensor(tokens, dtype=torch.int32, device="cuda"), torch.tensor(shares, dtype=torch.float64, device="cuda")
