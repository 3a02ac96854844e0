"""Refusals of rope, sample and kv8_shared_attention: argument checks that reach no device (no GPU)."""
import ctypes

import pytest
import torch

from xrgpu_amd import _native as nat
from xrgpu_amd import ops

MEM = (ctypes.c_uint8 * 4096)()
PTR = (ctypes.addressof(MEM) + 15) // 16 * 16  # a 16-byte aligned address that is never read
H16 = torch.float16


def rope(q=PTR, k=None, oq=PTR, ok=None, qs=128, ks=64, oqs=128, oks=64, dtype=nat.F16, f=PTR, R=64, m=1.0, pos=PTR, pt=nat.I32, lengths=None,
         starts=None, rows=0, B=0, Hq=2, Hk=0, D=64):
    return nat.lib().xrmm_rope(q, k, oq, ok, qs, ks, oqs, oks, dtype, f, R, m, pos, pt, lengths, starts, rows, B, Hq, Hk, D, 0, 0, None)


def sample(x=PTR, stride=100, dtype=nat.F16, u=PTR, t=1.0, k=0, p=1.0, m=0.0, tokens=PTR, shares=PTR, rows=0, V=100, ws=None, temperatures=None):
    return nat.lib().xrmm_sample(x, stride, dtype, u, temperatures, None, None, None, t, k, p, m, tokens, shares, rows, V, ws, 0, None)


def shared(q=PTR, qs=128, dtype=nat.F16, cd=nat.I8, sp=PTR, S=1, rows=0, B=1, W=1, page=16, Hq=2, H=1, D=64, scale=1.0, window=0, ws=None):
    return nat.lib().xrmm_kv8_shared_attention(q, qs, PTR, dtype, PTR, PTR, PTR, PTR, cd, sp, S, PTR, PTR, None, None, rows, 0, B, W, 1, page, Hq,
                                               H, D, scale, 1, window, ws, 0, None)


@pytest.mark.parametrize("call,kw,msg", [
    (rope, dict(dtype=nat.I8), "q and k"), (rope, dict(rows=-1), "rows"), (rope, dict(D=1025), "head size"), (rope, dict(D=0), "head size"),
    (rope, dict(R=0), "turned part"), (rope, dict(R=63), "turned part"), (rope, dict(R=66), "turned part"), (rope, dict(Hq=-1), "heads"),
    (rope, dict(m=float("nan")), "magnitude"), (rope, dict(m=float("inf")), "magnitude"), (rope, dict(rows=1, lengths=PTR, B=1), "either"),
    (rope, dict(rows=1, pos=None), "either"), (rope, dict(pt=nat.F32), "int32 or int64"), (rope, dict(starts=PTR), "belong to lengths"),
    (rope, dict(B=-1), "batch"), (rope, dict(rows=1, pos=None, lengths=PTR), "without sequences"),
    (rope, dict(rows=3, pos=None, lengths=PTR, B=2), "need starts"), (rope, dict(rows=2, qs=100), "strides"), (rope, dict(rows=2, oqs=100), "strides"),
    (rope, dict(rows=2, Hk=1, k=PTR, ok=PTR, ks=10), "strides"), (rope, dict(rows=1, q=None), "null"), (rope, dict(rows=1, f=None), "null"),
    (rope, dict(rows=1, Hk=1), "null"), (rope, dict(q=PTR + 1), "elements"), (rope, dict(f=PTR + 4), "elements"),
    (rope, dict(pt=nat.I64, pos=PTR + 4), "elements"), (rope, dict(rows=2, oq=PTR + 2), "overlap"), (rope, dict(rows=2, oq=PTR + 128), "overlap"),
    (rope, dict(rows=2, oqs=160), "overlap"), (rope, dict(rows=1, Hk=1, k=PTR + 128, ok=PTR + 1024), "overlap"),
    (rope, dict(rows=1, oq=PTR + 1024, Hk=1, k=PTR + 512, ok=PTR + 1152), "overlap"),
    (sample, dict(dtype=nat.I8), "logits"), (sample, dict(rows=-1), "rows"), (sample, dict(V=0), "2^24"), (sample, dict(V=(1 << 24) + 1), "2^24"),
    (sample, dict(rows=2, stride=99), "stride"), (sample, dict(t=-0.1), "temperature"), (sample, dict(t=float("nan")), "temperature"),
    (sample, dict(k=-1), "top_k"), (sample, dict(p=-0.1), "top_p"), (sample, dict(p=float("nan")), "top_p"), (sample, dict(m=1.1), "min_p"),
    (sample, dict(m=-0.1), "min_p"), (sample, dict(m=float("nan")), "min_p"), (sample, dict(rows=1, x=None), "null"), (sample, dict(rows=1, u=None), "null"),
    (sample, dict(rows=1, tokens=None), "null"), (sample, dict(rows=1, shares=None), "null"), (sample, dict(x=PTR + 1), "elements"),
    (sample, dict(u=PTR + 2), "4-byte"), (sample, dict(temperatures=PTR + 2), "4-byte"), (sample, dict(ws=PTR // 256 * 256 + 16), "256-byte"),
    (shared, dict(S=-1), "negative count"), (shared, dict(S=1 << 28, page=16), "2^31 tokens"), (shared, dict(rows=1, sp=None), "null"),
    (shared, dict(sp=PTR + 2), "4-byte"), (shared, dict(dtype=nat.F32), "q must be"), (shared, dict(Hq=3, H=2), "multiple"),
    (shared, dict(window=-1), "window"), (shared, dict(scale=float("nan")), "scale"), (shared, dict(rows=2, qs=64), "stride"),
    (shared, dict(rows=1, q=PTR + 1), "elements"), (shared, dict(D=80), "head size"), (shared, dict(cd=nat.U8), "int8 or float8"),
    (shared, dict(ws=PTR // 256 * 256 + 16), "256-byte"),
])
def test_c_entry_refuses(call, kw, msg):
    assert call(**kw) == nat.XRMM_EINVAL
    assert msg in nat.last_error()


@pytest.mark.parametrize("call", [rope, sample, shared])
def test_empty_calls_are_ok_without_a_device(call):
    assert call() == nat.XRMM_OK and nat.last_error() == ""


def z(*s, dt=H16):
    return torch.zeros(s, dtype=dt)


F = torch.ones(32, dtype=torch.float64)
P = torch.zeros(3, dtype=torch.int32)


@pytest.mark.parametrize("kw,msg", [
    (dict(q=z(3, 2, 64, dt=torch.int32)), "both be"), (dict(k=z(3, 2, 64, dt=torch.float32)), "both be"), (dict(q=z(3, 128)), "same tokens"),
    (dict(k=z(2, 2, 64)), "same tokens"), (dict(k=z(3, 2, 32)), "same tokens"), (dict(frequencies=F.float()), "float64"), (dict(frequencies=F[None]), "float64"),
    (dict(positions=None), "either"), (dict(lengths=P), "either"), (dict(positions=P.float()), "int32 or int64"), (dict(positions=P[:2]), "int32 or int64"),
    (dict(positions=None, lengths=P.long()), "lengths"), (dict(positions=None, lengths=P, starts=P), "starts"), (dict(starts=P), "starts"),
    (dict(k_out=z(3, 2, 64)), "k_out without"), (dict(out=z(3, 2, 32)), "out must"), (dict(k=z(3, 1, 64), k_out=z(3, 2, 64)), "k_out must"),
    (dict(q=z(3, 64, 2).transpose(1, 2)), "contiguous"), (dict(q=z(1, 2, 64).expand(3, 2, 64)), "overlap"), (dict(), "on the GPU"),
])
def test_rope_front_refuses(kw, msg):
    with pytest.raises(nat.XrmmInvalid, match=msg):
        ops.rope(**{**dict(q=z(3, 2, 64), frequencies=F, positions=P), **kw})


@pytest.mark.parametrize("args,kw,msg", [
    ((0,), {}, "even"), ((7,), {}, "even"), ((8, -1.0), {}, "positive"), ((8,), dict(factor=0.0), "positive"), ((8,), dict(scaling="other"), "scaling"),
    ((8,), dict(scaling="yarn"), "original_length"), ((8,), dict(scaling="bands", original_length=0), "original_length"),
    ((8,), dict(scaling="bands", original_length=10, low=4.0, high=1.0), "low"), ((2,), dict(scaling="ntk"), "two pairs"),
])
def test_rope_frequencies_refuse(args, kw, msg):
    with pytest.raises(nat.XrmmInvalid, match=msg):
        ops.rope_frequencies(*args, device="cpu", **kw)


@pytest.mark.parametrize("kw,msg", [
    (dict(logits=z(3, 10, dt=torch.int32)), "float32, float16 or bfloat16"), (dict(logits=z(10)), r"\[rows, vocab\]"), (dict(logits=z(3, 0)), "vocab positive"),
    (dict(logits=z(10, 3).t()), "contiguous"), (dict(logits=z(1, 10).expand(3, 10)), "overlap"), (dict(u=torch.zeros(2)), "u must"),
    (dict(u=torch.zeros(3, dtype=torch.float64)), "u must"), (dict(temperature=torch.zeros(2)), "temperature must"),
    (dict(top_k=torch.zeros(3)), "top_k must"), (dict(top_p=torch.zeros(3, dtype=torch.float64)), "top_p must"), (dict(min_p=torch.zeros(3, 1)), "min_p must"),
    (dict(), "on the GPU"),
])
def test_sample_front_refuses(kw, msg):
    with pytest.raises(nat.XrmmInvalid, match=msg):
        ops.sample(**{**dict(logits=z(3, 10), u=torch.zeros(3)), **kw})


def test_shared_front_refuses():
    from tests.test_lowbit_validation import cache
    q = z(1, 2, 64)
    for pages, msg in ((torch.zeros(2, dtype=torch.int64), "shared_pages"), (torch.zeros(1, 2, dtype=torch.int32), "shared_pages"),
                       (torch.zeros(2, dtype=torch.int32), "on the GPU")):
        with pytest.raises(nat.XrmmInvalid, match=msg):
            ops.kv8_shared_attention(q, shared_pages=pages, **cache())
    for x, msg in ((q.float(), "q must be"), (z(2, 3, 64), "multiple"), (z(2, 2, 96), r"\[tokens, 2, 64\]")):
        with pytest.raises(nat.XrmmInvalid, match=msg):
            ops.kv8_shared_attention(x, shared_pages=P, **cache())


def test_shared_attention_names_its_way(monkeypatch):
    f = lambda T, B, S, W, **kw: ops.kv8_shared_attention_kernel(T, 32, 8, 128, batch=B, shared_pages=S, table_width=W, page_size=64, **kw)
    size = lambda T, B, S, W: ops.kv8_shared_attention_workspace_bytes(T, 32, 8, 128, batch=B, shared_pages=S, table_width=W, page_size=64)
    assert f(64, 64, 128, 138) == "kv8_prefix_tile" and f(1, 1, 128, 138) == "kv8_walk" and f(64, 64, 0, 138) == "kv8_walk"
    assert size(64, 64, 128, 138) > size(64, 64, 0, 138)
    monkeypatch.setenv("XRMM_KV8_SHARED", "kv8_prefix_rows")
    assert f(64, 64, 128, 138) == "kv8_prefix_rows" and f(1, 1, 128, 138) == "kv8_walk"
    monkeypatch.setenv("XRMM_KV8_SHARED", "kv8_walk")
    assert f(64, 64, 128, 138) == "kv8_walk"
    with pytest.raises(nat.XrmmInvalid, match="head size"):
        ops.kv8_shared_attention_kernel(1, 8, 2, 80, batch=1, shared_pages=1, table_width=1, page_size=64)


def test_sample_workspaces():
    """None where a workgroup a row is estimated fastest whatever is asked for."""
    assert ops.sample_workspace_bytes(1, 128000) > 4096 and ops.sample_workspace_bytes(1, 2000) == 0 and ops.sample_workspace_bytes(500, 128000) == 0
    assert ops.sample_workspace_bytes(0, 128000) == 0 and ops.sample_workspace_bytes(4, 0) == 0


BIG = (1 << 63) - 1


def test_rope_strides_that_are_of_no_use_are_not_read():
    """Of one row, and of no heads: what they hold decides nothing, whether memory overlaps above all."""
    for rows, kw in ((1, {}), (0, {}), (1, dict(Hk=1, k=PTR + 1024, ok=PTR + 1024))):
        for stride in (BIG, -BIG, 0, 1 << 62):
            assert rope(rows=rows, oq=PTR + 2, qs=stride, ks=stride, oqs=stride, oks=stride, **kw) == (nat.XRMM_EINVAL if rows else nat.XRMM_OK)
            assert rows == 0 or "overlap" in nat.last_error()
    for stride in (BIG, -BIG, 1 << 62):
        assert rope(rows=2, oq=PTR + 2, ks=stride, oks=stride) == nat.XRMM_EINVAL and "overlap" in nat.last_error()


@pytest.mark.parametrize("name", ["qs", "ks", "oqs", "oks"])
def test_rope_refuses_strides_whose_ranges_no_memory_has(name):
    # 2^62 elements of 2 bytes are 2^63 bytes: they wrap to a range that overlaps nothing
    for stride in (BIG, 1 << 62, 1 << 61):
        assert rope(**{**dict(rows=3, Hk=1, k=PTR, ok=PTR), name: stride}) == nat.XRMM_EINVAL
        assert "past any memory" in nat.last_error(), nat.last_error()


INF = float("inf")


@pytest.mark.parametrize("kw,msg", [
    (dict(theta=1.0, scaling="yarn", original_length=4096, factor=4.0), "theta above 1"), (dict(theta=0.5, scaling="yarn", original_length=4096, factor=4.0), "theta above 1"),
    *[({**dict(scaling=s, original_length=4096, factor=4.0), **kw}, "finite") for s in ("yarn", "bands")
      for kw in (dict(original_length=INF), dict(original_length=float("nan")), dict(high=INF), dict(low=float("nan")), dict(low=INF, high=INF))],
    (dict(scaling="ntk", factor=1e300), "finite theta"), (dict(theta=1e308, scaling="ntk", factor=10.0), "finite theta"),
])
def test_rope_frequencies_refuse_numbers_that_give_none(kw, msg):
    """A division by the logarithm of 1, floors of infinities and powers past float64 raised Python's own errors, or none."""
    with pytest.raises(nat.XrmmInvalid, match=msg):
        ops.rope_frequencies(8, device="cpu", **kw)


@pytest.mark.parametrize("kw", [dict(theta=1.0), dict(theta=0.5, scaling="linear", factor=2.0), dict(theta=0.5, scaling="bands", original_length=100, factor=4.0),
                                dict(theta=1.0, scaling="bands", original_length=100, factor=4.0), dict(theta=1.0 + 2.0 ** -40, scaling="yarn", original_length=4096, factor=4.0)])
def test_rope_frequencies_take_the_others(kw):
    f, m = ops.rope_frequencies(8, device="cpu", **kw)
    assert f.shape == (4,) and f.isfinite().all() and m >= 1.0
