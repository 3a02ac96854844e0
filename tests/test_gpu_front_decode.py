"""GPU: the native front end's rope, sample and kv8_shared_attention give what the Python path gives, and leave it what they do not take."""
import pytest

from tests.test_gpu_front_lowbit import _ops, both, cache

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
def test_rope(gpu, dt):
    ops = _ops()
    f, _ = ops.rope_frequencies(48)
    wide = torch.randn(6, 6 * 64, device="cuda").to(dt)
    q, k = wide[:, :256].view(6, 4, 64), wide[:, 256:].view(6, 2, 64)
    pos = torch.arange(6, device="cuda") * 1000
    lengths = torch.tensor([9, 70, 3], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 3, 5, 6], dtype=torch.int32, device="cuda")
    for kw in (dict(positions=pos), dict(positions=pos.int(), interleaved=True), dict(lengths=lengths), dict(lengths=lengths, starts=starts),
               dict(positions=pos, inverse=True, magnitude=1.5), dict(positions=pos, magnitude=2)):
        both(lambda: ops.rope(q, k, frequencies=f, **kw))
        both(lambda: ops.rope(q, frequencies=f, **kw))
    r = ops._FRONT.rope
    assert r(q, k, f, pos, None, None, 1.0, False, False) is not None
    for args in ((q.cpu(), k, f, pos, None, None, 1.0, False, False), (q, k.double(), f, pos, None, None, 1.0, False, False),
                 (q, k[:3], f, pos, None, None, 1.0, False, False), (q, k, f.float(), pos, None, None, 1.0, False, False),
                 (q, k, f, None, None, None, 1.0, False, False), (q, k, f, pos, lengths, None, 1.0, False, False),
                 (q, k, f, pos.float(), None, None, 1.0, False, False), (q, k, f, pos, None, starts, 1.0, False, False),
                 (q, k, f, None, lengths, starts[:3], 1.0, False, False), (q, k, f, pos, None, None, None, False, False),
                 (q, k, f, pos, None, None, 1.0, 1, False), (q[:0], k[:0], f, pos[:0], None, None, 1.0, False, False)):
        assert r(*args) is None
    with pytest.raises(ValueError):
        ops.rope(q, k, frequencies=torch.ones(33, dtype=torch.float64, device="cuda"), positions=pos)


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
def test_sample(gpu, dt):
    ops = _ops()
    x = torch.randn(5, 9007, device="cuda").to(dt)[:, :9000]
    u = torch.rand(5, device="cuda")
    full = lambda v, t=torch.float32: torch.full((5,), v, device="cuda", dtype=t)
    for kw in (dict(), dict(temperature=0), dict(top_k=5, top_p=1), dict(top_p=0.7, min_p=0.01), dict(temperature=full(0.8), top_k=full(9, torch.int32)),
               dict(top_p=full(0.5), min_p=full(0.0)), dict(top_k=full(3, torch.int32), min_p=0.1)):
        both(lambda: ops.sample(x, u, **kw))
    s = ops._FRONT.sample
    ops.sample(x, u)
    assert type(s(x, u, 1.0, 0, 1.0, 0.0)) is tuple
    for args in ((x.cpu(), u, 1.0, 0, 1.0, 0.0), (x, u.double(), 1.0, 0, 1.0, 0.0), (x.double(), u, 1.0, 0, 1.0, 0.0), (x.t(), u, 1.0, 0, 1.0, 0.0),
                 (x, u[:4], 1.0, 0, 1.0, 0.0), (x, u, None, 0, 1.0, 0.0), (x, u, 1.0, None, 1.0, 0.0), (x, u, 1.0, 1 << 40, 1.0, 0.0),
                 (x, u, full(1.0).double(), 0, 1.0, 0.0), (x, u, 1.0, full(1.0), 1.0, 0.0), (x, u, 1.0, 0, full(1.0)[:3], 0.0), (x[:0], u[:0], 1.0, 0, 1.0, 0.0)):
        assert s(*args) is None
    both(lambda: ops.sample(x, u, top_k=1 << 40))
    for kw in (dict(temperature=-1.0), dict(top_k=-1), dict(top_p=-0.5), dict(min_p=2.0)):
        with pytest.raises(ValueError):
            ops.sample(x, u, **kw)


@pytest.mark.parametrize("dt", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("n", [1, 3, 30])
def test_shared(gpu, dt, n):
    ops = _ops()
    c = cache([500, 700], dt=dt)
    pages = c[4][0, :20].contiguous()
    wide = torch.randn(2 * n, 5 * 64, device="cuda").half()
    q = wide[:, 64:].view(2 * n, 4, 64)
    starts = torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda")
    args = (*c[:4], pages, *c[4:])

    def with_status(**kw):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        return ops.kv8_shared_attention(q, *args, status=status, **kw), status

    for st in (None, starts):
        both(lambda: ops.kv8_shared_attention(q, *args, starts=st, max_new=n))
        both(lambda: with_status(starts=st))
    both(lambda: ops.kv8_shared_attention(q, *args, causal=False, window=100, scale=0.2))
    both(lambda: ops.kv8_shared_attention(q, *args, scale=1))
    f = ops._FRONT.kv8_shared_attention
    assert torch.is_tensor(f(q, *args, None, None, None, True, 0, None))
    for bad in ((q.float(), *args), (q[:, :3], *args), (q, *c[:4], pages.long(), *c[4:]), (q, *c[:4], pages[None], *c[4:]), (q, *c[:4], pages, c[4], c[5].long())):
        assert f(*bad, None, None, None, True, 0, None) is None
    with pytest.raises(ValueError):
        ops.kv8_shared_attention(q, *args, window=-1)


@pytest.mark.parametrize("call", ["sample", "shared"])
def test_a_workspace_lives_until_the_launch_that_uses_it(gpu, call):
    """As in test_gpu_front_lowbit.py: another thread may replace the table's workspace while a call is without the lock."""
    import ctypes

    from xrgpu_amd import _native as nat
    ops = _ops()
    names = ["xrmm_rope", "xrmm_sample_workspace_bytes", "xrmm_sample", "xrmm_kv8_shared_attention_workspace_bytes", "xrmm_kv8_shared_attention"]
    address = [ctypes.cast(getattr(nat.lib(), n), ctypes.c_void_p).value for n in names]
    if call == "sample":
        x, u = torch.randn(1, 128000, device="cuda"), torch.rand(1, device="cuda")
        run, which = (lambda: ops._FRONT.sample(x, u, 1.0, 0, 0.9, 0.0)), 2
        ops.sample(x, u, top_p=0.9)
        need = ops.sample_workspace_bytes(1, 128000)
    else:
        c = cache([5000, 5100], H=1, D=128, page=64)
        pages = c[4][0, :70].contiguous()
        q = torch.randn(2, 4, 128, device="cuda").half()
        run, which = (lambda: ops._FRONT.kv8_shared_attention(q, *c[:4], pages, *c[4:], None, None, None, True, 0, None)), 4
        ops.kv8_shared_attention(q, *c[:4], pages, *c[4:])
        need = ops.kv8_shared_attention_workspace_bytes(2, 4, 1, 128, batch=2, shared_pages=70, table_width=c[4].shape[1], page_size=64)
    assert need > 0
    fn = getattr(nat.lib(), names[which])
    seen = []

    def entry(*args):
        ws, size = args[-3], args[-2]
        key = next(k for k, t in ops._WORKSPACES.items() if t.data_ptr() == ws)
        ops._WORKSPACES[key] = torch.zeros(2 * size, dtype=torch.uint8, device="cuda")
        seen.append((ws, [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(4)]))
        return 0

    fake = ctypes.CFUNCTYPE(fn.restype, *fn.argtypes)(entry)
    there = list(address)
    there[which] = ctypes.cast(fake, ctypes.c_void_p).value
    try:
        ops._FRONT.bind_decode(*there)
        assert run() is not None
    finally:
        ops._FRONT.bind_decode(*address)
    (ws, others), = seen
    assert ws and all(t.data_ptr() != ws for t in others)
