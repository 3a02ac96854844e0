"""GPU: the native front end's MX4 and kv8 calls give what the Python path gives, and leave it what they do not take."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def _ops():
    from xrgpu_amd import ops
    assert ops._front(), "the native front end is not built"
    return ops


def both(f):
    ops = _ops()
    a = f()
    front = ops._FRONT
    ops._FRONT = False
    try:
        b = f()
    finally:
        ops._FRONT = front
    a, b = (x if isinstance(x, tuple) else (x,) for x in (a, b))
    for x, y in zip(a, b, strict=True):
        assert x.dtype == y.dtype and x.shape == y.shape and torch.equal(x, y)


def weights(N, K):
    kb = -(-K // 32)
    return (torch.randint(0, 256, (N, kb, 16), dtype=torch.uint8, device="cuda"),
            torch.randint(120, 125, (N, kb), dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
def test_quantize(gpu, dt):
    ops = _ops()
    x = torch.randn(3, 5, 70, device="cuda").to(dt)
    assert ops._FRONT.mx4_quantize(x) is not None
    both(lambda: ops.mx4_quantize(x))
    assert ops._FRONT.mx4_quantize(x.transpose(0, 1)) is None and ops._FRONT.mx4_quantize(x.cpu()) is None
    assert ops._FRONT.mx4_quantize(x.int()) is None


@pytest.mark.parametrize("M", [1, 8, 40, 300])
def test_product(gpu, M):
    ops = _ops()
    B, S = weights(96, 4096)
    A = torch.randn(2, M, 4096, device="cuda").half()
    bias = torch.randn(96, device="cuda").half()
    both(lambda: ops.matmul_mx4(A, B, S, bias))
    both(lambda: ops.matmul_mx4(A.bfloat16(), B, S))
    c, s = ops.mx4_quantize(A)
    for o in (None, torch.float32, torch.bfloat16):
        both(lambda: ops.matmul_mx4(c, B, S, A_scales=s, out_dtype=o))
    assert ops._FRONT.matmul_mx4(A, B, S, bias.float(), None, None) is None
    assert ops._FRONT.matmul_mx4(A, B, S[:, :-1], None, None, None) is None
    assert ops._FRONT.matmul_mx4(A[..., :4000], B, S, None, None, None) is None
    assert ops._FRONT.matmul_mx4(A, B, S, None, None, torch.float32) is None
    assert ops._FRONT.matmul_mx4(c, B, S, None, None, None) is None


def test_a_missing_workspace_comes_back_as_its_bytes(gpu):
    ops = _ops()
    B, S = weights(64, 8192)
    A = torch.randn(40, 8192, device="cuda").half()
    need = ops.matmul_mx4_workspace_bytes(40, 8192, 64)
    assert need > 0
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        assert ops._FRONT.matmul_mx4(A, B, S, None, None, None) == need
        y = ops.matmul_mx4(A, B, S)
        z = ops._FRONT.matmul_mx4(A, B, S, None, None, None)
        st.synchronize()
    assert torch.equal(y, z)


def cache(lens, H=2, D=64, page=16, dt=torch.int8):
    B, W = len(lens), -(-max(lens) // page)
    mk = lambda: torch.randint(-90, 90, (B * W, H, page, D), device="cuda").to(torch.int8).view(dt) if dt == torch.int8 else \
        torch.randn(B * W, H, page, D, device="cuda").to(dt)
    sc = lambda: torch.full((B * W, H), 2.0 ** -5, device="cuda")
    return [mk(), mk(), sc(), sc(), torch.randperm(B * W, device="cuda").int().view(B, W),
            torch.tensor(lens, dtype=torch.int32, device="cuda")]


@pytest.mark.parametrize("dt", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("n", [1, 3, 30])
def test_append_and_attention(gpu, dt, n):
    ops = _ops()
    c = cache([500, 700], dt=dt)
    wide = torch.randn(2 * n, 8 * 64, device="cuda").half()
    q, k, v = wide[:, :256].view(2 * n, 4, 64), wide[:, 256:384].view(2 * n, 2, 64), wide[:, 384:].view(2 * n, 2, 64)
    starts = torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda")

    def append(st):
        d = [x.clone() for x in c[:4]]
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        assert ops.kv8_append(k, v, *d, *c[4:], starts=st, max_new=n, status=status) is None
        return tuple(x.view(torch.uint8) for x in d) + (status,)

    for st in (None, starts):
        both(lambda: append(st))
        both(lambda: ops.kv8_attention(q, *c, starts=st, max_new=n))
    both(lambda: ops.kv8_attention(q, *c, causal=False, window=100, scale=0.2))
    both(lambda: ops.kv8_attention(q, *c, scale=1))
    f = ops._FRONT
    assert f.kv8_attention(q, *c, None, None, None, True, 0, None) is not None
    assert f.kv8_append(k, v, *[x.clone() for x in c[:4]], *c[4:], None, None, None) is True
    assert f.kv8_attention(q.float(), *c, None, None, None, True, 0, None) is None
    assert f.kv8_attention(q[:, :3], *c, None, None, None, True, 0, None) is None
    assert f.kv8_attention(q, *c[:5], c[5].long(), None, None, None, True, 0, None) is None
    assert f.kv8_append(k, v[:1], *c, None, None, None) is None
    assert f.kv8_append(k[:0], v[:0], *c, None, None, None) is None
    with pytest.raises(ValueError):
        ops.kv8_attention(q, *c, window=-1)


@pytest.mark.parametrize("call", ["product", "attention"])
def test_a_workspace_lives_until_the_launch_that_uses_it(gpu, call):
    """Another thread may replace the table's workspace while a call is without the interpreter's lock: here the
    entry point itself does, in place of a launch. The call's workspace must not come back as another tensor's memory."""
    import ctypes

    from xrgpu_amd import _native as nat
    ops = _ops()
    names = ["xrmm_mx4_quantize", "xrmm_matmul_mx4_workspace_bytes", "xrmm_matmul_mx4", "xrmm_kv8_append",
             "xrmm_kv8_attention_workspace_bytes", "xrmm_kv8_attention"]
    address = [ctypes.cast(getattr(nat.lib(), n), ctypes.c_void_p).value for n in names]
    if call == "product":
        B, S = weights(64, 8192)
        A = torch.randn(40, 8192, device="cuda").half()
        run, which, at = (lambda: ops._FRONT.matmul_mx4(A, B, S, None, None, None)), 2, -3
        ops.matmul_mx4(A, B, S)
    else:
        c = cache([5000], H=1, D=128, page=64)
        q = torch.randn(1, 4, 128, device="cuda").half()
        run, which, at = (lambda: ops._FRONT.kv8_attention(q, *c, None, None, None, True, 0, None)), 5, -3
        ops.kv8_attention(q, *c)
    fn = getattr(nat.lib(), names[which])
    seen = []

    def entry(*args):
        ws, size = args[at], args[at + 1]
        key = next(k for k, t in ops._WORKSPACES.items() if t.data_ptr() == ws)
        ops._WORKSPACES[key] = torch.zeros(2 * size, dtype=torch.uint8, device="cuda")
        seen.append((ws, [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(4)]))
        return 0

    fake = ctypes.CFUNCTYPE(fn.restype, *fn.argtypes)(entry)
    there = list(address)
    there[which] = ctypes.cast(fake, ctypes.c_void_p).value
    bind = ops._FRONT.bind_lowbit
    try:
        bind(ops._WORKSPACES, torch._C._cuda_isCurrentStreamCapturing, *there)
        assert torch.is_tensor(run())
    finally:
        bind(ops._WORKSPACES, torch._C._cuda_isCurrentStreamCapturing, *address)
    (ws, others), = seen
    assert ws and all(t.data_ptr() != ws for t in others)
