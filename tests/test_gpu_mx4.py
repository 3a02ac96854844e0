"""GPU parity of mx4_quantize and matmul_mx4 against oracle/lowbit.py.

Quantisation follows from comparisons and powers of two: bit equality. Products: the codes' values and their
products with the activations are exact in float32, so a result is off by its one output rounding
(eps / 2 relative) and the float32 sum (K + 2 roundings of 2^-24 relative to the sum of magnitudes).
"""
import numpy as np
import pytest

from oracle import lowbit as LB

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def ops():
    from xrgpu_amd import ops as _ops
    return _ops


def check_quant(x):
    codes, scales = ops().mx4_quantize(x)
    c, s = LB.mx4_quantize(x.double().cpu().numpy().reshape(-1, x.shape[-1]))
    assert tuple(codes.shape) == tuple(x.shape[:-1]) + (c.shape[1], 16)
    assert np.array_equal(scales.cpu().numpy().reshape(s.shape), s)
    assert np.array_equal(codes.cpu().numpy().reshape(c.shape), c)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 32), (3, 31), (2, 33), (5, 40), (7, 100), (1, 4096), (33, 1002), (130, 96), (0, 64)])
def test_quantize_shapes(gpu, dt, rows, K):
    g = torch.Generator().manual_seed(rows * 1000 + K)
    x = torch.randn(rows, K, generator=g) * torch.exp2(torch.randint(-6, 7, (rows, 1), generator=g).float())
    check_quant(x.to(DT[dt]).cuda())


@pytest.mark.parametrize("dt", list(DT))
def test_quantize_ties_extremes_and_nonfinite(gpu, dt):
    t = DT[dt]
    fi = torch.finfo(t)
    grid = torch.arange(0, 8.01, 0.125)
    rows = [torch.cat([grid[i:i + 15], -grid[i:i + 15], torch.tensor([6.0, 0.0])])[:32] for i in range(0, 50, 5)]
    x = torch.stack(rows)
    x = torch.cat([x, x * 2.0 ** -13, x * 2.0 ** 9, torch.zeros(2, 32), -torch.zeros(1, 32)]).to(t)
    tiny = torch.zeros(6, 32, dtype=t)
    tiny[0, 3], tiny[1, 5], tiny[2, 7], tiny[3, 1], tiny[4, 2], tiny[5, 0] = fi.tiny, fi.max, -fi.max, fi.tiny / 4, float("inf"), float("nan")
    tiny[4:, 9] = 1.0
    check_quant(torch.cat([x, tiny]).cuda())


def test_quantize_odd_view_and_leading_axes(gpu):
    x = torch.randn(2 * 3 * 64 + 1, device="cuda").half()[1:].view(2, 3, 64)  # 2-byte aligned
    check_quant(x)


def check_product(A, codes, scales, bias, y, extra=None):
    """A float64 [M, K] (exact values)."""
    W = LB.mx4_decode(codes.cpu().numpy(), scales.cpu().numpy())[:, :A.shape[1]]
    ref, mag = A @ W.T, np.abs(A) @ np.abs(W).T
    if bias is not None:
        b = bias.double().cpu().numpy()
        ref, mag = ref + b, mag + np.abs(b)
    eps = torch.finfo(y.dtype).eps
    tol = eps / 2 * np.abs(ref) + (1 + eps) * (A.shape[1] + 2) * 2.0 ** -24 * mag + torch.finfo(y.dtype).tiny * eps
    got = y.double().cpu().numpy().reshape(ref.shape)
    assert np.isfinite(got).all()
    worst = (np.abs(got - ref) - tol).max() if ref.size else 0.0
    assert worst <= 0, (worst, np.abs(got - ref).max())


def weights(N, K, seed, spread=3, center=122):
    g = torch.Generator().manual_seed(seed)
    kb = -(-K // 32)
    codes = torch.randint(0, 256, (N, kb, 16), generator=g, dtype=torch.uint8)
    scales = torch.randint(center - spread, center + spread + 1, (N, kb), generator=g, dtype=torch.uint8)
    if K % 32:
        nib = torch.stack((codes & 15, codes >> 4), -1).view(N, kb * 32)
        nib[:, K:] = 0
        nib = nib.view(N, kb, 16, 2)
        codes = nib[..., 0] | (nib[..., 1] << 4)
    return codes.cuda(), scales.cuda()


SHAPES = [(1, 32, 1), (1, 64, 17), (1, 4096, 64), (2, 96, 33), (3, 1000, 70), (5, 333, 48), (8, 512, 256), (16, 2048, 100),
          (17, 256, 40), (31, 1056, 130), (33, 512, 257), (47, 2080, 96), (64, 768, 192), (65, 640, 65), (100, 1024, 300),
          (128, 512, 256), (129, 4096, 128), (200, 544, 513), (257, 256, 260), (300, 1000, 129), (513, 384, 640),
          (1, 5000, 9), (4, 14336, 64), (40, 14336, 64), (70, 8192, 48), (0, 64, 8)]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_product_float_activations(gpu, dt, M, K, N):
    codes, scales = weights(N, K, M + K + N)
    g = torch.Generator().manual_seed(M * 7 + K)
    A = torch.randn(M, K, generator=g).to(DT[dt])
    bias = torch.randn(N, generator=g).to(DT[dt]).cuda() if (M + N) % 2 else None
    y = ops().matmul_mx4(A.cuda(), codes, scales, bias)
    assert y.dtype == DT[dt] and tuple(y.shape) == (M, N)
    check_product(A.double().numpy(), codes, scales, bias, y)


@pytest.mark.parametrize("out", list(DT))
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_product_mx4_activations(gpu, out, M, K, N):
    codes, scales = weights(N, K, M + K + N)
    ac, as_ = weights(max(M, 1), K, M + 3 * K, spread=4, center=126)
    ac, as_ = ac[:M], as_[:M]
    g = torch.Generator().manual_seed(N)
    bias = torch.randn(N, generator=g).to(DT[out]).cuda() if (M + N) % 2 else None
    y = ops().matmul_mx4(ac, codes, scales, bias, A_scales=as_, out_dtype=DT[out])
    assert y.dtype == DT[out] and tuple(y.shape) == (M, N)
    check_product(LB.mx4_decode(ac.cpu().numpy(), as_.cpu().numpy()), codes, scales, bias, y)


@pytest.mark.parametrize("M", [1, 24, 80, 300])
@pytest.mark.parametrize("center", [1, 60, 100, 108, 139, 145])
def test_scales_outside_binary16(gpu, M, center):
    """Block scales far outside binary16's range meet float16 activations at full precision (outputs scaled into range
    by bfloat16 activations' twin: float16 results overflow to infinity or vanish exactly as the true values do)."""
    N, K = 130, 512
    codes, scales = weights(N, K, center, spread=0, center=center)
    scales[:, 3] = 120  # one ordinary block, among blocks that binary16 cannot hold
    A = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).half()
    y = ops().matmul_mx4(A.cuda(), codes, scales).double().cpu().numpy()
    W = LB.mx4_decode(codes.cpu().numpy(), scales.cpu().numpy())
    a = A.double().numpy()
    ref, mag = a @ W.T, np.abs(a) @ np.abs(W).T
    tol = 2.0 ** -11 * np.abs(ref) + (K + 2) * 2.0 ** -24 * mag + 2.0 ** -25
    sure = np.abs(ref) + tol < 65504
    over = np.abs(ref) - tol > 65520
    assert (np.abs(y - ref)[sure] <= tol[sure]).all()
    assert np.array_equal(y[over], np.sign(ref[over]) * np.inf)
    # the same weights alone: small ones must not vanish beside nothing
    A0 = torch.zeros_like(A)
    A0[:, :96] = A[:, :96] * 256
    y0 = ops().matmul_mx4(A0.cuda(), codes, scales).double().cpu().numpy()
    ref0 = A0.double().numpy() @ W.T
    fin = np.abs(ref0) < 60000
    lim = 2.0 ** -11 * np.abs(ref0) + 2.0 ** -14 * (np.abs(A0.double().numpy()) @ np.abs(W).T) + 2.0 ** -25
    assert (np.abs(y0 - ref0)[fin] <= lim[fin]).all()


@pytest.mark.parametrize("M", [1, 40, 150, 520])
@pytest.mark.parametrize("act", ["f16", "bf16", "mx4"])
def test_nonfinite_stays_in_its_row_and_column(gpu, M, act):
    N, K = 96, 256
    codes, scales = weights(N, K, 5)
    scales[7, 2] = 255
    if act == "mx4":
        ac, as_ = weights(M, K, 6, center=125)
        as_[M // 2, 1] = 255
        y = ops().matmul_mx4(ac, codes, scales, A_scales=as_, out_dtype=torch.float32)
    else:
        A = torch.randn(M, K, device="cuda").to(DT[act])
        A[M // 2, 40] = float("nan")
        y = ops().matmul_mx4(A, codes, scales)
    nan = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    nan[:, 7] = True
    nan[M // 2] = True
    assert torch.equal(y.isnan(), nan)


def test_unaligned_activations_and_leading_axes(gpu):
    N, K = 100, 520
    codes, scales = weights(N, K, 11)
    for M in (1, 30, 140, 300):
        flat = torch.randn(M * K + 1, device="cuda").half()
        A = flat[1:].view(M, K)
        check_product(A.double().cpu().numpy(), codes, scales, None, ops().matmul_mx4(A, codes, scales))
    A = torch.randn(2, 3, K, device="cuda").bfloat16()
    y = ops().matmul_mx4(A, codes, scales)
    assert tuple(y.shape) == (2, 3, N)
    check_product(A.double().cpu().numpy().reshape(6, K), codes, scales, None, y)


@pytest.mark.parametrize("M,K,N", [(1, 4096, 512), (40, 8192, 256), (160, 4096, 512), (700, 2048, 640)])
def test_repeats_are_equal_bit_for_bit_and_out_is_used(gpu, M, K, N):
    codes, scales = weights(N, K, 1)
    A = torch.randn(M, K, device="cuda").half()
    first = ops().matmul_mx4(A, codes, scales)
    out = torch.full((M, N), float("nan"), device="cuda", dtype=torch.float16)
    for _ in range(3):
        assert ops().matmul_mx4(A, codes, scales, out=out) is out
        assert torch.equal(out, first)
    ac, as_ = ops().mx4_quantize(A)
    a = ops().matmul_mx4(ac, codes, scales, A_scales=as_)
    assert torch.equal(a, ops().matmul_mx4(ac, codes, scales, A_scales=as_))


@pytest.mark.parametrize("M", [1, 40, 160])
def test_other_stream_workspace_and_graph(gpu, M):
    N, K = 320, 8192
    codes, scales = weights(N, K, 2)
    A = torch.randn(M, K, device="cuda").half()
    eager = ops().matmul_mx4(A, codes, scales)
    W = LB.mx4_decode(codes.cpu().numpy(), scales.cpu().numpy())
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    y = ops().matmul_mx4(A, codes, scales, stream=st)
    st.synchronize()
    assert torch.equal(y, eager)
    need = ops().matmul_mx4_workspace_bytes(M, K, N)
    ws = torch.zeros(max(need, 4096), dtype=torch.uint8, device="cuda")
    for _ in range(2):
        assert torch.equal(ops().matmul_mx4(A, codes, scales, workspace=ws), eager)
    assert not ws[:4096].any()
    if need:
        with pytest.raises(ValueError):
            ops().matmul_mx4(A, codes, scales, workspace=ws[: need - 1])
    for kw in ({}, {"workspace": ws}):
        out = torch.empty(M, N, dtype=torch.float16, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            qc, qs = ops().mx4_quantize(A)
            out4 = ops().matmul_mx4(qc, codes, scales, A_scales=qs, **({} if not kw else {"workspace": ws}))
            ops().matmul_mx4(A, codes, scales, out=out, **kw)
        for i in range(3):
            A.copy_(torch.randn(M, K, device="cuda").half())
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            check_product(A.double().cpu().numpy(), codes, scales, None, out)
            c, s = ops().mx4_quantize(A)
            check_product(LB.mx4_decode(c.cpu().numpy(), s.cpu().numpy()), codes, scales, None, out4)
            ops().matmul_mx4(A, codes, scales)


@pytest.mark.parametrize("M", [1, 2, 3, 4, 8, 40, 150])
@pytest.mark.parametrize("dt,center", [("f16", 139), ("bf16", 245)])
def test_subnormal_activations(gpu, M, dt, center):
    """Activations below the smallest normal value count in full."""
    N, K = 70, 224
    codes, scales = weights(N, K, M, spread=1, center=center)
    t = DT[dt]
    step = torch.finfo(t).tiny * torch.finfo(t).eps
    A = (torch.randint(-30, 31, (M, K), generator=torch.Generator().manual_seed(M)).double() * step).to(t)
    y = ops().matmul_mx4(A.cuda(), codes, scales)
    check_product(A.double().numpy(), codes, scales, None, y)


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 16])
@pytest.mark.parametrize("K,N", [(1, 1), (31, 17), (2048, 5), (2080, 33), (4097, 130), (20000, 40), (70000, 3)])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_product_few_rows(gpu, M, K, N, dt):
    codes, scales = weights(N, K, M + K + N)
    A = torch.randn(M, K, generator=torch.Generator().manual_seed(K)).to(DT[dt])
    bias = torch.randn(N, generator=torch.Generator().manual_seed(N)).to(DT[dt]).cuda()
    y = ops().matmul_mx4(A.cuda(), codes, scales, bias)
    check_product(A.double().numpy(), codes, scales, bias, y)


@pytest.mark.parametrize("M", [20, 33])
@pytest.mark.parametrize("act", ["f16", "mx4"])
def test_rows_past_the_tiled_products_k(gpu, M, act):
    K, N = (1 << 21) + 96, 3
    codes, scales = weights(N, K, 3, spread=1, center=119)
    if act == "mx4":
        ac, as_ = weights(M, K, 4, spread=1, center=124)
        y = ops().matmul_mx4(ac, codes, scales, A_scales=as_, out_dtype=torch.float32)
        A = LB.mx4_decode(ac.cpu().numpy(), as_.cpu().numpy())
    else:
        A = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).half()
        y, A = ops().matmul_mx4(A.cuda(), codes, scales), A.double().numpy()
    check_product(A, codes, scales, None, y)


def test_kernel_names(gpu):
    assert ops().matmul_mx4_kernel(1, 4096, 4096).startswith("mx4_")
    with pytest.raises(ValueError):
        ops().matmul_mx4_kernel(1, 0, 4096)


@pytest.mark.parametrize("act,K", [("mx4", 2080), ("mx4", 2240), ("f16", 1056)])
def test_wide_tiles_with_ragged_edges(gpu, act, K):
    """256-tiles: rows, columns and blocks that end inside them, and scales that start at any byte."""
    M, N = 2040, 8180
    codes, scales = weights(N, K, K)
    assert ops().matmul_mx4_kernel(M, K, N, torch.uint8 if act == "mx4" else DT[act]) == "mx4_gemm_256"
    g = torch.Generator().manual_seed(K)
    if act == "mx4":
        ac, as_ = weights(M, K, K + 1, spread=4, center=126)
        y = ops().matmul_mx4(ac, codes, scales, A_scales=as_, out_dtype=torch.float32)
        check_product(LB.mx4_decode(ac.cpu().numpy(), as_.cpu().numpy()), codes, scales, None, y)
    else:
        A = torch.randn(M, K, generator=g).to(DT[act])
        check_product(A.double().numpy(), codes, scales, None, ops().matmul_mx4(A.cuda(), codes, scales))
