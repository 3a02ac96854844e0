"""GPU parity of matmul_mx4 on each size of tile, with the tile asserted; tolerances as in test_gpu_mx4.py."""
import pytest

from oracle import lowbit as LB
from tests.test_gpu_mx4 import DT, check_product, ops, weights
from tests.test_mx4_plan import plan
from xrgpu_amd import _native as nat

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
AT = {"f16": nat.F16, "bf16": nat.BF16, "mx4": nat.U8}


def product(M, K, N, act, *, bias=False, out=torch.float32, odd=False):
    """One product of random operands, checked; `odd`: 16-bit activations that start at an odd element, scales at an odd byte."""
    codes, scales = weights(N, K, M + K + N)
    if odd:
        flat = torch.empty(scales.numel() + 1, dtype=torch.uint8, device="cuda")
        scales = flat[1:].copy_(scales.flatten()).view(scales.shape)
    g = torch.Generator().manual_seed(M + N)
    dt = out if act == "mx4" else DT[act]
    b = torch.randn(N, generator=g).to(dt).cuda() if bias else None
    if act == "mx4":
        ac, as_ = weights(M, K, M + 3 * K, spread=4, center=126)
        y = ops().matmul_mx4(ac, codes, scales, b, A_scales=as_, out_dtype=out)
        A = LB.mx4_decode(ac.cpu().numpy(), as_.cpu().numpy())
    else:
        A = torch.randn(M * K + 1, generator=g).to(dt).cuda()[1 if odd else 0:][:M * K].view(M, K)
        y = ops().matmul_mx4(A, codes, scales, b)
        A = A.double().cpu().numpy()
    check_product(A, codes, scales, b, y)


@pytest.mark.parametrize("act", list(AT))
@pytest.mark.parametrize("M,K,N,mixed", [(2040, 1000, 11000, False), (1000, 1056, 18900, False), (2048, 2080, 14300, True)])
def test_columns_of_192_end_inside_their_last_tile(gpu, act, M, K, N, mixed):
    t, mt, nb, ns, splits, _ = plan(M, K, N, AT[act])
    assert t == 256 and ns > 0 and (nb > 0) == mixed and (N - nb * 256) % 192 != 0
    product(M, K, N, act, bias=mixed)


# act, (M, K, N), tile, whether K is split: ragged rows, columns and blocks, and K that no 16-bit row's pieces divide
TILES = [("f16", (900, 544, 3900), 128, False), ("bf16", (1000, 257, 4000), 128, False), ("f16", (1010, 333, 3990), 128, False),
         ("bf16", (500, 4096, 4090), 128, True), ("f16", (65, 4157, 3265), 128, True), ("mx4", (900, 544, 3900), 128, False),
         ("mx4", (4231, 10776, 68), 128, True), ("f16", (2040, 1056, 8180), 256, False), ("bf16", (2030, 1001, 8170), 256, False),
         ("f16", (2040, 331, 8180), 256, False), ("bf16", (141, 4118, 16688), 256, True), ("f16", (250, 4104, 16600), 256, True),
         ("mx4", (2040, 2240, 8180), 256, False), ("mx4", (138, 28424, 5741), 256, True)]


@pytest.mark.parametrize("act,size,tile,split", TILES)
@pytest.mark.parametrize("odd", [False, True])
def test_tiles(gpu, act, size, tile, split, odd):
    t, mt, nb, ns, splits, nws = plan(*size, AT[act])
    assert t == tile and ns == 0 and (splits > 1) == split
    assert ops().matmul_mx4_kernel(*size, torch.uint8 if act == "mx4" else DT[act]) == f"mx4_gemm_{tile}"
    product(*size, act, bias=odd, odd=odd, out=torch.bfloat16 if odd else torch.float32)


@pytest.mark.parametrize("act,size,tile,split", [x for x in TILES if x[3]])
def test_split_tiles_without_a_workspace_and_again(gpu, act, size, tile, split):
    M, K, N = size
    codes, scales = weights(N, K, K)
    if act == "mx4":
        a, as_ = weights(M, K, M, spread=4, center=126)
        A, dt = LB.mx4_decode(a.cpu().numpy(), as_.cpu().numpy()), torch.float32
    else:
        a, as_, dt = torch.randn(M, K, generator=torch.Generator().manual_seed(K)).to(DT[act]).cuda(), None, DT[act]
        A = a.double().cpu().numpy()
    y = torch.full((M, N), float("nan"), device="cuda", dtype=dt)
    ptr = lambda t: None if t is None else t.data_ptr()
    nat.check(nat.lib().xrmm_matmul_mx4(ptr(a), ptr(as_), AT[act], ptr(codes), ptr(scales), None, ptr(y),
                                        {torch.float32: nat.F32, **{DT[k]: AT[k] for k in ("f16", "bf16")}}[dt], M, K, N, None, 0,
                                        torch.cuda.current_stream().cuda_stream))
    check_product(A, codes, scales, None, y)
    first = ops().matmul_mx4(a, codes, scales, A_scales=as_, out_dtype=dt)
    for _ in range(3):
        assert torch.equal(ops().matmul_mx4(a, codes, scales, A_scales=as_, out_dtype=dt), first)


# 16-bit activations alone, on each tile and on 192 columns
FLOATS = [x[:3] for x in TILES if x[0] == "f16"] + [("f16", (2040, 1000, 11000), 192), ("f16", (2048, 520, 14300), 192)]


@pytest.mark.parametrize("act,size,tile", FLOATS)
@pytest.mark.parametrize("odd", [False, True])
def test_scales_outside_binary16_on_tiles(gpu, act, size, tile, odd):
    """Some blocks' scales are 2^-40 or 2^18, met by activations that bring their products to ordinary ones or to nothing."""
    M, K, N = size
    t, _, _, ns, _, _ = plan(M, K, N, AT[act])
    assert t == min(256, tile + 64 * (tile == 192)) and (ns > 0) == (tile == 192)
    codes, scales = weights(N, K, K)
    scales[N // 3:N // 3 + 5, 1], scales[N - 1, 2] = 145, 87
    g = torch.Generator().manual_seed(M)
    A = torch.randn(M, K, generator=g)
    A[:, 32:64] *= 2.0 ** -14
    A = torch.cat([torch.zeros(1), A.flatten()]).half().cuda()[0 if odd else 1:]
    A = (A[1:] if odd else A.clone()).view(M, K)
    assert A.data_ptr() % 4 == (2 if odd else 0)
    check_product(A.double().cpu().numpy(), codes, scales, None, ops().matmul_mx4(A, codes, scales))


@pytest.mark.parametrize("act,size,tile", [x[:3] for x in TILES if x[1][1] < 5000] + [(a, (2040, 1000, 11000), 192) for a in AT])
def test_nonfinite_stays_in_its_row_and_column_on_tiles(gpu, act, size, tile):
    M, K, N = size
    codes, scales = weights(N, K, 5)
    scales[N - 3, 2] = 255
    if act == "mx4":
        a, as_ = weights(M, K, 6, center=125)
        as_[M - 2, 1] = 255
        y = ops().matmul_mx4(a, codes, scales, A_scales=as_, out_dtype=torch.float32)
    else:
        A = torch.randn(M, K, device="cuda").to(DT[act])
        A[M - 2, 40] = float("nan")
        y = ops().matmul_mx4(A, codes, scales)
    nan = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    nan[:, N - 3] = True
    nan[M - 2] = True
    assert torch.equal(y.isnan(), nan) and y[~nan].isfinite().all()
