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
