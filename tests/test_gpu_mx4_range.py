"""GPU: matmul_mx4 where operands are at the ends of their ranges and the products are not; tolerances as in test_gpu_mx4.py."""
import pytest

from oracle import lowbit as LB
from tests.test_gpu_mx4 import check_product, ops, weights

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

MS = pytest.mark.parametrize("M", [1, 2, 3, 16, 40, 300])


@MS
@pytest.mark.parametrize("K,N", [(224, 70), (4096, 33), (1000, 17)])
def test_largest_bfloat16_activations(gpu, M, K, N):
    codes, scales = weights(N, K, M, center=60)
    A = (torch.rand(M, K, generator=torch.Generator().manual_seed(M)) * 1e38 + 2.3e38).bfloat16()
    y = ops().matmul_mx4(A.cuda(), codes, scales)
    check_product(A.double().numpy(), codes, scales, None, y)


@MS
@pytest.mark.parametrize("a,w", [(4, 250), (250, 4), (1, 245), (200, 60)])
def test_mx4_scales_whose_product_is_in_range(gpu, M, a, w):
    K, N = 288, 70
    codes, scales = weights(N, K, M, spread=1, center=w)
    ac, as_ = weights(M, K, M + 1, spread=1, center=a)
    y = ops().matmul_mx4(ac, codes, scales, A_scales=as_, out_dtype=torch.float32)
    check_product(LB.mx4_decode(ac.cpu().numpy(), as_.cpu().numpy()), codes, scales, None, y)
