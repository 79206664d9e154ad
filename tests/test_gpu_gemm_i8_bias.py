"""gemm_i8 (include/gemm.h): the product with b_scales and the bias share one rounding, however the
product is cut. Scales of eight bits and a bias in multiples of 2^-16 leave whatever is not rounded
exact in 64 bits (below 2^10, in multiples of 2^-28), so the results are known to the bit."""
import pytest
import torch

from rows_util import TYPES
from test_gpu_gemm_i8 import Problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K", [(1, 768, 130), (16, 4096, 64), (30, 3000, 200), (64, 1600, 6400),
                                   (40, 4100, 96), (300, 700, 130), (1000, 4096, 48),
                                   (2100, 2300, 130)])
@pytest.mark.parametrize("name", list(TYPES))
def test_one_rounding(gpu, name, M, N, K):
    print("bias in one rounding", name, M, N, K, flush=True)
    p = Problem(M, N, K, name)
    g = torch.Generator().manual_seed(M + N + K)
    p.sa = torch.randint(1, 256, (M, 1), generator=g) * 2.0 ** -20
    p.sb = torch.randint(1, 256, (N, 1), generator=g) * 2.0 ** -8
    p.bias = torch.randint(-1 << 22, 1 << 22, (N, 1), generator=g) * 2.0 ** -16
    for buffer, values in ((p.SA, p.sa), (p.SB, p.sb), (p.BI, p.bias)):
        buffer.t.copy_(values)
    sums = torch.matmul(p.a.double(), p.b.double().t())
    assert sums.abs().max() < 1 << 22
    y = (sums.float() * p.sa).double() * p.sb.double().t()
    want = (y + p.bias.double().t()).float()
    if M * N > 1000:  # a rounding of their own for either would show
        assert (want != y.float() + p.bias.t()).double().mean() > 0.01
    p.run()
    assert p.C.holds(want.to(p.t))
    assert p.C.intact()
