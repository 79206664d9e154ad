"""gemm_i8 (include/gemm.h) against the product in 64 bits.

The sum is exact. Rounding it to fp32, its product with a_scales, and the product with b_scales
and the bias: three roundings of the product and one of the result, u = 2^-24 each, and half a
step of the result's type.
"""
import pytest
import torch

import bmb
from rows_util import TYPES, U, Rows, close, half_step, smallest

pytestmark = pytest.mark.gpu


def line(n):
    return -(-n // 16) * 16


class Problem:
    def __init__(self, M, N, K, name="f32", bias=True, lda=None, ldb=None, ldc=None, skew=0, seed=0,
                 fill=None):
        g = torch.Generator().manual_seed(seed + M * 31 + N * 7 + K)
        self.M, self.N, self.K = M, N, K
        kind, self.t = TYPES[name]
        lda, ldb, ldc = lda or line(max(K, 1)), ldb or line(max(K, 1)), ldc or N
        # What lies behind a row's K is never zero.
        whole = [torch.randint(-128, 128, (r, ld), generator=g, dtype=torch.int8) | 1
                 for r, ld in ((M, lda), (N, ldb))]
        if fill is not None:
            for w in whole:
                w.fill_(fill)
        # canaries of 64 bytes keep the rows' alignment
        self.A, self.B = (Rows(len(w), w.shape[1], torch.int8, values=w) for w in whole)
        self.a, self.b = whole[0][:, :K], whole[1][:, :K]
        self.sa = 0.01 + torch.rand(M, 1, generator=g)
        self.sb = 0.01 + torch.rand(N, 1, generator=g)
        self.bias = torch.randn(N, 1, generator=g) * 100 if bias else None
        self.SA, self.SB = (Rows(len(s), 1, torch.float32, values=s) for s in (self.sa, self.sb))
        self.BI = Rows(N, 1, torch.float32, values=self.bias) if bias else None
        self.C = Rows(M, N, self.t, ldc, skew)
        self.g = bmb.GemmI8(M=M, N=N, K=K, type=kind, A=self.A.ptr, B=self.B.ptr,
                            a_scales=self.SA.ptr, b_scales=self.SB.ptr,
                            bias=self.BI.ptr if bias else None, C=self.C.ptr, lda=lda, ldb=ldb,
                            ldc=ldc)

    def run(self, work=True, stream=0):
        need = bmb.gemm_i8_workspace(self.g)
        self.ws = Rows(1, max(need, 1), torch.uint8)
        if work and need:
            self.g.work, self.g.work_bytes = self.ws.ptr, need
        torch.cuda.synchronize()
        bmb.gemm_i8(self.g, stream)
        torch.cuda.synchronize()
        bmb.check("gemm_i8")
        assert self.ws.intact()
        return self.C.get()

    def check(self, got):
        p = torch.matmul(self.a.double(), self.b.double().t())
        assert p.abs().max() < 2 ** 31 if p.numel() else True
        p = p * self.sa.double() * self.sb.double().t()
        want = p + self.bias.double().t() if self.bias is not None else p
        bound = 3.01 * U * p.abs() + want.abs() * (half_step(self.t) + 1.01 * U) + smallest(self.t)
        # From half a step past the type's largest number on a result is infinite (next to there
        # the bound decides nothing).
        top = torch.finfo(self.t).max * (1.0 + half_step(self.t) / 2)
        off = 4.02 * U * (p.abs() + want.abs())
        want = torch.where(want.abs() - off >= top, want.sign() * float("inf"), want)
        near = torch.isfinite(want) & (want.abs() + off >= top)
        close(got, torch.where(near, got.double(), want), bound)
        assert self.C.intact() and self.A.intact() and self.B.intact()


SIZES = [(1, 1, 1), (1, 1, 16), (2, 3, 5), (1, 64, 128), (1, 2304, 768), (1, 50257, 64),
         (3, 100, 127), (5, 31, 129), (7, 2049, 255), (16, 768, 64), (17, 33, 1000), (31, 63, 65),
         (32, 64, 256), (33, 65, 257), (48, 1600, 1600), (64, 6400, 1600), (65, 129, 130),
         (100, 1000, 3), (127, 127, 127), (128, 128, 128), (129, 257, 383), (200, 768, 2048),
         (256, 256, 256), (300, 700, 15), (513, 1025, 640), (1000, 1601, 96), (2048, 17, 512),
         (2048, 2048, 272), (4096, 1, 129)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("name", list(TYPES))
def test_sizes(gpu, name, M, N, K):
    print("gemm_i8", name, M, N, K, flush=True)
    p = Problem(M, N, K, name, bias=(M + N + K) % 2 == 0)
    p.check(p.run())


@pytest.mark.parametrize("M,N,K", [(16, 4096, 64), (30, 3000, 200), (64, 1600, 6400), (40, 4100, 96),
                                   (300, 700, 130), (2100, 2300, 130)])
@pytest.mark.parametrize("name", list(TYPES))
def test_roundings(gpu, name, M, N, K):
    """Without a bias every rounding is known: the sum's, its product's with a_scales, that one's
    with b_scales, all to fp32, and the result's. To the bit, however the product is cut."""
    print("roundings", name, M, N, K, flush=True)
    p = Problem(M, N, K, name, bias=False)
    p.SA.t.mul_(2.0 ** -12)  # (fp16 holds the results)
    y = torch.matmul(p.a.double(), p.b.double().t()).float() * (p.sa * 2.0 ** -12)
    want = (y.double() * p.sb.double().t()).float().to(p.t)
    assert torch.isfinite(want).all()
    p.run()
    assert p.C.holds(want)


@pytest.mark.parametrize("M,N,K,name", [(4100, 4099, 130, "bf16"), (4096, 4096, 256, "f32"),
                                        (1000, 50257, 80, "f16"), (8192, 2050, 129, "f32")])
def test_many_tiles(gpu, M, N, K, name):
    print("many tiles", M, N, K, name, flush=True)
    p = Problem(M, N, K, name)
    p.check(p.run())


@pytest.mark.parametrize("M,N,K,name,more,skew", [
    (1000, 50257, 48, "f32", 0, 0), (2304, 7001, 70, "f32", 3, 1), (2304, 6945, 33, "f32", 0, 7),
    (4096, 8001, 64, "bf16", 0, 0), (4001, 8065, 40, "f16", 5, 3), (256, 57121, 16, "f32", 0, 2),
    (2100, 7168, 20, "f32", 0, 5), (2304, 7001, 40, "f32", 39, 17)])
def test_rows_inside_lines(gpu, M, N, K, name, more, skew):
    """Large results whose rows begin at odd places, or all at the same odd place: every element
    is stored once, and nothing between the rows."""
    print("rows inside lines", M, N, K, name, more, skew, flush=True)
    p = Problem(M, N, K, name, ldc=N + more, skew=skew)
    p.check(p.run())


@pytest.mark.parametrize("stages", list(range(1, 19)) + [25, 40])
@pytest.mark.parametrize("M,N", [(16, 48), (70, 80), (33, 50257), (2048, 2048), (2100, 2300),
                                 (4096, 4096)])
def test_stages(gpu, M, N, stages):
    """Every number of stages of 128 k, the last one whole or not, in each tile; the sums against
    the product in 64 bits on the device."""
    for K in (128 * stages, 128 * stages - 61):
        print("stages", M, N, K, flush=True)
        g = torch.Generator(device="cuda").manual_seed(stages)
        ld = line(K)
        A, B = (torch.randint(-128, 128, (r, ld), device="cuda", generator=g, dtype=torch.int8) | 1
                for r in (M, N))
        one = torch.ones(max(M, N), device="cuda")
        C = Rows(M, N, torch.float32)
        c = bmb.GemmI8(M=M, N=N, K=K, type=bmb.F32, A=A.data_ptr(), B=B.data_ptr(),
                       a_scales=one.data_ptr(), b_scales=one.data_ptr(), C=C.ptr, lda=ld, ldb=ld,
                       ldc=N)
        need = bmb.gemm_i8_workspace(c)
        work = torch.empty(max(need, 1), device="cuda", dtype=torch.uint8)
        c.work, c.work_bytes = work.data_ptr() if need else None, need
        torch.cuda.synchronize()
        bmb.gemm_i8(c)
        torch.cuda.synchronize()
        bmb.check("gemm_i8")
        # whole numbers below 2^53; rounded to fp32 as the call does
        want = torch.matmul(A[:, :K].double(), B[:, :K].double().t()).float()
        assert torch.equal(C.t, want) and C.intact()


@pytest.mark.parametrize("M,N,K", [(1, 70, 300), (40, 50, 700), (150, 200, 333), (300, 260, 64)])
@pytest.mark.parametrize("name", list(TYPES))
def test_strides(gpu, name, M, N, K):
    print("strides", name, M, N, K, flush=True)
    p = Problem(M, N, K, name, lda=line(K) + 48, ldb=line(K) + 4096, ldc=N + 5, skew=1)
    p.check(p.run())


@pytest.mark.parametrize("M,N", [(1, 1), (3, 40), (130, 70)])
def test_nothing_to_add(gpu, M, N):
    """K = 0: the bias, or zeros."""
    for bias in (True, False):
        p = Problem(M, N, 0, "bf16", bias=bias)
        p.check(p.run())


@pytest.mark.parametrize("M,N", [(1, 5), (20, 33), (70, 70)])
def test_largest_sum(gpu, M, N):
    """131071 products of -128 by -128: 2^31 - 2^14 in 32 bits."""
    p = Problem(M, N, 131071, "f32", fill=-128)
    p.check(p.run())


@pytest.mark.parametrize("M,N,K", [(1, 768, 6400), (8, 96, 40000), (64, 256, 16000),
                                   (150, 130, 20000), (512, 512, 8192)])
def test_long_k(gpu, M, N, K):
    """Few results of many products: with a workspace, and with the library's; the same bits."""
    print("long k", M, N, K, flush=True)
    p = Problem(M, N, K, "f32")
    got = p.run()
    p.check(got)
    q = Problem(M, N, K, "f32")
    assert torch.equal(q.run(work=False), got)


def test_scales_pass_through(gpu):
    """A scale of NaN (a row that could not be put into 8 bits) makes its row NaN and no other,
    also where the sum is 0; a scale of 0 gives the bias."""
    p = Problem(70, 90, 64, "f32")
    p.A.t[5] = 0
    p.a[5] = 0
    p.sa[5], p.sa[6], p.sb[80] = float("nan"), 0.0, 0.0
    p.SA.t.copy_(p.sa)
    p.SB.t.copy_(p.sb)
    got = p.run()
    p.check(got)
    assert torch.isnan(got[5]).all() and torch.equal(got[6], p.bias[:, 0])
    assert torch.isfinite(got[[i for i in range(70) if i != 5]]).all()


def test_overflow_is_infinite(gpu):
    """Results past fp16's range."""
    p = Problem(40, 40, 512, "f16", bias=False)
    p.sa[:], p.sb[:] = 30.0, 30.0
    p.SA.t.copy_(p.sa)
    p.SB.t.copy_(p.sb)
    got = p.run()
    want = torch.matmul(p.a.double(), p.b.double().t()) * 900.0
    assert torch.equal(got, want.float().to(torch.float16)) and torch.isinf(got).any()
