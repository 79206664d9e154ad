"""rms_norm_backward of wide rows (include/nn.h): many of them a workgroup, and rows of 2^16 to 2^20
elements, whose mean is held in 64 bits, so that its bound does not grow with C. u = 2^-24.

A term of the mean rounds dout * weight and inp * rstd once each, and the mean rounds to fp32: 3 u
of the terms' magnitude. What follows rounds at most five times (those two again, the product with
the mean under one rounding, the product with rstd, and the addition of dres).
"""
import pytest
import torch

from rows_util import TYPES, U, close, half_step, smallest
from test_gpu_norm import backward, check_backward, gen, values

pytestmark = pytest.mark.gpu


def check(dout, inp, weight, dres, dinp, rstd):
    C, t = inp.shape[1], inp.dtype
    d, x, w, r = dout.double(), inp.double(), weight.double(), rstd.double()
    xhat = x * r
    dot = (d * w * xhat).mean(1, keepdim=True)
    terms = (d * w * xhat).abs().mean(1, keepdim=True)
    want = r * (d * w - xhat * dot)
    size = r * ((d * w).abs() + (xhat * dot).abs())
    if dres is not None:
        want = want + dres.double()
        size = size + dres.double().abs()
    bound = r * xhat.abs() * terms * 3.01 * U + 5.01 * U * size
    close(dinp, want, bound + want.abs() * half_step(t) + smallest(t))


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("C", [1 << 16, (1 << 18) + 13, 1 << 20])
def test_even_rows(gpu, name, C):
    """Rows of one value: every addition to a long sum in fp32 would be off the same way."""
    print("even rows", name, C, flush=True)
    t = TYPES[name][1]
    g = gen(C)
    inp, dout = ((1.0 + torch.rand(6, 1, generator=g)).to(t).expand(6, C).contiguous()
                 for _ in range(2))
    weight = (1.0 + torch.rand(1, generator=g)).expand(C).contiguous()
    dinp, _, rstd = backward(dout, inp, weight)
    check(dout, inp, weight, None, dinp, rstd)


@pytest.mark.parametrize("name", list(TYPES))
def test_rows(gpu, name):
    """Ordinary values, all of one sign, with what reaches the sum past the norm."""
    C, g, t = (1 << 19) + 5, gen(3), TYPES[name][1]
    inp, dout = (values(3, C, torch.float32, g).abs().to(t) for _ in range(2))
    dres, weight = torch.randn(3, C, generator=g).to(t), 1.0 + 0.1 * torch.randn(C, generator=g)
    dinp, _, rstd = backward(dout, inp, weight, dres)
    check(dout, inp, weight, dres, dinp, rstd)


@pytest.mark.parametrize("name,C", [("f32", 2500), ("bf16", 4100), ("f32", 8200), ("f16", 8200),
                                    ("bf16", 16400)])
def test_many_rows(gpu, name, C):
    """Six rows a workgroup, the last with one: a row's sums are not the next one's."""
    print("many rows", name, C, flush=True)
    rows, t, g = 512 * 5 + 9, TYPES[name][1], gen(C)
    assert rows % 6 == 1
    inp, dout, dres = (values(rows, C, t, g) for _ in range(3))
    weight, dw0 = 1.0 + 0.3 * torch.randn(C, generator=g), torch.randn(C, generator=g)
    check_backward(dout, inp, weight, dres, dw0, backward(dout, inp, weight, dres, dw0))
