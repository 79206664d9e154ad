"""rotary_forward and rotary_backward (include/nn.h) against their formula in 64 bits.

The angle's fraction of a turn is rounded to fp32: at most 2^-26 of a turn, 1.6 u; sine and cosine
are off by at most 2 u more (u = 2^-24), and 1 u for the amplitude. Each product and their
difference round once: together below 8 u of amplitude * (|x| + |y|). Positions p add 2^-51 of
p * freq in radians.
"""
import math

import pytest
import torch

import bmb
from rows_util import TYPES, U, Rows, close, half_step, smallest

pytestmark = pytest.mark.gpu

LAYOUTS = {"half": bmb.ROTARY_HALF, "pairs": bmb.ROTARY_PAIRS}


def plan(hs, dims, layout="half", amplitude=1.0, base=10000.0, **kw):
    p = bmb.Rotary(head_size=hs, dims=dims, layout=LAYOUTS[layout], amplitude=amplitude)
    bmb.rotary_frequencies(p, base, **kw)
    return p


def expected(p, x, heads, pos, back):
    """(result, its bound) of host rows x (tokens, heads * hs)."""
    hs, n = p.head_size, p.dims
    freq = torch.tensor(list(p.freq)[:n // 2], dtype=torch.float64)
    angle = pos.double()[:, None] * freq
    if back:
        angle = -angle
    amp = float(p.amplitude)
    c, s = (torch.cos(angle) * amp)[:, None], (torch.sin(angle) * amp)[:, None]
    y = x.double().view(len(pos), heads, hs).clone()
    at = torch.arange(n // 2)
    i, j = (at, at + n // 2) if p.layout == bmb.ROTARY_HALF else (2 * at, 2 * at + 1)
    a, b = y[..., i].clone(), y[..., j].clone()
    y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    bound = torch.zeros_like(y)
    off = abs(amp) * (a.abs() + b.abs()) * (8 * U + 2.0 ** -51 * angle.abs()[:, None])
    bound[..., i], bound[..., j] = off, off
    y, bound = y.view(len(pos), -1), bound.view(len(pos), -1)
    turned = torch.zeros(hs, dtype=torch.bool)
    turned[i], turned[j] = True, True
    turned = turned.repeat(heads)
    bound = bound + torch.where(turned, y.abs() * half_step(x.dtype) + smallest(x.dtype), 0.0)
    return y, bound


def turn(p, x, heads, pos, back=False, in_stride=None, out_stride=None, skew=0, place=False,
         stream=0):
    T, width = x.shape
    kind = next(k for k, t in TYPES.values() if t == x.dtype)
    X = Rows(T, width, x.dtype, in_stride, skew, x)
    O = X if place else Rows(T, width, x.dtype, out_stride, skew)
    P = Rows(T, 1, torch.int32, values=pos[:, None])
    f = bmb.rotary_backward if back else bmb.rotary_forward
    f(p, O.ptr, O.stride, X.ptr, X.stride, kind, T, heads, P.ptr, stream)
    torch.cuda.synchronize()
    bmb.check("rotary")
    assert O.intact() and X.intact() and (place or X.holds(x))
    return O.get()


@pytest.mark.parametrize("hs,dims,heads", [(2, 2, 1), (4, 2, 3), (32, 32, 3), (64, 64, 24),
                                           (64, 32, 24), (64, 16, 1), (80, 20, 5), (80, 80, 2),
                                           (96, 90, 7), (127, 66, 3), (128, 128, 40), (128, 2, 9),
                                           (256, 256, 4), (256, 130, 16), (63, 62, 300)])
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("name", list(TYPES))
def test_heads(gpu, name, layout, hs, dims, heads):
    print("rotary", name, layout, hs, dims, heads, flush=True)
    g = torch.Generator().manual_seed(hs + dims)
    p = plan(hs, dims, layout, 1.25)
    x = torch.randn(7, heads * hs, generator=g).to(TYPES[name][1])
    pos = torch.randint(0, 5000, (7,), generator=g, dtype=torch.int32)
    for back in (False, True):
        want, bound = expected(p, x, heads, pos, back)
        out = turn(p, x, heads, pos, back)
        close(out, want, bound)
        assert torch.equal(turn(p, x, heads, pos, back, place=True), out)
        assert torch.equal(turn(p, x, heads, pos, back, heads * hs + 5, heads * hs + 3, 1), out)


@pytest.mark.parametrize("tokens", [1, 2, 255, 4097])
def test_tokens(gpu, tokens):
    g = torch.Generator().manual_seed(tokens)
    p = plan(32, 32)
    x = torch.randn(tokens, 64, generator=g)
    pos = torch.arange(tokens, dtype=torch.int32)
    want, bound = expected(p, x, 2, pos, False)
    close(turn(p, x, 2, pos), want, bound)


def test_any_position(gpu):
    """Far ones, the type's ends, and negative ones (their bound grows with p * freq)."""
    pos = torch.tensor([0, 1, -1, 131071, 10 ** 6, 2 ** 24 + 1, -2 ** 24 - 1, 2 ** 31 - 1, -2 ** 31],
                       dtype=torch.int32)
    x = torch.randn(len(pos), 128, generator=torch.Generator().manual_seed(1))
    for layout in LAYOUTS:
        p = plan(128, 128, layout)
        want, bound = expected(p, x, 1, pos, False)
        out = turn(p, x, 1, pos)
        close(out, want, bound)
        assert torch.equal(out[0], x[0])


def test_backward_undoes_forward(gpu):
    """The transpose of a turn is its inverse: two roundings of each element apart."""
    g = torch.Generator().manual_seed(2)
    p = plan(64, 48, "pairs")
    x = torch.randn(50, 5 * 64, generator=g)
    pos = torch.randint(0, 1 << 17, (50,), generator=g, dtype=torch.int32)
    back = turn(p, turn(p, x, 5, pos), 5, pos, back=True)
    pairs = x.view(50, 5, 32, 2).abs().sum(3, keepdim=True).expand(50, 5, 32, 2).reshape(50, -1)
    close(back, x, pairs * 32 * U)


def test_part_of_fused_rows(gpu):
    """Queries and keys of fused rows in place; the values stay."""
    g = torch.Generator().manual_seed(3)
    heads, kv, hs, T = 6, 2, 64, 33
    p = plan(hs, hs)
    x = torch.randn(T, (heads + 2 * kv) * hs, generator=g).to(torch.bfloat16)
    pos = torch.randint(0, 999, (T,), generator=g, dtype=torch.int32)
    X, P = Rows(T, x.shape[1], x.dtype, values=x), Rows(T, 1, torch.int32, values=pos[:, None])
    bmb.rotary_forward(p, X.ptr, X.stride, X.ptr, X.stride, bmb.BF16, T, heads + kv, P.ptr)
    got = X.get()
    width = (heads + kv) * hs
    want, bound = expected(p, x[:, :width], heads + kv, pos, False)
    close(got[:, :width], want, bound)
    assert torch.equal(got[:, width:], x[:, width:])


def test_one_row_for_all(gpu):
    """An input of stride 0: one row at many positions."""
    p = plan(32, 32)
    x = torch.randn(1, 32, generator=torch.Generator().manual_seed(4))
    pos = torch.arange(100, dtype=torch.int32)
    X, O = Rows(1, 32, torch.float32, values=x), Rows(100, 32, torch.float32)
    P = Rows(100, 1, torch.int32, values=pos[:, None])
    bmb.rotary_forward(p, O.ptr, 32, X.ptr, 0, bmb.F32, 100, 1, P.ptr)
    want, bound = expected(p, x.expand(100, 32), 1, pos, False)
    close(O.get(), want, bound)


def test_not_finite_stays_in_its_pair(gpu):
    p = plan(8, 8)
    x = torch.ones(3, 16)
    x[1, 2] = float("inf")
    x[2, 9] = float("nan")
    got = turn(p, x, 2, torch.full((3,), 3, dtype=torch.int32))
    bad = ~torch.isfinite(got)
    assert bad.nonzero().tolist() == [[1, 2], [1, 6], [2, 9], [2, 13]]


def test_caller_frequencies(gpu):
    """freq may be the caller's own."""
    p = bmb.Rotary(head_size=16, dims=16, layout=bmb.ROTARY_PAIRS, amplitude=0.5)
    for i in range(8):
        p.freq[i] = math.sqrt(i + 0.5)
    x = torch.randn(20, 16, generator=torch.Generator().manual_seed(5))
    pos = torch.arange(20, dtype=torch.int32) * 1000
    want, bound = expected(p, x, 1, pos, False)
    close(turn(p, x, 1, pos), want, bound)
