"""rms_norm_forward, rms_norm_backward and quantize_rows (include/nn.h) against their formulas in
64 bits. 8-bit numbers have to be equal. u = 2^-24 is half a step of fp32.

Forward: out rounds s * rstd, that times weight, and rstd (a rounding of 64 bits): 3 u, and the
result's own half step.
Backward: dout * weight and xhat round once each; the sum over a row is at most 32 additions a
thread (C / 1024 in wide rows) and 22 more: together below (57 + C / 1024) u of the sum of its
terms' magnitudes; what follows rounds at most four times. dweight: at most 64 + 4 roundings of
sums, and one of each term.
"""
import itertools

import pytest
import torch

import bmb
from rows_util import TYPES, U, Rows, close, half_step, smallest

pytestmark = pytest.mark.gpu
EPS = 1e-5
NAMES = list(TYPES)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def values(rows, C, t, g):
    big = torch.where(torch.rand(C, generator=g) < 0.05, 20.0, 1.0)
    return (torch.randn(rows, C, generator=g) * big).to(t)


def i8_of(v):
    """(numbers, largest magnitude) of 64-bit rows."""
    a = v.abs().amax(1, keepdim=True)
    q = torch.where(a > 0, torch.round(v * 127.0 / a), torch.zeros_like(v))
    return q, a


def forward(x, weight, res=None, out_type="same", kept=True, eps=EPS, stride=None, skew=0,
            rstd=True, stream=0):
    """(out, scales, rstd, sum) as Rows from host tensors."""
    rows, C = x.shape
    name = next(n for n in NAMES if TYPES[n][1] == x.dtype)
    kind, t = TYPES[name]
    X = Rows(rows, C, t, stride, skew, x)
    W = Rows(1, C, torch.float32, values=weight[None])
    i8 = out_type == "i8"
    O = Rows(rows, C, torch.int8 if i8 else t, stride, skew)
    S, R = Rows(rows, 1, torch.float32), Rows(rows, 1, torch.float32)
    n = bmb.RmsNorm(rows=rows, C=C, type=kind, out_type=bmb.I8 if i8 else kind, eps=eps, x=X.ptr,
                    x_stride=X.stride, weight=W.ptr, out=O.ptr, out_stride=O.stride)
    if i8:
        n.scales = S.ptr
    if rstd:
        n.rstd = R.ptr
    keep = [X, W]
    K = None
    if res is not None:
        Q = Rows(rows, C, t, stride, skew, res)
        keep.append(Q)
        n.residual, n.residual_stride = Q.ptr, Q.stride
        if kept:
            K = Rows(rows, C, t, stride, skew)
            n.sum, n.sum_stride = K.ptr, K.stride
    bmb.rms_norm_forward(n, stream)
    torch.cuda.synchronize()
    bmb.check("rms_norm_forward")
    assert X.holds(x) and X.intact() and O.intact() and S.intact() and R.intact()
    assert K is None or K.intact()
    return O, S, R, K


def check_forward(x, weight, res, out_type, got, eps=EPS):
    O, S, R, K = got
    t = x.dtype
    s = x if res is None else (x.float() + res.float()).to(t)
    if K is not None:
        assert torch.equal(K.get(), s)
    f, w = s.double(), weight.double()
    rstd = 1.0 / torch.sqrt((f * f).mean(1, keepdim=True) + torch.tensor(eps).double())
    close(R.get(), rstd, rstd * (U * 1.001))
    if out_type == "i8":
        q, a = i8_of(f * w)
        assert torch.equal(O.get(), q.to(torch.int8))
        scale = a * rstd / 127.0
        close(S.get(), scale, scale * (U * 1.001) + 2.0 ** -150)
    else:
        y = f * rstd * w
        close(O.get(), y, y.abs() * (half_step(t) + 3.01 * U) + smallest(t))


# One piece of a row, whole waves of them, odd ends, each number of threads and pieces, and rows
# that are read twice.
WIDTHS = [1, 3, 7, 8, 64, 255, 768, 1023, 1025, 1600, 2048, 2049, 4097, 6400, 8192, 8193, 12289,
          16384, 16392, 20011]


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("name,out_type,added", [
    (n, o, a) for n, o, a in itertools.product(NAMES, ("same", "i8"), (True, False))])
def test_forward(gpu, name, out_type, added, C):
    print("rms_norm_forward", name, out_type, added, C, flush=True)
    g = gen(C * 7 + added)
    t, rows = TYPES[name][1], 5 if C > 2048 else 13
    x, weight = values(rows, C, t, g), 1.0 + 0.3 * torch.randn(C, generator=g)
    res = values(rows, C, t, g) if added else None
    check_forward(x, weight, res, out_type, forward(x, weight, res, out_type))


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("out_type", ["same", "i8"])
@pytest.mark.parametrize("C,stride,skew", [(768, 771, 1), (65, 2304, 3), (1600, 1600, 5),
                                           (16385, 16400, 1)])
def test_forward_strided(gpu, name, out_type, C, stride, skew):
    print("strided", name, out_type, C, stride, skew, flush=True)
    g = gen(C)
    t = TYPES[name][1]
    x, weight = values(6, C, t, g), 1.0 + 0.3 * torch.randn(C, generator=g)
    res = values(6, C, t, g)
    got = forward(x, weight, res, out_type, stride=stride, skew=skew)
    check_forward(x, weight, res, out_type, got)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 257, 5000])
def test_forward_rows(gpu, rows):
    g = gen(rows)
    x, weight = values(rows, 96, torch.bfloat16, g), torch.randn(96, generator=g)
    res = values(rows, 96, torch.bfloat16, g)
    for out_type in ("same", "i8"):
        check_forward(x, weight, res, out_type, forward(x, weight, res, out_type))


def test_forward_without_sum_and_rstd(gpu):
    """What is not kept changes nothing."""
    g = gen(5)
    x, weight = values(4, 200, torch.float16, g), torch.randn(200, generator=g)
    res = values(4, 200, torch.float16, g)
    a = forward(x, weight, res, "i8")
    b = forward(x, weight, res, "i8", kept=False, rstd=False)
    assert torch.equal(a[0].get(), b[0].get()) and torch.equal(a[1].get(), b[1].get())
    a, b = forward(x, weight, res), forward(x, weight, res, kept=False, rstd=False)
    assert torch.equal(a[0].get(), b[0].get())


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("C", [100, 5000, 16500])
def test_forward_in_place(gpu, name, C):
    """sum over x or residual, out over the other one; the same bits."""
    print("in place", name, C, flush=True)
    g = gen(C)
    kind, t = TYPES[name]
    x, res = values(3, C, t, g), values(3, C, t, g)
    weight = torch.randn(C, generator=g)
    O, _, R, K = forward(x, weight, res)
    for swap in (False, True):
        X, Q = Rows(3, C, t, values=x), Rows(3, C, t, values=res)
        W, R2 = Rows(1, C, torch.float32, values=weight[None]), Rows(3, 1, torch.float32)
        a, b = (Q, X) if swap else (X, Q)
        bmb.rms_norm_forward(bmb.RmsNorm(
            rows=3, C=C, type=kind, out_type=kind, eps=EPS, x=X.ptr, x_stride=C, residual=Q.ptr,
            residual_stride=C, sum=a.ptr, sum_stride=C, out=b.ptr, out_stride=C, weight=W.ptr,
            rstd=R2.ptr))
        assert torch.equal(a.get(), K.get()) and torch.equal(b.get(), O.get())
        assert torch.equal(R2.get(), R.get()) and a.intact() and b.intact()


def test_columns_of_one_buffer(gpu):
    """x, residual and both results are column ranges of the same rows."""
    g = gen(3)
    C, rows = 40, 7
    whole = Rows(rows, 4 * C, torch.float32, values=torch.randn(rows, 4 * C, generator=g))
    before = whole.get().clone()
    weight = torch.randn(C, generator=g)
    W = Rows(1, C, torch.float32, values=weight[None])
    p = whole.ptr
    bmb.rms_norm_forward(bmb.RmsNorm(
        rows=rows, C=C, type=bmb.F32, out_type=bmb.F32, eps=EPS, x=p, x_stride=4 * C,
        residual=p + 4 * C, residual_stride=4 * C, sum=p + 8 * C, sum_stride=4 * C,
        out=p + 12 * C, out_stride=4 * C, weight=W.ptr))
    O, _, _, K = forward(before[:, :C].contiguous(), weight, before[:, C:2 * C].contiguous())
    got = whole.get()
    assert torch.equal(got[:, :2 * C], before[:, :2 * C])
    assert torch.equal(got[:, 2 * C:3 * C], K.get()) and torch.equal(got[:, 3 * C:], O.get())


def test_one_row_for_all(gpu):
    """A residual of stride 0: one row added to all."""
    g = gen(4)
    x, res = values(9, 70, torch.float32, g), values(1, 70, torch.float32, g)
    weight = torch.randn(70, generator=g)
    O, _, _, _ = forward(x, weight, res.expand(9, 70).contiguous())
    X, Q, P = (Rows(9, 70, torch.float32, values=x), Rows(1, 70, torch.float32, values=res),
               Rows(9, 70, torch.float32))
    W = Rows(1, 70, torch.float32, values=weight[None])
    bmb.rms_norm_forward(bmb.RmsNorm(rows=9, C=70, type=bmb.F32, out_type=bmb.F32, eps=EPS,
                                     x=X.ptr, x_stride=70, residual=Q.ptr, residual_stride=0,
                                     out=P.ptr, out_stride=70, weight=W.ptr))
    assert torch.equal(P.get(), O.get())


@pytest.mark.parametrize("C", [32, 3000, 17000])
def test_extreme_rows(gpu, C):
    """Zeros, one nonzero, the type's largest and smallest numbers: their squares and products
    pass fp32's range on both sides."""
    top, low = torch.finfo(torch.float32).max, 1e-45
    x = torch.zeros(6, C)
    x[1, C // 2] = 3.0
    x[2] = top
    x[3] = low
    x[4, ::2], x[4, 1::2] = top, low
    x[5] = torch.linspace(-1e-30, 1e-30, C)
    weight = torch.linspace(0.5, 2.0, C)
    for out_type in ("same", "i8"):
        check_forward(x, weight, None, out_type, forward(x, weight, None, out_type))
    check_forward(x, weight * 1e30, None, "i8", forward(x, weight * 1e30, None, "i8"))


def test_not_finite(gpu):
    """A row with an infinity or a NaN (or a weight with one): 8 bits give zeros and a scale of
    NaN; the other rows are not touched by it. In the input's type the formula speaks."""
    x = torch.ones(5, 50)
    x[1, 7], x[2, 9], x[3, 49] = float("inf"), float("nan"), float("-inf")
    weight = torch.ones(50)
    O, S, R, _ = forward(x, weight, None, "i8")
    q, s = O.get(), S.get()[:, 0]
    assert torch.isnan(s[1:4]).all() and (q[1:4] == 0).all()
    assert (q[0] == 127).all() and torch.isfinite(s[[0, 4]]).all()
    O, _, _, _ = forward(x, weight)
    y = O.get()
    assert torch.isnan(y[1, 7]) and (y[1, :7] == 0).all() and torch.isnan(y[2]).all()
    for bad in (float("inf"), float("nan")):
        weight[3] = bad
        O, S, _, _ = forward(torch.ones(2, 50), weight, None, "i8")
        assert torch.isnan(S.get()).all() and (O.get() == 0).all()


def quantize(x, stride=None, skew=0, out_stride=None):
    rows, C = x.shape
    kind = next(k for k, t in TYPES.values() if t == x.dtype)
    X = Rows(rows, C, x.dtype, stride, skew, x)
    O, S = Rows(rows, C, torch.int8, out_stride, skew), Rows(rows, 1, torch.float32)
    bmb.quantize_rows(O.ptr, O.stride, S.ptr, X.ptr, X.stride, kind, rows, C)
    torch.cuda.synchronize()
    bmb.check("quantize_rows")
    assert O.intact() and S.intact() and X.holds(x)
    return O.get(), S.get()


def check_quantize(x, got):
    q, a = i8_of(x.double())
    assert torch.equal(got[0], q.to(torch.int8))
    close(got[1], a / 127.0, a / 127.0 * (U * 1.001) + 2.0 ** -150)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("C", WIDTHS)
def test_quantize(gpu, name, C):
    print("quantize_rows", name, C, flush=True)
    x = values(9, C, TYPES[name][1], gen(C))
    check_quantize(x, quantize(x))
    check_quantize(x, quantize(x, C + 3, 1, C + 5))


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("C", [256, 4096, 33000])
def test_quantize_half_way(gpu, name, C):
    """Numbers half-way between two steps, and next to it on both sides: largest magnitude 127/64
    makes every (2k + 1) / 128 half-way; an odd largest magnitude puts them where fp32 cannot
    tell."""
    t = TYPES[name][1]
    x = torch.zeros(4, C)
    odd = (torch.arange(C) % 254 * 2 - 253).float()
    x[0] = odd / 128.0
    x[0, 0] = 127.0 / 64.0
    x[1] = odd * (77.25 / 256)
    x[1, 5] = 127 * (77.25 / 128)
    x[2] = torch.nextafter(odd / 128.0, torch.tensor(1e9))
    x[2, 0] = 127.0 / 64.0
    x[3] = torch.nextafter(odd / 128.0, torch.tensor(-1e9))
    x[3, 0] = 127.0 / 64.0
    x = x.to(t)
    check_quantize(x, quantize(x))
    # the same half-way numbers as products with a weight
    w = torch.where(torch.arange(C) % 3 == 0, 0.5, 2.0)
    y = (x.double() / w.double()).to(t)
    check_forward(y, w, None, "i8", forward(y, w, None, "i8"))


@pytest.mark.parametrize("C", [254, 5000, 17000])
def test_half_way_products(gpu, C):
    """Products of 48 bits half-way between two steps, and next to it: 127 m w is the largest, so
    that (2k + 1) / 2 m w is half-way, which whole numbers tell without a rounding."""
    print("half-way products", C, flush=True)
    g = gen(C)
    m = torch.randint(1 << 14, 1 << 15, (8, 1), generator=g) * 2 + 1
    odd = torch.arange(C) % 254 * 2 - 253
    w = (torch.randint(1 << 23, 1 << 24, (1,), generator=g) | 1).expand(C)
    s = odd * m  # twice the value, so that it is whole
    s[:, 0] = 254 * m[:, 0]
    s[4:6, 1:] += 1
    s[6:8, 1:] -= 1
    x, weight = s.float() / 2, w.float()
    assert torch.equal((x.double() * 2).long(), s)
    O, _, _, _ = forward(x, weight, None, "i8")
    # q = 127 s / s[0], to the nearest, half-way to the even one
    num, den = 2 * 127 * s + s[:, :1], 2 * s[:, :1]
    q = num.div(den, rounding_mode="floor")
    q -= ((num % den == 0) & (q % 2 != 0)).long()
    assert torch.equal(O.get().long(), q)


def test_quantize_extremes(gpu):
    x = torch.zeros(7, 90)
    x[1] = torch.finfo(torch.float32).max
    x[1, ::2] *= 0.3
    x[2] = 1e-45
    x[3, 8] = -1e-40
    x[4, 3] = float("nan")
    x[5, 89] = float("-inf")
    x[6] = torch.linspace(-1e-37, 2e-37, 90)
    q, s = quantize(x)
    fine = [0, 1, 2, 3, 6]
    check_quantize(x[fine], (q[fine], s[fine]))
    assert (q[4:6] == 0).all() and torch.isnan(s[4:6]).all()
    assert (q[3, 8] == -127) and q.min() >= -127


# ------------------------------------------------------------------- backward
def backward(dout, inp, weight, dres=None, dw0=None, stride=None, skew=0, place=None, work=True,
             rstd=None):
    rows, C = inp.shape
    kind = next(k for k, t in TYPES.values() if t == inp.dtype)
    t = inp.dtype
    f = inp.double()
    if rstd is None:
        rstd = (1.0 / torch.sqrt((f * f).mean(1, keepdim=True) + EPS)).float()
    R = Rows(rows, 1, torch.float32, values=rstd)
    W = Rows(1, C, torch.float32, values=weight[None])
    b = dict(dout=Rows(rows, C, t, stride, skew, dout), inp=Rows(rows, C, t, stride, skew, inp))
    if dres is not None:
        b["dres"] = Rows(rows, C, t, stride, skew, dres)
    b["dinp"] = b[place] if place else Rows(rows, C, t, stride, skew)
    g = bmb.RmsNormGrad(rows=rows, C=C, type=kind, weight=W.ptr, rstd=R.ptr)
    for k, r in b.items():
        setattr(g, k, r.ptr)
        setattr(g, k + "_stride", r.stride)
    D = None
    if dw0 is not None:
        D = Rows(1, C, torch.float32, values=dw0[None])
        g.dweight = D.ptr
    need = bmb.rms_norm_backward_workspace(g)
    assert (need > 0) == (dw0 is not None)
    if work and need:
        ws = Rows(1, need, torch.uint8)
        g.work, g.work_bytes = ws.ptr, need
    bmb.rms_norm_backward(g)
    torch.cuda.synchronize()
    bmb.check("rms_norm_backward")
    assert all(r.intact() for r in b.values()) and (D is None or D.intact())
    assert not (work and need) or ws.intact()
    return b["dinp"].get(), None if D is None else D.get()[0], rstd


def check_backward(dout, inp, weight, dres, dw0, got):
    dinp, dw, rstd = got
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
    bound = r * xhat.abs() * terms * (57 + C / 1024) * U + 5 * U * size
    close(dinp, want, bound + want.abs() * half_step(t) + smallest(t))
    if dw0 is not None:
        sums = (d * xhat).sum(0)
        close(dw, dw0.double() + sums, 70 * U * (d * xhat).abs().sum(0)
              + 1.01 * U * (dw0.double() + sums).abs())


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("name,added", [(n, a) for n in NAMES for a in (True, False)])
def test_backward(gpu, name, added, C):
    print("rms_norm_backward", name, added, C, flush=True)
    g = gen(C + added)
    t, rows = TYPES[name][1], 6 if C > 2048 else 37
    inp, dout = values(rows, C, t, g), torch.randn(rows, C, generator=g).to(t)
    weight, dw0 = 1.0 + 0.3 * torch.randn(C, generator=g), torch.randn(C, generator=g)
    dres = torch.randn(rows, C, generator=g).to(t) if added else None
    check_backward(dout, inp, weight, dres, dw0, backward(dout, inp, weight, dres, dw0))


@pytest.mark.parametrize("rows", [1, 2, 5, 63, 64, 65, 1000, 4099, 70001])
def test_backward_rows(gpu, rows):
    print("backward rows", rows, flush=True)
    g = gen(rows)
    inp, dout = values(rows, 40, torch.float32, g), torch.randn(rows, 40, generator=g)
    weight, dw0 = torch.randn(40, generator=g), torch.zeros(40)
    got = backward(dout, inp, weight, None, dw0)
    check_backward(dout, inp, weight, None, dw0, got)
    again = backward(dout, inp, weight, None, dw0, work=False)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("C", [50, 2500, 16500])
def test_backward_places(gpu, name, C):
    """Rows of a stride off their alignment; dinp over each input; without dweight: one result."""
    print("backward places", name, C, flush=True)
    g = gen(C)
    t = TYPES[name][1]
    inp, dout, dres = (values(11, C, t, g) for _ in range(3))
    weight, dw0 = torch.randn(C, generator=g), torch.randn(C, generator=g)
    want = backward(dout, inp, weight, dres, dw0)
    check_backward(dout, inp, weight, dres, dw0, want)
    for kw in (dict(stride=C + 3, skew=1), dict(place="dout"), dict(place="inp"),
               dict(place="dres")):
        got = backward(dout, inp, weight, dres, dw0, **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), kw
    assert torch.equal(backward(dout, inp, weight, dres)[0], want[0])


def test_backward_against_differences(gpu):
    """The gradient of a weighted sum of the outputs, by central differences of the formula in 64
    bits (whose own error at steps of 1e-5 is below 1e-9 here)."""
    g = gen(11)
    C = 37
    x, weight, c = (torch.randn(3, C, generator=g), 1.0 + 0.3 * torch.randn(C, generator=g),
                    torch.randn(3, C, generator=g))

    def loss(x, w):
        return float((c.double() * x * w / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)).sum())

    dinp, dw, _ = backward(c, x, weight, None, torch.zeros(C))
    h = 1e-5
    for r, i in [(0, 0), (1, 17), (2, 36)]:
        d = torch.zeros(3, C, dtype=torch.float64)
        d[r, i] = h
        num = (loss(x.double() + d, weight.double()) - loss(x.double() - d, weight.double())) / 2 / h
        assert abs(num - dinp[r, i].item()) < 1e-5
        num = (loss(x.double(), weight.double() + d[r]) - loss(x.double(), weight.double() - d[r]))
        assert abs(num / 2 / h - dw[i].item()) < 1e-5
