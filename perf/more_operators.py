"""Performance cases of the operators around the paged cache: what a decoder's layer does between
the residual stream and its attention.

  norm      residual addition and root-mean-square norm, out in the input's type or in 8 bits
  grad      its backward pass
  quantize  rows to 8 bits with a scale each: activations, and weights by their output channels
  linear    product of 8-bit rows with 8-bit weights, scaled for each token and channel
  rotary    rotary positions of queries and keys, and their gradients

A case is a dict of plain values; listed() gives the ones quoted, draw() more of the same ranges.
With `own` false run() computes an operator in elementary torch operations; with `own` true it
makes the library's calls. What is held in 8 bits is returned as the numbers it stands for.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-5
_I8_LINE = 16  # rows of 8-bit numbers start at multiples of this


def listed():
    return [
        # The next token of one sequence of GPT-2 small's width, out for an 8-bit linear layer.
        # Latency.
        dict(name="norm_token", op="norm", rows=1, C=768, type="bf16", residual=True, out="i8"),
        # GPT-2 small's training batch of 8 x 1024 tokens, fp32 as the trainer keeps it.
        dict(name="norm_prompt", op="norm", rows=8192, C=768, type="f32", residual=True,
             out="same"),
        # Its backward pass.
        dict(name="norm_grad_gpt2", op="grad", rows=8192, C=768, type="f32", residual=True),
        # A wide model's, in 16 bits, sequences packed without padding (odd rows).
        dict(name="norm_grad_wide", op="grad", rows=16381, C=4096, type="bf16", residual=True),
        # Activations of an odd width.
        dict(name="quantize_odd", op="quantize", rows=333, C=6401, type="f16"),
        # GPT-2 small's token embedding as the weights of its output layer.
        dict(name="quantize_weights", op="quantize", rows=50257, C=768, type="f32"),
        # The next token of one sequence through GPT-2 small's QKV projection. Latency.
        dict(name="linear_token", op="linear", M=1, N=2304, K=768, type="f32", bias=True),
        # 64 of them through GPT-2 XL's first MLP layer: the weights' bytes.
        dict(name="linear_batch", op="linear", M=64, N=6400, K=1600, type="f16", bias=True),
        # Logits of 1000 positions over the unpadded vocabulary (odd rows).
        dict(name="linear_logits", op="linear", M=1000, N=50257, K=768, type="f32", bias=False),
        # Prompts through a wide model.
        dict(name="linear_large", op="linear", M=8192, N=8192, K=8192, type="bf16", bias=False),
        # One decoding step of 64 requests far into a context that was made longer after
        # training, out of the fused rows. Latency.
        dict(name="rotary_step", op="rotary", tokens=64, heads=32, kv=8, hs=128, dims=128,
             type="bf16", layout="half", scaling="parts", factor=8.0, far=131072, back=False,
             place=False),
        # Gradients of GPT-2 small's queries and keys with half of each head turned, in place.
        dict(name="rotary_grad_gpt2", op="rotary", tokens=8192, heads=12, kv=12, hs=64, dims=32,
             type="f32", layout="pairs", scaling="none", factor=1.0, far=1024, back=True,
             place=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "grad", "quantize", "linear", "linear", "linear", "rotary"])
    t = rng.choice(["f32", "f16", "bf16"])
    if op in ("norm", "grad", "quantize"):
        C = rng.choice([64, 384, 768, 1024, 1600, 2048, 4096, 6400, 8192, 12288,
                        _log(rng, 1, 16384), _log(rng, 1, 16384) | 1])
        rows = _log(rng, 1, max(1, min(50257, (1 << 26) // C)))
        c = dict(op=op, rows=rows, C=C, type=t)
        if op != "quantize":
            c["residual"] = rng.random() < 0.7
        if op == "norm":
            c["out"] = rng.choice(["same", "i8"])
        return c
    if op == "linear":
        M = rng.choice([_log(rng, 1, 64), _log(rng, 1, 8192), 1 << rng.randrange(13)])
        N = rng.choice([768, 1600, 2304, 4096, 4800, 6400, 50257, _log(rng, 1, 16384)])
        K = rng.choice([64, 768, 1600, 4096, 6400, _log(rng, 1, 16384)])
        while M > 1 and M * N * K > 1 << 39 or M * N > 1 << 26:
            M = M * 2 // 3
        return dict(op=op, M=M, N=N, K=K, type=t, bias=rng.random() < 0.5)
    kv, group = rng.choice([1, 2, 6, 8, 12]), rng.choice([1, 2, 4, 8])
    hs = rng.choice([32, 64, 64, 80, 128, 128, 256])
    tokens = _log(rng, 1, 16384)
    while tokens > 1 and tokens * kv * (group + 1) * hs > 1 << 27:
        tokens //= 2
    scaling = rng.choice(["none", "none", "linear", "base", "parts"])
    return dict(op=op, tokens=tokens, heads=kv * group, kv=kv, hs=hs,
                dims=rng.choice([hs, hs, hs // 2, hs // 4]), type=t,
                layout=rng.choice(["half", "pairs"]), scaling=scaling,
                factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0, 32.0]),
                far=_log(rng, 64, 1 << 20), back=rng.random() < 0.4, place=rng.random() < 0.4)


# ------------------------------------------------------------------- inputs
class _Rng:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        t = torch.empty(shape, device="cuda", dtype=dtype)
        return t.normal_(0.0, std, generator=self.g)

    def uniform(self, *shape):
        return torch.rand(shape, device="cuda", generator=self.g)

    def bytes(self, *shape):
        """8-bit numbers as quantised normal values have them, the ends included."""
        t = torch.empty(shape, device="cuda", dtype=torch.float16)
        return t.normal_(0.0, 36.0, generator=self.g).clamp_(-127, 127).to(torch.int8)

    def below(self, n, *shape):
        return torch.randint(0, n, shape, device="cuda", generator=self.g, dtype=torch.int32)


def _bmb():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "bare-metal-bard_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import bmb
    return bmb


def _line(n):
    return -(-n // _I8_LINE) * _I8_LINE


def prepare(case, seed):
    c, r = dict(case), _Rng(seed)
    s = dict(c=c)
    _PREPARE[c["op"]](s, c, r)
    return s


def _stream_values(r, rows, C, t):
    """A residual stream: normal values, some channels far larger than the others."""
    big = torch.where(r.uniform(C) < 0.01, 12.0, 1.0)
    return (r.normal(rows, C) * big).to(t)


def _i8_rows(s, rows, C):
    s.update(q=torch.zeros(rows, _line(C), device="cuda", dtype=torch.int8),
             scales=torch.zeros(rows, device="cuda"))


def _prepare_norm(s, c, r):
    rows, C, t = c["rows"], c["C"], _TYPES[c["type"]]
    s.update(x=_stream_values(r, rows, C, t), weight=1.0 + 0.2 * r.normal(C),
             rstd=torch.zeros(rows, device="cuda"))
    if c["residual"]:
        s.update(residual=_stream_values(r, rows, C, t), sum=torch.zeros_like(s["x"]))
    if c["out"] == "i8":
        _i8_rows(s, rows, C)
    else:
        s["out"] = torch.zeros_like(s["x"])
    if own:
        bmb = s["bmb"] = _bmb()
        n = s["norm"] = bmb.RmsNorm(rows=rows, C=C, type=bmb.ELEMENT_TYPES[c["type"]], eps=_EPS,
                                    x=s["x"].data_ptr(), x_stride=C,
                                    weight=s["weight"].data_ptr(), rstd=s["rstd"].data_ptr())
        if c["residual"]:
            n.residual, n.residual_stride = s["residual"].data_ptr(), C
            n.sum, n.sum_stride = s["sum"].data_ptr(), C
        if c["out"] == "i8":
            n.out_type, n.out, n.out_stride = bmb.I8, s["q"].data_ptr(), s["q"].stride(0)
            n.scales = s["scales"].data_ptr()
        else:
            n.out_type, n.out, n.out_stride = n.type, s["out"].data_ptr(), C


def _prepare_grad(s, c, r):
    rows, C, t = c["rows"], c["C"], _TYPES[c["type"]]
    inp = _stream_values(r, rows, C, t)
    s.update(inp=inp, weight=1.0 + 0.2 * r.normal(C), dout=r.normal(rows, C, std=1e-2, dtype=t),
             dinp=torch.zeros(rows, C, device="cuda", dtype=t),
             rstd=torch.rsqrt(inp.float().square().mean(1) + _EPS),
             # what the batch's earlier part has left in the weights' gradient
             dweight=r.normal(C, std=1e-2))
    if c["residual"]:
        s["dres"] = r.normal(rows, C, std=1e-2, dtype=t)
    if own:
        bmb = s["bmb"] = _bmb()
        g = s["grad"] = bmb.RmsNormGrad(rows=rows, C=C, type=bmb.ELEMENT_TYPES[c["type"]],
                                        dinp_stride=C, dout_stride=C, inp_stride=C,
                                        **{k: s[k].data_ptr() for k in ("dinp", "dout", "inp",
                                                                        "weight", "rstd",
                                                                        "dweight")})
        if c["residual"]:
            g.dres, g.dres_stride = s["dres"].data_ptr(), C
        need = bmb.rms_norm_backward_workspace(g)
        s["work"] = torch.empty(need, device="cuda", dtype=torch.uint8)
        g.work, g.work_bytes = s["work"].data_ptr(), need


def _prepare_quantize(s, c, r):
    s["x"] = _stream_values(r, c["rows"], c["C"], _TYPES[c["type"]])
    _i8_rows(s, c["rows"], c["C"])
    if own:
        bmb = s["bmb"] = _bmb()
        s["type"] = bmb.ELEMENT_TYPES[c["type"]]


def _prepare_linear(s, c, r):
    M, N, K, t = c["M"], c["N"], c["K"], _TYPES[c["type"]]
    s.update(A=r.bytes(M, _line(K)), B=r.bytes(N, _line(K)),
             a_scales=0.01 + 0.04 * r.uniform(M), b_scales=2e-4 + 6e-4 * r.uniform(N),
             bias=r.normal(N, std=0.1) if c["bias"] else None,
             out=torch.zeros(M, N, device="cuda", dtype=t))
    if own:
        bmb = s["bmb"] = _bmb()
        g = s["gemm"] = bmb.GemmI8(M=M, N=N, K=K, type=bmb.ELEMENT_TYPES[c["type"]],
                                   A=s["A"].data_ptr(), B=s["B"].data_ptr(),
                                   a_scales=s["a_scales"].data_ptr(),
                                   b_scales=s["b_scales"].data_ptr(), C=s["out"].data_ptr(),
                                   lda=_line(K), ldb=_line(K), ldc=N)
        if c["bias"]:
            g.bias = s["bias"].data_ptr()
        need = bmb.gemm_i8_workspace(g)
        s["work"] = torch.empty(need, device="cuda", dtype=torch.uint8)
        g.work, g.work_bytes = s["work"].data_ptr(), need


_BASE, _TRAINED, _SLOW, _FAST = 10000.0, 8192, 1.0, 32.0


def _amplitude(c):
    """The temperature that goes with a context scaled by parts."""
    return 0.1 * math.log(c["factor"]) + 1.0 if c["scaling"] == "parts" and not c["place"] else 1.0


def _prepare_rotary(s, c, r):
    T, hs, t = c["tokens"], c["hs"], _TYPES[c["type"]]
    turned, width = (c["heads"] + c["kv"]) * hs, (c["heads"] + 2 * c["kv"]) * hs
    # Rows of the fused projection (or their gradients): queries, keys, values.
    s.update(qkv=r.normal(T, width, dtype=t), positions=r.below(c["far"], T))
    if not c["place"]:
        s["out"] = torch.zeros(T, turned, device="cuda", dtype=t)
    if own:
        bmb = s["bmb"] = _bmb()
        p = s["plan"] = bmb.Rotary(head_size=hs, dims=c["dims"], amplitude=_amplitude(c),
                                   layout={"half": bmb.ROTARY_HALF,
                                           "pairs": bmb.ROTARY_PAIRS}[c["layout"]])
        kind = {"none": bmb.ROTARY_UNSCALED, "linear": bmb.ROTARY_LINEAR,
                "base": bmb.ROTARY_BASE, "parts": bmb.ROTARY_PARTS}[c["scaling"]]
        bmb.rotary_frequencies(p, _BASE, kind, c["factor"], _TRAINED, _SLOW, _FAST)
        s["type"] = bmb.ELEMENT_TYPES[c["type"]]


_PREPARE = dict(norm=_prepare_norm, grad=_prepare_grad, quantize=_prepare_quantize,
                linear=_prepare_linear, rotary=_prepare_rotary)


# --------------------------------------------------------------------- runs
def run(s):
    op = s["c"]["op"]
    return (_OWN if own else _PLAIN)[op](s, s["c"])


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _values(s, C):
    """The numbers that 8-bit rows stand for."""
    return torch.mul(s["q"][:, :C], s["scales"][:, None])


def _own_norm(s, c):
    s["bmb"].rms_norm_forward(s["norm"], _stream())
    out = s["out"] if c["out"] == "same" else _values(s, c["C"])
    return (out, s["rstd"], s["sum"]) if c["residual"] else (out, s["rstd"])


def _own_grad(s, c):
    s["bmb"].rms_norm_backward(s["grad"], _stream())
    return s["dinp"], s["dweight"]


def _own_quantize(s, c):
    s["bmb"].quantize_rows(s["q"].data_ptr(), s["q"].stride(0), s["scales"].data_ptr(),
                           s["x"].data_ptr(), c["C"], s["type"], c["rows"], c["C"], _stream())
    return _values(s, c["C"])


def _own_linear(s, c):
    s["bmb"].gemm_i8(s["gemm"], _stream())
    return s["out"]


def _own_rotary(s, c):
    bmb = s["bmb"]
    turn = bmb.rotary_backward if c["back"] else bmb.rotary_forward
    width = s["qkv"].stride(0)
    out, stride = (s["qkv"], width) if c["place"] else (s["out"], s["out"].stride(0))
    turn(s["plan"], out.data_ptr(), stride, s["qkv"].data_ptr(), width, s["type"], c["tokens"],
         c["heads"] + c["kv"], s["positions"].data_ptr(), _stream())
    return out


def _plain_i8(v):
    """(whole numbers, largest magnitude / 127) of 64-bit rows; where a number is half-way
    between two, 32 bits would not do."""
    a = v.abs().amax(1, keepdim=True)
    return torch.where(a > 0, torch.round(v * 127.0 / a), 0.0), a / 127.0


def _plain_norm(s, c):
    x = s["x"]
    if c["residual"]:
        s["sum"].copy_(x.float() + s["residual"].float())
        x = s["sum"]
    f = x.float()
    rstd = torch.rsqrt((f * f).mean(1, keepdim=True) + _EPS)
    s["rstd"].copy_(rstd[:, 0])
    if c["out"] == "i8":
        q, step = _plain_i8(x.double() * s["weight"].double())
        s["scales"].copy_((step * rstd.double())[:, 0])
        s["q"][:, :c["C"]] = q.to(torch.int8)
        out = _values(s, c["C"])
    else:
        s["out"].copy_(f * rstd * s["weight"])
        out = s["out"]
    return (out, s["rstd"], s["sum"]) if c["residual"] else (out, s["rstd"])


def _plain_grad(s, c):
    rstd = s["rstd"][:, None]
    dout, xhat = s["dout"].float(), s["inp"].float() * rstd
    d = dout * s["weight"]
    g = rstd * (d - xhat * (d * xhat).mean(1, keepdim=True))
    s["dinp"].copy_(g + s["dres"].float() if c["residual"] else g)
    s["dweight"].add_((dout * xhat).sum(0, dtype=torch.float64))
    return s["dinp"], s["dweight"]


def _plain_quantize(s, c):
    q, step = _plain_i8(s["x"].double())
    s["scales"].copy_(step[:, 0])
    s["q"][:, :c["C"]] = q.to(torch.int8)
    return _values(s, c["C"])


def _plain_linear(s, c):
    K = c["K"]
    y = torch.matmul(s["A"][:, :K].float(), s["B"][:, :K].float().t())
    y = y * s["a_scales"][:, None] * s["b_scales"]
    s["out"].copy_(y + s["bias"] if c["bias"] else y)
    return s["out"]


def _plain_frequencies(c):
    n = c["dims"]
    base, i = _BASE, torch.arange(0, n, 2, device="cuda", dtype=torch.float64)
    if c["scaling"] == "base" and n > 2:
        base = base * c["factor"] ** (n / (n - 2))
    f = torch.exp(-math.log(base) * i / n)
    if c["scaling"] == "linear":
        f = f / c["factor"]
    if c["scaling"] == "parts":
        keep = ((_TRAINED * f / (2 * math.pi) - _SLOW) / (_FAST - _SLOW)).clamp(0.0, 1.0)
        f = f * keep + f / c["factor"] * (1.0 - keep)
    return f


def _plain_rotary(s, c):
    T, hs, n, H = c["tokens"], c["hs"], c["dims"], c["heads"] + c["kv"]
    angle = s["positions"].double()[:, None] * _plain_frequencies(c)  # far positions
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if c["back"]:
        sin = -sin
    amp = _amplitude(c)
    src = s["qkv"][:, :H * hs].view(T, H, hs)
    out = src if c["place"] else s["out"].view(T, H, hs)
    x = src.float()
    if c["layout"] == "half":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], 2)
    else:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], 3).flatten(2)
    out[..., :n] = (turned * amp).to(out.dtype)
    if not c["place"]:
        out[..., n:] = src[..., n:]
    return s["qkv"] if c["place"] else s["out"]


_OWN = dict(norm=_own_norm, grad=_own_grad, quantize=_own_quantize, linear=_own_linear,
            rotary=_own_rotary)
_PLAIN = dict(norm=_plain_norm, grad=_plain_grad, quantize=_plain_quantize, linear=_plain_linear,
              rotary=_plain_rotary)


# --------------------------------------------------------------------- work
def work(case):
    c, op = case, case["op"]
    if op == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        return dict(bytes=(M + N) * K + 4 * (M + N) + 4 * N * c["bias"] + M * N * _SIZE[c["type"]],
                    flops=2 * M * N * K)
    size = _SIZE[c["type"]]
    if op == "rotary":
        T, hs, H = c["tokens"], c["hs"], c["heads"] + c["kv"]
        n = c["dims"] if c["place"] else hs
        return dict(bytes=2 * T * H * n * size + 4 * T, flops=3 * T * H * c["dims"])
    rows, C = c["rows"], c["C"]
    n = rows * C
    if op == "norm":
        # the norm's rows (x and the residual, and their sum); the result
        moved = n * size * (3 if c["residual"] else 1)
        moved += n * size if c["out"] == "same" else 9 * n  # 8-bit rows, read again as values
        return dict(bytes=moved + 4 * C + 8 * rows, flops=6 * n)
    if op == "grad":
        return dict(bytes=n * size * (4 if c["residual"] else 3) + 12 * C + 4 * rows,
                    flops=10 * n)
    return dict(bytes=n * size + 6 * n + 8 * rows, flops=3 * n)


# -------------------------------------------------------------------- exact
def exact(case, seed):
    c = dict(case)
    s = {}
    _plain_inputs(s, c, seed)
    return _EXACT[c["op"]](s, c)


def _plain_inputs(s, c, seed):
    """The case's inputs without the library's handles."""
    global own
    kept, own = own, False
    try:
        s.update(prepare(c, seed))
    finally:
        own = kept


def _exact_rows(rows, C):
    """Slices of rows that take about half a gigabyte in 64 bits."""
    step = max(1, (1 << 26) // C)
    return [slice(i, min(rows, i + step)) for i in range(0, rows, step)]


def _exact_i8(v):
    """The number nearest to each of v among 255 even steps over its row's range (the even one of
    two as near)."""
    top = v.abs().max(1).values.clamp(min=1e-300)[:, None]
    n = torch.div(v * 127.0, top)
    low = torch.floor(n)
    up = (n - low > 0.5) | ((n - low == 0.5) & (low % 2 != 0))
    return (low + up) * top / 127.0


def _exact_norm(s, c):
    parts = []
    for i in _exact_rows(c["rows"], c["C"]):
        x = s["x"][i].double()
        if c["residual"]:
            x = (x + s["residual"][i].double()).to(s["x"].dtype).double()
        scale = 1.0 / torch.sqrt(torch.linalg.vector_norm(x, dim=1) ** 2 / c["C"] + _EPS)
        y = torch.mul(x, s["weight"].double()[None, :])
        y = (_exact_i8(y) if c["out"] == "i8" else y) * scale[:, None]
        parts.append((y, scale) + ((x,) if c["residual"] else ()))
    return tuple(torch.cat(p) for p in zip(*parts))


def _exact_grad(s, c):
    w, dw, parts = s["weight"].double(), s["dweight"].double(), []
    for i in _exact_rows(c["rows"], c["C"]):
        x, r = s["inp"][i].double(), s["rstd"][i].double()[:, None]
        g = s["dout"][i].double()
        dw = dw + (g * (x * r)).sum(0)
        dot = torch.linalg.vecdot(g * w, x)[:, None]
        d = r * w * g - x * r ** 3 * dot / c["C"]
        parts.append(d + s["dres"][i].double() if c["residual"] else d)
    return torch.cat(parts), dw


def _exact_quantize(s, c):
    return torch.cat([_exact_i8(s["x"][i].double()) for i in _exact_rows(c["rows"], c["C"])])


def _exact_linear(s, c):
    K = c["K"]
    a = s["A"][:, :K].double() * s["a_scales"].double()[:, None]
    b = s["B"][:, :K].double() * s["b_scales"].double()[:, None]
    start = s["bias"].double() if c["bias"] else torch.zeros(c["N"], device="cuda").double()
    return torch.addmm(start, a, b.t())


def _exact_rotary(s, c):
    """Pairs as complex numbers, each frequency from its own definition."""
    T, hs, n, H = c["tokens"], c["hs"], c["dims"], c["heads"] + c["kv"]
    freq = []
    for i in range(n // 2):
        base = _BASE
        if c["scaling"] == "base" and n > 2:
            base *= math.pow(c["factor"], n / (n - 2))
        f = math.pow(base, -2.0 * i / n)
        if c["scaling"] == "linear":
            f /= c["factor"]
        if c["scaling"] == "parts":
            turns = _TRAINED * f / math.tau
            keep = min(1.0, max(0.0, (turns - _SLOW) / (_FAST - _SLOW)))
            f = (1.0 - keep) * f / c["factor"] + keep * f
        freq.append(f)
    sign = -1.0 if c["back"] else 1.0
    p = s["positions"].double()[:, None] * torch.tensor(freq, device="cuda", dtype=torch.float64)
    turn = torch.polar(torch.full_like(p, _amplitude(c)), sign * p)[:, None]
    whole = s["qkv"].double()
    out = whole[:, :H * hs].reshape(T, H, hs).clone()
    at = torch.arange(n // 2, device="cuda")
    i, j = (at, at + n // 2) if c["layout"] == "half" else (2 * at, 2 * at + 1)
    z = torch.complex(out[..., i], out[..., j]) * turn
    out[..., i], out[..., j] = z.real, z.imag
    out = out.view(T, H * hs)
    return torch.cat([out, whole[:, H * hs:]], 1) if c["place"] else out


_EXACT = dict(norm=_exact_norm, grad=_exact_grad, quantize=_exact_quantize, linear=_exact_linear,
              rotary=_exact_rotary)
