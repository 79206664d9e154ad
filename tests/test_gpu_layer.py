"""The operators around the paged cache together, as a decoder's layer uses them: a generation step
in 8 bits (pages, norm, QKV, positions, append, attention, projection, next norm), eager and as a
replayed graph, and a layer's training pass in fp32 with its gradients.

The step is checked link by link: each operator against its formula in 64 bits on what the one
before it left on the device (so no link's tolerance has to cover another's rounding)."""
import math

import pytest
import torch

import bmb
from gpu_util import fp32_order_bound
from rows_util import TYPES, U, Rows, close, half_step, smallest
from test_gpu_norm import i8_of
from test_gpu_rotary import expected

pytestmark = pytest.mark.gpu
EPS = 1e-5


class Step:
    """One layer's part of a generation step: R requests, each with one new token, some of them
    idle."""

    def __init__(self, R, lens, width, heads, kv, hs, name, page=16, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.kind, self.t = TYPES[name]
        t = self.t
        self.R, self.width, self.heads, self.kv, self.hs, self.page = R, width, heads, kv, hs, page
        self.lens = torch.tensor(lens, dtype=torch.int32)
        new = torch.ones(R, dtype=torch.int32)
        new[1::4] = 0  # idle
        held = -(-self.lens // page)
        self.max_pages = int(held.max()) + 2
        pages = self.pages = int(held.sum()) + R + 3
        order = torch.randperm(pages, generator=g).to(torch.int32)
        table = torch.full((R, self.max_pages), -1, dtype=torch.int32)
        at = 0
        for r in range(R):
            table[r, :held[r]] = order[at:at + int(held[r])]
            at += int(held[r])
        free = torch.full((pages,), -1, dtype=torch.int32)
        free[:pages - at] = order[at:]
        d = "cuda"
        i32 = dict(dtype=torch.int32, device=d)
        self.start = dict(table=table, free=free, lens_dev=self.lens.clone(),
                          state=torch.tensor([0, pages - at], dtype=torch.int32),
                          k=torch.randn(pages, page, kv, hs, generator=g).to(t),
                          v=torch.randn(pages, page, kv, hs, generator=g).to(t))
        for k, x in self.start.items():
            setattr(self, k, x.to(d).clone())
        self.new = new.to(d)
        self.slots, self.positions = torch.zeros(R, **i32), torch.zeros(R, **i32)
        self.rows, self.offsets = torch.zeros(R, **i32), torch.zeros(R + 1, **i32)
        self.plan = bmb.PagedPlan(
            requests=R, max_pages=self.max_pages, pages=pages, page_size=page, max_tokens=R,
            new_tokens=self.new.data_ptr(), lens=self.lens_dev.data_ptr(),
            lens_out=self.lens_dev.data_ptr(), state=self.state.data_ptr(),
            state_out=self.state.data_ptr(), free_pages=self.free.data_ptr(),
            block_table=self.table.data_ptr(), slots=self.slots.data_ptr(),
            positions=self.positions.data_ptr(), rows=self.rows.data_ptr(),
            offsets=self.offsets.data_ptr())
        # Weights, in 8 bits once.
        self.qkv_width = (heads + 2 * kv) * hs
        self.w_qkv, self.s_qkv, self.b_qkv = self.weights(self.qkv_width, width, g)
        self.w_out, self.s_out, self.b_out = self.weights(width, heads * hs, g)
        self.norm1, self.norm2 = ((1.0 + 0.2 * torch.randn(width, generator=g)).to(d)
                                  for _ in range(2))
        self.x = torch.randn(R, width, generator=g).to(t).to(d)
        self.res = torch.randn(R, width, generator=g).to(t).to(d)
        line = -(-width // 16) * 16
        z = lambda *s, dtype=t: torch.zeros(*s, dtype=dtype, device=d)  # noqa: E731
        self.sum1, self.sum2, self.y2 = z(R, width), z(R, width), z(R, width)
        self.q1, self.s1 = z(R, line, dtype=torch.int8), z(R, dtype=torch.float32)
        self.qkv = z(R, self.qkv_width)
        self.att, self.lse = z(R, heads * hs), z(R, heads, dtype=torch.float32)
        self.q2, self.s2 = z(R, heads * hs, dtype=torch.int8), z(R, dtype=torch.float32)
        self.proj = z(R, width)
        self.rstd1, self.rstd2 = z(R, dtype=torch.float32), z(R, dtype=torch.float32)
        self.rot = bmb.Rotary(head_size=hs, dims=hs, layout=bmb.ROTARY_HALF, amplitude=1.0)
        bmb.rotary_frequencies(self.rot, 10000.0, bmb.ROTARY_PARTS, 8.0, 4096, 1.0, 32.0)
        self.cache = bmb.PagedCache(k=self.k.data_ptr(), v=self.v.data_ptr(), type=self.kind,
                                    pages=pages, page_size=page, kv_heads=kv, head_size=hs,
                                    page_stride=page * kv * hs, token_stride=kv * hs,
                                    head_stride=hs)
        self.batch = bmb.PagedBatch(requests=R, max_len=int(self.lens.max()) + 1,
                                    table_stride=self.max_pages, heads=heads, n_rows=R,
                                    type=self.kind, scale=1.0 / math.sqrt(hs),
                                    q_stride=self.qkv_width, out_stride=heads * hs,
                                    block_table=self.table.data_ptr(),
                                    lens=self.lens_dev.data_ptr(), rows=self.rows.data_ptr())
        need = bmb.paged_attention_workspace(self.cache, self.batch)
        self.work = torch.empty(max(need, 1), dtype=torch.uint8, device=d)
        self.batch.work, self.batch.work_bytes = self.work.data_ptr(), need
        p = lambda x: x.data_ptr()  # noqa: E731
        self.n1 = bmb.RmsNorm(rows=R, C=width, type=self.kind, out_type=bmb.I8, eps=EPS, x=p(self.x),
                              x_stride=width, residual=p(self.res), residual_stride=width,
                              sum=p(self.sum1), sum_stride=width, weight=p(self.norm1),
                              out=p(self.q1), out_stride=line, scales=p(self.s1),
                              rstd=p(self.rstd1))
        self.n2 = bmb.RmsNorm(rows=R, C=width, type=self.kind, out_type=self.kind, eps=EPS,
                              x=p(self.proj), x_stride=width, residual=p(self.sum1),
                              residual_stride=width, sum=p(self.sum2), sum_stride=width,
                              weight=p(self.norm2), out=p(self.y2), out_stride=width,
                              rstd=p(self.rstd2))
        self.g1 = self.linear(self.q1, self.s1, self.w_qkv, self.s_qkv, self.b_qkv, self.qkv,
                              width)
        self.g2 = self.linear(self.q2, self.s2, self.w_out, self.s_out, self.b_out, self.proj,
                              heads * hs)

    def weights(self, n, k, g):
        w = (torch.randn(n, k, generator=g) * 0.05).cuda()
        line = -(-k // 16) * 16
        q = torch.zeros(n, line, dtype=torch.int8, device="cuda")
        s = torch.zeros(n, device="cuda")
        bmb.quantize_rows(q.data_ptr(), line, s.data_ptr(), w.data_ptr(), k, bmb.F32, n, k)
        torch.cuda.synchronize()
        ref, a = i8_of(w.double().cpu())
        assert torch.equal(q[:, :k].cpu(), ref.to(torch.int8))
        return q, s, (torch.randn(n, generator=g) * 0.1).cuda()

    def linear(self, a, sa, b, sb, bias, c, K):
        g = bmb.GemmI8(M=a.shape[0], N=b.shape[0], K=K, type=self.kind, A=a.data_ptr(),
                       B=b.data_ptr(), a_scales=sa.data_ptr(), b_scales=sb.data_ptr(),
                       bias=bias.data_ptr(), C=c.data_ptr(), lda=a.stride(0), ldb=b.stride(0),
                       ldc=c.stride(0))
        need = bmb.gemm_i8_workspace(g)
        if need:
            w = torch.empty(need, dtype=torch.uint8, device="cuda")
            g.work, g.work_bytes = w.data_ptr(), need
            self.keep = getattr(self, "keep", []) + [w]
        return g

    def reset(self):
        for k, x in self.start.items():
            getattr(self, k).copy_(x)
        for k in self.results:
            getattr(self, k).zero_()

    results = ("sum1", "q1", "s1", "qkv", "att", "lse", "q2", "s2", "proj", "sum2", "y2",
               "rstd1", "rstd2", "slots", "positions", "rows", "offsets")

    def run(self, stream):
        """The step, queued on `stream`."""
        R, size = self.R, self.qkv.element_size()
        turned = (self.heads + self.kv) * self.hs
        bmb.paged_plan(self.plan, stream)
        bmb.rms_norm_forward(self.n1, stream)
        bmb.gemm_i8(self.g1, stream)
        # queries and keys in place in the fused rows
        qkv = self.qkv.data_ptr()
        bmb.rotary_forward(self.rot, qkv, self.qkv_width, qkv, self.qkv_width, self.kind, R,
                           self.heads + self.kv, self.positions.data_ptr(), stream)
        bmb.paged_append(self.cache, qkv + self.heads * self.hs * size, qkv + turned * size,
                         self.kind, self.qkv_width, self.slots.data_ptr(), R, stream)
        bmb.paged_attention(self.cache, self.batch, self.att.data_ptr(), self.lse.data_ptr(),
                            qkv, stream)
        bmb.quantize_rows(self.q2.data_ptr(), self.heads * self.hs, self.s2.data_ptr(),
                          self.att.data_ptr(), self.heads * self.hs, self.kind, R,
                          self.heads * self.hs, stream)
        bmb.gemm_i8(self.g2, stream)
        bmb.rms_norm_forward(self.n2, stream)

    def get(self):
        torch.cuda.synchronize()
        names = self.results + ("k", "v", "table", "free", "state", "lens_dev")
        return {k: getattr(self, k).cpu().clone() for k in names}


def check_norm(x, res, weight, out, scales, rstd, kept, C):
    s = (x.float() + res.float()).to(x.dtype)
    assert torch.equal(kept, s)
    f, w = s.double(), weight.double()
    r = 1.0 / torch.sqrt((f * f).mean(1, keepdim=True) + torch.tensor(EPS).double())
    close(rstd[:, None], r, r * (U * 1.001))
    if scales is not None:
        q, a = i8_of(f * w)
        assert torch.equal(out[:, :C], q.to(torch.int8))
        close(scales[:, None], a * r / 127, a * r / 127 * (U * 1.001))
    else:
        y = f * r * w
        close(out, y, y.abs() * (half_step(x.dtype) + 3.01 * U) + smallest(x.dtype))


def check_linear(q, s, w, sw, bias, out, K):
    p = torch.matmul(q[:, :K].double(), w[:, :K].double().t()) * s.double()[:, None] * sw.double()
    want = p + bias.double()
    close(out, want, 3.01 * U * p.abs() + want.abs() * (half_step(out.dtype) + 1.01 * U)
          + smallest(out.dtype))


@pytest.mark.parametrize("name,R,width,heads,kv,hs,top", [
    ("bf16", 5, 768, 12, 12, 64, 40), ("f16", 33, 1600, 25, 5, 64, 300),
    ("f32", 3, 100, 4, 2, 32, 70), ("bf16", 64, 1024, 32, 8, 128, 2000)])
def test_generation_step(gpu, name, R, width, heads, kv, hs, top):
    print("generation step", name, R, width, heads, kv, hs, top, flush=True)
    g = torch.Generator().manual_seed(R)
    lens = torch.randint(1, top, (R,), generator=g).tolist()
    s = Step(R, lens, width, heads, kv, hs, name)
    s.reset()
    torch.cuda.synchronize()
    s.run(0)
    got = s.get()
    bmb.check("step")
    live = (got["rows"] >= 0).nonzero()[:, 0]
    assert len(live) == R - len(range(1, R, 4))
    check_norm(s.x.cpu(), s.res.cpu(), s.norm1.cpu(), got["q1"], got["s1"], got["rstd1"],
               got["sum1"], width)
    # the fused rows as the linear layer left them
    s.reset()
    bmb.paged_plan(s.plan, 0)
    bmb.rms_norm_forward(s.n1)
    bmb.gemm_i8(s.g1)
    torch.cuda.synchronize()
    qkv, turned = s.qkv.cpu(), (heads + kv) * hs
    check_linear(got["q1"], got["s1"], s.w_qkv.cpu(), s.s_qkv.cpu(), s.b_qkv.cpu(), qkv, width)
    want, bound = expected(s.rot, qkv[:, :turned], heads + kv, got["positions"], False)
    close(got["qkv"][:, :turned], want, bound)
    assert torch.equal(got["qkv"][:, turned:], qkv[:, turned:])
    # the cache holds the turned keys and the values at the step's slots
    keys, values = (got[k].view(-1, kv * hs) for k in ("k", "v"))
    for r in live.tolist():
        row = int(got["rows"][r])
        slot = int(got["slots"][row])
        assert int(got["positions"][row]) == lens[r]
        assert torch.equal(keys[slot], got["qkv"][row, heads * hs:turned])
        assert torch.equal(values[slot], qkv[row, turned:])
        # attention of the request's tokens
        n = lens[r] + 1
        page = got["table"][r].long()
        at = torch.arange(n)
        idx = page[at // s.page] * s.page + at % s.page
        k = keys[idx].double().view(n, kv, hs)
        v = values[idx].double().view(n, kv, hs)
        q = got["qkv"][row, :heads * hs].double().view(kv, heads // kv, hs)
        x = torch.matmul(q, k.permute(1, 2, 0)) / math.sqrt(hs)
        p = torch.softmax(x, 2)
        o = torch.matmul(p, v.permute(1, 0, 2)).reshape(-1)
        top_v = torch.matmul(p, v.abs().permute(1, 0, 2)).reshape(-1)
        # scores and weights in fp32 (a few u of the scores' terms), 2^-17 of a weight in bf16
        terms = torch.matmul(q.abs(), k.abs().permute(1, 2, 0)).amax() / math.sqrt(hs)
        off = top_v * (2.0 ** -17 + (hs + 8) * 2 * U * terms + (n + 16) * U)
        close(got["att"][row], o, off + o.abs() * half_step(s.t) + smallest(s.t))
    q2, a2 = i8_of(got["att"].double())
    assert torch.equal(got["q2"], q2.to(torch.int8))
    close(got["s2"][:, None], a2 / 127, a2 / 127 * (U * 1.001))
    check_linear(got["q2"], got["s2"], s.w_out.cpu(), s.s_out.cpu(), s.b_out.cpu(), got["proj"],
                 heads * hs)
    check_norm(got["proj"], got["sum1"], s.norm2.cpu(), got["y2"], None, got["rstd2"],
               got["sum2"], width)


@pytest.mark.parametrize("name,R,width,heads,kv,hs,top", [("bf16", 33, 768, 12, 4, 64, 700),
                                                          ("f32", 2, 4096, 32, 8, 128, 50)])
def test_captured_step(gpu, name, R, width, heads, kv, hs, top):
    """The step as a graph, replayed with eager work of the same program between the replays."""
    print("captured step", name, R, width, flush=True)
    g = torch.Generator().manual_seed(R)
    s = Step(R, torch.randint(1, top, (R,), generator=g).tolist(), width, heads, kv, hs, name)
    s.reset()
    torch.cuda.synchronize()
    s.run(0)
    want = s.get()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        s.run(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        s.reset()
        torch.cuda.synchronize()
        graph.replay()
        got = s.get()
        for k in want:
            assert torch.equal(got[k], want[k]), (i, k)
        s.reset()  # an eager step between the replays
        torch.cuda.synchronize()
        s.run(0)
        again = s.get()
        assert all(torch.equal(again[k], want[k]) for k in want), i
    bmb.check("captured step")


def test_training_pass(gpu):
    """x -> norm -> QKV (fp32 gemm) -> positions -> causal attention, and back: every gradient
    against automatic differentiation in 64 bits. Each of the chain's links is held to 1e-5
    normwise by its own tests; five of them on the longest path."""
    B, T, C, NH = 2, 70, 128, 2
    hs, N = C // NH, B * T
    g = torch.Generator().manual_seed(8)
    x, res = (torch.randn(N, C, generator=g) for _ in range(2))
    nw = 1.0 + 0.2 * torch.randn(C, generator=g)
    w = torch.randn(3 * C, C, generator=g) / math.sqrt(C)
    dout, dres = torch.randn(N, C, generator=g), torch.randn(N, C, generator=g)
    pos = torch.arange(T, dtype=torch.int32).repeat(B) + 500
    plan = bmb.Rotary(head_size=hs, dims=48, layout=bmb.ROTARY_PAIRS, amplitude=1.0)
    bmb.rotary_frequencies(plan, 10000.0)

    # in 64 bits
    X, RES, NW, W = (t.double().requires_grad_() for t in (x, res, nw, w))
    S = X + RES
    r = 1.0 / torch.sqrt((S * S).mean(1, keepdim=True) + EPS)
    QKV = (S * r * NW) @ W.t()
    freq = torch.tensor(list(plan.freq)[:24], dtype=torch.float64)
    angle = pos.double()[:, None] * freq
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    qk = QKV[:, :2 * C].view(N, 2 * NH, hs)
    a, b = qk[..., 0:48:2], qk[..., 1:48:2]
    turned = torch.stack([a * c - b * s, b * c + a * s], 3).flatten(2)
    qk = torch.cat([turned, qk[..., 48:]], 2).view(B, T, 2, NH, hs)
    V = QKV[:, 2 * C:].view(B, T, NH, hs)
    sc = torch.einsum("bthd,bshd->bhts", qk[:, :, 0], qk[:, :, 1]) / math.sqrt(hs)
    sc = sc.masked_fill(torch.ones(T, T).triu(1).bool(), -math.inf)
    OUT = torch.einsum("bhts,bshd->bthd", torch.softmax(sc, 3), V).reshape(N, C)
    (OUT * dout.double()).sum().backward(retain_graph=True)
    (S * dres.double()).sum().backward()

    # on the device
    d = lambda t: t.cuda().contiguous()  # noqa: E731
    z = lambda *sh: torch.zeros(*sh, device="cuda")  # noqa: E731
    dx, dr, dnw, dw = d(x), d(res), d(nw), d(w)
    kept, y, rstd, qkv = z(N, C), z(N, C), z(N), z(N, 3 * C)
    p = d(pos)
    bmb.rms_norm_forward(bmb.RmsNorm(
        rows=N, C=C, type=bmb.F32, out_type=bmb.F32, eps=EPS, x=dx.data_ptr(), x_stride=C,
        residual=dr.data_ptr(), residual_stride=C, sum=kept.data_ptr(), sum_stride=C,
        weight=dnw.data_ptr(), out=y.data_ptr(), out_stride=C, rstd=rstd.data_ptr()))
    with bmb.gemm_math(bmb.GEMM_MATH_FP32):
        bmb.gemm(False, True, N, 3 * C, C, 1.0, y.data_ptr(), dw.data_ptr(), 0.0, qkv.data_ptr())
    bmb.rotary_forward(plan, qkv.data_ptr(), 3 * C, qkv.data_ptr(), 3 * C, bmb.F32, N, 2 * NH,
                       p.data_ptr())
    out, lse = z(N, C), z(B * NH * T)
    bmb.flash_forward(out.data_ptr(), lse.data_ptr(), qkv.data_ptr(), B, T, C, NH)
    dqkv, dsum, do = z(N, 3 * C), z(B * NH * T), d(dout)
    bmb.flash_backward(dqkv.data_ptr(), dsum.data_ptr(), do.data_ptr(), qkv.data_ptr(),
                       out.data_ptr(), lse.data_ptr(), B, T, C, NH)
    bmb.rotary_backward(plan, dqkv.data_ptr(), 3 * C, dqkv.data_ptr(), 3 * C, bmb.F32, N, 2 * NH,
                        p.data_ptr())
    dy, gw, gnw = z(N, C), z(3 * C, C), z(C)
    dinp = d(dres)
    with bmb.gemm_math(bmb.GEMM_MATH_FP32):
        bmb.gemm(False, False, N, C, 3 * C, 1.0, dqkv.data_ptr(), dw.data_ptr(), 0.0,
                 dy.data_ptr())
        bmb.gemm(True, False, 3 * C, C, N, 1.0, dqkv.data_ptr(), y.data_ptr(), 0.0, gw.data_ptr())
    bmb.rms_norm_backward(bmb.RmsNormGrad(
        rows=N, C=C, type=bmb.F32, dout=dy.data_ptr(), dout_stride=C, inp=kept.data_ptr(),
        inp_stride=C, dres=dinp.data_ptr(), dres_stride=C, weight=dnw.data_ptr(),
        rstd=rstd.data_ptr(), dinp=dinp.data_ptr(), dinp_stride=C, dweight=gnw.data_ptr()))
    torch.cuda.synchronize()
    bmb.check("training pass")
    assert fp32_order_bound(3 * C) < 1e-5
    for got, want in ((out, OUT.detach()), (dinp, X.grad), (dinp, RES.grad), (gnw, NW.grad),
                      (gw, W.grad)):
        err = (got.double().cpu() - want).abs().max() / want.abs().max()
        assert err < 5e-5, float(err)
