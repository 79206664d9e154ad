"""rms_norm_*, quantize_rows, gemm_i8 and rotary_* on streams, in graphs and from several host
threads: the bits of a call on the null stream every time."""
import threading

import pytest
import torch

import bmb
from rows_util import TYPES

pytestmark = pytest.mark.gpu


class Calls:
    """One call of each operator, with results of its own; `work`: with workspaces of the
    caller's."""

    def __init__(self, seed, work=True, name="bf16", rows=300, C=1000, M=64, N=400, K=8192):
        g = torch.Generator(device="cuda").manual_seed(seed)
        kind, t = TYPES[name]
        rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        z = lambda *s, dtype=t: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa: E731
        f32 = torch.float32
        self.keep = keep = {}
        x, res, dout = (rnd(rows, C).to(t) for _ in range(3))
        w = 1.0 + 0.1 * rnd(C)
        keep.update(x=x, res=res, dout=dout, w=w)
        out = dict(sum=z(rows, C), out=z(rows, C), rstd=z(rows, dtype=f32),
                   q=z(rows, C, dtype=torch.int8), scales=z(rows, dtype=f32),
                   qx=z(rows, C, dtype=torch.int8), sx=z(rows, dtype=f32), dinp=z(rows, C),
                   dweight=z(C, dtype=f32), C=z(M, N), turned=z(rows, 10 * 64))
        self.out = out
        p = {k: v.data_ptr() for k, v in {**keep, **out}.items()}
        n = dict(rows=rows, C=C, type=kind, eps=1e-5, x=p["x"], x_stride=C, residual=p["res"],
                 residual_stride=C, sum=p["sum"], sum_stride=C, weight=p["w"], rstd=p["rstd"],
                 out_stride=C)
        self.norm = bmb.RmsNorm(out_type=kind, out=p["out"], **n)
        self.norm8 = bmb.RmsNorm(out_type=bmb.I8, out=p["q"], scales=p["scales"], **n)
        self.grad = bmb.RmsNormGrad(rows=rows, C=C, type=kind, dout=p["dout"], dout_stride=C,
                                    inp=p["sum"], inp_stride=C, weight=p["w"], rstd=p["rstd"],
                                    dinp=p["dinp"], dinp_stride=C, dweight=p["dweight"])
        A, B = (torch.randint(-127, 128, (r, K), device="cuda", generator=g, dtype=torch.int8)
                for r in (M, N))
        sa, sb = (torch.rand(r, device="cuda", generator=g) for r in (M, N))
        keep.update(A=A, B=B, sa=sa, sb=sb)
        self.gemm = bmb.GemmI8(M=M, N=N, K=K, type=kind, A=A.data_ptr(), B=B.data_ptr(),
                               a_scales=sa.data_ptr(), b_scales=sb.data_ptr(), C=p["C"], lda=K,
                               ldb=K, ldc=N)
        assert bmb.gemm_i8_workspace(self.gemm) > 0  # a product that is split
        if work:
            for s, need in ((self.grad, bmb.rms_norm_backward_workspace(self.grad)),
                            (self.gemm, bmb.gemm_i8_workspace(self.gemm))):
                keep["work%d" % need] = b = torch.empty(need, device="cuda", dtype=torch.uint8)
                s.work, s.work_bytes = b.data_ptr(), need
        self.rot = bmb.Rotary(head_size=64, dims=64, layout=bmb.ROTARY_HALF, amplitude=1.0)
        bmb.rotary_frequencies(self.rot, 10000.0)
        keep["heads"] = rnd(rows, 10 * 64).to(t)
        keep["pos"] = torch.arange(rows, device="cuda", dtype=torch.int32)
        self.kind, self.rows, self.C = kind, rows, C
        torch.cuda.synchronize()

    def run(self, stream, backward=True):
        p = {k: v.data_ptr() for k, v in {**self.keep, **self.out}.items()}
        bmb.rms_norm_forward(self.norm, stream)
        bmb.rms_norm_forward(self.norm8, stream)
        bmb.quantize_rows(p["qx"], self.C, p["sx"], p["x"], self.C, self.kind, self.rows, self.C,
                          stream)
        if backward:
            bmb.rms_norm_backward(self.grad, stream)
        bmb.gemm_i8(self.gemm, stream)
        bmb.rotary_forward(self.rot, p["turned"], 640, p["heads"], 640, self.kind, self.rows, 10,
                           p["pos"], stream)
        bmb.rotary_backward(self.rot, p["turned"], 640, p["turned"], 640, self.kind, self.rows, 7,
                            p["pos"], stream)

    def clear(self):
        for t in self.out.values():
            t.zero_()
        torch.cuda.synchronize()

    def get(self):
        torch.cuda.synchronize()
        bmb.check("calls")
        return {k: v.clone() for k, v in self.out.items()}

    def want(self):
        self.clear()
        self.run(0)
        return self.get()


def same(a, b, skip=()):
    for k in a:
        if k not in skip:
            assert torch.equal(a[k], b[k]), k


@pytest.mark.parametrize("work", [True, False])
def test_streams(gpu, work):
    """A side stream behind work of its own that fills the inputs late; leases of the library's
    when no workspace is given."""
    c = Calls(1, work)
    want = c.want()
    for _ in range(3):
        c.clear()
        s = torch.cuda.Stream()
        late = c.keep["x"].clone()
        c.keep["x"].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            big = torch.zeros(1 << 28, device="cuda")
            for _ in range(3):
                big.add_(1.0)
            c.keep["x"].copy_(late)
        c.run(s.cuda_stream)
        same(c.get(), want)


def test_two_graphs_at_once(gpu):
    """Two captured graphs with workspaces of their own, replayed on two streams together, with
    eager calls between the replays."""
    calls = [Calls(2), Calls(3)]
    wants = [c.want() for c in calls]
    graphs, streams = [], [torch.cuda.Stream() for _ in calls]
    for c, s in zip(calls, streams):
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            c.run(torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for i in range(4):
        for c in calls:
            c.clear()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        for c, w in zip(calls, wants):
            same(c.get(), w)
        same(calls[i % 2].want(), wants[i % 2])


def test_capture_without_workspaces(gpu):
    """gemm_i8 runs unsplit (the same bits: whole numbers), rms_norm_backward refuses."""
    c = Calls(4, work=False)
    want = c.want()
    c.clear()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s = torch.cuda.current_stream().cuda_stream
        with pytest.raises(ValueError):
            bmb.rms_norm_backward(c.grad, s)
        c.run(s, backward=False)
    for _ in range(3):
        c.clear()
        g.replay()
        same(c.get(), want, skip=("dinp", "dweight"))


def test_host_threads(gpu):
    """Four host threads on the null stream, leases at once."""
    calls = [Calls(10 + i, work=False) for i in range(4)]
    wants = [c.want() for c in calls]
    for c in calls:
        c.clear()
    errors, barrier = [], threading.Barrier(4)

    def go(c):
        try:
            barrier.wait()
            c.run(0)
            bmb.check("thread")
        except Exception as e:  # reported below
            errors.append(repr(e))

    threads = [threading.Thread(target=go, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=60)
    assert not any(t.is_alive() for t in threads) and not errors, errors
    for c, w in zip(calls, wants):
        same(c.get(), w)


def test_repeated_calls(gpu):
    """The same bits again and again; dweight adds up."""
    c = Calls(5)
    want = c.want()
    for i in range(3):
        c.run(0)
    got = c.get()
    same(got, want, skip=("dweight",))
    ratio = (got["dweight"] / want["dweight"]).median()
    assert abs(float(ratio) - 4.0) < 1e-5
