"""What rms_norm_forward, rms_norm_backward, quantize_rows, gemm_i8 and the rotary entry points
refuse, on the host, before anything is launched; the layout of their structs; and the
frequencies, which are host code. No GPU: every pointer here is a number."""
import ctypes
import math
import os
import subprocess

import pytest

import bmb

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 24  # addresses, never used: buffers are this far apart


def at(i):
    return (i + 1) * P


def refused(capfd, what, f, *args):
    with pytest.raises(ValueError):
        f(*args)
    assert what in capfd.readouterr().err
    assert bmb.last_error() == 0


def norm(**kw):
    f = dict(rows=4, C=64, type=bmb.F32, out_type=bmb.F32, eps=1e-5, x=at(0), residual=at(1),
             sum=at(2), weight=at(3), out=at(4), scales=at(5), rstd=at(6), x_stride=64,
             residual_stride=64, sum_stride=64, out_stride=64)
    f.update(kw)
    return bmb.RmsNorm(**f)


NORMS = [(dict(type=3), "type"), (dict(type=-1), "type"), (dict(out_type=bmb.F16), "out_type"),
         (dict(out_type=4), "out_type"), (dict(rows=-1), "rows"), (dict(C=0), "C not"),
         (dict(C=(1 << 24) + 1), "C not"), (dict(eps=0.0), "eps"), (dict(eps=-1.0), "eps"),
         (dict(eps=math.nan), "eps"), (dict(eps=math.inf), "eps"), (dict(x=None), "null"),
         (dict(weight=None), "null"), (dict(out=None), "null"),
         (dict(out_type=bmb.I8, scales=None), "null"), (dict(residual=None), "without residual"),
         (dict(x=at(0) + 2), "element"), (dict(sum=at(2) + 1), "element"),
         (dict(weight=at(3) + 2), "element"), (dict(rstd=at(6) + 1), "element"),
         (dict(x_stride=63), "stride"), (dict(x_stride=-64), "stride"),
         (dict(residual_stride=1), "stride"), (dict(sum_stride=0), "stride"),
         (dict(out_stride=0), "stride"), (dict(out_stride=(1 << 40) + 1), "stride"),
         (dict(out=at(2)), "overlap"), (dict(out=at(0) + 4), "overlap"),
         (dict(sum=at(0) + 256), "overlap"), (dict(sum=at(0), sum_stride=128), "overlap"),
         (dict(out_type=bmb.I8, out=at(0)), "overlap"), (dict(rstd=at(0)), "overlap"),
         (dict(out_type=bmb.I8, rstd=at(5)), "overlap"), (dict(weight=at(4)), "overlap"),
         (dict(weight=at(2)), "overlap"),
         (dict(out_type=bmb.I8, scales=at(4) + 64), "overlap")]


@pytest.mark.parametrize("kw,why", NORMS)
def test_norm_refuses(capfd, kw, why):
    refused(capfd, why, bmb.rms_norm_forward, norm(**kw))


def test_nothing_is_no_launch():
    bmb.rms_norm_forward(norm(rows=0, x=None))
    bmb.rms_norm_backward(grad(rows=0, inp=None))
    bmb.quantize_rows(None, 64, None, None, 64, bmb.F32, 0, 64)
    bmb.gemm_i8(gemm(M=0, A=None))
    bmb.gemm_i8(gemm(N=0, C=None))
    bmb.rotary_forward(rotary(), None, 64, None, 64, bmb.F32, 0, 1, None)
    assert bmb.last_error() == 0


def test_none_is_refused(capfd):
    for f in (bmb.rms_norm_forward, bmb.rms_norm_backward, bmb.gemm_i8):
        refused(capfd, "no arguments", f, None)
    refused(capfd, "no plan", bmb.rotary_forward, None, at(0), 64, at(1), 64, bmb.F32, 4, 1, at(2))
    assert bmb.rms_norm_backward_workspace(None) == 0 and bmb.gemm_i8_workspace(None) == 0


def grad(**kw):
    f = dict(rows=4, C=64, type=bmb.F32, dout=at(0), inp=at(1), dres=at(2), weight=at(3),
             rstd=at(4), dinp=at(5), dweight=at(6), dout_stride=64, inp_stride=64, dres_stride=64,
             dinp_stride=64, work=at(7), work_bytes=1 << 20)
    f.update(kw)
    return bmb.RmsNormGrad(**f)


@pytest.mark.parametrize("kw,why", [
    (dict(type=3), "type"), (dict(rows=-1), "rows"), (dict(C=0), "C not"),
    (dict(C=1 << 25), "C not"), (dict(dout=None), "null"), (dict(inp=None), "null"),
    (dict(weight=None), "null"), (dict(rstd=None), "null"), (dict(dinp=None), "null"),
    (dict(dres=at(2) + 2), "element"), (dict(dweight=at(6) + 1), "element"),
    (dict(work=at(7) + 2), "element"), (dict(dout_stride=63), "stride"),
    (dict(dinp_stride=0), "stride"), (dict(dres_stride=-1), "stride"),
    (dict(dinp=at(0) + 4), "overlap"), (dict(dinp=at(2), dinp_stride=65), "overlap"),
    (dict(dweight=at(1)), "overlap"), (dict(dweight=at(5)), "overlap"),
    (dict(dweight=at(3)), "overlap"), (dict(dinp=at(3)), "overlap"), (dict(rstd=at(5)), "overlap"),
    (dict(work_bytes=255), "too small"), (dict(work=at(5)), "overlap"),
    (dict(work=at(0) + 16), "overlap"), (dict(work=at(6)), "overlap")])
def test_backward_refuses(capfd, kw, why):
    refused(capfd, why, bmb.rms_norm_backward, grad(**kw))


def test_backward_workspace():
    """Sums of at most 64 rows each; none without dweight, none for what is refused."""
    assert bmb.rms_norm_backward_workspace(grad()) >= 256
    assert bmb.rms_norm_backward_workspace(grad(dweight=None)) == 0
    assert bmb.rms_norm_backward_workspace(grad(rows=0)) == 0
    assert bmb.rms_norm_backward_workspace(grad(C=0)) == 0
    assert bmb.rms_norm_backward_workspace(grad(type=9)) == 0
    big = bmb.rms_norm_backward_workspace(grad(rows=(1 << 31) - 1, C=16384))
    assert big >= ((1 << 31) // 64) * 16384 * 4


@pytest.mark.parametrize("kw,why", [
    (dict(type=3), "type"), (dict(rows=-1), "rows"), (dict(C=0), "C not"), (dict(out=None), "null"),
    (dict(scales=None), "null"), (dict(x=None), "null"), (dict(x=at(1) + 2), "element"),
    (dict(scales=at(2) + 1), "element"), (dict(x_stride=63), "stride"),
    (dict(out_stride=63), "stride"), (dict(out_stride=0), "stride"), (dict(out=at(1)), "overlap"),
    (dict(scales=at(1)), "overlap"), (dict(scales=at(0)), "overlap")])
def test_quantize_refuses(capfd, kw, why):
    f = dict(out=at(0), out_stride=64, scales=at(2), x=at(1), x_stride=64, type=bmb.F32, rows=4,
             C=64)
    f.update(kw)
    refused(capfd, why, bmb.quantize_rows, *f.values())


def gemm(**kw):
    f = dict(M=4, N=8, K=64, type=bmb.F32, A=at(0), B=at(1), a_scales=at(2), b_scales=at(3),
             bias=at(4), C=at(5), lda=64, ldb=64, ldc=8)
    f.update(kw)
    return bmb.GemmI8(**f)


@pytest.mark.parametrize("kw,why", [
    (dict(type=3), "type"), (dict(M=-1), "negative"), (dict(N=-1), "negative"),
    (dict(K=-1), "negative"), (dict(K=131072, lda=131072, ldb=131072), "131071"),
    (dict(A=None), "null"), (dict(B=None), "null"), (dict(a_scales=None), "null"),
    (dict(b_scales=None), "null"), (dict(C=None), "null"), (dict(lda=48), "lda"),
    (dict(ldb=63), "ldb"), (dict(lda=1 << 23), "lda"), (dict(lda=72), "16 bytes"),
    (dict(ldb=65), "16 bytes"), (dict(A=at(0) + 8), "16 bytes"), (dict(B=at(1) + 1), "16 bytes"),
    (dict(ldc=7), "ldc"), (dict(C=at(5) + 2), "element"), (dict(a_scales=at(2) + 2), "element"),
    (dict(bias=at(4) + 1), "element"), (dict(C=at(0)), "overlap"), (dict(C=at(1) + 64), "overlap"),
    (dict(C=at(3)), "overlap"), (dict(C=at(4) - 16), "overlap"),
    (dict(M=1 << 30, N=1 << 30), "too many")])
def test_gemm_refuses(capfd, kw, why):
    refused(capfd, why, bmb.gemm_i8, gemm(**kw))


@pytest.mark.parametrize("kw,why", [
    (dict(work_bytes=16), "too small"), (dict(work=at(6) + 8), "16 bytes"),
    (dict(work=at(0)), "overlap"), (dict(work=at(1) - 256), "overlap"),
    (dict(work=at(2)), "overlap"), (dict(work=at(3)), "overlap"), (dict(work=at(4)), "overlap"),
    (dict(work=at(5)), "overlap")])
def test_gemm_refuses_workspace(capfd, kw, why):
    g = gemm(M=64, N=64, K=16384, lda=16384, ldb=16384, ldc=64, work=at(6), work_bytes=1 << 22)
    need = bmb.gemm_i8_workspace(g)
    assert 2 * 64 * 64 * 4 <= need <= 1 << 22
    for k, v in kw.items():
        setattr(g, k, v)
    refused(capfd, why, bmb.gemm_i8, g)


def test_gemm_workspace():
    """Only what is split needs one; none for what is refused."""
    assert bmb.gemm_i8_workspace(gemm()) == 0
    assert bmb.gemm_i8_workspace(gemm(K=0, A=None, B=None)) == 0
    assert bmb.gemm_i8_workspace(gemm(M=0, K=16384)) == 0
    assert bmb.gemm_i8_workspace(gemm(K=131072)) == 0
    assert bmb.gemm_i8_workspace(gemm(type=7, K=16384)) == 0


def rotary(**kw):
    f = dict(head_size=64, dims=64, layout=bmb.ROTARY_HALF, amplitude=1.0)
    f.update(kw)
    return bmb.Rotary(**f)


@pytest.mark.parametrize("plan,kw,why", [
    (dict(head_size=1), {}, "head size"), (dict(head_size=257), {}, "head size"),
    (dict(dims=0), {}, "dims"), (dict(dims=63), {}, "dims"), (dict(dims=66), {}, "dims"),
    (dict(layout=2), {}, "layout"), ({}, dict(type=3), "type"), ({}, dict(tokens=-1), "tokens"),
    ({}, dict(heads=0), "heads"), ({}, dict(heads=65537), "heads"), ({}, dict(out=None), "null"),
    ({}, dict(inp=None), "null"), ({}, dict(positions=None), "null"),
    ({}, dict(out=at(0) + 2), "element"), ({}, dict(positions=at(2) + 2), "element"),
    ({}, dict(out_stride=127), "stride"), ({}, dict(inp_stride=127), "stride"),
    ({}, dict(out_stride=0), "stride"), ({}, dict(out=at(1) + 256), "overlap"),
    ({}, dict(out=at(1), out_stride=129), "overlap"), ({}, dict(positions=at(0)), "overlap")])
@pytest.mark.parametrize("f", [bmb.rotary_forward, bmb.rotary_backward])
def test_rotary_refuses(capfd, f, plan, kw, why):
    a = dict(out=at(0), out_stride=128, inp=at(1), inp_stride=128, type=bmb.F32, tokens=4, heads=2,
             positions=at(2))
    a.update(kw)
    refused(capfd, why, f, rotary(**plan), *a.values())


@pytest.mark.parametrize("plan,kw,why", [
    (dict(dims=63), {}, "dims"), (dict(head_size=300, dims=2), {}, "head size"),
    ({}, dict(base=0.0), "base"), ({}, dict(base=math.nan), "base"),
    ({}, dict(base=math.inf), "base"), ({}, dict(scaling=4), "scaling"),
    ({}, dict(scaling=-1), "scaling"), ({}, dict(scaling=1, factor=0.5), "factor"),
    ({}, dict(scaling=2, factor=math.nan), "factor"), ({}, dict(scaling=3, factor=2.0), "trained"),
    ({}, dict(scaling=3, factor=2.0, trained_len=9, slow=2.0, fast=2.0), "slow"),
    ({}, dict(scaling=3, factor=2.0, trained_len=9, slow=-1.0, fast=2.0), "slow"),
    ({}, dict(scaling=3, factor=2.0, trained_len=9, slow=1.0, fast=math.inf), "slow")])
def test_frequencies_refuse(capfd, plan, kw, why):
    a = dict(base=10000.0)
    a.update(kw)
    refused(capfd, why, lambda: bmb.rotary_frequencies(rotary(**plan), **a))


@pytest.mark.parametrize("dims", [2, 4, 20, 64, 128, 256])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
def test_frequencies(dims, base):
    """Each scaling from its definition (pow is good to a step or two of 64 bits)."""
    def of(scaling, factor=1.0, **kw):
        p = rotary(head_size=dims, dims=dims)
        bmb.rotary_frequencies(p, base, scaling, factor, **kw)
        return list(p.freq)[:dims // 2]

    plain = [base ** (-2.0 * i / dims) for i in range(dims // 2)]
    assert of(bmb.ROTARY_UNSCALED) == pytest.approx(plain, rel=1e-15)
    assert of(bmb.ROTARY_LINEAR, 8.0) == pytest.approx([f / 8 for f in plain], rel=1e-15)
    wide = base * 8.0 ** (dims / (dims - 2.0)) if dims > 2 else base
    assert of(bmb.ROTARY_BASE, 8.0) == pytest.approx(
        [wide ** (-2.0 * i / dims) for i in range(dims // 2)], rel=1e-14)
    got = of(bmb.ROTARY_PARTS, 8.0, trained_len=4096, slow=1.0, fast=32.0)
    for f, p in zip(got, plain):
        turns = 4096 * p / (2 * math.pi)
        if turns >= 32:
            assert f == pytest.approx(p, rel=1e-15)
        elif turns <= 1:
            assert f == pytest.approx(p / 8, rel=1e-15)
        else:
            k = (turns - 1) / 31
            assert f == pytest.approx(k * p + (1 - k) * p / 8, rel=1e-13)
    # the longest wave of a base scaled so turns as far in the longer context as it did before
    if dims > 2:
        assert of(bmb.ROTARY_BASE, 8.0)[-1] * 8 == pytest.approx(plain[-1], rel=1e-13)


def test_struct_layouts(tmp_path):
    """The ctypes mirrors have the C headers' sizes and offsets."""
    structs = [("gemm.h", bmb.GemmI8), ("nn.h", bmb.RmsNorm), ("nn.h", bmb.RmsNormGrad),
               ("nn.h", bmb.Rotary)]
    src = ["#define __HIP_PLATFORM_AMD__", "#include <stdio.h>", "#include <stddef.h>",
           '#include "gemm.h"', '#include "nn.h"', "int main(void){"]
    want = []
    for _, s in structs:
        n = s.__name__
        src.append('printf("%%zu\\n", sizeof(%s));' % n)
        want.append(ctypes.sizeof(s))
        for f, _ in s._fields_:
            src.append('printf("%%zu\\n", offsetof(%s, %s));' % (n, f))
            want.append(getattr(s, f).offset)
    for name, value in (("BMB_I8", bmb.I8), ("BMB_ROTARY_PAIRS", bmb.ROTARY_PAIRS),
                        ("BMB_ROTARY_LINEAR", bmb.ROTARY_LINEAR),
                        ("BMB_ROTARY_BASE", bmb.ROTARY_BASE),
                        ("BMB_ROTARY_PARTS", bmb.ROTARY_PARTS)):
        src.append('printf("%%d\\n", %s);' % name)
        want.append(value)
    src += ["return 0;}"]
    c, exe = tmp_path / "layout.c", tmp_path / "layout"
    c.write_text("\n".join(src))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), "-I/opt/rocm/include",
                    str(c), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in out] == want
