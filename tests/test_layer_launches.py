"""What rms_norm_*, quantize_rows, gemm_i8 and rotary_* queue for their largest calls, on the host:
a small program loads the library and stands in for the HIP calls that launch a kernel, so nothing
runs and every pointer is a number. A dispatch holds fewer than 2^32 lanes: larger work has to
come in several."""
import os
import subprocess

import pytest

import bmb

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#define __HIP_PLATFORM_AMD__
#include <dlfcn.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include "gemm.h"
#include "nn.h"
static dim3 grid, block;
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t lds, hipStream_t stream) {
    grid = g, block = b;
    return 0;
}
hipError_t __hipPopCallConfiguration(dim3 *g, dim3 *b, size_t *lds, hipStream_t *stream) {
    *g = grid, *b = block, *lds = 0, *stream = 0;
    return 0;
}
hipError_t hipLaunchKernel(const void *f, dim3 g, dim3 b, void **args, size_t lds,
                           hipStream_t stream) {
    printf("launch %llu %u\n", 1ull * g.x * g.y * g.z, b.x);
    return 0;
}
hipError_t hipGetLastError(void) { return 0; }
hipError_t hipGetDevice(int *d) { *d = 0; return 0; }
hipError_t hipFuncSetAttribute(const void *f, hipFuncAttribute what, int value) { return 0; }
static void *at(long long n) { return (void *)(n << 56); }
int main(int argc, char **argv) {
    void *lib = dlopen(argv[1], RTLD_NOW);
    if (!lib) { fprintf(stderr, "%s\n", dlerror()); return 2; }
    const char *what = argv[2];
    long long n[8] = {0};
    for (int i = 3; i < argc; ++i) n[i - 3] = atoll(argv[i]);
    int rc = 2;
    if (!strcmp(what, "norm")) {  /* type, out_type, rows, C */
        int (*f)(const RmsNorm *, void *) = dlsym(lib, "rms_norm_forward");
        RmsNorm a = {n[2], n[3], n[0], n[1], 1e-5f, at(1), 0, 0, at(2), at(3), at(4), 0,
                     0, 0, 0, n[3]};
        rc = f(&a, 0);
    }
    if (!strcmp(what, "quantize")) {  /* type, rows, C */
        int (*f)(signed char *, long long, float *, const void *, long long, int, int, int,
                 void *) = dlsym(lib, "quantize_rows");
        rc = f(at(1), n[2], at(2), at(3), 0, n[0], n[1], n[2], 0);
    }
    if (!strcmp(what, "grad")) {  /* type, rows, C */
        int (*f)(const RmsNormGrad *, void *) = dlsym(lib, "rms_norm_backward");
        RmsNormGrad a = {n[1], n[2], n[0], at(1), at(2), 0, at(3), at(4), at(5), at(6),
                         0, 0, 0, n[2], at(7), ~0ull >> 20};
        rc = f(&a, 0);
    }
    if (!strcmp(what, "rotary")) {  /* type, tokens, heads, head size */
        int (*f)(const Rotary *, void *, long long, const void *, long long, int, int, int,
                 const int *, void *) = dlsym(lib, "rotary_forward");
        Rotary r = {n[3], n[3], BMB_ROTARY_HALF, 1.0f};
        rc = f(&r, at(1), n[2] * n[3], at(2), 0, n[0], n[1], n[2], at(3), 0);
    }
    if (!strcmp(what, "gemm")) {  /* type, M, N, K */
        int (*f)(const GemmI8 *, void *) = dlsym(lib, "gemm_i8");
        long long ld = (n[3] + 15) / 16 * 16;
        GemmI8 g = {n[1], n[2], n[3], n[0], at(1), at(2), at(3), at(4), 0, at(5), ld, ld, n[2],
                    at(6), ~0ull >> 20};
        rc = f(&g, 0);
    }
    printf("end %d\n", rc);
    return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    d = tmp_path_factory.mktemp("layer_launches")
    src, exe = d / "p.c", d / "p"
    src.write_text(PROGRAM)
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-rdynamic", "-I",
                    os.path.join(ROOT, "include"), "-I/opt/rocm/include", str(src), "-o", str(exe),
                    "-ldl"], check=True)
    return str(exe)


def launches(program, what, *args):
    """(workgroups, lanes of one) of each launch of a call that is accepted."""
    r = subprocess.run([program, bmb.LIB_PATH, what] + [str(a) for a in args],
                       capture_output=True, text=True, timeout=60)
    lines = r.stdout.split("\n")[:-1]
    assert r.returncode == 0 and lines[-1] == "end 0", (r.stdout, r.stderr)
    got = [tuple(int(x) for x in line.split()[1:]) for line in lines[:-1]]
    assert got and all(blocks * lanes < 1 << 32 for blocks, lanes in got), got
    return got


ROWS = [1, (1 << 24) + 5, (1 << 31) - 1]


@pytest.mark.parametrize("type", [bmb.F32, bmb.F16])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("C", [1, 768, 4096, 16384, 20000])
def test_rows(program, type, rows, C):
    each = 4 if C <= 1024 else 1  # rows of a workgroup
    for got in (launches(program, "norm", type, type, rows, C),
                launches(program, "norm", type, bmb.I8, rows, C),
                launches(program, "quantize", type, rows, C)):
        assert sum(blocks for blocks, _ in got) == -(-rows // each)


@pytest.mark.parametrize("type", [bmb.F32, bmb.F16])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("C", [1, 768, 4096, 16384, 20000])
def test_grad(program, type, rows, C):
    got = launches(program, "grad", type, rows, C)
    span = min(64, max(4, -(-rows // 512)))
    if C <= 16384:
        assert sum(blocks for blocks, _ in got[:-1]) == -(-rows // span)
    else:
        chunks = -(-C // (256 * (4 if type == bmb.F32 else 8)))
        assert sum(blocks for blocks, _ in got[:-1]) == chunks * -(-rows // span) + rows
    assert got[-1] == (-(-C // 16), 1024)


@pytest.mark.parametrize("type", [bmb.F32, bmb.BF16])
@pytest.mark.parametrize("tokens", ROWS)
@pytest.mark.parametrize("heads,hs", [(1, 2), (40, 128), (1000, 256)])
def test_rotary(program, type, tokens, heads, hs):
    got = launches(program, "rotary", type, tokens, heads, hs)
    assert sum(blocks * lanes for blocks, lanes in got) >= tokens


@pytest.mark.parametrize("M,N,K", [(1, 1, 0), (1, 1 << 20, 64), (1 << 17, 1 << 17, 128),
                                   (1 << 28, 1, 16), (1, 1 << 28, 16), (64, 64, 131071)])
def test_gemm(program, M, N, K):
    launches(program, "gemm", bmb.BF16, M, N, K)
