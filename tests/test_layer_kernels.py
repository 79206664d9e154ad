"""Every kernel that the library holds for the operators around the paged cache is one that some
call reaches. On the host: a small program loads the library, notes the kernels that it registers,
and stands in for the HIP calls that launch them, so nothing runs and every pointer is a number."""
import os
import subprocess

import pytest

import bmb
from test_layer_launches import ROOT

PROGRAM = r"""
#define __HIP_PLATFORM_AMD__
#include <dlfcn.h>
#include <stdio.h>
#include <string.h>
#include "gemm.h"
#include "nn.h"
static struct { const void *host; const char *name; } kernels[4096];
static int count;
void __hipRegisterFunction(void **modules, const void *host, char *f, const char *name,
                           unsigned limit, void *tid, void *bid, void *block, void *grid,
                           int *wave) {
    kernels[count].host = host;
    kernels[count++].name = name;
}
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t lds, hipStream_t stream) { return 0; }
hipError_t __hipPopCallConfiguration(dim3 *g, dim3 *b, size_t *lds, hipStream_t *stream) {
    *g = *b = (dim3){1, 1, 1}, *lds = 0, *stream = 0;
    return 0;
}
hipError_t hipLaunchKernel(const void *f, dim3 g, dim3 b, void **args, size_t lds,
                           hipStream_t stream) {
    for (int i = 0; i < count; ++i)
        if (kernels[i].host == f) printf("launched %s\n", kernels[i].name);
    return 0;
}
hipError_t hipGetLastError(void) { return 0; }
hipError_t hipGetDevice(int *d) { *d = 0; return 0; }
hipError_t hipFuncSetAttribute(const void *f, hipFuncAttribute what, int value) { return 0; }
static void *at(long long n) { return (void *)(n << 56); }
int main(int argc, char **argv) {
    void *lib = dlopen(argv[1], RTLD_NOW);
    if (!lib) { fprintf(stderr, "%s\n", dlerror()); return 2; }
    int (*norm)(const RmsNorm *, void *) = dlsym(lib, "rms_norm_forward");
    int (*grad)(const RmsNormGrad *, void *) = dlsym(lib, "rms_norm_backward");
    int (*rows8)(signed char *, long long, float *, const void *, long long, int, int, int,
                 void *) = dlsym(lib, "quantize_rows");
    int (*turn)(const Rotary *, void *, long long, const void *, long long, int, int, int,
                const int *, void *) = dlsym(lib, "rotary_forward");
    int (*gemm)(const GemmI8 *, void *) = dlsym(lib, "gemm_i8");
    for (int i = 0; i < count; ++i) printf("registered %s\n", kernels[i].name);
    char what[16];
    long long n[5];
    while (scanf("%15s %lld %lld %lld %lld %lld", what, n, n + 1, n + 2, n + 3, n + 4) == 6) {
        int rc = 2;
        if (!strcmp(what, "rows")) {  /* type, rows, C */
            RmsNorm a = {n[1], n[2], n[0], n[0], 1e-5f, at(1), 0, 0, at(2), at(3), at(4), 0,
                         0, 0, 0, n[2]};
            rc = norm(&a, 0);
            a.out_type = BMB_I8;
            rc |= norm(&a, 0);
            rc |= rows8(at(1), n[2], at(2), at(3), 0, n[0], n[1], n[2], 0);
            RmsNormGrad g = {n[1], n[2], n[0], at(1), at(2), 0, at(3), at(4), at(5), at(6),
                             0, 0, 0, n[2], at(7), ~0ull >> 20};
            rc |= grad(&g, 0);
        }
        if (!strcmp(what, "turn")) {  /* type, layout, heads, head size, dims */
            Rotary r = {n[3], n[4], n[1], 1.0f};
            rc = turn(&r, at(1), n[2] * n[3], at(2), 0, n[0], 7, n[2], at(3), 0);
        }
        if (!strcmp(what, "gemm")) {  /* type, M, N, K */
            long long ld = (n[3] + 15) / 16 * 16;
            GemmI8 g = {n[1], n[2], n[3], n[0], at(1), at(2), at(3), at(4), 0, at(5), ld, ld, n[2],
                        at(6), ~0ull >> 20};
            rc = gemm(&g, 0);
        }
        if (rc) { fprintf(stderr, "%s refused\n", what); return 3; }
    }
    return 0;
}
"""

TYPES = (bmb.F32, bmb.F16, bmb.BF16)


def calls():
    """Sizes on both sides of every limit, and far from them."""
    for t in TYPES:
        for C in [1, 64, 256, 257, 512, 513, 768, 1024, 1025, 2048, 2049, 4096, 4097, 6144, 6145,
                  8192, 8193, 12288, 12289, 16384, 16385, 1 << 20]:
            yield "rows", t, 5, C, 0, 0
        for layout in (bmb.ROTARY_HALF, bmb.ROTARY_PAIRS):
            for hs, dims in [(2, 2), (4, 4), (8, 8), (16, 16), (6, 6), (12, 12), (24, 24),
                             (64, 64), (64, 32), (80, 20), (127, 126), (256, 256)]:
                yield "turn", t, layout, 3, hs, dims
        for M in (1, 2, 4, 5, 16, 17, 32, 33, 64, 65, 128, 300, 512, 1024, 2048, 4096, 8192):
            for N in (1, 64, 768, 2304, 4096, 4097, 8192, 16384, 50257, 1 << 20):
                for K in (16, 768, 4096, 4608, 8192, 8193, 16384):
                    yield "gemm", t, M, N, K, 0


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """(names that are registered, names that are launched)."""
    d = tmp_path_factory.mktemp("layer_kernels")
    src, exe = d / "p.c", d / "p"
    src.write_text(PROGRAM)
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-rdynamic", "-I",
                    os.path.join(ROOT, "include"), "-I/opt/rocm/include", str(src), "-o", str(exe),
                    "-ldl"], check=True)
    lines = "\n".join(" ".join(map(str, c)) for c in calls())
    r = subprocess.run([str(exe), bmb.LIB_PATH], input=lines, capture_output=True, text=True,
                       timeout=120)
    assert r.returncode == 0, r.stderr
    got = [line.split() for line in r.stdout.split("\n")[:-1]]
    return [{name for what, name in got if what == w} for w in ("registered", "launched")]


@pytest.mark.parametrize("family", ["i8_kernel", "i8_few_kernel", "i8_join_kernel", "rows_kernel",
                                    "wide_rows_kernel", "grad_kernel", "wide_grad_kernel",
                                    "wide_sums_kernel", "join_sums_kernel", "rotary_kernel"])
def test_reached(kernels, family):
    mangled = "_GLOBAL__N_1%d%s" % (len(family), family)
    registered, launched = ({n for n in names if mangled in n} for names in kernels)
    assert registered and launched <= registered
    assert not registered - launched, sorted(registered - launched)
