"""What the generation entry points queue for their largest calls, on the host:
a small program loads the library and stands in for the HIP calls that launch a
kernel, so nothing runs and every pointer is a number. A dispatch holds fewer
than 2^32 lanes: larger work has to come in several."""
import os
import subprocess

import pytest

import bmb

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <dlfcn.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include "flash.h"
#include "nn.h"
typedef struct { unsigned x, y, z; } dim3;
static dim3 grid, block;
int __hipPushCallConfiguration(dim3 g, dim3 b, size_t lds, void *stream) {
    grid = g, block = b;
    return 0;
}
int __hipPopCallConfiguration(dim3 *g, dim3 *b, size_t *lds, void **stream) {
    *g = grid, *b = block, *lds = 0, *stream = 0;
    return 0;
}
int hipLaunchKernel(const void *f, dim3 g, dim3 b, void **args, size_t lds, void *stream) {
    printf("launch %u %u\n", g.x * g.y * g.z, b.x);
    return 0;
}
int hipGetLastError(void) { return 0; }
int hipGetDevice(int *d) { *d = 0; return 0; }
int hipFuncSetAttribute(const void *f, int what, int value) { return 0; }
static void *at(long long n) { return (void *)(n << 20); }
int main(int argc, char **argv) {
    void *lib = dlopen(argv[1], RTLD_NOW);
    if (!lib) { fprintf(stderr, "%s\n", dlerror()); return 2; }
    const char *what = argv[2];
    long long n[8] = {0};
    for (int i = 3; i < argc; ++i) n[i - 3] = atoll(argv[i]);
    int rc = 2;
    if (!strcmp(what, "logits")) {  /* type, rows, V */
        int (*f)(void *, const void *, int, int, int, long long, const LogitsRules *, void *) =
            dlsym(lib, "logits_process");
        LogitsRules r = {0};
        rc = f(at(1), at(1), n[0], n[1], n[2], n[2], &r, 0);
    }
    if (!strcmp(what, "append")) {  /* type, cache's type, kv, hs, tokens */
        int (*f)(const PagedCache *, const void *, const void *, int, long long, const int *, int,
                 void *) = dlsym(lib, "paged_append");
        PagedCache c = {at(1), at(2), n[1], 8, 16, n[2], n[3], 16 * n[2] * n[3], n[2] * n[3], n[3]};
        rc = f(&c, at(3), at(4), n[0], 0, at(5), n[4], 0);
    }
    if (!strcmp(what, "attend")) {  /* type, cache's type, hs, heads, kv, requests, max_len */
        int (*f)(const PagedCache *, const PagedBatch *, void *, float *, const void *, void *) =
            dlsym(lib, "paged_attention");
        PagedCache c = {at(1), at(2), n[1], 1, 1 << 24, n[4], n[2], 0, n[2] * n[4], n[2]};
        PagedBatch b = {n[5], n[6], 1, n[3], n[5], n[0], 1.0f, 0, n[2] * n[3]};
        b.block_table = b.lens = at(3);
        b.work = at(4), b.work_bytes = ~0ull;
        rc = f(&c, &b, at(5), 0, at(6), 0);
    }
    printf("end %d\n", rc);
    return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    d = tmp_path_factory.mktemp("launches")
    src, exe = d / "p.c", d / "p"
    src.write_text(PROGRAM)
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-rdynamic", "-I",
                    os.path.join(ROOT, "include"), str(src), "-o", str(exe), "-ldl"], check=True)
    return str(exe)


def launches(program, what, *args):
    """(workgroups, lanes of one) of each launch of a call that is accepted."""
    r = subprocess.run([program, bmb.LIB_PATH, what] + [str(a) for a in args],
                       capture_output=True, text=True, timeout=60)
    lines = r.stdout.split("\n")[:-1]
    assert r.returncode == 0 and lines[-1] == "end 0", (r.stdout, r.stderr)
    return [tuple(int(x) for x in line.split()[1:]) for line in lines[:-1]]


def covered(got, workgroups):
    assert all(blocks * lanes < 1 << 32 for blocks, lanes in got), got
    assert sum(blocks for blocks, _ in got) == workgroups, got


@pytest.mark.parametrize("type,ids", [(bmb.F32, 2048), (bmb.F16, 2048), (bmb.BF16, 2048)])
@pytest.mark.parametrize("rows,V", [(4, 50257), ((1 << 24) - 1, 65), (1 << 24, 65),
                                    ((1 << 24) + 5, 65), (1 << 26, 4096), ((1 << 31) - 1, 1)])
def test_logits(program, type, ids, rows, V):
    few = rows * V < 512 * ids and type == bmb.F32
    chunks = -(-V // (ids // 2 if few else ids))
    covered(launches(program, "logits", type, rows, V), rows * chunks)


@pytest.mark.parametrize("type,cache", [(bmb.F32, bmb.F32), (bmb.F32, bmb.F16),
                                        (bmb.F32, bmb.BF16), (bmb.F16, bmb.F16)])
@pytest.mark.parametrize("kv,hs,tokens", [(1, 32, 1), (12, 64, 32), (8, 128, (1 << 25) - 1),
                                          (8, 128, 1 << 25), (1, 64, (1 << 29) + 9),
                                          (3, 32, (1 << 29) + 1), (1, 128, (1 << 31) - 1)])
def test_append(program, type, cache, kv, hs, tokens):
    covered(launches(program, "append", type, cache, kv, hs, tokens),
            -(-tokens * kv * hs // 8 // 256))


@pytest.mark.parametrize("type,cache", [(bmb.F32, bmb.F32), (bmb.F32, bmb.BF16),
                                        (bmb.F16, bmb.F16)])
@pytest.mark.parametrize("heads,kv", [(32, 32), (64, 16), (66, 2), (256, 8)])
@pytest.mark.parametrize("requests,split", [(3, False), (3, True), ((1 << 18) + 1, False),
                                            (1 << 19, False), ((1 << 19) + 9, False),
                                            ((1 << 23) + 1, False)])
def test_attention(program, type, cache, heads, kv, requests, split):
    if heads > 64 and requests > 1 << 20:
        requests = 1 << 22
    tiles = -(-heads // kv // (32 if type != bmb.F32 and heads // kv > 16 else 16))
    blocks = -(-(requests + split * (2048 // (kv * tiles))) // 8) * 8 * kv * tiles
    got = launches(program, "attend", type, cache, 32, heads, kv, requests,
                   1 << 20 if split else 3)
    covered(got, blocks + split * requests * heads)


@pytest.mark.parametrize("type,cache", [(bmb.F32, bmb.F32), (bmb.F16, bmb.F16)])
@pytest.mark.parametrize("requests", [(1 << 11) - 1, 1 << 11, (1 << 11) + 1])
def test_attention_joins(program, type, cache, requests):
    """Split sequences: as many joins as a dispatch has lanes for, and more."""
    heads, kv, max_len = 1 << 13, 256, 1 << 23
    tiles = 1 if type == bmb.F16 else 2
    blocks = -(-(requests + 2048 // (kv * tiles)) // 8) * 8 * kv * tiles
    covered(launches(program, "attend", type, cache, 32, heads, kv, requests, max_len),
            blocks + requests * heads)
