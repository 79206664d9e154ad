"""What the generation entry points (paged_plan, paged_append, paged_attention,
logits_process) refuse, on the host, before anything is launched; and the
layout of their structs. No GPU: every pointer here is a number."""
import ctypes
import os
import subprocess

import pytest

import bmb

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # an address, never used


def plan(**kw):
    f = dict(requests=2, max_pages=4, pages=8, page_size=16, max_tokens=8, new_tokens=P, lens=P,
             lens_out=P + 64, state=P, state_out=P + 64, free_pages=P, block_table=P, slots=P,
             positions=P, rows=P, offsets=P)
    f.update(kw)
    return bmb.PagedPlan(**f)


def cache(**kw):
    f = dict(k=P, v=P, type=bmb.F32, pages=8, page_size=16, kv_heads=2, head_size=64,
             page_stride=2048, token_stride=128, head_stride=64)
    f.update(kw)
    return bmb.PagedCache(**f)


def batch(**kw):
    f = dict(requests=2, max_len=64, table_stride=4, heads=4, n_rows=2, type=bmb.F32, scale=1.0,
             q_stride=256, out_stride=256, block_table=P, lens=P)
    f.update(kw)
    return bmb.PagedBatch(**f)


def refused(capfd, what, f, *args):
    with pytest.raises(ValueError):
        f(*args)
    assert what in capfd.readouterr().err


BAD_PLANS = [(dict(requests=0), "requests"), (dict(requests=8193), "requests"),
             (dict(max_pages=0), "least"), (dict(pages=0), "least"), (dict(page_size=0), "least"),
             (dict(max_tokens=-1), "least"), (dict(pages=1 << 28), "2^31"),
             (dict(max_pages=1 << 28), "2^31"), (dict(lens_out=P + 4), "overlaps"),
             (dict(state_out=P - 4), "overlaps")]
BAD_PLANS += [({k: None}, "null") for k in ("new_tokens", "lens", "lens_out", "state", "state_out",
                                            "free_pages", "block_table", "slots", "positions",
                                            "rows", "offsets")]


@pytest.mark.parametrize("kw,why", BAD_PLANS)
def test_plan_refuses(capfd, kw, why):
    refused(capfd, why, bmb.paged_plan, plan(**kw))


def test_plan_refuses_none(capfd):
    refused(capfd, "no plan", bmb.paged_plan, None)


BAD_CACHES = [(dict(k=None), "no cache"), (dict(v=None), "no cache"), (dict(type=3), "type"),
              (dict(type=-1), "type"), (dict(pages=0), "empty"), (dict(page_size=0), "empty"),
              (dict(kv_heads=0), "empty"), (dict(head_size=48), "head size"),
              (dict(head_size=256), "head size"), (dict(pages=1 << 27), "2^31"),
              (dict(k=P + 8), "16 bytes"), (dict(v=P + 4), "16 bytes"),
              (dict(page_stride=2046), "16 bytes"), (dict(token_stride=130), "16 bytes"),
              (dict(head_stride=65), "16 bytes"),
              (dict(type=bmb.F16, token_stride=132), "16 bytes"),
              (dict(page_stride=-2048), "negative"),
              (dict(token_stride=1 << 26), "token_stride")]


@pytest.mark.parametrize("kw,why", BAD_CACHES)
def test_cache_is_refused(capfd, kw, why):
    c = cache(**kw)
    refused(capfd, why, bmb.paged_append, c, P, P, bmb.F32, 128, P, 4)
    refused(capfd, why, bmb.paged_attention, c, batch(), P, P, P)
    assert bmb.paged_attention_workspace(c, batch(max_len=64)) == 0


@pytest.mark.parametrize("kw,why", [(dict(type=7), "type"), (dict(type=bmb.F16), "own type"),
                                    (dict(tokens=-1), "negative"), (dict(k=None), "null"),
                                    (dict(v=None), "null"), (dict(slots=None), "null"),
                                    (dict(k=P + 2), "4 bytes"),
                                    (dict(tokens=(1 << 30)), "too many")])
def test_append_refuses(capfd, kw, why):
    a = dict(k=P, v=P, type=bmb.F32, row_stride=128, slots=P, tokens=4)
    a.update(kw)
    refused(capfd, why, bmb.paged_append, cache(), *a.values())


def test_append_refuses_odd_rows_of_16_bits(capfd):
    c = cache(type=bmb.BF16)
    refused(capfd, "4 bytes", bmb.paged_append, c, P, P, bmb.BF16, 129, P, 4)
    refused(capfd, "own type", bmb.paged_append, c, P, P, bmb.F16, 128, P, 4)


def test_nothing_to_append_is_no_launch():
    bmb.paged_append(cache(), None, None, bmb.F32, 128, None, 0)
    assert bmb.last_error() == 0


@pytest.mark.parametrize("kw,why", [(dict(requests=0), "least"), (dict(max_len=-1), "least"),
                                    (dict(heads=0), "least"), (dict(n_rows=0), "least"),
                                    (dict(heads=5), "multiple"), (dict(type=9), "type"),
                                    (dict(type=bmb.F16), "own type"),
                                    (dict(max_len=65), "table_stride"),
                                    (dict(table_stride=3), "table_stride"),
                                    (dict(requests=1 << 29), "too many"),
                                    (dict(max_len=(1 << 31) - 4096, table_stride=1 << 27), "4097"),
                                    (dict(out_stride=255), "overlap"),
                                    (dict(block_table=None), "null"), (dict(lens=None), "null")])
def test_attention_refuses(capfd, kw, why):
    refused(capfd, why, bmb.paged_attention, cache(), batch(**kw), P, P, P)


def test_attention_refuses_buffers(capfd):
    refused(capfd, "null", bmb.paged_attention, cache(), batch(), None, P, P)
    refused(capfd, "null", bmb.paged_attention, cache(), batch(), P, P, None)
    refused(capfd, "4 bytes", bmb.paged_attention, cache(), batch(), P + 2, P, P)
    refused(capfd, "no batch", bmb.paged_attention, cache(), None, P, P, P)
    c = cache(type=bmb.BF16)
    refused(capfd, "4 bytes", bmb.paged_attention, c, batch(type=bmb.BF16, q_stride=257), P, P, P)
    refused(capfd, "own type", bmb.paged_attention, c, batch(type=bmb.F16), P, P, P)


def test_attention_refuses_huge_caches_of_odd_pages(capfd):
    c = cache(pages=1 << 22, page_size=24, page_stride=1 << 13, token_stride=256)
    refused(capfd, "64 GiB", bmb.paged_attention, c, batch(table_stride=64), P, P, P)


@pytest.mark.parametrize("page_size,last,why", [(24, (1 << 36) - 16, "64 GiB"),
                                                (24, (1 << 36) - 32, "too small"),
                                                (32, 1 << 40, "too small")])
def test_attention_odd_pages_by_their_places(capfd, page_size, last, why):
    """Not the cache's size: where its last token starts, behind the first. (A
    workspace that is too small is refused behind that.)"""
    c = cache(pages=2, page_size=page_size, page_stride=last // 4 - (page_size - 1) * 128)
    b = batch(max_len=64000, table_stride=4000)
    b.work, b.work_bytes = P, 16
    refused(capfd, why, bmb.paged_attention, c, b, P, P, P)


def test_attention_refuses_small_workspaces(capfd):
    b = batch(max_len=64000, table_stride=4000)
    need = bmb.paged_attention_workspace(cache(), b)
    assert need > 0
    b.work, b.work_bytes = P, need - 1
    refused(capfd, "too small", bmb.paged_attention, cache(), b, P, P, P)
    b.work, b.work_bytes = P + 4, need
    refused(capfd, "16 bytes", bmb.paged_attention, cache(), b, P, P, P)


@pytest.mark.parametrize("kw", [dict(k=None, v=None), dict(k=None), dict(v=None),
                                dict(k=P + 8), dict(v=P + 4)])
def test_workspace_looks_at_no_pointer(kw):
    """Its bytes are known before the cache and the batch have their buffers."""
    b = batch(max_len=64000, table_stride=4000)
    need = bmb.paged_attention_workspace(cache(), b)
    b.block_table = b.lens = None
    assert need > 0 and bmb.paged_attention_workspace(cache(**kw), b) == need
    assert bmb.paged_attention_workspace(cache(head_size=48, **kw), b) == 0


def test_workspace_of_nothing():
    assert bmb.paged_attention_workspace(None, batch()) == 0
    assert bmb.paged_attention_workspace(cache(), None) == 0


def rules(**kw):
    f = dict(tokens=P, token_stride=8, lens=P, repetition=P, bias_offsets=P, bias_ids=P,
             bias_values=P, biases=2, mask=P, masks=4, mask_stride=4)
    f.update(kw)
    return bmb.LogitsRules(**f)


@pytest.mark.parametrize("kw,why", [(dict(lens=None), "lens"),
                                    (dict(token_stride=-1), "token_stride"),
                                    (dict(tokens=None), "penalties"),
                                    (dict(bias_ids=None), "bias"), (dict(bias_values=None), "bias"),
                                    (dict(biases=-1), "bias"), (dict(mask_stride=3), "V bits"),
                                    (dict(masks=0), "V bits"), (dict(masks=3), "fewer masks")])
def test_logits_refuses_rules(capfd, kw, why):
    refused(capfd, why, bmb.logits_process, P, P, bmb.F32, 4, 100, 104, rules(**kw))


@pytest.mark.parametrize("args,why", [((P, P, 3, 4, 100, 104), "type"),
                                      ((P, P, 0, -1, 100, 104), "least"),
                                      ((P, P, 0, 4, 0, 104), "least"),
                                      ((P, P, 0, 4, 100, 99), "least"),
                                      ((None, P, 0, 4, 100, 104), "null"),
                                      ((P, None, 0, 4, 100, 104), "null"),
                                      ((P + 2, P, 0, 4, 100, 104), "element"),
                                      ((P + 1, P, 1, 4, 100, 104), "element"),
                                      ((P + 16, P, 0, 4, 100, 104), "overlaps"),
                                      ((P, P + 400, 0, 2, 100, 104), "overlaps"),
                                      ((P, P, 0, 1 << 30, 1 << 14, 1 << 14), "too many")])
def test_logits_refuses(capfd, args, why):
    refused(capfd, why, bmb.logits_process, *args, rules(masks=1 << 30, mask_stride=1 << 10))


def test_logits_refuses_no_rules(capfd):
    refused(capfd, "null", bmb.logits_process, P, P, 0, 4, 100, 104, None)


def test_no_rows_is_no_launch():
    bmb.logits_process(P, P, bmb.F32, 0, 100, 104, rules())
    assert bmb.last_error() == 0


def test_struct_layouts_match_headers(tmp_path):
    """The ctypes mirrors have the C headers' sizes and offsets."""
    structs = [bmb.PagedCache, bmb.PagedPlan, bmb.PagedBatch, bmb.LogitsRules]
    src = ["#include <stdio.h>", "#include <stddef.h>", '#include "flash.h"', '#include "nn.h"',
           "int main(void){"]
    want = []
    for s in structs:
        src.append('printf("%%zu\\n", sizeof(%s));' % s.__name__)
        want.append(ctypes.sizeof(s))
        for f in s._fields_:
            src.append('printf("%%zu\\n", offsetof(%s, %s));' % (s.__name__, f[0]))
            want.append(getattr(s, f[0]).offset)
    src.append("return 0;}")
    c, exe = tmp_path / "layout.c", tmp_path / "layout"
    c.write_text("\n".join(src))
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"),
                    str(c), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    assert got == want


def test_headers_meet_the_runtime_header(tmp_path):
    """flash.h and nn.h name the stream without including the HIP runtime; a
    C++ caller that does passes its hipStream_t."""
    cpp = tmp_path / "caller.cpp"
    cpp.write_text('#include "flash.h"\n#include "nn.h"\n#include <hip/hip_runtime_api.h>\n'
                   "int f(hipStream_t s) { return paged_plan(nullptr, s) + "
                   "logits_process(nullptr, nullptr, 0, 0, 0, 0, nullptr, s); }\n")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-D__HIP_PLATFORM_AMD__", "-I",
                    os.path.join(ROOT, "include"), "-I/opt/rocm/include", "-c", str(cpp), "-o",
                    str(tmp_path / "caller.o")], check=True)
