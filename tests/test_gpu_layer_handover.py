"""rms_norm_backward and gemm_i8 with workspaces of the library's, on busy streams: a workspace
passes from one stream's call to another's while work is queued on both, and the results are a lone
call's to the bit."""
import threading

import pytest
import torch

import bmb
from rows_util import U
from test_gpu_layer_streams import Calls, same

pytestmark = pytest.mark.gpu
TURNS = 3


def wants(calls):
    """What TURNS runs of each leave (dweight adds up), on the null stream."""
    got = []
    for c in calls:
        c.clear()
        for _ in range(TURNS):
            c.run(0)
        got.append(c.get())
    for c in calls:
        c.clear()
    return got


def occupy(stream, big):
    with torch.cuda.stream(stream):
        for _ in range(3):
            big.add_(1.0)


@pytest.mark.parametrize("streams", [2, 6])
def test_between_streams(gpu, streams):
    """Calls on several streams in turn, nothing waited for: each stream's first call is behind
    work of its own, so that a later call meets a workspace whose last user has not run."""
    calls = [Calls(20 + i, work=False) for i in range(streams)]
    expect = wants(calls)
    side = [torch.cuda.Stream() for _ in calls]
    big = [torch.zeros(1 << 27, device="cuda") for _ in calls]
    for late in range(2):
        for c in calls:
            c.clear()
        occupy(side[late], big[late])
        for _ in range(TURNS):
            for c, s in zip(calls, side):
                c.run(s.cuda_stream)
        for c, want in zip(calls, expect):
            same(c.get(), want)


def test_null_stream_and_another(gpu):
    """From the null stream to a side stream and back."""
    calls = [Calls(30 + i, work=False) for i in range(2)]
    expect = wants(calls)
    side = torch.cuda.Stream()
    big = torch.zeros(1 << 27, device="cuda")
    for first in (0, 1):
        for c in calls:
            c.clear()
        if first:
            occupy(side, big)
        for _ in range(TURNS):
            calls[0].run(0)
            calls[1].run(side.cuda_stream)
        for c, want in zip(calls, expect):
            same(c.get(), want)


def test_threads_with_streams(gpu):
    """Four host threads, a stream each."""
    calls = [Calls(40 + i, work=False) for i in range(4)]
    expect = wants(calls)
    side = [torch.cuda.Stream() for _ in calls]
    errors, barrier = [], threading.Barrier(len(calls))

    def go(c, s):
        try:
            barrier.wait()
            for _ in range(TURNS):
                c.run(s.cuda_stream)
            bmb.check("thread")
        except Exception as e:  # reported below
            errors.append(repr(e))

    threads = [threading.Thread(target=go, args=a) for a in zip(calls, side)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=60)
    assert not any(t.is_alive() for t in threads) and not errors, errors
    for c, want in zip(calls, expect):
        same(c.get(), want)


@pytest.mark.parametrize("work", [True, False])
def test_every_sum_adds_up(gpu, work):
    """dweight after n calls is n times one call's: the call's sum S is held in 64 bits, so the
    first result is off by u |S| and the k-th addition by u |k S|."""
    c = Calls(50, work)
    once = c.want()["dweight"].double()
    n = 4
    c.clear()
    for _ in range(n):
        c.run(0)
    got = c.get()["dweight"].double()
    assert (once != 0).all()
    off = (n + n * (n + 1) / 2) * 1.01 * U * once.abs()
    assert ((got - n * once).abs() <= off).all()
