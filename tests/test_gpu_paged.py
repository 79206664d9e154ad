"""The paged key-value cache (include/flash.h) on the GPU: paged_plan,
paged_append and paged_attention against exact host computations, and a run of
them together against the whole-sequence attention.

Bars: paged_plan's whole numbers are equal; paged_append's elements are the
rounded inputs, bit for bit; paged_attention is within the rounding bound that
paged_util.Problem.exact derives for its sizes and types."""
import math
import threading

import numpy as np
import pytest
import torch

import bmb
import oracle as O
from paged_util import DTYPES, U32, Pool, Problem, cache_struct, ints, pages_of, plan_exact

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]
EDGES = [0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 256]


# ------------------------------------------------------------------- plan
def test_plan_of_many_tokens(gpu):
    """More tokens than the workgroups have threads, long prompts beside single
    tokens; on a side stream."""
    r = np.random.default_rng(5)
    lens = r.integers(0, 3000, 40)
    lens[::4] = 0
    pool = Pool(lens, 32, width=pages_of(45000, 32), free=14000, seed=6)
    side = torch.cuda.Stream()
    for in_place in (False, True):
        new = np.ones(40, np.int64)
        new[::4] = r.integers(1, 40000, 10)
        new[3] = -1
        torch.cuda.synchronize()
        pool.step(new, int(new[new > 0].sum()) + 5, in_place, side.cuda_stream)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("R,page,prompt", [(1, 16, 1), (1, 1, 3), (3, 5, 40), (64, 16, 1),
                                           (65, 16, 300), (1024, 8, 7), (1500, 3, 5),
                                           (8192, 16, 2)])
def test_plan_steps(gpu, R, page, prompt, in_place):
    """Several steps of one pool: prompts, single tokens, idle and ended
    requests, more than fit."""
    r = np.random.default_rng(R + page)
    lens = r.integers(0, 50, R)
    pool = Pool(lens, page, width=pages_of(80, page), free=2 * R + 8, seed=R)
    for step in range(5):
        new = r.integers(1, prompt + 1, R)
        new[r.random(R) < 0.2] = 0
        new[r.random(R) < 0.15] = -1
        total = int(new[new > 0].sum())
        cap = max(0, total if step % 2 == 0 else total * 2 // 3)
        print("plan R=%d page=%d step %d: %d tokens, room %d" % (R, page, step, total, cap),
              flush=True)
        pool.step(new, cap, in_place)


def test_plan_grants_in_order(gpu):
    """No page left for one request: later ones that need none still go; past
    max_tokens nothing more goes; a request past its table never counts."""
    # held 4 of 4 places each; the pool has two free pages
    pool = Pool([4, 4, 4, 3, 3, 8], 4, width=2, free=2, seed=1)
    pool.step([1, 5, 1, 1, 1, 1], 8)      # 1: its table ends; 5: too; 0, 2 take the pages
    assert pool.lens.tolist() == [5, 4, 5, 4, 4, 8]
    pool.step([1, 1, 1, 1, 0, -1], 8)     # no page for 1 and 3; 5 ends
    assert pool.lens.tolist() == [6, 4, 6, 4, 4, 0] and pool.state[1] == 2
    pool.step([1, 1, 1, 1, 1, 0], 2)      # two tokens' room
    assert pool.lens.tolist() == [7, 5, 6, 4, 4, 0]
    pool.step([0, 0, 0, 0, 0, 0], 0)
    pool.step([-1] * 6, 4)
    assert pool.lens.tolist() == [0] * 6 and pool.state[1] == pool.pages


def test_plan_room_is_passed_across_scan_rounds(gpu):
    """A request past the room for tokens stops every later one, also those
    that a later round of the scan reads."""
    new = np.ones(3000, np.int64)
    new[1000] = 64
    pool = Pool(np.zeros(3000, np.int64), 64, width=1, free=3000, seed=3)
    pool.step(new, 1020, in_place=False)
    assert pool.lens[:1000].sum() == 1000 and pool.lens[1000:].sum() == 0


def test_plan_reads_bad_device_values_safely(gpu):
    """Lengths, states and table entries outside their ranges: no place outside
    the buffers is touched, and slots of unknown pages are -1."""
    pool = Pool([5, 6, 7], 4, width=3, free=3, seed=2)
    d = pool.d
    table = torch.tensor([[9999, -1, 0], [2, 1 << 30, 0], [0, 1, 2]], dtype=torch.int32).cuda()
    lens = ints([6, 1 << 30, -5])
    state, ring = ints([-1, 1 << 30]), d["ring"].clone()
    new = ints([1, -1, 1])
    guard = torch.full((64,), 4242, device="cuda", dtype=torch.int32)
    outs = {k: guard.clone() for k in ("slots", "positions", "rows", "offsets", "lens_out",
                                       "state_out")}
    plan = bmb.PagedPlan(requests=3, max_pages=3, pages=pool.pages, page_size=4, max_tokens=8,
                         new_tokens=new.data_ptr(), lens=lens.data_ptr(), state=state.data_ptr(),
                         free_pages=ring.data_ptr(), block_table=table.data_ptr(),
                         **{k: v.data_ptr() for k, v in outs.items()})
    bmb.paged_plan(plan)
    torch.cuda.synchronize()
    bmb.check("paged_plan")
    assert outs["slots"][0].item() == -1            # page -1 of request 0
    assert (outs["slots"][8:] == 4242).all() and (outs["rows"][3:] == 4242).all()
    assert outs["lens_out"][:3].tolist() == [7, 0, 1]
    assert 0 <= outs["state_out"][1].item() <= pool.pages


def test_plan_captured(gpu):
    """A captured step, in place, replayed: each replay is the next step."""
    pool = Pool([3] * 70, 4, width=8, free=300, seed=5)
    new = [1] * 60 + [0] * 5 + [7] * 5
    pool.step(new, 128)
    d_new = ints(new)
    bufs = {k: torch.zeros(n, device="cuda", dtype=torch.int32)
            for k, n in (("slots", 2048), ("positions", 2048), ("rows", 70), ("offsets", 71))}
    plan = bmb.PagedPlan(requests=70, max_pages=8, pages=pool.pages, page_size=4, max_tokens=2048,
                         new_tokens=d_new.data_ptr(), lens=pool.d["lens"].data_ptr(),
                         lens_out=pool.d["lens"].data_ptr(), state=pool.d["state"].data_ptr(),
                         state_out=pool.d["state"].data_ptr(),
                         free_pages=pool.d["ring"].data_ptr(),
                         block_table=pool.d["table"].data_ptr(),
                         **{k: t.data_ptr() for k, t in bufs.items()})
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        bmb.paged_plan(plan, side.cuda_stream)
    for i in range(3):
        want = plan_exact(pool.table, pool.lens, np.array(new), pool.ring, pool.state, 4, 2048)
        graph.replay()
        torch.cuda.synchronize()
        for name, t in (("slots", bufs["slots"]), ("positions", bufs["positions"]),
                        ("rows", bufs["rows"]), ("offsets", bufs["offsets"]),
                        ("block_table", pool.d["table"]), ("lens_out", pool.d["lens"]),
                        ("state_out", pool.d["state"]), ("free_pages", pool.d["ring"])):
            assert np.array_equal(t.cpu().numpy(), want[name]), (i, name)
        pool.table, pool.ring = want["block_table"], want["free_pages"]
        pool.lens, pool.state = want["lens_out"], want["state_out"]


# ----------------------------------------------------------------- append
@pytest.mark.parametrize("type,cache", TYPES)
@pytest.mark.parametrize("tokens,kv,hs,page,layout",
                         [(1, 12, 64, 16, "token"), (37, 1, 32, 5, "head"),
                          (300, 3, 128, 24, "head"), (257, 7, 64, 1, "token")])
def test_append(gpu, type, cache, tokens, kv, hs, page, layout):
    g = torch.Generator().manual_seed(tokens)
    pages = pages_of(tokens, page) + 2
    width = kv * hs
    rows = (torch.randn(tokens, 3 * width + 2, generator=g) * 3).to(DTYPES[type])
    rows[0, width] = math.inf
    rows[-1, 2 * width] = math.nan
    shape = (pages, page, kv, hs) if layout == "token" else (pages, kv, page, hs)
    k0, v0 = (torch.randn(shape, generator=g).to(DTYPES[cache]) for _ in range(2))
    slots = torch.randperm(pages * page, generator=g)[:tokens].to(torch.int32)
    if tokens > 3:
        slots[1], slots[2], slots[3] = -1, pages * page, 1 << 30
    k, v, d_rows, d_slots = k0.cuda(), v0.cuda(), rows.cuda(), slots.cuda()
    c = cache_struct(k, v, layout, page, kv, hs, cache)
    item = d_rows.element_size()
    bmb.paged_append(c, d_rows.data_ptr() + width * item, d_rows.data_ptr() + 2 * width * item,
                     bmb.ELEMENT_TYPES[type], 3 * width + 2, d_slots.data_ptr(), tokens)
    torch.cuda.synchronize()
    bmb.check("paged_append")
    for got, want, i in ((k, k0, 1), (v, v0, 2)):
        want = want if layout == "token" else want.permute(0, 2, 1, 3).contiguous()
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < pages * page:
                want[s // page, s % page] = (rows[t, i * width:(i + 1) * width].view(kv, hs)
                                             .to(DTYPES[cache]))
        got = got.cpu() if layout == "token" else got.cpu().permute(0, 2, 1, 3)
        same = (got == want) | (torch.isnan(got) & torch.isnan(want))
        assert same.all()


def test_append_tokens_of_several_launches(gpu):
    """More elements than one dispatch has lanes for: the tokens with a slot, at
    both ends and around where a launch ends, arrive; nothing else is written."""
    kv, hs, page, tokens = 8, 128, 4, (1 << 25) + 3
    ends = ((1 << 32) - 1) // 256 // 8 * 8 * 256 // (kv * hs // 8)
    live = [0, 1, ends - 1, ends, ends + 1, (1 << 25) - 1, 1 << 25, tokens - 1]
    # rows one element apart: row t is elements t..t+1023
    rows = torch.randn(2, tokens + kv * hs, device="cuda")
    slots = torch.full((tokens,), -1, dtype=torch.int32, device="cuda")
    at = [2 * i + 1 for i in range(len(live))]
    slots[torch.tensor(live, device="cuda")] = ints(at)
    k = torch.full((5, page, kv, hs), 768.0, device="cuda")
    v = k.clone()
    want_k, want_v = k.clone().view(-1, kv * hs), v.clone().view(-1, kv * hs)
    for t, s in zip(live, at):
        want_k[s], want_v[s] = rows[0, t:t + kv * hs], rows[1, t:t + kv * hs]
    bmb.paged_append(cache_struct(k, v, "token", page, kv, hs, "f32"), rows[0].data_ptr(),
                     rows[1].data_ptr(), bmb.F32, 1, slots.data_ptr(), tokens)
    torch.cuda.synchronize()
    bmb.check("paged_append")
    assert torch.equal(k.view(-1, kv * hs), want_k) and torch.equal(v.view(-1, kv * hs), want_v)


# -------------------------------------------------------------- attention
@pytest.mark.parametrize("type,cache", TYPES)
@pytest.mark.parametrize("hs", [32, 64, 128])
@pytest.mark.parametrize("heads,kv,page,layout", [(3, 3, 16, "token"), (8, 2, 16, "head"),
                                                  (5, 1, 7, "token"), (34, 2, 64, "head"),
                                                  (2, 2, 1, "head"), (66, 2, 32, "token")])
def test_attention_edges(gpu, type, cache, hs, heads, kv, page, layout):
    print("attention edges", type, cache, hs, heads, kv, page, flush=True)
    p = Problem(EDGES, heads, kv, hs, type, cache, page, layout, seed=hs + heads).device()
    p.run()
    p.check()


@pytest.mark.parametrize("type,cache", TYPES)
@pytest.mark.parametrize("hs", [32, 64, 128])
@pytest.mark.parametrize("lens,heads,kv,page", [([4500], 12, 12, 16), ([257, 0, 1, 2500], 8, 2, 24),
                                                ([3000, 2], 20, 1, 32), ([2600, 129], 3, 1, 48),
                                                ([2500, 700], 40, 1, 10),
                                                ([300] * 70 + [0, 1, 5000], 2, 2, 16),
                                                ([40] * 190 + [9000], 2, 2, 8)])
def test_attention_split(gpu, type, cache, hs, lens, heads, kv, page):
    print("attention split", type, cache, hs, lens[:4], heads, kv, page, flush=True)
    p = Problem(lens, heads, kv, hs, type, cache, page, "head", seed=hs).device()
    assert p.workspace() > 0
    p.run()
    p.check()


def large_batch(lens, heads, kv, hs, type, cache, page, max_len, seed):
    """A batch made on the device, run once with leased scratch, and checked for
    its first and last live requests and heads: Problem.exact's bound, with what
    flash.h allows a probability's two 16-bit numbers to lose."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    held = [pages_of(n, page) for n in lens]
    pages, width = sum(held) + 1, pages_of(max_len, page)
    order = torch.randperm(pages, device="cuda", generator=g)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    k = torch.full((pages, page, kv, hs), math.nan, device="cuda", dtype=DTYPES[cache])
    v, at = torch.full_like(k, math.inf), 0
    for r, n in enumerate(lens):
        table[r, :held[r]] = order[at:at + held[r]]
        at += held[r]
        t = torch.arange(n, device="cuda")
        for half in (k, v):
            half[table[r].long()[t // page], t % page] = torch.empty(
                n, kv, hs, device="cuda", dtype=half.dtype).normal_(generator=g)
    R, W, G = len(lens), heads * hs, heads // kv
    q = torch.empty(R, W, device="cuda", dtype=DTYPES[type]).normal_(generator=g)
    out, lse = torch.full_like(q, 768.0), torch.full((R, heads), 768.0, device="cuda")
    d_lens, scale = ints(lens), 1 / math.sqrt(hs)
    batch = bmb.PagedBatch(requests=R, max_len=max_len, table_stride=width, heads=heads, n_rows=R,
                           type=bmb.ELEMENT_TYPES[type], scale=scale, q_stride=W, out_stride=W,
                           block_table=table.data_ptr(), lens=d_lens.data_ptr())
    handle = cache_struct(k, v, "token", page, kv, hs, cache)
    bmb.paged_attention(handle, batch, out.data_ptr(), lse.data_ptr(), q.data_ptr())
    torch.cuda.synchronize()
    bmb.check("paged_attention")
    half_step = torch.finfo(DTYPES[type]).eps / 2
    lost, floor = dict(f32=(0.0, 0.0), f16=(2.0 ** -23, 2.0 ** -40), bf16=(2.0 ** -17, 0.0))[type]
    live = [r for r, n in enumerate(lens) if n]
    assert torch.isfinite(out[live].float()).all() and torch.isfinite(lse[live]).all()
    for r, n in enumerate(lens):
        if n == 0:
            assert (out[r] == 0).all() and (lse[r] == -math.inf).all()
    for r in live[:2] + live[-2:]:
        n, t = lens[r], torch.arange(lens[r], device="cuda")
        for h in sorted({0, kv - 1}):
            keys, values = (x[table[r].long()[t // page], t % page, h].double() for x in (k, v))
            qh = q[r].view(kv, G, hs)[h].double()
            x = qh @ keys.t() * scale
            mag = (qh.abs() @ keys.abs().t()).amax(1) * scale
            z = torch.logsumexp(x, 1)
            p = torch.exp(x - z[:, None])
            want = p @ values
            ds = 4 * (math.sqrt(hs) + 1) * U32 * mag + 4 * U32 * x.abs().amax(1)
            eps = 2 * ds + (4 * math.sqrt(n) + 16) * U32 + lost
            bound = (eps[:, None] * (p @ values.abs()) + floor * values.abs().sum(0)
                     + half_step * want.abs() + (2.0 ** -25 if type == "f16" else 0.0))
            got = out[r].view(kv, G, hs)[h].double()
            assert ((got - want).abs() <= bound).all(), (r, h, ((got - want).abs() / bound).max())
            zb = ds + (4 * math.sqrt(n) + 16) * U32 + 4 * U32 * z.abs()
            assert ((lse[r].view(kv, G)[h].double() - z).abs() <= zb).all(), (r, h)
    return handle, batch


# Batches whose keys and values pass what stays in the caches (1.2e8 bytes), by 128 keys:
# their loads are non-temporal ones.
PAST_CACHES = 1.2e8


@pytest.mark.parametrize("type,cache", TYPES)
@pytest.mark.parametrize("hs", [32, 64, 128])
@pytest.mark.parametrize("group", [1, 3, 5, 20])
@pytest.mark.parametrize("page", [16, 24])
def test_attention_split_past_the_caches(gpu, type, cache, hs, group, page):
    kv = 1024 // hs
    if type == "f32" and group == 20:
        group = 16  # (more take two workgroups, which keep the rows for each other)
    lens = [8300, 1, 8129] if cache == "f32" else [8300, 129, 8129, 0, 8200, 8300]
    size = DTYPES[cache].itemsize
    assert sum(lens) * 2 * 1024 * size > PAST_CACHES
    print("past the caches", type, cache, hs, group, page, flush=True)
    handle, batch = large_batch(lens, kv * group, kv, hs, type, cache, page, max(lens), seed=hs)
    assert bmb.paged_attention_workspace(handle, batch) > 0


@pytest.mark.parametrize("type,cache", TYPES)
@pytest.mark.parametrize("hs", [32, 64, 128])
@pytest.mark.parametrize("group", [1, 5])
@pytest.mark.parametrize("page", [16, 24])
def test_attention_whole_past_the_caches(gpu, type, cache, hs, group, page):
    """The same loads for sequences of one part each."""
    kv, size = 1024 // hs, DTYPES[cache].itemsize
    max_len = (512 << 10) // (2 * hs * size)
    lens = [max_len, 1, 0] + [(37 * i) % max_len for i in range(60)] + [max_len - 1]
    assert 0.5 * len(lens) * max_len * 2 * 1024 * size > PAST_CACHES
    handle, batch = large_batch(lens, kv * group, kv, hs, type, cache, page, max_len, seed=hs + 1)
    assert bmb.paged_attention_workspace(handle, batch) == 0


@pytest.mark.parametrize("type,cache,heads", [("bf16", "bf16", 2), ("f32", "f16", 1)])
@pytest.mark.parametrize("requests", [4097, 4300])
def test_attention_split_of_thousands_of_requests(gpu, type, cache, heads, requests):
    """More than 64 requests to a lane of the search for a part: every request's
    rows, those of the long ones in two of them included."""
    lens = [i % 3 for i in range(requests)]
    share = -(-requests // 64)
    lens[10 * share + share - 1], lens[-1], lens[20 * share] = 9000, 700, 20000
    d = Problem(lens, heads, 1, 32, type, cache, 16, seed=requests).device()
    assert share > 64 and d.workspace() > 0
    d.run()
    d.check()


@pytest.mark.parametrize("type,cache", [("f32", "f32"), ("f16", "f16")])
def test_attention_many_requests(gpu, type, cache):
    """More workgroups than the device holds at once, every request whole."""
    lens = [(7 * i) % 61 for i in range(1500)]
    lens[1234] = 1300
    d = Problem(lens, 4, 2, 64, type, cache, 16, seed=16).device()
    assert bmb.paged_attention_workspace(d.cache, d.batch) == 0
    d.run()
    d.check()


@pytest.mark.parametrize("type,cache", [("f32", "f32"), ("bf16", "bf16")])
def test_attention_rows(gpu, type, cache):
    """Rows in another order, idle requests, rows outside the range, short and
    split sequences: unnamed rows stay."""
    for lens in ([5, 60, 0, 33, 7], [5, 700, 0, 33, 900]):
        rows = [4, -1, 2, 0, 1000000]
        d = Problem(lens, 4, 2, 64, type, cache, 16, rows=[4, -1, 2, 0, -9], seed=3).device()
        d.rows.copy_(ints(rows))
        d.run()
        d.check()


@pytest.mark.parametrize("type,cache", TYPES)
def test_attention_sharp_and_negative_scale(gpu, type, cache):
    """Scores of hundreds (one key takes all), and a negative scale."""
    for scale, spread in ((1.0, 12.0), (-0.4, 2.0), (0.0, 1.0)):
        d = Problem([1, 40, 400, 1000], 6, 3, 64, type, cache, 16, scale=scale, spread=spread,
                    seed=4).device()
        d.run()
        d.check()


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("heads,page", [(2, 16), (5, 10), (40, 16)])
@pytest.mark.parametrize("gap", [8, 14, 18, 20])
def test_attention_weak_keys_beside_a_strong_one(gpu, type, heads, page, gap):
    """One key `gap` nats above all others, its value 0, theirs large: the result
    is what the weak keys bring, to its last bits.

    The bound is Problem.exact's, but for what the two 16-bit numbers of a
    probability lose: at most 2^-17 (bf16) or 2^-23 (fp16) of it, and in fp16 up
    to 2^-40 of the largest, once for each key."""
    lens = [2, 40, 700, 3000, 129]
    strong = [0, 39, 350, 2999, 17]
    p = Problem(lens, heads, 1, 64, type, type, page, seed=gap)
    p.q.zero_()
    p.q[:, :heads * 64:64] = 1.0  # the score is scale times the key's first element
    p.scale = gap / 16.0
    g = torch.Generator().manual_seed(gap)
    for r, n in enumerate(lens):
        t = torch.arange(n)
        at = (p.table[r].long()[t // page], t % page)
        p.k[at] = 0.0
        p.v[at] = (30000.0 + 30000.0 * torch.rand(n, 1, 64, generator=g)).to(p.v.dtype)
        one = (int(p.table[r, strong[r] // page]), strong[r] % page)
        p.k[one] = 16.0
        p.v[one] = 0.0
    d = p.device()
    d.run()
    torch.cuda.synchronize()
    bmb.check("paged_attention")
    half_step, lost = torch.finfo(DTYPES[type]).eps / 2, 2.0 ** (-17 if type == "bf16" else -23)
    for r, (want, lse, _, lse_bound) in p.exact().items():
        n = lens[r]
        ds = 4 * (math.sqrt(64) + 1) * U32 * gap + 4 * U32 * gap
        eps = 2 * ds + (4 * math.sqrt(n) + 16) * U32 + lost
        # (all values are at least 0: the sum of their magnitudes is the result)
        bound = (eps + half_step) * want
        if type == "f16":
            bound = bound + 2.0 ** -40 * 60000 * n + 2.0 ** -25
        got = d.out[r, :heads * 64].cpu().double().view(heads, 64)
        worst = ((got - want).abs() / bound).max().item()
        assert worst <= 1.0, (r, n, worst, got[0, :4], want[0, :4])
        assert ((d.lse[r].cpu().double() - lse).abs() <= lse_bound).all()


@pytest.mark.parametrize("type,cache", TYPES)
@pytest.mark.parametrize("page", [16, 6])
def test_attention_pages_outside_the_cache(gpu, type, cache, page):
    """Tokens in pages outside [0, pages) count as absent; a request with no
    other gives 0 and -inf."""
    d = Problem([page, 4 * page, 900], 4, 4, 32, type, cache, page, seed=5).device()
    p = d.p
    bad = d.table.clone()
    bad[0, 0], bad[1, 1], bad[1, 3], bad[2, 0], bad[2, 9] = -1, p.pages, 1 << 30, -(1 << 30), -2
    d.table.copy_(bad)
    d.run()
    torch.cuda.synchronize()
    bmb.check("paged_attention")
    W = p.heads * p.hs
    assert (d.out[0, :W] == 0).all() and (d.lse[0] == -math.inf).all()
    for r in (1, 2):
        keep = [t for t in range(p.lens[r]) if 0 <= bad[r, t // page] < p.pages]
        q = p.q[r, :W].double().view(p.heads, p.hs)
        k, v = p.tokens(r, p.k)[keep], p.tokens(r, p.v)[keep]
        x = torch.einsum("hd,nhd->hn", q, k) * p.scale
        out = torch.einsum("hn,nhd->hd", torch.softmax(x, 1), v)
        # scores below 8 here; 2^-7 covers an output's half step in any type
        tol = {"f32": 1e-5, "f16": 2e-3, "bf16": 2.0 ** -7}[type]
        assert (d.out[r, :W].cpu().double().view(p.heads, p.hs) - out).abs().max() < tol
        assert (d.lse[r].cpu().double() - torch.logsumexp(x, 1)).abs().max() < 1e-4


def test_attention_infinite_and_nan_keys(gpu):
    """A live key of -inf scores takes no part; all of them: an empty row. A NaN
    in a live key reaches its heads and no others."""
    p = Problem([3, 3, 3], 2, 2, 32, "f32", "f32", 16, seed=6)
    p.q[:, :64] = 1.0
    place = lambda r, t: (int(p.table[r, 0]), t)
    p.k[place(0, 1)] = -math.inf
    for t in range(3):
        p.k[place(1, t)] = -math.inf
    p.k[place(2, 0)][0, 5] = math.nan
    d = p.device()
    d.run()
    torch.cuda.synchronize()
    k, v = p.tokens(0, p.k)[[0, 2]], p.tokens(0, p.v)[[0, 2]]
    x = torch.einsum("hd,nhd->hn", torch.ones(2, 32, dtype=torch.float64), k) * p.scale
    want = torch.einsum("hn,nhd->hd", torch.softmax(x, 1), v)
    assert (d.out[0, :64].cpu().double().view(2, 32) - want).abs().max() < 1e-5
    assert (d.out[1, :64] == 0).all() and (d.lse[1] == -math.inf).all()
    assert torch.isnan(d.out[2, :32]).all() and torch.isfinite(d.out[2, 32:64]).all()


def test_attention_longer_than_max_len(gpu):
    """The rest of a longer sequence is not read."""
    d = Problem([100, 700], 2, 2, 64, "f32", "f32", 16, seed=7).device()
    d.batch.max_len = 96
    d.run()
    torch.cuda.synchronize()
    d.p.lens = [96, 96]
    d.check()


def test_attention_of_no_tokens(gpu):
    """max_len 0: every request is empty, and its table is not looked at."""
    d = Problem([3, 40], 2, 2, 64, "bf16", "bf16", 16, seed=7).device()
    d.batch.max_len, d.batch.table_stride = 0, 0
    d.run()
    torch.cuda.synchronize()
    d.p.lens = [0, 0]
    d.check()


@pytest.mark.parametrize("type,cache", TYPES)
def test_attention_subnormal_values(gpu, type, cache):
    """fp16 values below 2^-14 (and results, where the type holds them) keep
    their digits."""
    p = Problem([50, 300], 8, 1, 64, type, cache, 16, seed=14)
    p.v = (p.v.float() * 2.0 ** -19).to(p.v.dtype)
    p.k = torch.where(torch.rand(p.k.shape, generator=torch.Generator().manual_seed(1)) < 0.3,
                      (p.k.float() * 2.0 ** -19).to(p.k.dtype), p.k)
    d = p.device()
    d.run()
    d.check()


def test_attention_broadcast_query(gpu):
    """q_stride 0: one query for all requests."""
    d = Problem([20, 33, 900], 4, 2, 64, "f32", "f32", 16, seed=15).device()
    d.batch.q_stride = 0
    d.p.q[1:] = d.p.q[0]
    d.run()
    d.check()


def test_attention_interleaved_halves_and_null_lse(gpu):
    """K and V in one buffer (pages, 2, page, kv, hs); no lse."""
    d = Problem([40, 300], 4, 2, 64, "f16", "f16", 16, seed=8).device()
    both = torch.stack([d.k, d.v], 1).contiguous()
    d.cache.k, d.cache.v = both.data_ptr(), both.data_ptr() + both[0, 0].numel() * 2
    d.cache.page_stride *= 2
    bmb.paged_attention(d.cache, d.batch, d.out.data_ptr(), None, d.q.data_ptr())
    torch.cuda.synchronize()
    assert (d.lse == 768.0).all()
    d.run()
    d.check()


@pytest.mark.parametrize("page", [16, 12])
def test_attention_offsets_past_32_bits(gpu, page):
    """Pages whose places lie more than 2^32 elements into the buffer."""
    kv, hs = 8, 128
    pages = (1 << 32) // (page * kv * hs) + 8
    k = torch.zeros(pages, page, kv, hs, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    small = Problem([70], kv, kv, hs, "f16", "f16", page, seed=9)
    d = small.device()
    shift = pages - small.pages
    k[shift:], v[shift:] = d.k, d.v
    d.table.add_(shift)
    d.k, d.v = k, v
    d.cache = cache_struct(k, v, "token", page, kv, hs, "f16")
    d.run()
    d.check()
    rows = torch.randn(2, 2 * kv * hs, device="cuda").half()
    slots = ints([pages * page - 1, 5])
    bmb.paged_append(d.cache, rows.data_ptr(), rows.data_ptr() + 2 * kv * hs, bmb.F16, 2 * kv * hs,
                     slots.data_ptr(), 2)
    torch.cuda.synchronize()
    assert torch.equal(k[-1, -1].view(-1), rows[0, :kv * hs])
    assert torch.equal(v[0, 5].view(-1), rows[1, kv * hs:])


@pytest.mark.parametrize("type,cache,heads", [("f32", "f32", 32), ("f16", "f16", 64)])
def test_attention_parts_of_several_launches(gpu, type, cache, heads):
    """More requests than one dispatch has lanes for: the bits of a few of them
    alone, over and over."""
    kv, hs, few = 32, 32, 61
    small = Problem([i % 4 for i in range(few)], heads, kv, hs, type, cache, 16, seed=23)
    d = small.device()
    d.run()
    d.check()
    requests, W = (1 << 19) + 11, heads * hs
    times = -(-requests // few)
    table, lens, q = (x.repeat(times, *[1] * (x.dim() - 1))[:requests].contiguous()
                      for x in (d.table, d.lens, d.q[:, :W]))
    out = torch.full((requests, W), 768.0, dtype=DTYPES[type], device="cuda")
    lse = torch.full((requests, heads), 768.0, device="cuda")
    b = d.batch
    b.requests = b.n_rows = requests
    b.q_stride = b.out_stride = W
    b.block_table, b.lens = table.data_ptr(), lens.data_ptr()
    assert bmb.paged_attention_workspace(d.cache, b) == 0
    bmb.paged_attention(d.cache, b, out.data_ptr(), lse.data_ptr(), q.data_ptr())
    torch.cuda.synchronize()
    bmb.check("paged_attention")
    for got, want in ((out, d.out[:, :W]), (lse, d.lse)):
        whole = requests // few * few
        assert (got[:whole].view(-1, *want.shape) == want).all()
        assert torch.equal(got[whole:], want[:requests - whole])


def test_attention_joins_of_several_launches(gpu):
    """More heads of requests than one dispatch has lanes for, the last request
    split: its joined rows within the bound, every other the one value it has."""
    requests, heads, kv, hs, page, n = 2051, 8192, 256, 32, 4096, 100000
    pages, max_len, G, W = pages_of(n, page), 1 << 21, heads // kv, heads * hs
    g = torch.Generator(device="cuda").manual_seed(24)
    k, v = (torch.empty(pages, page, kv, hs, device="cuda", dtype=torch.float16)
            .normal_(generator=g) for _ in range(2))
    q = torch.empty(W, device="cuda", dtype=torch.float16).normal_(generator=g)
    table = torch.zeros(requests, pages_of(max_len, page) + 1, dtype=torch.int32, device="cuda")
    table[:, 0] = torch.arange(requests, device="cuda") % pages
    table[-1, :pages] = torch.arange(pages, device="cuda")
    lens = torch.ones(requests, dtype=torch.int32, device="cuda")
    lens[-1] = n
    out = torch.full((requests, W), 768.0, dtype=torch.float16, device="cuda")
    batch = bmb.PagedBatch(requests=requests, max_len=max_len + 1, table_stride=table.shape[1],
                           heads=heads, n_rows=requests, type=bmb.F16, scale=1 / math.sqrt(hs),
                           q_stride=0, out_stride=W, block_table=table.data_ptr(),
                           lens=lens.data_ptr())
    cache = cache_struct(k, v, "token", page, kv, hs, "f16")
    need = bmb.paged_attention_workspace(cache, batch)
    assert need > 0 and requests * heads * 256 > 1 << 32
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    batch.work, batch.work_bytes = work.data_ptr(), need
    bmb.paged_attention(cache, batch, out.data_ptr(), None, q.data_ptr())
    torch.cuda.synchronize()
    bmb.check("paged_attention")
    for p in range(pages):  # one key: its value
        assert (out[p:-1:pages].view(-1, kv, G, hs) == v[p, 0][:, None]).all()
    for h in (0, 100, kv - 1):
        x = (q.view(kv, G, hs)[h].double() @ k.view(-1, kv, hs)[:n, h].double().t()) / math.sqrt(hs)
        values = v.view(-1, kv, hs)[:n, h].double()
        weights = torch.softmax(x, 1)
        want = weights @ values
        # as Problem.exact
        mag = (q.view(kv, G, hs)[h].abs().double()
               @ k.view(-1, kv, hs)[:n, h].abs().double().t()).amax(1) / math.sqrt(hs)
        eps = (2 * (4 * (math.sqrt(hs) + 1) * U32 * mag + 4 * U32 * x.abs().amax(1))
               + (4 * math.sqrt(n) + 16) * U32 + 2.0 ** -23)
        bound = (eps[:, None] * (weights @ values.abs()) + 2.0 ** -40 * values.abs().sum(0)
                 + 2.0 ** -11 * want.abs() + 2.0 ** -25)
        got = out[-1].view(kv, G, hs)[h].double()
        assert ((got - want).abs() <= bound).all(), ((got - want).abs() / bound).max()


def test_attention_streams_and_scratch(gpu):
    """Leased scratch on two streams in turn, and the same bits as with a
    workspace of the caller's, every time."""
    a = Problem([2000, 1, 700], 8, 2, 64, "bf16", "bf16", 16, seed=10).device()
    b = Problem([900] * 9, 4, 4, 64, "f32", "f32", 16, seed=11).device()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    bits = []
    for i in range(6):
        for d in (a, b):
            s = streams[i % 2]
            d.run(s.cuda_stream)
        torch.cuda.synchronize()
        bits.append([d.out.cpu().view(torch.int16).numpy().copy() for d in (a, b)])
    a.check()
    b.check()
    for d in (a, b):
        d.workspace()
        d.run()
        d.check()
    bits.append([d.out.cpu().view(torch.int16).numpy().copy() for d in (a, b)])
    for x in bits[1:]:
        for y, z in zip(x, bits[0]):
            assert np.array_equal(y, z)


def test_attention_captured(gpu):
    """Captured with a workspace, replayed with other lengths and queries each
    time; without one the capture is refused before anything is queued."""
    lens = [600, 3, 1400]
    d = Problem(lens, 8, 2, 64, "bf16", "bf16", 16, seed=12).device()
    d.workspace()
    side = torch.cuda.Stream()
    d.run(side.cuda_stream)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        d.run(side.cuda_stream)
        work, d.batch.work = d.batch.work, None
        with pytest.raises(ValueError):
            d.run(side.cuda_stream)
        d.batch.work = work
    other = Problem([50, 60], 4, 4, 64, "f32", "f32", 16, seed=13).device()
    for now in ([600, 3, 1400], [599, 0, 17], [1, 2, 1399]):
        d.p.lens = now
        d.lens.copy_(ints(now))
        d.out.fill_(768.0)
        d.p.q = torch.randn(d.p.q.shape).to(torch.bfloat16)
        d.q.copy_(d.p.q)
        torch.cuda.synchronize()
        graph.replay()
        d.check()
        other.run()
        other.check()


def test_attention_two_graphs_at_once(gpu):
    """Two captured calls with a workspace each, replayed at once on two
    streams: the eager bits, every time."""
    problems = [Problem([3000, 5, 1200], 8, 2, 64, "bf16", "bf16", 16, seed=17),
                Problem([900] * 9 + [0], 4, 4, 64, "f32", "f32", 12, seed=18)]
    ds, graphs, streams, bits = [p.device() for p in problems], [], [], []
    for d in ds:
        assert d.workspace() > 0
        d.run()
        d.check()
        bits.append(d.out.cpu().view(torch.int16).numpy().copy())
        side = torch.cuda.Stream()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            d.run(side.cuda_stream)
        graphs.append(g)
        streams.append(side)
    for _ in range(4):
        for d in ds:
            d.out.fill_(768.0)
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for d, b in zip(ds, bits):
            assert np.array_equal(d.out.cpu().view(torch.int16).numpy(), b)


def test_attention_from_host_threads(gpu):
    """Four host threads with leased scratch on the null stream at once."""
    ds = [Problem([1500 + 100 * i, 40], 8, 2, 64, "f16", "f16", 16, seed=20 + i).device()
          for i in range(4)]
    torch.cuda.synchronize()
    barrier, errors = threading.Barrier(4), []

    def work(d):
        try:
            barrier.wait()
            for _ in range(10):
                d.run()
            torch.cuda.synchronize()
            bmb.check("paged_attention")
        except Exception as e:  # reported by the main thread
            errors.append(repr(e))

    threads = [threading.Thread(target=work, args=(d,)) for d in ds]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=60)
    assert not any(t.is_alive() for t in threads) and not errors, errors
    for d in ds:
        d.check()


# --------------------------------------------------------------- together
def test_generation_matches_whole_sequence_attention(gpu):
    """Prompts through the fused whole-sequence attention, then token by token
    through plan, append and paged attention: every new row equals the row that
    whole-sequence attention over everything gives (both fp32: the two bounds,
    1e-5 each at these sizes), and the cache never mixes requests up."""
    NH, hs, page, T = 4, 64, 16, 96
    C = NH * hs
    prompts, steps = [33, 1, 64, 17], 20
    R = len(prompts)
    g = torch.Generator().manual_seed(21)
    qkv = torch.randn(R, T, 3 * C, generator=g).cuda()
    pool = Pool([0] * R, page, width=pages_of(T, page), free=R * pages_of(T, page), seed=4)
    k = torch.full((pool.pages, page, NH, hs), math.nan, device="cuda")
    v = k.clone()
    cache = cache_struct(k, v, "token", page, NH, hs, "f32")
    ref_o, _ = O.attn_fwd_f64(qkv.cpu().numpy(), R, T, C, NH)
    for step in range(steps):
        new = prompts if step == 0 else [1] * R
        if step == 7:
            new = [1, 0, 1, 1]  # request 1 waits
        total = sum(new)
        before = pool.lens.copy()
        o = pool.step(new, total + 3)
        rows = torch.cat([qkv[r, before[r]:before[r] + n] for r, n in enumerate(new)])
        bmb.paged_append(cache, rows.data_ptr() + C * 4, rows.data_ptr() + 2 * C * 4, bmb.F32,
                         3 * C, o["slots"].data_ptr(), total)
        att = torch.zeros(total, C, device="cuda")
        batch = bmb.PagedBatch(requests=R, max_len=T, table_stride=pool.table.shape[1], heads=NH,
                               n_rows=total, type=bmb.F32, scale=1 / math.sqrt(hs),
                               q_stride=3 * C, out_stride=C,
                               block_table=pool.d["table"].data_ptr(),
                               lens=pool.d["lens"].data_ptr(), rows=o["rows"].data_ptr())
        bmb.paged_attention(cache, batch, att.data_ptr(), None, rows.data_ptr())
        torch.cuda.synchronize()
        bmb.check("generation step")
        at = 0
        for r, n in enumerate(new):
            at += n
            if n:
                want = ref_o.reshape(R, T, C)[r, pool.lens[r] - 1]
                err = np.abs(att[at - 1].cpu().numpy() - want).max()
                assert err < 2e-5, (step, r, err)
        if step == 0:  # the prompts' own rows, by the whole-sequence kernel
            for r, n in enumerate(prompts):
                x = qkv[r, :n].contiguous()
                y, lse = torch.empty(n, C, device="cuda"), torch.empty(NH * n, device="cuda")
                bmb.flash_forward(y.data_ptr(), lse.data_ptr(), x.data_ptr(), 1, n, C, NH)
                torch.cuda.synchronize()
                last = att[sum(prompts[:r + 1]) - 1]
                assert (y[n - 1] - last).abs().max() < 2e-5
