"""Performance cases of the generation operators: what a program that serves a trained GPT token by
token has the library do between two forward passes.

  plan    a step's pages, slots and positions from each request's length, for a pool of pages
  append  the keys and values of the step's tokens into the paged cache
  attend  attention of one new token a request over its pages
  logits  penalties for repeated tokens, biases and grammar masks on the logits

A case is a dict of plain values; listed() gives the ones quoted, draw() more of the same ranges.
With `own` false run() computes an operator in elementary torch operations; with `own` true it
makes the library's calls.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_I32 = torch.int32


def listed():
    return [
        # One decoding step of 64 requests of up to 1024 tokens: one token each, a few of them
        # ending. Latency.
        dict(name="plan_decode", op="plan", requests=64, page=16, lo=1, hi=1023, prompt=0,
             prompts=0.0, ended=0.05, idle=0.05, spare=1.5, mix=1),
        # A server that admits many prompts at once beside running requests.
        dict(name="plan_prompts", op="plan", requests=512, page=16, lo=1, hi=4096, prompt=4096,
             prompts=0.6, ended=0.05, idle=0.05, spare=1.2, mix=2),
        # GPT-2 small (12 heads of 64): one token of each of 32 requests, out of the fused QKV
        # rows into an fp32 cache. Latency.
        dict(name="append_decode_gpt2", op="append", tokens=32, kv=12, hs=64, type="f32",
             cache="f32", page=16, layout="token", padded=0.0),
        # Its prompts: 8 x 1024 tokens, kept in 16 bits.
        dict(name="append_prompts_gpt2", op="append", tokens=8192, kv=12, hs=64, type="f32",
             cache="bf16", page=16, layout="token", padded=0.02),
        # A long prompt of a wide model, head by head inside a page.
        dict(name="append_large", op="append", tokens=65536, kv=8, hs=128, type="bf16",
             cache="bf16", page=64, layout="head", padded=0.0),
        # One sequence of GPT-2 small near its full length, everything fp32. Latency.
        dict(name="attend_gpt2_one", op="attend", requests=1, heads=12, kv=12, hs=64, type="f32",
             cache="f32", page=16, layout="token", lo=1000, hi=1000, idle=0.0, mix=3),
        # 64 of them of any length, the cache in 16 bits.
        dict(name="attend_gpt2_batch", op="attend", requests=64, heads=12, kv=12, hs=64,
             type="f32", cache="bf16", page=16, layout="token", lo=1, hi=1024, idle=0.0, mix=4),
        # Shared key-value heads, many requests from a few tokens to thousands.
        dict(name="attend_gqa_ragged", op="attend", requests=128, heads=32, kv=8, hs=128,
             type="f16", cache="f16", page=16, layout="head", lo=1, hi=8192, idle=0.0, mix=5),
        # fp32 cache, pages that are no whole number of 16 keys.
        dict(name="attend_f32_pages24", op="attend", requests=16, heads=8, kv=8, hs=128,
             type="f32", cache="f32", page=24, layout="token", lo=3000, hi=4000, idle=0.0, mix=6),
        # Two very long contexts: the cache's length has to fill the device.
        dict(name="attend_long", op="attend", requests=2, heads=32, kv=8, hs=128, type="bf16",
             cache="bf16", page=64, layout="head", lo=131072, hi=131072, idle=0.0, mix=7),
        # The next token of one sequence over the unpadded vocabulary (odd rows). Latency.
        dict(name="logits_one", op="logits", rows=1, V=50257, type="f32", lo=1000, hi=1000,
             biases=16, grammar=1.0, mix=8),
        # A large batch of them, some rows under a grammar, some free.
        dict(name="logits_batch", op="logits", rows=512, V=50257, type="f32", lo=16, hi=2048,
             biases=64, grammar=0.3, mix=9),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend", "logits", "logits"])
    mix = rng.randrange(1 << 30)
    page = rng.choice([8, 16, 16, 32, 64, 128, 5, 24])
    if op == "plan":
        return dict(op=op, requests=_log(rng, 1, 1024), page=page, lo=1, hi=_log(rng, 64, 4096),
                    prompt=_log(rng, 1, 2048), prompts=rng.choice([0.0, 0.1, 0.5, 1.0]),
                    ended=rng.choice([0.0, 0.1]), idle=rng.choice([0.0, 0.1]),
                    spare=rng.choice([0.6, 1.0, 2.0]), mix=mix)
    if op == "append":
        t, cache = rng.choice([("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"),
                               ("f16", "f16")])
        return dict(op=op, tokens=_log(rng, 1, 16384), kv=rng.choice([1, 2, 6, 8, 12]),
                    hs=rng.choice([32, 64, 128]), type=t, cache=cache, page=page,
                    layout=rng.choice(["token", "head"]), padded=rng.choice([0.0, 0.1]))
    if op == "attend":
        t, cache = rng.choice([("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"),
                               ("f16", "f16")])
        kv, group = rng.choice([1, 2, 4, 6, 8, 12]), rng.choice([1, 1, 2, 3, 4, 8, 16])
        hs = rng.choice([32, 64, 64, 128])
        hi = _log(rng, 1, 65536)
        requests = _log(rng, 1, 256)
        while requests > 1 and requests * hi * kv * hs > 1e8:
            requests = requests * 2 // 3
        return dict(op=op, requests=requests, heads=kv * group, kv=kv, hs=hs, type=t, cache=cache,
                    page=page, layout=rng.choice(["token", "head"]), lo=max(1, hi // 64), hi=hi,
                    idle=rng.choice([0.0, 0.0, 0.2]), mix=mix)
    V = rng.choice([65, 4096, 32000, 50257, 50257, 50304, 131073])
    rows = _log(rng, 1, 256)
    return dict(op=op, rows=rows, V=V, type=rng.choice(["f32", "f32", "f16", "bf16"]), lo=1,
                hi=_log(rng, 8, 8192), biases=rng.choice([0, 4, 100]),
                grammar=rng.choice([0.0, 0.5, 1.0]), mix=mix)


# ------------------------------------------------------------ shapes of a case
def _plan_shape(c):
    """(tokens held, tokens of this step) of each request: a new prompt holds none and brings
    many, a running request brings one, an idle one none, and -1 ends a request."""
    r = random.Random(c["mix"])
    held, new = [], []
    for _ in range(c["requests"]):
        n, kind = _log(r, c["lo"], c["hi"]), r.random()
        if kind < c["ended"]:
            held.append(n)
            new.append(-1)
        elif kind < c["ended"] + c["idle"]:
            held.append(n)
            new.append(0)
        elif r.random() < c["prompts"]:
            held.append(0)
            new.append(_log(r, max(1, c["prompt"] // 64), max(1, c["prompt"])))
        else:
            held.append(n)
            new.append(1)
    return held, new


def _pages(tokens, page):
    return (tokens + page - 1) // page


def _plan_sizes(c):
    held, new = _plan_shape(c)
    P = c["page"]
    need = sum(_pages(h + n, P) - _pages(h, P) for h, n in zip(held, new) if n > 0)
    used = sum(_pages(h, P) for h in held)
    width = max(_pages(h + max(n, 0), P) for h, n in zip(held, new)) + 2
    return dict(held=held, new=new, width=width, used=used, free=int(need * c["spare"]) + 1,
                tokens=sum(n for n in new if n > 0))


def _lens(c):
    r = random.Random(c["mix"])
    return [_log(r, c["lo"], c["hi"]) for _ in range(c["requests"])]


def _idle(c):
    """The requests that take no part in this step (their rows are -1)."""
    r = random.Random(c["mix"] + 1)
    return [r.random() < c["idle"] for _ in range(c["requests"])]


def _history(c):
    """(tokens, prompt tokens among them) of each row."""
    r = random.Random(c["mix"])
    out = []
    for _ in range(c["rows"]):
        n = _log(r, c["lo"], c["hi"])
        out.append((n, int(n * r.random())))
    return out


def _masked(c):
    r = random.Random(c["mix"] + 1)
    return [r.random() < c["grammar"] for _ in range(c["rows"])]


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

    def perm(self, n):
        return torch.randperm(n, device="cuda", dtype=_I32, generator=self.g)


def _ints(values):
    return torch.tensor(values, device="cuda", dtype=_I32)


def _bmb():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "bare-metal-bard_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import bmb
    return bmb


def _cache(r, pages, c):
    """The two halves of a cache of `pages` pages, the type's values everywhere (pages that hold
    no request's tokens keep those of requests that ended)."""
    P, kv, hs = c["page"], c["kv"], c["hs"]
    shape = (pages, P, kv, hs) if c["layout"] == "token" else (pages, kv, P, hs)
    return (r.normal(*shape, dtype=_TYPES[c["cache"]]), r.normal(*shape, dtype=_TYPES[c["cache"]]))


def _cache_handle(bmb, s, c):
    P, kv, hs = c["page"], c["kv"], c["hs"]
    token, head = (kv * hs, hs) if c["layout"] == "token" else (hs, P * hs)
    return bmb.PagedCache(k=s["k_cache"].data_ptr(), v=s["v_cache"].data_ptr(),
                          type=bmb.ELEMENT_TYPES[c["cache"]], pages=s["k_cache"].shape[0],
                          page_size=P, kv_heads=kv, head_size=hs, page_stride=P * kv * hs,
                          token_stride=token, head_stride=head)


def prepare(case, seed):
    c, r = dict(case), _Rng(seed)
    s = dict(c=c)
    _PREPARE[c["op"]](s, c, r)
    return s


def _prepare_plan(s, c, r):
    z = _plan_sizes(c)
    R, P, width = c["requests"], c["page"], z["width"]
    pages = z["used"] + z["free"]
    order = r.perm(pages)
    # Pages are handed to the requests in a random order; the rest are free, in a ring.
    held = _ints([_pages(h, P) for h in z["held"]])
    start = (torch.cumsum(held, 0) - held)[:, None]
    col = torch.arange(width, device="cuda")[None, :]
    inside = col < held[:, None]
    table = torch.where(inside, order[torch.where(inside, start + col, 0)], -1).to(_I32)
    head = int(torch.randint(0, pages, (1,), device="cuda", generator=r.g))
    ring = torch.full((pages,), -1, device="cuda", dtype=_I32)
    at = (head + torch.arange(z["free"], device="cuda")) % pages
    ring[at] = order[z["used"]:]
    T = max(1, z["tokens"])
    s.update(table=table, ring=ring, state=_ints([head, z["free"]]), lens=_ints(z["held"]),
             new=_ints(z["new"]), T=T, pages=pages, width=width,
             lens_out=torch.zeros(R, device="cuda", dtype=_I32),
             state_out=torch.zeros(2, device="cuda", dtype=_I32),
             slots=torch.zeros(T, device="cuda", dtype=_I32),
             positions=torch.zeros(T, device="cuda", dtype=_I32),
             rows=torch.zeros(R, device="cuda", dtype=_I32),
             offsets=torch.zeros(R + 1, device="cuda", dtype=_I32))
    if own:
        bmb = s["bmb"] = _bmb()
        p = {k: s[k].data_ptr() for k in ("lens", "lens_out", "state", "state_out", "slots",
                                          "positions", "rows", "offsets")}
        s["plan"] = bmb.PagedPlan(requests=R, max_pages=width, pages=pages, page_size=P,
                                  max_tokens=T, new_tokens=s["new"].data_ptr(),
                                  free_pages=ring.data_ptr(), block_table=table.data_ptr(), **p)


def _prepare_append(s, c, r):
    n, P, kv, hs = c["tokens"], c["page"], c["kv"], c["hs"]
    pages = _pages(n, P) * 5 // 4 + 1
    s["k_cache"], s["v_cache"] = _cache(r, pages, c)
    # The step's tokens fill pages in a random order of pages; a padded batch has rows without one.
    t = torch.arange(n, device="cuda")
    slots = r.perm(pages)[t // P].long() * P + t % P
    slots = torch.where(r.uniform(n) < c["padded"], -1, slots)
    s["slots"] = slots.to(_I32)
    # Rows of the fused projection: queries, keys, values.
    s["qkv"] = r.normal(n, 3 * kv * hs, dtype=_TYPES[c["type"]])
    if own:
        bmb = s["bmb"] = _bmb()
        s["cache"], s["type"] = _cache_handle(bmb, s, c), bmb.ELEMENT_TYPES[c["type"]]


def _prepare_attend(s, c, r):
    R, P, kv, hs, heads = c["requests"], c["page"], c["kv"], c["hs"], c["heads"]
    lens = _lens(c)
    held = [_pages(n, P) for n in lens]
    pages, width = sum(held) + 3, max(held) + 1
    order = r.perm(pages)
    cnt = _ints(held)
    start = (torch.cumsum(cnt, 0) - cnt)[:, None]
    col = torch.arange(width, device="cuda")[None, :]
    inside = col < cnt[:, None]
    s["table"] = torch.where(inside, order[torch.where(inside, start + col, 0)], -1).to(_I32)
    s["k_cache"], s["v_cache"] = _cache(r, pages, c)
    row, rows = 0, []
    for idle in _idle(c):
        rows.append(-1 if idle else row)
        row += not idle
    t = _TYPES[c["type"]]
    s.update(lens=_ints(lens), host_lens=lens, host_rows=rows, rows=_ints(rows),
             qkv=r.normal(R, (heads + 2 * kv) * hs, dtype=t),
             out=torch.zeros(R, heads * hs, device="cuda", dtype=t),
             lse=torch.zeros(R, heads, device="cuda"), scale=1.0 / math.sqrt(hs))
    if own:
        bmb = s["bmb"] = _bmb()
        s["cache"] = _cache_handle(bmb, s, c)
        s["batch"] = bmb.PagedBatch(requests=R, max_len=max(lens), table_stride=width,
                                    heads=heads, n_rows=R, type=bmb.ELEMENT_TYPES[c["type"]],
                                    scale=s["scale"], q_stride=(heads + 2 * kv) * hs,
                                    out_stride=heads * hs, block_table=s["table"].data_ptr(),
                                    lens=s["lens"].data_ptr(), rows=s["rows"].data_ptr())
        need = bmb.paged_attention_workspace(s["cache"], s["batch"])
        s["work"] = torch.empty(need, device="cuda", dtype=torch.uint8)
        s["batch"].work, s["batch"].work_bytes = s["work"].data_ptr(), need


def _prepare_logits(s, c, r):
    rows, V = c["rows"], c["V"]
    hist = _history(c)
    width = max(n for n, _ in hist)
    lens, prompts = _ints([n for n, _ in hist]), _ints([p for _, p in hist])
    # Text: the frequent words are the low ids, and they repeat.
    ids = (V ** r.uniform(rows, width)).to(_I32).clamp_(max=V) - 1
    s["tokens"] = torch.where(torch.arange(width, device="cuda")[None, :] < lens[:, None], ids, -1)
    nb = c["biases"]
    masked = _masked(c)
    index, m = [], 0
    for on in masked:
        index.append(m if on else -1)
        m += on
    words = (V + 31) // 32
    # A grammar allows a few words, or most of them.
    few = r.uniform(max(m, 1), 1) < 0.5
    bits = r.uniform(max(m, 1), words, 32) < torch.where(few, 0.01, 0.9)[:, :, None]
    weight = torch.ones(32, device="cuda", dtype=torch.int64) << torch.arange(32, device="cuda")
    mask = (bits * weight).sum(2)
    mask = torch.where(mask >= 1 << 31, mask - (1 << 32), mask).to(_I32)
    s.update(lens=lens, prompts=prompts, logits=r.normal(rows, V, std=3.0, dtype=_TYPES[c["type"]]),
             out=torch.zeros(rows, V, device="cuda", dtype=_TYPES[c["type"]]),
             repetition=1.0 + 0.3 * r.uniform(rows), frequency=0.5 * r.uniform(rows),
             presence=0.5 * r.uniform(rows), mask=mask, mask_index=_ints(index),
             bias_offsets=_ints([nb * i for i in range(rows + 1)]),
             # distinct ids in a row: every (V // biases)-th, shifted
             bias_ids=((torch.arange(max(nb, 1), device="cuda") * (V // max(nb, 1)))[None, :]
                       + torch.randint(0, max(1, V // max(nb, 1)), (rows, 1), device="cuda",
                                       generator=r.g)).to(_I32).contiguous(),
             bias_values=r.normal(rows, max(nb, 1), std=4.0))
    if own:
        bmb = s["bmb"] = _bmb()
        s["type"] = bmb.ELEMENT_TYPES[c["type"]]
        p = {k: s[k].data_ptr() for k in ("tokens", "repetition", "frequency", "presence")}
        if nb:
            p.update({k: s[k].data_ptr() for k in ("bias_offsets", "bias_ids", "bias_values")})
            p.update(biases=nb * rows)
        if m:
            p.update(mask=s["mask"].data_ptr(), mask_index=s["mask_index"].data_ptr(),
                     mask_stride=words, masks=m)
        s["rules"] = bmb.LogitsRules(token_stride=width, lens=lens.data_ptr(),
                                     prompt_lens=prompts.data_ptr(), **p)


_PREPARE = dict(plan=_prepare_plan, append=_prepare_append, attend=_prepare_attend,
                logits=_prepare_logits)


# --------------------------------------------------------------------- runs
def run(s):
    op = s["c"]["op"]
    return (_OWN if own else _PLAIN)[op](s, s["c"])


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _plan_outputs(s):
    return (s["table"], s["ring"], s["lens_out"], s["state_out"], s["slots"], s["positions"],
            s["rows"], s["offsets"])


def _own_plan(s, c):
    s["bmb"].paged_plan(s["plan"], _stream())
    return _plan_outputs(s)


def _own_append(s, c):
    width, item = c["kv"] * c["hs"], _SIZE[c["type"]]
    qkv = s["qkv"].data_ptr()
    s["bmb"].paged_append(s["cache"], qkv + width * item, qkv + 2 * width * item, s["type"],
                          3 * width, s["slots"].data_ptr(), c["tokens"], _stream())
    return s["k_cache"], s["v_cache"]


def _own_attend(s, c):
    s["bmb"].paged_attention(s["cache"], s["batch"], s["out"].data_ptr(), s["lse"].data_ptr(),
                             s["qkv"].data_ptr(), _stream())
    return s["out"], s["lse"]


def _own_logits(s, c):
    s["bmb"].logits_process(s["out"].data_ptr(), s["logits"].data_ptr(), s["type"], c["rows"],
                            c["V"], c["V"], s["rules"], _stream())
    return s["out"]


def _plain_plan(s, c):
    R, P, T, pages, width = c["requests"], c["page"], s["T"], s["pages"], s["width"]
    lens, new = s["lens"].long(), s["new"].long()
    head, free = s["state"][0].long(), s["state"][1].long()
    have = (lens + P - 1) // P
    fits = (new > 0) & (lens + new <= width * P)
    need = torch.where(fits, (lens + new + P - 1) // P - have, 0)
    upto = torch.cumsum(need, 0)
    fits = fits & ((need == 0) | (upto <= free))
    fits = fits & (torch.cumsum(torch.where(fits, new, 0), 0) <= T)
    grant = torch.where(fits, new, 0)
    offsets = torch.cat([torch.zeros_like(grant[:1]), torch.cumsum(grant, 0)])
    gone = torch.where(new < 0, have, 0)
    s["offsets"].copy_(offsets)
    s["lens_out"].copy_(torch.where(new < 0, 0, lens + grant))
    s["rows"].copy_(torch.where(fits, offsets[1:] - 1, -1))
    taken = torch.where(fits, need, 0).sum()
    s["state_out"].copy_(torch.stack([(head + taken) % pages, free - taken + gone.sum()]))
    # every token of the step
    t = torch.arange(T, device="cuda")
    live = t < offsets[R]
    req = torch.searchsorted(offsets[1:], t, right=True).clamp_(max=R - 1)
    pos = lens[req] + t - offsets[req]
    j = torch.where(live, pos // P, 0)
    fresh = live & (j >= have[req])
    at = (head + (upto - need)[req] + j - have[req]) % pages
    page = torch.where(fresh, s["ring"][at], s["table"][req, j]).long()
    s["slots"].copy_(torch.where(live, page * P + pos % P, -1))
    s["positions"].copy_(torch.where(live, pos, 0))
    first = fresh & (pos % P == 0)
    s["table"][req[first], j[first]] = page[first].to(_I32)
    # pages of ended requests join the end of the ring
    col = torch.arange(width, device="cuda")[None, :]
    held = col < gone[:, None]
    freed = s["table"][held]
    s["ring"][(head + free + torch.arange(freed.numel(), device="cuda")) % pages] = freed
    return _plan_outputs(s)


def _by_token(cache, c):
    """(pages, page, kv, hs) view of a cache half."""
    return cache if c["layout"] == "token" else cache.permute(0, 2, 1, 3)


def _plain_append(s, c):
    n, kv, hs, P = c["tokens"], c["kv"], c["hs"], c["page"]
    slots = s["slots"].long()
    live = slots >= 0
    at = slots[live]
    rows = s["qkv"].view(n, 3, kv, hs)[live]
    for half, i in (("k_cache", 1), ("v_cache", 2)):
        _by_token(s[half], c)[at // P, at % P] = rows[:, i].to(_TYPES[c["cache"]])
    return s["k_cache"], s["v_cache"]


def _plain_attend(s, c):
    kv, hs, heads, P = c["kv"], c["hs"], c["heads"], c["page"]
    k_all, v_all = _by_token(s["k_cache"], c), _by_token(s["v_cache"], c)
    for i, (n, row) in enumerate(zip(s["host_lens"], s["host_rows"])):
        if row < 0:
            continue
        pages = s["table"][i, :_pages(n, P)].long()
        k = k_all[pages].reshape(-1, kv, hs)[:n].float().permute(1, 2, 0).contiguous()
        v = v_all[pages].reshape(-1, kv, hs)[:n].float().permute(1, 0, 2).contiguous()
        q = s["qkv"][row, :heads * hs].float().view(kv, heads // kv, hs)
        x = torch.matmul(q, k) * s["scale"]
        m = x.amax(2, keepdim=True)
        e = torch.exp(x - m)
        z = e.sum(2, keepdim=True)
        s["out"][row] = (torch.matmul(e, v) / z).view(-1).to(s["out"].dtype)
        s["lse"][row] = (m + torch.log(z)).view(-1)
    return s["out"], s["lse"]


def _plain_logits(s, c):
    rows, V = c["rows"], c["V"]
    ids, width = s["tokens"].long(), s["tokens"].shape[1]
    col = torch.arange(width, device="cuda")[None, :]
    held = (col < s["lens"][:, None]) & (ids >= 0) & (ids < V)
    safe = torch.where(held, ids, 0)
    seen = torch.zeros(rows, V, device="cuda", dtype=_I32)
    seen.scatter_add_(1, safe, held.to(_I32))
    made = torch.zeros(rows, V, device="cuda", dtype=_I32)
    made.scatter_add_(1, safe, (held & (col >= s["prompts"][:, None])).to(_I32))
    x = s["logits"].float()
    rep = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * made.float()
    x = x - s["presence"][:, None] * (made > 0).float()
    if c["biases"]:
        x.scatter_add_(1, s["bias_ids"].long(), s["bias_values"])
    v = torch.arange(V, device="cuda")
    index = s["mask_index"].long()
    words = s["mask"][index.clamp(min=0)][:, v // 32]
    allowed = ((words >> (v % 32)[None, :]) & 1).bool() | (index < 0)[:, None]
    s["out"].copy_(torch.where(allowed, x, -math.inf))
    return s["out"]


_OWN = dict(plan=_own_plan, append=_own_append, attend=_own_attend, logits=_own_logits)
_PLAIN = dict(plan=_plain_plan, append=_plain_append, attend=_plain_attend, logits=_plain_logits)


# --------------------------------------------------------------------- work
def work(case):
    c, op = case, case["op"]
    if op == "plan":
        z = _plan_sizes(c)
        R, P = c["requests"], c["page"]
        fresh = sum(_pages(h + n, P) - _pages(h, P) for h, n in zip(z["held"], z["new"]) if n > 0)
        gone = sum(_pages(h, P) for h, n in zip(z["held"], z["new"]) if n < 0)
        # lens, new and their results a request; slot and position a token; a page id read and
        # written a page
        return dict(bytes=4 * (6 * R + 2 * z["tokens"] + 2 * (fresh + gone)), flops=0)
    if op == "append":
        n = c["tokens"] * c["kv"] * c["hs"] * 2
        live = 1.0 - c["padded"]
        return dict(bytes=int(n * live * (_SIZE[c["type"]] + _SIZE[c["cache"]])) + 4 * c["tokens"],
                    flops=0)
    if op == "attend":
        keys = sum(n for n, idle in zip(_lens(c), _idle(c)) if not idle)
        held = sum(_pages(n, c["page"]) for n, idle in zip(_lens(c), _idle(c)) if not idle)
        live = sum(not i for i in _idle(c))
        return dict(bytes=keys * c["kv"] * c["hs"] * 2 * _SIZE[c["cache"]] + 4 * held
                    + live * c["heads"] * (2 * c["hs"] * _SIZE[c["type"]] + 4),
                    flops=4 * keys * c["heads"] * c["hs"])
    words, hist = (c["V"] + 31) // 32, sum(n for n, _ in _history(c))
    return dict(bytes=2 * c["rows"] * c["V"] * _SIZE[c["type"]] + 4 * hist
                + 4 * words * sum(_masked(c)) + 8 * c["rows"] * c["biases"],
                flops=4 * c["rows"] * c["V"])


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


def _exact_plan(s, c):
    """Request by request, on the host."""
    P, T, pages, width = c["page"], s["T"], s["pages"], s["width"]
    table, ring = s["table"].cpu().numpy().copy(), s["ring"].cpu().numpy().copy()
    lens, new = s["lens"].tolist(), s["new"].tolist()
    head, free = s["state"].tolist()
    slots, positions = np.full(T, -1, np.int32), np.zeros(T, np.int32)
    rows, offsets, after = [], [0], []
    asked, used, done, full = 0, 0, 0, False
    released = []
    for r, (h, n) in enumerate(zip(lens, new)):
        rows.append(-1)
        after.append(0 if n < 0 else h)
        if n < 0:
            released.extend(table[r, :_pages(h, P)].tolist())
        elif n > 0 and h + n <= width * P:
            have, want = _pages(h, P), _pages(h + n, P)
            asked += want - have
            if want == have or asked <= free:
                full = full or done + n > T
                if not full:
                    for j in range(have, want):
                        table[r, j] = ring[(head + used) % pages]
                        used += 1
                    p = np.arange(h, h + n)
                    positions[done:done + n] = p
                    slots[done:done + n] = table[r, p // P] * P + p % P
                    done += n
                    rows[-1], after[-1] = done - 1, h + n
        offsets.append(done)
    for i, page in enumerate(released):
        ring[(head + free + i) % pages] = page
    state = [(head + used) % pages, free - used + len(released)]
    whole = [table, ring, np.array(after), np.array(state), slots, positions, np.array(rows),
             np.array(offsets)]
    return tuple(torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda() for a in whole)


def _exact_append(s, c):
    n, kv, hs, P = c["tokens"], c["kv"], c["hs"], c["page"]
    slots = s["slots"].cpu().tolist()
    tokens = torch.tensor([t for t, x in enumerate(slots) if x >= 0], device="cuda")
    at = torch.tensor([x for x in slots if x >= 0], device="cuda")
    out = []
    for i, half in ((1, "k_cache"), (2, "v_cache")):
        whole = s[half].double()
        for h in range(kv):
            cols = slice((i * kv + h) * hs, (i * kv + h + 1) * hs)
            values = s["qkv"][:, cols].double()[tokens]
            if c["layout"] == "token":
                whole[:, :, h].index_put_((at // P, at % P), values)
            else:
                whole[:, h].index_put_((at // P, at % P), values)
        out.append(whole)
    return tuple(out)


def _exact_attend(s, c):
    kv, hs, heads, P = c["kv"], c["hs"], c["heads"], c["page"]
    group = heads // kv
    out, lse = s["out"].double(), s["lse"].double()
    for i, (n, row) in enumerate(zip(s["host_lens"], s["host_rows"])):
        if row < 0:
            continue
        key = torch.arange(n, device="cuda")
        page, at = s["table"][i].long()[key // P], key % P
        for h in range(kv):
            pick = (page, at, h) if c["layout"] == "token" else (page, h, at)
            k, v = s["k_cache"][pick].double(), s["v_cache"][pick].double()
            q = s["qkv"][row, h * group * hs:(h + 1) * group * hs].double().view(group, hs)
            x = (k @ q.t()) * s["scale"]
            z = torch.logsumexp(x, 0)
            lse[row, h * group:(h + 1) * group] = z
            out[row, h * group * hs:(h + 1) * group * hs] = (v.t() @ torch.exp(x - z)).t().reshape(-1)
    return out, lse


def _exact_logits(s, c):
    V = c["V"]
    out = s["logits"].double()
    words = s["mask"].cpu().numpy().view(np.uint32)
    index = s["mask_index"].tolist()
    for r, (n, prompt) in enumerate(_history(c)):
        x = out[r]
        made = torch.bincount(s["tokens"][r, prompt:n].long(), minlength=V).double()
        seen = torch.bincount(s["tokens"][r, :n].long(), minlength=V) > 0
        rep = s["repetition"][r].double()
        y = torch.where(x > 0, x / rep, x * rep)
        x = torch.where(seen, y, x) - s["frequency"][r].double() * made
        x = x - torch.where(made > 0, s["presence"][r].double(), 0.0)
        if c["biases"]:
            x[s["bias_ids"][r].long()] += s["bias_values"][r].double()
        if index[r] >= 0:
            bits = np.unpackbits(words[index[r]].view(np.uint8), bitorder="little")[:V]
            x[torch.from_numpy(bits == 0).cuda()] = -math.inf
        out[r] = x
    return out


_EXACT = dict(plan=_exact_plan, append=_exact_append, attend=_exact_attend, logits=_exact_logits)
