"""Paged-cache problems on the host, their exact answers in fp64, and the
library's calls on them, for the tests of the generation operators."""
import math

import numpy as np
import torch

import bmb

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U32 = 2.0 ** -24


def pages_of(tokens, page):
    return -(-tokens // page)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Problem:
    """A cache with `lens` tokens a request, its pages in a random order, every
    other place (behind a request's end, in pages of nobody) NaN or infinite,
    and queries in fused rows. All on the host; `device()` uploads."""

    def __init__(self, lens, heads, kv, hs, type, cache, page, layout="token", seed=0,
                 rows=None, scale=None, spread=1.0, extra_columns=1):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.heads, self.kv, self.hs, self.page = list(lens), heads, kv, hs, page
        self.type, self.cache, self.layout = type, cache, layout
        R = len(self.lens)
        held = [pages_of(n, page) for n in self.lens]
        self.pages = sum(held) + 3
        width = max(held) + extra_columns
        order = torch.randperm(self.pages, generator=g).tolist()
        self.table = torch.full((R, width), -7, dtype=torch.int32)
        at = 0
        for r, n in enumerate(held):
            for j in range(n):
                self.table[r, j] = order[at]
                at += 1
        shape = (self.pages, page, kv, hs)
        junk = torch.where(torch.rand(shape, generator=g) < 0.5, math.nan, math.inf)
        self.k, self.v = junk.to(DTYPES[cache]), junk.neg().to(DTYPES[cache])
        for r, n in enumerate(self.lens):
            t = torch.arange(n)
            at = (self.table[r].long()[t // page], t % page)
            self.k[at] = torch.randn(n, kv, hs, generator=g).to(DTYPES[cache])
            self.v[at] = torch.randn(n, kv, hs, generator=g).to(DTYPES[cache])
        self.n_rows = R
        self.rows = rows
        if rows is not None:
            self.n_rows = max([x for x in rows] + [0]) + 2
        self.q_stride = (heads + 2 * kv) * hs
        self.q = (torch.randn(self.n_rows, self.q_stride, generator=g) * spread).to(DTYPES[type])
        self.scale = 1.0 / math.sqrt(hs) if scale is None else scale

    def tokens(self, r, half):
        """(len, kv, hs) of request r in fp64."""
        n = self.lens[r]
        t = np.arange(n)
        return half[self.table[r].long()[t // self.page], t % self.page].double()

    def row(self, r):
        row = r if self.rows is None else self.rows[r]
        return row if 0 <= row < self.n_rows else -1

    def exact(self):
        """{row: (out (heads, hs), lse (heads), bound of out, bound of lse)}.

        The bounds count the roundings of the computation. Scores: fp32 sums of
        exact products (random-walk model, 4 sqrt(n) 2^-24 of the sum of their
        magnitudes, as for the fp32 GEMMs), then three roundings of the scaled
        score. A probability moves by twice the scores' error; the sum over the
        keys adds the same model's 4 sqrt(n) 2^-24, the weights of up to 64
        joined parts and the final division a few more. With a 16-bit cache
        and queries the probabilities enter as two 16-bit roundings: 2^-16
        (bf16) or 2^-21 (fp16) of each, and what fp16 cannot hold, 2^-25 of the
        largest. At the end half a step of the output's type."""
        res = {}
        half_step = torch.finfo(DTYPES[self.type]).eps / 2
        for r, n in enumerate(self.lens):
            row = self.row(r)
            if row < 0:
                continue
            G = self.heads // self.kv
            q = self.q[row, :self.heads * self.hs].double().view(self.kv, G, self.hs)
            k, v = self.tokens(r, self.k).permute(1, 0, 2), self.tokens(r, self.v).permute(1, 0, 2)
            if n == 0:
                z = torch.zeros(self.heads, self.hs, dtype=torch.float64)
                res[row] = (z, torch.full((self.heads,), -math.inf, dtype=torch.float64), z,
                            torch.zeros(self.heads, dtype=torch.float64))
                continue
            x = torch.matmul(q, k.transpose(1, 2)) * self.scale
            mag = (torch.matmul(q.abs(), k.abs().transpose(1, 2)) * abs(self.scale)).amax(2)
            lse = torch.logsumexp(x, 2)
            p = torch.exp(x - lse[:, :, None])
            out = torch.matmul(p, v)
            ds = 4 * (math.sqrt(self.hs) + 1) * U32 * mag + 4 * U32 * x.abs().amax(2)
            eps = 2 * ds + (4 * math.sqrt(n) + 16) * U32
            weight = torch.matmul(p, v.abs())
            extra = 0.0
            if self.type != "f32":
                eps = eps + (2.0 ** -16 if self.type == "bf16" else 2.0 ** -21)
                if self.type == "f16":
                    extra = 2.0 ** -25 * v.abs().sum(1)[:, None, :]
            bound = eps[:, :, None] * weight + extra + half_step * out.abs() + 1e-37
            if self.type == "f16":
                bound = bound + 2.0 ** -25  # subnormal outputs
            lse_bound = ds + (4 * math.sqrt(n) + 16) * U32 + 4 * U32 * lse.abs()
            res[row] = (out.reshape(self.heads, self.hs), lse.reshape(-1),
                        bound.reshape(self.heads, self.hs), lse_bound.reshape(-1))
        return res

    def device(self):
        return DeviceProblem(self)


def cache_struct(k, v, layout, page, kv, hs, cache):
    """PagedCache of device halves laid out (pages, page, kv, hs) ("token") or
    (pages, kv, page, hs) ("head")."""
    token, head = (kv * hs, hs) if layout == "token" else (hs, page * hs)
    return bmb.PagedCache(k=k.data_ptr(), v=v.data_ptr(), type=bmb.ELEMENT_TYPES[cache],
                          pages=k.shape[0], page_size=page, kv_heads=kv, head_size=hs,
                          page_stride=page * kv * hs, token_stride=token, head_stride=head)


class DeviceProblem:
    def __init__(self, p):
        self.p = p
        self.k, self.v = (x.permute(0, 2, 1, 3).contiguous().cuda() if p.layout == "head"
                          else x.cuda() for x in (p.k, p.v))
        self.table, self.lens = p.table.cuda(), ints(p.lens)
        self.rows = None if p.rows is None else ints(p.rows)
        self.q = p.q.cuda()
        W = p.heads * p.hs
        self.out_stride = W + 6  # rows apart by more than they hold
        self.out = torch.full((p.n_rows, self.out_stride), 768.0, device="cuda",
                              dtype=DTYPES[p.type])
        self.lse = torch.full((p.n_rows, p.heads), 768.0, device="cuda")
        self.cache = cache_struct(self.k, self.v, p.layout, p.page, p.kv, p.hs, p.cache)
        self.batch = bmb.PagedBatch(
            requests=len(p.lens), max_len=max(max(p.lens), 0), table_stride=p.table.shape[1],
            heads=p.heads, n_rows=p.n_rows, type=bmb.ELEMENT_TYPES[p.type], scale=p.scale,
            q_stride=p.q_stride, out_stride=self.out_stride, block_table=self.table.data_ptr(),
            lens=self.lens.data_ptr(), rows=None if self.rows is None else self.rows.data_ptr())
        self.work = None

    def workspace(self):
        need = bmb.paged_attention_workspace(self.cache, self.batch)
        # the last bytes are a canary
        self.work = torch.full((need + 64,), 0x5A, device="cuda", dtype=torch.uint8)
        self.batch.work, self.batch.work_bytes = self.work.data_ptr(), need
        return need

    def run(self, stream=0):
        bmb.paged_attention(self.cache, self.batch, self.out.data_ptr(), self.lse.data_ptr(),
                            self.q.data_ptr(), stream)

    def check(self):
        """Results within the bounds; every other place as it was."""
        p = self.p
        torch.cuda.synchronize()
        bmb.check("paged_attention")
        out, lse = self.out.cpu().double(), self.lse.cpu().double()
        W = p.heads * p.hs
        assert (out[:, W:] == 768.0).all()
        exact = p.exact()
        worst = 0.0
        for row in range(p.n_rows):
            if row not in exact:
                assert (out[row] == 768.0).all() and (lse[row] == 768.0).all(), row
                continue
            o, z, ob, zb = exact[row]
            got = out[row, :W].view(p.heads, p.hs)
            bad = ~((got - o).abs() <= ob)
            assert not bad.any(), (row, bad.nonzero()[:4].tolist(), got[bad][:4], o[bad][:4],
                                   ob[bad][:4])
            same = (lse[row] == z) | ((lse[row] - z).abs() <= zb)
            assert same.all(), (row, lse[row], z, zb)
            worst = max(worst, float(((got - o).abs() / (ob + 1e-300)).max()))
        if self.work is not None:
            assert (self.work[-64:] == 0x5A).all()
        return worst


def plan_exact(table, lens, new, ring, state, page, max_tokens):
    """paged_plan request by request; numpy int arrays in, all results out."""
    R, width = table.shape
    table, ring = table.copy(), ring.copy()
    pages = len(ring)
    head, count = int(state[0]), int(state[1])
    slots, pos = np.full(max_tokens, -1, np.int32), np.zeros(max_tokens, np.int32)
    rows, offsets, after = np.full(R, -1, np.int32), np.zeros(R + 1, np.int32), np.array(lens)
    asked = used = tokens = brought = 0
    released = []
    for r in range(R):
        h, n = int(lens[r]), int(new[r])
        if n < 0:
            released += [int(x) for x in table[r, :pages_of(h, page)]]
            after[r] = 0
        elif n > 0 and h + n <= width * page:
            have, want = pages_of(h, page), pages_of(h + n, page)
            asked += want - have
            if want == have or asked <= count:
                brought += n
                if brought <= max_tokens:
                    for j in range(have, want):
                        table[r, j] = ring[(head + used) % pages]
                        used += 1
                    for t in range(h, h + n):
                        slots[tokens] = table[r, t // page] * page + t % page
                        pos[tokens] = t
                        tokens += 1
                    rows[r], after[r] = tokens - 1, h + n
        offsets[r + 1] = tokens
    for i, x in enumerate(released):
        ring[(head + count + i) % pages] = x
    out = np.array([(head + used) % pages, count - used + len(released)], np.int32)
    return dict(block_table=table, free_pages=ring, lens_out=after, state_out=out, slots=slots,
                positions=pos, rows=rows, offsets=offsets)


class Pool:
    """Device state of paged_plan with its host copy; in place or not."""

    def __init__(self, lens, page, width, free, seed=0):
        r = np.random.default_rng(seed)
        held = [pages_of(n, page) for n in lens]
        self.page, self.R = page, len(lens)
        self.pages = sum(held) + free
        order = r.permutation(self.pages).astype(np.int32)
        self.table = np.full((self.R, width), -3, np.int32)
        at = 0
        for i, n in enumerate(held):
            self.table[i, :n] = order[at:at + n]
            at += n
        head = int(r.integers(0, self.pages)) if self.pages else 0
        self.ring = np.full(max(self.pages, 1), -5, np.int32)
        self.ring[(head + np.arange(free)) % max(self.pages, 1)] = order[at:]
        self.state, self.lens = np.array([head, free], np.int32), np.array(lens, np.int32)
        self.d = {k: torch.from_numpy(getattr(self, k)).cuda()
                  for k in ("table", "ring", "state", "lens")}

    def step(self, new, max_tokens, in_place=True, stream=0):
        """Runs paged_plan, checks every result against plan_exact, and takes
        them over as the next state. Returns the device results."""
        d, R = self.d, self.R
        new = np.array(new, np.int32)
        want = plan_exact(self.table, self.lens, new, self.ring, self.state, self.page, max_tokens)

        def buf(n):
            return torch.full((n + 16,), 4242, device="cuda", dtype=torch.int32)

        o = dict(slots=buf(max_tokens), positions=buf(max_tokens), rows=buf(R), offsets=buf(R + 1))
        o["lens_out"] = d["lens"] if in_place else buf(R)
        o["state_out"] = d["state"] if in_place else buf(2)
        d_new = torch.from_numpy(new).cuda()
        plan = bmb.PagedPlan(requests=R, max_pages=self.table.shape[1], pages=self.pages,
                             page_size=self.page, max_tokens=max_tokens,
                             new_tokens=d_new.data_ptr(), lens=d["lens"].data_ptr(),
                             state=d["state"].data_ptr(), free_pages=d["ring"].data_ptr(),
                             block_table=d["table"].data_ptr(),
                             **{k: t.data_ptr() for k, t in o.items()})
        bmb.paged_plan(plan, stream)
        torch.cuda.synchronize()
        bmb.check("paged_plan")
        got = dict(o, block_table=d["table"], free_pages=d["ring"])
        for name, w in want.items():
            x = got[name].cpu().numpy()
            assert np.array_equal(x.reshape(-1)[:w.size], w.reshape(-1)), (name, x, w)
            assert (x.reshape(-1)[w.size:] == 4242).all(), name
        self.table, self.ring = want["block_table"], want["free_pages"]
        self.lens, self.state = want["lens_out"], want["state_out"]
        d["lens"], d["state"] = o["lens_out"][:R], o["state_out"][:2]
        o["new"] = d_new
        return o
