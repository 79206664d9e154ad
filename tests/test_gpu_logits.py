"""logits_process (include/nn.h) on the GPU against a host computation in fp64.

Bar: each of the up to four fp32 operations rounds once (2^-24 of what it
gives), the result once to its type (half a step, eps / 2, or half a subnormal
step). Masked places, and places no rule touches, are equal."""
import math

import numpy as np
import pytest
import torch

import bmb

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


class Case:
    def __init__(self, rows, V, type, stride=None, hist=40, biases=5, seed=0, shift=0):
        r = np.random.default_rng(seed)
        self.rows, self.V, self.type, self.shift = rows, V, type, shift
        self.stride = stride or V
        x = torch.from_numpy(r.standard_normal((rows, self.stride)) * 4).to(DTYPES[type])
        x[0, min(V - 1, 2)], x[0, 0] = math.inf, -math.inf
        if V > 3:
            x[-1, 3] = math.nan
        self.x = x
        self.tokens = r.integers(0, V, (rows, hist))
        self.tokens[:, ::7] = self.tokens[:, :1]           # a repeated id
        if hist > 2:
            self.tokens[:, 1], self.tokens[:, 2] = -1, V   # ids outside the vocabulary
        self.lens = r.integers(0, hist + 1, rows)
        self.prompts = (self.lens * r.random(rows)).astype(int)
        if rows > 2:
            self.lens[1], self.prompts[2] = hist + 100, hist + 5
        self.rep = 1 + r.random(rows).astype(np.float32)
        self.freq, self.pres = (r.random(rows).astype(np.float32) for _ in range(2))
        counts = r.integers(0, biases + 1, rows) if biases else np.zeros(rows, int)
        self.offsets = np.concatenate([[0], np.cumsum(counts)])
        n = int(self.offsets[-1])
        self.bias_ids = r.integers(-2, V + 2, max(n, 1))
        if n > 1:
            self.bias_ids[1] = self.bias_ids[0]            # the last entry counts
        self.bias = (r.standard_normal(max(n, 1)) * 5).astype(np.float32)
        self.words = (V + 31) // 32 + 1
        self.masks = 3
        self.mask = r.integers(0, 1 << 32, (self.masks, self.words),
                               dtype=np.uint64).astype(np.uint32)
        self.mask[1] = 0                                   # nothing is allowed
        self.index = r.integers(-1, self.masks + 1, rows)
        if rows > 3:
            self.index[:4] = [0, 1, -1, 2]

    def exact(self, penalties, biases, masks):
        x = self.x[:, :self.V].double().numpy().copy()
        tol = np.zeros_like(x)
        u = 2.0 ** -24
        for r in range(self.rows):
            n = min(max(int(self.lens[r]), 0), self.tokens.shape[1])
            t = self.tokens[r, :n]
            if penalties:
                ok = (t >= 0) & (t < self.V)
                seen = np.unique(t[ok])
                first = max(int(self.prompts[r]), 0)
                out = t[first:][ok[first:]]
                made = np.bincount(out, minlength=self.V)
                for i in seen:
                    rep = float(self.rep[r])
                    x[r, i] = x[r, i] / rep if x[r, i] > 0 else x[r, i] * rep
                    tol[r, i] += u * abs(x[r, i])
                    if made[i]:
                        f = float(self.freq[r]) * made[i]
                        x[r, i] -= f
                        tol[r, i] += u * (abs(f) + abs(x[r, i]))
                        x[r, i] -= float(self.pres[r])
                        tol[r, i] += u * abs(x[r, i])
            if biases:
                last = {}
                for e in range(self.offsets[r], self.offsets[r + 1]):
                    if 0 <= self.bias_ids[e] < self.V:
                        last[int(self.bias_ids[e])] = float(self.bias[e])
                for i, b in last.items():
                    x[r, i] += b
                    tol[r, i] += u * abs(x[r, i])
            if masks and 0 <= self.index[r] < self.masks:
                bits = np.unpackbits(self.mask[self.index[r]].view(np.uint8),
                                     bitorder="little")[:self.V]
                x[r, bits == 0] = -math.inf
                tol[r, bits == 0] = 0
        return x, tol

    def run(self, penalties=True, biases=True, masks=True, in_place=False, stream=0):
        rows, V = self.rows, self.V
        t = DTYPES[self.type]
        # `shift` elements off 16-byte alignment, a canary behind
        n = rows * self.stride
        self.inp = torch.empty(n + self.shift, dtype=t, device="cuda")
        self.inp[self.shift:] = self.x.reshape(-1).cuda()
        src = self.inp[self.shift:]
        if in_place:
            self.out, dst = self.inp, src
        else:
            self.out = torch.full((n + 24,), 55.0, dtype=t, device="cuda")
            dst = self.out[:n]
        self.keep = [i32(self.tokens), i32(self.lens), i32(self.prompts),
                     torch.from_numpy(self.rep).cuda(), torch.from_numpy(self.freq).cuda(),
                     torch.from_numpy(self.pres).cuda(), i32(self.offsets), i32(self.bias_ids),
                     torch.from_numpy(self.bias).cuda(),
                     torch.from_numpy(self.mask.view(np.int32)).cuda(), i32(self.index)]
        p = [k.data_ptr() for k in self.keep]
        f = {}
        if penalties:
            f.update(tokens=p[0], token_stride=self.tokens.shape[1], lens=p[1], prompt_lens=p[2],
                     repetition=p[3], frequency=p[4], presence=p[5])
        if biases:
            f.update(bias_offsets=p[6], bias_ids=p[7], bias_values=p[8],
                     biases=int(self.offsets[-1]))
        if masks:
            f.update(mask=p[9], masks=self.masks, mask_stride=self.words, mask_index=p[10])
        self.rules = bmb.LogitsRules(**f)
        self.args = (dst.data_ptr(), src.data_ptr(), bmb.ELEMENT_TYPES[self.type], rows, V,
                     self.stride, self.rules)
        bmb.logits_process(*self.args, stream)
        torch.cuda.synchronize()
        bmb.check("logits_process")
        self.dst = dst
        if not in_place:
            assert (self.out[n:] == 55.0).all()
            pad = dst.view(rows, self.stride)[:, V:]
            assert (pad == 55.0).all()
        else:
            pad = dst.view(rows, self.stride)[:, V:].cpu()
            assert torch.equal(pad, self.x[:, V:])
        self.check(penalties, biases, masks)

    def check(self, penalties, biases, masks):
        got = self.dst.view(self.rows, self.stride)[:, :self.V].cpu().double().numpy()
        want, tol = self.exact(penalties, biases, masks)
        f = torch.finfo(DTYPES[self.type])
        step = f.eps / 2 * np.abs(want) + (f.tiny * f.eps / 2 if self.type != "f32" else 0)
        tol = tol + np.where(tol > 0, step, 0)  # what no rule touched is equal
        with np.errstate(invalid="ignore"):
            same = (got == want) | (np.isnan(got) & np.isnan(want)) | (np.abs(got - want) <= tol)
        assert same.all(), (np.argwhere(~same)[:4], got[~same][:4], want[~same][:4])


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,V,stride", [(1, 1, None), (5, 65, 128), (4, 4095, None),
                                           (3, 4096, 4096),
                                           (4, 4097, 4100), (6, 50257, None), (5, 50257, 50304),
                                           (3, 12289, 12291), (70, 33, 33),
                                           # results past 32 MB, and just below
                                           (340, 50257, None), (160, 50257, 50259)])
def test_logits(gpu, type, rows, V, stride):
    print("logits", type, rows, V, stride, flush=True)
    Case(rows, V, type, stride, seed=V).run()


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("penalties", [False, True])
@pytest.mark.parametrize("biases", [False, True])
@pytest.mark.parametrize("masks", [False, True])
def test_logits_each_rule(gpu, type, penalties, biases, masks):
    for in_place in (False, True):
        Case(5, 5003, type, 5005, seed=3).run(penalties, biases, masks, in_place)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shift", [1, 2, 3, 7])
def test_logits_alignment(gpu, type, shift):
    """Input and output rows that start at different places of 16 bytes."""
    Case(4, 9001, type, 9001, seed=shift, shift=shift).run()


@pytest.mark.parametrize("hist,biases", [(1, 0), (1, 1), (3000, 500), (70001, 3)])
def test_logits_history(gpu, hist, biases):
    Case(3, 20011, "f32", None, hist=hist, biases=biases, seed=hist).run()


def test_logits_clipped_device_values(gpu):
    """Negative lengths, offsets outside the list."""
    c = Case(4, 500, "f32", seed=5)
    c.lens[:] = [-3, 10, -1, 0]
    c.prompts[:] = [0, -5, 2, 0]
    c.run()
    off = i32([-4, 2, 1, 1 << 30, 3])
    c.rules.bias_offsets = off.data_ptr()
    bmb.logits_process(*c.args)
    torch.cuda.synchronize()
    bmb.check("logits_process")


def test_logits_clipped_bias_offsets(gpu):
    """Offsets outside the list are read as its ends, and a range that ends before
    it begins is empty."""
    c = Case(6, 500, "f32", biases=0, seed=6)
    n = 40
    c.bias_ids = (np.arange(n) * 11) % 250  # each a few times: the last entry counts
    c.bias = (np.arange(n) + 1).astype(np.float32)
    c.offsets = np.array([0, 0, 0, 0, 0, 0, n])
    c.run()
    given = [-4, 7, 3, -1, 1 << 30, 25, n + 1]
    clipped = [min(max(x, 0), n) for x in given]
    off = i32(given)
    c.rules.bias_offsets = off.data_ptr()
    bmb.logits_process(*c.args)
    torch.cuda.synchronize()
    bmb.check("logits_process")
    got = c.dst.view(c.rows, c.stride)[:, :c.V].cpu()
    for r in range(c.rows):
        b, e = clipped[r], clipped[r + 1]
        assert (b < e) == (r in (0, 3, 5))
        c.offsets = np.zeros(c.rows + 1, int)  # of row r alone
        c.offsets[r], c.offsets[r + 1] = b, max(b, e)
        want, tol = c.exact(True, True, True)
        with np.errstate(invalid="ignore"):
            x = got[r].double().numpy()
            same = (x == want[r]) | (np.isnan(x) & np.isnan(want[r])) | (
                np.abs(x - want[r]) <= tol[r] + 2.0 ** -24 * np.abs(want[r]) * (tol[r] > 0))
        assert same.all(), (r, np.argwhere(~same)[:4])


def test_logits_offsets_past_32_bits(gpu):
    """Rows that start more than 2^31 elements into the buffers."""
    V, rows = 1 << 20, 2080
    x = torch.zeros(rows, V, dtype=torch.float16, device="cuda")
    x[-1] = 2.0
    out = torch.zeros_like(x)
    tok = torch.full((rows, 1), V - 1, dtype=torch.int32, device="cuda")
    lens, rep = i32([1] * rows), torch.full((rows,), 2.0, device="cuda")
    rules = bmb.LogitsRules(tokens=tok.data_ptr(), token_stride=1, lens=lens.data_ptr(),
                            repetition=rep.data_ptr())
    bmb.logits_process(out.data_ptr(), x.data_ptr(), bmb.F16, rows, V, V, rules)
    torch.cuda.synchronize()
    bmb.check("logits_process")
    assert (out[-1, :-1] == 2.0).all() and out[-1, -1] == 1.0 and (out[:-1] == 0).all()


def test_logits_rows_of_several_launches(gpu):
    """More rows than one dispatch has lanes for: every row follows its rules."""
    rows, V = (1 << 24) + 5, 65
    x = torch.full((rows, V), 4.0, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros_like(x)
    row = torch.arange(rows, device="cuda")
    tok = (row * 7 % V).to(torch.int32)
    lens = torch.ones(rows, dtype=torch.int32, device="cuda")
    rep = (1 + row % 2).float()                                   # 1 or 2
    offsets = torch.arange(rows + 1, device="cuda", dtype=torch.int32)
    ids, values = ((tok + 1) % V).to(torch.int32), (row % 5).float()
    words = torch.tensor([~(1 << 3), -1, -1], dtype=torch.int32, device="cuda")
    index = torch.where(row % 3 == 0, 0, -1).to(torch.int32)
    rules = bmb.LogitsRules(tokens=tok.data_ptr(), token_stride=1, lens=lens.data_ptr(),
                            repetition=rep.data_ptr(), bias_offsets=offsets.data_ptr(),
                            bias_ids=ids.data_ptr(), bias_values=values.data_ptr(), biases=rows,
                            mask=words.data_ptr(), masks=1, mask_stride=3,
                            mask_index=index.data_ptr())
    bmb.logits_process(out.data_ptr(), x.data_ptr(), bmb.BF16, rows, V, V, rules)
    torch.cuda.synchronize()
    bmb.check("logits_process")
    x.scatter_(1, tok[:, None].long(), (4.0 / rep).to(x.dtype)[:, None])
    x.scatter_add_(1, ids[:, None].long(), values.to(x.dtype)[:, None])
    x[:, 3] = torch.where(row % 3 == 0, -math.inf, x[:, 3])
    assert torch.equal(out, x)


def test_logits_longest_history(gpu):
    """2^31 - 1 tokens, the most that a length can say, the last two of them the
    only ones of the vocabulary."""
    n, V = (1 << 31) - 1, 70
    tokens = torch.full((1, n), -1, dtype=torch.int32, device="cuda")
    tokens[0, -2:] = ints = i32([7, 69])
    x = torch.full((1, V), 8.0, device="cuda")
    out = torch.zeros_like(x)
    lens, prompt = i32([n]), i32([n - 1])
    rep, freq = torch.full((1,), 2.0, device="cuda"), torch.full((1,), 0.5, device="cuda")
    rules = bmb.LogitsRules(tokens=tokens.data_ptr(), token_stride=n, lens=lens.data_ptr(),
                            prompt_lens=prompt.data_ptr(), repetition=rep.data_ptr(),
                            frequency=freq.data_ptr())
    bmb.logits_process(out.data_ptr(), x.data_ptr(), bmb.F32, 1, V, V, rules)
    torch.cuda.synchronize()
    bmb.check("logits_process")
    x[0, ints.long()] = torch.tensor([4.0, 3.5], device="cuda")
    assert torch.equal(out, x)


def test_logits_biases_at_the_largest_offsets(gpu):
    """A row's entries at the end of a list of 2^31 - 1, of which only they exist."""
    n, V = 700, 90
    b1 = (1 << 31) - 1
    b0 = b1 - n
    ids = torch.arange(n, device="cuda", dtype=torch.int32) % 100
    values = torch.arange(n, device="cuda").float()
    offsets = i32([b0, b1])
    x, out = torch.zeros(1, V, device="cuda"), torch.ones(1, V, device="cuda")
    rules = bmb.LogitsRules(bias_offsets=offsets.data_ptr(), bias_ids=ids.data_ptr() - 4 * b0,
                            bias_values=values.data_ptr() - 4 * b0, biases=b1)
    bmb.logits_process(out.data_ptr(), x.data_ptr(), bmb.F32, 1, V, V, rules)
    torch.cuda.synchronize()
    bmb.check("logits_process")
    assert out[0].tolist() == [600.0 + i for i in range(V)]  # the last entry of each id


def test_logits_captured(gpu):
    """Captured on a side stream and replayed on changed inputs."""
    c = Case(8, 5003, "bf16", None, seed=9)
    c.run()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        bmb.logits_process(*c.args, side.cuda_stream)
    for i in range(3):
        c.x = torch.randn(8, 5003).to(torch.bfloat16)
        c.inp.copy_(c.x.reshape(-1))
        c.lens = np.minimum(c.lens + i, 40)
        c.keep[1].copy_(i32(c.lens))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        c.check(True, True, True)
