"""Device buffers of rows for the tests of the operators around the paged cache."""
import numpy as np
import torch

import bmb

TYPES = {"f32": (bmb.F32, torch.float32), "f16": (bmb.F16, torch.float16),
         "bf16": (bmb.BF16, torch.bfloat16)}
U = 2.0 ** -24  # half a step of fp32
CANARY = 0x5A
SIDE = 64  # elements of canary on either side


def half_step(t):
    return torch.finfo(t).eps / 2


def smallest(t):
    """Half of the type's smallest positive number: what a result that small is off by."""
    return float(torch.finfo(t).smallest_normal) * torch.finfo(t).eps / 2


class Rows:
    """rows x width of a type, `stride` elements apart, canaries on both sides and between the
    rows, `skew` elements behind a multiple of 256 bytes."""

    def __init__(self, rows, width, dtype, stride=None, skew=0, values=None):
        self.rows, self.width, self.dtype = rows, width, dtype
        self.stride = width if stride is None else stride
        span = (rows - 1) * self.stride + width if rows else 0
        size = torch.empty(0, dtype=dtype).element_size()
        self.buf = torch.full(((SIDE * 2 + skew + span) * size,), CANARY, dtype=torch.uint8,
                              device="cuda")
        flat = self.buf.view(dtype)
        self.flat = flat
        self.at = SIDE + skew
        self.t = torch.as_strided(flat, (rows, width), (self.stride, 1), self.at)
        if values is not None:
            self.t.copy_(values)

    @property
    def ptr(self):
        return self.flat.data_ptr() + self.at * self.flat.element_size()

    def get(self):
        """The rows on the host."""
        torch.cuda.synchronize()
        return self.t.cpu()

    def holds(self, values):
        """The rows are `values` to the bit (NaN too)."""
        as_int = {1: torch.int8, 2: torch.int16, 4: torch.int32}[self.flat.element_size()]
        return torch.equal(self.get().contiguous().view(as_int), values.contiguous().view(as_int))

    def intact(self):
        """Nothing but the rows was written."""
        torch.cuda.synchronize()
        keep = torch.ones(self.flat.numel(), dtype=torch.bool, device="cuda")
        torch.as_strided(keep, (self.rows, self.width), (self.stride, 1), self.at).fill_(False)
        size = self.flat.element_size()
        rest = self.buf.view(-1, size)[keep]
        return bool((rest == CANARY).all())


def close(got, want, bound):
    """|got - want| <= bound, element by element, and NaN and infinities where they belong; the
    message names the worst place."""
    got, want, bound = got.double(), want.double(), torch.as_tensor(bound).double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    over = torch.where(fine, (got - want).abs() - bound, torch.zeros_like(want))
    worst = int(over.reshape(-1).argmax()) if over.numel() else 0
    assert not (over > 0).any(), (
        np.unravel_index(worst, tuple(over.shape)), got.reshape(-1)[worst].item(),
        want.reshape(-1)[worst].item(), int((over > 0).sum()))
