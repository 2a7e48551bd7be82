"""Tensors and calls shared by the GPU tests of the layer norm and the gated
linear recurrence.  Every tensor lies in a larger buffer filled with NaN
(inputs, so that a read outside shows) or with a sentinel (outputs, so that
a write outside shows)."""
import ctypes as C

import numpy as np
import torch

import kmamba_b200 as kb

SENTINEL = -77.0
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}  # output rounding: half a step of 8 bits
TINY = 1e-30


def typed(a, dtype):
    """float64 array -> the nearest values of dtype, as float64 (what the kernel is given)."""
    return torch.from_numpy(np.asarray(a)).to(dtype).double().numpy()


class Banded:
    """A [rows, D] or [batch, L, D] tensor inside a wider buffer."""

    def __init__(self, shape, dtype, fill, gap=0, shift=0, time_major=False):
        D, lead = shape[-1], 1
        for n in shape[:-1]:
            lead *= n
        self.ld = D + gap
        self.flat = torch.full((max(lead, 1) * self.ld + 64 + shift + 64,), fill, dtype=dtype, device="cuda")
        self.fill = fill
        if len(shape) == 3 and time_major:
            st = (self.ld, shape[0] * self.ld, 1)
        elif len(shape) == 3:
            st = (shape[1] * self.ld, self.ld, 1)
        else:
            st = (self.ld, 1)
        self.t = self.flat.as_strided(shape, st, 64 + shift)

    def set(self, a):
        self.t.copy_(torch.from_numpy(np.ascontiguousarray(a)).to(self.t.dtype))
        return self

    def np(self):
        return self.t.double().cpu().numpy()

    def untouched_outside(self):
        """Whether everything outside the view still holds the fill."""
        f = self.flat.clone()
        f.as_strided(self.t.shape, self.t.stride(), self.t.storage_offset()).fill_(self.fill)
        return bool((f == self.fill).all())

    def rows(self):
        st = self.t.stride()
        return kb.KmbRows(self.t.data_ptr(), st[-2], st[0] if self.t.dim() == 3 else 0)


def within(name, got, want, bound, dtype=torch.float32):
    """Every entry within its bound, plus half a step of the output type."""
    lim = bound + HALF[dtype] * (np.abs(want) + bound) + TINY
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert np.all(np.isfinite(got) == np.isfinite(want)), name
    if not got.size:
        return
    off = np.abs(got - want) - lim
    k = np.unravel_index(np.argmax(off), off.shape)
    assert off[k] <= 0, (name, k, got[k], want[k], lim[k])


def byref(a):
    return C.byref(a)
