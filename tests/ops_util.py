"""Device buffers for the operators' tests: every matrix sits in a larger allocation filled with a pattern, so that a write
next to it shows."""
import numpy as np
import torch

import hcomm_amd as h
import ops_reference as ref

TORCH = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DT = {"bf16": h.HcommDataType.BFP16, "fp16": h.HcommDataType.FP16, "fp32": h.HcommDataType.FP32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
GUARD = 0xA5


class Dense:
    """rows x cols of a type at an element offset, `stride` elements from row to row."""

    def __init__(self, rows, cols, t, stride=None, offset=0, values=None):
        self.rows, self.cols, self.t = rows, cols, t
        self.stride = cols if stride is None else stride
        n = offset + max(rows - 1, 0) * self.stride + cols + 64
        self.raw = torch.full((n * SIZE[t],), GUARD, dtype=torch.uint8, device="cuda")
        self.all = self.raw.view(TORCH[t])
        self.view = torch.as_strided(self.all, (rows, cols), (self.stride, 1), offset)
        if values is not None:
            self.view.copy_(torch.as_tensor(values).to(TORCH[t]).reshape(rows, cols))
        self.ptr = self.all.data_ptr() + offset * SIZE[t]

    def double(self):
        return self.view.double().cpu().numpy()

    def guards_hold(self):
        """Everything outside the rows x cols elements is as it was."""
        keep = torch.ones(self.all.shape, dtype=torch.bool, device="cuda")
        torch.as_strided(keep, (self.rows, self.cols), (self.stride, 1), (self.ptr - self.all.data_ptr()) // SIZE[self.t]).fill_(False)
        return bool((self.raw.view(-1, SIZE[self.t])[keep] == GUARD).all())


class Mx:
    """A matrix in the 4-bit format; `pad`: extra blocks and scale bytes from row to row, `shift`: where the scales begin."""

    def __init__(self, rows, cols, pad=0, shift=0, code=None, scale=None):
        self.rows, self.cols, self.nb = rows, cols, ref.blocks_of(cols)
        self.ps, self.ss = (self.nb + pad) * 16, self.nb + pad
        self.packed = torch.full((rows * self.ps + 64,), GUARD, dtype=torch.uint8, device="cuda")
        self.scales = torch.full((rows * self.ss + 64 + shift,), GUARD, dtype=torch.uint8, device="cuda")
        self.shift = shift
        if code is not None:
            self._blocks().copy_(torch.from_numpy(ref.mx_pack(code)))
            self._scales().copy_(torch.from_numpy(scale))
        self.item = (self.packed.data_ptr(), self.ps, self.scales.data_ptr() + shift, self.ss)

    def _blocks(self):
        return torch.as_strided(self.packed, (self.rows, self.nb, 16), (self.ps, 16, 1))

    def _scales(self):
        return torch.as_strided(self.scales, (self.rows, self.nb), (self.ss, 1), self.shift)

    def code(self):
        return ref.mx_unpack(self._blocks().cpu().numpy())

    def scale(self):
        return self._scales().cpu().numpy()

    def values(self):
        return ref.mx_values(self.code(), self.scale(), self.cols)

    def guards_hold(self):
        p, s = self.packed.clone(), self.scales.clone()
        torch.as_strided(p, (self.rows, self.nb, 16), (self.ps, 16, 1)).fill_(GUARD)
        torch.as_strided(s, (self.rows, self.nb), (self.ss, 1), self.shift).fill_(GUARD)
        return bool((p == GUARD).all()) and bool((s == GUARD).all())


def random_mx(rows, cols, rng, pad=0, shift=0, spread=6, unit=0, tail=None):
    """Random elements under scales 2^(unit - 127 + 0..spread); `tail`: what the last block holds past cols (0 by default)."""
    nb = ref.blocks_of(cols)
    code = rng.integers(0, 16, (rows, nb, 32)).astype(np.uint8)
    scale = rng.integers(unit, unit + spread + 1, (rows, nb)).astype(np.uint8)
    if cols % 32:
        code[:, -1, cols % 32:] = 0 if tail is None else tail
    return Mx(rows, cols, pad, shift, code, scale)


def close(got, want, t, slack, what):
    """|got - want| <= slack (an absolute bound for each element, computed in 64 bits) + the output's own rounding."""
    smallest = {"bf16": 2.0 ** -133, "fp16": 2.0 ** -24, "fp32": 2.0 ** -149}[t] / 2
    bound = slack + (np.abs(want) + slack) * ref.EPS_HALF[t] + smallest
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), "%s: %d of %d off, first %r: got %r want %r bound %r" % (
        what, bad.sum(), bad.size, tuple(np.argwhere(bad)[0]), got[bad][0], want[bad][0], np.broadcast_to(bound, got.shape)[bad][0])
