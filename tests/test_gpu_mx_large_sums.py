"""Folds whose sums pass the range of their results: what is quantised again, and what the dense results become."""
import numpy as np
import pytest
import torch

import hcomm_amd as h
import ops_reference as ref
from ops_util import DT, Dense, Mx, close, random_mx

pytestmark = pytest.mark.gpu

# half a step above a type's largest number: from here on a result is infinite
INFINITE_FROM = {"fp32": (2 - 2.0 ** -24) * 2.0 ** 127, "bf16": (2 - 2.0 ** -8) * 2.0 ** 127, "fp16": (2 - 2.0 ** -11) * 2.0 ** 15}


def fold(thread, t, src, addend, rows, cols):
    dst, again = Dense(rows, cols, t), Mx(rows, cols, 1, 1)
    torch.cuda.synchronize()
    h.check(h.HcommGfxMxReduceKOnThread(
        thread, dst.ptr, cols, DT[t], h.mx_views([again.item]), h.mx_views([x.item for x in src]), len(src),
        addend.ptr if addend else None, cols, rows, cols))
    h.check(h.HcommGfxThreadSynchronize(thread))
    v = addend.double() if addend else np.zeros((rows, cols))
    for x in src:
        v = v + x.values()
    return dst, again, v


@pytest.mark.parametrize("t", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("k,with_addend", [(2, False), (8, False), (1, True), (8, True), (9, False), (32, True)])
def test_sums_past_fp32_are_quantised_at_the_largest_scale(gpu_thread, k, with_addend, t):
    """Every contribution is finite in fp32, their sums are not: a block of them has the scale of fp32's largest numbers and its
    elements stop at 6 times that; dense results are infinite."""
    rows, cols = 40, 200
    rng = np.random.default_rng(1000 * k + with_addend)
    src = [random_mx(rows, cols, rng, unit=249, spread=3) for _ in range(k)]
    addend = None
    if with_addend:
        top = {"fp32": 3.3e38, "bf16": 3.3e38, "fp16": 6e4}[t]
        addend = Dense(rows, cols, t, values=rng.uniform(-top, top, (rows, cols)))
    dst, again, v = fold(gpu_thread, t, src, addend, rows, cols)
    past = np.abs(v) >= 2.0 ** 128
    assert past.any() or k == 1 and t == "fp16"
    code, scale = ref.mx_encode(v)
    got = again.code()
    zero = (code & 7) == 0
    assert np.array_equal(again.scale(), scale) and scale.max() == 252
    assert np.array_equal(got[~zero], code[~zero]) and not (got[zero] & 7).any() and again.guards_hold()
    infinite = np.abs(v) >= INFINITE_FROM[t]
    out = dst.double()
    assert np.array_equal(out[infinite], np.copysign(np.inf, v[infinite])) and np.isfinite(out[~infinite]).all()
    close(np.where(infinite, 0.0, out), np.where(infinite, 0.0, v), t, 0.0, "dst")


@pytest.mark.parametrize("k", [2, 9])
def test_infinities_and_nan_make_their_block_nan(gpu_thread, k):
    """An infinite or NaN term is no sum past the range: its block, and no other, becomes NaN."""
    rows, cols = 6, 160
    rng = np.random.default_rng(k)
    src = [random_mx(rows, cols, rng, unit=246, spread=4) for _ in range(k)]
    for t, value in (("fp32", np.inf), ("fp32", -np.inf), ("bf16", np.nan)):
        own = rng.standard_normal((rows, cols))
        own[2, 70] = value
        addend = Dense(rows, cols, t, values=own)
        dst, again, v = fold(gpu_thread, t, src, addend, rows, cols)
        code, scale = ref.mx_encode(v)
        assert (scale == 255).sum() == 1 and np.array_equal(again.scale(), scale)
        assert not again.code()[2, 2].any() and again.guards_hold()
        at = dst.double()[2, 70]
        assert np.isnan(at) if np.isnan(value) else at == value
