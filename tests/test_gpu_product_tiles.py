"""Products that go through tiles in LDS, at the sizes at which each of those forms is taken (tests/product_forms.py, pinned by
tests/test_product_forms.py), against the format's definition in 64 bits.  The bound: every one of a product's additions loses
at most one step of fp32 of the sum of magnitudes."""
import numpy as np
import pytest
import torch

import hcomm_amd as h
from ops_util import DT, Dense, close, random_mx
from product_forms import MID_128, MID_64, SIZES, TILE, form_of
from test_gpu_mx import product_case, test_product_of_a_block_that_is_nan as nan_case

pytestmark = pytest.mark.gpu

ALL = [(form, size) for form in (MID_64, MID_128, TILE) for size in SIZES[form]]


@pytest.mark.parametrize("t", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("form,size", ALL)
def test_sizes(gpu_thread, form, size, t):
    """Matrices one behind another, then padded ones with garbage past the rows' ends and results inside a larger matrix."""
    m, n, cols, k = size
    assert form_of(*size) == form
    rng = np.random.default_rng(m + 7 * n + 31 * cols + k)
    product_case(gpu_thread, m, n, cols, k, t, rng)
    product_case(gpu_thread, m, n, cols, k, t, rng, pad=1, shift=1, tail=0xF, stride=3)


@pytest.mark.parametrize("form,m,n,cols", [(MID_64, 600, 700, 600), (MID_128, 1450, 1502, 500), (TILE, 2830, 2890, 300), (TILE, 257, 16400, 225),
                                           (TILE, 33000, 3, 513)])
def test_a_block_that_is_nan(gpu_thread, form, m, n, cols):
    assert form_of(m, n, cols, 1) == form
    nan_case(gpu_thread, m, n, cols)


def with_strides(x, blocks, scale_bytes):
    """x's matrix with so many more blocks and bytes of scales from row to row, which hold what would show."""
    packed = torch.full((x.rows, x.nb + blocks, 16), 0x77, dtype=torch.uint8, device="cuda")
    scales = torch.full((x.rows, x.nb + scale_bytes), 255, dtype=torch.uint8, device="cuda")
    packed[:, :x.nb], scales[:, :x.nb] = x._blocks(), x._scales()
    return packed, scales, (packed.data_ptr(), (x.nb + blocks) * 16, scales.data_ptr(), x.nb + scale_bytes)


@pytest.mark.parametrize("side", ["a", "b"])
@pytest.mark.parametrize("what", ["blocks", "scales"])
@pytest.mark.parametrize("form,m,n,cols,k", [(MID_64, 600, 700, 600, 2), (MID_128, 1450, 1502, 470, 3), (TILE, 2830, 2890, 256, 2)])
def test_the_last_rank_with_a_stride_of_its_own(gpu_thread, form, m, n, cols, k, side, what):
    """One stride of one rank differs, at sizes that take these forms when all ranks' are equal."""
    last = [0] * (k - 1) + [1]
    assert form_of(m, n, cols, k) == form and form_of(m, n, cols, k, **{side + "_" + what: last}) < MID_64
    rng = np.random.default_rng(m + n + cols)
    a, b = ([random_mx(rows, cols, rng, unit=120, tail=0x5) for _ in range(k)] for rows in (m, n))
    laid = {s: [with_strides(x, p if (s, what) == (side, "blocks") else 0, p if (s, what) == (side, "scales") else 0) for x, p in zip(ranks, last)]
            for s, ranks in (("a", a), ("b", b))}
    dst = Dense(m, n, "fp32", n + 1, 1)
    torch.cuda.synchronize()
    h.check(h.HcommGfxMxProductKOnThread(gpu_thread, dst.ptr, n + 1, DT["fp32"], h.mx_views([x[2] for x in laid["a"]]),
                                         h.mx_views([x[2] for x in laid["b"]]), k, m, n, cols))
    h.check(h.HcommGfxThreadSynchronize(gpu_thread))
    want = sum(x.values() @ y.values().T for x, y in zip(a, b))
    magnitude = sum(np.abs(x.values()) @ np.abs(y.values()).T for x, y in zip(a, b))
    close(dst.double(), want, "fp32", k * cols * 2.0 ** -23 * magnitude, "dst")
    assert dst.guards_hold()
