"""Products that go through tiles in LDS, at the sizes at which each of those forms is taken (tests/product_forms.py, pinned by
tests/test_product_forms.py), against the format's definition in 64 bits.  The bound: every one of a product's additions loses
at most one step of fp32 of the sum of magnitudes."""
import numpy as np
import pytest

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
