"""Which form every product of the GPU tests takes: a rule that moves may not leave a form without its tests (no GPU)."""
import pytest

import test_gpu_mx as mx
from product_forms import DIRECT_16, DIRECT_32, MID_128, MID_64, SIZES, TILE, WAVE_32, form_of


@pytest.mark.parametrize("form", sorted(SIZES))
def test_sizes_by_form(form):
    for size in SIZES[form]:
        assert form_of(*size) == form, size


def test_sizes_of_the_other_product_tests():
    assert [form_of(*s) for s in mx.PRODUCTS] == [DIRECT_16] * 13 + [DIRECT_32] * 2 + [MID_64] * 2
    assert [form_of(*s) for s in mx.SHORT] == [WAVE_32, WAVE_32, DIRECT_32, DIRECT_32, DIRECT_32, WAVE_32, WAVE_32, MID_128, MID_64, MID_128, WAVE_32, MID_128]
    assert form_of(1, (1 << 30) + 5003, 256, 1) == TILE


@pytest.mark.parametrize("form", sorted(SIZES))
def test_ranks_with_strides_of_their_own_take_no_form_of_one_stride(form):
    """The forms through LDS walk every rank's matrices by the first one's strides."""
    for m, n, cols, k in SIZES[form]:
        if k == 1:
            continue
        one, last = [1] * k, [0] * (k - 1) + [1]
        assert form_of(m, n, cols, k, one, one, one, one) == form           # equal strides, padded
        for side, rows in (("a", m), ("b", n)):
            for what in ("blocks", "scales"):
                if rows > 1:                                                # a single row has no stride
                    assert form_of(m, n, cols, k, **{side + "_" + what: last}) in (DIRECT_16, DIRECT_32, WAVE_32), (m, n, cols, k, side, what)


def test_rows_of_few_blocks_take_no_form_of_whole_stages():
    for cols in (1, 32, 100, 224):
        assert form_of(2900, 2900, cols, 1) == WAVE_32
    assert form_of(2900, 2900, 225, 1) == TILE
    assert form_of(2900, 2900, 481, 2, [0, 1]) == DIRECT_32                 # too long for the form of short rows
