"""A product whose rows of results are longer than 4 GiB."""
import numpy as np
import pytest
import torch

import hcomm_amd as h
import ops_reference as ref
from ops_util import DT, random_mx

pytestmark = pytest.mark.gpu


def test_columns_past_two_to_the_thirtieth(gpu_thread):
    """One token times more than 2^30 rows of weights, of which only the first and the last ones are not zero: every fp32
    result lies in its own column, and those behind 2^30 elements not in the row's first ones."""
    cols, blocks, front, back = 256, 8, 4096, 5003
    n = (1 << 30) + back
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 160e9:
        pytest.skip("150 GB of device memory are not free")
    rng = np.random.default_rng(30)
    a = random_mx(1, cols, rng, unit=120)
    ends = [random_mx(rows, cols, rng, unit=118) for rows in (front, back)]
    packed = torch.zeros((n, blocks, 16), dtype=torch.uint8, device="cuda")
    scales = torch.zeros((n, blocks), dtype=torch.uint8, device="cuda")
    for part, e in ((slice(0, front), ends[0]), (slice(n - back, n), ends[1])):
        packed[part].copy_(e._blocks())
        scales[part].copy_(e._scales())
    dst = torch.full((n + 64,), float("nan"), dtype=torch.float32, device="cuda")
    b = h.mx_views([(packed.data_ptr(), blocks * 16, scales.data_ptr(), blocks)])
    torch.cuda.synchronize()
    h.check(h.HcommGfxMxProductKOnThread(gpu_thread, dst.data_ptr(), n, DT["fp32"], h.mx_views([a.item]), b, 1, 1, n, cols))
    h.check(h.HcommGfxThreadSynchronize(gpu_thread))
    try:
        for part, e in ((slice(0, front), ends[0]), (slice(n - back, n), ends[1])):
            want, magnitude = (a.values() @ e.values().T)[0], (np.abs(a.values()) @ np.abs(e.values()).T)[0]
            # one step of fp32 of the sum of magnitudes for every addition and the rounding of the result
            off = np.abs(dst[part].double().cpu().numpy() - want)
            assert (off <= cols * 2.0 ** -23 * magnitude + np.abs(want) * ref.EPS_HALF["fp32"]).all(), part
        assert not bool((dst[front:n - back] != 0).any())
        assert bool(torch.isnan(dst[n:]).all())
    finally:
        del packed, scales, dst
        torch.cuda.empty_cache()  # 150 GB that no other test needs
