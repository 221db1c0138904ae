"""The norms behind a fold and their gradient where they move more than the L2s hold (32 MiB) in rows of whole groups of eight,
and folds of more than eight ranks: the variants that pass by the caches, for every way in which lanes share rows.  Bounds as in
test_gpu_reduce_norm.py."""
import pytest
import torch

import hcomm_amd as h
from test_gpu_reduce_norm import Case

pytestmark = pytest.mark.gpu

L2S = 32 << 20
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}

# rows, cols, type, parameters: 1, 8 and 32 lanes to a row; one wavefront and two; more; two groups a lane; above 8,192 columns
LARGE = [(263000, 8, "fp32", "fp32"), (66001, 64, "bf16", "fp32"), (8300, 256, "fp32", "fp32"), (8209, 512, "fp16", "fp16"), (2063, 1024, "fp32", "fp32"),
         (2057, 2048, "bf16", "bf16"), (1031, 2048, "fp32", "fp32"), (1033, 4096, "fp16", "fp32"), (515, 8192, "bf16", "fp32"), (130, 16384, "fp32", "fp32")]


@pytest.mark.parametrize("rows,cols,t,p", LARGE)
@pytest.mark.parametrize("gates", ["one for all", "one for each", "few", "none"])
def test_more_than_the_caches_hold(gpu_thread, rows, cols, t, p, gates):
    assert cols % 8 == 0 and rows * cols * SIZE[t] * 4 > L2S
    per = {"one for all": rows, "one for each": 1, "few": rows // 7, "none": 0}[gates]
    Case(rows, cols, t, k=2, per=per, p=p).run(gpu_thread)


@pytest.mark.parametrize("rows,cols,t,p", [LARGE[1], LARGE[4], LARGE[7], LARGE[9]])
def test_over_their_inputs(gpu_thread, rows, cols, t, p):
    """y over the residual and the sum over the first partial; dSum over the sum, dResidual over dy: the bits of calls with outputs
    of their own."""
    a, b = (Case(rows, cols, t, k=2, per=rows // 3, p=p) for _ in range(2))
    torch.cuda.synchronize()
    h.check(a.forward(gpu_thread))
    h.check(b.forward(gpu_thread, y=b.residual.ptr, sum=b.x[0].ptr))
    h.check(h.HcommGfxThreadSynchronize(gpu_thread))
    assert torch.equal(a.y.view, b.residual.view) and torch.equal(a.sum.view, b.x[0].view) and torch.equal(a.z.view, b.z.view)
    da, db = a.gradient_desc(), b.gradient_desc(sum=b.x[0].ptr, y=b.residual.ptr, dSum=b.x[0].ptr, dResidual=b.dy.ptr)
    torch.cuda.synchronize()
    h.check(h.HcommGfxReduceNormGradOnThread(gpu_thread, da))
    h.check(h.HcommGfxReduceNormGradOnThread(gpu_thread, db))
    h.check(h.HcommGfxThreadSynchronize(gpu_thread))
    for want, got in ((a.ds, b.x[0]), (a.dres, b.dy), (a.dpost, b.dpost), (a.dpre, b.dpre), (a.dgate, b.dgate)):
        assert torch.equal(want.view, got.view)


@pytest.mark.parametrize("k", [9, 17, 32])
@pytest.mark.parametrize("rows,cols", [(1, 8), (1, 1024), (6, 64), (6, 776), (7, 1024), (3, 2048), (2, 8200), (1, 16384)])
@pytest.mark.parametrize("t", ["bf16", "fp32"])
def test_more_than_eight_ranks(gpu_thread, rows, cols, k, t):
    """Rows of whole groups; rows that start off 16-byte boundaries too."""
    Case(rows, cols, t, k=k, per=2).run(gpu_thread)
    Case(rows, cols, t, k=k, per=2, pad=3, seed=1).run(gpu_thread)
