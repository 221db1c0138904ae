"""A shard of a batch that has no rows: the weights' gradients are 0, the gate has no row and its gradient's memory stays as it is."""
import pytest
import torch

import hcomm_amd as h
from ops_util import DT, Dense

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("per", [1, 100])
@pytest.mark.parametrize("cols,p", [(7, "fp32"), (600, "bf16"), (9000, "fp32")])
def test_gradient_of_no_rows(gpu_thread, cols, p, per):
    some, gate, d_gate = Dense(1, cols, "bf16"), Dense(1, cols, p), Dense(1, cols, p)
    w1, w2, d1, d2 = (Dense(1, cols, p) for _ in range(4))
    d = h.ReduceNormGradDesc(
        rows=0, cols=cols, dataType=DT["bf16"], paramType=DT[p], residualScale=1.0, eps=1e-5, rowsPerGate=per, sum=some.ptr, sumStride=cols,
        y=some.ptr, yStride=cols, dy=some.ptr, dyStride=cols, dz=some.ptr, dzStride=cols, postWeight=w1.ptr, preWeight=w2.ptr, gate=gate.ptr,
        gateStride=cols, dSum=some.ptr, dSumStride=cols, dPostWeight=d1.ptr, dPreWeight=d2.ptr, dGate=d_gate.ptr, dGateStride=cols)
    assert h.reduce_norm_grad_workspace_bytes(d) == 0
    torch.cuda.synchronize()
    h.check(h.HcommGfxReduceNormGradOnThread(gpu_thread, d))
    h.check(h.HcommGfxThreadSynchronize(gpu_thread))
    for x in (d1, d2):
        assert not bool(x.view.any()) and x.guards_hold()
    for x in (some, gate, d_gate, w1, w2):
        assert bool((x.raw == 0xA5).all())
