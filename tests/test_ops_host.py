"""What the operators around a fold refuse, and the launches they make, on a recorder thread (no GPU)."""
import pytest

import hcomm_amd as h
from hcomm_amd import HcclResult as R, HcommDataType as DT, Kernel

A, B, C_, D, E, F = (0x10000000 * i for i in range(1, 7))


@pytest.fixture()
def rec():
    code, t = h.HcommGfxRecorderThreadAlloc()
    assert code == 0
    yield t
    h.HcommThreadFree([t])


def view(packed=A, scales=B, cols=64, rows=4, pad=0):
    nb = -(-cols // 32) + pad
    return h.mx_views([(packed, nb * 16, scales, nb)])


def ranks(k, cols=64):
    nb = -(-cols // 32)
    return h.mx_views([(A + 0x100000 * j, nb * 16, B + 0x100000 * j, nb) for j in range(k)])


def nothing_ran(rec):
    assert h.launch_log(rec) == []


def test_quantize_refusals(rec):
    q = lambda thread=rec, out=None, src=C_, stride=64, rows=4, cols=64, t=DT.BFP16: h.HcommGfxMxQuantizeOnThread(  # noqa: E731
        thread, view(cols=max(cols, 1)) if out is None else out, src, stride, rows, cols, t)
    assert h.HcommGfxMxQuantizeOnThread(rec, None, C_, 64, 4, 64, DT.BFP16) == R.E_PTR
    assert q(out=view(packed=0)) == R.E_PTR and q(out=view(scales=0)) == R.E_PTR and q(src=None) == R.E_PTR
    assert q(thread=0) == R.E_PTR and q(thread=0x1234) == R.E_PTR
    for t in (DT.INT8, DT.INT32, DT.FP64, DT.FP8E4M3, 255):
        assert q(t=t) == R.E_PARA
    assert q(src=C_ + 1) == R.E_PARA and q(src=C_ + 2, t=DT.FP32) == R.E_PARA
    assert q(stride=63) == R.E_PARA                                     # rows would overlap
    assert q(out=view(packed=A + 8)) == R.E_PARA                        # blocks are 16-byte units
    assert q(out=h.mx_views([(A, 40, B, 2)])) == R.E_PARA and q(out=h.mx_views([(A, 16, B, 2)])) == R.E_PARA
    assert q(out=h.mx_views([(A, 32, B, 1)])) == R.E_PARA               # scales of neighbouring rows would overlap
    assert q(out=view(packed=C_ + 16)) == R.E_PARA and q(out=view(scales=C_ + 5)) == R.E_PARA  # over the source
    assert q(out=view(scales=A + 3)) == R.E_PARA
    assert q(stride=1 << 63) == R.E_PARA and q(src=(1 << 64) - 64) == R.E_PARA  # ends wrap
    assert q(rows=1, cols=(1 << 34) + 1, stride=0) == R.E_NOT_SUPPORT
    nothing_ran(rec)
    h.HcommBatchModeStart(None)
    assert q() == R.E_NOT_SUPPORT
    h.HcommBatchModeEnd(None)
    assert q(rows=0) == R.SUCCESS and q(cols=0) == R.SUCCESS
    nothing_ran(rec)
    assert q() == R.SUCCESS and q(rows=1, stride=0) == R.SUCCESS        # a single row has no stride
    a, b = h.launch_log(rec)
    assert (a.kind, a.dtype, a.bytes, a.blocks) == (Kernel.MX_QUANTIZE, DT.BFP16, 4 * 2 * 17, 1) and b.bytes == 34


def test_columns_of_a_larger_matrix_do_not_meet(rec):
    """Inputs and outputs that interleave row by row are taken; the same with one element in common is refused."""
    own = lambda off: h.HcommGfxMxReduceKOnThread(rec, C_, 200, DT.FP32, None, view(), 1, C_ + 4 * off, 200, 4, 64)  # noqa: E731
    assert own(64) == R.SUCCESS and own(136) == R.SUCCESS and own(0) == R.SUCCESS
    assert own(63) == R.E_PARA and own(137) == R.E_PARA and own(200) == R.E_PARA


def test_fold_refusals(rec):
    def fold(thread=rec, dst=C_, ds=64, t=DT.FP32, again=None, srcs=None, k=3, addend=None, stride=64, rows=4, cols=64):
        return h.HcommGfxMxReduceKOnThread(thread, dst, ds, t, again, ranks(3) if srcs is None else srcs, k, addend, stride, rows, cols)
    assert fold(dst=None) == R.E_PTR and fold(thread=0) == R.E_PTR
    assert h.HcommGfxMxReduceKOnThread(rec, C_, 64, DT.FP32, None, None, 1, None, 0, 4, 64) == R.E_PTR
    assert fold(again=view(packed=0)) == R.E_PTR
    assert fold(srcs=h.mx_views([(A, 32, B, 2), (0, 32, B, 2), (A, 32, B, 2)])) == R.E_PTR
    assert fold(k=0) == R.E_PARA and fold(k=33) == R.E_PARA
    assert fold(t=DT.INT32) == R.E_PARA and fold(dst=C_ + 2) == R.E_PARA and fold(ds=63) == R.E_PARA
    assert fold(addend=C_ + 4) == R.E_PARA and fold(addend=C_, stride=65) == R.E_PARA   # meets dst without being it
    assert fold(dst=A) == R.E_PARA and fold(dst=B + 0x200000) == R.E_PARA               # over an input
    assert fold(again=view(packed=C_, scales=D)) == R.E_PARA and fold(again=view(packed=D, scales=D + 8)) == R.E_PARA
    assert fold(again=view()) == R.E_PARA
    h.HcommBatchModeStart(None)
    assert fold() == R.E_NOT_SUPPORT
    h.HcommBatchModeEnd(None)
    assert fold(rows=0) == R.SUCCESS and fold(cols=0) == R.SUCCESS
    nothing_ran(rec)
    assert fold() == R.SUCCESS and fold(addend=C_) == R.SUCCESS
    assert fold(dst=None, again=view(packed=D, scales=E)) == R.SUCCESS
    assert fold(srcs=ranks(1), k=1) == R.SUCCESS
    assert [(r.kind, r.nseg, r.bytes) for r in h.launch_log(rec)] == \
        [(Kernel.MX_REDUCE, 3, 1024), (Kernel.MX_REDUCE, 3, 1024), (Kernel.MX_REDUCE, 3, 4 * 34), (Kernel.MX_REDUCE, 1, 1024)]


def test_product_refusals(rec):
    def product(thread=rec, dst=E, ds=8, t=DT.BFP16, a=None, b=None, k=2, m=4, n=8, cols=64):
        at = lambda base: h.mx_views([(base + 0x1000 * j, 32, base + 0x100000 + 0x1000 * j, 2) for j in range(2)])  # noqa: E731
        return h.HcommGfxMxProductKOnThread(thread, dst, ds, t, at(A) if a is None else a, at(C_) if b is None else b, k, m, n, cols)
    assert product(dst=None) == R.E_PTR and product(thread=0) == R.E_PTR
    assert h.HcommGfxMxProductKOnThread(rec, E, 8, DT.BFP16, None, view(), 1, 4, 8, 64) == R.E_PTR
    assert product(b=h.mx_views([(A, 32, B, 2), (A, 32, 0, 2)])) == R.E_PTR
    assert product(k=0) == R.E_PARA and product(k=33) == R.E_PARA and product(t=DT.INT8) == R.E_PARA and product(cols=0) == R.E_PARA
    assert product(ds=7) == R.E_PARA and product(dst=E + 1) == R.E_PARA and product(dst=A) == R.E_PARA
    assert product(a=h.mx_views([(A + 4, 32, B, 2)] * 2)) == R.E_PARA
    assert product(cols=1 << 28) == R.E_NOT_SUPPORT
    assert product(a=h.mx_views([(A, 1 << 23, B, 2)] * 2)) == R.E_NOT_SUPPORT
    h.HcommBatchModeStart(None)
    assert product() == R.E_NOT_SUPPORT
    h.HcommBatchModeEnd(None)
    assert product(m=0) == R.SUCCESS and product(n=0) == R.SUCCESS
    nothing_ran(rec)
    assert product() == R.SUCCESS
    assert product(b=h.mx_views([(C_, 32, C_ + 0x1000, 2)] * 2)) == R.SUCCESS    # the same weights twice
    assert all((r.kind, r.nseg, r.bytes) == (Kernel.MX_PRODUCT, 2, 64) for r in h.launch_log(rec))


def norm(**change):
    f = dict(rows=4, cols=64, dataType=DT.BFP16, paramType=DT.BFP16, srcs=[A, A + 0x1000], srcStride=64, residual=B, residualStride=64,
             residualScale=1.0, eps=1e-5, postWeight=C_, preWeight=C_ + 0x1000, gate=C_ + 0x2000, gateStride=64, rowsPerGate=4,
             sum=D, sumStride=64, y=D + 0x1000, yStride=64, z=D + 0x2000, zStride=64)
    f.update(change)
    return h.ReduceNormDesc(**f)


def test_norm_refusals(rec):
    run = lambda thread=rec, **c: h.HcommGfxReduceNormOnThread(thread, norm(**c))  # noqa: E731
    assert h.HcommGfxReduceNormOnThread(rec, None) == R.E_PTR and run(thread=0) == R.E_PTR
    assert run(y=None) == R.E_PTR and run(z=None) == R.E_PTR and run(preWeight=None) == R.E_PTR and run(srcs=[A, 0]) == R.E_PTR
    assert run(srcs=[]) == R.E_PARA and run(srcs=[A + 0x1000 * j for j in range(33)]) == R.E_PARA
    assert run(dataType=DT.INT8) == R.E_PARA and run(paramType=DT.FP16) == R.E_PARA and run(dataType=DT.FP32) == R.E_PARA
    nan = float("nan")
    assert run(eps=-1.0) == R.E_PARA and run(eps=nan) == R.E_PARA and run(residualScale=nan) == R.E_PARA and run(eps=float("inf")) == R.E_PARA
    assert run(rowsPerGate=0) == R.E_PARA
    for name in ("srcStride", "residualStride", "sumStride", "yStride", "zStride"):
        assert run(**{name: 63}) == R.E_PARA, name
    assert run(gateStride=63, rowsPerGate=2) == R.E_PARA and run(gateStride=63) == R.SUCCESS  # one row of gates has no stride
    h.HcommGfxLaunchLogClear(rec)
    for name, at in (("y", A), ("y", D + 2), ("z", B), ("z", D + 0x1000), ("sum", A + 0x1000), ("sum", B), ("y", C_), ("z", C_ + 0x2000), ("y", D + 0x2000), ("z", D + 1)):
        assert run(**{name: at}) == R.E_PARA, (name, at)
    assert run(y=B, yStride=72) == R.E_PARA and run(sum=A, srcs=[A, A]) == R.E_PARA
    assert run(cols=16385, srcStride=16385, residualStride=16385, sumStride=16385, yStride=16385, zStride=16385) == R.E_NOT_SUPPORT
    h.HcommBatchModeStart(None)
    assert run() == R.E_NOT_SUPPORT
    h.HcommBatchModeEnd(None)
    assert run(rows=0) == R.SUCCESS and run(cols=0) == R.SUCCESS
    nothing_ran(rec)
    assert run() == R.SUCCESS and run(y=B, sum=A) == R.SUCCESS and run(sum=None, residual=None, gate=None, postWeight=None) == R.SUCCESS
    assert run(preWeight=None, z=None, rowsPerGate=0, gate=None) == R.SUCCESS and run(paramType=DT.FP32) == R.SUCCESS
    assert [(r.kind, r.bytes, r.nseg) for r in h.launch_log(rec)] == [(Kernel.NORM, n * 512, 2) for n in (3, 3, 2, 2, 3)]


def grad(work=True, **change):
    f = dict(rows=4, cols=64, dataType=DT.BFP16, paramType=DT.BFP16, residualScale=1.0, eps=1e-5, rowsPerGate=4, sum=A, sumStride=64,
             y=A + 0x1000, yStride=64, dy=A + 0x2000, dyStride=64, dz=A + 0x3000, dzStride=64, postWeight=B, preWeight=B + 0x1000,
             gate=B + 0x2000, gateStride=64, dSum=C_, dSumStride=64, dResidual=C_ + 0x1000, dResidualStride=64, dPostWeight=D,
             dPreWeight=D + 0x1000, dGate=D + 0x2000, dGateStride=64)
    f.update(change)
    d = h.ReduceNormGradDesc(**f)
    if work:
        try:
            d.workspace, d.workspaceBytes = E, h.reduce_norm_grad_workspace_bytes(d)
        except h.HcommError:
            pass
    return d


def test_norm_gradient_refusals(rec):
    run = lambda thread=rec, **c: h.HcommGfxReduceNormGradOnThread(thread, grad(**c))  # noqa: E731
    assert h.HcommGfxReduceNormGradOnThread(rec, None) == R.E_PTR and run(thread=0) == R.E_PTR
    for name in ("sum", "dy", "dSum", "dz", "y"):
        assert run(**{name: None}) == R.E_PTR, name
    assert run(work=False) == R.E_PTR
    d = grad()
    d.workspaceBytes -= 1
    assert h.HcommGfxReduceNormGradOnThread(rec, d) == R.E_PARA
    d = grad()
    d.workspace += 4
    assert h.HcommGfxReduceNormGradOnThread(rec, d) == R.E_PARA
    assert run(postWeight=None) == R.E_PARA and run(gate=None) == R.E_PARA and run(preWeight=None, dz=None) == R.E_PARA
    assert run(dataType=DT.INT8) == R.E_PARA and run(paramType=DT.FP16) == R.E_PARA and run(eps=-1.0) == R.E_PARA and run(rowsPerGate=0) == R.E_PARA
    for name in ("sumStride", "yStride", "dyStride", "dzStride", "dSumStride", "dResidualStride"):
        assert run(**{name: 63}) == R.E_PARA, name
    assert run(dGateStride=63, rowsPerGate=1) == R.E_PARA
    for name, at in (("dSum", A + 0x3000), ("dSum", A + 0x1000), ("dResidual", A), ("dResidual", C_), ("dPostWeight", B), ("dGate", D), ("dSum", E), ("dPreWeight", C_ + 2)):
        assert run(**{name: at}) == R.E_PARA, (name, at)
    assert run(dSum=A + 0x2000, dResidual=A + 0x2000) == R.E_PARA       # both over dy
    assert run(cols=16385) == R.E_NOT_SUPPORT
    h.HcommBatchModeStart(None)
    assert run() == R.E_NOT_SUPPORT
    h.HcommBatchModeEnd(None)
    nothing_ran(rec)
    assert run() == R.SUCCESS and run(dSum=A, dResidual=A + 0x1000) == R.SUCCESS and run(dSum=A + 0x2000) == R.SUCCESS and run(dResidual=A + 0x2000) == R.SUCCESS
    assert [r.kind for r in h.launch_log(rec)] == [Kernel.NORM_GRAD, Kernel.NORM_SUMS] * 4
    h.HcommGfxLaunchLogClear(rec)
    none = dict(dPostWeight=None, dPreWeight=None, dGate=None)
    assert h.reduce_norm_grad_workspace_bytes(grad(**none)) == 0 and run(work=False, **none) == R.SUCCESS
    assert [r.kind for r in h.launch_log(rec)] == [Kernel.NORM_GRAD]
    h.HcommGfxLaunchLogClear(rec)
    assert run(cols=0) == R.SUCCESS
    nothing_ran(rec)
    assert run(rows=0) == R.SUCCESS                                       # the weights' gradients become 0
    assert [r.kind for r in h.launch_log(rec)] == [Kernel.NORM_SUMS]


def test_workspace_is_bounded_by_the_runs_and_not_by_the_rows():
    for rows, cols, per in ((8192, 4096, 8192), (1 << 20, 4096, 1), (1 << 20, 64, 100), (1 << 30, 16384, 1 << 30)):
        n = h.reduce_norm_grad_workspace_bytes(grad(work=False, rows=rows, cols=cols, rowsPerGate=per))
        assert 0 < n <= 3 * 4 * 2048 * 512 * 2 * 2, (rows, cols, per, n)
    with pytest.raises(h.HcommError):
        h.reduce_norm_grad_workspace_bytes(grad(work=False, rowsPerGate=0))


def test_a_thread_in_another_batch_is_refused(rec):
    """A thread that holds recorded operations of another host thread's batch takes nothing from this one."""
    import threading
    go, stop = threading.Event(), threading.Event()

    def other():
        h.HcommBatchModeStart(None)
        h.HcommLocalCopyOnThread(rec, A, B, 64)
        go.set()
        stop.wait(20)
        h.HcommBatchModeEnd(None)
    t = threading.Thread(target=other)
    t.start()
    assert go.wait(20)
    try:
        assert h.HcommGfxMxQuantizeOnThread(rec, view(), C_, 64, 4, 64, DT.BFP16) == R.E_UNAVAIL
        assert h.HcommGfxReduceNormOnThread(rec, norm()) == R.E_UNAVAIL
        assert h.HcommGfxReduceNormGradOnThread(rec, grad()) == R.E_UNAVAIL
    finally:
        stop.set()
        t.join()
    assert h.HcommGfxMxQuantizeOnThread(rec, view(), C_, 64, 4, 64, DT.BFP16) == R.SUCCESS


def test_launches_of_more_lanes_than_a_grid_counts(rec):
    """A limit of its own, next to it the last size that is taken; nothing of a refused call is queued."""
    big = lambda at: at << 20  # noqa: E731  (apart from one another by more than the matrices are long)
    fold = lambda cols: h.HcommGfxMxReduceKOnThread(rec, big(A), 0, DT.BFP16, None, h.mx_views([(big(B), 0, big(C_), 0)]), 1, None, 0, 1, cols)  # noqa: E731
    last = ((1 << 24) - 1) * 256 * 8
    assert last > 1 << 34 and fold((1 << 34) + 32) == R.E_NOT_SUPPORT and fold(1 << 34) == R.SUCCESS
    rows = lambda n: h.HcommGfxMxReduceKOnThread(rec, big(A), 64, DT.BFP16, None, h.mx_views([(big(B), 32, big(C_), 2)]), 1, None, 0, n, 33)  # noqa: E731
    assert rows(32 * ((1 << 24) - 1)) == R.SUCCESS and rows(32 * ((1 << 24) - 1) + 1) == R.E_NOT_SUPPORT
    norm = lambda n: h.HcommGfxReduceNormOnThread(rec, h.ReduceNormDesc(  # noqa: E731
        rows=n, cols=64, dataType=DT.BFP16, paramType=DT.BFP16, residualScale=1.0, eps=1e-5, srcs=[big(A)], srcStride=64, y=big(B), yStride=64))
    assert norm(32 * ((1 << 24) - 1)) == R.SUCCESS and norm(32 * ((1 << 24) - 1) + 1) == R.E_NOT_SUPPORT and norm(1 << 31) == R.E_NOT_SUPPORT
    one = lambda m, n: h.HcommGfxMxProductKOnThread(rec, big(A), n, DT.BFP16, h.mx_views([(big(B), 16, big(C_), 1)]),  # noqa: E731
                                                    h.mx_views([(big(D), 16, big(E), 1)]), 1, m, n, 32)
    assert one(1, 32 * ((1 << 23) - 1)) == R.SUCCESS and one(1, 32 * ((1 << 23) - 1) + 1) == R.E_NOT_SUPPORT
    assert one(1 << 16, (1 << 17) - 32) == R.SUCCESS and one(1 << 16, 1 << 17) == R.E_NOT_SUPPORT
    assert [r.kind for r in h.launch_log(rec)] == [Kernel.MX_REDUCE] * 2 + [Kernel.NORM] + [Kernel.MX_PRODUCT] * 2
