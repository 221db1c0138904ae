"""The operators around a fold as they are used together, every stage against its formula on what the stage before left:
a tensor-parallel block's boundary (quantise, product, fold with norms, quantise, product; the gradient back through the
norms), and an allreduce whose messages travel in four bits."""
import numpy as np
import pytest
import torch

import hcomm_amd as h
import ops_reference as ref
from ops_util import DT, Dense, Mx, close

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def on(thread, *calls):
    for c in calls:
        h.check(c)
    h.check(h.HcommGfxThreadSynchronize(thread))


@pytest.mark.parametrize("tokens", [1, 37])
def test_block_boundary(gpu_thread, tokens):
    ranks, inner, cols, alpha, eps = 4, 200, 328, 1.0, 1e-6
    rng = np.random.default_rng(tokens)
    acts = [Dense(tokens, inner, "bf16", values=rng.standard_normal((tokens, inner))) for _ in range(ranks)]
    weights = [Dense(cols, inner, "bf16", values=rng.standard_normal((cols, inner)) / 28) for _ in range(ranks)]
    residual = Dense(tokens, cols, "bf16", values=rng.standard_normal((tokens, cols)))
    post, pre, gate = (Dense(1, cols, "bf16", values=1 + 0.1 * rng.standard_normal((1, cols))) for _ in range(3))
    qa, qw = [Mx(tokens, inner) for _ in range(ranks)], [Mx(cols, inner) for _ in range(ranks)]
    partial = [Dense(tokens, cols, "bf16") for _ in range(ranks)]
    whole = Dense(tokens, cols, "fp32")
    s, y, z, qz = (Dense(tokens, cols, "bf16") for _ in range(3)), None, None, Mx(tokens, cols)
    s, y, z = s
    nxt = Dense(tokens, 50, "bf16")
    w_next = Dense(50, cols, "bf16", values=rng.standard_normal((50, cols)))
    qn = Mx(50, cols)
    torch.cuda.synchronize()
    one = lambda m: h.mx_views([m.item])  # noqa: E731
    for j in range(ranks):
        on(gpu_thread,
           h.HcommGfxMxQuantizeOnThread(gpu_thread, one(qa[j]), acts[j].ptr, inner, tokens, inner, DT["bf16"]),
           h.HcommGfxMxQuantizeOnThread(gpu_thread, one(qw[j]), weights[j].ptr, inner, cols, inner, DT["bf16"]),
           h.HcommGfxMxProductKOnThread(gpu_thread, partial[j].ptr, cols, DT["bf16"], one(qa[j]), one(qw[j]), 1, tokens, cols, inner))
    desc = h.ReduceNormDesc(
        rows=tokens, cols=cols, dataType=DT["bf16"], paramType=DT["bf16"], srcs=[p.ptr for p in partial], srcStride=cols, residual=residual.ptr,
        residualStride=cols, residualScale=alpha, eps=eps, postWeight=post.ptr, preWeight=pre.ptr, gate=gate.ptr, gateStride=cols,
        rowsPerGate=tokens, sum=s.ptr, sumStride=cols, y=y.ptr, yStride=cols, z=z.ptr, zStride=cols)
    on(gpu_thread,
       h.HcommGfxReduceNormOnThread(gpu_thread, desc),
       h.HcommGfxMxQuantizeOnThread(gpu_thread, one(qz), z.ptr, cols, tokens, cols, DT["bf16"]),
       h.HcommGfxMxQuantizeOnThread(gpu_thread, one(qn), w_next.ptr, cols, 50, cols, DT["bf16"]),
       h.HcommGfxMxProductKOnThread(gpu_thread, nxt.ptr, 50, DT["bf16"], one(qz), one(qn), 1, tokens, 50, cols),
       h.HcommGfxMxProductKOnThread(gpu_thread, whole.ptr, cols, DT["fp32"], h.mx_views([q.item for q in qa]), h.mx_views([q.item for q in qw]),
                                    ranks, tokens, cols, inner))
    total, size = 0.0, 0.0
    for j in range(ranks):
        for q, d in ((qa[j], acts[j]), (qw[j], weights[j])):
            code, scale = ref.mx_encode(d.double())
            assert np.array_equal(q.code(), code) and np.array_equal(q.scale(), scale)
        p, m = qa[j].values() @ qw[j].values().T, np.abs(qa[j].values()) @ np.abs(qw[j].values()).T
        close(partial[j].double(), p, "bf16", inner * 2 * U * m, "partial")
        total, size = total + p, size + m
    # the product over all ranks in one call: the partial sums that the ranks would have rounded
    close(whole.double(), total, "fp32", ranks * inner * 2 * U * size, "whole")
    want = ref.norm(np.stack([p.double() for p in partial]), residual.double(), alpha, eps, post.double()[0], pre.double()[0], gate.double(), tokens)
    magnitude = sum(np.abs(p.double()) for p in partial).max()
    for got, exp, what in zip((s, y, z), want, ("sum", "y", "z")):
        close(got.double(), exp, "bf16", 64 * U * (np.abs(exp).max() + magnitude), what)
    code, scale = ref.mx_encode(z.double())
    assert np.array_equal(qz.code(), code) and np.array_equal(qz.scale(), scale)
    close(nxt.double(), qz.values() @ qn.values().T, "bf16", cols * 2 * U * (np.abs(qz.values()) @ np.abs(qn.values()).T), "next")
    # back through the norms: what y and z receive reaches every rank's partial and the residual
    dy, dz = (Dense(tokens, cols, "bf16", values=rng.standard_normal((tokens, cols))) for _ in range(2))
    ds, dres, dpost, dpre, dgate = (Dense(n, cols, "bf16") for n in (tokens, tokens, 1, 1, 1))
    g = h.ReduceNormGradDesc(
        rows=tokens, cols=cols, dataType=DT["bf16"], paramType=DT["bf16"], residualScale=alpha, eps=eps, rowsPerGate=tokens, sum=s.ptr,
        sumStride=cols, y=y.ptr, yStride=cols, dy=dy.ptr, dyStride=cols, dz=dz.ptr, dzStride=cols, postWeight=post.ptr, preWeight=pre.ptr,
        gate=gate.ptr, gateStride=cols, dSum=ds.ptr, dSumStride=cols, dResidual=dres.ptr, dResidualStride=cols, dPostWeight=dpost.ptr,
        dPreWeight=dpre.ptr, dGate=dgate.ptr, dGateStride=cols)
    work = torch.empty(h.reduce_norm_grad_workspace_bytes(g), dtype=torch.uint8, device="cuda")
    g.workspace, g.workspaceBytes = work.data_ptr(), work.numel()
    torch.cuda.synchronize()
    on(gpu_thread, h.HcommGfxReduceNormGradOnThread(gpu_thread, g))
    want = ref.norm_grad(s.double(), y.double(), dy.double(), dz.double(), alpha, eps, post.double()[0], pre.double()[0], gate.double(), tokens)
    for got, name in ((ds, "sum"), (dres, "residual"), (dpost, "post"), (dpre, "pre"), (dgate, "gate")):
        exp = want[name].reshape(got.double().shape)
        close(got.double(), exp, "bf16", (128 + tokens) * U * np.abs(exp).max() * 4, name)


def test_allreduce_in_four_bits(gpu_thread):
    """Reduce-scatter and all-gather of quantised slices with the copies of the framework's own batch mode: every rank's own
    share stays in full precision, every rank ends with the same bits."""
    ranks, count = 5, 5 * 1031
    slice_ = count // ranks
    nb = ref.blocks_of(slice_)
    rng = np.random.default_rng(3)
    x = [Dense(1, count, "bf16", values=rng.standard_normal((1, count)) * 1e-3) for _ in range(ranks)]
    sent = [[Mx(1, slice_) for _ in range(ranks)] for _ in range(ranks)]        # sent[r][d]: rank r's message to rank d
    there = [[Mx(1, slice_) for _ in range(ranks)] for _ in range(ranks)]       # there[d][r]: the same, arrived
    folded, gathered = [Mx(1, slice_) for _ in range(ranks)], [[Mx(1, slice_) for _ in range(ranks)] for _ in range(ranks)]
    out = [Dense(1, count, "bf16") for _ in range(ranks)]
    at = lambda d, i: d.ptr + i * slice_ * 2  # noqa: E731
    torch.cuda.synchronize()
    t = gpu_thread
    for r in range(ranks):
        for d in range(ranks):
            if r != d:
                h.check(h.HcommGfxMxQuantizeOnThread(t, h.mx_views([sent[r][d].item]), at(x[r], d), slice_, 1, slice_, DT["bf16"]))

    def move(pairs):
        h.check(h.HcommBatchModeStart(b"four bits"))
        for dst, src in pairs:
            h.check(h.HcommLocalCopyOnThread(t, dst.item[0], src.item[0], nb * 16))
            h.check(h.HcommLocalCopyOnThread(t, dst.item[2], src.item[2], nb))
        h.check(h.HcommBatchModeEnd(b"four bits"))
    move([(there[d][r], sent[r][d]) for r in range(ranks) for d in range(ranks) if r != d])
    for d in range(ranks):
        views = h.mx_views([there[d][r].item for r in range(ranks) if r != d])
        h.check(h.HcommGfxMxReduceKOnThread(t, None, 0, DT["bf16"], h.mx_views([folded[d].item]), views, ranks - 1, at(x[d], d), slice_, 1, slice_))
    move([(gathered[r][d], folded[d]) for r in range(ranks) for d in range(ranks)])
    for r in range(ranks):
        for d in range(ranks):
            h.check(h.HcommGfxMxReduceKOnThread(t, at(out[r], d), slice_, DT["bf16"], None, h.mx_views([gathered[r][d].item]), 1, None, 0, 1, slice_))
    h.check(h.HcommGfxThreadSynchronize(t))
    for d in range(ranks):
        part = slice(d * slice_, (d + 1) * slice_)
        v = x[d].double()[:, part]
        for r in range(ranks):
            if r != d:
                code, scale = ref.mx_encode(x[r].double()[:, part])
                v = v + ref.mx_values(code, scale, slice_)
        code, scale = ref.mx_encode(v)
        want = ref.mx_values(code, scale, slice_)
        for r in range(ranks):
            assert np.array_equal(out[r].double()[:, part], want)
    for r in range(ranks):
        assert out[r].guards_hold() and torch.equal(out[r].raw, out[0].raw)
