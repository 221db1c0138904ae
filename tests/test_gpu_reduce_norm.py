"""The norms, gate and residual behind a fold, and their gradient, against their formulas in 64 bits.

Bounds count roundings of fp32 (u = 2^-24).  A sum over a row of at most 16,384 elements goes through at most 16 additions in a
lane, 6 between lanes and 16 between wavefronts, so a sum of squares is off by at most 40 u relative, the mean by 2 u more and
1 / rms by half of that and an instruction good to one unit in the last place (2 u): 23 u, RHO = 24 u.  The output's own rounding is added by close()."""
import numpy as np
import pytest
import torch

import hcomm_amd as h
import ops_reference as ref
from ops_util import DT, Dense, close

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
RHO = 24 * U
SUM = 42 * U  # of a mean over a row, relative to the mean of magnitudes
ALPHA, EPS = 0.75, 1e-5


def rms(v):
    return np.sqrt((v * v).mean(1, keepdims=True) + EPS)


def mean(v):
    return np.abs(v).mean(1, keepdims=True)


class Case:
    def __init__(self, rows, cols, t, k=3, post=True, pre=True, per=0, p=None, residual=True, seed=0, pad=0, scale=1.0):
        rng = np.random.default_rng(seed * 7919 + rows * 31 + cols)
        self.rows, self.cols, self.t, self.p, self.per = rows, cols, t, p or t, per
        stride = cols + pad

        def dense(v, kind=None, one=False):
            kind = kind or t
            return Dense(v.shape[0], cols, kind, cols if one else stride, 0 if one else pad, v)
        normal = rng.standard_normal
        self.x = [dense(normal((rows, cols)) * scale) for _ in range(k)]
        self.residual = dense(2 * normal((rows, cols))) if residual else None
        self.post = dense(1 + 0.2 * normal((1, cols)), self.p, True) if post else None
        self.pre = dense(1 + 0.2 * normal((1, cols)), self.p, True) if pre else None
        gates = -(-rows // per) if per else 0
        self.gate = dense(0.5 + 0.2 * normal((gates, cols)), self.p) if gates else None
        self.sum, self.y = Dense(rows, cols, t, stride, pad), Dense(rows, cols, t, stride, pad)
        self.z = Dense(rows, cols, t, stride, pad) if pre else None
        self.dy, self.dz = dense(normal((rows, cols))), dense(normal((rows, cols))) if pre else None
        self.ds, self.dres = Dense(rows, cols, t, stride, pad), Dense(rows, cols, t, stride, pad)
        self.dpost = Dense(1, cols, self.p) if post else None
        self.dpre = Dense(1, cols, self.p) if pre else None
        self.dgate = Dense(gates, cols, self.p, stride, pad) if gates else None
        self.stride = stride

    def params(self):
        one = lambda d: None if d is None else d.double()[0]  # noqa: E731
        return dict(post=one(self.post), pre=one(self.pre), gate=None if self.gate is None else self.gate.double(), per=max(self.per, 1))

    def forward(self, thread, **change):
        ptr = lambda d: None if d is None else d.ptr  # noqa: E731
        s = self.stride
        fields = dict(rows=self.rows, cols=self.cols, dataType=DT[self.t], paramType=DT[self.p], srcs=[x.ptr for x in self.x], srcStride=s,
                      residual=ptr(self.residual), residualStride=s, residualScale=ALPHA, eps=EPS, postWeight=ptr(self.post),
                      preWeight=ptr(self.pre), gate=ptr(self.gate), gateStride=s, rowsPerGate=self.per, sum=self.sum.ptr, sumStride=s,
                      y=self.y.ptr, yStride=s, z=ptr(self.z), zStride=s)
        fields.update(change)
        self.desc = h.ReduceNormDesc(**fields)
        return h.HcommGfxReduceNormOnThread(thread, self.desc)

    def gradient_desc(self, **change):
        ptr = lambda d: None if d is None else d.ptr  # noqa: E731
        s = self.stride
        fields = dict(rows=self.rows, cols=self.cols, dataType=DT[self.t], paramType=DT[self.p], residualScale=ALPHA, eps=EPS,
                      rowsPerGate=self.per, sum=self.sum.ptr, sumStride=s, y=self.y.ptr, yStride=s, dy=self.dy.ptr, dyStride=s,
                      dz=ptr(self.dz), dzStride=s, postWeight=ptr(self.post), preWeight=ptr(self.pre), gate=ptr(self.gate), gateStride=s,
                      dSum=self.ds.ptr, dSumStride=s, dResidual=self.dres.ptr, dResidualStride=s, dPostWeight=ptr(self.dpost),
                      dPreWeight=ptr(self.dpre), dGate=ptr(self.dgate), dGateStride=s)
        fields.update(change)
        d = h.ReduceNormGradDesc(**fields)
        need = h.reduce_norm_grad_workspace_bytes(d)
        self.work = torch.full((need + 64,), 0xA5, dtype=torch.uint8, device="cuda")
        d.workspace, d.workspaceBytes = self.work.data_ptr(), need
        return d

    def check_forward(self):
        p = self.params()
        x = np.stack([v.double() for v in self.x])
        res = None if self.residual is None else self.residual.double()
        s, y, z = ref.norm(x, res, ALPHA, EPS, **p)
        off_s = (len(x) - 1) * U * np.abs(x).sum(0)
        close(self.sum.double(), s, self.t, off_s, "sum")
        hh, off_h = s, off_s
        if p["post"] is not None:
            hh = s / rms(s) * p["post"]
            rho = RHO + 2 * np.sqrt((off_s ** 2).mean(1, keepdims=True)) / rms(s)
            off_h = np.abs(p["post"] / rms(s)) * off_s + np.abs(hh) * (rho + 3 * U)
        if p["gate"] is not None:
            g = p["gate"][np.arange(self.rows) // p["per"]]
            hh, off_h = hh * g, off_h * np.abs(g) + np.abs(hh * g) * U
        off_y = off_h if res is None else off_h + 2 * U * (np.abs(ALPHA * res) + np.abs(hh))
        close(self.y.double(), y, self.t, off_y, "y")
        if z is not None:
            rho = RHO + 2 * np.sqrt((off_y ** 2).mean(1, keepdims=True)) / rms(y)
            close(self.z.double(), z, self.t, np.abs(p["pre"] / rms(y)) * off_y + np.abs(z) * (rho + 3 * U), "z")
        for d in (self.sum, self.y, self.z):
            assert d is None or d.guards_hold()

    def check_gradient(self):
        p = self.params()
        s, y, dy = self.sum.double(), self.y.double(), self.dy.double()
        dz = None if self.dz is None else self.dz.double()
        want = ref.norm_grad(s, y, dy, dz, ALPHA, EPS, **p)
        total, off = dy, np.zeros_like(dy)
        if dz is not None:
            r = 1 / rms(y)
            a, b = dz * p["pre"] * r, y * r ** 3 * (dz * p["pre"] * y).mean(1, keepdims=True)
            total = dy + a - b
            off = np.abs(a) * (RHO + 4 * U) + np.abs(y) * r ** 3 * mean(dz * p["pre"] * y) * (3 * RHO + SUM + 6 * U) + 3 * U * (np.abs(dy) + np.abs(a) + np.abs(b))
            n = np.abs(dz * y * r)
            close(self.dpre.double()[0], want["pre"], self.p, n.sum(0) * (RHO + (self.rows + 4) * U), "dPreWeight")
        close(self.dres.double(), want["residual"], self.t, ALPHA * off + np.abs(want["residual"]) * U, "dResidual")
        r = 1 / rms(s)
        hh = s if p["post"] is None else s * r * p["post"]
        d, off_d = total, off
        if p["gate"] is not None:
            index = np.arange(self.rows) // p["per"]
            each = np.abs(hh) * off + np.abs(total * hh) * (RHO + (self.per + 5) * U)
            bound = np.zeros_like(p["gate"])
            np.add.at(bound, index, each)
            close(self.dgate.double(), want["gate"], self.p, bound, "dGate")
            g = p["gate"][index]
            d, off_d = total * g, off * np.abs(g) + np.abs(total * g) * U
        if p["post"] is not None:
            n = s * r
            each = np.abs(n) * off_d + np.abs(d * n) * (RHO + (self.rows + 4) * U)
            close(self.dpost.double()[0], want["post"], self.p, each.sum(0), "dPostWeight")
            d, off_d = d * p["post"], off_d * np.abs(p["post"]) + np.abs(d * p["post"]) * U
            m = mean(d * s) * (3 * RHO + SUM + 6 * U) + mean(off_d * s)
            off_d = r * off_d + np.abs(d * r) * (RHO + 4 * U) + np.abs(s) * r ** 3 * m + 3 * U * (np.abs(d * r) + np.abs(want["sum"]))
        close(self.ds.double(), want["sum"], self.t, off_d, "dSum")
        for o in (self.ds, self.dres, self.dpost, self.dpre, self.dgate):
            assert o is None or o.guards_hold()
        assert bool((self.work[-64:] == 0xA5).all())

    def run(self, thread):
        torch.cuda.synchronize()
        h.check(self.forward(thread))
        d = self.gradient_desc()
        torch.cuda.synchronize()
        h.check(h.HcommGfxReduceNormGradOnThread(thread, d))
        h.check(h.HcommGfxThreadSynchronize(thread))
        self.check_forward()
        self.check_gradient()


SHAPES = [(1, 1), (1, 7), (3, 8), (5, 100), (2, 511), (9, 513), (7, 1001), (130, 1024), (33, 1500), (20, 2048), (4, 4097), (3, 8192), (2, 8200), (3, 16383), (2, 16384),
          (700, 64), (2500, 40)]


@pytest.mark.parametrize("t", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_shapes(gpu_thread, rows, cols, t):
    Case(rows, cols, t, per=rows).run(gpu_thread)
    Case(rows, cols, t, per=max(1, rows // 3), pad=3, seed=1).run(gpu_thread)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("per", [0, 1, 7, 40])
@pytest.mark.parametrize("t,p", [("bf16", "fp32"), ("fp16", "fp16"), ("fp32", "fp32")])
def test_parts_left_out(gpu_thread, post, pre, per, t, p):
    Case(40, 600, t, post=post, pre=pre, per=per, p=p, residual=per != 7, pad=1).run(gpu_thread)


@pytest.mark.parametrize("k", [1, 2, 4, 5, 8, 17, 32])
def test_ranks(gpu_thread, k):
    Case(6, 777, "bf16", k=k, per=2).run(gpu_thread)


@pytest.mark.parametrize("rows,per", [(5000, 1), (5000, 2), (5003, 3), (5000, 2500), (4999, 100), (2049, 2049), (3000, 100000)])
@pytest.mark.parametrize("cols", [24, 1030])
def test_rows_that_share_a_gate(gpu_thread, rows, per, cols):
    """Fewer gate rows than runs of rows (each joined from several runs) and more (each inside one run)."""
    Case(rows, cols, "fp32", k=1, per=per).run(gpu_thread)


def test_gradients_that_are_not_wanted(gpu_thread):
    for leave in (("dResidual",), ("dGate",), ("dPostWeight",), ("dPreWeight", "dGate"), ("dPostWeight", "dPreWeight", "dGate", "dResidual")):
        c, full = (Case(50, 300, "fp32", per=8) for _ in range(2))
        torch.cuda.synchronize()
        for case, change in ((full, {}), (c, {n: None for n in leave})):
            h.check(case.forward(gpu_thread))
            d = case.gradient_desc(**change)
            torch.cuda.synchronize()
            h.check(h.HcommGfxReduceNormGradOnThread(gpu_thread, d))
            h.check(h.HcommGfxThreadSynchronize(gpu_thread))
        for name, out, want in (("dResidual", c.dres, full.dres), ("dGate", c.dgate, full.dgate), ("dPostWeight", c.dpost, full.dpost),
                                ("dPreWeight", c.dpre, full.dpre), ("dSum", c.ds, full.ds)):
            if name in leave:
                assert bool((out.raw == 0xA5).all()), name
            else:  # the runs of rows may be cut elsewhere: the same sums in another order
                a, b = out.double(), want.double()
                assert np.abs(a - b).max() <= 1e-5 * np.abs(b).max(), name


def test_no_rows(gpu_thread):
    """Nothing is written but the weights' gradients, which are 0."""
    c = Case(0, 100, "bf16", per=4)
    torch.cuda.synchronize()
    h.check(c.forward(gpu_thread))
    h.check(h.HcommGfxReduceNormGradOnThread(gpu_thread, c.gradient_desc()))
    h.check(h.HcommGfxThreadSynchronize(gpu_thread))
    assert not c.dpost.double().any() and not c.dpre.double().any()
    for d in (c.sum, c.y, c.z, c.ds, c.dres):
        assert bool((d.raw == 0xA5).all())


def test_in_place(gpu_thread):
    """y over the residual, the sum over the first partial; dSum over the sum, dResidual over dy."""
    a, b = Case(30, 500, "bf16", per=30), Case(30, 500, "bf16", per=30)
    torch.cuda.synchronize()
    h.check(a.forward(gpu_thread))
    h.check(b.forward(gpu_thread, y=b.residual.ptr, sum=b.x[0].ptr))
    h.check(h.HcommGfxThreadSynchronize(gpu_thread))
    assert torch.equal(a.y.view, b.residual.view) and torch.equal(a.sum.view, b.x[0].view) and torch.equal(a.z.view, b.z.view)
    da = a.gradient_desc()
    torch.cuda.synchronize()
    h.check(h.HcommGfxReduceNormGradOnThread(gpu_thread, da))
    h.check(h.HcommGfxThreadSynchronize(gpu_thread))
    want = [t.view.clone() for t in (a.ds, a.dres, a.dpost, a.dpre, a.dgate)]
    d = a.gradient_desc(dSum=a.sum.ptr, dResidual=a.dy.ptr)
    torch.cuda.synchronize()
    h.check(h.HcommGfxReduceNormGradOnThread(gpu_thread, d))
    h.check(h.HcommGfxThreadSynchronize(gpu_thread))
    for got, exp in zip((a.sum, a.dy, a.dpost, a.dpre, a.dgate), want):
        assert torch.equal(got.view, exp)


def test_large_values_and_a_row_of_zeros(gpu_thread):
    c = Case(5, 300, "fp32", scale=1e15, per=1)
    for x in c.x:
        x.view[2] = 0
    c.residual.view[2] = 0
    c.run(gpu_thread)


def test_a_nan_stays_in_its_row(gpu_thread):
    c = Case(6, 300, "bf16", per=6)
    c.x[1].view[3, 17] = float("nan")
    torch.cuda.synchronize()
    h.check(c.forward(gpu_thread))
    h.check(h.HcommGfxThreadSynchronize(gpu_thread))
    bad = np.isnan(c.y.double())
    assert bad[3].all() and not bad[[0, 1, 2, 4, 5]].any() and np.isnan(c.z.double())[3].all() and np.isnan(c.sum.double()).sum() == 1


def test_gradient_against_differences(gpu_thread):
    """A directional derivative of the library's own forward pass, in fp32: (f(v + e d) - f(v - e d)) / 2 e.  The difference
    quotient is off by e^2 times a third derivative and by the forward pass's roundings over e."""
    rows, cols, k, e = 4, 48, 2, 2.0 ** -8
    c = Case(rows, cols, "fp32", k=k, per=2)
    rng = np.random.default_rng(8)
    torch.cuda.synchronize()
    h.check(c.forward(gpu_thread))
    d = c.gradient_desc()
    torch.cuda.synchronize()
    h.check(h.HcommGfxReduceNormGradOnThread(gpu_thread, d))
    h.check(h.HcommGfxThreadSynchronize(gpu_thread))
    dy, dz = c.dy.double(), c.dz.double()
    parts = [(c.x[0], c.ds), (c.x[1], c.ds), (c.residual, c.dres), (c.post, c.dpost), (c.pre, c.dpre), (c.gate, c.dgate)]
    for what, grad in parts:
        way = rng.standard_normal(what.view.shape)
        before = what.view.clone()
        got = []
        for sign in (1, -1):
            what.view.copy_(before + sign * e * torch.from_numpy(way).float().cuda())
            torch.cuda.synchronize()
            h.check(c.forward(gpu_thread))
            h.check(h.HcommGfxThreadSynchronize(gpu_thread))
            got.append((c.y.double() * dy).sum() + (c.z.double() * dz).sum())
        what.view.copy_(before)
        want, is_ = (grad.double() * way).sum(), (got[0] - got[1]) / (2 * e)
        scale = np.abs(grad.double() * way).sum()
        assert abs(is_ - want) <= 2e-3 * scale, (is_, want, scale)


def test_captured_gradients_repeat_their_bits():
    c = Case(600, 520, "bf16", per=150)
    stream = torch.cuda.Stream()
    code, thread = h.HcommThreadAllocWithStream(stream.cuda_stream)
    h.check(code)
    d = c.gradient_desc()
    torch.cuda.synchronize()
    h.check(c.forward(thread))
    h.check(h.HcommGfxReduceNormGradOnThread(thread, d))
    torch.cuda.synchronize()
    outs = (c.sum, c.y, c.z, c.ds, c.dres, c.dpost, c.dpre, c.dgate)
    want = [o.raw.clone() for o in outs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        h.check(c.forward(thread))
        h.check(h.HcommGfxReduceNormGradOnThread(thread, d))
    for _ in range(3):
        for o in outs:
            o.raw.fill_(0xA5)
        c.work.fill_(0xFF)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o.raw, w) for o, w in zip(outs, want))
    h.HcommThreadFreeWithStream([thread])


def test_rows_past_32_bits(gpu_thread):
    """Rows 4 GiB apart in every matrix of the forward pass and the gradient."""
    rows, cols, far = 3, 40, (1 << 31) + 3
    rng = np.random.default_rng(4)
    big = torch.empty((rows - 1) * far + 16 * cols, dtype=torch.bfloat16, device="cuda")

    class Far:
        def __init__(self, i, v=None):
            self.view = torch.as_strided(big, (rows, cols), (far, 1), i * cols)
            self.ptr = big.data_ptr() + i * cols * 2
            if v is not None:
                self.view.copy_(torch.from_numpy(v).bfloat16())

        def double(self):
            return self.view.double().cpu().numpy()

        def guards_hold(self):
            return True
    c = Case(rows, cols, "bf16", k=1, per=1)
    n = lambda: rng.standard_normal((rows, cols))  # noqa: E731
    c.x, c.residual, c.gate, c.dy, c.dz = [Far(0, n())], Far(1, n()), Far(2, n()), Far(3, n()), Far(4, n())
    c.sum, c.y, c.z, c.ds, c.dres, c.dgate = (Far(i) for i in range(5, 11))
    c.stride = far
    c.run(gpu_thread)


@pytest.mark.parametrize("t,p", [("bf16", "bf16"), ("fp16", "fp32"), ("fp32", "fp32")])
def test_ends_of_rows(gpu_thread, t, p):
    """Every place in a group of eight elements at which a row can end, around the sizes at which another wavefront joins."""
    for cols in list(range(1, 18)) + [512 + d for d in range(-1, 9)] + [1030, 2047, 4099, 8193, 8198]:
        Case(4, cols, t, k=2, p=p, per=3, pad=1).run(gpu_thread)


@pytest.mark.parametrize("rows,per", [(6200, 2), (6149, 3), (700, 2), (1030, 257), (530, 0), (300, 1000), (9, 1), (1, 1)])
@pytest.mark.parametrize("cols,t,p", [(3, "fp16", "fp32"), (8, "fp32", "fp32"), (9, "bf16", "bf16"), (16, "fp16", "fp16"), (31, "bf16", "fp32"), (33, "fp32", "fp32"), (64, "bf16", "fp32"), (65, "fp32", "fp32"), (128, "fp16", "fp16"), (203, "bf16", "bf16"), (256, "fp32", "fp32"), (257, "bf16", "fp32")])
def test_rows_that_share_a_wavefront(gpu_thread, rows, per, cols, t, p):
    """1 to 32 lanes to a row and the first length of a wavefront of its own; gates inside a set of lanes' rows and across sets."""
    Case(rows, cols, t, k=2, per=per, p=p, pad=5 * (cols % 2)).run(gpu_thread)


@pytest.mark.parametrize("rows,per", [(530, 2), (519, 0), (260, 100)])
@pytest.mark.parametrize("cols,t,p", [(4104, "fp32", "fp32"), (6007, "bf16", "fp32"), (8192, "fp16", "fp16"), (8201, "bf16", "bf16"), (12296, "bf16", "fp32"), (16384, "fp32", "fp32")])
def test_more_rows_than_runs_of_long_ones(gpu_thread, rows, per, cols, t, p):
    Case(rows, cols, t, k=1, per=per, p=p).run(gpu_thread)


@pytest.mark.parametrize("cols", [40, 130, 4099, 8200, 16377])
@pytest.mark.parametrize("t", ["bf16", "fp32"])
def test_gradients_over_their_inputs(gpu_thread, cols, t):
    """dSum over the sum or dy, dResidual over dy or y: the bits of a call with outputs of its own."""
    a = Case(20, cols, t, k=1, per=3)
    torch.cuda.synchronize()
    h.check(a.forward(gpu_thread))
    h.check(h.HcommGfxReduceNormGradOnThread(gpu_thread, a.gradient_desc()))
    h.check(h.HcommGfxThreadSynchronize(gpu_thread))
    results = ("ds", "dres", "dpost", "dpre", "dgate")
    want = {n: getattr(a, n).view.clone() for n in results}
    for ds, dres in (("sum", "dy"), ("sum", "y"), ("dy", "y"), ("dy", "dres"), ("sum", "dres")):
        b = Case(20, cols, t, k=1, per=3)
        torch.cuda.synchronize()
        h.check(b.forward(gpu_thread))
        d = b.gradient_desc(dSum=getattr(b, ds).ptr, dResidual=getattr(b, dres).ptr)
        torch.cuda.synchronize()
        h.check(h.HcommGfxReduceNormGradOnThread(gpu_thread, d))
        h.check(h.HcommGfxThreadSynchronize(gpu_thread))
        for n, got in zip(results, (ds, dres, "dpost", "dpre", "dgate")):
            assert torch.equal(getattr(b, got).view, want[n]), (ds, dres, n)


@pytest.mark.parametrize("power", [0, -60, 50])
def test_small_and_large_rows_without_eps(gpu_thread, power):
    """1 / rms scales with the row: means of squares of 2^-120 and 2^100 and eps = 0 leave z as it is for rows around 1."""
    rows, cols = 3, 200
    rng = np.random.default_rng(11)
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    src, y, z = Dense(rows, cols, "fp32", cols, 0, x.astype(np.float64) * 2.0 ** power), Dense(rows, cols, "fp32"), Dense(rows, cols, "fp32")
    w = Dense(1, cols, "fp32", cols, 0, 1 + 0.2 * rng.standard_normal((1, cols)))
    d = h.ReduceNormDesc(srcs=[src.ptr], srcStride=cols, rows=rows, cols=cols, dataType=h.HcommDataType.FP32, paramType=h.HcommDataType.FP32,
                         residualScale=1.0, eps=0.0, y=y.ptr, yStride=cols, z=z.ptr, zStride=cols, preWeight=w.ptr)
    torch.cuda.synchronize()
    h.check(h.HcommGfxReduceNormOnThread(gpu_thread, d))
    h.check(h.HcommGfxThreadSynchronize(gpu_thread))
    v = x.astype(np.float64)
    want = v / np.sqrt((v * v).mean(1, keepdims=True)) * w.double()
    close(z.double(), want, "fp32", np.abs(want) * (RHO + 2 * U), "z")
    assert np.array_equal(y.double(), v * 2.0 ** power)


@pytest.mark.parametrize("rows,per", [(536, 1), (300, 2), (1999, 3), (255, 9), (1300, 20), (5, 4)])
@pytest.mark.parametrize("cols,t,p", [(20, "fp32", "fp32"), (132, "fp16", "fp16"), (626, "bf16", "fp32"), (5001, "bf16", "bf16"), (9000, "fp32", "fp32")])
def test_a_row_of_the_gate_in_one_run(gpu_thread, rows, per, cols, t, p):
    """Fewer gate rows than runs, each with so few rows that one run has them all."""
    Case(rows, cols, t, k=1, per=per, p=p, pad=cols % 3).run(gpu_thread)
