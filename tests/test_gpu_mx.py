"""Messages in microscaled 4-bit floating point against the format's definition in 64 bits (tests/ops_reference.py).

Quantising and the fold are compared exactly: codes and scales bit for bit, dense results within the one rounding to the
output's type.  The product's bound: every one of its additions loses at most one step of fp32 of the sum of magnitudes."""
import numpy as np
import pytest
import torch

import hcomm_amd as h
import ops_reference as ref
from ops_util import DT, Dense, Mx, close, random_mx

pytestmark = pytest.mark.gpu

TYPES = ["bf16", "fp16", "fp32"]


def sync(t):
    h.check(h.HcommGfxThreadSynchronize(t))


def ready():
    torch.cuda.synchronize()  # the inputs were made on torch's stream


def awkward(rows, cols, t, rng):
    """Values that meet every branch of the format: ties, saturation, zeros of both signs, far exponents, subnormals."""
    v = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-12, 12, (rows, cols)))
    pick = rng.integers(0, 8, (rows, cols))
    v = np.where(pick == 0, np.round(v * 4) / 4, v)                                   # many ties
    v = np.where(pick == 1, 0.0, v)
    v = np.where(pick == 2, -0.0, v)
    v = np.where(pick == 3, rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.75], (rows, cols)) * rng.choice([-1, 1], (rows, cols)), v)
    for b in range(0, cols, 32):                                                      # some blocks: all zero, tiny, subnormal, huge
        kind = rng.integers(0, 8)
        part = slice(b, b + 32)
        if kind == 0:
            v[:, part] = 0.0
        elif kind == 1:
            v[:, part] *= {"bf16": 2.0 ** -120, "fp16": 2.0 ** -12, "fp32": 2.0 ** -130}[t]
        elif kind == 2:
            v[:, part] *= {"bf16": 2.0 ** 100, "fp16": 2.0 ** 1, "fp32": 2.0 ** 104}[t]
    return v


SHAPES = [(1, 1), (1, 31), (1, 32), (3, 33), (5, 1), (3, 100), (1025, 7), (77, 1009), (1, 8191), (2, 8232), (3, 9000), (1, 100003), (255, 257)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize(gpu_thread, rows, cols, t):
    rng = np.random.default_rng(rows * 1000003 + cols)
    for stride, offset, pad, shift in ((cols, 0, 0, 0), (cols + 5, 3, 2, 1)):
        src = Dense(rows, cols, t, stride, offset, awkward(rows, cols, t, rng))
        out = Mx(rows, cols, pad, shift)
        ready()
        h.check(h.HcommGfxMxQuantizeOnThread(gpu_thread, h.mx_views([out.item]), src.ptr, src.stride, rows, cols, DT[t]))
        sync(gpu_thread)
        code, scale = ref.mx_encode(src.double())
        assert np.array_equal(out.scale(), scale)
        assert np.array_equal(out.code(), code)
        assert out.guards_hold() and src.guards_hold()


@pytest.mark.parametrize("t", TYPES)
def test_quantize_infinities_and_nan(gpu_thread, t):
    v = np.random.default_rng(5).standard_normal((4, 160))
    v[0, 0], v[0, 40], v[1, 64:96], v[2, 159], v[3, 31] = np.inf, np.nan, -np.inf, -np.nan, np.inf
    src, out = Dense(4, 160, t, values=v), Mx(4, 160)
    ready()
    h.check(h.HcommGfxMxQuantizeOnThread(gpu_thread, h.mx_views([out.item]), src.ptr, 160, 4, 160, DT[t]))
    sync(gpu_thread)
    code, scale = ref.mx_encode(src.double())
    assert (scale == 255).sum() == 5 and np.array_equal(out.scale(), scale) and np.array_equal(out.code(), code)


@pytest.mark.parametrize("t", ["bf16", "fp16"])
def test_quantize_every_value_of_a_sixteen_bit_type(gpu_thread, t):
    """All 65,536 patterns as the largest of a block and, shuffled, beside others."""
    bits = np.arange(65536, dtype=np.uint16)
    shuffled = np.random.default_rng(1).permutation(bits)
    alone = np.zeros((65536, 32), np.uint16)
    alone[:, 7] = bits
    for b in (alone, shuffled.reshape(1, -1)):
        rows, cols = b.shape
        src, out = Dense(rows, cols, t), Mx(rows, cols)
        src.raw[:b.size * 2].copy_(torch.from_numpy(b.reshape(-1).view(np.uint8).copy()))
        ready()
        h.check(h.HcommGfxMxQuantizeOnThread(gpu_thread, h.mx_views([out.item]), src.ptr, cols, rows, cols, DT[t]))
        sync(gpu_thread)
        code, scale = ref.mx_encode(src.double())
        assert np.array_equal(out.scale(), scale) and np.array_equal(out.code(), code)


@pytest.mark.parametrize("rows,cols,k", [(1, 1, 1), (3, 33, 2), (1, 8191, 7), (77, 1009, 8), (2, 8232, 9), (5, 100, 17), (300, 70, 32), (1, 70000, 3)])
@pytest.mark.parametrize("t", TYPES)
def test_fold(gpu_thread, rows, cols, k, t):
    """dst alone, again alone, both, with and without the addend; garbage past the row's end in the inputs' last blocks."""
    rng = np.random.default_rng(rows + 31 * cols + 1007 * k)
    for want_dst, want_again, want_addend, spread in ((1, 0, 0, 6), (1, 1, 1, 12), (0, 1, 0, 17), (1, 1, 0, 30)):
        # scales around 1 keep fp16 in range; 30 apart is beyond an fp32 sum and exact in fp64
        unit = 112 if t == "fp16" else 100
        spread = min(spread, 16) if t == "fp16" else spread
        src = [random_mx(rows, cols, rng, j % 3, j % 4, spread, unit, tail=0xF if j % 2 else 0x7) for j in range(k)]
        addend = Dense(rows, cols, t, cols + 3, 1, rng.standard_normal((rows, cols)) * 2.0 ** (unit - 120)) if want_addend else None
        dst = Dense(rows, cols, t, cols + 1, 2) if want_dst else None
        again = Mx(rows, cols, 1, 3) if want_again else None
        ready()
        h.check(h.HcommGfxMxReduceKOnThread(
            gpu_thread, dst.ptr if dst else None, dst.stride if dst else 0, DT[t], h.mx_views([again.item]) if again else None,
            h.mx_views([x.item for x in src]), k, addend.ptr if addend else None, addend.stride if addend else 0, rows, cols))
        sync(gpu_thread)
        v = addend.double() if addend else np.zeros((rows, cols))
        for x in src:
            v = v + x.values()
        if dst:
            close(dst.double(), v, t, 0.0, "dst")
            assert dst.guards_hold()
        if again:
            code, scale = ref.mx_encode(v)
            got = again.code()
            zero = (code & 7) == 0  # the sign of a sum of zeros is not part of the contract
            assert np.array_equal(again.scale(), scale) and np.array_equal(got[~zero], code[~zero]) and not (got[zero] & 7).any()
            assert again.guards_hold()


def test_fold_scales_far_apart_and_at_the_ends_of_their_range(gpu_thread):
    """Scales from 0 to 254: sums in fp64 of fp32 contributions, infinite where those are; 255 makes its block NaN alone."""
    rng = np.random.default_rng(11)
    rows, cols, k = 64, 96, 6
    src = [random_mx(rows, cols, rng, unit=0, spread=252) for _ in range(k)]
    special = Mx(rows, cols, code=rng.integers(0, 16, (rows, 3, 32)).astype(np.uint8),
                 scale=rng.choice(np.array([0, 1, 2, 250, 253, 254, 255], np.uint8), (rows, 3)))
    src.append(special)
    dst = Dense(rows, cols, "fp32")
    ready()
    h.check(h.HcommGfxMxReduceKOnThread(gpu_thread, dst.ptr, cols, DT["fp32"], None, h.mx_views([x.item for x in src]), k + 1, None, 0, rows, cols))
    sync(gpu_thread)
    with np.errstate(over="ignore", invalid="ignore"):
        parts = [x.values().astype(np.float32).astype(np.float64) for x in src]
        v = parts[0]
        for p in parts[1:]:
            v = v + p
        want = v.astype(np.float32)
    got = dst.view.cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(want).any() and np.isinf(want).any()
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    # fp64 additions of seven terms and one rounding to fp32
    magnitude = sum(np.abs(p) for p in parts)[fine]
    assert (np.abs(got[fine].astype(np.float64) - v[fine]) <= 7 * 2.0 ** -53 * magnitude + np.abs(v[fine]) * 2.0 ** -24 + 2.0 ** -150).all()


@pytest.mark.parametrize("t", TYPES)
def test_dequantize_keeps_every_value(gpu_thread, t):
    """k = 1: all 16 elements under every scale the type can hold, signs of zeros included."""
    lo, hi = {"bf16": (0, 252), "fp32": (0, 252), "fp16": (104, 138)}[t]
    scale = np.arange(lo, hi + 1, dtype=np.uint8).reshape(-1, 1)
    code = np.tile(np.arange(32, dtype=np.uint8) % 16, (len(scale), 1, 1))
    src, dst = Mx(len(scale), 32, code=code, scale=scale), Dense(len(scale), 32, t)
    ready()
    h.check(h.HcommGfxMxReduceKOnThread(gpu_thread, dst.ptr, 32, DT[t], None, h.mx_views([src.item]), 1, None, 0, len(scale), 32))
    sync(gpu_thread)
    assert np.array_equal(dst.double(), src.values()) and np.array_equal(np.signbit(dst.double()), np.signbit(src.values()))


def test_fold_into_the_addend(gpu_thread):
    rng = np.random.default_rng(3)
    src = [random_mx(9, 200, rng, unit=120) for _ in range(4)]
    own = Dense(9, 200, "bf16", 203, 1, rng.standard_normal((9, 200)))
    v = own.double() + sum(x.values() for x in src)
    ready()
    h.check(h.HcommGfxMxReduceKOnThread(gpu_thread, own.ptr, 203, DT["bf16"], None, h.mx_views([x.item for x in src]), 4, own.ptr, 203, 9, 200))
    sync(gpu_thread)
    close(own.double(), v, "bf16", 0.0, "dst")
    assert own.guards_hold()


def product_case(thread, m, n, cols, k, t, rng, pad=0, shift=0, tail=None, stride=0):
    a = [random_mx(m, cols, rng, pad, shift, unit=120, tail=tail) for _ in range(k)]
    b = [random_mx(n, cols, rng, pad * 2, shift + 1, unit=116, tail=tail) for _ in range(k)]
    dst = Dense(m, n, t, n + stride, stride)
    ready()
    h.check(h.HcommGfxMxProductKOnThread(thread, dst.ptr, dst.stride, DT[t], h.mx_views([x.item for x in a]), h.mx_views([x.item for x in b]), k, m, n, cols))
    sync(thread)
    want, magnitude = np.zeros((m, n)), np.zeros((m, n))
    for x, y in zip(a, b):
        p, q = x.values(), y.values()
        want += p @ q.T
        magnitude += np.abs(p) @ np.abs(q).T
    close(dst.double(), want, t, k * cols * 2.0 ** -23 * magnitude, "dst")
    assert dst.guards_hold()


PRODUCTS = [(1, 1, 1, 1), (1, 16, 32, 1), (1, 17, 33, 2), (5, 40, 100, 3), (16, 16, 512, 1), (16, 15, 544, 32), (17, 33, 513, 2), (33, 31, 31, 5),
            (1, 300, 4096, 8), (40, 100, 1009, 3), (64, 64, 2048, 1), (100, 130, 96, 9), (129, 257, 700, 2), (300, 520, 256, 1), (257, 255, 1500, 3),
            (513, 700, 1024, 1), (520, 1030, 2080, 2)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,cols,k", PRODUCTS)
def test_product(gpu_thread, m, n, cols, k, t):
    rng = np.random.default_rng(m + 7 * n + 31 * cols + k)
    product_case(gpu_thread, m, n, cols, k, t, rng)
    product_case(gpu_thread, m, n, cols, k, t, rng, pad=1, shift=1, tail=0xF, stride=3)


@pytest.mark.parametrize("m,n,cols", [(3, 40, 200), (200, 300, 520), (600, 600, 600)])
def test_product_of_a_block_that_is_nan(gpu_thread, m, n, cols):
    """Scale 255 makes the row of a (or of b) NaN and nothing else; bytes behind a row's scales are not read as scales."""
    rng = np.random.default_rng(1)
    a, b = random_mx(m, cols, rng, 1, 0, unit=120), random_mx(n, cols, rng, 1, 0, unit=120)
    a.scales.fill_(255), b.scales.fill_(255)  # the padding too
    sa, sb = np.full((m, a.nb), 120, np.uint8), np.full((n, b.nb), 121, np.uint8)
    sa[m // 2, -1], sb[n - 1, 0] = 255, 255
    a._scales().copy_(torch.from_numpy(sa)), b._scales().copy_(torch.from_numpy(sb))
    dst = Dense(m, n, "fp32")
    ready()
    h.check(h.HcommGfxMxProductKOnThread(gpu_thread, dst.ptr, n, DT["fp32"], h.mx_views([a.item]), h.mx_views([b.item]), 1, m, n, cols))
    sync(gpu_thread)
    nan = np.zeros((m, n), bool)
    nan[m // 2], nan[:, n - 1] = True, True
    got = dst.double()
    assert np.array_equal(np.isnan(got), nan)
    with np.errstate(invalid="ignore"):
        want = np.nan_to_num(a.values()) @ np.nan_to_num(b.values()).T
    assert (np.abs(got - want)[~nan] <= cols * 2.0 ** -22 * 36 * 4 * cols * 2.0 ** -13).all()


def test_offsets_past_32_bits(gpu_thread):
    """Rows more than 4 GiB apart, in every dense and packed operand that may be."""
    rows, cols, far = 3, 70, (1 << 31) + 11
    rng = np.random.default_rng(2)
    v = rng.standard_normal((rows, cols))
    big = torch.empty((rows - 1) * far + cols, dtype=torch.bfloat16, device="cuda")
    src = torch.as_strided(big, (rows, cols), (far, 1))
    src.copy_(torch.from_numpy(v).bfloat16())
    step = (1 << 32) + 16
    packed, scales = (torch.empty((rows - 1) * step + 64, dtype=torch.uint8, device="cuda") for _ in range(2))
    views = h.mx_views([(packed.data_ptr(), step, scales.data_ptr(), step)])
    ready()
    h.check(h.HcommGfxMxQuantizeOnThread(gpu_thread, views, big.data_ptr(), far, rows, cols, DT["bf16"]))
    sync(gpu_thread)
    code, scale = ref.mx_encode(src.double().cpu().numpy())
    assert np.array_equal(torch.as_strided(scales, (rows, 3), (step, 1)).cpu().numpy(), scale)
    assert np.array_equal(torch.as_strided(packed, (rows, 3, 16), (step, 16, 1)).cpu().numpy(), ref.mx_pack(code))
    h.check(h.HcommGfxMxReduceKOnThread(gpu_thread, big.data_ptr(), far, DT["bf16"], None, views, 1, None, 0, rows, cols))
    sync(gpu_thread)
    assert np.array_equal(src.double().cpu().numpy(), ref.mx_values(code, scale, cols))
    a = random_mx(rows, 64, rng, unit=120)
    b = random_mx(cols, 64, rng, unit=120)
    h.check(h.HcommGfxMxProductKOnThread(gpu_thread, big.data_ptr(), far, DT["bf16"], h.mx_views([a.item]), h.mx_views([b.item]), 1, rows, cols, 64))
    sync(gpu_thread)
    close(src.double().cpu().numpy(), a.values() @ b.values().T, "bf16", 64 * 2.0 ** -23 * (np.abs(a.values()) @ np.abs(b.values()).T), "dst")


def test_two_streams_and_a_graph_give_the_eager_bits():
    """The three operators on a stream of torch's, captured and replayed between eager calls on another thread."""
    rng = np.random.default_rng(9)
    rows, cols, n, k = 40, 1000, 90, 3
    x = [Dense(rows, cols, "bf16", values=rng.standard_normal((rows, cols))) for _ in range(k)]
    w = [random_mx(n, cols, rng, unit=118) for _ in range(k)]
    wv = h.mx_views([y.item for y in w])

    def buffers():
        return [Mx(rows, cols) for _ in range(k)], Dense(rows, cols, "fp32"), Dense(rows, n, "bf16"), Mx(rows, cols)

    def calls(thread, to):
        q, total, out, again = to
        views, av = h.mx_views([y.item for y in q]), h.mx_views([again.item])
        for j in range(k):
            one = h.mx_views([q[j].item])
            h.check(h.HcommGfxMxQuantizeOnThread(thread, one, x[j].ptr, cols, rows, cols, DT["bf16"]))
        h.check(h.HcommGfxMxReduceKOnThread(thread, total.ptr, cols, DT["fp32"], av, views, k, None, 0, rows, cols))
        h.check(h.HcommGfxMxProductKOnThread(thread, out.ptr, n, DT["bf16"], views, wv, k, rows, n, cols))
        return views, av

    eager, graphed, other = buffers(), buffers(), buffers()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    threads = [h.HcommThreadAllocWithStream(s.cuda_stream)[1] for s in streams]
    torch.cuda.synchronize()
    calls(threads[0], eager)
    torch.cuda.synchronize()
    want = [t.clone() for t in (eager[1].raw, eager[2].raw, eager[3].packed, eager[3].scales)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        keep = calls(threads[0], graphed)
    for step in range(3):
        for to in (graphed, other):
            to[1].raw.fill_(0xA5), to[2].raw.fill_(0xA5), to[3].packed.fill_(0xA5), to[3].scales.fill_(0xA5)
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            graph.replay()
        calls(threads[1], other)
        torch.cuda.synchronize()
        for to in (graphed, other):
            for got, exp in zip((to[1].raw, to[2].raw, to[3].packed, to[3].scales), want):
                assert torch.equal(got, exp), step
    del keep
    h.HcommThreadFreeWithStream(threads)


@pytest.mark.parametrize("t", TYPES)
def test_ends_of_rows(gpu_thread, t):
    """Every place in a block at which a row can end, in rows shorter than a group, long ones and ones just past a workgroup's
    piece; what lies in front of a row is not part of it."""
    rng = np.random.default_rng(6)
    for cols in list(range(1, 42)) + [2048 + d for d in (0, 1, 3, 7, 8, 9)] + [8192 + d for d in (1, 5, 31, 33)]:
        rows = 3
        src = Dense(rows, cols, t, cols + 9, 5, awkward(rows, cols, t, rng))
        out, total = Mx(rows, cols, 1), Dense(rows, cols, t, cols + 2, 1)
        ready()
        view = h.mx_views([out.item])
        h.check(h.HcommGfxMxQuantizeOnThread(gpu_thread, view, src.ptr, src.stride, rows, cols, DT[t]))
        h.check(h.HcommGfxMxReduceKOnThread(gpu_thread, total.ptr, total.stride, DT[t], None, view, 1, src.ptr, src.stride, rows, cols))
        sync(gpu_thread)
        code, scale = ref.mx_encode(src.double())
        assert np.array_equal(out.scale(), scale) and np.array_equal(out.code(), code), cols
        close(total.double(), src.double() + ref.mx_values(code, scale, cols), t, 0.0, cols)
        assert out.guards_hold() and total.guards_hold()


@pytest.mark.parametrize("m,n,cols,k", [(70, 90, 480, 2), (70, 90, 481, 1), (70, 200, 1009, 3), (130, 140, 2080, 2), (300, 400, 500, 3), (400, 300, 2049, 2)])
def test_product_of_ranks_with_strides_of_their_own(gpu_thread, m, n, cols, k):
    """Every rank's matrices padded by another number of blocks, then the same sizes with equal strides."""
    rng = np.random.default_rng(m + n + cols)
    for pads in ([0] * k, list(range(k))):
        a = [random_mx(m, cols, rng, p, p, unit=120, tail=0x5) for p in pads]
        b = [random_mx(n, cols, rng, 2 * p, p, unit=118, tail=0xD) for p in pads]
        dst = Dense(m, n, "fp32", n + 1, 1)
        ready()
        h.check(h.HcommGfxMxProductKOnThread(gpu_thread, dst.ptr, n + 1, DT["fp32"], h.mx_views([x.item for x in a]), h.mx_views([x.item for x in b]), k, m, n, cols))
        sync(gpu_thread)
        want = sum(x.values() @ y.values().T for x, y in zip(a, b))
        magnitude = sum(np.abs(x.values()) @ np.abs(y.values()).T for x, y in zip(a, b))
        close(dst.double(), want, "fp32", k * cols * 2.0 ** -23 * magnitude, "dst")
        assert dst.guards_hold()


AROUND = [(rows, cols) for rows in (1, 3, 300) for cols in (992, 1024, 1025, 1056, 2048, 2049, 4064, 4096, 4097, 8193)]


@pytest.mark.parametrize("rows,cols", AROUND + [(140000, 33), (8300, 1000), (2100, 4090), (1100, 4100)])
def test_rows_around_what_a_workgroup_holds(gpu_thread, rows, cols):
    """One row, a few and many of the lengths at which a workgroup goes from several rows to one and to pieces of one, and
    the fold of what was quantised with itself."""
    rng = np.random.default_rng(rows + cols)
    src = Dense(rows, cols, "bf16", cols + 1, 1, rng.standard_normal((rows, cols)))
    out, dst, again = Mx(rows, cols, 1, 1), Dense(rows, cols, "fp32", cols + 2, 1), Mx(rows, cols, 2, 3)
    ready()
    h.check(h.HcommGfxMxQuantizeOnThread(gpu_thread, h.mx_views([out.item]), src.ptr, src.stride, rows, cols, DT["bf16"]))
    h.check(h.HcommGfxMxReduceKOnThread(gpu_thread, dst.ptr, dst.stride, DT["fp32"], h.mx_views([again.item]), h.mx_views([out.item] * 2), 2, None, 0,
                                        rows, cols))
    sync(gpu_thread)
    code, scale = ref.mx_encode(src.double())
    assert np.array_equal(out.scale(), scale) and np.array_equal(out.code(), code) and out.guards_hold()
    twice = 2 * out.values()
    assert np.array_equal(dst.double(), twice) and dst.guards_hold()
    assert np.array_equal(again.values(), ref.mx_values(*ref.mx_encode(twice), cols)) and again.guards_hold()


SHORT = [(600, 700, 32, 1), (600, 700, 33, 3), (600, 700, 200, 9), (520, 1030, 224, 32), (1100, 600, 100, 17), (2050, 2050, 97, 2), (900, 1100, 128, 4),
         (1500, 1600, 250, 2), (600, 700, 300, 5), (1500, 1600, 470, 2), (1400, 4100, 256, 1), (2050, 2300, 300, 3)]


@pytest.mark.parametrize("m,n,cols,k", SHORT)
def test_product_of_short_rows(gpu_thread, m, n, cols, k):
    """Many results of one to fifteen blocks a rank."""
    product_case(gpu_thread, m, n, cols, k, "bf16", np.random.default_rng(m + n + cols), pad=2, shift=3, tail=0xE, stride=1)


@pytest.mark.parametrize("m,n,cols", [(600, 800, 40), (600, 800, 220), (700, 800, 250), (1500, 1600, 400), (1400, 4100, 300)])
def test_product_of_short_rows_with_nan(gpu_thread, m, n, cols):
    test_product_of_a_block_that_is_nan(gpu_thread, m, n, cols)
