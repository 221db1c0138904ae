"""The operators around a fold in 64 bits, from their formulas alone (numpy; nothing of the library)."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = 32
EPS_HALF = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}  # half a step, relative


def blocks_of(cols):
    return -(-cols // BLOCK)


def mx_encode(v):
    """v [rows, cols] float64 -> (codes [rows, blocks, 32] 0..15, scales [rows, blocks] 0..255)."""
    rows, cols = v.shape
    nb = blocks_of(cols)
    w = np.zeros((rows, nb * BLOCK))
    w[:, :cols] = v
    w = w.reshape(rows, nb, BLOCK)
    bad = ~np.isfinite(w).all(-1)
    w = np.where(bad[..., None], 0.0, w)
    top = np.abs(w).max(-1)
    with np.errstate(divide="ignore"):
        e = np.frexp(top)[1] - 1                      # 2^e <= top < 2^(e+1)
    s = np.where(top > 0, np.clip(e - 2 + 127, 0, 252), 0)
    a = np.abs(w) / np.ldexp(1.0, s - 127)[..., None]
    mid = (GRID[1:] + GRID[:-1]) / 2
    below = np.searchsorted(mid, a, side="left")     # middles that lie below a: a tie stays at the lower element
    upto = np.searchsorted(mid, a, side="right")     # ... or goes to the upper one
    code = np.where(below % 2 == 0, below, upto)
    code = code + 8 * np.signbit(w)
    code = np.where(bad[..., None], 0, code)
    return code.astype(np.uint8), np.where(bad, 255, s).astype(np.uint8)


def mx_values(code, s, cols):
    v = np.where(code >= 8, -1.0, 1.0) * GRID[code & 7] * np.ldexp(1.0, s.astype(np.int64) - 127)[..., None]
    v = np.where((s == 255)[..., None], np.nan, v)
    return v.reshape(v.shape[0], -1)[:, :cols]


def mx_pack(code):
    return (code[..., 0::2] | (code[..., 1::2] << 4)).astype(np.uint8)


def mx_unpack(packed):
    return np.stack((packed & 15, packed >> 4), -1).reshape(*packed.shape[:-1], BLOCK)


def norm(x, residual, alpha, eps, post=None, pre=None, gate=None, per=1):
    """x [k, rows, cols] -> s, y, z (None without pre)."""
    s = x[0].copy()
    for p in x[1:]:
        s = s + p
    h = s if post is None else s / np.sqrt((s * s).mean(1, keepdims=True) + eps) * post
    if gate is not None:
        h = h * gate[np.arange(s.shape[0]) // per]
    y = h if residual is None else alpha * residual + h
    z = None if pre is None else y / np.sqrt((y * y).mean(1, keepdims=True) + eps) * pre
    return s, y, z


def norm_grad(s, y, dy, dz, alpha, eps, post=None, pre=None, gate=None, per=1):
    """The vector-Jacobian products of norm() at the stored s and y."""
    out = {}
    total = dy.copy()
    if pre is not None:
        q = (y * y).mean(1, keepdims=True) + eps
        total += pre * dz / np.sqrt(q) - y * q ** -1.5 * (pre * dz * y).mean(1, keepdims=True)
        out["pre"] = (dz * y / np.sqrt(q)).sum(0)
    out["residual"] = alpha * total
    q = (s * s).mean(1, keepdims=True) + eps
    h = s if post is None else s / np.sqrt(q) * post
    d = total
    if gate is not None:
        index = np.arange(s.shape[0]) // per
        dg = np.zeros_like(gate)
        np.add.at(dg, index, total * h)
        out["gate"] = dg
        d = total * gate[index]
    if post is not None:
        out["post"] = (d * s / np.sqrt(q)).sum(0)
        d = d * post
        d = d / np.sqrt(q) - s * q ** -1.5 * (d * s).mean(1, keepdims=True)
    out["sum"] = d
    return out
