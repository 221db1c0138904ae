"""What is measured of the operators around a rank fold: messages in microscaled 4-bit floating point (quantised, folded,
multiplied) and the norms, gate and residual behind a tensor-parallel fold, with their gradient.

The plain forms are elementary torch operations in fp32; with ``own`` set the same passes go through the library's
entry points on a thread bound to torch's current stream."""
import math

import torch

own = False

BLOCK = 32  # elements that share a scale
BLOCK_BYTES = 17  # sixteen of elements, one of scale
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5
ALPHA = 0.75  # the residual's scale


def listed():
    return [
        # a ragged decode batch's activations on their way into a product: small, rows that end inside a block
        {"name": "quantize_ragged", "op": "quantize", "rows": 77, "cols": 5005, "type": "fp16"},
        # a 128 MiB rank message of gradients (the headline allreduce's message)
        {"name": "quantize_message", "op": "quantize", "rows": 1, "cols": 67108864, "type": "bf16"},
        # eight ranks' small messages folded: a decode step's allreduce
        {"name": "fold_small", "op": "fold", "k": 8, "rows": 1, "cols": 16384, "type": "bf16", "addend": False, "requant": False},
        # the slice a rank owns of the headline message (16 MiB of bf16): its own share in full precision, the others'
        # quantised, the result quantised again for the gather
        {"name": "fold_slice", "op": "fold", "k": 7, "rows": 1, "cols": 8388608, "type": "bf16", "addend": True, "requant": True},
        # a seven-rank reduce-scatter slice of 100,000,003 elements: no power of two anywhere
        {"name": "fold_odd", "op": "fold", "k": 7, "rows": 1, "cols": 14285715, "type": "fp32", "addend": False, "requant": False},
        # a row-parallel layer over eight ranks: one token, the weights are read once
        {"name": "product_token", "op": "product", "k": 8, "m": 1, "n": 8192, "cols": 1024, "type": "bf16"},
        # a ragged decode batch on odd lengths
        {"name": "product_ragged", "op": "product", "k": 3, "m": 77, "n": 5003, "cols": 1009, "type": "fp32"},
        # the same layer on a prompt
        {"name": "product_prompt", "op": "product", "k": 8, "m": 4096, "n": 8192, "cols": 1024, "type": "bf16"},
        # behind the fold of a decode step: one row
        {"name": "norm_token", "op": "norm", "k": 8, "rows": 1, "cols": 8192, "type": "bf16", "post": True, "pre": True, "gate": 1},
        # behind the fold of a training step, the sum kept for the gradient; one learned gate for all rows
        {"name": "norm_train", "op": "norm", "k": 8, "rows": 8192, "cols": 4096, "type": "bf16", "post": True, "pre": True, "gate": 8192},
        # gradients with a gate for each sample of a batch, odd sizes, the last sample shorter
        {"name": "norm_grad_samples", "op": "norm_grad", "rows": 1333, "cols": 1001, "type": "fp16", "post": True, "pre": True, "gate": 100},
        # the gradient of norm_train
        {"name": "norm_grad_train", "op": "norm_grad", "rows": 8192, "cols": 4096, "type": "bf16", "post": True, "pre": True, "gate": 8192},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "fold", "product", "norm", "norm_grad"])
    case = {"op": op, "type": rng.choice(sorted(TYPES))}
    if op == "quantize":
        case["rows"] = rng.choice([1, _spread(rng, 1, 4096)])
        case["cols"] = _spread(rng, 1, (1 << 25) // case["rows"])
    elif op == "fold":
        case["k"] = rng.randint(1, 16)
        case["rows"] = rng.choice([1, _spread(rng, 1, 1024)])
        case["cols"] = _spread(rng, 1, (1 << 26) // (case["rows"] * case["k"]))
        case["addend"] = rng.random() < 0.5
        case["requant"] = rng.random() < 0.5
    elif op == "product":
        case["k"] = rng.choice([1, rng.randint(1, 16)])
        case["m"] = _spread(rng, 1, 4096)
        case["n"] = _spread(rng, 1, 8192)
        case["cols"] = _spread(rng, 1, 8192 // case["k"])
    else:
        if op == "norm":
            case["k"] = rng.randint(1, 16)
        case["cols"] = _spread(rng, 16, 16384)
        case["rows"] = _spread(rng, 1, (1 << 25) // case["cols"])
        case["post"] = rng.random() < 0.75
        case["pre"] = rng.random() < 0.75
        # rows that share a row of gates: none (no gate), one each, a sample's, all
        case["gate"] = rng.choice([0, 1, _spread(rng, 1, case["rows"]), case["rows"]])
    return case


def work(case):
    u = SIZE[case["type"]]
    if case["op"] == "product":
        k, m, n, cols = case["k"], case["m"], case["n"], case["cols"]
        blocks = k * (m + n) * -(-cols // BLOCK)
        return {"bytes": blocks * BLOCK_BYTES + m * n * u, "flops": 2 * m * n * k * cols}
    el = case["rows"] * case["cols"]
    packed = case["rows"] * -(-case["cols"] // BLOCK) * BLOCK_BYTES
    if case["op"] == "quantize":  # read, the packed form written, its values written
        return {"bytes": el * u + packed + el * 2, "flops": 4 * el}
    if case["op"] == "fold":
        k = case["k"]
        out = el * u + (packed + el * 2 if case["requant"] else 0)
        return {"bytes": k * packed + (el * u if case["addend"] else 0) + out, "flops": 2 * k * el}
    gates = -(-case["rows"] // case["gate"]) * case["cols"] if case["gate"] else 0
    params = gates + case["cols"] * (case["post"] + case["pre"])
    if case["op"] == "norm":  # the partials and the residual; the sum, y and (with a norm in front of the next block) z
        return {"bytes": (el * (case["k"] + 1 + 2 + case["pre"]) + params) * u, "flops": (case["k"] + 12) * el}
    # s, y, dy (and dz) in, ds and the residual's gradient out; parameters in, their gradients out
    return {"bytes": (el * (3 + case["pre"] + 2) + 2 * params) * u, "flops": 30 * el}


# ---- microscaled 4-bit floating point, plain -------------------------------------------------------------------------


def _power(e):
    """2^e as fp32 for -127 <= e <= 127, by its bits (2^-127 is subnormal)."""
    e = e.to(torch.int32)
    return torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).view(torch.float32)


def _encode(x):
    """x [..., rows, cols] -> (elements [..., rows, blocks, 16], scales [..., rows, blocks]), both uint8.  Sums come in
    fp64: many of them lie in the middle between two elements, where the last bit of an fp32 sum would decide."""
    cols = x.shape[-1]
    blocks = -(-cols // BLOCK)
    x = x if x.dtype == torch.float64 else x.float()
    v = torch.nn.functional.pad(x, (0, blocks * BLOCK - cols)).reshape(*x.shape[:-1], blocks, BLOCK)
    amax = v.abs().amax(-1)
    bad = ~torch.isfinite(amax)
    scale = torch.where(amax > 0, torch.frexp(amax)[1] + (127 - 1 - 2), 0).clamp(0, 252)
    v = v * _power(127 - scale)[..., None]
    a = v.abs().clamp(max=6.0)
    code = torch.where(a < 2, torch.round(a * 2), torch.where(a < 4, torch.round(a) + 2, torch.round(a / 2) + 4))
    code = torch.where(bad[..., None], torch.zeros_like(code), code + 8 * torch.signbit(v)).to(torch.uint8)
    scale = torch.where(bad, torch.full_like(scale, 255), scale).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def _decode(packed, scale, cols):
    """The fp32 values [..., rows, cols] of packed elements and scales."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=packed.device)
    e = torch.stack((packed & 15, packed >> 4), -1).reshape(*packed.shape[:-1], BLOCK)
    f = torch.where(scale == 255, torch.full_like(scale, 0, dtype=torch.float32) / 0, _power(scale.to(torch.int32) - 127))
    v = table[e.to(torch.int32)] * f[..., None]
    return v.reshape(*v.shape[:-2], -1)[..., :cols]


# ---- inputs ----------------------------------------------------------------------------------------------------------


def _normal(shape, gen, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda") * scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, t = case["op"], TYPES[case["type"]]
    s = {"op": op, "case": case, "plan": None}
    if op == "product":
        k, m, n, cols = case["k"], case["m"], case["n"], case["cols"]
        s["a"], s["a_scale"] = _encode(_normal((k, m, cols), gen))
        s["b"], s["b_scale"] = _encode(_normal((k, n, cols), gen, (k * cols) ** -0.5))
        s["out"] = torch.empty((m, n), dtype=t, device="cuda")
        return s
    rows, cols = case["rows"], case["cols"]
    blocks = -(-cols // BLOCK)
    if op == "quantize":
        # gradients and activations: normal, with a few columns far larger than the rest
        x = _normal((rows, cols), gen)
        x *= torch.where(torch.rand((cols,), generator=gen, device="cuda") < 0.01, 20.0, 1.0)
        s["x"] = x.to(t)
    elif op == "fold":
        s["x"], s["x_scale"] = _encode(_normal((case["k"], rows, cols), gen, 1e-3))
        if case["addend"]:
            s["addend"] = _normal((rows, cols), gen, 1e-3).to(t)
        s["out"] = torch.empty((rows, cols), dtype=t, device="cuda")
    else:
        gates = -(-rows // case["gate"]) if case["gate"] else 0
        s["post"] = (1 + _normal((cols,), gen, 0.1)).to(t) if case["post"] else None
        s["pre"] = (1 + _normal((cols,), gen, 0.1)).to(t) if case["pre"] else None
        s["gate"] = (0.5 + _normal((gates, cols), gen, 0.1)).to(t) if gates else None
        if op == "norm":
            s["x"] = _normal((case["k"], rows, cols), gen, case["k"] ** -0.5).to(t)
            s["residual"] = _normal((rows, cols), gen, 2.0).to(t)
            names = ("sum", "y") + (("z",) if case["pre"] else ())
        else:
            s["sum"] = _normal((rows, cols), gen).to(t)
            s["y"] = _normal((rows, cols), gen, 2.0).to(t)
            s["dy"] = _normal((rows, cols), gen).to(t)
            s["dz"] = _normal((rows, cols), gen).to(t) if case["pre"] else None
            names = ("dsum", "dresidual")
            for name in ("post", "pre", "gate"):
                if s[name] is not None:
                    s["d" + name] = torch.empty_like(s[name])
        for name in names:
            s["out_" + name] = torch.empty((rows, cols), dtype=t, device="cuda")
    if op == "quantize" or case.get("requant"):
        # where the packed message goes, and its values
        s["packed"] = torch.empty((rows, blocks, BLOCK // 2), dtype=torch.uint8, device="cuda")
        s["scales"] = torch.empty((rows, blocks), dtype=torch.uint8, device="cuda")
        s["values"] = torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda")
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------


def run(s):
    if own:
        return _OWN[s["op"]](s)
    return _PLAIN[s["op"]](s)


def _rows_gate(s):
    """The gate of every row, or None."""
    g, each, rows = s["gate"], s["case"]["gate"], s["case"]["rows"]
    if g is None:
        return None
    g = g.float()
    return g if g.shape[0] == 1 else g[torch.arange(rows, device=g.device) // each]


def _inverse_rms(v):
    return torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)


def _plain_quantize(s):
    packed, scale = _encode(s["x"])
    return {"values": _decode(packed, scale, s["case"]["cols"]).to(torch.bfloat16)}


def _plain_fold(s):
    case = s["case"]
    v = _decode(s["x"], s["x_scale"], case["cols"]).sum(0, dtype=torch.float64)
    if case["addend"]:
        v = s["addend"].double() + v
    out = {"out": v.to(TYPES[case["type"]])}
    if case["requant"]:
        packed, scale = _encode(v)
        out["values"] = _decode(packed, scale, case["cols"]).to(torch.bfloat16)
    return out


def _plain_product(s):
    case = s["case"]
    # the ranks' shares of the inner length side by side: one product sums over all of them
    a = _decode(s["a"], s["a_scale"], case["cols"]).permute(1, 0, 2).reshape(case["m"], -1)
    b = _decode(s["b"], s["b_scale"], case["cols"]).permute(1, 0, 2).reshape(case["n"], -1)
    return {"out": (a @ b.t()).to(TYPES[case["type"]])}


def _plain_norm(s):
    t = TYPES[s["case"]["type"]]
    v = s["x"].float().sum(0)
    h = v if s["post"] is None else v * _inverse_rms(v) * s["post"].float()
    g = _rows_gate(s)
    y = ALPHA * s["residual"].float() + (h if g is None else g * h)
    out = {"sum": v.to(t), "y": y.to(t)}
    if s["pre"] is not None:
        out["z"] = (y * _inverse_rms(y) * s["pre"].float()).to(t)
    return out


def _plain_norm_grad(s):
    case, t = s["case"], TYPES[s["case"]["type"]]
    v, y, total, out = s["sum"].float(), s["y"].float(), s["dy"].float(), {}
    if s["pre"] is not None:
        r, dz = _inverse_rms(y), s["dz"].float()
        n = y * r
        d = dz * s["pre"].float()
        total = total + r * (d - n * (d * n).mean(-1, keepdim=True))
        out["dpre"] = (dz * n).sum(0).to(t)
    out["dresidual"] = (ALPHA * total).to(t)
    r = _inverse_rms(v)
    h = v if s["post"] is None else v * r * s["post"].float()
    g = _rows_gate(s)
    d = total if g is None else total * g
    if g is not None:
        gates = s["gate"].shape[0]
        dg = torch.nn.functional.pad(total * h, (0, 0, 0, gates * case["gate"] - case["rows"]))
        out["dgate"] = dg.reshape(gates, case["gate"], -1).sum(1).to(t)
    if s["post"] is not None:
        n = v * r
        out["dpost"] = (d * n).sum(0).to(t)
        d = d * s["post"].float()
        d = r * (d - n * (d * n).mean(-1, keepdim=True))
    out["dsum"] = d.to(t)
    return out


_PLAIN = {"quantize": _plain_quantize, "fold": _plain_fold, "product": _plain_product, "norm": _plain_norm, "norm_grad": _plain_norm_grad}


# ---- the same pass through the library -------------------------------------------------------------------------------

_threads = {}


def _thread():
    """The library's thread on torch's current stream."""
    import hcomm_amd as h
    stream = torch.cuda.current_stream().cuda_stream
    if stream not in _threads:
        code, handle = h.HcommThreadAllocWithStream(stream)
        h.check(code, "HcommThreadAllocWithStream")
        _threads[stream] = handle
    return h, _threads[stream]


def _type(h, name):
    return {"bf16": h.HcommDataType.BFP16, "fp16": h.HcommDataType.FP16, "fp32": h.HcommDataType.FP32}[name]


def _views(h, packed, scale):
    """One view for each rank of packed [k, rows, blocks, 16] and scale [k, rows, blocks]."""
    stride = packed.shape[-2] * packed.shape[-1]
    return h.mx_views([(p.data_ptr(), stride, q.data_ptr(), q.shape[-1]) for p, q in zip(packed, scale)])


def _own_quantize(s):
    h, thread = _thread()
    case, x = s["case"], s["x"]
    if s["plan"] is None:  # the descriptions of the buffers that a program keeps beside them
        s["plan"] = (_views(h, s["packed"][None], s["scales"][None]), _type(h, case["type"]))
    view, t = s["plan"]
    rows, cols = case["rows"], case["cols"]
    h.check(h.HcommGfxMxQuantizeOnThread(thread, view, x.data_ptr(), cols, rows, cols, t))
    h.check(h.HcommGfxMxReduceKOnThread(thread, s["values"].data_ptr(), cols, h.HcommDataType.BFP16, None, view, 1, None, 0, rows, cols))
    return {"values": s["values"]}


def _own_fold(s):
    h, thread = _thread()
    case = s["case"]
    if s["plan"] is None:
        again = _views(h, s["packed"][None], s["scales"][None]) if case["requant"] else None
        s["plan"] = (_views(h, s["x"], s["x_scale"]), again, s["addend"].data_ptr() if case["addend"] else None, _type(h, case["type"]))
    views, again, addend, t = s["plan"]
    rows, cols = case["rows"], case["cols"]
    h.check(h.HcommGfxMxReduceKOnThread(thread, s["out"].data_ptr(), cols, t, again, views, case["k"], addend, cols, rows, cols))
    out = {"out": s["out"]}
    if again is not None:
        h.check(h.HcommGfxMxReduceKOnThread(thread, s["values"].data_ptr(), cols, h.HcommDataType.BFP16, None, again, 1, None, 0, rows, cols))
        out["values"] = s["values"]
    return out


def _own_product(s):
    h, thread = _thread()
    case = s["case"]
    if s["plan"] is None:
        s["plan"] = (_views(h, s["a"], s["a_scale"]), _views(h, s["b"], s["b_scale"]), _type(h, case["type"]))
    a, b, t = s["plan"]
    h.check(h.HcommGfxMxProductKOnThread(thread, s["out"].data_ptr(), case["n"], t, a, b, case["k"], case["m"], case["n"], case["cols"]))
    return {"out": s["out"]}


def _pointer(x):
    return None if x is None else x.data_ptr()


def _own_norm(s):
    h, thread = _thread()
    case = s["case"]
    if s["plan"] is None:
        t, cols = _type(h, case["type"]), case["cols"]
        s["plan"] = h.ReduceNormDesc(
            rows=case["rows"], cols=cols, dataType=t, paramType=t, srcs=[x.data_ptr() for x in s["x"]], srcStride=cols,
            residual=s["residual"].data_ptr(), residualStride=cols, residualScale=ALPHA, eps=EPS,
            postWeight=_pointer(s["post"]), preWeight=_pointer(s["pre"]),
            gate=_pointer(s["gate"]), gateStride=cols, rowsPerGate=case["gate"],
            sum=s["out_sum"].data_ptr(), sumStride=cols, y=s["out_y"].data_ptr(), yStride=cols,
            z=_pointer(s.get("out_z")), zStride=cols)
    h.check(h.HcommGfxReduceNormOnThread(thread, s["plan"]))
    return {n: s["out_" + n] for n in ("sum", "y", "z") if "out_" + n in s}


def _own_norm_grad(s):
    h, thread = _thread()
    case = s["case"]
    if s["plan"] is None:
        t, cols = _type(h, case["type"]), case["cols"]
        s["plan"] = h.ReduceNormGradDesc(
            rows=case["rows"], cols=cols, dataType=t, paramType=t, residualScale=ALPHA, eps=EPS,
            sum=s["sum"].data_ptr(), sumStride=cols, y=s["y"].data_ptr(), yStride=cols,
            dy=s["dy"].data_ptr(), dyStride=cols, dz=_pointer(s["dz"]), dzStride=cols,
            postWeight=_pointer(s["post"]), preWeight=_pointer(s["pre"]),
            gate=_pointer(s["gate"]), gateStride=cols, rowsPerGate=case["gate"],
            dSum=s["out_dsum"].data_ptr(), dSumStride=cols, dResidual=s["out_dresidual"].data_ptr(), dResidualStride=cols,
            dPostWeight=_pointer(s.get("dpost")), dPreWeight=_pointer(s.get("dpre")), dGate=_pointer(s.get("dgate")), dGateStride=cols)
        s["workspace"] = torch.empty(h.reduce_norm_grad_workspace_bytes(s["plan"]), dtype=torch.uint8, device="cuda")
        s["plan"].workspace, s["plan"].workspaceBytes = s["workspace"].data_ptr(), s["workspace"].numel()
    h.check(h.HcommGfxReduceNormGradOnThread(thread, s["plan"]))
    out = {n: s["out_" + n] for n in ("dsum", "dresidual")}
    out.update({n: s[n] for n in ("dpost", "dpre", "dgate") if n in s})
    return out


_OWN = {"quantize": _own_quantize, "fold": _own_fold, "product": _own_product, "norm": _own_norm, "norm_grad": _own_norm_grad}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------

_GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]  # what three bits without their sign stand for


def _two_to(e):
    """2^e in fp64 by its bits: a power or an exponential may be a last place off."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_mx(v):
    """v rounded to the format, as the format's definition has it: the block's exponent is that of its largest magnitude
    less two, elements go to the nearest of _GRID, at the middle to the one with an even code."""
    cols = v.shape[-1]
    blocks = -(-cols // BLOCK)
    w = torch.zeros((*v.shape[:-1], blocks * BLOCK), dtype=torch.float64, device=v.device)
    w[..., :cols] = v
    w = w.reshape(*v.shape[:-1], blocks, BLOCK)
    top = w.abs().amax(-1, keepdim=True)
    unit = _two_to(torch.where(top > 0, torch.frexp(top)[1] - 3, -127).clamp(min=-127))
    grid = torch.tensor(_GRID, dtype=torch.float64, device=v.device)
    middle = (grid[1:] + grid[:-1]) / 2
    a = w.abs() / unit
    below, up_to = torch.bucketize(a, middle, out_int32=True), torch.bucketize(a, middle, out_int32=True, right=True)
    q = grid[torch.where(below % 2 == 0, below, up_to)]
    return (torch.copysign(q, w) * unit).reshape(*v.shape[:-1], -1)[..., :cols]


def _exact_values(packed, scale, cols):
    n = packed.to(torch.int16)
    n = torch.stack((n % 16, n // 16), -1).flatten(-2)
    grid = torch.tensor(_GRID, dtype=torch.float64, device=packed.device)
    v = torch.where(n < 8, 1.0, -1.0).double() * grid[(n % 8).to(torch.int32)]
    v = v * _two_to(scale.to(torch.int64) - 127)[..., None]
    return v.flatten(-2)[..., :cols]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return {"values": _exact_mx(s["x"].double())}
    if op == "fold":
        v = torch.zeros((case["rows"], case["cols"]), dtype=torch.float64, device="cuda")
        for j in range(case["k"]):
            v += _exact_values(s["x"][j], s["x_scale"][j], case["cols"])
        if case["addend"]:
            v += s["addend"].double()
        return {"out": v, "values": _exact_mx(v)} if case["requant"] else {"out": v}
    if op == "product":
        v = torch.zeros((case["m"], case["n"]), dtype=torch.float64, device="cuda")
        for j in range(case["k"]):
            v += _exact_values(s["a"][j], s["a_scale"][j], case["cols"]) @ _exact_values(s["b"][j], s["b_scale"][j], case["cols"]).t().contiguous()
        return {"out": v}
    one = torch.ones((1, 1), dtype=torch.float64, device="cuda")
    w1 = one if s["post"] is None else s["post"].double()
    w2 = one if s["pre"] is None else s["pre"].double()
    gate = one if s["gate"] is None else s["gate"].double().repeat_interleave(case["gate"], 0)[:case["rows"]]
    if op == "norm":
        v = s["x"][0].double()
        for j in range(1, case["k"]):
            v = v + s["x"][j].double()
        h = v if s["post"] is None else v / (v.pow(2).mean(1, keepdim=True) + EPS).sqrt() * w1
        y = ALPHA * s["residual"].double() + gate * h
        out = {"sum": v, "y": y}
        if s["pre"] is not None:
            out["z"] = y / (y.pow(2).mean(1, keepdim=True) + EPS).sqrt() * w2
        return out
    v, y, upstream = s["sum"].double(), s["y"].double(), s["dy"].double()
    out = {}
    if s["pre"] is not None:
        dz, q = s["dz"].double(), y.pow(2).mean(1, keepdim=True) + EPS
        # z_i = y_i w_i q^-1/2, so y_j gathers w_j dz_j q^-1/2 - y_j q^-3/2 mean(w dz y)
        upstream = upstream + w2 * dz / q.sqrt() - y * q.pow(-1.5) * (w2 * dz * y).mean(1, keepdim=True)
        out["dpre"] = (dz * y / q.sqrt()).sum(0)
    out["dresidual"] = ALPHA * upstream
    q = v.pow(2).mean(1, keepdim=True) + EPS
    h = v if s["post"] is None else v * w1 / q.sqrt()
    if s["gate"] is not None:
        each = (upstream * h).split(case["gate"])
        out["dgate"] = torch.stack([e.sum(0) for e in each])
    into = gate * upstream
    if s["post"] is not None:
        out["dpost"] = (into * v / q.sqrt()).sum(0)
        into = w1 * into / q.sqrt() - v * q.pow(-1.5) * (w1 * into * v).mean(1, keepdim=True)
    out["dsum"] = into.expand_as(v)
    return out
