"""Measured cases of the few-bit affine layer operators: 8-bit activation checkpoints, the gated unit
that writes and reads them, the affine weight gradient from a checkpoint, and the affine layer with
4-bit weights. `run` computes a case with elementary torch operations, or, where `own` is true, with
this package's operators.
"""
import math
import os
import sys

import torch

own = False

_PY = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nnabla-ext-cuda_b200", "python")
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _ops():
    if _PY not in sys.path:
        sys.path.insert(0, _PY)
    from dwbnq import ops
    return ops


def listed():
    return [
        # a checkpoint written in the forward pass and read back in the backward pass: the hidden
        # state of a few tokens (launch latency), of a training batch, and of a ragged fp32 batch
        {"name": "ckpt8-small", "op": "ckpt8", "type": "bf16", "rows": 8, "cols": 2048},
        {"name": "ckpt8-batch", "op": "ckpt8", "type": "bf16", "rows": 16384, "cols": 8192},
        {"name": "ckpt8-ragged", "op": "ckpt8", "type": "f32", "rows": 4099, "cols": 5003},
        # the gated unit of an MLP layer: forward with checkpoints of both inputs and backward from
        # them for a training batch; an odd width in fp16; the bare forward of a few served tokens
        {"name": "glu-train", "op": "glu_train", "type": "bf16", "act": "silu", "rows": 8192, "cols": 11008, "product": 0},
        {"name": "glu-train-ragged", "op": "glu_train", "type": "f16", "act": "gelu", "rows": 1021, "cols": 4999, "product": 1},
        {"name": "glu-serve", "op": "glu", "type": "bf16", "act": "silu", "rows": 4, "cols": 14336},
        # weight gradient of an affine layer whose input was kept in 8 bits: a square projection over a
        # training batch; a long batch through a narrow layer; the 1280 -> 1000 classifier in fp32 with
        # its bias; a handful of tokens, gradients summed over micro-batches
        {"name": "dw-square", "op": "dw", "type": "bf16", "tokens": 8192, "c_in": 4096, "c_out": 4096, "bias": 0, "accum": 0},
        {"name": "dw-long", "op": "dw", "type": "f16", "tokens": 65536, "c_in": 512, "c_out": 320, "bias": 1, "accum": 0},
        {"name": "dw-classifier", "op": "dw", "type": "f32", "tokens": 1021, "c_in": 1280, "c_out": 1000, "bias": 1, "accum": 0},
        # one token through a layer with 4-bit weights: the small classifier (latency), a wide layer,
        # and a served batch of 16 through a square one, with zero points
        {"name": "w4-classifier", "op": "w4", "type": "f32", "rows": 1, "c_in": 1280, "c_out": 1000, "group": 32, "zeros": 0, "bias": 1},
        {"name": "w4-token", "op": "w4", "type": "bf16", "rows": 1, "c_in": 4096, "c_out": 14336, "group": 128, "zeros": 0, "bias": 0},
        {"name": "w4-batch", "op": "w4", "type": "f16", "rows": 16, "c_in": 8192, "c_out": 8192, "group": 64, "zeros": 1, "bias": 0},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ckpt8", "glu_train", "glu", "dw", "dw", "w4", "w4"])
    case = {"op": op, "type": rng.choice(["bf16", "bf16", "f16", "f32"])}
    while True:
        if op == "ckpt8":
            case.update(rows=_log_int(rng, 1, 16384), cols=_log_int(rng, 1, 8192))
            cost = case["rows"] * case["cols"] / (16384 * 8192)
        elif op in ("glu_train", "glu"):
            case.update(act=rng.choice(["silu", "gelu", "relu"]), rows=_log_int(rng, 1, 8192), cols=_log_int(rng, 1, 14336))
            if op == "glu_train":
                case["product"] = rng.randrange(2)
            cost = 2 * case["rows"] * case["cols"] / (8192 * 11008)
        elif op == "dw":
            case.update(tokens=_log_int(rng, 1, 65536), c_in=_log_int(rng, 16, 4096), c_out=_log_int(rng, 16, 4096),
                        bias=rng.randrange(2), accum=rng.randrange(2))
            parts = {"bf16": 1, "f16": 2, "f32": 3}[case["type"]]
            cost = 2 * parts * case["tokens"] * case["c_in"] * case["c_out"] / (8192 * 4096 * 4096)
        else:
            case.update(rows=_log_int(rng, 1, 16), c_in=_log_int(rng, 32, 14336), c_out=_log_int(rng, 1, 14336),
                        group=rng.choice([32, 64, 128]), zeros=rng.randrange(2), bias=rng.randrange(2))
            cost = case["c_in"] * case["c_out"] / (8192 * 8192)
        if cost <= 1:
            return case


# ---- inputs -----------------------------------------------------------------------------------

def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _activations(gen, rows, cols, dtype, width=None):
    """Hidden states: normal values, a few channels far larger than the rest, some rows near zero."""
    n = cols if width is None else width
    x = torch.randn((rows, n), generator=gen, device="cuda")
    channel = torch.randn((1, n), generator=gen, device="cuda")
    x *= torch.where(channel > 2.5, 12.0, 1.0)
    row = torch.rand((rows, 1), generator=gen, device="cuda")
    x *= torch.where(row < 0.01, 1e-3, 1.0)
    return x.to(dtype)


def _exponents(x):
    """Exponent byte of each group of 32 columns: the one of the largest magnitude, at least 7; 255 where a value is not finite."""
    pad = (-x.shape[1]) % 32
    g = torch.nn.functional.pad(x.float(), (0, pad)).view(x.shape[0], -1, 32)
    amax = (g.view(torch.int32) & 0x7fffffff).amax(-1)
    return g, (amax >> 23).clamp_min(7)


def _encode(x):
    """Codes [rows, 32 * groups] (columns past the last are 0) and exponent bytes [rows, groups] of a checkpoint."""
    g, b = _exponents(x)
    inv = ((260 - b) << 23).view(torch.float32)[..., None]
    code = torch.round(g * inv).clamp(-127, 127)
    code = torch.where((b == 255)[..., None], torch.zeros_like(code), code)
    return code.view(x.shape[0], -1).to(torch.int8), b.to(torch.uint8)


def _decode(codes, exps, cols):
    b = exps.int()
    step = torch.where(b == 255, torch.full_like(b, 0x7fc00000), (b - 6) << 23).view(torch.float32)
    v = codes.float().view(codes.shape[0], -1, 32) * step[..., None]
    return v.view(codes.shape[0], -1)[:, :cols]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[case["type"]]
    op = case["op"]
    s = {"case": dict(case), "dtype": t}
    if op == "ckpt8":
        s["x"] = _activations(gen, case["rows"], case["cols"], t)
    elif op in ("glu", "glu_train"):
        # gate and up are the halves of one projection's output, as are their gradients
        both = _activations(gen, case["rows"], case["cols"], t, width=2 * case["cols"])
        s["gate"], s["up"] = both[:, :case["cols"]], both[:, case["cols"]:]
        if op == "glu_train":
            s["dy"] = _normal(gen, (case["rows"], case["cols"]), t, 0.1)
    elif op == "dw":
        x = _activations(gen, case["tokens"], case["c_in"], t)
        s["codes"], s["exps"] = _encode(x)
        s["dy"] = _normal(gen, (case["tokens"], case["c_out"]), t, 0.1)
        if case["accum"]:
            s["dw"] = _normal(gen, (case["c_out"], case["c_in"]), torch.float32)
    else:
        k, n, g = case["c_in"], case["c_out"], case["group"]
        groups = (k + g - 1) // g
        s["x"] = _normal(gen, (case["rows"], k), t)
        s["q"] = torch.randint(0, 16, (n, k), generator=gen, device="cuda", dtype=torch.uint8)
        s["scales"] = ((torch.rand((n, groups), generator=gen, device="cuda") + 0.5) * (0.25 / math.sqrt(k))).to(t)
        s["zeros"] = torch.randint(6, 11, (n, groups), generator=gen, device="cuda", dtype=torch.uint8) if case["zeros"] else None
        s["b"] = _normal(gen, (n,), t) if case["bias"] else None
        if own:
            s["w4"] = _ops().pack_w4(s["q"], s["scales"], s["zeros"], group=g)
    return s


# ---- one pass -----------------------------------------------------------------------------------

def _act(name, g):
    if name == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        # 1 + erf(t) loses its digits in the left tail in 32 bits
        d = g.double()
        p = 0.5 * torch.special.erfc(-d * math.sqrt(0.5))
        return (d * p).float(), (p + d * torch.exp(-0.5 * d * d) / math.sqrt(2 * math.pi)).float()
    return torch.clamp_min(g, 0), (g > 0).float()


def run(state):
    case, t = state["case"], state["dtype"]
    op = case["op"]
    if own:
        ops = _ops()
        if op == "ckpt8":
            return ops.restore_code8(ops.checkpoint_code8(state["x"]))
        if op == "glu":
            return ops.glu(state["gate"], state["up"], act=case["act"])
        if op == "glu_train":
            y, cg, cu = ops.glu(state["gate"], state["up"], act=case["act"], checkpoint=True)
            both = torch.empty((case["rows"], 2 * case["cols"]), dtype=t, device=y.device)
            res = ops.glu_backward(cg, cu, state["dy"], act=case["act"], product=bool(case["product"]),
                                   dgate=both[:, :case["cols"]], dup=both[:, case["cols"]:])
            out = {"y": y, "dgate": res[0], "dup": res[1]}
            if case["product"]:
                out["h"] = ops.restore_code8(res[2])
            return out
        if op == "dw":
            ck = ops.Code8Checkpoint(state["codes"], state["exps"], (case["tokens"], case["c_in"]), t)
            dw = state["dw"].clone() if case["accum"] else None
            dw, db = ops.affine_weight_backward(ck, state["dy"], dw=dw, need=(True, bool(case["bias"])),
                                                accum=(bool(case["accum"]), False))
            # beside a 32-bit dw the call returns db in 32 bits too
            return {"dw": dw, "db": db.to(t)} if case["bias"] else {"dw": dw}
        return ops.affine_w4(state["x"], state["w4"], state["b"])

    if op == "ckpt8":
        return _decode(*_encode(state["x"]), case["cols"]).to(t)
    if op == "glu":
        a, _ = _act(case["act"], state["gate"].float())
        return (a * state["up"].float()).to(t)
    if op == "glu_train":
        a, _ = _act(case["act"], state["gate"].float())
        y = (a * state["up"].float()).to(t)
        g = _decode(*_encode(state["gate"]), case["cols"])
        u = _decode(*_encode(state["up"]), case["cols"])
        a, da = _act(case["act"], g)
        dy = state["dy"].float()
        out = {"y": y, "dgate": (dy * u * da).to(t), "dup": (dy * a).to(t)}
        if case["product"]:
            out["h"] = _decode(*_encode(a * u), case["cols"]).to(t)
        return out
    if op == "dw":
        x = _decode(state["codes"], state["exps"], case["c_in"])
        dy = state["dy"].float()
        dw = (dy.t() @ x)
        if case["accum"]:
            # the sum of this pass and the earlier ones: the gradient buffer of accumulated passes is 32 bits wide
            dw = dw + state["dw"]
            out = {"dw": dw}
        else:
            out = {"dw": dw.to(t)}
        if case["bias"]:
            out["db"] = dy.sum(0).to(t)
        return out
    k, g = case["c_in"], case["group"]
    z = state["zeros"].float() if case["zeros"] else torch.full_like(state["scales"], 8.0, dtype=torch.float32)
    z = z.repeat_interleave(g, 1)[:, :k]
    w = (state["q"].float() - z) * state["scales"].float().repeat_interleave(g, 1)[:, :k]
    y = state["x"].float() @ w.t()
    if case["bias"]:
        y = y + state["b"].float()
    return y.to(t)


# ---- the definitions in 64 bits -------------------------------------------------------------------

def _two_to(e):
    """2^e in 64 bits, from the bits: torch.pow is not exact on the GPU and the codes have ties."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _round_trip64(x):
    """Value of every element after its group of 32 kept 8 bits."""
    rows, cols = x.shape
    groups = (cols + 31) // 32
    v = torch.zeros((rows, groups * 32), dtype=torch.float64, device=x.device)
    v[:, :cols] = x
    v = v.reshape(rows, groups, 32)
    top = v.abs().max(-1, keepdim=True).values
    # top = m * 2^e with 0.5 <= m < 1: the step leaves it between 64 and 128 steps
    _, e = torch.frexp(top)
    step = _two_to(torch.where(top > 0, (e - 7).clamp_min(-126), -126))
    code = torch.clamp(torch.round(v / step), -127.0, 127.0)
    return (code * step).reshape(rows, groups * 32)[:, :cols]


def _act64(name, g):
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * torch.sigmoid(-g)
    if name == "gelu":
        cdf = torch.special.ndtr(g)
        return g * cdf, cdf + g * torch.exp(-g * g / 2) * (1 / math.sqrt(2 * math.pi))
    zero = torch.zeros_like(g)
    return torch.maximum(g, zero), torch.where(g > 0, torch.ones_like(g), zero)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "ckpt8":
        return _round_trip64(s["x"])
    if op == "glu":
        return _act64(case["act"], s["gate"].double())[0] * s["up"].double()
    if op == "glu_train":
        out = {"y": _act64(case["act"], s["gate"].double())[0] * s["up"].double()}
        g, u, dy = _round_trip64(s["gate"]), _round_trip64(s["up"]), s["dy"].double()
        a, da = _act64(case["act"], g)
        out["dgate"], out["dup"] = dy * da * u, dy * a
        if case["product"]:
            # the code of the product depends on the rounding of the product itself: no 64-bit value
            out["h"] = None
        return out
    if op == "dw":
        step = _two_to(s["exps"].int() - 133)
        x = (s["codes"].double() * step.repeat_interleave(32, 1))[:, :case["c_in"]]
        dy = s["dy"].double()
        dw = torch.einsum("to,ti->oi", dy, x)
        if case["accum"]:
            dw += s["dw"].double()
        return {"dw": dw, "db": dy.sum(0)} if case["bias"] else {"dw": dw}
    n, k = s["q"].shape
    grp = torch.arange(k, device="cuda") // case["group"]
    zero = s["zeros"].double() if case["zeros"] else torch.full(s["scales"].shape, 8.0, dtype=torch.float64, device="cuda")
    w = s["scales"].double()[:, grp] * (s["q"].double() - zero[:, grp])
    y = torch.einsum("ri,oi->ro", s["x"].double(), w)
    return y + s["b"].double() if case["bias"] else y


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    op, b = case["op"], _BYTES[case["type"]]
    if op == "ckpt8":
        r, c = case["rows"], case["cols"]
        ck = r * c + r * ((c + 31) // 32)
        # x and the restored tensor once each, the checkpoint written and read
        return {"bytes": 2 * r * c * b + 2 * ck, "flops": 2 * r * c}
    if op == "glu":
        return {"bytes": 3 * case["rows"] * case["cols"] * b, "flops": 4 * case["rows"] * case["cols"]}
    if op == "glu_train":
        r, c = case["rows"], case["cols"]
        ck = r * c + r * ((c + 31) // 32)
        # forward: gate, up, y and two checkpoints; backward: both checkpoints, dy, dgate, dup
        # (and the checkpoint of the product, written, read back and restored)
        extra = 2 * ck + r * c * b if case["product"] else 0
        return {"bytes": 6 * r * c * b + 4 * ck + extra, "flops": 16 * r * c}
    if op == "dw":
        t, i, o = case["tokens"], case["c_in"], case["c_out"]
        out = o * i * (8 if case["accum"] else b) + (o * b if case["bias"] else 0)
        return {"bytes": t * o * b + t * i + t * ((i + 31) // 32) + out, "flops": 2 * t * i * o}
    n, k, r = case["c_out"], case["c_in"], case["rows"]
    groups = (k + case["group"] - 1) // case["group"]
    return {"bytes": (n * k + 1) // 2 + n * groups * (b + (1 if case["zeros"] else 0)) + r * (n + k) * b + (n * b if case["bias"] else 0),
            "flops": 2 * r * n * k}
