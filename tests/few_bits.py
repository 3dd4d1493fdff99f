"""Plain 64-bit implementations of the affine layer in few bits (the oracle of the tests, NumPy / torch on the CPU)."""
import math

import numpy as np
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(dtype):
    """Largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def ckpt8(x):
    """(codes int8 [rows, 32 groups], exponents uint8 [rows, groups], values float64 [rows, cols]) of a CPU tensor [rows, cols]."""
    v = x.to(torch.float64).numpy()
    rows, cols = v.shape
    groups = (cols + 31) // 32
    padded = np.zeros((rows, groups * 32))
    padded[:, :cols] = v
    g = padded.reshape(rows, groups, 32)
    finite = np.isfinite(g).all(-1)
    top = np.where(finite, np.abs(np.where(np.isfinite(g), g, 0)).max(-1), 1.0)
    _, e = np.frexp(top)  # top = m 2^e, 0.5 <= m < 1: biased exponent e - 1 + 127
    b = np.where(top > 0, np.maximum(e + 126, 7), 7)
    step = np.ldexp(1.0, b - 133)
    codes = np.clip(np.rint(np.where(finite[..., None], g, 0) / step[..., None]), -127, 127)
    b = np.where(finite, b, 255)
    values = np.where(finite[..., None], codes * step[..., None], np.nan)
    return (codes.reshape(rows, -1).astype(np.int8), b.astype(np.uint8),
            torch.from_numpy(values.reshape(rows, -1)[:, :cols].copy()))


def act(name, g):
    """(act(g), act'(g), size of the terms act' is added up from) in float64."""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * torch.sigmoid(-g), s + g.abs() * s * torch.sigmoid(-g)
    if name == "gelu":
        p, d = 0.5 * torch.special.erfc(-g * math.sqrt(0.5)), torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
        return g * p, p + g * d, p + g.abs() * d
    one = (g > 0).double()
    return g.clamp_min(0), one, one


def w4_weight(codes, scales, zeros, group):
    k = codes.shape[1]
    idx = torch.arange(k) // group
    z = 8.0 if zeros is None else zeros.double()[:, idx]
    return (codes.double() - z) * scales.double()[:, idx]


def quantize_w4(w, group):
    """codes and scales as dwbnq_w4_quantize defines them (fp32 division), for finite weights."""
    n, k = w.shape
    groups = (k + group - 1) // group
    p = np.zeros((n, groups * group), np.float32)
    p[:, :k] = w.float().numpy()
    g = p.reshape(n, groups, group)
    s = torch.from_numpy(np.abs(g).max(-1) / np.float32(7)).to(w.dtype)
    s32 = s.float().numpy()[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(s32 > 0, np.clip(np.rint(g / s32), -8, 7), 0) + 8
    return torch.from_numpy(q.reshape(n, -1)[:, :k].astype(np.uint8)), s
