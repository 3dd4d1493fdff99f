"""The five operators of the path and the fused layer, on torch CUDA tensors.

Names, argument order and argument meaning follow nnabla's functional API
(``F.depthwise_convolution``, ``F.batch_normalization``, ``F.fixed_point_quantize``,
``F.pow2_quantize``, ``F.min_max_quantize``), which is what resolves to the ``*Cuda``
classes of nnabla-ext-cuda under ``get_extension_context('cuda')``. torch is used only
for device memory and streams; every computation is a call into libdwbnq through the
C ABI with raw device pointers.
"""
import ctypes

import torch

from . import _lib as L


def _dtype_code(t):
    if t.dtype == torch.float32:
        return L.F32
    if t.dtype == torch.float16:
        return L.F16
    raise TypeError("dwbnq supports float32 and float16 tensors, got %s" % t.dtype)


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _chk_cuda(*ts):
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("dwbnq operators take CUDA tensors (there is no CPU fallback)")
        if not t.is_contiguous():
            raise ValueError("dwbnq operators take contiguous tensors")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError("all tensors must live on one device")
    return dev


def _stream(dev):
    return ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)


def _pair(v, ndim=2):
    if isinstance(v, int):
        return (v,) * ndim
    v = tuple(int(a) for a in v)
    return v


class _ShapeOf:
    """What conv_desc reads of a tensor: its shape and element type."""

    def __init__(self, shape, dtype):
        self.shape, self.dtype = tuple(shape), dtype

    def dim(self):
        return len(self.shape)


def conv_desc(x, w, base_axis=1, pad=None, stride=None, dilation=None, multiplier=1):
    """dwbnq_conv_desc for x [..., C, (H,) W] and w [C*mult, (kh,) kw]."""
    sdims = x.dim() - base_axis - 1
    if sdims not in (1, 2):
        raise ValueError("depthwise_convolution supports 1-D and 2-D convolutions")
    if w.dim() != sdims + 1:
        raise ValueError("weight rank %d does not match %d spatial dims" % (w.dim(), sdims))
    pad = _pair(0 if pad is None else pad, sdims)
    stride = _pair(1 if stride is None else stride, sdims)
    dilation = _pair(1 if dilation is None else dilation, sdims)
    n = 1
    for s in x.shape[:base_axis]:
        n *= int(s)
    c = int(x.shape[base_axis])
    if int(w.shape[0]) != c * multiplier:
        raise ValueError("weight has %d output maps, expected C*multiplier = %d" % (w.shape[0], c * multiplier))
    if sdims == 2:
        h, wd = int(x.shape[-2]), int(x.shape[-1])
        kh, kw = int(w.shape[1]), int(w.shape[2])
        (ph, pw), (sh, sw), (dh, dw) = pad, stride, dilation
    else:
        h, wd = 1, int(x.shape[-1])
        kh, kw = 1, int(w.shape[1])
        ph, sh, dh = 0, 1, 1
        pw, sw, dw = pad[0], stride[0], dilation[0]
    d = L.ConvDesc(dtype=_dtype_code(x), c=c, n=n, h=h, w=wd, kh=kh, kw=kw, stride_h=sh, stride_w=sw,
                   pad_h=ph, pad_w=pw, dil_h=dh, dil_w=dw, multiplier=multiplier)
    ho, wo = ctypes.c_int32(), ctypes.c_int32()
    L.check(L.lib().dwbnq_conv_out_shape(ctypes.byref(d), ctypes.byref(ho), ctypes.byref(wo)))
    oshape = tuple(x.shape[:base_axis]) + (c * multiplier,) + ((ho.value, wo.value) if sdims == 2 else (wo.value,))
    return d, oshape


def depthwise_convolution(x, w, b=None, base_axis=1, pad=None, stride=None, dilation=None,
                          multiplier=1, out=None):
    dev = _chk_cuda(x, w, b, out)
    d, oshape = conv_desc(x, w, base_axis, pad, stride, dilation, multiplier)
    y = out if out is not None else torch.empty(oshape, dtype=x.dtype, device=dev)
    L.check(L.lib().dwbnq_dwconv_fwd(ctypes.byref(d), _ptr(x), _ptr(w), _ptr(b), _ptr(y), dev.index,
                                     _stream(dev)))
    return y


def _bn_view(x, axes):
    if len(axes) != 1:
        raise ValueError("batch_normalization: exactly one channel axis is supported")
    ax = axes[0] % x.dim()
    size0 = 1
    for s in x.shape[:ax]:
        size0 *= int(s)
    size2 = 1
    for s in x.shape[ax + 1:]:
        size2 *= int(s)
    return size0, int(x.shape[ax]), size2


def batch_normalization(x, beta, gamma, mean, variance, axes=(1,), decay_rate=0.9, eps=1e-5,
                        batch_stat=False, out=None):
    """Inference mode only (batch_stat=False): the training path is outside this library."""
    if batch_stat:
        raise NotImplementedError("dwbnq implements BatchNormalization with batch_stat=False only")
    dev = _chk_cuda(x, beta, gamma, mean, variance, out)
    size0, size1, size2 = _bn_view(x, list(axes))
    y = out if out is not None else torch.empty_like(x)
    L.check(L.lib().dwbnq_bn_infer_fwd(_dtype_code(x), size0, size1, size2, float(eps), _ptr(x), _ptr(beta),
                                       _ptr(gamma), _ptr(mean), _ptr(variance), _ptr(y), dev.index,
                                       _stream(dev)))
    return y


def fixed_point_quantize(x, sign=True, n=8, delta=2.0 ** -4, ste_fine_grained=True, out=None):
    dev = _chk_cuda(x, out)
    y = out if out is not None else torch.empty_like(x)
    L.check(L.lib().dwbnq_fpq_fwd(_dtype_code(x), x.numel(), int(sign), int(n), float(delta), _ptr(x),
                                  _ptr(y), dev.index, _stream(dev)))
    return y


def pow2_quantize(x, sign=True, with_zero=True, n=8, m=1, ste_fine_grained=True, out=None):
    dev = _chk_cuda(x, out)
    y = out if out is not None else torch.empty_like(x)
    L.check(L.lib().dwbnq_pow2q_fwd(_dtype_code(x), x.numel(), int(sign), int(with_zero), int(n), int(m),
                                    _ptr(x), _ptr(y), dev.index, _stream(dev)))
    return y


def workspace(channels, device):
    """Scratch for the MinMaxQuantize entry points (torch's allocator returns 512-byte aligned blocks)."""
    nbytes = int(L.lib().dwbnq_workspace_bytes(int(channels)))
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _mm_args(x, qr_min, qr_max, ql_min, ql_max, channels):
    for t in (qr_min, qr_max, ql_min, ql_max):
        if t.numel() != channels or t.dtype != x.dtype:
            raise ValueError("MinMaxQuantize ranges must hold one %s value per channel (%d)" % (x.dtype, channels))
    return L.MinMaxPtrs(qr_min.data_ptr(), qr_max.data_ptr(), ql_min.data_ptr(), ql_max.data_ptr())


def min_max_quantize(x, qr_min, qr_max, ql_min, ql_max, decay=0.999, x_min_max=False, ema=False,
                     ste_fine_grained=True, eps=0.01, axis=1, comm=None, ws=None, out=None):
    """Per-channel MinMaxQuantize: ranges of shape [1, C, 1, 1] along ``axis``. qr_min and
    qr_max are updated in place when x_min_max is set. ``comm`` (a dwbnq.comm.Communicator)
    all-reduces the per-channel min/max across the ranks that share a sharded batch."""
    dev = _chk_cuda(x, qr_min, qr_max, ql_min, ql_max, out)
    size0, c, size2 = _bn_view(x, [axis])
    mm = _mm_args(x, qr_min, qr_max, ql_min, ql_max, c)
    q = L.QuantDesc(kind=L.Q_MINMAX, decay=float(decay), eps=float(eps), x_min_max=int(x_min_max), ema=int(ema))
    ws = ws if ws is not None else workspace(c, dev)
    y = out if out is not None else torch.empty_like(x)
    L.check(L.lib().dwbnq_minmaxq_fwd(_dtype_code(x), size0, c, size2, ctypes.byref(q), _ptr(x),
                                      ctypes.byref(mm), _ptr(y), _ptr(ws),
                                      None if comm is None else comm.handle, dev.index, _stream(dev)))
    return y


def quant_desc(quant):
    """dict {"kind": "none"|"fpq"|"pow2"|"minmax", ...} -> QuantDesc."""
    kind = quant["kind"] if quant else "none"
    if kind == "none":
        return L.QuantDesc(kind=L.Q_NONE)
    if kind == "fpq":
        return L.QuantDesc(kind=L.Q_FPQ, sign=int(quant["sign"]), n=int(quant["n"]), delta=float(quant["delta"]))
    if kind == "pow2":
        return L.QuantDesc(kind=L.Q_POW2, sign=int(quant["sign"]), with_zero=int(quant["with_zero"]),
                           n=int(quant["n"]), m=int(quant["m"]))
    if kind == "minmax":
        return L.QuantDesc(kind=L.Q_MINMAX, decay=float(quant.get("decay", 0.999)),
                           eps=float(quant.get("eps", 0.01)), x_min_max=int(quant.get("x_min_max", True)),
                           ema=int(quant.get("ema", False)))
    raise ValueError("unknown quantizer kind %r" % (kind,))


def fused_dw_bn_quant(x, w, b, beta, gamma, mean, variance, eps=1e-5, pad=None, stride=None,
                      dilation=None, multiplier=1, quant=None, base_axis=1, comm=None, ws=None, out=None):
    """The layer the graph pass produces: quantizer(BN_inference(depthwise_convolution(x))).

    ``mean is None`` skips BatchNormalization. For kind "minmax" the dict also carries the
    tensors qr_min, qr_max, ql_min, ql_max (qr_* updated in place when x_min_max)."""
    mmt = [quant[k] for k in ("qr_min", "qr_max", "ql_min", "ql_max")] if quant and quant["kind"] == "minmax" else []
    dev = _chk_cuda(x, w, b, beta, gamma, mean, variance, out, *mmt)
    d, oshape = conv_desc(x, w, base_axis, pad, stride, dilation, multiplier)
    q = quant_desc(quant)
    y = out if out is not None else torch.empty(oshape, dtype=x.dtype, device=dev)
    mm = None
    if mmt:
        oc = int(w.shape[0])
        mm = ctypes.byref(_mm_args(x, mmt[0], mmt[1], mmt[2], mmt[3], oc))
        ws = ws if ws is not None else workspace(oc, dev)
    L.check(L.lib().dwbnq_fused_fwd(ctypes.byref(d), float(eps), ctypes.byref(q), _ptr(x), _ptr(w), _ptr(b),
                                    _ptr(beta), _ptr(gamma), _ptr(mean), _ptr(variance), mm, _ptr(y),
                                    _ptr(ws) if mmt else None, None if comm is None else comm.handle,
                                    dev.index, _stream(dev)))
    return y


# ---- training side -------------------------------------------------------------------------------

def fixed_point_quantize_backward(dy, x=None, sign=True, n=8, delta=2.0 ** -4, ste_fine_grained=True, dx=None,
                                  accum=False):
    """STE backward of fixed_point_quantize: returns dx (``dx`` given and ``accum``: added onto)."""
    dev = _chk_cuda(dy, x, dx)
    out = dx if dx is not None else torch.empty_like(dy)
    L.check(L.lib().dwbnq_fpq_bwd(_dtype_code(dy), dy.numel(), int(sign), int(n), float(delta), int(ste_fine_grained),
                                  int(accum), _ptr(x), _ptr(dy), _ptr(out), dev.index, _stream(dev)))
    return out


def pow2_quantize_backward(dy, x=None, sign=True, with_zero=True, n=8, m=1, ste_fine_grained=True, dx=None,
                           accum=False):
    """STE backward of pow2_quantize."""
    dev = _chk_cuda(dy, x, dx)
    out = dx if dx is not None else torch.empty_like(dy)
    L.check(L.lib().dwbnq_pow2q_bwd(_dtype_code(dy), dy.numel(), int(sign), int(with_zero), int(n), int(m),
                                    int(ste_fine_grained), int(accum), _ptr(x), _ptr(dy), _ptr(out), dev.index,
                                    _stream(dev)))
    return out


def depthwise_convolution_backward(x, w, dy, base_axis=1, pad=None, stride=None, dilation=None, multiplier=1,
                                   dx=None, dw=None, db=None, need=(True, True, True), accum=(False, False, False)):
    """Gradients of depthwise_convolution: returns (dx, dw, db), None where ``need`` is False
    (propagate_down); ``accum[i]`` adds onto the given tensor instead of overwriting it."""
    dev = _chk_cuda(x, w, dy, dx, dw, db)
    d, oshape = conv_desc(x, w, base_axis, pad, stride, dilation, multiplier)
    if tuple(dy.shape) != tuple(oshape):
        raise ValueError("dy has shape %s, the convolution's output is %s" % (tuple(dy.shape), tuple(oshape)))
    dx = (dx if dx is not None else torch.empty_like(x)) if need[0] else None
    dw = (dw if dw is not None else torch.empty_like(w)) if need[1] else None
    db = (db if db is not None else torch.empty(w.shape[0], dtype=w.dtype, device=dev)) if need[2] else None
    mask = (1 if accum[0] else 0) | (2 if accum[1] else 0) | (4 if accum[2] else 0)
    L.check(L.lib().dwbnq_dwconv_bwd(ctypes.byref(d), _ptr(x), _ptr(w), _ptr(dy), _ptr(dx), _ptr(dw), _ptr(db), mask,
                                     dev.index, _stream(dev)))
    return dx, dw, db


# ---- 8-bit storage of quantized activations -------------------------------------------------

def quantize_linear_code8(x, scale, zero_point=0, round_mode="HALF_AWAY_FROM_ZERO", signed=False,
                          min_range=None, max_range=None, out=None):
    """QuantizeLinear (scalar scale / zero point) with the result stored as int8 / uint8 codes:
    saturate(round(x / scale + zero_point)). The argument names are nnabla's
    ``F.quantize_linear``; ``signed`` picks the narrow type, the range defaults to all of it."""
    dev = _chk_cuda(x, out)
    lo = (-128 if signed else 0) if min_range is None else int(min_range)
    hi = (127 if signed else 255) if max_range is None else int(max_range)
    mode = {"HALF_AWAY_FROM_ZERO": L.ROUND_HALF_AWAY_FROM_ZERO, "HALF_TO_EVEN": L.ROUND_HALF_TO_EVEN}[round_mode]
    y = out if out is not None else torch.empty(x.shape, dtype=torch.int8 if lo < 0 else torch.uint8, device=dev)
    L.check(L.lib().dwbnq_quantize_linear_code8_fwd(_dtype_code(x), x.numel(), float(scale), int(zero_point), mode,
                                                    lo, hi, _ptr(x), _ptr(y), dev.index, _stream(dev)))
    return y


def dequantize_linear_code8(codes, scale, zero_point=0, dtype=torch.float32, out=None):
    """DequantizeLinear from int8 / uint8 codes: (code - zero_point) * scale."""
    dev = _chk_cuda(codes, out)
    if codes.dtype not in (torch.int8, torch.uint8):
        raise TypeError("codes must be int8 or uint8")
    y = out if out is not None else torch.empty(codes.shape, dtype=dtype, device=dev)
    L.check(L.lib().dwbnq_dequantize_linear_code8_fwd(_dtype_code(y), codes.numel(), float(scale), int(zero_point),
                                                      int(codes.dtype == torch.int8), _ptr(codes), _ptr(y), dev.index,
                                                      _stream(dev)))
    return y


def fused_dw_bn_quant_code8(x_codes, in_delta, w, b, beta, gamma, mean, variance, eps=1e-5, pad=None, stride=None,
                            dilation=None, multiplier=1, quant=None, base_axis=1, out=None):
    """The fused layer on 8-bit codes: x_codes (int8 / uint8) stands for x = code * in_delta,
    the result is the code of FixedPointQuantize(BN(conv(x))), int8 when the quantizer is
    signed, else uint8. ``quant`` is a FixedPointQuantize dict with n <= 8 and a power-of-two
    delta; w, b and the BN vectors are float32."""
    if x_codes.dtype not in (torch.int8, torch.uint8):
        raise TypeError("x_codes must be int8 or uint8")
    if not quant or quant["kind"] != "fpq":
        raise ValueError("8-bit storage needs a FixedPointQuantize quantizer")
    dev = _chk_cuda(x_codes, w, b, beta, gamma, mean, variance, out)
    # geometry from the code tensor's shape, parameter dtype from w
    d, oshape = conv_desc(_ShapeOf(x_codes.shape, w.dtype), w, base_axis, pad, stride, dilation, multiplier)
    q = quant_desc(quant)
    io = L.Code8Desc(in_signed=int(x_codes.dtype == torch.int8), in_delta=float(in_delta))
    ydt = torch.int8 if quant["sign"] else torch.uint8
    y = out if out is not None else torch.empty(oshape, dtype=ydt, device=dev)
    if y.dtype != ydt:
        raise TypeError("out must be %s for this quantizer" % ydt)
    L.check(L.lib().dwbnq_fused_fwd_code8(ctypes.byref(d), float(eps), ctypes.byref(q), ctypes.byref(io), _ptr(x_codes),
                                          _ptr(w), _ptr(b), _ptr(beta), _ptr(gamma), _ptr(mean), _ptr(variance),
                                          _ptr(y), dev.index, _stream(dev)))
    return y


# ---- the affine layer of a transformer in few bits ----------------------------------------------
# 8-bit activation checkpoints with the backward passes that read them, and 4-bit weights. These
# take float32, float16 and bfloat16 tensors [..., channels] whose last axis is contiguous; the leading
# axes are rows and may have any one stride (the halves of a wider tensor, a padded buffer).

_FEW_BITS_TYPES = {torch.float32: L.F32, torch.float16: L.F16, torch.bfloat16: L.BF16}
_GLU_ACTS = {"silu": L.ACT_SILU, "gelu": L.ACT_GELU, "relu": L.ACT_RELU}
CODE8_GROUP = 32


def _few_bits_code(dtype):
    if dtype not in _FEW_BITS_TYPES:
        raise TypeError("the few-bit affine operators take float32, float16 and bfloat16 tensors, got %s" % dtype)
    return _FEW_BITS_TYPES[dtype]


def _one_device(*ts):
    dev = None
    for t in ts:
        if t is None:
            continue
        d = t.device
        if d != dev:
            if not t.is_cuda:
                raise ValueError("dwbnq operators take CUDA tensors (there is no CPU fallback)")
            if dev is not None:
                raise ValueError("all tensors must live on one device")
            dev = d
    return dev


def _launch(name, dev, *args):
    """Calls an entry point of the library on dev's current stream, with dev current for the call only. These operators are called
    thousands of times a second by a serving loop: the common case makes no context object and wraps no pointer."""
    fn = getattr(L.lib(), name)
    index = dev.index
    if torch.cuda.current_device() == index:
        status = fn(*args, index, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, index, torch._C._cuda_getCurrentRawStream(index))
    if status:
        L.check(status)


def _addr(t):
    return None if t is None else t.data_ptr()


def _rows_view(t, name):
    """(rows, cols, row stride) of [..., cols] seen as a matrix."""
    dim = t.dim()
    if dim == 2 or (dim > 0 and t.is_contiguous()):
        cols = t.shape[-1]
        if dim == 2:
            rows, (ld, unit) = t.shape[0], t.stride()
            if cols > 0 and unit == 1:
                if rows == 1:
                    return 1, cols, cols
                if rows > 1 and ld >= cols:
                    return rows, cols, ld
        elif cols > 0:
            return t.numel() // cols, cols, cols
    if dim < 1:
        raise ValueError("%s must have at least one axis" % name)
    cols = int(t.shape[-1])
    rows = 1
    for s in t.shape[:-1]:
        rows *= int(s)
    if cols > 1 and rows > 0 and t.stride(-1) != 1:
        raise ValueError("%s: the last axis must be contiguous" % name)
    ld = None  # stride of the innermost leading axis that is longer than 1; the outer ones must continue it
    span = 1
    for s, st in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if s == 1:
            continue
        if ld is None:
            ld = int(st)
        elif rows > 0 and st != ld * span:
            raise ValueError("%s: the leading axes must be one run of rows with one stride" % name)
        span *= int(s)
    if ld is None or rows == 0:
        ld = cols
    if rows > 1 and ld < cols:
        raise ValueError("%s: rows overlap (stride %d below %d columns)" % (name, ld, cols))
    return rows, cols, max(ld, cols)


def _like(t, name, shape, dtype, device, like=None):
    """A given output (or a second input) checked against what it has to be; a new one when it is None (``like``: a tensor of its
    type and device, from which it is made faster)."""
    if t is None:
        return like.new_empty(shape) if like is not None else torch.empty(shape, dtype=dtype, device=device)
    if t.shape != shape or t.dtype != dtype:
        raise ValueError("%s must be %s of shape %s, got %s of shape %s" % (name, dtype, tuple(shape), t.dtype, tuple(t.shape)))
    return t


class Code8Checkpoint:
    """A tensor kept in 8 bits: int8 ``codes`` [rows, 32 * groups], uint8 ``exponents`` [rows, groups], the tensor's
    ``shape`` and ``dtype``. Value = code * 2^(exponent - 133), NaN where the exponent is 255."""

    def __init__(self, codes, exponents, shape, dtype):
        shape = tuple(int(s) for s in shape)
        if not shape:
            raise ValueError("a checkpoint has at least one axis")
        rows = 1
        for s in shape[:-1]:
            rows *= s
        groups = (shape[-1] + CODE8_GROUP - 1) // CODE8_GROUP
        if codes.dtype != torch.int8 or tuple(codes.shape) != (rows, CODE8_GROUP * groups) or not codes.is_contiguous():
            raise ValueError("codes must be contiguous int8 of shape %s" % ((rows, CODE8_GROUP * groups),))
        if exponents.dtype != torch.uint8 or tuple(exponents.shape) != (rows, groups) or not exponents.is_contiguous():
            raise ValueError("exponents must be contiguous uint8 of shape %s" % ((rows, groups),))
        _few_bits_code(dtype)
        self.codes, self.exponents, self.shape, self.dtype, self.rows, self.cols = codes, exponents, shape, dtype, rows, shape[-1]

    @classmethod
    def empty(cls, shape, dtype, device, like=None):
        ck = cls.__new__(cls)
        rows = 1
        for s in shape[:-1]:
            rows *= s
        groups = (shape[-1] + CODE8_GROUP - 1) // CODE8_GROUP
        like = torch.empty(0, device=device) if like is None else like
        ck.codes = like.new_empty((rows, CODE8_GROUP * groups), dtype=torch.int8)
        ck.exponents = like.new_empty((rows, groups), dtype=torch.uint8)
        ck.shape, ck.dtype, ck.rows, ck.cols = tuple(shape), dtype, rows, shape[-1]
        return ck


def _ck_out(ck, name, shape, dtype, like):
    if ck is None:
        return Code8Checkpoint.empty(shape, dtype, like.device, like)
    if ck.shape != tuple(shape) or ck.dtype != dtype:
        raise ValueError("%s must be a checkpoint of a %s tensor of shape %s" % (name, dtype, tuple(shape)))
    return ck


def checkpoint_code8(x, out=None):
    """The 8-bit checkpoint of x [..., channels] (groups of 32 channels share a power-of-two step)."""
    code = _few_bits_code(x.dtype)
    if x.dim() < 1:
        raise ValueError("x must have at least one axis")
    ck = _ck_out(out, "out", x.shape, x.dtype, x)
    dev = _one_device(x, ck.codes, ck.exponents)
    rows, cols, ld = _rows_view(x, "x")
    _launch("dwbnq_ckpt8_store", dev, code, rows, cols, ld, x.data_ptr(), ck.codes.data_ptr(), ck.exponents.data_ptr())
    return ck


def restore_code8(ck, dtype=None, out=None):
    """The values a checkpoint stands for, in the checkpointed tensor's type or ``dtype``."""
    y = _like(out, "out", ck.shape, out.dtype if out is not None and dtype is None else dtype or ck.dtype, ck.codes.device)
    code = _few_bits_code(y.dtype)
    dev = _one_device(ck.codes, ck.exponents, y)
    rows, cols, ld = _rows_view(y, "out")
    _launch("dwbnq_ckpt8_load", dev, code, rows, cols, ck.codes.data_ptr(), ck.exponents.data_ptr(), ld, y.data_ptr())
    return y


def glu(gate, up, act="silu", checkpoint=False, out=None):
    """act(gate) * up, act one of "silu", "gelu" (erf form) and "relu". With ``checkpoint`` the result is (y,
    checkpoint of gate, checkpoint of up), all written in one pass. ``out`` may be ``gate`` or ``up``."""
    code = _few_bits_code(gate.dtype)
    _like(up, "up", gate.shape, gate.dtype, gate.device)
    y = _like(out, "out", gate.shape, gate.dtype, gate.device, gate)
    dev = _one_device(gate, up, y)
    (rows, cols, ldg), (_, _, ldu), (_, _, ldy) = _rows_view(gate, "gate"), _rows_view(up, "up"), _rows_view(y, "out")
    if not checkpoint:
        _launch("dwbnq_glu_fwd", dev, code, _GLU_ACTS[act], rows, cols, ldg, gate.data_ptr(), ldu, up.data_ptr(), ldy,
                y.data_ptr(), None, None, None, None)
        return y
    cg, cu = (Code8Checkpoint.empty(gate.shape, gate.dtype, dev, gate) for _ in range(2))
    _launch("dwbnq_glu_fwd", dev, code, _GLU_ACTS[act], rows, cols, ldg, gate.data_ptr(), ldu, up.data_ptr(), ldy, y.data_ptr(),
            cg.codes.data_ptr(), cg.exponents.data_ptr(), cu.codes.data_ptr(), cu.exponents.data_ptr())
    return y, cg, cu


def glu_backward(ck_gate, ck_up, dy, act="silu", product=False, dgate=None, dup=None, need=(True, True),
                 accum=(False, False)):
    """Gradients of glu from the checkpoints of its inputs: (dgate, dup), None where ``need`` is False; with
    ``product`` also the checkpoint of act(gate) * up, the input of the layer behind. ``accum[i]`` adds onto
    the given tensor. dgate / dup may be views with a row stride, and either may be ``dy`` itself."""
    shape, dtype = ck_gate.shape, ck_gate.dtype
    if ck_up.shape != shape or ck_up.dtype != dtype:
        raise ValueError("the checkpoints of gate and up must have one shape and type")
    if (accum[0] and need[0] and dgate is None) or (accum[1] and need[1] and dup is None):
        raise ValueError("accumulating needs the tensor to accumulate onto")
    code = _few_bits_code(dtype)
    if dy is None and (need[0] or need[1]):
        raise ValueError("dy is needed for dgate and dup")
    device = ck_gate.codes.device
    cols = ck_gate.cols
    ldd = ldg = ldu = cols
    if dy is not None:
        ldd = _rows_view(_like(dy, "dy", shape, dtype, device), "dy")[2]
    dgate = _like(dgate, "dgate", shape, dtype, device, dy) if need[0] else None
    dup = _like(dup, "dup", shape, dtype, device, dy) if need[1] else None
    if dgate is not None:
        ldg = _rows_view(dgate, "dgate")[2]
    if dup is not None:
        ldu = _rows_view(dup, "dup")[2]
    dev = _one_device(ck_gate.codes, ck_gate.exponents, ck_up.codes, ck_up.exponents, dy, dgate, dup)
    ck = Code8Checkpoint.empty(shape, dtype, dev, ck_gate.codes) if product else None
    mask = (1 if accum[0] else 0) | (2 if accum[1] else 0)
    _launch("dwbnq_glu_bwd_ckpt8", dev, code, _GLU_ACTS[act], ck_gate.rows, cols, ck_gate.codes.data_ptr(),
            ck_gate.exponents.data_ptr(), ck_up.codes.data_ptr(), ck_up.exponents.data_ptr(), ldd, _addr(dy), ldg, _addr(dgate),
            ldu, _addr(dup), ck.codes.data_ptr() if product else None, ck.exponents.data_ptr() if product else None, mask)
    return (dgate, dup, ck) if product else (dgate, dup)


def affine_workspace(desc, device):
    """A workspace tensor of the size affine_weight_backward asks for (``desc``: AffineDesc)."""
    return torch.empty(int(L.lib().dwbnq_affine_bwd_workspace_bytes(ctypes.byref(desc))), dtype=torch.uint8, device=device)


def affine_weight_backward(ck_x, dy, dw=None, db=None, need=(True, True), accum=(False, False), dtype=None, ws=None):
    """Weight and bias gradients (dw [c_out, c_in], db [c_out]) of an affine layer y = x w^T + b from the checkpoint
    of x [..., c_in] and dy [..., c_out]; None where ``need`` is False. They have dy's type, or float32 when
    ``dtype`` (or the given dw / db) says so; ``accum[i]`` adds onto the given tensor."""
    code = _few_bits_code(dy.dtype)
    if ck_x.shape[:-1] != tuple(dy.shape[:-1]):
        raise ValueError("dy %s has other rows than the checkpoint %s" % (tuple(dy.shape), ck_x.shape))
    if ws is not None and not ws.is_contiguous():
        raise ValueError("ws must be contiguous")
    if any(a and n and t is None for a, n, t in zip(accum, need, (dw, db))):
        raise ValueError("accumulating needs the tensor to accumulate onto")
    if dtype is None:
        dtype = dw.dtype if dw is not None else db.dtype if db is not None else dy.dtype
    rows, c_out, ld = _rows_view(dy, "dy")
    c_in = ck_x.cols
    like = dy if dtype == dy.dtype else None
    dw = _like(dw, "dw", (c_out, c_in), dtype, dy.device, like) if need[0] else None
    db = _like(db, "db", (c_out,), dtype, dy.device, like) if need[1] else None
    for t, n in ((dw, "dw"), (db, "db")):
        if t is not None and not t.is_contiguous():
            raise ValueError("%s must be contiguous" % n)
    dev = _one_device(dy, ck_x.codes, ck_x.exponents, dw, db, ws)
    # without dw nothing of x is read, and no scratch is needed for the parts of dy
    d = L.AffineDesc(dtype=code, dw_dtype=_few_bits_code(dtype), rows=rows, c_in=c_in if need[0] else 0, c_out=c_out, ld_dy=ld,
                     dy_unaligned=int(dy.data_ptr() % 16 != 0))
    mask = (2 if accum[0] else 0) | (4 if accum[1] else 0)
    if ws is None:
        ws = affine_workspace(d, dev)
    elif ws.numel() * ws.element_size() < int(L.lib().dwbnq_affine_bwd_workspace_bytes(ctypes.byref(d))):
        raise ValueError("ws is smaller than dwbnq_affine_bwd_workspace_bytes asks for")
    _launch("dwbnq_affine_bwd_ckpt8", dev, ctypes.byref(d), ck_x.codes.data_ptr(), ck_x.exponents.data_ptr(), dy.data_ptr(),
            _addr(dw), _addr(db), mask, ws.data_ptr())
    return dw, db


class W4Weight:
    """4-bit weights [c_out, c_in] laid out for affine_w4 (``packed``: the bytes that pack_w4 made), with the type of the layer's
    tensors. ``packed`` may be None until it is set."""

    def __init__(self, packed, c_out, c_in, group, dtype, has_zeros):
        self.c_out, self.c_in, self.group, self.dtype, self.has_zeros = c_out, c_in, group, dtype, has_zeros
        self._desc = L.W4Desc(dtype=_few_bits_code(dtype), group=group, c_in=c_in, c_out=c_out, has_zeros=int(has_zeros))
        self._ref = ctypes.byref(self._desc)
        self.packed = packed

    @property
    def packed(self):
        return self._packed

    @packed.setter
    def packed(self, t):
        if t is not None:
            need = int(L.lib().dwbnq_w4_packed_bytes(self._ref))
            if t.dtype != torch.uint8 or not t.is_contiguous() or t.numel() < need:
                raise ValueError("packed must be contiguous uint8 of %d bytes for this layer" % need)
        self._packed = t

    def desc(self):
        """The layer's dwbnq_w4_desc, by reference."""
        return self._ref


def _w4_groups(c_in, group):
    if group not in (32, 64, 128):
        raise L.DwbnqError(L.ERR_UNSUPPORTED, "group of %s input channels: 32, 64 and 128 are supported" % (group,))
    return (c_in + group - 1) // group


def quantize_w4(w, group=128):
    """Round-to-nearest 4-bit weights of w [c_out, c_in]: (codes uint8 [c_out, c_in] in 0..15, scales [c_out, groups]);
    the weight is (code - 8) * scale. Lay them out with pack_w4."""
    if w.dim() != 2:
        raise ValueError("w must be [c_out, c_in]")
    code = _few_bits_code(w.dtype)
    groups = _w4_groups(int(w.shape[1]), group)
    dev = _one_device(w)
    c_out, c_in, ld = _rows_view(w, "w")
    codes = torch.empty((c_out, c_in), dtype=torch.uint8, device=dev)
    scales = torch.empty((c_out, groups), dtype=w.dtype, device=dev)
    _launch("dwbnq_w4_quantize", dev, code, c_out, c_in, group, ld, _addr(w), _addr(codes), _addr(scales))
    return codes, scales


def pack_w4(codes, scales, zeros=None, group=128):
    """Lays 4-bit weights out for affine_w4, once per layer: codes uint8 [c_out, c_in] (0..15), scales [c_out, groups] of
    the layer's type, zeros uint8 [c_out, groups] or None (8 everywhere); weight = (code - zero) * scale."""
    if codes.dim() != 2 or codes.dtype != torch.uint8:
        raise ValueError("codes must be uint8 [c_out, c_in]")
    c_out, c_in = (int(s) for s in codes.shape)
    groups = _w4_groups(c_in, group)
    dev = _one_device(codes, scales, zeros)
    _like(scales, "scales", (c_out, groups), scales.dtype, dev)
    if zeros is not None:
        _like(zeros, "zeros", (c_out, groups), torch.uint8, dev)
    if not all(t is None or t.is_contiguous() for t in (codes, scales, zeros)):
        raise ValueError("codes, scales and zeros must be contiguous")
    w4 = W4Weight(None, c_out, c_in, int(group), scales.dtype, zeros is not None)
    d = w4.desc()
    w4.packed = torch.empty(int(L.lib().dwbnq_w4_packed_bytes(d)), dtype=torch.uint8, device=dev)
    _launch("dwbnq_w4_pack", dev, d, codes.data_ptr(), scales.data_ptr(), _addr(zeros), w4.packed.data_ptr())
    return w4


def affine_w4(x, w4, b=None, out=None):
    """x w^T + b with 4-bit weights, for a few rows (the weights are read once per 16 rows): x [..., c_in]."""
    if x.dtype != w4.dtype:
        raise TypeError("x is %s, the weights' scales are %s" % (x.dtype, w4.dtype))
    rows, c_in, ldx = _rows_view(x, "x")
    if c_in != w4.c_in:
        raise ValueError("x has %d channels, the weights %d" % (c_in, w4.c_in))
    y = _like(out, "out", x.shape[:-1] + (w4.c_out,), x.dtype, x.device, x)
    if b is not None and not _like(b, "b", (w4.c_out,), x.dtype, x.device).is_contiguous():
        raise ValueError("b must be contiguous")
    packed = w4._packed
    if packed is None:
        raise ValueError("the layer has no packed weights yet")
    dev = _one_device(x, packed, b, y)
    _launch("dwbnq_w4_affine_fwd", dev, w4.desc(), rows, ldx, x.data_ptr(), packed.data_ptr(), _addr(b),
            _rows_view(y, "out")[2], y.data_ptr())
    return y


_ACTS = {None: L.ACT_NONE, "none": L.ACT_NONE, "relu": L.ACT_RELU, "relu6": L.ACT_RELU6}
_MATHS = {"fp32": L.PW_MATH_FP32, "tf32": L.PW_MATH_TF32}


def pwconv_desc(x, w, base_axis=1, math="fp32", act=None):
    """PwConvDesc for x [..., c_in, h, w] and a Convolution weight w [c_out, c_in, 1, 1] (or [c_out, c_in])."""
    if x.dim() != base_axis + 3:
        raise ValueError("pointwise convolution takes [..., c_in, h, w]")
    if w.dim() not in (2, 4) or (w.dim() == 4 and tuple(w.shape[2:]) != (1, 1)) or w.shape[1] != x.shape[base_axis]:
        raise ValueError("weight %s is not a 1x1 kernel over %d input channels" % (tuple(w.shape), x.shape[base_axis]))
    if x.dtype != w.dtype:
        raise TypeError("x and w must have one dtype")
    n = 1
    for s in x.shape[:base_axis]:
        n *= int(s)
    d = L.PwConvDesc(dtype=_dtype_code(x), c_in=int(w.shape[1]), c_out=int(w.shape[0]), h=int(x.shape[base_axis + 1]),
                     w=int(x.shape[base_axis + 2]), n=n, math=_MATHS[math], act=_ACTS[act])
    return d, tuple(x.shape[:base_axis]) + (int(w.shape[0]),) + tuple(x.shape[base_axis + 1:])


def pwconv_workspace(x, w, base_axis=1):
    """A workspace tensor of the size the pointwise entry points ask for."""
    d, _ = pwconv_desc(x, w, base_axis)
    nbytes = int(L.lib().dwbnq_pwconv_workspace_bytes(ctypes.byref(d)))
    return torch.empty(nbytes, dtype=torch.uint8, device=w.device)


def pointwise_convolution(x, w, b=None, base_axis=1, math="fp32", ws=None, out=None):
    """Convolution with a 1x1 kernel (pad 0, stride 1, dilation 1, group 1): y = w * x + b."""
    dev = _chk_cuda(x, w, b, out, ws)
    d, oshape = pwconv_desc(x, w, base_axis, math)
    ws = ws if ws is not None else pwconv_workspace(x, w, base_axis)
    y = out if out is not None else torch.empty(oshape, dtype=x.dtype, device=dev)
    L.check(L.lib().dwbnq_pwconv_fwd(ctypes.byref(d), _ptr(x), _ptr(w), _ptr(b), _ptr(y), _ptr(ws), dev.index, _stream(dev)))
    return y


def fused_pw_bn_quant(x, w, b, beta, gamma, mean, variance, eps=1e-5, quant=None, act=None, base_axis=1, math="fp32",
                      ws=None, out=None):
    """quantizer(act(BN_inference(pointwise_convolution(x)))) in one kernel. ``mean is None`` skips
    BatchNormalization; ``act`` is None, "relu" or "relu6"; ``quant`` a "fpq" / "pow2" dict or None."""
    dev = _chk_cuda(x, w, b, beta, gamma, mean, variance, out, ws)
    d, oshape = pwconv_desc(x, w, base_axis, math, act)
    q = quant_desc(quant)
    ws = ws if ws is not None else pwconv_workspace(x, w, base_axis)
    y = out if out is not None else torch.empty(oshape, dtype=x.dtype, device=dev)
    L.check(L.lib().dwbnq_pwconv_fused_fwd(ctypes.byref(d), float(eps), ctypes.byref(q), _ptr(x), _ptr(w), _ptr(b), _ptr(beta),
                                           _ptr(gamma), _ptr(mean), _ptr(variance), _ptr(y), _ptr(ws), dev.index,
                                           _stream(dev)))
    return y


def pwconv_prepare(x, w, b, beta, gamma, mean, variance, eps=1e-5, act=None, base_axis=1, math="fp32", ws=None):
    """One-time part of fused_pw_bn_quant for parameters that do not change between calls: fills
    (and returns) the workspace; ``x`` only gives the shape."""
    dev = _chk_cuda(w, b, beta, gamma, mean, variance, ws)
    d, _ = pwconv_desc(x, w, base_axis, math, act)
    ws = ws if ws is not None else pwconv_workspace(x, w, base_axis)
    L.check(L.lib().dwbnq_pwconv_prepare(ctypes.byref(d), float(eps), _ptr(w), _ptr(b), _ptr(beta), _ptr(gamma), _ptr(mean),
                                         _ptr(variance), _ptr(ws), dev.index, _stream(dev)))
    return ws


def fused_pw_bn_quant_prepared(x, w_shape_like, ws, has_bn=True, quant=None, act=None, base_axis=1, math="fp32", out=None):
    """The per-call part: one kernel launch on a workspace ``pwconv_prepare`` filled with the same
    ``act`` and ``math``. ``w_shape_like`` is the weight (or anything with its shape and dtype)."""
    dev = _chk_cuda(x, ws, out)
    d, oshape = pwconv_desc(x, w_shape_like, base_axis, math, act)
    q = quant_desc(quant)
    y = out if out is not None else torch.empty(oshape, dtype=x.dtype, device=dev)
    L.check(L.lib().dwbnq_pwconv_fused_fwd_prepared(ctypes.byref(d), ctypes.byref(q), int(bool(has_bn)), _ptr(x), _ptr(y),
                                                    _ptr(ws), dev.index, _stream(dev)))
    return y


def pwconv_plan(x, w, base_axis=1, math="fp32"):
    """1 when the tcgen05 kernel takes this call, 0 for the plain FMA kernel (diagnostic)."""
    d, _ = pwconv_desc(x, w, base_axis, math)
    path = ctypes.c_int()
    L.check(L.lib().dwbnq_pwconv_plan(ctypes.byref(d), _ptr(x), _ptr(w), ctypes.byref(path)))
    return path.value


def pwconv_tiling(desc, x_address=4096, sms=148):
    """Launch shape of the tcgen05 pointwise kernel for a PwConvDesc (host only, diagnostic)."""
    out = (ctypes.c_int * 8)()
    L.check(L.lib().dwbnq_debug_pwconv_tiling(ctypes.byref(desc), ctypes.c_void_p(x_address), int(sms), out))
    keys = ("columns", "channel_tiles", "x_path", "tiles", "ctas", "stages", "accumulators", "shared_columns")
    return dict(zip(keys, list(out)))


def set_forced_pw_path(path):
    L.check(L.lib().dwbnq_set_forced_pw_path(int(path)))


def set_pw_max_ctas(ctas):
    L.check(L.lib().dwbnq_set_pw_max_ctas(int(ctas)))


def fused_plan(x, w, y=None, base_axis=1, pad=None, stride=None, dilation=None, multiplier=1):
    """Kernel family and tile geometry the library would choose (diagnostic)."""
    d, _ = conv_desc(x, w, base_axis, pad, stride, dilation, multiplier)
    path, p, th, thr, smem = (ctypes.c_int() for _ in range(5))
    ctas = ctypes.c_int64()
    L.check(L.lib().dwbnq_fused_plan(ctypes.byref(d), _ptr(x), _ptr(y if y is not None else x), ctypes.byref(path),
                                     ctypes.byref(p), ctypes.byref(th), ctypes.byref(thr), ctypes.byref(ctas),
                                     ctypes.byref(smem)))
    return {"path": path.value, "planes_per_cta": p.value, "rows_per_tile": th.value, "threads": thr.value,
            "ctas": ctas.value, "smem_bytes": smem.value}


def set_forced_path(path):
    L.check(L.lib().dwbnq_set_forced_path(int(path)))


def set_tuning(planes_per_cta=0, row_blocks_per_tile=0, threads=0, rows_per_patch=0):
    L.check(L.lib().dwbnq_set_tuning(int(planes_per_cta), int(row_blocks_per_tile), int(threads),
                                     int(rows_per_patch)))


def check_device_flag(device=-1):
    L.check(L.lib().dwbnq_check_device_flag(int(device)))
