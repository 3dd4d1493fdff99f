"""What the entry points of the affine layer in few bits refuse, and with which status (CPU: the arguments are checked
before a device is touched, and the pointers given here are never followed)."""
import ctypes

import pytest
import torch

from dwbnq import _lib as L
from dwbnq import ops

P = 1 << 20  # an address that is aligned to anything


def call(name, *args):
    lib = L.lib()
    status = getattr(lib, name)(*args)
    return status, lib.dwbnq_last_error_string().decode()


# accepted arguments come as far as the device: without one ERR_CUDA, and with one nothing is launched for empty tensors
REACHED = (L.OK, L.ERR_CUDA)


def test_checkpoint_refusals():
    good = [L.BF16, 4, 40, 40, P, P, P, -1, None]

    def bad(i, v, status=L.ERR_INVALID_ARG):
        a = list(good)
        a[i] = v
        st, msg = call("dwbnq_ckpt8_store", *a)
        assert st == status and msg, (i, v, msg)
        b = [a[0], a[1], a[2], a[5], a[6], a[3], a[4], a[7], a[8]]
        st, msg = call("dwbnq_ckpt8_load", *b)
        assert st == status and msg, (i, v, msg)

    for i, vs in {0: (-1, 3, 99), 1: (-1, 1 << 60), 2: (-1, 41, 1 << 34), 3: (39, -1, (1 << 62)), 4: (None, P + 1), 5: (None, P + 8),
                  6: (None,)}.items():
        for v in vs:
            bad(i, v)
    for empty in ((1, 0), (2, 0)):
        a = list(good)
        a[empty[0]] = empty[1]
        a[4] = a[5] = a[6] = None
        assert call("dwbnq_ckpt8_store", *a)[0] in REACHED


def test_glu_refusals():
    good = dict(dtype=L.F16, act=L.ACT_SILU, rows=3, cols=8, ldg=8, g=P, ldu=8, u=P, ldy=8, y=P, gc=P, ge=P, uc=P, ue=P, dev=-1, s=None)
    for k, v in (("dtype", 5), ("act", L.ACT_NONE), ("act", L.ACT_RELU6), ("act", 9), ("rows", -1), ("ldg", 7), ("ldu", 0), ("ldy", 7),
                 ("g", None), ("u", None), ("y", None), ("y", P + 1), ("gc", None), ("ge", None), ("uc", None), ("ue", None), ("uc", P + 4)):
        st, msg = call("dwbnq_glu_fwd", *dict(good, **{k: v}).values())
        assert st == L.ERR_INVALID_ARG and msg, (k, v)
    back = dict(dtype=L.F16, act=L.ACT_GELU, rows=3, cols=8, gc=P, ge=P, uc=P, ue=P, ldy=8, dy=P, ldg=8, g=P, ldu=8, u=P, pc=P, pe=P,
                accum=0, dev=-1, s=None)
    for k, v in (("dtype", -1), ("act", 0), ("cols", -1), ("gc", None), ("ue", None), ("gc", P + 2), ("ldy", 7), ("dy", None), ("dy", P + 1),
                 ("ldg", 1), ("g", P + 1), ("ldu", 7), ("u", P + 1), ("pc", None), ("pe", None), ("pc", P + 15)):
        st, msg = call("dwbnq_glu_bwd_ckpt8", *dict(back, **{k: v}).values())
        assert st == L.ERR_INVALID_ARG and msg, (k, v)
    assert call("dwbnq_glu_bwd_ckpt8", *dict(back, g=None, u=None, pc=None, pe=None, gc=None).values())[0] == L.OK  # nothing asked for


def test_affine_backward_refusals():
    def desc(**kw):
        return L.AffineDesc(**dict(dict(dtype=L.BF16, dw_dtype=L.F32, rows=64, c_in=40, c_out=24, ld_dy=24), **kw))

    def run(d, codes=P, exps=P, dy=P, dw=P, db=P, ws=P):
        return call("dwbnq_affine_bwd_ckpt8", ctypes.byref(d), codes, exps, dy, dw, db, 0, ws, -1, None)

    lib = L.lib()
    for kw in (dict(dtype=7), dict(dw_dtype=L.F16), dict(dtype=L.F32, dw_dtype=L.BF16), dict(rows=-1), dict(rows=1 << 31), dict(c_in=-1),
               dict(c_out=1 << 25), dict(ld_dy=23), dict(c_in=1 << 24, c_out=1 << 24, ld_dy=1 << 24)):
        assert run(desc(**kw))[0] == L.ERR_INVALID_ARG, kw
        assert lib.dwbnq_affine_bwd_workspace_bytes(ctypes.byref(desc(**kw))) == 0
    assert call("dwbnq_affine_bwd_ckpt8", None, P, P, P, P, P, 0, P, -1, None)[0] == L.ERR_INVALID_ARG
    assert lib.dwbnq_affine_bwd_workspace_bytes(None) == 0
    for kw in (dict(codes=None), dict(codes=P + 8), dict(exps=None), dict(dy=None), dict(dy=P + 1), dict(dw=P + 2), dict(db=P + 1), dict(ws=None),
               dict(ws=P + 16)):
        assert run(desc(), **kw)[0] == L.ERR_INVALID_ARG, kw
    assert run(desc(), dw=None, db=None, ws=None)[0] == L.OK
    assert run(desc(c_out=0, ld_dy=0), dy=None)[0] == L.OK
    assert lib.dwbnq_affine_bwd_workspace_bytes(ctypes.byref(desc())) > 0


def test_affine_backward_unaligned_dy_is_declared():
    """A dy off the 16-byte grid needs a workspace that only a descriptor which says so is given."""
    def desc(**kw):
        return L.AffineDesc(**dict(dict(dtype=L.BF16, dw_dtype=L.F32, rows=640, c_in=40, c_out=24, ld_dy=24), **kw))

    size = lambda **kw: L.lib().dwbnq_affine_bwd_workspace_bytes(ctypes.byref(desc(**kw)))  # noqa: E731
    st, msg = call("dwbnq_affine_bwd_ckpt8", ctypes.byref(desc()), P, P, P + 2, P, P, 0, P, -1, None)
    assert st == L.ERR_INVALID_ARG and "dy_unaligned" in msg
    assert size(dy_unaligned=1) == size() + 640 * 24 * 2 and size(ld_dy=25) == size(dy_unaligned=1)
    assert size(dtype=L.F32, c_in=0) < 10000  # db alone
    # three parts, and 30 chunks of 64 tokens instead of 10, each with a tile of 128 x 256 sums
    assert size(dtype=L.F32) == size() + 3 * 640 * 24 * 2 + (30 - 10) * 128 * 256 * 4


def test_w4_refusals():
    def desc(**kw):
        return L.W4Desc(**dict(dict(dtype=L.BF16, group=64, c_in=128, c_out=24, has_zeros=0), **kw))

    lib = L.lib()
    for kw, st in ((dict(dtype=3), L.ERR_INVALID_ARG), (dict(group=16), L.ERR_UNSUPPORTED), (dict(group=0), L.ERR_UNSUPPORTED),
                   (dict(c_in=-1), L.ERR_INVALID_ARG), (dict(c_out=-4), L.ERR_INVALID_ARG), (dict(c_in=1 << 25), L.ERR_INVALID_ARG),
                   (dict(c_in=1 << 23, c_out=1 << 23), L.ERR_INVALID_ARG)):
        d = desc(**kw)
        assert call("dwbnq_w4_pack", ctypes.byref(d), P, P, None, P, -1, None)[0] == st
        assert call("dwbnq_w4_affine_fwd", ctypes.byref(d), 1, 128, P, P, None, 24, P, -1, None)[0] == st
        assert call("dwbnq_w4_quantize", d.dtype, d.c_out, d.c_in, d.group, 1 << 20, P, P, P, -1, None)[0] == st
        assert lib.dwbnq_w4_packed_bytes(ctypes.byref(d)) == 0
    assert lib.dwbnq_w4_packed_bytes(ctypes.byref(desc())) == 2048 + 256  # two tiles of 1 KiB, 2 x 2 x 16 scales padded to 256 bytes
    d = desc()
    for a in ((None, P, None, P), (P, None, None, P), (P, P, P, P), (P, P, None, None), (P, P, None, P + 16), (P, P + 1, None, P)):
        assert call("dwbnq_w4_pack", ctypes.byref(d), *a, -1, None)[0] == L.ERR_INVALID_ARG
    assert call("dwbnq_w4_pack", ctypes.byref(desc(has_zeros=1)), P, P, None, P, -1, None)[0] == L.ERR_INVALID_ARG
    for rows, ldx, x, pk, b, ldy, y in ((-1, 128, P, P, None, 24, P), (1, 127, P, P, None, 24, P), (1, 128, None, P, None, 24, P),
                                        (1, 128, P, None, None, 24, P), (1, 128, P, P, None, 23, P), (1, 128, P, P, None, 24, None),
                                        (1, 128, P, P + 8, None, 24, P), (1, 128, P + 1, P, None, 24, P), (1, 128, P, P, P + 1, 24, P)):
        assert call("dwbnq_w4_affine_fwd", ctypes.byref(d), rows, ldx, x, pk, b, ldy, y, -1, None)[0] == L.ERR_INVALID_ARG
    assert call("dwbnq_w4_affine_fwd", ctypes.byref(d), 1 << 21, 128, P, P, None, 24, P, -1, None)[0] == L.ERR_UNSUPPORTED
    assert call("dwbnq_w4_quantize", L.F32, 4, 64, 32, 63, P, P, P, -1, None)[0] == L.ERR_INVALID_ARG
    assert call("dwbnq_w4_quantize", L.F32, 4, 64, 32, 64, None, P, P, -1, None)[0] == L.ERR_INVALID_ARG


def test_other_operators_refuse_bfloat16():
    with pytest.raises(TypeError):
        ops._dtype_code(torch.zeros(1, dtype=torch.bfloat16))
    assert call("dwbnq_fpq_fwd", L.BF16, 4, 1, 8, 0.5, P, P, -1, None)[0] == L.ERR_INVALID_ARG


def test_wrapper_refusals():
    x = torch.zeros(4, 40)
    with pytest.raises(ValueError):  # there is no CPU path
        ops.checkpoint_code8(x)
    with pytest.raises(TypeError):
        ops.checkpoint_code8(x.double())
    with pytest.raises(ValueError):
        ops.glu(x, x[:, :39])
    with pytest.raises(ValueError):
        ops.glu(x, x.half())
    with pytest.raises(KeyError):
        ops.glu(x.to("meta").expand(4, 40), x.to("meta"), act="tanh") if torch.cuda.is_available() else ops._GLU_ACTS["tanh"]
    codes, exps = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.uint8)
    ck = ops.Code8Checkpoint(codes, exps, (4, 40), torch.float32)
    for c, e, shape in ((codes[:, :40], exps, (4, 40)), (codes, exps[:, :1], (4, 40)), (codes, exps, (4, 65)), (codes, exps, ()),
                        (codes.float(), exps, (4, 40)), (codes, exps.int(), (4, 40)), (codes.T.contiguous().T, exps, (4, 40))):
        with pytest.raises(ValueError):
            ops.Code8Checkpoint(c, e, shape, torch.float32)
    with pytest.raises(TypeError):
        ops.Code8Checkpoint(codes, exps, (4, 40), torch.float64)
    with pytest.raises(ValueError):
        ops.restore_code8(ck, out=torch.zeros(4, 41))
    with pytest.raises(ValueError):
        ops.affine_weight_backward(ck, torch.zeros(5, 8))
    with pytest.raises(ValueError):
        ops.affine_weight_backward(ck, torch.zeros(4, 8), accum=(True, False))
    with pytest.raises(ValueError):
        ops.affine_weight_backward(ck, torch.zeros(4, 8), dw=torch.zeros(40, 8))
    with pytest.raises(ValueError):
        ops.glu_backward(ck, ck, torch.zeros(4, 40), accum=(False, True))
    with pytest.raises(ValueError):
        ops.glu_backward(ck, ck, None)
    with pytest.raises(ValueError):
        ops.pack_w4(torch.zeros(4, 40), torch.zeros(4, 1))
    with pytest.raises(ValueError):
        ops.quantize_w4(torch.zeros(4))
    w4 = ops.W4Weight(None, 8, 40, 128, torch.float32, False)
    with pytest.raises(TypeError):
        ops.affine_w4(x.half(), w4)
    with pytest.raises(ValueError):
        ops.affine_w4(x[:, :39], w4)


def test_row_views():
    """What counts as rows of one stride."""
    t = torch.zeros(4, 6, 10)
    assert ops._rows_view(t, "t") == (24, 10, 10)
    assert ops._rows_view(t[:, :, 2:9], "t") == (24, 7, 10)
    assert ops._rows_view(t[:, 1], "t") == (4, 10, 60)
    assert ops._rows_view(t[1:2, :, :3], "t") == (6, 3, 10)
    assert ops._rows_view(t[0, 0], "t") == (1, 10, 10)
    assert ops._rows_view(t[:, :, :1], "t") == (24, 1, 10)
    assert ops._rows_view(t[:0], "t")[:2] == (0, 10)
    for bad in (t[:, :5], t[..., ::2], t.transpose(1, 2), t[:, :1].expand(4, 6, 10), t[:1, :1].expand(1, 6, 10)):
        with pytest.raises(ValueError):
            ops._rows_view(bad, "t")
