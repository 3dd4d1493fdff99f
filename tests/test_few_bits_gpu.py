"""The affine layer in few bits on the GPU against plain 64-bit implementations: 8-bit checkpoints bit for bit,
the gated unit, the weight gradient from a checkpoint and 4-bit weights within derived bounds, and bit for bit
where the sums are exact."""
import numpy as np
import pytest
import torch

import few_bits as fb
from dwbnq import ops

pytestmark = pytest.mark.gpu
TYPES = ["bf16", "f16", "f32"]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def placed(t, device, how):
    """A device copy of the CPU matrix t: contiguous, as a column slice of a wider buffer, or at an odd element offset."""
    rows, cols = t.shape
    if how == "dense":
        return t.to(device).contiguous()
    pad, off = {"slice16": (32, 16), "odd": (3, 1)}[how]
    buf = torch.full((rows, cols + pad), 77.0, dtype=t.dtype, device=device)
    buf[:, off:off + cols] = t.to(device)
    return buf[:, off:off + cols]


def untouched(view, before):
    """The buffer around a column slice still holds its filling."""
    base = view._base
    off = view.storage_offset()
    assert torch.equal(base[:, :off], before[:, :off]) and torch.equal(base[:, off + view.shape[1]:], before[:, off + view.shape[1]:])


def activations(rows, cols, dtype, seed):
    g = gen(seed)
    x = torch.randn(rows, cols, generator=g)
    x *= torch.where(torch.rand(1, cols, generator=g) > 0.97, 30.0, 1.0) * torch.where(torch.rand(rows, 1, generator=g) > 0.9, 1e-3, 1.0)
    return x.to(dtype)


# ---- checkpoints ------------------------------------------------------------------------------

def hard_values(dtype, seed):
    """Groups where the format has to decide: ties, the clamp, zeros, the ends of the type's range, non-finite values."""
    fi = torch.finfo(dtype)
    rows = []
    for e in (-14, -3, 0, 5, 14):
        rows.append(torch.tensor([127.5, 126.5, 0.5, 1.5, -0.5, -127.5, -2.5, 64.0] * 4, dtype=torch.float64) * 2.0 ** e / 64)
    rows.append(torch.zeros(32, dtype=torch.float64))
    rows.append(torch.full((32,), -0.0, dtype=torch.float64))
    rows.append(torch.linspace(-1, 1, 32, dtype=torch.float64) * fi.max)
    rows.append(torch.linspace(-1, 1, 32, dtype=torch.float64) * fi.tiny)
    rows.append(torch.linspace(-1, 1, 32, dtype=torch.float64) * fi.smallest_normal * fi.eps * 40)
    x = torch.stack(rows).to(dtype)
    bad = torch.randn(3, 32, generator=gen(seed)).to(dtype)
    bad[0, 3], bad[1, 31], bad[2, 0] = float("nan"), float("inf"), float("-inf")
    return torch.cat([x, bad])


def check_ckpt(ck, x):
    codes, exps, values = fb.ckpt8(x)
    np.testing.assert_array_equal(ck.exponents.cpu().numpy(), exps)
    np.testing.assert_array_equal(ck.codes.cpu().numpy(), codes)
    return values


@pytest.mark.parametrize("how", ["dense", "slice16", "odd"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (1, 32), (5, 33), (17, 64), (64, 100), (2, 1000), (129, 2048)])
@pytest.mark.parametrize("dt", TYPES)
def test_checkpoint_and_restore_bit_for_bit(cuda_device, dt, rows, cols, how):
    dtype = fb.TYPES[dt]
    x = activations(rows, cols, dtype, rows * 1000 + cols)
    xd = placed(x, cuda_device, how)
    ck = ops.checkpoint_code8(xd)
    values = check_ckpt(ck, x)
    out = placed(torch.zeros(rows, cols, dtype=dtype), cuda_device, how)
    before = out._base.clone() if how != "dense" else None
    got = ops.restore_code8(ck, out=out)
    assert torch.equal(got.cpu(), values.to(dtype))
    if how != "dense":
        untouched(out, before)
    for other in fb.TYPES.values():  # the value is exact in float32 and bfloat16, rounded once in float16
        assert torch.equal(ops.restore_code8(ck, dtype=other).cpu(), values.to(other))


@pytest.mark.parametrize("dt", TYPES)
def test_checkpoint_of_hard_values(cuda_device, dt):
    x = hard_values(fb.TYPES[dt], 5)
    ck = ops.checkpoint_code8(x.to(cuda_device))
    values = check_ckpt(ck, x)
    got = ops.restore_code8(ck).cpu()
    assert torch.equal(got.isnan(), values.isnan())
    assert torch.equal(got.nan_to_num(nan=0.0), values.to(got.dtype).nan_to_num(nan=0.0))
    assert got[~values.isnan()].isfinite().all()  # a finite tensor never comes back infinite
    # the stated error bound, in steps
    fin = ~values.isnan()
    step = torch.from_numpy(np.ldexp(1.0, ck.exponents.cpu().numpy().astype(int) - 133))
    err = (x.double() - values).abs() / step
    assert (err[fin] < 1).all() and (err[fin & (x.double().abs() / step <= 127.5)] <= 0.5).all()


def test_checkpoint_shapes_and_reuse(cuda_device):
    x = torch.randn(2, 3, 5, 40, device=cuda_device)
    ck = ops.checkpoint_code8(x)
    assert ck.shape == (2, 3, 5, 40) and ck.codes.shape == (30, 64) and ck.exponents.shape == (30, 2)
    y = torch.randn_like(x)
    assert ops.checkpoint_code8(y, out=ck) is ck
    check_ckpt(ck, y.reshape(30, 40).cpu())
    v = torch.randn(7, device=cuda_device)
    check_ckpt(ops.checkpoint_code8(v), v[None].cpu())
    t = torch.randn(6, 4, 50, device=cuda_device)[:, 1]  # rows of another tensor's middle axis
    check_ckpt(ops.checkpoint_code8(t), t.cpu())
    for shape in ((0, 5), (5, 0), (0,)):
        ck = ops.checkpoint_code8(torch.empty(shape, device=cuda_device))
        assert ops.restore_code8(ck).shape == shape


# ---- gated unit ----------------------------------------------------------------------------------

def near(got, want, size, dtype, unit, what, tiny):
    """|got - want| within `unit` fp32 half-steps of `size` and one rounding to the type. `tiny`: what multiplies the sigmoid (or
    normal distribution) and its exponential: where those are below the normal range 2^-126 (e^-g above 3.4e38 is infinite in
    fp32), fp32 keeps none of their digits, so they are off by up to 2^-126 each."""
    got, want = got.double().cpu(), want
    lim = unit * 2.0 ** -24 * size + half_abs(want, dtype) + 2.0 ** -125 * tiny.abs()
    bad = (got - want).abs() > lim
    assert not bad.any(), (what, got[bad][:4], want[bad][:4], lim[bad][:4])


def half_abs(want, dtype):
    # one rounding, of a value that is itself a little off: 2% covers a step of the fp32 value across a binade
    return want.abs() * fb.half_step(dtype) * 1.02 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


# fp32 rounding steps of the evaluation, as half-steps 2^-24 of the terms' size. For 32-bit tensors: expf 2, erfcf 8 (its
# documented 4 ulp), sums, products and the division one each: under 16. The argument of an exponential or of erfc is rounded
# once or twice before, which the function turns into at most 2 g^2 half-steps. For 16-bit tensors the fast exponential may be
# used (2 + 1.2 |g| ulp, and 2 ulp of a fast division): 8 + 3 |g| more.
def units(g, dtype):
    extra = 0.0 if dtype == torch.float32 else 8 + 3 * g.abs()
    return 16 + 4 * g * g + extra


@pytest.mark.parametrize("how", ["dense", "slice16", "odd"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (2, 64), (33, 100), (65, 1032)])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dt", TYPES)
def test_glu_forward_and_backward(cuda_device, dt, act, rows, cols, how):
    dtype = fb.TYPES[dt]
    gate, up = activations(rows, cols, dtype, 1) * 2, activations(rows, cols, dtype, 2)
    dy = torch.randn(rows, cols, generator=gen(3)).to(dtype)
    gd, ud, dyd = (placed(t, cuda_device, how) for t in (gate, up, dy))
    y, cg, cu = ops.glu(gd, ud, act=act, checkpoint=True)
    g64, u64 = gate.double(), up.double()
    a, _, _ = fb.act(act, g64)
    near(y, a * u64, (a * u64).abs(), dtype, units(g64, dtype), "y", (g64.abs() + 1) * u64)
    assert torch.equal(ops.glu(gd, ud, act=act), y)
    gv, uv = check_ckpt(cg, gate), check_ckpt(cu, up)
    dgate = placed(torch.zeros(rows, cols, dtype=dtype), cuda_device, how)
    dup = placed(torch.zeros(rows, cols, dtype=dtype), cuda_device, how)
    before = [t._base.clone() for t in (dgate, dup)] if how != "dense" else []
    ops.glu_backward(cg, cu, dyd, act=act, dgate=dgate, dup=dup)
    a, d, size = fb.act(act, gv)
    dy64 = dy.double()
    near(dgate, dy64 * uv * d, (dy64 * uv).abs() * size, dtype, units(gv, dtype), "dgate", (gv.abs() + 1) * dy64 * uv)
    near(dup, dy64 * a, (dy64 * a).abs(), dtype, units(gv, dtype), "dup", (gv.abs() + 1) * dy64)
    for t, b in zip((dgate, dup), before):
        untouched(t, b)
    # the product's checkpoint: its codes are those of an fp32 product within the same bound, so at most one step off
    dg2, none, prod = ops.glu_backward(cg, cu, dyd, act=act, product=True, need=(True, False))
    assert none is None and torch.equal(dg2, dgate.contiguous())
    h = (a * uv)
    codes, exps, _ = fb.ckpt8(h.float())
    step = np.ldexp(1.0, prod.exponents.cpu().numpy().astype(int) - 133).repeat(32, 1)[:, :cols]
    got = ops.restore_code8(prod, dtype=torch.float32).cpu().double()
    assert ((got - h).abs() <= torch.from_numpy(step) * 1.001).all()
    same = prod.exponents.cpu().numpy() == exps
    assert same.mean() > 0.95 and (prod.codes.cpu().numpy().reshape(rows, -1, 32)[same] == codes.reshape(rows, -1, 32)[same]).mean() > 0.95


@pytest.mark.parametrize("dt", TYPES)
def test_glu_accumulates_and_aliases(cuda_device, dt):
    dtype = fb.TYPES[dt]
    gate, up, dy = (activations(9, 80, dtype, s).to(cuda_device) for s in (1, 2, 3))
    y, cg, cu = ops.glu(gate, up, checkpoint=True)
    dg, du = ops.glu_backward(cg, cu, dy)
    base = activations(9, 80, dtype, 4).to(cuda_device)
    acc_g, acc_u = base.clone(), base.clone()
    ops.glu_backward(cg, cu, dy, dgate=acc_g, dup=acc_u, accum=(True, False))
    assert torch.equal(acc_u, du)
    # base + the fp32 gradient, rounded once: within one rounding of the sum, and one of the gradient we have at hand
    want = base.double() + dg.double()
    lim = (dg.double().abs() + want.abs()) * fb.half_step(dtype) * 1.01 + 1e-7
    assert ((acc_g.double() - want).abs() <= lim).all()
    t = dy.clone()
    assert torch.equal(ops.glu_backward(cg, cu, t, dgate=t)[0], dg) and torch.equal(t, dg)
    g2 = gate.clone()
    assert torch.equal(ops.glu(g2, up, out=g2), y)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_glu_extremes(cuda_device, act):
    g = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 20.0, -20.0, 87.0, -87.0, 100.0, -100.0, 3e38, -3e38, 1e-45, 13.0, -13.0, -1.2785])
    u = torch.ones(16)
    y, cg, cu = ops.glu(g[None].to(cuda_device), u[None].to(cuda_device), act=act, checkpoint=True)
    want, _, _ = fb.act(act, g.double())
    # results below the normal range may be flushed or rounded in the subnormal range
    assert ((y.cpu().double()[0] - want).abs() <= want.abs() * (16 + 4 * torch.clamp(g.double() ** 2, max=400)) * 2 ** -24 + 2e-38).all()
    nan = torch.tensor([[float("nan"), 1.0]], device=cuda_device)
    one = torch.ones_like(nan)
    y, cg, cu = ops.glu(nan, one, act=act, checkpoint=True)
    assert y[0, 0].isnan() and not y[0, 1].isnan()
    dg, du = ops.glu_backward(cg, cu, one, act=act)
    assert dg.isnan().all() and du.isnan().all()  # the group of the NaN stands for NaN


def test_glu_gradient_against_differences(cuda_device):
    """Central differences of the 64-bit unit at the checkpointed values."""
    gate, up, dy = (activations(4, 64, torch.float32, s) for s in (11, 12, 13))
    for act in ("silu", "gelu"):
        _, cg, cu = ops.glu(gate.to(cuda_device), up.to(cuda_device), act=act, checkpoint=True)
        dg, du = ops.glu_backward(cg, cu, dy.to(cuda_device), act=act)
        gv, uv, h = fb.ckpt8(gate)[2], fb.ckpt8(up)[2], 1e-5
        num_g = dy.double() * uv * (fb.act(act, gv + h)[0] - fb.act(act, gv - h)[0]) / (2 * h)
        num_u = dy.double() * fb.act(act, gv)[0]
        # difference quotient: h^2/6 f''' <= 1e-10 f''', rounding 1e-16 |f| / h; both far below the bound
        assert ((dg.cpu().double() - num_g).abs() <= 1e-5 * (1 + num_g.abs())).all()
        assert ((du.cpu().double() - num_u).abs() <= 1e-5 * (1 + num_u.abs())).all()


# ---- weight gradient ---------------------------------------------------------------------------------

DW_SHAPES = [(1, 1, 1), (1, 33, 5), (5, 64, 64), (63, 127, 129), (64, 128, 256), (65, 129, 257), (200, 300, 40), (1000, 96, 520),
             (4097, 160, 130), (130, 1280, 1000)]


def dw_case(rows, c_in, c_out, dtype, seed, exact):
    g = gen(seed)
    if exact:
        # integer values times powers of two: every product and every sum is exact in fp32 (|sum| < 2^24 units)
        big = max(1, min(8, (1 << 24) // (rows * 128)))
        x = torch.randint(-127, 128, (rows, c_in), generator=g).double()
        x[:, ::32] = 127  # every group has step 1
        dy = torch.randint(-big, big + 1, (rows, c_out), generator=g).double()
        return x.to(torch.float32), dy.to(dtype)
    return activations(rows, c_in, torch.float32, seed), (torch.randn(rows, c_out, generator=g) * 0.1).to(dtype)


@pytest.mark.parametrize("how", ["dense", "slice16", "odd"])
@pytest.mark.parametrize("rows,c_in,c_out", DW_SHAPES)
@pytest.mark.parametrize("dt", TYPES)
def test_affine_gradients_exact_sums(cuda_device, dt, rows, c_in, c_out, how):
    dtype = fb.TYPES[dt]
    x, dy = dw_case(rows, c_in, c_out, dtype, rows + c_in, True)
    ck = ops.checkpoint_code8(x.to(cuda_device))
    dyd = placed(dy, cuda_device, how)
    want, wantb = dy.double().T @ x.double(), dy.double().sum(0)
    for out in {dtype, torch.float32}:
        dw, db = ops.affine_weight_backward(ck, dyd, dtype=out)
        assert dw.dtype == out and torch.equal(dw.cpu(), want.to(out)) and torch.equal(db.cpu(), wantb.to(out))
    base = torch.randint(-50, 50, (c_out, c_in), generator=gen(9)).float()
    acc, none = ops.affine_weight_backward(ck, dyd, dw=base.to(cuda_device), need=(True, False), accum=(True, False))
    assert none is None and torch.equal(acc.cpu(), (want + base.double()).float())
    _, db = ops.affine_weight_backward(ck, dyd, db=base[:, 0].to(cuda_device).contiguous(), need=(False, True), accum=(False, True))
    assert torch.equal(db.cpu(), (wantb + base[:, 0].double()).float())
    ops.check_device_flag()


@pytest.mark.parametrize("rows,c_in,c_out", [(3, 40, 24), (777, 200, 136), (5000, 64, 320)])
@pytest.mark.parametrize("dt", TYPES)
def test_affine_gradients_real_values(cuda_device, dt, rows, c_in, c_out):
    dtype = fb.TYPES[dt]
    x, dy = dw_case(rows, c_in, c_out, dtype, 31, False)
    ck = ops.checkpoint_code8(x.to(cuda_device))
    xv = fb.ckpt8(x)[2]
    want, size = dy.double().T @ xv, dy.double().abs().T @ xv.abs()
    dw, db = ops.affine_weight_backward(ck, dy.to(cuda_device), dtype=torch.float32)
    # exact products; a partial sum of n of them is off by at most n steps 2^-23 of its size (a truncating adder included)
    assert ((dw.cpu().double() - want).abs() <= (rows + 8) * 2.0 ** -23 * size).all()
    # and on the whole by far less: the tensor cores' sums are cut into short runs that are added in fp32
    assert (dw.cpu().double() - want).norm() <= 1.5e-6 * want.norm()
    wantb = dy.double().sum(0)
    assert ((db.cpu().double() - wantb).abs() <= (rows + 8) * 2.0 ** -24 * dy.double().abs().sum(0)).all()
    again, _ = ops.affine_weight_backward(ck, dy.to(cuda_device), dtype=torch.float32)
    assert torch.equal(again, dw)  # the order of the sum is fixed
    # 16-bit results are summed in longer runs: the first bound, and one rounding
    narrow, _ = ops.affine_weight_backward(ck, dy.to(cuda_device))
    lim = (rows + 8) * 2.0 ** -23 * size + want.abs() * fb.half_step(dtype) * 1.02
    assert ((narrow.cpu().double() - want).abs() <= lim).all()


@pytest.mark.parametrize("rows,c_in,c_out", [(4300, 1536, 3200), (9001, 64, 96), (20011, 130, 300)])
@pytest.mark.parametrize("dt", ["f16", "f32"])
def test_affine_gradients_of_long_batches(cuda_device, dt, rows, c_in, c_out):
    """dy in several bfloat16 parts over more tokens than a run of the lower parts, in whole tiles and in tiles cut anywhere."""
    dtype = fb.TYPES[dt]
    x, dy = (t.to(cuda_device) for t in dw_case(rows, c_in, c_out, dtype, 37, False))
    dy[:, 0] = 1 + dy[:, 0].abs() / 16  # one sign and every digit in use
    ck = ops.checkpoint_code8(x)
    xv = ops.restore_code8(ck, torch.float32).double()
    want, size = dy.double().T @ xv, dy.double().abs().T @ xv.abs()
    dw, _ = ops.affine_weight_backward(ck, dy, need=(True, False), dtype=torch.float32)
    # the bounds of the shorter batches
    assert ((dw.double() - want).abs() <= (rows + 8) * 2.0 ** -23 * size).all()
    assert (dw.double() - want).norm() <= 1.5e-6 * want.norm()
    base = torch.randn(c_out, c_in, generator=gen(4)).to(cuda_device)
    acc, _ = ops.affine_weight_backward(ck, dy, dw=base.clone(), need=(True, False), accum=(True, False))
    # one addition more per run: a run has at least 512 tokens
    assert ((acc.double() - base.double() - want).abs() <= (rows + 8) * 2.0 ** -23 * size + (rows / 512 + 2) * 2.0 ** -24 * base.abs()).all()
    assert torch.equal(ops.affine_weight_backward(ck, dy, need=(True, False), dtype=torch.float32)[0], dw)
    ops.check_device_flag()


def test_affine_gradients_of_nothing(cuda_device):
    ck = ops.checkpoint_code8(torch.empty(0, 40, device=cuda_device))
    dy = torch.empty(0, 24, device=cuda_device)
    dw, db = ops.affine_weight_backward(ck, dy)
    assert dw.shape == (24, 40) and not dw.any() and not db.any()
    base = torch.ones(24, 40, device=cuda_device)
    dw, _ = ops.affine_weight_backward(ck, dy, dw=base, need=(True, False), accum=(True, False))
    assert torch.equal(dw, torch.ones_like(dw))
    ck = ops.checkpoint_code8(torch.empty(7, 0, device=cuda_device))
    dw, db = ops.affine_weight_backward(ck, torch.ones(7, 3, device=cuda_device))
    assert dw.shape == (3, 0) and torch.equal(db, torch.full((3,), 7.0, device=cuda_device))


@pytest.mark.parametrize("dt", TYPES)
def test_affine_gradients_non_finite(cuda_device, dt):
    """A NaN group of the checkpoint reaches the 32 channels it stands for, an infinity of dy its output channel."""
    dtype = fb.TYPES[dt]
    x, dy = torch.ones(70, 96), torch.ones(70, 40)
    x[69, 40] = float("nan")
    dy[3, 7], dy[4, 9] = float("inf"), float("nan")
    ck = ops.checkpoint_code8(x.to(cuda_device))
    dw, db = ops.affine_weight_backward(ck, dy.to(dtype).to(cuda_device), dtype=torch.float32)
    bad = torch.zeros(40, 96, dtype=torch.bool)
    bad[:, 32:64] = True
    bad[9] = True
    inf = torch.zeros_like(bad)
    inf[7, :32] = inf[7, 64:] = True
    assert torch.equal(dw.cpu().isnan(), bad) and torch.equal(dw.cpu().isinf(), inf)
    assert (dw.cpu()[~bad & ~inf] == 70).all() and db[7].isinf() and db[9].isnan() and db[0] == 70


# ---- 4-bit weights ----------------------------------------------------------------------------------------

W4_SHAPES = [(1, 1, 1), (1, 32, 16), (1, 100, 7), (2, 127, 33), (1, 128, 1000), (3, 1280, 200), (8, 300, 65), (9, 256, 48),
             (16, 520, 130), (17, 96, 20), (40, 1000, 24), (1, 5000, 8)]


def w4_case(rows, k, n, group, dtype, seed, exact, zero_points):
    g = gen(seed)
    groups = (k + group - 1) // group
    codes = torch.randint(0, 16, (n, k), generator=g).to(torch.uint8)
    zeros = torch.randint(0, 16, (n, groups), generator=g).to(torch.uint8) if zero_points else None
    if exact:
        # small integers and power-of-two scales of a small range: exact in fp32 whatever the order
        x = torch.randint(-3, 4, (rows, k), generator=g).to(dtype)
        scales = (2.0 ** torch.randint(-2, 2, (n, groups), generator=g)).to(dtype)
        b = torch.randint(-9, 10, (n,), generator=g).to(dtype)
    else:
        x = torch.randn(rows, k, generator=g).to(dtype)
        scales = (torch.rand(n, groups, generator=g) * 0.02 + 0.01).to(dtype)
        b = torch.randn(n, generator=g).to(dtype)
    return x, codes, scales, zeros, b


@pytest.mark.parametrize("zero_points", [False, True], ids=["mid", "zeros"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,k,n", W4_SHAPES)
@pytest.mark.parametrize("dt", TYPES)
def test_w4_affine(cuda_device, dt, rows, k, n, group, zero_points):
    dtype = fb.TYPES[dt]
    dev = lambda t: None if t is None else t.to(cuda_device)  # noqa: E731
    x, codes, scales, zeros, b = w4_case(rows, k, n, group, dtype, rows + k, True, zero_points)
    w4 = ops.pack_w4(dev(codes), dev(scales), dev(zeros), group=group)
    want = x.double() @ fb.w4_weight(codes, scales, zeros, group).T
    for how in ("dense", "odd"):
        assert torch.equal(ops.affine_w4(placed(x, cuda_device, how), w4).cpu(), want.to(dtype))
    out = placed(torch.zeros(rows, n, dtype=dtype), cuda_device, "odd")
    before = out._base.clone()
    ops.affine_w4(dev(x), w4, dev(b), out=out)
    assert torch.equal(out.cpu(), (want + b.double()).to(dtype))
    untouched(out, before)
    x, codes, scales, zeros, b = w4_case(rows, k, n, group, dtype, rows + k, False, zero_points)
    w4 = ops.pack_w4(dev(codes), dev(scales), dev(zeros), group=group)
    w = fb.w4_weight(codes, scales, zeros, group)
    want, size = x.double() @ w.T + b.double(), x.double().abs() @ w.abs().T + b.double().abs()
    got = ops.affine_w4(dev(x), w4, dev(b)).cpu().double()
    # exact products (one more rounding where the scale is multiplied in first), k of them added in fp32
    lim = (k + 8) * 2.0 ** -23 * size + want.abs() * fb.half_step(dtype) * 1.02
    assert ((got - want).abs() <= lim).all()
    ops.check_device_flag()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(1, 1), (5, 100), (64, 256), (33, 1000)])
@pytest.mark.parametrize("dt", TYPES)
def test_w4_quantize(cuda_device, dt, n, k, group):
    dtype = fb.TYPES[dt]
    w = (torch.randn(n, k, generator=gen(n + k)) * 0.05)
    w[0, :min(k, 40)] = 0
    w = w.to(dtype)
    for how in ("dense", "odd"):
        codes, scales = ops.quantize_w4(placed(w, cuda_device, how), group=group)
        wc, ws = fb.quantize_w4(w, group)
        assert torch.equal(scales.cpu(), ws) and torch.equal(codes.cpu(), wc)
    # through the layer: rows of the identity read the weights back
    w4 = ops.pack_w4(codes, scales, group=group)
    eye = torch.eye(k, dtype=dtype, device=cuda_device)[:16]
    got = ops.affine_w4(eye, w4).cpu().double()
    assert torch.equal(got, fb.w4_weight(wc, ws, None, group).T[:16].to(dtype).double())


def test_w4_non_finite(cuda_device):
    w = torch.randn(3, 256, generator=gen(1))
    w[1, 200] = float("nan")
    codes, scales = ops.quantize_w4(w.to(cuda_device), group=128)
    w4 = ops.pack_w4(codes, scales, group=128)
    x = torch.ones(2, 256)
    x[1, 3] = float("inf")
    y = ops.affine_w4(x.to(cuda_device), w4).cpu()
    assert y[0].isfinite().tolist() == [True, False, True] and not y[1].isfinite().any()
    assert not ops.affine_w4(torch.empty(0, 256, device=cuda_device), w4).numel()
    none = ops.pack_w4(torch.empty(4, 0, dtype=torch.uint8, device=cuda_device), torch.empty(4, 0, device=cuda_device))
    b = torch.arange(4.0, device=cuda_device)
    assert torch.equal(ops.affine_w4(torch.empty(3, 0, device=cuda_device), none, b), b.expand(3, 4))
    assert not ops.affine_w4(torch.empty(3, 0, device=cuda_device), none).any()


# ---- together -------------------------------------------------------------------------------------------------

class Mlp:
    """A gated MLP layer as its user writes it: training with 8-bit checkpoints, serving with 4-bit weights."""

    def __init__(self, d, h, dtype, device, seed):
        g = gen(seed)
        self.w_in = (torch.randn(2 * h, d, generator=g) / d ** 0.5).to(dtype).to(device)
        self.w_out = (torch.randn(d, h, generator=g) / h ** 0.5).to(dtype).to(device)
        self.h = h

    def forward(self, x):
        both = x @ self.w_in.T
        y, cg, cu = ops.glu(both[..., :self.h], both[..., self.h:], checkpoint=True)
        return y @ self.w_out.T, (ops.checkpoint_code8(x), cg, cu)

    def backward(self, kept, dout):
        cx, cg, cu = kept
        dh = dout @ self.w_out
        dboth = torch.empty(*dh.shape[:-1], 2 * self.h, dtype=dh.dtype, device=dh.device)
        _, _, ch = ops.glu_backward(cg, cu, dh, product=True, dgate=dboth[..., :self.h], dup=dboth[..., self.h:])
        dw_out, _ = ops.affine_weight_backward(ch, dout, need=(True, False), dtype=torch.float32)
        dw_in, _ = ops.affine_weight_backward(cx, dboth, need=(True, False), dtype=torch.float32)
        return dw_in, dw_out, dboth @ self.w_in


@pytest.mark.parametrize("dt", TYPES)
def test_mlp_training_step(cuda_device, dt):
    dtype = fb.TYPES[dt]
    m = Mlp(96, 200, dtype, cuda_device, 1)
    x = activations(6 * 37, 96, dtype, 2).reshape(6, 37, 96).to(cuda_device)
    dout = (torch.randn(6, 37, 96, generator=gen(3))).to(dtype).to(cuda_device)
    _, kept = m.forward(x)
    got = m.backward(kept, dout)
    w_in, w_out, xd = (t.double().requires_grad_() for t in (m.w_in, m.w_out, x))
    both = xd @ w_in.T
    out = (torch.nn.functional.silu(both[..., :200]) * both[..., 200:]) @ w_out.T
    want = torch.autograd.grad(out, (w_in, w_out, xd), dout.double())
    # a kept value is off by step / sqrt(12) on average, the step being at most 1/64 of its group's largest value and the group's
    # norm at least that value: sqrt(32) / (64 sqrt(12)) = 2.6% per tensor at worst, three tensors: 4.5%, and the roundings to the type
    for a, b in zip(got, want):
        assert (a.double() - b).norm() <= 0.06 * b.norm()


@pytest.mark.parametrize("dt", TYPES)
def test_mlp_serving_step(cuda_device, dt):
    dtype = fb.TYPES[dt]
    m = Mlp(160, 352, dtype, cuda_device, 1)
    q_in, q_out = ops.quantize_w4(m.w_in, group=32), ops.quantize_w4(m.w_out, group=32)
    w_in, w_out = ops.pack_w4(*q_in, group=32), ops.pack_w4(*q_out, group=32)
    x = torch.randn(2, 1, 160, generator=gen(4)).to(dtype).to(cuda_device)
    both = ops.affine_w4(x, w_in)
    y = ops.affine_w4(ops.glu(both[..., :352], both[..., 352:]), w_out)
    wi, wo = (fb.w4_weight(c.cpu(), s.cpu(), None, 32) for c, s in (q_in, q_out))
    b64 = x.cpu().double() @ wi.T
    want = (torch.nn.functional.silu(b64[..., :352]) * b64[..., 352:]) @ wo.T
    # three roundings to the type along the way, averaged over hundreds of terms
    assert (y.cpu().double() - want).norm() <= (6 * fb.half_step(dtype) + 2e-6) * want.norm()


def test_streams_and_graphs(cuda_device):
    """A training and a serving step captured into two graphs, replayed in turn on new inputs, on a side stream."""
    m = Mlp(64, 128, torch.bfloat16, cuda_device, 1)
    codes, scales = ops.quantize_w4(m.w_in, group=64)
    w4 = ops.pack_w4(codes, scales, group=64)
    x = torch.randn(80, 64, device=cuda_device).bfloat16()
    dout = torch.randn(80, 64, device=cuda_device).bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train = lambda: m.backward(m.forward(x)[1], dout)  # noqa: E731
        serve = lambda: ops.affine_w4(x[:3], w4)  # noqa: E731
        train(), serve()
        side.synchronize()
        g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g1, stream=side):
            r1 = train()
        with torch.cuda.graph(g2, stream=side):
            r2 = serve()
        for seed in range(3):
            x.copy_(torch.randn(80, 64, generator=gen(seed)).bfloat16())
            dout.copy_(torch.randn(80, 64, generator=gen(seed + 9)).bfloat16())
            want1, want2 = train(), serve()
            g2.replay()
            g1.replay()
            g2.replay()
            side.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(r1, want1)) and torch.equal(r2, want2)
    ops.check_device_flag()


def test_threads_share_nothing(cuda_device):
    """Two host threads on streams of their own, the same calls at once."""
    import threading
    m = Mlp(64, 96, torch.float32, cuda_device, 1)
    xs = [torch.randn(300, 64, generator=gen(s)).to(cuda_device) for s in range(2)]
    want = [m.backward(m.forward(x)[1], x) for x in xs]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i] = m.backward(m.forward(xs[i])[1], xs[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


# ---- sizes and places ---------------------------------------------------------------------------------------------

def test_offsets_past_32_bits(cuda_device):
    """Tensors of more than 2^31 elements: what lies at their far end is what the same rows give by themselves."""
    rows, cols = 70001, 32768
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=cuda_device)
    tail = torch.randn(3, cols, generator=gen(1)).bfloat16().to(cuda_device)
    x[-3:] = tail
    ck, part = ops.checkpoint_code8(x), ops.checkpoint_code8(tail)
    assert torch.equal(ck.codes[-3:], part.codes) and torch.equal(ck.exponents[-3:], part.exponents)
    y = ops.restore_code8(ck, out=x)
    assert torch.equal(y[-3:], ops.restore_code8(part)) and not y[:-3].any()
    dy = torch.zeros(rows, 24, dtype=torch.bfloat16, device=cuda_device)
    dy[-3:] = 1.0
    dw, db = ops.affine_weight_backward(ck, dy, dtype=torch.float32)
    want = ops.restore_code8(part, dtype=torch.float32).sum(0)
    assert torch.allclose(dw, want.expand(24, cols), rtol=3 * 2.0 ** -23, atol=0) and (db == 3).all()
    ops.check_device_flag()


def test_w4_offsets_past_32_bits(cuda_device):
    n, k = 65552, 65600
    codes = torch.full((n, k), 8, dtype=torch.uint8, device=cuda_device)
    codes[-5:] = torch.randint(0, 16, (5, k), generator=gen(2)).to(torch.uint8).to(cuda_device)
    scales = torch.full((n, (k + 127) // 128), 0.5, dtype=torch.bfloat16, device=cuda_device)
    w4 = ops.pack_w4(codes, scales, group=128)
    assert w4.packed.numel() > 1 << 31
    x = torch.randint(-1, 2, (2, k), generator=gen(3)).bfloat16().to(cuda_device)
    y = ops.affine_w4(x, w4)
    want = x.double() @ ((codes[-5:].double() - 8) * 0.5).T
    assert torch.equal(y[:, -5:], want.bfloat16()) and not y[:, :-5].any()


@pytest.mark.parametrize("dt", TYPES)
def test_every_row_count(cuda_device, dt):
    """Token counts around the chunk and run sizes of the weight gradient, and row counts of the 4-bit layer around its blocks."""
    dtype = fb.TYPES[dt]
    for rows in (2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1023, 1025):
        x, dy = dw_case(rows, 48, 40, dtype, rows, True)
        dw, db = ops.affine_weight_backward(ops.checkpoint_code8(x.to(cuda_device)), dy.to(cuda_device), dtype=torch.float32)
        assert torch.equal(dw.cpu(), (dy.double().T @ x.double()).float()) and torch.equal(db.cpu(), dy.double().sum(0).float())
    x, codes, scales, zeros, _ = w4_case(35, 384, 40, 64, dtype, 5, True, True)
    w4 = ops.pack_w4(*(t.to(cuda_device) for t in (codes, scales, zeros)), group=64)
    want = (x.double() @ fb.w4_weight(codes, scales, zeros, 64).T).to(dtype)
    for rows in range(1, 36):
        assert torch.equal(ops.affine_w4(x[:rows].to(cuda_device), w4).cpu(), want[:rows])


def test_w4_splits_agree(cuda_device):
    """Layers that are narrow and deep (a cluster of CTAs per output tile), wide (CTAs that walk over many tiles) and in between."""
    for n, k in ((16, 16384), (200, 9000), (4096, 640), (20000, 256), (2400, 2304)):
        for dt, rows in (("bf16", 1), ("f16", 11), ("f32", 2)):
            x, codes, scales, zeros, b = w4_case(rows, k, n, 128, fb.TYPES[dt], n, True, True)
            w4 = ops.pack_w4(*(t.to(cuda_device) for t in (codes, scales, zeros)), group=128)
            want = x.to(cuda_device).double() @ fb.w4_weight(codes, scales, zeros, 128).to(cuda_device).T + b.to(cuda_device).double()
            assert torch.equal(ops.affine_w4(x.to(cuda_device), w4, b.to(cuda_device)), want.to(fb.TYPES[dt])), (n, k, dt)
    ops.check_device_flag()


def test_another_stream_than_the_current_devices_default(cuda_device):
    """The work goes to the stream that is current at the call: a long copy in front of it on that stream is waited for."""
    side = torch.cuda.Stream()
    src = torch.randn(4096, 4096, device=cuda_device).bfloat16()
    x = torch.zeros_like(src)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            x.copy_(src)
            x.zero_()
        x.copy_(src)
        ck = ops.checkpoint_code8(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(ck.codes, ops.checkpoint_code8(src).codes)


class Fenced:
    """Tensors between two bands of a known pattern."""

    BAND = 4096

    def __init__(self, device):
        self.device, self.buffers = device, []

    def __call__(self, shape, dtype, fill=None):
        n = int(np.prod(shape)) * torch.empty(0, dtype=dtype).element_size()
        buf = torch.full((self.BAND + (n + 255) // 256 * 256 + self.BAND,), 0xA5, dtype=torch.uint8, device=self.device)
        self.buffers.append((buf, n))
        t = buf[self.BAND:self.BAND + n].view(dtype).view(shape)
        if fill is not None:
            t.copy_(fill)
        return t

    def check(self):
        for buf, n in self.buffers:
            assert (buf[:self.BAND] == 0xA5).all() and (buf[self.BAND + n:] == 0xA5).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,c_in,c_out", [(1, 1, 1), (65, 100, 36), (130, 257, 300), (1027, 64, 513)])
def test_nothing_beside_the_tensors_is_written(cuda_device, dt, rows, c_in, c_out):
    import ctypes

    from dwbnq import _lib as L
    dtype, fence = fb.TYPES[dt], Fenced(cuda_device)
    groups = (c_in + 31) // 32
    x = fence((rows, c_in), dtype, activations(rows, c_in, dtype, 1))
    up = fence((rows, c_in), dtype, activations(rows, c_in, dtype, 2))
    dy = fence((rows, c_out), dtype, activations(rows, c_out, dtype, 3))
    ck = [ops.Code8Checkpoint(fence((rows, 32 * groups), torch.int8), fence((rows, groups), torch.uint8), (rows, c_in), dtype) for _ in range(3)]
    y, dg, du = (fence((rows, c_in), dtype) for _ in range(3))
    ops.checkpoint_code8(x, out=ck[0])
    ops.restore_code8(ck[0], out=y)
    lib, stream = L.lib(), torch.cuda.current_stream().cuda_stream
    ptr = lambda c: (c.codes.data_ptr(), c.exponents.data_ptr())  # noqa: E731
    code = L.BF16 if dt == "bf16" else L.F16 if dt == "f16" else L.F32
    L.check(lib.dwbnq_glu_fwd(code, L.ACT_GELU, rows, c_in, c_in, x.data_ptr(), c_in, up.data_ptr(), c_in, y.data_ptr(), *ptr(ck[0]), *ptr(ck[1]),
                              0, stream))
    L.check(lib.dwbnq_glu_bwd_ckpt8(code, L.ACT_GELU, rows, c_in, *ptr(ck[0]), *ptr(ck[1]), c_in, y.data_ptr(), c_in, dg.data_ptr(), c_in,
                                    du.data_ptr(), *ptr(ck[2]), 3 if rows % 2 else 0, 0, stream))
    for out in {code, L.F32}:
        d = L.AffineDesc(dtype=code, dw_dtype=out, rows=rows, c_in=c_in, c_out=c_out, ld_dy=c_out)
        t = torch.float32 if out == L.F32 else dtype
        ws = fence((int(lib.dwbnq_affine_bwd_workspace_bytes(ctypes.byref(d))),), torch.uint8)
        ops.affine_weight_backward(ck[0], dy, dw=fence((c_out, c_in), t), db=fence((c_out,), t), ws=ws)
    q, s = ops.quantize_w4(x, group=64)
    w4 = ops.pack_w4(q, s, group=64)
    w4.packed = fence(tuple(w4.packed.shape), torch.uint8, w4.packed)
    for r in (1, 9, 20):
        xs = fence((r, c_in), dtype, activations(r, c_in, dtype, 4))
        ops.affine_w4(xs, w4, out=fence((r, rows), dtype))
    torch.cuda.synchronize()
    fence.check()
    ops.check_device_flag()
