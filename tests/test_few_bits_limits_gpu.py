"""The affine layer in few bits at the ends of its range on the GPU, against plain 64-bit implementations: batches so long that
the bias of a sum would show, values that are not finite or as large as the type holds, terms that cancel."""
import pytest
import torch

import few_bits as fb
from dwbnq import ops

pytestmark = pytest.mark.gpu
TYPES = ["bf16", "f16", "f32"]


def gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("accum", [False, True], ids=["new", "accum"])
@pytest.mark.parametrize("rows", [8192, 65536])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_sixteen_bit_weight_gradients_have_no_bias(cuda_device, dt, rows, accum):
    """148 tiles (none is cut along the tokens), everything of one sign: an adder that drops digits shows as a mean error."""
    dtype, c_in, c_out = fb.TYPES[dt], 4736, 1024
    g = torch.Generator(device=cuda_device).manual_seed(rows)
    rand = lambda *s: torch.rand(*s, generator=g, device=cuda_device)  # noqa: E731
    # every channel has a size of its own, so that the results lie everywhere between two neighbours of the type
    x = (0.4 + 0.5 * rand(1, c_in)) * (0.9 + 0.1 * rand(rows, c_in))
    dy = ((0.05 + 0.05 * rand(1, c_out)) * (0.5 + 0.5 * rand(rows, c_out))).to(dtype)
    ck = ops.checkpoint_code8(x)
    del x
    want = torch.zeros(c_out, c_in, dtype=torch.float64, device=cuda_device)
    for part in range(0, rows, 8192):
        some = ops.Code8Checkpoint(ck.codes[part:part + 8192], ck.exponents[part:part + 8192], (min(8192, rows - part), c_in), torch.float32)
        want += dy[part:part + 8192].double().T @ ops.restore_code8(some).double()
    dw, none = None, None
    if accum:
        dw = rand(c_out, c_in).to(dtype)
        want += dw.double()
    dw, none = ops.affine_weight_backward(ck, dy, dw=dw, need=(True, False), accum=(accum, False))
    assert none is None and dw.dtype == dtype
    err = (dw.double() - want) / want
    # Products are exact. Sums are cut into runs of at most 1024 tokens, 64 steps of the adder, each of which may drop less than
    # 2^-23 of the run's sum: 2^-17 in all. The runs, at least 256 tokens each in two parts of dy at most, are added in fp32.
    drift = 2.0 ** -17 + rows / 128 * 2.0 ** -24
    half = fb.half_step(dtype)
    assert err.abs().max() <= half * 1.001 + drift
    # the roundings are spread evenly over +-half a step: their mean over n values is off by half / sqrt(3 n), times six
    assert err.mean().abs() <= drift + 6 * half / (3 * err.numel()) ** 0.5
    ops.check_device_flag()


# ---- 4-bit weights -------------------------------------------------------------------------------


def w4_layer(n, k, group, dtype, zero_points, device, seed):
    g = gen(seed)
    groups = (k + group - 1) // group
    codes = torch.randint(0, 16, (n, k), generator=g).to(torch.uint8)
    zeros = torch.randint(0, 16, (n, groups), generator=g).to(torch.uint8) if zero_points else None
    scales = (torch.rand(n, groups, generator=g) * 0.004 + 0.002).to(dtype)
    b = torch.randn(n, generator=g).to(dtype)
    return codes, scales, zeros, b


def packed(codes, scales, zeros, group, device):
    return ops.pack_w4(codes.to(device), scales.to(device), None if zeros is None else zeros.to(device), group=group)


def w4_bound(x, w, b, k, dtype):
    """(64-bit result, limit): exact products, k of them and one bias added in fp32 (whatever the order, an adder that truncates
    included), one rounding of the result. A weight of 0 takes no part, however large its x."""
    want = x.double() @ w.T + b.double()
    size = x.double().abs() @ w.abs().T + b.double().abs()
    return want, (k + 8) * 2.0 ** -23 * size + want.abs() * fb.half_step(dtype) * 1.02


@pytest.mark.parametrize("zero_points", [False, True], ids=["mid", "zeros"])
@pytest.mark.parametrize("rows,k,n,group", [(3, 256, 48, 128), (11, 1000, 130, 64), (2, 520, 700, 32), (1, 4096, 4800, 128)])
@pytest.mark.parametrize("dt", TYPES)
def test_w4_values_that_are_not_finite_or_huge(cuda_device, dt, rows, k, n, group, zero_points):
    """An infinity gives infinities of the weights' signs and NaN where the weight is 0; the largest number of the type gives numbers."""
    dtype = fb.TYPES[dt]
    top = torch.finfo(dtype).max
    codes, scales, zeros, b = w4_layer(n, k, group, dtype, zero_points, cuda_device, k + n)
    w4 = packed(codes, scales, zeros, group, cuda_device)
    w = fb.w4_weight(codes, scales, zeros, group)
    for case in (("inf", "-inf"), ("inf", "inf", "nan"), (top,), (top, -top, top), (top / 128, 1.0)):
        x = torch.randn(rows, k, generator=gen(len(case))).to(dtype)
        for i, v in enumerate(case):
            x[-1, (37 * i + 5) % k] = float(v)
        got = ops.affine_w4(x.to(cuda_device), w4, b.to(cuda_device)).cpu().double()
        want, lim = w4_bound(x, w, b, k, dtype)
        fin = want.isfinite()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf() & ~fin, want.isinf())
        assert torch.equal(got[want.isinf()], want[want.isinf()])
        assert ((got - want).abs() <= lim)[fin].all()
        assert fin[:-1].all() and (not isinstance(case[0], float) or fin.all())
    ops.check_device_flag()


@pytest.mark.parametrize("outlier", [1e2, 1e4, 6e4])
@pytest.mark.parametrize("rows,k,n,group", [(1, 1024, 160, 128), (16, 640, 64, 32), (2, 512, 4800, 64)])
@pytest.mark.parametrize("dt", TYPES)
def test_w4_outliers_of_unused_channels(cuda_device, dt, rows, k, n, group, outlier):
    """One channel of every group is far larger than the others and has weight 0: it does not show in the result."""
    dtype = fb.TYPES[dt]
    codes, scales, zeros, b = w4_layer(n, k, group, dtype, True, cuda_device, 3)
    idle = torch.arange(0, k, group) + 17 % group
    codes[:, idle] = zeros
    x = torch.randn(rows, k, generator=gen(5)).to(dtype)
    x[:, idle] = outlier
    want, lim = w4_bound(x, fb.w4_weight(codes, scales, zeros, group), b, k, dtype)
    got = ops.affine_w4(x.to(cuda_device), packed(codes, scales, zeros, group, cuda_device), b.to(cuda_device)).cpu().double()
    assert ((got - want).abs() <= lim).all()
    # rows with a large common part, which cancels where a group's weights do (float16: so large that the results stay in range)
    x = (outlier / (64 if dtype == torch.float16 else 1) + torch.randn(rows, k, generator=gen(6))).to(dtype)
    want, lim = w4_bound(x, fb.w4_weight(codes, scales, zeros, group), b, k, dtype)
    got = ops.affine_w4(x.to(cuda_device), packed(codes, scales, zeros, group, cuda_device), b.to(cuda_device)).cpu().double()
    assert ((got - want).abs() <= lim).all()


@pytest.mark.parametrize("rows", [1, 12])
@pytest.mark.parametrize("dt", TYPES)
def test_w4_weights_of_zero_give_the_bias(cuda_device, dt, rows):
    dtype, n, k, group = fb.TYPES[dt], 4800, 1100, 64
    codes, scales, zeros, b = w4_layer(n, k, group, dtype, True, cuda_device, 8)
    codes = zeros.repeat_interleave(group, 1)[:, :k].contiguous()
    x = (100 + torch.randn(rows, k, generator=gen(7))).to(dtype)
    got = ops.affine_w4(x.to(cuda_device), packed(codes, scales, zeros, group, cuda_device), b.to(cuda_device))
    assert torch.equal(got.cpu(), b.expand(rows, n))
    # groups whose scale is not finite stand for NaN
    scales[5, 2], scales[7, 0] = float("nan"), float("inf")
    got = ops.affine_w4(x.to(cuda_device), packed(codes, scales, zeros, group, cuda_device), b.to(cuda_device)).cpu()
    bad = torch.zeros(rows, n, dtype=torch.bool)
    bad[:, 5] = bad[:, 7] = True
    assert torch.equal(got.isnan(), bad) and torch.equal(got[~bad], b.expand(rows, n)[~bad])


# ---- gated unit ----------------------------------------------------------------------------------

MAGNITUDES = [1e-30, 1e-8, 2.0 ** -14, 1e-3, 0.1, 0.5, 0.75, 1.0, 1.2785, 1.5, 2.0, 2.75, 3.0, 4.0, 5.5, 7.0, 9.0, 11.0, 13.0, 13.25, 15.0, 16.0,
              17.5, 20.0, 40.0, 64.0, 87.0, 88.0, 89.0, 100.0, 104.0, 500.0, 6e4, 1e10, 1e19, 1e30, 3e38]


def act_near(got, want, size, g, scale, dtype):
    """One rounding to the type; the evaluation in fp32, 24 half-steps of the terms' size and the rounding of an exponential's argument
    (3 |g|; 4 g^2 where the exponential is of g^2, whose results vanish beyond 15); and 0 for what fp32 holds below 2^-126."""
    unit = 24 + 3 * g.abs() + 4 * torch.clamp(g * g, max=225.0)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    lim = want.abs() * fb.half_step(dtype) * 1.02 + tiny + unit * 2.0 ** -24 * size + 2.0 ** -125 * (g.abs() + 1) * scale
    bad = ~((got.double().cpu() - want).abs() <= lim)
    assert not bad.any(), (g[bad][:4], got.cpu()[bad][:4], want[bad][:4], lim[bad][:4])


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dt", TYPES)
def test_glu_over_the_whole_range(cuda_device, dt, act):
    """Both signs of every size that the type holds, a group of 32 each, forward and backward."""
    dtype = fb.TYPES[dt]
    top = torch.finfo(dtype).max
    m = torch.tensor([v for v in MAGNITUDES if v <= top and v >= torch.finfo(dtype).smallest_normal], dtype=torch.float64)
    steps = torch.tensor([1.0, 0.99, 0.9, 0.75, 0.6, 0.51, 0.3, 0.1] * 2, dtype=torch.float64)
    gate = (m[:, None] * torch.cat([steps, -steps])).to(dtype)
    up = torch.full_like(gate, 0.5)
    up[:, ::3] = -1.0
    dy = torch.full_like(gate, 2.0)
    y, cg, cu = ops.glu(gate.to(cuda_device), up.to(cuda_device), act=act, checkpoint=True)
    g, u = gate.double(), up.double()
    a, _, _ = fb.act(act, g)
    act_near(y, a * u, (a * u).abs(), g, u.abs(), dtype)
    dg, du = ops.glu_backward(cg, cu, dy.to(cuda_device), act=act)
    gv, uv = fb.ckpt8(gate)[2], fb.ckpt8(up)[2]
    a, d, size = fb.act(act, gv)
    act_near(dg, 2 * uv * d, (2 * uv).abs() * size, gv, (2 * uv).abs(), dtype)
    inside = (2 * a).abs() < top * 0.999
    act_near(du.cpu()[inside], (2 * a)[inside], (2 * a).abs()[inside], gv[inside], torch.full_like(gv, 2.0)[inside], dtype)
    assert torch.equal(du.cpu().double()[~inside], (2 * a)[~inside].to(dtype).double())
    # what is not finite
    g = torch.tensor([[float("inf"), float("-inf"), float("nan"), 0.0, -0.0, 1.0]]).to(dtype)
    y = ops.glu(g.to(cuda_device), torch.ones_like(g).to(cuda_device), act=act).cpu()
    want = fb.act(act, g.double())[0].to(dtype)
    if act == "relu":
        want = torch.tensor([[float("inf"), 0.0, float("nan"), 0.0, 0.0, 1.0]]).to(dtype)
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.nan_to_num(nan=7.0, posinf=9.0)[:, :5], want.nan_to_num(nan=7.0, posinf=9.0)[:, :5])


# ---- gradients near the end of the range -------------------------------------------------------------


@pytest.mark.parametrize("exponent", [-100, -109, -113, -120, -127])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_weight_gradient_of_tiny_dy(cuda_device, dt, exponent):
    """A dy down to the last numbers below the normal range, times an x that brings the result back."""
    dtype, rows, c_in, c_out = fb.TYPES[dt], 200, 96, 40
    x = torch.randn(rows, c_in, generator=gen(1)) * 2.0 ** 90
    dy = (torch.randn(rows, c_out, generator=gen(2)).double() * 2.0 ** exponent).to(dtype)
    ck = ops.checkpoint_code8(x.to(cuda_device))
    xv = fb.ckpt8(x)[2]
    want, size = dy.double().T @ xv, dy.double().abs().T @ xv.abs()
    dw, db = ops.affine_weight_backward(ck, dy.to(cuda_device), dtype=torch.float32)
    # float32: the last of the three parts ends at bfloat16's last number, 2^-133
    lost = 2.0 ** -133 * xv.abs().sum(0) if dt == "f32" else torch.zeros(c_in, dtype=torch.float64)
    assert ((dw.cpu().double() - want).abs() <= (rows + 8) * 2.0 ** -23 * size + lost).all()
    wantb = dy.double().sum(0)
    assert ((db.cpu().double() - wantb).abs() <= (rows + 8) * 2.0 ** -24 * dy.double().abs().sum(0) + 2.0 ** -149).all()


@pytest.mark.parametrize("dt", TYPES)
def test_checkpoints_and_weights_near_zero(cuda_device, dt):
    """4-bit weights and rows whose products lie below the normal range of the type, brought back by the other factor."""
    dtype, rows, k, n, group = fb.TYPES[dt], 5, 256, 96, 64
    small, large = (2.0 ** -14, 1.0) if dt == "f16" else (2.0 ** -110, 2.0 ** 100)
    codes, scales, zeros, _ = w4_layer(n, k, group, torch.float32, True, cuda_device, 4)
    for xs, ss in ((small, large), (large, small)):
        x = (torch.randn(rows, k, generator=gen(3)).double() * xs).to(dtype)
        s = (scales.double() * ss).to(dtype)
        w = fb.w4_weight(codes, s, zeros, group)
        want, lim = w4_bound(x, w, torch.zeros(n), k, dtype)
        lim = lim + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        if dt == "f32":  # the parts of a row end at 2^-133
            lim = lim + 2.0 ** -133 * w.abs().sum(1)
        got = ops.affine_w4(x.to(cuda_device), packed(codes, s, zeros, group, cuda_device)).cpu().double()
        assert ((got - want).abs() <= lim).all()


@pytest.mark.parametrize("rows,c_in,c_out", [(1, 4500, 5000), (70, 4096, 6000), (129, 256, 20000), (600, 1024, 1100)])
@pytest.mark.parametrize("dt", TYPES)
def test_weight_gradient_units_of_every_length(cuda_device, dt, rows, c_in, c_out):
    """More tiles than SMs with one chunk of tokens each, two or a few; the exponents on and off a word boundary, accumulated too."""
    dtype = fb.TYPES[dt]
    g = torch.Generator(device=cuda_device).manual_seed(rows)
    # whole numbers: every sum is exact
    x = torch.randint(-127, 128, (rows, c_in), generator=g, device=cuda_device).float()
    x[:, ::32] = 127
    dy = torch.randint(-4, 5, (rows, c_out), generator=g, device=cuda_device).to(dtype)
    want = (dy.double().T @ x.double()).float()
    ck = ops.checkpoint_code8(x)
    buf = torch.zeros(ck.exponents.numel() + 1, dtype=torch.uint8, device=cuda_device)
    buf[1:] = ck.exponents.flatten()
    odd = ops.Code8Checkpoint(ck.codes, buf[1:].view(ck.exponents.shape), ck.shape, ck.dtype)
    for c in (ck, odd):
        dw, _ = ops.affine_weight_backward(c, dy, need=(True, False), dtype=torch.float32)
        assert torch.equal(dw, want)
        assert torch.equal(ops.affine_weight_backward(c, dy, need=(True, False))[0], want.to(dtype))
    acc, _ = ops.affine_weight_backward(odd, dy, dw=torch.ones_like(want), need=(True, False), accum=(True, False))
    assert torch.equal(acc, want + 1)
    ops.check_device_flag()


FIRST_CALL = """
import sys, torch
sys.path[:0] = sys.argv[1:]
from dwbnq import ops
x, dy = torch.randn(300, 256, device="cuda").half(), torch.randn(300, 200, device="cuda").half()
codes, scales = torch.randint(0, 16, (96, 256), device="cuda", dtype=torch.uint8), torch.rand(96, 2, device="cuda").half()
def step():
    y, cg, cu = ops.glu(x, x, checkpoint=True)
    dg, du = ops.glu_backward(cg, cu, x)
    dw, db = ops.affine_weight_backward(ops.checkpoint_code8(y), dy, dtype=torch.float32)
    return dg, du, dw, db, ops.affine_w4(x[:5], ops.pack_w4(codes, scales))
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = step()
x.copy_(torch.randn(300, 256, device="cuda"))
g.replay()
assert all(torch.equal(a, b) for a, b in zip(got, step()))
ops.check_device_flag()
print("same")
"""


def test_the_first_calls_of_a_process_may_be_captured(cuda_device):
    import os
    import subprocess
    import sys
    paths = [os.path.dirname(os.path.dirname(os.path.abspath(ops.__file__)))]
    out = subprocess.run([sys.executable, "-c", FIRST_CALL] + paths, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "same", out.stderr[-2000:]
