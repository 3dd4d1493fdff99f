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
