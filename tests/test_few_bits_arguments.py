"""Arguments of the few-bit wrappers that would reach past a tensor if they were taken, or that fail in a way of their own (CPU: they
are refused before a device is asked for)."""
import pytest
import torch

from dwbnq import _lib as L
from dwbnq import ops


def checkpoint(rows=64, cols=40):
    groups = (cols + 31) // 32
    return ops.Code8Checkpoint(torch.zeros(rows, 32 * groups, dtype=torch.int8), torch.zeros(rows, groups, dtype=torch.uint8), (rows, cols),
                               torch.float32)


def test_a_workspace_is_memory_of_its_size():
    """A broadcast or strided tensor has as many elements as its shape says, but not as many bytes behind its address."""
    dy = torch.zeros(64, 24)
    for ws in (torch.zeros(1, dtype=torch.uint8).expand(1 << 24), torch.zeros(1 << 12, 1).expand(1 << 12, 1 << 12),
               torch.zeros(1 << 12, 1 << 12, dtype=torch.uint8)[:, ::2], torch.zeros(64, 1 << 17).T):
        with pytest.raises(ValueError, match="ws must be contiguous"):
            ops.affine_weight_backward(checkpoint(), dy, ws=ws)


def test_packed_weights_are_as_large_as_their_layer():
    """Packed weights kept by the caller (from a file, of another layer or group size) are checked where they are given."""
    need = 2048 + 256  # 8 channels of 240 in groups of 128: two blocks of 1 KiB, 2 x 16 scales of 2 bytes each
    new = lambda packed, **kw: ops.W4Weight(packed, *(kw.get(k, v) for k, v in (("c_out", 8), ("c_in", 240), ("group", 128))),  # noqa: E731
                                            torch.bfloat16, False)
    assert new(torch.zeros(need, dtype=torch.uint8)).packed.numel() == need
    assert new(torch.zeros(need + 5, dtype=torch.uint8)).packed is not None
    for bad in (torch.zeros(need - 256, dtype=torch.uint8), torch.zeros(need), torch.zeros(1, dtype=torch.uint8).expand(need),
                torch.zeros(2 * need, dtype=torch.uint8)[::2], torch.zeros(need, dtype=torch.int8)):
        with pytest.raises(ValueError, match="packed"):
            new(bad)
        w4 = new(torch.zeros(need, dtype=torch.uint8))
        with pytest.raises(ValueError, match="packed"):
            w4.packed = bad
    for other in (dict(c_in=257), dict(c_out=17), dict(c_in=512, group=32)):
        with pytest.raises(ValueError, match="packed"):
            new(torch.zeros(need, dtype=torch.uint8), **other)
    w4 = new(None)
    with pytest.raises(ValueError, match="packed"):
        ops.affine_w4(torch.zeros(1, 240, dtype=torch.bfloat16), w4)


@pytest.mark.parametrize("group", [0, -32, 16, 48, 256])
def test_group_sizes_are_refused_alike(group):
    """A group size that does not exist is the library's refusal, whatever the number."""
    codes, scales = torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 4)
    for call in (lambda: ops.quantize_w4(torch.zeros(4, 64), group=group), lambda: ops.pack_w4(codes, scales, group=group)):
        with pytest.raises(L.DwbnqError) as e:
            call()
        assert e.value.status == L.ERR_UNSUPPORTED


def test_tensors_without_an_axis_are_refused():
    one = torch.zeros(())
    for call in (lambda: ops.checkpoint_code8(one), lambda: ops.glu(one, one), lambda: ops.affine_weight_backward(checkpoint(), one)):
        with pytest.raises(ValueError):
            call()
