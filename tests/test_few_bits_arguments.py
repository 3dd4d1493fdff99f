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
