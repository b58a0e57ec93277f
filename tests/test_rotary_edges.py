"""Rotary positions at the ends of their arguments: positions of every type and size, gradients of the
inverse and of the table, captured and replayed."""
import pytest
import torch

from osp_next_b200 import ops
from osp_next_b200.models import functional as Fn
from osp_next_b200.ops import reference as ref
from test_gated_rotary import close, turned

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("far", [2 ** 32 + 5, 2 ** 40, -2 ** 32 + 5, 2 ** 31, -2 ** 31, 2 ** 63 - 1, -2 ** 63])
def test_gpu_positions_beyond_32_bits(far):
    """Outside the table, whatever their low 32 bits."""
    table = ops.rotary_table(64, 100)
    q = torch.randn(9, 3, 64, device="cuda").bfloat16()
    pos = torch.arange(9, device="cuda")
    want = ops.rotary(q, None, pos, table)[0]
    ops.check_device_errors()
    pos[4] = far
    got = ops.rotary(q, None, pos, table)[0]
    with pytest.raises(ops.DeviceWaitError, match="rotary position"):
        ops.check_device_errors()
    rest = torch.arange(9, device="cuda") != 4
    assert torch.isnan(got[4]).all() and torch.equal(got[rest], want[rest])


@gpu
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64, torch.uint16,
                                   torch.uint32, torch.uint64])
def test_gpu_types_of_positions(dtype):
    table = ops.rotary_table(64, 100)
    q = torch.randn(2, 9, 3, 64, device="cuda").bfloat16()
    pos = torch.tensor([0, 99, 3, 5, 98, 1, 2, 77, 50], device="cuda")
    close(ops.rotary(q, None, pos.to(dtype), table)[0][1], turned(q[1], pos[:, None], table, "half", [32]), str(dtype))
    two = torch.stack([pos, pos.flip(0)], 1)
    close(ops.rotary(q, None, two.to(dtype), table, "interleaved", [20, 12])[0][1],
          turned(q[1], two, table, "interleaved", [20, 12]), str(dtype))
    ops.check_device_errors()
