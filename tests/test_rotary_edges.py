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


@gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rot,sections", [(32, None), (64, [10, 12, 10]), (24, [12, 0]), (0, None), (2, [0, 1])])
def test_gpu_a_bad_position_makes_its_whole_token_nan(layout, dtype, rot, sections):
    """The copied elements, the pairs of the other axes and heads of k too, from any axis, also one without pairs."""
    table = ops.rotary_table(rot, 100) if rot else torch.zeros(100, 0, 2, device="cuda")
    g = torch.Generator("cuda").manual_seed(1)
    q, k = (torch.randn(9, h, 64, generator=g, device="cuda").to(dtype) for h in (5, 2))
    axes = 1 if sections is None else len(sections)
    pos = torch.randint(0, 100, (9, axes), generator=g, device="cuda")
    kw = dict(layout=layout, sections=sections)
    want = ops.rotary(q, k, pos, table, **kw)
    ops.check_device_errors()
    for axis in range(axes):
        for value in (100, -1):
            bad = pos.clone()
            bad[4, axis] = value
            got = ops.rotary(q, k, bad, table, **kw)
            with pytest.raises(ops.DeviceWaitError, match="rotary position"):
                ops.check_device_errors()
            rest = torch.arange(9, device="cuda") != 4
            for a, b in zip(got, want):
                assert torch.isnan(a[4]).all() and torch.equal(a[rest], b[rest])
            with pytest.raises(IndexError, match="positions 0 to 99"):
                ops.rotary(q.cpu(), k.cpu(), bad.cpu(), table.cpu(), **kw)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("layout,inverse", [("half", False), ("interleaved", True)])
def test_gradient_of_the_table(device, layout, inverse):
    """No call drops it: against differences, alone and beside that of q, and refused where nothing is recorded."""
    g = torch.Generator().manual_seed(1)
    table = torch.randn(10, 4, 2, generator=g).to(device)
    q, do = (torch.randn(3, 2, 8, generator=g).to(device) for _ in range(2))
    pos = torch.tensor([2, 9, 2], device=device)
    leaf = table.clone().requires_grad_()
    for x in (q, q.clone().requires_grad_()):
        got, = torch.autograd.grad(Fn.rotary(x, None, pos, leaf, layout, inverse=inverse)[0], leaf, do)
        for at in ((2, 0, 0), (2, 3, 1), (9, 1, 1), (4, 0, 0)):
            step = torch.zeros_like(table)
            step[at] = 0.5                                              # the rotation is linear in the table
            want = sum(s * (ref.rotary(q.double(), pos[:, None], table + s * step, layout, [4], inverse) * do).sum()
                       for s in (1, -1))
            # cosines and sines of some 3 as fp32, 2^-23 each, times 3 x 2 x 8 products of some 1
            assert abs(got[at] - want) <= 48 * 3 * 2.0 ** -23 * 4, at
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.rotary(q, None, pos, leaf)
    with torch.no_grad():
        assert not ops.rotary(q, None, pos, leaf)[0].requires_grad


@gpu
def test_gpu_inverse_and_second_derivatives_are_captured():
    """The inverse under autograd, its gradient and the gradient of that, in a graph: no copy from the host."""
    table = ops.rotary_table(64, 100)
    pos = torch.arange(20, device="cuda")
    g = torch.Generator("cuda").manual_seed(1)
    static = [torch.randn(20, 3, 64, generator=g, device="cuda") for _ in range(3)]

    def step(x, do, dd):
        x, do = x.detach().requires_grad_(True), do.detach().requires_grad_(True)
        y = Fn.rotary(x, None, pos, table, inverse=True)[0]
        gx, = torch.autograd.grad(y, x, do, create_graph=True)
        gdo, = torch.autograd.grad(gx, do, dd)
        return y.detach(), gx.detach(), gdo
    want = step(*static)
    for i, back in ((0, True), (1, False), (2, True)):
        close(want[i], turned(static[i], pos[:, None], table, "half", [32], back), str(i))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = step(*static)
    for t in static:
        t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, step(*static)))


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.uint16, torch.uint32,
                                   torch.uint64])
def test_types_of_positions(dtype):
    table = ops.rotary_table(8, 100, device="cpu")
    q, pos = torch.randn(3, 2, 8), torch.tensor([0, 99, 3])
    assert torch.equal(ops.rotary(q, None, pos.to(dtype), table)[0], ops.rotary(q, None, pos, table)[0])
    if dtype.is_signed:
        with pytest.raises(IndexError, match="positions 0 to 99"):
            ops.rotary(q, None, torch.tensor([0, -1, 3], dtype=dtype), table)
    with pytest.raises(IndexError, match="positions 0 to 99"):
        ops.rotary(q, None, torch.tensor([0, 100, 3], dtype=dtype), table)
