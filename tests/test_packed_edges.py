"""Packed attention at the ends of its arguments: scales of any sign, biases to the largest values, heads
and forms that the sizes of the other tests do not reach.  Bounds as there."""
import math
import pathlib

import pytest
import torch

from osp_next_b200 import ops
from osp_next_b200.models import functional as Fn
from osp_next_b200.ops import packed
from test_packed_attention import _pass, close, oracle, tensors, tiles  # noqa: F401

gpu = pytest.mark.gpu


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 1e39])
def test_scale_refusals(scale):
    pack = ops.SequencePack([3], device="cpu")
    q, k, v, do = tensors(pack, 2, 2, 8, "cpu", dtype=torch.float32)
    for call in (ops.packed_attention, Fn.packed_attention):
        with pytest.raises(ValueError, match="finite scale"):
            call(q, k, v, pack, scale=scale)
    with pytest.raises(ValueError, match="finite scale"):
        ops.packed_attention_bwd(q, k, v, q, do, q[..., 0], pack, scale=scale)


def _negative(pack, heads, kv, dim, causal, scale, std, bias=None):
    """The same as -q at the scale -scale, where the oracle's bounds have their sign."""
    q, k, v, do = tensors(pack, heads, kv, dim, "cuda", std=std)
    want = oracle(-q, k, v, pack, causal, -scale, bias, do if bias is None else None)
    o, lse = ops.packed_attention(q, k, v, pack, causal=causal, scale=scale, rel_bias=bias, return_lse=True)
    close(o, want["o"], want["eo"], "o")
    close(lse, want["lse"], want["else"], "lse")
    if bias is None:
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        grads = torch.autograd.grad(Fn.packed_attention(*leaves, pack, causal=causal, scale=scale), leaves, do)
        close(-grads[0], want["dq"], want["edq"], "dq")
        close(grads[1], want["dk"], want["edk"], "dk")
        close(grads[2], want["dv"], want["edv"], "dv")
    ops.check_device_errors()


@gpu
@pytest.mark.parametrize("causal", [True, False])
def test_gpu_negative_scale(causal, tiles):  # noqa: F811
    """Rows that see nothing of a key tile (limits not aligned with tiles), scores that spread over hundreds."""
    for lengths, keys in (([100], [150]), ([300, 5], None), ([1, 40], [2000, 130])):
        for heads, kv, dim in ((4, 4, 64), (6, 2, 128), (7, 1, 80)):
            _negative(ops.SequencePack(lengths, keys), heads, kv, dim, causal, -0.11, 1.0)
            _negative(ops.SequencePack(lengths, keys), heads, kv, dim, causal, -0.125, 6.0)
    pack = ops.SequencePack([100, 200])
    _negative(pack, 4, 2, 64, causal, -0.11, 1.0, torch.randn(4, 399, device="cuda"))


@gpu
def test_gpu_scale_of_zero_and_refusals(tiles):  # noqa: F811
    pack = ops.SequencePack([100, 3], [150, 3])
    _pass(pack, 6, 2, 64, True, scale=0.0)
    q, k, v, do = tensors(pack, 6, 2, 64, "cuda")
    for scale in (math.nan, math.inf, 1e39):
        for call in (ops.packed_attention, Fn.packed_attention):
            with pytest.raises(ValueError, match="finite scale"):
                call(q, k, v, pack, scale=scale)
        with pytest.raises(ValueError, match="finite scale"):
            ops.packed_attention_bwd(q, k, v, q, do, torch.zeros(103, 6, device="cuda"), pack, scale=scale)
