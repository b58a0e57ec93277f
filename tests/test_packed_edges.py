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


def _masking_bias(pack, heads, low):
    """Each head hides another stretch of relative positions by the lowest value of the type: near keys, far
    keys, those behind, those ahead, all of them; the rest is some +-1."""
    m = pack.longest
    d = torch.arange(1 - m, m, device="cuda")
    hide = [d.abs() < 140, d.abs() > 130, d < 0, d > 0, d == d, d == 3][:heads]
    b = torch.randn(heads, 2 * m - 1, generator=torch.Generator("cuda").manual_seed(3), device="cuda")
    return torch.where(torch.stack(hide), low, b)


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,keys,dim", [([300, 77], None, 64), ([1, 20], [2500, 1300], 64), ([300], [700], 128)])
def test_gpu_bias_of_the_lowest_value(lengths, keys, dim, causal, tiles):  # noqa: F811
    """Hidden keys have no weight, also where they fill the first key tiles of a row; a row all of whose keys are
    hidden weighs them alike, as scores that such a value swallows do (split along the keys or not)."""
    pack = ops.SequencePack(lengths, keys)
    q, k, v, _ = tensors(pack, 6, 3, dim, "cuda")
    low = torch.finfo(torch.float32).min
    bias = _masking_bias(pack, 6, low)
    o, lse = ops.packed_attention(q, k, v, pack, causal=causal, scale=0.1, rel_bias=bias, return_lse=True)
    ops.check_device_errors()
    HALF, F32 = 2.0 ** -8, 2.0 ** -23
    for a0, a, b0, b in zip(pack.starts, pack.lengths, pack.key_starts, pack.key_lengths):
        place, key = torch.arange(b - a, b, device="cuda")[:, None], torch.arange(b, device="cuda")[None]
        for h in range(6):
            qs, ks, vs = q[a0:a0 + a, h].double(), k[b0:b0 + b, h // 2].double(), v[b0:b0 + b, h // 2].double()
            add = bias[h][key - place + pack.longest - 1].double()
            seen = key <= place if causal else torch.ones(a, b, dtype=torch.bool, device="cuda")
            open_ = seen & (add > low)
            none = seen.any(1) & ~open_.any(1)
            s = qs @ ks.t() * 0.1
            es = (dim + 2) * F32 * 0.1 * (qs.abs() @ ks.abs().t()) + 8 * F32 * (s.abs() + 4)
            s = torch.where(none[:, None], 0.0, s + add).masked_fill(~torch.where(none[:, None], seen, open_), -math.inf)
            want = torch.logsumexp(s, 1)
            p = torch.where(torch.isinf(want)[:, None], 0.0, torch.exp(s - want[:, None]))
            off = (2 * es.masked_fill(~open_, 0.0).amax(1, keepdim=True) + 16 * F32 + F32 * b ** 0.5 * 4).expm1()
            ov = p @ vs
            close(o[a0:a0 + a, h], ov, HALF * ov.abs() + (1 + HALF) * (HALF + off + b * F32) * (p @ vs.abs()), f"o {h}")
            got = lse[a0:a0 + a, h].double()
            assert torch.isfinite(got[none]).all() and (got[none] < -6e37).all()
            close(got[~none], want[~none], (es.masked_fill(~open_, 0.0).amax(1) + 64 * F32 * (1 + s.masked_fill(
                torch.isinf(s), 0.0).abs().amax(1)))[~none], f"lse {h}")


@gpu
def test_gpu_bias_of_the_largest_value(tiles):  # noqa: F811
    """A row's keys of the largest value share its weight alike; a NaN stays one."""
    pack = ops.SequencePack([200])
    q, k, v, _ = tensors(pack, 2, 2, 64, "cuda")
    bias = torch.zeros(2, 399, device="cuda")
    bias[:, 199 - 4:199 + 1] = torch.finfo(torch.float32).max          # the last five positions
    o = ops.packed_attention(q, k, v, pack, scale=0.1, rel_bias=bias)
    want = torch.stack([v[max(0, i - 4):i + 1].double().mean(0) for i in range(200)])
    size = torch.stack([v[max(0, i - 4):i + 1].double().abs().mean(0) for i in range(200)])
    close(o, want, 2.0 ** -8 * want.abs() + 1.01 * 2.0 ** -8 * size, "o")
    bias[1, 199 - 150] = math.nan
    o = ops.packed_attention(q, k, v, pack, scale=0.1, rel_bias=bias)
    assert torch.isnan(o[150:, 1]).all() and torch.isfinite(o[:, 0]).all() and torch.isfinite(o[:150, 1]).all()
    ops.check_device_errors()


def test_waits_of_the_forward_kernel_are_bounded():
    """Warps that may give up at a bounded wait meet others only at waits that are bounded too, and once, all
    of them, before the block ends."""
    src = (pathlib.Path(ops.__file__).parent / "csrc" / "packed_attn_fwd.cu").read_text()
    kernel = src[src.index("packed_fwd_kernel(const __grid_constant__"):src.index("packed_combine_kernel(const int* joins")]
    assert "named_bar_sync" not in kernel and "bar.sync" not in kernel
    assert kernel.count("__syncthreads()") == 2
    roles = kernel[kernel.index("if (warp == L::kProdWarp) {\n    // ---"):kernel.rindex("__syncthreads()")]
    assert "__syncthreads" not in roles and "return;" not in roles


@gpu
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 128), (6, 2, 80), (3, 1, 72), (2, 2, 120), (4, 2, 40)])
@pytest.mark.parametrize("causal", [True, False])
def test_gpu_bias_with_other_heads(heads, kv, dim, causal, tiles):  # noqa: F811
    for lengths, keys in (([77, 1, 300], None), ([3, 130], [700, 131]), ([2], [3000])):
        pack = ops.SequencePack(lengths, keys)
        bias = torch.randn(heads, 2 * pack.longest + 5, generator=torch.Generator("cuda").manual_seed(3), device="cuda")
        _pass(pack, heads, kv, dim, causal, bias=bias, train=False, scale=0.05)


@gpu
def test_gpu_pack_first_used_in_inference_mode():
    """Work lists laid out in inference mode serve calls under autograd and captured ones."""
    with torch.inference_mode():
        pack = ops.SequencePack([100, 7])
        q, k, v, do = tensors(pack, 4, 2, 64, "cuda")
        want = ops.packed_attention(q, k, v, pack)
        ops.packed_attention_bwd(q, k, v, want, do, torch.zeros(107, 4, device="cuda"), pack)
    q, k, v, do = (t.clone() for t in (q, k, v, do))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = Fn.packed_attention(*leaves, pack)
    grads = torch.autograd.grad(out, leaves, do)
    fresh = ops.SequencePack([100, 7])
    again = torch.autograd.grad(Fn.packed_attention(*leaves, fresh), leaves, do)
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(grads, again))


def _rounded_run(q, k, v, do, pack, causal, scale):
    """dq, dk in 64 bits, and from weights, outputs and results rounded as the kernels round them (dS is not): the
    weights relative to their row's largest, o to bf16 and a byte of what that left."""
    b16 = lambda t: t.to(torch.bfloat16).double()  # noqa: E731
    out = [[torch.zeros_like(t, dtype=torch.float64) for t in (q, k)] for _ in range(2)]
    group = q.shape[1] // k.shape[1]
    for a0, n in zip(pack.starts, pack.lengths):
        for h in range(q.shape[1] if n else 0):
            at, g = slice(a0, a0 + n), h // group
            qs, ks, vs, ds_ = (t.double() for t in (q[at, h], k[at, g], v[at, g], do[at, h]))
            s = qs @ ks.t() * scale
            if causal:
                s = s.masked_fill(torch.ones_like(s).triu(1) > 0, -math.inf)
            p, e = torch.softmax(s, 1), torch.exp(s - s.amax(1, keepdim=True))
            o = (b16(e) @ vs) / e.sum(1, keepdim=True)
            low = ((o - b16(o)) * 256).to(torch.float8_e5m2).double() / 256
            dp = ds_ @ vs.t()
            for i, out_ in enumerate((p @ vs, b16(o) + low)):
                ds = p * (dp - (ds_ * out_).sum(1, keepdim=True)) * scale
                out[i][0][at, h] += ds @ ks
                out[i][1][at, g] += ds.t() @ qs
    return out[0], [b16(t) for t in out[1]]


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,heads,kv,dim", [([2] * 60, 8, 8, 64), ([1, 3, 5, 2, 8, 32] * 4, 4, 2, 128), ([17] * 30, 7, 1, 80),
                                                  ([32, 20, 31] * 6, 6, 1, 40), ([7] * 40, 16, 1, 96)])
def test_gpu_gradients_of_short_sequences(lengths, heads, kv, dim, causal):
    """As near to 64 bits as the rounding of weights and results allows; with dS rounded to bf16, 1.3 times as far.
    1.1: the kernels take the largest weight of a row some 2^8 late, which moves its roundings, and sums in fp32."""
    pack = ops.SequencePack(lengths)
    q, k, v, do = tensors(pack, heads, kv, dim, "cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(Fn.packed_attention(*leaves, pack, causal=causal), leaves, do)
    want, rounded = _rounded_run(q.detach(), k.detach(), v.detach(), do, pack, causal, dim ** -0.5)
    for g, w, r, n in zip(got, want, rounded, ("dq", "dk")):
        assert (g.double() - w).norm() <= 1.1 * (r - w).norm(), n
    ops.check_device_errors()


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,keys", [([1] * 11, None), ([1, 40, 1], [1, 1, 1]), ([3000], [1]), ([300, 1, 20], None)])
def test_gpu_gradients_of_rows_with_one_key(lengths, keys, causal):
    """A row that sees one key weighs it by 1 whatever the scores: its dq is zero, and the dk of a sequence of one
    key.  Zero, not what two sums over the same products leave."""
    pack = ops.SequencePack(lengths, keys)
    q, k, v, do = tensors(pack, 8, 2, 128, "cuda", std=3.0)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(Fn.packed_attention(*leaves, pack, causal=causal), leaves, do)
    for a0, a, b0, b in zip(pack.starts, pack.lengths, pack.key_starts, pack.key_lengths):
        sees = torch.arange(b - a + 1, b + 1).clamp(min=0) if causal else torch.full((a,), int(b))
        at = torch.arange(a0, a0 + a)[sees <= 1]
        assert not dq[at.cuda()].any()
        rest = torch.arange(a0, a0 + a)[sees > 1]
        assert len(rest) == 0 or dq[rest.cuda()].any(2).all()
        if b == 1:
            assert not dk[b0:b0 + 1].any() and dv[b0:b0 + 1].any()
    ops.check_device_errors()
