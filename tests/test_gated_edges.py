"""The gated feed-forward block at the ends of its range and in the forms that the sizes of the other tests do
not reach.  Bounds as there: half a bf16 step is 2^-8 of a value, sums run in fp32."""
import math

import pytest
import torch

from osp_next_b200 import ops
from osp_next_b200.models import functional as Fn
from test_gated_rotary import CURVE, F32, HALF, act64, close, ffn_tensors

gpu = pytest.mark.gpu


def kept(v):
    """What keeping a projection may lose: half a step of 9 bits of mantissa, of 6 far from 1."""
    a = v.abs()
    return torch.where((a >= 2.0 ** -19) & (a < 2.0 ** 15), 2.0 ** -10, 2.0 ** -7) * a + 2.0 ** -132


def gradients(x, wg, wu, wd, act, dy):
    """name -> (value in 64 bits, largest error), relative to the products at every size of the values."""
    x, wg, wu, wd, dy = (t.double() for t in (x, wg, wu, wd, dy))
    M, K, F, C = x.shape[0], x.shape[1], wg.shape[0], wd.shape[0]
    g, u = x @ wg.t(), x @ wu.t()
    kg, ku = (K * F32 * (x.abs() @ w.abs().t()) + kept(t) for w, t in ((wg, g), (wu, u)))
    a, d = act64(g.clamp(-1e5, 1e5), act)                              # the same from there on
    a, d = torch.where(g.abs() > 1e5, g.clamp(min=0), a), torch.where(g.abs() > 1e5, (g > 0).double(), d)
    fast = 2.0 ** -16                                                  # an exponential of up to 88
    da = 1.13 * kg + fast * a.abs()
    # beyond 200 the derivative is 0 or 1 on either side of the rounding
    dd = torch.where(g.abs() > 200, 0.0, CURVE * kg) + fast
    h, dh = a * u, dy @ wd
    edh = C * F32 * (dy.abs() @ wd.abs())
    eh = (da * u.abs() + (a.abs() + da) * ku) * (1 + HALF) + HALF * h.abs()
    dg, du = dh * u * d, dh * a
    edg = (edh * u.abs() * d.abs() + (dh.abs() + edh) * (ku * d.abs() + (u.abs() + ku) * dd)) * (1 + HALF) + HALF * dg.abs()
    edu = (edh * a.abs() + (dh.abs() + edh) * da) * (1 + HALF) + HALF * du.abs()

    def product(p, ep, q, terms):
        v = p @ q
        return v, (1 + HALF) * (ep @ q.abs() + terms * F32 * (p.abs() @ q.abs())) + HALF * v.abs()
    dx = [product(dg, edg, wg, 2 * F), product(du, edu, wu, 2 * F)]
    v = dx[0][0] + dx[1][0]
    return {"dx": (v, dx[0][1] + dx[1][1] + HALF * v.abs()), "dwg": product(dg.t(), edg.t(), x, M),
            "dwu": product(du.t(), edu.t(), x, M),
            "dwd": tuple(t.t() for t in product(h.t(), eh.t(), dy, M))}


@gpu
@pytest.mark.parametrize("size", [2.0 ** -50, 2.0 ** -32, 2.0 ** -18, 2.0 ** 14, 2.0 ** 33, 2.0 ** 50])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("M,K,F", [(40, 64, 136), (2600, 64, 2312)])
def test_gpu_gradients_of_small_and_large_projections(size, act, M, K, F):
    """Gradients stay within their roundings whatever the size of the projections: few rows and tiles."""
    x, wg, wu, wd, dy = ffn_tensors(M, K, F)
    x = x * size
    want = gradients(x, wg, wu, wd, act, dy)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    grads = torch.autograd.grad(Fn.gated_ffn(*leaves, act=act), leaves, dy)
    for got, n in zip(grads, ("dx", "dwg", "dwu", "dwd")):
        close(got, want[n], n)
    ops.check_device_errors()


@gpu
def test_gpu_kept_projections_at_their_ends():
    """One projection a column, from the smallest to the largest number and across the ends of the fine range: the
    gradient of the up weight is act(g), that of the down weight act(g) u."""
    e = torch.tensor([-133, -126, -125, -60, -31, -21, -20, -19, -1, 0, 6, 15, 16, 17, 31, 32, 60, 110, 126], dtype=torch.float64)
    vals = (torch.cat([s * m * 2 ** e for m in (1.0, 1.9921875) for s in (1, -1)])).float().bfloat16()
    vals = torch.cat([vals, vals.new_zeros(-len(vals) % 8)])
    F = len(vals)
    x = torch.zeros(1, 8, device="cuda", dtype=torch.bfloat16)
    x[0, 0] = 1.0
    wg, wu = (torch.zeros(F, 8, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    wg[:, 0], wu[:, 0] = vals.cuda(), 1.0
    wd, dy = torch.eye(F, device="cuda").bfloat16(), torch.ones(1, F, device="cuda").bfloat16()
    g = vals.cuda().double()
    for act in ("silu", "gelu_tanh"):
        leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
        _, dwg, dwu, dwd = torch.autograd.grad(Fn.gated_ffn(*leaves, act=act), leaves, dy)
        a, d = act64(g.clamp(-1e5, 1e5), act)
        a, d = torch.where(g.abs() > 1e5, g.clamp(min=0), a), torch.where(g.abs() > 1e5, (g > 0).double(), d)
        err = 1.13 * kept(g) + 2.0 ** -16 * a.abs() + HALF * a.abs()
        close(dwu[:, 0], (a, err + 2.0 ** -126), "act")               # products below 2^-126 may be cut
        close(dwd.diagonal(), (a, err + 2.0 ** -126), "h")
        close(dwg[:, 0], (d, torch.where(g.abs() > 200, 0.0, CURVE * kept(g)) + 2.0 ** -16 + HALF * d.abs()), "act'")
    ops.check_device_errors()


def _kernels(f):
    """Names of the block's kernels that a call launches."""
    from torch.profiler import ProfilerActivity, profile
    f()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        f()
        torch.cuda.synchronize()
    return [e.name for e in p.events() if "osp::ffn::" in e.name]


@gpu
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("M,K,F,C", [(2499, 2056, 2312, 2064), (5003, 776, 1032, 1160)])
def test_gpu_tiled_form(act, M, K, F, C):
    """Every product in whole tiles, with several blocks along K and ragged last tiles: values, all gradients,
    and gradients of fp32 leaves."""
    from test_gated_rotary import ffn_oracle
    x, wg, wu, wd, dy = ffn_tensors(M, K, F, C)
    want = ffn_oracle(x, wg, wu, wd, act, dy)
    close(ops.gated_linear(x, wg, wu, act), want["h"], "h")
    close(ops.gated_ffn(x, wg, wu, wd, act), want["y"], "y")
    for dtype in (torch.bfloat16, torch.float32):
        leaves = [t.to(dtype).requires_grad_(True) for t in (x, wg, wu, wd)]

        def step():
            return torch.autograd.grad(Fn.gated_ffn(*leaves, act=act), leaves, dy)
        if torch.cuda.get_device_properties(0).multi_processor_count <= 148:
            names = _kernels(step)                          # none where another profiler watches the process
            assert not names or (len(names) == 6 and all("::gemm<" in n for n in names)), names
        for got, n in zip(step(), ("dx", "dwg", "dwu", "dwd")):
            assert got.dtype == dtype
            close(got, want[n], n)
    ops.check_device_errors()


@gpu
def test_gpu_calls_at_once():
    """Both forms of the block, rotary and packed attention on streams of their own at once: what they give alone."""
    w = [ffn_tensors(1, K, F, seed=i)[1:4] for i, (K, F) in enumerate(((1024, 2048), (512, 4096), (2048, 512)))]
    xs = [[ffn_tensors(m, k[0].shape[1], 8, seed=m)[0] for m in (1, 40, 154, 256, 3000)] for k in w]
    pack = ops.SequencePack([300, 5, 77])
    q = torch.randn(382, 8, 64, device="cuda").bfloat16()
    table, pos = ops.rotary_table(64, 400), torch.arange(382, device="cuda")

    def work(i):
        out = [ops.gated_ffn(x, *w[i]) for x in xs[i]]
        z = ops.rotary(q, None, pos, table)[0]
        return out + [z, ops.packed_attention(z, z, z, pack, causal=bool(i % 2))]
    want = [work(i) for i in range(3)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [[], [], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(work(i))
    torch.cuda.synchronize()
    for i in range(3):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[i]))
    ops.check_device_errors()
