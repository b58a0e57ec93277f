"""The gated feed-forward block and rotary positions against their formulas in 64 bits, and a layer made
of them and packed attention.  Bounds count roundings: half a bf16 step is 2^-8 of a value; sums run in
fp32 (2^-23 a term); the activation's exponential and reciprocal are within 2^-20."""
import math

import pytest
import torch

from osp_next_b200 import ops
from osp_next_b200.models import functional as Fn
from osp_next_b200.ops import reference as ref

HALF, F32 = 2.0 ** -8, 2.0 ** -23
gpu = pytest.mark.gpu


def act64(g, kind):
    """act(g) and its derivative in 64 bits."""
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


CURVE = 1.2      # largest |act''| of both


def ffn_oracle(x, wg, wu, wd, act, dy=None):
    """name -> (value in 64 bits, largest error)."""
    x, wg, wu, wd = (t.double() for t in (x, wg, wu, wd))
    K, F, M = x.shape[1], wg.shape[0], x.shape[0]
    g, u = x @ wg.t(), x @ wu.t()
    eg, eu = (K * F32 * (x.abs() @ w.abs().t()) for w in (wg, wu))
    a, d = act64(g, act)
    h = a * u
    fast = 2.0 ** -20
    eh = (1.13 * eg + fast * a.abs()) * u.abs() + a.abs() * eu + HALF * h.abs()
    eh = eh * (1 + HALF)
    y = h @ wd.t()
    out = {"h": (h, eh), "y": (y, HALF * y.abs() + (1 + HALF) * (eh @ wd.abs().t() + F * F32 * (h.abs() @ wd.abs().t())))}
    if dy is None:
        return out
    dy = dy.double()
    C = wd.shape[0]
    dh = dy @ wd
    edh = C * F32 * (dy.abs() @ wd.abs())
    # kept projections have 9 bits of mantissa: off by half a step, 2^-10; zero below 2^-31
    kg, ku = eg + 2.0 ** -10 * g.abs() + 2.0 ** -31, eu + 2.0 ** -10 * u.abs() + 2.0 ** -31
    da = 1.13 * kg + fast * (a.abs() + 1)
    h2 = (h, (da * u.abs() + (a.abs() + da) * ku) * (1 + HALF) + HALF * h.abs())
    dg, du = dh * u * d, dh * a
    edg = (edh * u.abs() * d.abs() + dh.abs() * ku * (d.abs() + 0.01) + dh.abs() * (u.abs() + ku) * (CURVE * kg + 2 * fast)
           ) * (1 + HALF) + HALF * dg.abs()
    edu = (edh * a.abs() + (dh.abs() + edh) * da) * (1 + HALF) + HALF * du.abs()

    def product(p, ep, q, terms):
        v = p @ q
        return v, (1 + HALF) * (ep @ q.abs() + terms * F32 * (p.abs() @ q.abs())) + HALF * v.abs()
    dx1, e1 = product(dg, edg, wg, 2 * F)
    dx2, e2 = product(du, edu, wu, 2 * F)
    out["dx"] = (dx1 + dx2, e1 + e2 + HALF * (dx1 + dx2).abs())
    out["dwg"] = product(dg.t(), edg.t(), x, M)
    out["dwu"] = product(du.t(), edu.t(), x, M)
    v = dy.t() @ h
    out["dwd"] = (v, (1 + HALF) * (dy.abs().t() @ h2[1] + M * F32 * (dy.abs().t() @ h.abs())) + HALF * v.abs())
    return out


def close(got, want, what):
    v, e = want
    d = (got.double() - v).abs()
    assert got.shape == v.shape and not torch.isnan(d).any(), what
    worst = (d - e).max().item() if d.numel() else -1.0
    assert worst <= 1e-30, f"{what}: {worst:.3g} over the bound (largest error {d.max().item():.3g})"


def ffn_tensors(M, K, F, C=None, device="cuda", seed=0, dtype=torch.bfloat16):
    g = torch.Generator(device=device).manual_seed(seed)

    def rand(*s, std=1.0):
        return (torch.randn(*s, generator=g, device=device) * std).to(dtype)
    C = K if C is None else C
    return rand(M, K), rand(F, K, std=K ** -0.5), rand(F, K, std=K ** -0.5), rand(C, F, std=F ** -0.5), rand(M, C)


# ---------------------------------------------------------------------------- CPU

@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_ffn_reference(act):
    x, wg, wu, wd, dy = ffn_tensors(3, 5, 7, 4, "cpu", dtype=torch.float64)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    assert torch.autograd.gradcheck(lambda *t: Fn.gated_ffn(*t, act=act), leaves)
    want = ffn_oracle(*[t.detach() for t in leaves], act, dy)
    with torch.no_grad():
        assert torch.allclose(ops.gated_linear(x, wg, wu, act), want["h"][0], atol=1e-12)
        assert torch.allclose(ops.gated_ffn(x, wg, wu, wd, act), want["y"][0], atol=1e-12)
    grads = torch.autograd.grad(Fn.gated_ffn(*leaves, act=act), leaves, dy)
    for got, n in zip(grads, ("dx", "dwg", "dwu", "dwd")):
        assert torch.allclose(got, want[n][0], atol=1e-12), n


def test_ffn_refusals():
    x, wg, wu, wd, _ = ffn_tensors(3, 8, 16, 8, "cpu", dtype=torch.float32)
    with pytest.raises(ValueError, match="act one of"):
        ops.gated_linear(x, wg, wu, "relu")
    with pytest.raises(ValueError, match="against weights"):
        ops.gated_linear(x[:, :4], wg, wu)
    with pytest.raises(ValueError, match="against weights"):
        ops.gated_linear(x, wg, wu[:8])
    with pytest.raises(ValueError, match="down weight"):
        Fn.gated_ffn(x, wg, wu, wd[:, :8])
    with pytest.raises(TypeError, match="floating-point"):
        ops.gated_linear(x.int(), wg, wu)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.gated_ffn(x, wg, wu, wd.requires_grad_())


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("scaling", [None, {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 4.0},
                                     {"type": "yarn", "factor": 8.0, "original_len": 64}])
def test_rotary_reference(layout, scaling):
    table = ops.rotary_table(8, 50, 100.0, scaling, device="cpu")
    f, mult = ops.rotary_angles(8, 100.0, scaling)
    pos = torch.tensor([0, 49, 7])
    q = torch.randn(3, 2, 12, dtype=torch.float64)
    got, none = ops.rotary(q, None, pos, table, layout)
    assert none is None
    z = torch.polar(torch.full((3, 4), mult, dtype=torch.float64), pos.double()[:, None] * f)[:, None]
    head = q[..., :8]
    pairs = torch.complex(head[..., :4], head[..., 4:]) if layout == "half" else torch.view_as_complex(
        head.reshape(3, 2, 4, 2).contiguous())
    w = pairs * z
    want = torch.cat([w.real, w.imag], -1) if layout == "half" else torch.view_as_real(w).flatten(-2)
    assert torch.allclose(got[..., :8], want, atol=1e-6) and torch.equal(got[..., 8:], q[..., 8:])
    back, _ = ops.rotary(got, None, pos, table, layout, inverse=True)
    assert torch.allclose(back[..., :8], head * mult ** 2, atol=1e-6)
    q.requires_grad_()
    assert torch.autograd.gradcheck(lambda t: Fn.rotary(t, None, pos, table, layout)[0], [q])


def test_rotary_scaling_ends():
    """Fast pairs keep their angle, slow ones take the factor; turns within the trained length decide."""
    f, _ = ops.rotary_angles(64)
    y, mult = ops.rotary_angles(64, scaling={"type": "yarn", "factor": 8.0, "original_len": 4096})
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(y[turns > 40], f[turns > 40]) and torch.allclose(y[turns < 0.7], f[turns < 0.7] / 8)
    assert math.isclose(mult, 0.1 * math.log(8) + 1)
    n, _ = ops.rotary_angles(64, scaling={"type": "ntk", "factor": 8.0})
    assert math.isclose(float(n[0]), 1.0) and math.isclose(float(n[-1] * 8), float(f[-1]), rel_tol=1e-12)


def test_rotary_of_the_dit_matches_the_reference():
    pos = torch.stack([torch.randint(0, 60, (11,)) for _ in range(3)], 1)
    freqs = ref.rope_freqs(64)
    x = torch.randn(2, 11, 3, 64)
    want = ref.apply_rope(x, pos, freqs)
    table = torch.stack([freqs.double().cos(), freqs.double().sin()], -1).float()
    got, _ = ops.rotary(x, None, pos, table, "interleaved", ref.rope_split(64))
    assert torch.allclose(got, want, atol=1e-5)


def test_rotary_refusals():
    table = ops.rotary_table(8, 10, device="cpu")
    q = torch.randn(3, 2, 8)
    pos = torch.arange(3)
    with pytest.raises(ValueError, match="layout"):
        ops.rotary(q, None, pos, table, "both")
    with pytest.raises(ValueError, match=r"\[..., n, heads, head_dim\]"):
        ops.rotary(q, q[:2], pos, table)
    with pytest.raises(TypeError, match="one type"):
        ops.rotary(q, q.double(), pos, table)
    with pytest.raises(ValueError, match="table of 4 pairs"):
        ops.rotary(q[..., :6], None, pos, table)
    with pytest.raises(ValueError, match="table fp32"):
        ops.rotary(q, None, pos, table.double())
    with pytest.raises(TypeError, match="whole positions"):
        ops.rotary(q, None, pos.float(), table)
    with pytest.raises(ValueError, match=r"pos \[3\]"):
        ops.rotary(q, None, pos[:2], table)
    with pytest.raises(ValueError, match="sections"):
        ops.rotary(q, None, pos[:, None].repeat(1, 2), table, sections=[2, 1])
    with pytest.raises(IndexError, match="positions 0 to 9"):
        ops.rotary(q, None, pos + 8, table)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.rotary(q.requires_grad_(), None, pos, table)
    with pytest.raises(ValueError, match="even"):
        ops.rotary_table(7, 10, device="cpu")
    with pytest.raises(ValueError, match="scaling type"):
        ops.rotary_angles(8, scaling={"type": "cubic", "factor": 2})
    with pytest.raises(ValueError, match="unknown scaling keys"):
        ops.rotary_angles(8, scaling={"type": "linear", "factor": 2, "original_len": 3})
    with pytest.raises(ValueError, match="original_len"):
        ops.rotary_angles(8, scaling={"type": "yarn", "factor": 2})


# ---------------------------------------------------------------------------- GPU

FFN_SIZES = [(1, 64, 128, None), (1, 4096, 1024, None), (3, 136, 264, 72), (64, 256, 136, None), (65, 512, 1000, 520),
             (129, 72, 8, 8), (154, 1024, 2560, None), (300, 1536, 520, None), (1000, 200, 2200, None)]


@gpu
@pytest.mark.parametrize("M,K,F,C", FFN_SIZES)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_gpu_ffn(M, K, F, C, act):
    x, wg, wu, wd, dy = ffn_tensors(M, K, F, C)
    want = ffn_oracle(x, wg, wu, wd, act, dy)
    close(ops.gated_linear(x, wg, wu, act), want["h"], "h")
    close(ops.gated_ffn(x, wg, wu, wd, act), want["y"], "y")
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = Fn.gated_ffn(*leaves, act=act)
    close(y.detach(), want["y"], "y under autograd")
    for g, n in zip(torch.autograd.grad(y, leaves, dy), ("dx", "dwg", "dwu", "dwd")):
        close(g, want[n], n)
    ops.check_device_errors()


@gpu
def test_gpu_ffn_odd_sizes_views_and_types():
    x, wg, wu, wd, dy = ffn_tensors(7, 45, 83, 31)
    want = ffn_oracle(x, wg, wu, wd, "silu", dy)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = Fn.gated_ffn(*leaves)
    close(y.detach(), want["y"], "y")
    for g, n in zip(torch.autograd.grad(y, leaves, dy), ("dx", "dwg", "dwu", "dwd")):
        close(g, want[n], n)
    x, wg, wu, wd, dy = ffn_tensors(40, 128, 256)
    want = ops.gated_ffn(x, wg, wu, wd)
    stacked = torch.cat([wg, wu])                                      # both projections in one parameter
    assert torch.equal(ops.gated_ffn(x, *stacked.chunk(2), wd), want)
    wide = torch.zeros(40, 129, device="cuda", dtype=torch.bfloat16)
    wide[:, 1:] = x
    assert torch.equal(ops.gated_ffn(wide[:, 1:], wg, wu, wd), want)
    assert torch.equal(ops.gated_ffn(x.view(2, 20, 128), wg, wu, wd), want.view(2, 20, 128))
    leaves = [t.float().requires_grad_(True) for t in (x, wg, wu, wd)]     # fp32 master weights
    y = Fn.gated_ffn(*leaves)
    assert y.dtype == torch.bfloat16 and torch.equal(y, want)
    exact = ffn_oracle(x, wg, wu, wd, "silu", dy)
    for g, n in zip(torch.autograd.grad(y, leaves, dy), ("dx", "dwg", "dwu", "dwd")):
        assert g.dtype == torch.float32
        close(g, exact[n], n)
    frozen = [x.detach().requires_grad_(True), wg, wu.detach().requires_grad_(True), wd]
    y = Fn.gated_ffn(*frozen)
    gx, gu = torch.autograd.grad(y, [frozen[0], frozen[2]], dy.expand_as(y))
    close(gx, exact["dx"], "dx")
    close(gu, exact["dwu"], "dwu alone")
    for shape in ((0, 128), (2, 0, 128)):
        e = torch.zeros(shape, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        out = Fn.gated_ffn(e, wg, wu, wd)
        assert out.shape == shape
        g, = torch.autograd.grad(out.sum(), e)
        assert g.shape == shape
    leaf = wg.detach().requires_grad_(True)
    g, = torch.autograd.grad(Fn.gated_ffn(x[:0], leaf, wu, wd).sum(), leaf)
    assert (g == 0).all()


@gpu
def test_gpu_ffn_far_values():
    """Projections to +-1e4: the activation's ends, no NaN from its exponential."""
    x = torch.tensor([[1.0, -1.0] * 4], device="cuda").bfloat16()
    wg = torch.zeros(16, 8, device="cuda")
    wg[:, 0] = torch.tensor([0, 1, -1, 20, -20, 90, -90, 200, -200, 1e3, -1e3, 1e4, -1e4, 3, -3, 0.01])
    wu, wd = torch.eye(16, 8, device="cuda").bfloat16() + 1, torch.eye(16, device="cuda").bfloat16()
    wg = wg.bfloat16()
    dy = torch.ones(1, 16, device="cuda").bfloat16()
    for act in ("silu", "gelu_tanh"):
        want = ffn_oracle(x, wg, wu, wd, act, dy)
        leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
        y = Fn.gated_ffn(*leaves, act=act)
        close(y.detach(), want["y"], "y")
        for g, n in zip(torch.autograd.grad(y, leaves, dy), ("dx", "dwg", "dwu", "dwd")):
            assert torch.isfinite(g).all()
            close(g, want[n], n)


def turned(x, pos, table, layout, sections, inverse=False):
    """(value in 64 bits, largest error) from the table as it is: two products and a sum in fp32."""
    r = 2 * table.shape[1]
    axis = torch.repeat_interleave(torch.tensor(sections, device=x.device))
    cs = table.double()[pos.long()[:, axis], torch.arange(r // 2, device=x.device)]
    c, s = cs[:, None, :, 0], cs[:, None, :, 1] * (-1 if inverse else 1)
    y = x.double()
    a, b = (y[..., :r // 2], y[..., r // 2:r]) if layout == "half" else (y[..., 0:r:2], y[..., 1:r:2])
    parts = (a * c - b * s, a * s + b * c)
    errs = ((a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs())

    def join(p):
        return torch.cat(p, -1) if layout == "half" else torch.stack(p, -1).flatten(-2)
    half = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps              # half a step of the smallest values
    v = torch.cat([join(parts), y[..., r:]], -1)
    e = torch.cat([half * join(parts).abs() + 2 * 2.0 ** -24 * (1 + half) * join(errs) + tiny,
                   torch.zeros_like(y[..., r:])], -1)
    return v, e


@gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,heads,kv,dim,rot", [(1, 12, 2, 128, 128), (33, 5, 1, 80, 40), (7, 1, 1, 256, 256), (100, 3, 3, 64, 6),
                                                (9, 2, 1, 10, 4), (65, 40, 8, 96, 2)])
def test_gpu_rotary(layout, dtype, n, heads, kv, dim, rot):
    table = ops.rotary_table(rot, 500, 1000.0)
    g = torch.Generator("cuda").manual_seed(1)
    qkv = torch.randn(n, heads + 2 * kv, dim, generator=g, device="cuda").to(dtype)
    q, k = qkv[:, :heads], qkv[:, heads:heads + kv]
    for sections in ([rot // 2], [rot // 2 - 2 * (rot // 6), rot // 6, rot // 6]):
        pos = torch.randint(0, 500, (n, len(sections)), generator=g, device="cuda")
        kw = dict(layout=layout, sections=None if len(sections) == 1 else sections)
        p = pos[:, 0] if len(sections) == 1 else pos
        gq, gk = ops.rotary(q, k, p, table, **kw)
        close(gq, turned(q, pos, table, layout, sections), "q")
        close(gk, turned(k, pos, table, layout, sections), "k")
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k)]
        dq, dk = (torch.randn(t.shape, generator=g, device="cuda").to(dtype) for t in (q, k))
        grads = torch.autograd.grad(Fn.rotary(*leaves, p, table, **kw), leaves, [dq, dk])
        close(grads[0], turned(dq, pos, table, layout, sections, True), "dq")
        close(grads[1], turned(dk, pos, table, layout, sections, True), "dk")
    ops.check_device_errors()


@gpu
def test_gpu_rotary_addresses_batches_and_bad_positions():
    table = ops.rotary_table(64, 100)
    x = torch.randn(50 * 3 * 64 + 3, device="cuda").bfloat16()
    pos = torch.arange(50, device="cuda")
    for off in (0, 1, 2, 3):
        q = x[off:off + 50 * 3 * 64].view(50, 3, 64)
        for layout in ("half", "interleaved"):
            close(ops.rotary(q, None, pos, table, layout)[0], turned(q, pos[:, None], table, layout, [32]), str(off))
    q = x[:50 * 3 * 64].view(2, 25, 3, 64)
    got, _ = ops.rotary(q, None, pos[:25], table)
    assert torch.equal(got[1], ops.rotary(q[1], None, pos[:25], table)[0])
    one = q[0, :, :1].expand(25, 3, 64)
    assert torch.equal(ops.rotary(one, None, pos[:25], table)[0], ops.rotary(one.contiguous(), None, pos[:25], table)[0])
    e, _ = ops.rotary(q[:, :0], None, pos[:0], table)
    assert e.shape == (2, 0, 3, 64)
    ops.check_device_errors()
    bad = pos[:25].clone()
    bad[3], bad[7] = 100, -1
    got, _ = ops.rotary(q[0], None, bad, table)
    with pytest.raises(ops.DeviceWaitError, match="rotary position"):
        ops.check_device_errors()
    rest = torch.ones(25, dtype=torch.bool, device="cuda")
    rest[[3, 7]] = False
    assert torch.isnan(got[~rest]).all() and torch.equal(got[rest], ops.rotary(q[0], None, pos[:25], table)[0][rest])
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        ops.rotary(q.double(), None, pos[:25], table)


@gpu
def test_gpu_offsets_past_32_bits():
    """Rows beyond 2^31 elements of the kept projections, and of a rotated tensor."""
    M, K, F = 90000, 64, 12296
    x, wg, wu, wd, dy = ffn_tensors(M, K, F)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = Fn.gated_ffn(*leaves)
    dx, = torch.autograd.grad(y, leaves[0], dy)
    assert 2 * M * F > 1 << 31
    at = torch.tensor([0, 1, M // 2, M - 130, M - 1], device="cuda")
    want = ffn_oracle(x.detach()[at], *[t.detach() for t in leaves[1:]], "silu", dy[at])
    close(y.detach()[at], want["y"], "y")
    close(dx[at], want["dx"], "dx")
    n = 140000
    q = torch.zeros(n, 64, 256, device="cuda", dtype=torch.bfloat16)
    q[-3:] = torch.randn(3, 64, 256, device="cuda")
    table = ops.rotary_table(256, 16)
    pos = torch.arange(n, device="cuda") % 16
    got = ops.rotary(q, None, pos, table)[0]
    assert q.numel() > 1 << 31
    close(got[-3:], turned(q[-3:], pos[-3:, None], table, "half", [128]), "far rows")
    assert not got[:-3].any()


def _layer(x, ws, pos, table, pack, heads, kv, dim, rotary, attend, ffn, rnd):
    """A causal layer: projections, rotary positions, attention, gated feed-forward, both residuals."""
    qkv = rnd(x @ ws[0].t())
    q, k, v = (t.unflatten(1, (-1, dim)) for t in qkv.split([heads * dim, kv * dim, kv * dim], 1))
    q, k = rotary(q, k)
    x = x + rnd(attend(q, k, v).flatten(1) @ ws[1].t())
    return x + ffn(x, *ws[2:])


@gpu
def test_gpu_layer_forward_and_backward():
    """The three together, with gradients through all of them.  The bound is the error that a 64-bit run
    makes whose intermediate values and gradients are rounded to bf16 in the same places, three times."""
    heads, kv, dim, F = 8, 2, 64, 320
    pack = ops.SequencePack([1, 70, 200])
    n, C = pack.rows, heads * dim
    g = torch.Generator("cuda").manual_seed(5)

    def rand(*s, std):
        return (torch.randn(*s, generator=g, device="cuda") * std).bfloat16()
    ws = [rand((heads + 2 * kv) * dim, C, std=C ** -0.5), rand(C, C, std=C ** -0.5), rand(F, C, std=C ** -0.5),
          rand(F, C, std=C ** -0.5), rand(C, F, std=F ** -0.5)]
    x, do = rand(n, C, std=1.0), rand(n, C, std=1.0)
    pos = torch.cat([torch.arange(int(m), device="cuda") for m in pack.lengths])
    table = ops.rotary_table(dim, 256, scaling={"type": "yarn", "factor": 4.0, "original_len": 64})
    cpu = ops.SequencePack(pack.lengths, device="cpu")

    class Round(torch.autograd.Function):
        @staticmethod
        def forward(ctx, t):
            return t.bfloat16().double()

        @staticmethod
        def backward(ctx, t):
            return t.bfloat16().double()

    def run64(rnd):
        leaves = [t.double().requires_grad_(True) for t in [x] + ws]
        p = pos[:, None]

        def rot(q, k):
            return tuple(rnd(ref.rotary(t, p, table, "half", [dim // 2])) for t in (q, k))

        def att(q, k, v):
            return rnd(ref.packed_attention(q, k, v, cpu, True, dim ** -0.5)[0])

        def ffn(t, wg, wu, wd):
            t = rnd(t)
            return rnd(rnd(ref.gated_act(rnd(t @ wg.t()), "silu") * rnd(t @ wu.t())) @ wd.t())
        out = _layer(rnd(leaves[0]), leaves[1:], pos, table, pack, heads, kv, dim, rot, att, ffn, rnd)
        return [out.detach(), *torch.autograd.grad(out, leaves, do.double())]

    want, rounded = run64(lambda t: t), run64(Round.apply)
    leaves = [t.detach().requires_grad_(True) for t in [x] + ws]

    def rot(q, k):
        return Fn.rotary(q, k, pos, table)
    out = _layer(leaves[0], leaves[1:], pos, table, pack, heads, kv, dim, rot,
                 lambda q, k, v: Fn.packed_attention(q, k, v, pack), lambda t, *w: Fn.gated_ffn(t, *w), lambda t: t)
    got = [out.detach(), *torch.autograd.grad(out, leaves, do)]
    for i, (a, b, c) in enumerate(zip(got, want, rounded)):
        off, allowed = (a.double() - b).norm(), (c - b).norm()
        assert off <= 3 * allowed + 3 * HALF * b.norm(), (i, float(off / b.norm()), float(allowed / b.norm()))
    ops.check_device_errors()


@gpu
def test_gpu_layer_captured_with_its_backward():
    """Forward and backward of the operators captured into a graph and replayed on new inputs."""
    pack = ops.SequencePack([40, 90])
    table = ops.rotary_table(64, 128)
    pos = torch.cat([torch.arange(40, device="cuda"), torch.arange(90, device="cuda")])
    g = torch.Generator("cuda").manual_seed(5)
    ws = [(torch.randn(*s, generator=g, device="cuda") * 0.06).bfloat16() for s in ((384, 256), (384, 256), (256, 384))]
    x = torch.randn(130, 12, 64, generator=g, device="cuda").bfloat16()

    def step(x):
        x = x.detach().requires_grad_(True)
        q, k = Fn.rotary(x[:, :4], x[:, 4:8], pos, table)
        o = Fn.packed_attention(q, k, x[:, 8:], pack)
        y = Fn.gated_ffn(o.flatten(1), *ws, act="gelu_tanh")
        return y.detach(), torch.autograd.grad(y.float().square().sum(), x)[0]
    step(x)
    torch.cuda.synchronize()
    static = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for seed in (1, 2):
        new = torch.randn(x.shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").bfloat16()
        static.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step(new)))
