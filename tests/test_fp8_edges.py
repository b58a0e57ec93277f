"""Calls at the edges of the 8-bit operators: gradients that start at any address, empty sizes,
second derivatives, weights that change after they were packed or frozen, long lists of tensors."""
import copy
import glob
import os
import re

import pytest
import torch

from osp_next_b200 import ops
from osp_next_b200.models.lora import _PACKS, LoraLinear, LoraModel, fused_lora_operands, inject_lora
from osp_next_b200.models.osp_next import OSPNextModel
from osp_next_b200.ops import reference as ref
from osp_next_b200.parallel.ema import FSDPEMAModel
from osp_next_b200.parallel.optim import FusedAdamW
from osp_next_b200.quant import (FP8Linear, HIF8Linear, fp8_linear, fp8_multi_linear, freeze_fp8_weights,
                                 hif8_multi_linear)

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _randn(*shape, device="cpu", seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(device=device, dtype=dtype)


# ----------------------------------------------------------------------------- addresses

def test_vector_kernels_get_aligned_tensors(monkeypatch):
    """A contiguous view that starts at any element reaches the kernels that read vectors of 4 and 8
    bf16 as a copy from an aligned address, with the same values."""
    seen = []

    class Recorder:
        def gelu_tanh_bwd(self, dh, pre, dpre):
            seen.extend((t, 8) for t in (dh, pre, dpre))

        def bias_grad(self, g, part):
            seen.append((g, 16))
    monkeypatch.setattr(ops, "ext", Recorder)
    monkeypatch.setattr(ops, "_cuda", lambda *t: True)
    flat = _randn(200, dtype=torch.bfloat16)
    for start in range(9):
        a, b = flat[start:start + 48].view(6, 8), flat[100 + start:148 + start].view(6, 8)
        ops.gelu_tanh_bwd(a, b)
        ops.bias_grad(a)
        assert torch.equal(seen[-4][0], a) and torch.equal(seen[-3][0], b) and torch.equal(seen[-1][0], a)
    assert all(t.is_contiguous() and t.data_ptr() % align == 0 for t, align in seen)
    aligned = flat[:48].view(6, 8)
    ops.bias_grad(aligned)
    assert seen[-1][0].data_ptr() == aligned.data_ptr()          # no copy where none is needed


def _gelu64(x):
    return 0.5 * x * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (x + 0.044715 * x ** 3)))


@pytest.mark.parametrize("device", DEVICES)
def test_linear_gelu_with_gradients_from_any_address(device):
    """Two layers' outputs joined: the second's gradient is a contiguous view that starts 2 * 6 or
    2 * 3 bytes into the joined one, of a multiple of four elements."""
    for rows, n in (((1, 2), 6), ((1, 4), 3), ((3, 8), 5)):
        xs = [_randn(r, 64, device=device, seed=r, dtype=torch.bfloat16).requires_grad_() for r in rows]
        ws = [_randn(n, 64, device=device, seed=10 + i).div_(8).requires_grad_() for i in range(2)]
        y = torch.cat([fp8_linear(x, w, act="gelu_tanh") for x, w in zip(xs, ws)])
        dy = _randn(*y.shape, device=device, seed=3, dtype=torch.bfloat16)
        got = torch.autograd.grad(y, xs, dy)
        for x, w, d, g in zip(xs, ws, dy.split(rows), got):
            wr, wc = ops.fp8_quantize(w, block_rows=128, layout="both")
            pre = ops.fp8_matmul(x.detach(), wr, out_dtype=torch.float32).bfloat16().double().requires_grad_()
            (dpre,) = torch.autograd.grad(_gelu64(pre), pre, d.double())
            want = ops.fp8_quantize(dpre.bfloat16()).dequantize().double() @ wc.dequantize().double().t()
            # a last bit of the derivative in bf16 can move its code by a step, at most 2^-3 of the value;
            # a gradient read from another address is off by its own size
            assert ((g.double() - want).norm() / want.norm()).item() < 2.0 ** -3


@pytest.mark.parametrize("device", DEVICES)
def test_linear_bias_gradient_from_any_address(device):
    """The bias gradient of a layer without a weight gradient, from a gradient 2 bytes into its buffer."""
    x = _randn(5, 32, device=device, dtype=torch.bfloat16)
    w, b = _randn(16, 32, device=device), torch.zeros(16, device=device, requires_grad=True)
    head = torch.zeros(1, device=device, dtype=torch.bfloat16, requires_grad=True)
    y = torch.cat([head, fp8_linear(x, w, b).flatten()])
    dy = _randn(*y.shape, device=device, seed=3, dtype=torch.bfloat16)
    (got,) = torch.autograd.grad(y, [b], dy)
    want = dy[1:].view(5, 16).double().sum(0)
    assert bool(((got.double() - want).abs() <= 5 * 2.0 ** -24 * dy[1:].view(5, 16).double().abs().sum(0)).all())


@pytest.mark.gpu
def test_vector_kernels_refuse_other_addresses():
    flat = torch.zeros(64, device="cuda", dtype=torch.bfloat16)
    good, odd = flat[:32].view(4, 8), flat[1:33].view(4, 8)
    for args in ((odd, good, good), (good, odd, good), (good, good, odd)):
        with pytest.raises(RuntimeError):
            ops.ext().gelu_tanh_bwd(*args)
    with pytest.raises(RuntimeError):
        ops.ext().bias_grad(odd, torch.zeros(1, 8, device="cuda"))


# ----------------------------------------------------------------------------- loads and launches

def _csrc():
    return os.path.join(os.path.dirname(ops.__file__), "csrc")


def test_kernels_that_start_early_have_no_read_only_loads():
    """A kernel launched while the one before it runs must not read through the read-only path: its
    inputs may still be written, and such loads are not held behind the wait."""
    early = [f for f in glob.glob(os.path.join(_csrc(), "*.cu")) if "launch_kernel(" in open(f).read()]
    assert {os.path.basename(f) for f in early} >= {"fp8_gemm.cu", "fp8_quant.cu", "adamw_multi.cu"}
    shared = [os.path.join(_csrc(), h) for h in ("common.cuh", "fp8.cuh", "launch.h")]
    for f in early + shared:
        code = re.sub(r"//[^\n]*", "", open(f).read())
        assert not re.search(r"__ldg\b|ld\.global\.nc|__restrict", code), os.path.basename(f)


def test_cluster_barriers_are_reached_converged():
    """``barrier.cluster`` in its aligned form is undefined for a warp whose lanes are apart."""
    found = 0
    for f in glob.glob(os.path.join(_csrc(), "*.cu")) + glob.glob(os.path.join(_csrc(), "*.cuh")):
        code = re.sub(r"//[^\n]*", "", open(f).read())
        for m in re.finditer(r"asm volatile\(\s*\"barrier\.cluster\.arrive\.[a-z.]*aligned", code):
            assert code[:m.start()].rstrip().endswith("__syncwarp();"), os.path.basename(f)
            found += 1
    assert found


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 6, 13, 33, 64])
@pytest.mark.parametrize("N", [1, 100, 129, 1000])
def test_split_products_of_ragged_tiles(M, N):
    """Few rows over a K split on a cluster, where a warp's last lanes have no column of the result.
    Small integers: every sum is exact, whatever its order."""
    g = torch.Generator().manual_seed(M + N)
    x = torch.randint(-4, 5, (M, 4096), generator=g).to(device="cuda", dtype=torch.bfloat16)
    w = torch.randint(-4, 5, (N, 4096), generator=g).to(device="cuda", dtype=torch.float32)
    want = x.double() @ w.double().t()
    y = ops.fp8_matmul(x, ops.fp8_quantize(w, block_rows=128), out_dtype=torch.float32)
    assert torch.equal(y.double(), want)
    ops.check_device_errors()


# ----------------------------------------------------------------------------- optimizer

def _trained(device, dtype, steps, **kw):
    torch.manual_seed(0)
    params = [torch.nn.Parameter(torch.randn(n, device=device).to(dtype)) for n in (300, 7)]
    opt = FusedAdamW([{"params": params[:1]}, {"params": params[1:], "lr": 1e-3}], lr=1e-2, **kw)
    _steps(params, opt, 0, steps)
    return params, opt


def _steps(params, opt, first, n):
    for i in range(first, first + n):
        for j, p in enumerate(params):
            p.grad = 1e-3 * _randn(*p.shape, device=p.device, seed=100 * i + j, dtype=p.dtype)
        opt.step()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("save_bits", [8, 32])
@pytest.mark.parametrize("load_bits", [8, 32])
def test_checkpoints_keep_fp32_moments_of_16_bit_parameters(device, dtype, save_bits, load_bits):
    params, opt = _trained(device, dtype, 3, multi_tensor=True, state_bits=save_bits)
    sd = copy.deepcopy(opt.state_dict())
    saved = [dict(sd["state"][i]) for i in range(2)]
    assert all(st[k].dtype == torch.float32 for st in saved for k in ("exp_avg", "exp_avg_sq"))
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    again = FusedAdamW([{"params": twins[:1]}, {"params": twins[1:]}], multi_tensor=True, state_bits=load_bits)
    again.load_state_dict(copy.deepcopy(sd))
    for p, st in zip(twins, saved):
        got = again.state[p]
        assert got["step"] == st["step"] == 3
        if load_bits == 32:
            assert all(torch.equal(got[k], st[k]) and got[k].dtype == torch.float32 for k in ("exp_avg", "exp_avg_sq"))
        else:
            m, v = ops.adamw8_decode(*(got[k] for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")))
            # to the nearest of 3 mantissa bits (2^-4), or of the subnormal step: of the block's largest 2^-9 / 224
            # below for m, 2^-17 / 2^15 for v, which keeps a positive value positive
            for a, b, floor in ((m, st["exp_avg"], 2.0 ** -16), (v, st["exp_avg_sq"], 2.0 ** -30)):
                assert bool(((a - b).abs() <= 2.0 ** -4 * b.abs() + floor * b.abs().max()).all())
                # the same values again where they were 8-bit ones
                assert save_bits == 32 or torch.equal(a, b)
    _steps(params, opt, 3, 1)
    _steps(twins, again, 3, 1)
    if load_bits == save_bits == 32:                 # as if there had been no break
        assert all(torch.equal(p, q) for p, q in zip(params, twins))
    assert all(bool(q.isfinite().all()) for q in twins)


@pytest.mark.parametrize("device", DEVICES)
def test_per_tensor_moments_of_16_bit_parameters_load_into_lists(device):
    """The per-tensor form keeps moments in the parameter's type: they come back in fp32."""
    if device == "cuda":
        pytest.skip("the per-tensor kernel takes fp32 parameters")
    params, opt = _trained(device, torch.bfloat16, 2)
    assert opt.state[params[0]]["exp_avg"].dtype == torch.bfloat16
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    again = FusedAdamW([{"params": twins[:1]}, {"params": twins[1:]}], multi_tensor=True)
    again.load_state_dict(copy.deepcopy(opt.state_dict()))
    for p, q in zip(params, twins):
        assert again.state[q]["exp_avg"].dtype == torch.float32
        assert torch.equal(again.state[q]["exp_avg"], opt.state[p]["exp_avg"].float())
    _steps(twins, again, 2, 1)


# ----------------------------------------------------------------------------- weights that change

class _Projections(torch.nn.Module):
    def __init__(self, device):
        super().__init__()
        self.q, self.k = FP8Linear(64, 128, device=device), FP8Linear(64, 128, device=device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("frozen", [True, False])
def test_merging_an_adapter_into_fp8_layers(device, frozen):
    """The merged layers are those of the merged weights, frozen before or not, also stacked."""
    torch.manual_seed(0)
    lora = LoraModel(_Projections(device), r=4, lora_alpha=8.0, target_modules=["k"])
    net = lora.base_model.model
    x = _randn(3, 64, device=device, dtype=torch.bfloat16)
    if frozen:
        freeze_fp8_weights(net)
        with torch.no_grad():
            fp8_multi_linear(x, (net.q, net.k.base_layer))         # a stack of the weights as they are
    with torch.no_grad():
        net.k.lora_B["default"].weight.normal_()
        want_k = net.k.merged_weight()
        before = net.q(x)
        merged = lora.merge_and_unload()
        assert type(merged.k) is FP8Linear and torch.equal(merged.k.weight, want_k)
        assert (merged.k._frozen is not None) == frozen
        want = ops.fp8_matmul(x, ops.fp8_quantize(want_k, block_rows=128), merged.k.bias, out_dtype=merged.k(x).dtype)
        assert torch.equal(merged.k(x), want) and torch.equal(merged.q(x), before)
        assert torch.equal(fp8_multi_linear(x, (merged.q, merged.k)), torch.cat([before, want], -1))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kw", [{}, {"multi_tensor": True}, {"state_bits": 8}])
def test_an_optimizer_step_counts_as_a_change_of_the_weights(device, kw):
    """What is packed from weights looks at their version; torch's optimizers advance it, so do these."""
    params = [torch.nn.Parameter(torch.ones(n, device=device)) for n in (300, 5)]
    opt = FusedAdamW(params, lr=1e-2, **kw)
    for _ in range(2):
        before = [(p._version, p.detach().clone()) for p in params]
        for p in params:
            p.grad = torch.ones_like(p)
        opt.step()
        assert all(p._version > v and not torch.equal(p.detach(), old) for p, (v, old) in zip(params, before))
    ema = FSDPEMAModel(torch.nn.ParameterList(params))
    start = [p._version for p in params]
    ema.store(torch.nn.ParameterList(params))
    ema.ema_copy_to_model(torch.nn.ParameterList(params))
    swapped = [p._version for p in params]
    ema.restore(torch.nn.ParameterList(params))
    assert all(a < b < p._version for a, b, p in zip(start, swapped, params))


@pytest.mark.gpu
def test_list_step_counts_as_a_change_of_all_its_tensors():
    p, g = [torch.ones(300, device="cuda")], [torch.ones(300, device="cuda")]
    state = [[t] for t in ops.adamw8_state(p[0])]
    versions = [x[0]._version for x in (p, g, *state)]
    ops.adamw_multi_(p, g, *state, lr=1e-2, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, step=1)
    after = [x[0]._version for x in (p, g, *state)]
    assert after[1] == versions[1]
    assert all(a > b for i, (a, b) in enumerate(zip(after, versions)) if i != 1)
    with torch.inference_mode():                     # tensors without a version
        q = [torch.ones(300, device="cuda")]
        ops.adamw_multi_(q, [torch.ones_like(q[0])], [torch.zeros_like(q[0])], [torch.zeros_like(q[0])], lr=1e-2,
                         beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, step=1)
        assert bool((q[0] < 1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{}, {"multi_tensor": True}, {"state_bits": 8}])
@pytest.mark.parametrize("lora", [False, True])
def test_no_grad_outputs_follow_the_optimizer(kw, lora):
    """Packed q/k/v weights and folded adapters are those of the weights as they are: outputs equal
    those of a model built from a copy of the weights."""
    torch.manual_seed(0)

    def build():
        with torch.device("cuda"):
            m = OSPNextModel(dim=256, ffn_dim=512, num_heads=2, num_layers=2, text_len=16,
                             skiparse_model_type="dual_end", sparse_ratio=2, num_full_blocks=0)
        if lora:
            inject_lora(m, 4, 4.0, ["self_attn.q", "self_attn.k", "self_attn.v", "self_attn.o", "ffn.0", "ffn.2"])
        return m
    model = build()
    torch.nn.init.normal_(model.head.head.weight, std=0.02)
    params = [p for n, p in model.named_parameters() if not lora or "lora_" in n]
    opt = FusedAdamW(params, lr=3e-2, **kw)
    g = torch.Generator().manual_seed(1)
    x, t, ctx = (torch.randn(1, 16, 3, 16, 16, generator=g).cuda(), torch.tensor([500.0], device="cuda"),
                 torch.randn(1, 16, 4096, generator=g).cuda())
    with torch.no_grad():
        first = model(x, t, ctx)
    for step in range(2):
        for i, p in enumerate(params):
            p.grad = _randn(*p.shape, device="cuda", seed=10 * step + i, dtype=p.dtype)
        opt.step()
        twin = build()
        twin.load_state_dict(copy.deepcopy(model.state_dict()))
        with torch.no_grad():
            y = model(x, t, ctx)
            assert torch.equal(y, twin(x, t, ctx)) and not torch.equal(y, first)
    assert len(_PACKS.get(model.blocks[0].self_attn.q, {})) <= 2          # nothing of the old weights is kept


def test_packs_of_gathered_weights_follow_the_optimizer():
    """FSDP writes the weights that it gathers without advancing their version, often where they
    were before: an optimizer step and a swap of averaged weights count by themselves."""
    layer = LoraLinear(torch.nn.Linear(64, 32), r=4, alpha=8.0)
    shard = torch.nn.ParameterList([torch.nn.Parameter(torch.ones(4))])
    opt, ema, x = FusedAdamW(shard, lr=1e-2), FSDPEMAModel(shard), _randn(3, 64)

    def gathered():                                  # the same memory, the same version, other values
        w = layer.lora_B["default"].weight
        at = w.data_ptr(), w._version
        w.data.normal_()
        layer.base_layer.weight.data.normal_()
        assert (w.data_ptr(), w._version) == at

    def check():
        W, _, (_, B) = fused_lora_operands([layer], x)
        assert torch.equal(W, layer.base_layer.weight.detach().bfloat16())
        assert torch.equal(B, (2 * layer.lora_B["default"].weight.detach()).bfloat16())
        return W
    check()
    assert len(_PACKS[layer]) == 2 and copy.deepcopy(layer) not in _PACKS        # not in copies or checkpoints
    for write in (opt.step, lambda: ema.ema_copy_to_model(shard), lambda: ema.restore(shard)):
        shard[0].grad = torch.ones(4)
        write()
        gathered()
        W = check()
        assert check() is W                          # and kept as long as nothing changes


@pytest.mark.gpu
def test_hif8_copies_of_gathered_weights_follow_the_optimizer():
    p = torch.nn.Parameter(torch.ones(4, device="cuda"))
    opt = FusedAdamW([p])
    layer, x = HIF8Linear(64, 32, bias=False, device="cuda"), _randn(3, 64, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        for f in (layer, lambda v: hif8_multi_linear(v, (layer, layer))):
            before = f(x)
            p.grad = torch.ones_like(p)
            opt.step()
            layer.weight.data.neg_()
            assert torch.equal(f(x), -before) and bool(before.any())


# ----------------------------------------------------------------------------- second derivatives

@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("act", [None, "gelu_tanh"])
def test_second_derivatives_raise(device, act):
    """A penalty on a gradient would otherwise add nothing, without a word."""
    x = _randn(4, 64, device=device, dtype=torch.bfloat16).requires_grad_()
    w = _randn(8, 64, device=device, seed=1).requires_grad_()
    (dx,) = torch.autograd.grad(fp8_linear(x, w, act=act).float().square().sum(), x, create_graph=True)
    (plain,) = torch.autograd.grad(fp8_linear(x, w, act=act).float().square().sum(), x)
    assert torch.equal(dx.detach(), plain)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.float().square().sum().backward()


@pytest.mark.parametrize("device", DEVICES)
def test_matmul_refuses_to_drop_a_gradient(device):
    w = ops.fp8_quantize(_randn(8, 64, device=device), block_rows=128)
    x, b = _randn(4, 64, device=device, dtype=torch.bfloat16), torch.zeros(8, device=device)
    want = ops.fp8_matmul(x, w, b)
    for args in ((x.clone().requires_grad_(), w, b), (x, w, b.clone().requires_grad_()),
                 (ops.fp8_quantize(x), w, b.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="no gradient"):
            ops.fp8_matmul(*args)
        with torch.no_grad():
            assert torch.equal(ops.fp8_matmul(*args), want)
        with torch.inference_mode():
            assert torch.equal(ops.fp8_matmul(*args), want)


# ----------------------------------------------------------------------------- empty sizes

@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lead", [(), (3,), (2, 3), (0,), (2, 0)])
@pytest.mark.parametrize("K,N", [(0, 5), (64, 0), (0, 0), (64, 8)])
@pytest.mark.parametrize("act", [None, "gelu_tanh"])
def test_linear_without_rows_columns_or_outputs(device, lead, K, N, act):
    """As nn.Linear: an empty sum is the bias, gradients of what is empty are zero."""
    x = _randn(*lead, K, device=device, dtype=torch.bfloat16).requires_grad_()
    w, b = _randn(N, K, device=device, seed=1).requires_grad_(), _randn(N, device=device, seed=2).requires_grad_()
    y = fp8_linear(x, w, b, act)
    assert y.shape == lead + (N,)
    if K == 0:
        want = _gelu64(b.detach().double()) if act else b.detach().double()
        assert bool(((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20).all())
    dx, dw, db = torch.autograd.grad(y.float().square().sum(), (x, w, b))
    assert all(g.shape == t.shape and g.dtype == t.dtype for g, t in ((dx, x), (dw, w), (db, b)))
    assert all(bool(g.isfinite().all()) for g in (dx, dw, db))
    if x.numel() == 0 or N == 0:
        assert not bool(dw.any()) and not bool(dx.any())
    if 0 in lead:
        assert not bool(db.any())
    with torch.no_grad():
        layer = FP8Linear(K, N, device=device) if K and N else None
        if layer is not None:
            assert layer(x).shape == y.shape


# ----------------------------------------------------------------------------- AdamW over long lists

HYPER = dict(lr=1.0, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01)


def _param_bound(p, g, m, v, step, grad_scale):
    """64-bit parameters after a step and how far fp32 may be off.  Roundings to 2^-24: three of p; of
    the update three of each term of m, two of v, the constants, two products and a sum below the
    line, a square root and a division approximate to 2^-22 each: below 2^-20 of it, with m taken as
    the sum of its terms' magnitudes."""
    p, g, m, v = (t.double() for t in (p, g * grad_scale, m, v))
    b1, b2 = HYPER["beta1"], HYPER["beta2"]
    rate, bc2 = HYPER["lr"] / (1 - b1 ** step), (1 - b2 ** step) ** 0.5
    den = (b2 * v + (1 - b2) * g * g).sqrt() / bc2 + HYPER["eps"]
    want = p * (1 - HYPER["lr"] * HYPER["weight_decay"]) - rate * (b1 * m + (1 - b1) * g) / den
    return want, 2.0 ** -22 * (p.abs() + want.abs()) + 2.0 ** -20 * rate * (b1 * m.abs() + (1 - b1) * g.abs()) / den


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("step", [1, 2, 500])
def test_adamw_parameters_to_fp32_accuracy(device, bits, step):
    """Also where 1 - b2^t is small, which formed in fp32 would be off by 2^-14."""
    n = 5000
    p, g = _randn(n, device=device), 1e-3 * _randn(n, device=device, seed=1)
    m, v = 1e-3 * _randn(n, device=device, seed=2), (1e-3 * _randn(n, device=device, seed=3)) ** 2
    if bits == 8:
        half = torch.full((n,), 0x80008000, dtype=torch.int64, device=device)
        state = list(ref.adamw8_encode(m, v, half))
        m, v = ops.adamw8_decode(*state)
    else:
        m, v = (m, v) if step > 1 else (torch.zeros_like(m), torch.zeros_like(v))
        state = [m.clone(), v.clone()]
    want, bound = _param_bound(p, g, m, v, step, 0.5)
    ops.adamw_multi_([p], [g], *([t] for t in state), step=step, grad_scale=0.5, seed=3, **HYPER)
    assert bool(((p.double() - want).abs() <= bound).all()), float(((p.double() - want).abs() / bound).max())


LONG_LISTS = {   # tensors -> chunks of 4096 elements: more than 512 a launch, so that a step of the table has several
    "few": [3_000_001, 1, 4096, 4097, 129] + [700 + 97 * i for i in range(20)] + [1_234_567, 5, 8192],
    "small at the end": [2_500_000] + [1 + 61 * i for i in range(50)],
    "many": [1 + 641 * (i % 29) for i in range(300)] + [2_000_003] + [4095 + i % 3 for i in range(170)] + [1_000_000],
    "two launches": [9000 + 13 * i for i in range(700)],
}


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", list(LONG_LISTS))
@pytest.mark.parametrize("pdtype,gdtype,bits", [(torch.float32, torch.float32, 8), (torch.bfloat16, torch.bfloat16, 8),
                                                (torch.bfloat16, torch.float32, 8), (torch.float32, torch.bfloat16, 32)])
def test_adamw_long_lists(sizes, pdtype, gdtype, bits):
    """Every tensor by its own state, key and length: codes and scales as the CPU form has them."""
    sizes = LONG_LISTS[sizes]
    assert sum(-(-n // 4096) for n in sizes[:480]) > 512
    p = [_randn(n, seed=i, dtype=pdtype) for i, n in enumerate(sizes)]
    g = [(1e-3 * (1 + i % 7) * _randn(n, seed=5000 + i)).to(gdtype) for i, n in enumerate(sizes)]
    if bits == 8:
        state = [list(x) for x in zip(*(ops.adamw8_state(t) for t in p))]
    else:
        state = [[torch.zeros(n) for n in sizes] for _ in range(2)]
    host = [p, g] + state
    dev = [[t.cuda() for t in x] for x in host]
    hyper = dict(HYPER, lr=1e-2)
    for step in (1, 2):
        for lists in (host, dev):
            ops.adamw_multi_(*lists, step=step, grad_scale=0.7, seed=41 * step, **hyper)
        for a, b in zip(host[2:], dev[2:]):
            if bits == 8:
                assert all(torch.equal(x.view(torch.uint8), y.cpu().view(torch.uint8)) for x, y in zip(a, b))
            else:                                    # two products and a sum, which the kernel may contract
                assert all(bool(((x - y.cpu()).abs() <= 2.0 ** -20 * x.abs() + 1e-9).all()) for x, y in zip(a, b))
    # p moved by less than 0.1 a step: the update to 2^-20, its own roundings, in bf16 one place a step
    rel = 2.0 ** -6 if pdtype == torch.bfloat16 else 2.0 ** -22
    for x, y in zip(host[0], dev[0]):
        x, y = x.double(), y.cpu().double()
        assert bool(((x - y).abs() <= rel * x.abs() + 2.0 ** -20).all())


# ----------------------------------------------------------------------------- narrow products

@pytest.mark.gpu
@pytest.mark.parametrize("M", [65, 129, 5000])
@pytest.mark.parametrize("N", [1, 40, 63, 64])
def test_narrow_products(M, N):
    """One tile of 64 columns, in both result types, over one run of blocks and over several.  Small
    integers: every sum is exact, and so is its rounding."""
    for K in (128, 1000, 4096):
        g = torch.Generator().manual_seed(M + N + K)
        x = torch.randint(-4, 5, (M, K), generator=g).to(device="cuda", dtype=torch.bfloat16)
        w = torch.randint(-4, 5, (N, K), generator=g).to(device="cuda", dtype=torch.float32)
        want = x.double() @ w.double().t()
        wq = ops.fp8_quantize(w, block_rows=128)
        for dt in (torch.float32, torch.bfloat16):
            assert torch.equal(ops.fp8_matmul(x, wq, out_dtype=dt), want.to(dt))
    ops.check_device_errors()


# ----------------------------------------------------------------------------- sampling in fp8

def _small_model(device, quant):
    torch.manual_seed(0)
    with torch.device(device):
        m = OSPNextModel(dim=256, ffn_dim=512, num_heads=2, num_layers=2, text_len=16,
                         skiparse_model_type="dual_end", sparse_ratio=2, num_full_blocks=0, quant=quant)
    torch.nn.init.normal_(m.head.head.weight, std=0.02)
    return m


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("quant", [None, "fp8"])
def test_a_model_first_run_in_inference_mode(device, quant):
    """Its tables are made there and kept: later steps, gradients among them, find ordinary tensors."""
    model = _small_model(device, quant)
    g = torch.Generator().manual_seed(1)
    # a grid that no other test runs, so that the shared tables are made here
    x, t, ctx = (torch.randn(1, 16, 3, 12, 20, generator=g).to(device), torch.tensor([500.0], device=device),
                 torch.randn(1, 16, 4096, generator=g).to(device))
    with torch.inference_mode():
        y = model(x, t, ctx)
        assert torch.equal(model(x, t, ctx), y)
    with torch.no_grad():
        assert torch.equal(model(x, t, ctx), y.clone())
    model(x, t, ctx).float().square().mean().backward()
    assert all(bool(p.grad.isfinite().all()) for p in model.parameters() if p.grad is not None)


@pytest.mark.parametrize("device", DEVICES)
def test_rope_table_of_an_inference_tensor(device):
    with torch.inference_mode():
        f = torch.arange(12.0, device=device).view(3, 4)
        a = ops.rope_cos_sin(f, device).clone()
        f.add_(1)
        b = ops.rope_cos_sin(f, device)
        assert torch.equal(b[..., 0], f.double().cos().float()) and not torch.equal(a, b)



class _Text:
    """Stands in for tokenizer and text encoder: a sequence of 16 made from the prompt's length."""
    def __init__(self, device):
        self.device, self.tokenizer = device, self._tokenize
        self.dtype = torch.float32 if torch.device(device).type == "cpu" else torch.bfloat16

    def _tokenize(self, texts, **kw):
        return torch.tensor([[len(t)] for t in texts]), torch.ones(len(texts), 1)

    def __call__(self, ids, mask):
        return torch.cat([_randn(1, 16, 4096, device=self.device, seed=int(i), dtype=self.dtype) for i in ids])


class _Frames:
    """Stands in for the VAE: the first three channels of the latents."""
    dtype = torch.float32

    def decode(self, z):
        return torch.tanh(z.float())[:, :3]


@pytest.mark.parametrize("device", DEVICES)
def test_inference_script_in_fp8(device, tmp_path, monkeypatch):
    """``model_config.quant: fp8``: the weights are quantised once, every step runs on the frozen
    copies, and the videos are those of layers that quantise their weight in each call."""
    import torch.distributed as dist
    from osp_next_b200.data.utils import video_io
    from osp_next_b200.engine import builders
    monkeypatch.syspath_prepend(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "infer"))
    import infer_osp
    for k, v in dict(MASTER_ADDR="127.0.0.1", MASTER_PORT="29637", RANK="0", WORLD_SIZE="1", LOCAL_RANK="0").items():
        monkeypatch.setenv(k, v)
    (tmp_path / "prompts.txt").write_text("a dog runs\nthe sea at night, seen from above\n")
    cfg = {"model_name": "osp_next", "seed": 3, "prompt_txt": str(tmp_path / "prompts.txt"), "num_frames": 5,
           "height": 64, "width": 64, "output_dir": str(tmp_path / "out"), "timeout_s": 120,
           "weight_dtype": "fp32" if device == "cpu" else "bf16",
           "model_config": dict(dim=256, ffn_dim=512, num_heads=2, num_layers=2, text_len=16, quant="fp8",
                                skiparse_model_type="dual_end", sparse_ratio=2, num_full_blocks=0),
           "scheduler_config": {"scheduler_name": "flow_matching", "num_inference_steps": 2, "guidance_scale": 5.0}}
    built, videos, build_model = [], [], builders.build_model

    def build(*a, **k):
        built.append(build_model(*a, **k))
        torch.manual_seed(5)
        torch.nn.init.normal_(built[-1].head.head.weight, std=0.02)      # the head starts at zero
        return built[-1]
    monkeypatch.setattr(builders, "build_model", build)
    monkeypatch.setattr(builders, "build_vae", lambda *a: _Frames())
    monkeypatch.setattr(builders, "build_text_encoder", lambda c, dev: _Text(dev))
    monkeypatch.setattr(video_io, "save_video", lambda v, path, fps: videos.append((os.path.basename(path), v)))

    def run():
        videos.clear()
        infer_osp.main(copy.deepcopy(cfg))
        if dist.is_initialized():
            dist.destroy_process_group()
        assert [n for n, _ in videos] == ["00000.mp4", "00001.mp4", "grid.mp4"]
        return [v for n, v in videos if n != "grid.mp4"]
    frozen = run()
    layers = [m for m in built[-1].modules() if isinstance(m, FP8Linear)]
    assert len(layers) == 20 and all(m._frozen is not None for m in layers)
    assert all(v.shape == (2, 8, 8, 3) and v.dtype == torch.uint8 for v in frozen)
    assert not torch.equal(frozen[0], frozen[1])
    monkeypatch.setattr(FP8Linear, "freeze_weight", lambda self: self)
    again = run()
    assert all(torch.equal(a, b) for a, b in zip(frozen, again))
    cfg["model_config"].pop("quant")
    plain = run()
    assert not all(torch.equal(a, b) for a, b in zip(frozen, plain))
    # uint8 frames of tanh values: the quantisation moves them by a few of 255 in the mean
    assert max((a.float() - b.float()).abs().mean().item() for a, b in zip(frozen, plain)) < 25


# ----------------------------------------------------------------------------- long sums in fp32

@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(1, 512), (40, 300), (100, 64), (130, 300), (5000, 512)])
def test_a_large_first_term_costs_no_more_than_an_fp32_sum(M, N):
    """Sums near 1.5 from their first product on, with small ones of both signs behind it: each step
    of 32 products forms its sum in quarters of a place of 2^-23 and cuts it toward zero, by 3/8 of a
    place in the mean, for as long as a run goes on (12 blocks, 48 steps: 18 places), and the sum of the
    runs is rounded (1 more)."""
    K = 2048
    g = torch.Generator().manual_seed(M + N)

    def small(rows):                                 # +- 2^-11 (8 .. 15) / 8: products far below 2^-23
        v = torch.randint(8, 16, (rows, K), generator=g) / 8 * 2.0 ** -11
        return v * (torch.randint(0, 2, (rows, K), generator=g) * 2 - 1)
    x, w = small(M), small(N)
    x[:, 0], w[:, 0] = 1.5, 1.0
    a, b = ops.fp8_quantize(x.cuda()), ops.fp8_quantize(w.cuda())
    want = a.dequantize().double() @ b.dequantize().double().t()
    assert torch.equal(a.dequantize().cpu(), x) and torch.equal(b.dequantize().cpu(), w)
    assert 1 < want.min().item() and want.max().item() < 2
    places = (want - ops.fp8_matmul(a, b, out_dtype=torch.float32).double()) * 2 ** 23
    assert abs(places.mean().item()) <= 19
