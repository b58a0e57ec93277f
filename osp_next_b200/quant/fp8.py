"""Linear layers in block-scaled fp8 (format and kernels: :mod:`osp_next_b200.ops.fp8`).

Forward: y = x_q·W_qᵀ + b, x quantised in blocks 1 x 128 along its features, W in tiles
128 x 128.  Backward: dx = dy_q·W_q with the same codes of W read the other way, dW = dy_q'ᵀ·x_q'
with dy and x quantised in blocks of 128 tokens (straight-through estimator: the quantisers
have gradient 1).  All three products run on the block-scaled tensor-core kernel; the bias
gradient is summed from dy itself.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from .. import ops


def _grad_dtype(dt: torch.dtype) -> torch.dtype:
    return torch.bfloat16 if dt == torch.bfloat16 else torch.float32


def _out_dtype(x: torch.Tensor) -> torch.dtype:
    """bf16 on the GPU (the DiT's activations), the input's own type on the CPU."""
    return torch.float32 if not x.is_cuda and x.dtype == torch.float32 else torch.bfloat16


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x [..., K] as a matrix, also without columns (where -1 would be ambiguous)."""
    return x.reshape(x.shape[:-1].numel(), x.shape[-1])


class _FP8LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, act):
        x2 = _rows(x)
        need_x, need_w = ctx.needs_input_grad[:2]
        # one read of x gives the forward operand and the one of dW; the same for W and dx
        if x.is_cuda and x2.numel() and weight.numel():
            y, pre, *saved = ops.ext().fp8_linear_forward(x2, weight, bias, 1 if act else 0, act is not None, need_x,
                                                          need_w)
        else:
            xr, xc = ops.fp8_quantize(x2, layout="both")
            wr, wc = ops.fp8_quantize(weight, block_rows=ops.fp8.BLOCK, layout="both")
            y, pre = ops.fp8_matmul(xr, wr, bias, act, _out_dtype(x), aux=True)
            saved = [xc.data, xc.scale, wc.data, wc.scale]
        ctx.save_for_backward(pre if act else None, *saved)
        ctx.meta = (x.shape, x.dtype, weight.shape, weight.dtype, None if bias is None else bias.dtype)
        return y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        pre, *saved = ctx.saved_tensors
        xshape, xdt, wshape, wdt, bdt = ctx.meta
        g = _rows(gy)
        if pre is not None:
            g = _gelu_tanh_bwd(g, pre)
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx = dw = db = None
        if need_x or need_w:
            xdo, wdo = _grad_dtype(xdt), _grad_dtype(wdt)
            if g.is_cuda and g.numel() and xshape[-1]:
                dx, dw, db = ops.ext().fp8_linear_backward(g, *saved, need_b, xdo == torch.float32,
                                                           wdo == torch.float32)
            else:
                gr, gc, db = ops.fp8_quantize_with_sums(g)
                tokens, (N, K) = g.shape[0], wshape
                if need_x:
                    dx = ops.fp8_matmul(gr, ops.Fp8Tensor(saved[2], saved[3], K, N, ops.fp8.BLOCK), out_dtype=xdo)
                if need_w:
                    dw = ops.fp8_matmul(gc, ops.Fp8Tensor(saved[0], saved[1], K, tokens), out_dtype=wdo)
            dx = None if dx is None else dx.to(xdt).view(xshape)
            dw = None if dw is None else dw.to(wdt)
        db = (ops.bias_grad(g) if db is None else db).to(bdt) if need_b else None
        return dx, dw, db, None


def _gelu_tanh_bwd(g, pre):
    if g.is_cuda and g.numel() % 4 == 0:
        return ops.gelu_tanh_bwd(g, pre)
    with torch.enable_grad():
        p = pre.detach().float().requires_grad_(True)
        (d,) = torch.autograd.grad(F.gelu(p, approximate="tanh"), p, g.float())
    return d.to(torch.bfloat16)


def fp8_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
               act: Optional[str] = None) -> torch.Tensor:
    """``act(x·Wᵀ + b)`` (bf16; fp32 for fp32 CPU tensors) in block-scaled fp8 with an fp8
    backward pass.

    x [..., K] and weight [N, K] in bf16, fp16 or fp32, bias [N]; act None or ``"gelu_tanh"``.
    Both operands are quantised in the call (a weight that does not change is better kept as
    ``ops.fp8_quantize(weight, block_rows=128)`` for ``ops.fp8_matmul``).  First derivatives only:
    differentiating a gradient again raises."""
    if x.dim() == 0 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"fp8_linear: x {tuple(x.shape)} against weight {tuple(weight.shape)}")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError(f"fp8_linear: bias [{weight.shape[0]}], got {tuple(bias.shape)}")
    return _FP8LinearFn.apply(x, weight, bias, act)


class FP8Linear(nn.Linear):
    """``nn.Linear`` in block-scaled fp8 (forward and backward), with its parameters and state.
    The output is bf16 on the GPU, whatever the input's type (see :func:`fp8_linear`).

    Under autograd both operands are quantised every call.  For sampling, :meth:`freeze_weight`
    quantises the weight once and later no-grad calls use that copy until :meth:`thaw_weight`,
    ``train()`` or ``load_state_dict``: the layer never guesses whether a weight changed."""
    is_fp8 = True

    def __init__(self, in_features, out_features, bias=True, device=None, dtype=None):
        super().__init__(in_features, out_features, bias, device=device, dtype=dtype)
        self._frozen = None
        self._pack = None

    def freeze_weight(self):
        self._frozen = ops.fp8_quantize(self.weight.detach(), block_rows=ops.fp8.BLOCK)
        return self

    def thaw_weight(self):
        self._frozen = self._pack = None
        return self

    def refreeze_weight(self):
        """After a change of the weight: a frozen layer quantises it again, another stays as it is."""
        return self if self._frozen is None else self.freeze_weight()

    def train(self, mode: bool = True):
        if mode:
            self.thaw_weight()
        return super().train(mode)

    def _load_from_state_dict(self, *a, **k):
        self.thaw_weight()
        super()._load_from_state_dict(*a, **k)

    def _apply(self, fn, *a, **k):
        self.thaw_weight()
        return super()._apply(fn, *a, **k)

    def forward(self, x, act: Optional[str] = None):
        if torch.is_grad_enabled() and (x.requires_grad or self.weight.requires_grad
                                        or (self.bias is not None and self.bias.requires_grad)):
            return fp8_linear(x, self.weight, self.bias, act)
        w = self._frozen if self._frozen is not None else ops.fp8_quantize(self.weight, block_rows=ops.fp8.BLOCK)
        return ops.fp8_matmul(x, w, self.bias, act, _out_dtype(x))


def fp8_multi_linear(x: torch.Tensor, linears, act: Optional[str] = None) -> torch.Tensor:
    """[FP8Linear_1(x) | ... | FP8Linear_n(x)] of layers that read one input (q/k/v): x is
    quantised once and one product runs on the stacked weights.  With output sizes that are
    multiples of 128 (whole weight tiles) the values are those of the separate layers; others
    are run one by one."""
    if len(linears) == 1:
        return linears[0](x, act)
    has_bias = [m.bias is not None for m in linears]
    if any(m.out_features % ops.fp8.BLOCK for m in linears) or any(has_bias) != all(has_bias):
        return torch.cat([m(x, act) for m in linears], -1)
    bias = torch.cat([m.bias for m in linears]) if all(has_bias) else None
    params = [p for m in linears for p in (m.weight, m.bias) if p is not None]
    if torch.is_grad_enabled() and (x.requires_grad or any(p.requires_grad for p in params)):
        return fp8_linear(x, torch.cat([m.weight for m in linears]), bias, act)
    parts = [m._frozen for m in linears]
    if all(p is not None for p in parts):
        pack = linears[0]._pack        # (the frozen weights it was stacked from, the stack)
        if pack is None or len(pack[0]) != len(parts) or any(a is not b for a, b in zip(pack[0], parts)):
            w = ops.Fp8Tensor(torch.cat([p.data for p in parts]), torch.cat([p.scale for p in parts]),
                              sum(p.rows for p in parts), parts[0].cols, ops.fp8.BLOCK)
            pack = linears[0]._pack = (parts, w)
        w = pack[1]
    else:
        w = ops.fp8_quantize(torch.cat([m.weight.detach() for m in linears]), block_rows=ops.fp8.BLOCK)
    return ops.fp8_matmul(x, w, bias, act, _out_dtype(x))


def freeze_fp8_weights(module: nn.Module) -> nn.Module:
    """Quantise the weight of every :class:`FP8Linear` in ``module`` once (sampling)."""
    for m in module.modules():
        if isinstance(m, FP8Linear):
            m.freeze_weight()
    return module
