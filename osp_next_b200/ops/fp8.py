"""Block-128 fp8: quantisation and block-scaled products, and AdamW over lists of tensors.

Format (kernels: ``ops/csrc/fp8.cuh``): a matrix [R, K] is e4m3 codes [R, Kp] (Kp = K rounded
up to 128, zero-padded) with one power-of-two scale for each block of 128 along K, for one row
(``block_rows=1``) or for 128 rows together (``block_rows=128``, weights).  The scale is the
smallest 2^k, k >= -126, with max|x| / 2^k <= 448, kept as the byte k + 127.  Non-finite
elements do not count for the maximum and are stored as NaN.  The bytes lie in chunks of
128 rows x 4 blocks, ``scale[r // 128, kb // 4, r % 32, r % 128 // 32, kb % 4]``, as the tensor
core reads them; bytes of rows and blocks outside the matrix are zero.

CPU tensors run the PyTorch reference (:mod:`.reference`); CUDA tensors run the kernels.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import reference as ref
from ._ext import ext

BLOCK = 128
_IN_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_LAYOUTS = ("rows", "cols", "both")


class Fp8Tensor:
    """A quantised matrix: ``data`` e4m3 [rows, Kp], ``scale`` uint8 [ceil(rows / 128),
    ceil(cols / 512), 32, 4, 4], its logical sizes and the rows that share a scale."""

    __slots__ = ("data", "scale", "rows", "cols", "block_rows")

    def __init__(self, data: torch.Tensor, scale: torch.Tensor, rows: int, cols: int, block_rows: int = 1):
        self.data, self.scale = data, scale
        self.rows, self.cols, self.block_rows = rows, cols, block_rows

    @property
    def shape(self):
        return torch.Size((self.rows, self.cols))

    @property
    def device(self):
        return self.data.device

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        """The values it stands for, [rows, cols] (PyTorch ops; for inspection and tests)."""
        return ref.fp8_dequantize(self.data, self.scale, self.rows, self.cols).to(dtype)

    def __repr__(self):
        return f"Fp8Tensor([{self.rows}, {self.cols}], block {self.block_rows}x{BLOCK}, {self.data.device})"


def fp8_quantize(x: torch.Tensor, block_rows: int = 1, layout: str = "rows"):
    """Block-128 fp8 of a matrix x [R, K] (bf16, fp16 or fp32; any strides).

    ``layout="rows"``: blocks along K, of x; ``"cols"``: blocks along R, of the transpose
    (an :class:`Fp8Tensor` [K, R], what a weight-gradient product reads); ``"both"``: the pair
    (rows, cols) from one read of x.  ``block_rows=128`` gives each 128 x 128 tile one scale,
    so that both orientations hold the same values."""
    if x.dim() != 2:
        raise ValueError(f"fp8_quantize: a matrix is needed, got {tuple(x.shape)}")
    if x.dtype not in _IN_TYPES:
        raise TypeError(f"fp8_quantize: bf16, fp16 or fp32, got {x.dtype}")
    if block_rows not in (1, BLOCK):
        raise ValueError(f"fp8_quantize: block_rows 1 or {BLOCK}, got {block_rows}")
    if layout not in _LAYOUTS:
        raise ValueError(f"fp8_quantize: layout one of {_LAYOUTS}, got {layout!r}")
    R, K = x.shape
    if not x.is_cuda:
        sides = [Fp8Tensor(*ref.fp8_quantize(x if s == "rows" else x.t(), block_rows),
                           *((R, K) if s == "rows" else (K, R)), block_rows)
                 for s in ("rows", "cols") if layout in (s, "both")]
        return tuple(sides) if layout == "both" else sides[0]
    q, qs, t, ts, _ = ext().fp8_quantize(x, block_rows != 1, layout != "cols", layout != "rows", False)
    rows = None if q is None else Fp8Tensor(q, qs, R, K, block_rows)
    cols = None if t is None else Fp8Tensor(t, ts, K, R, block_rows)
    return (rows, cols) if layout == "both" else (cols if rows is None else rows)


def fp8_quantize_with_sums(g: torch.Tensor):
    """``fp8_quantize(g, layout="both")`` and the fp32 column sums of g [R, K] (an output gradient
    and its bias gradient) from one read of g: (rows, cols, sums [K])."""
    if not g.is_cuda:
        return (*fp8_quantize(g, layout="both"), g.float().sum(0))
    if g.dim() != 2 or g.dtype not in _IN_TYPES:
        raise TypeError(f"fp8_quantize_with_sums: a matrix in bf16, fp16 or fp32, got {g.dtype} {tuple(g.shape)}")
    R, K = g.shape
    q, qs, t, ts, part = ext().fp8_quantize(g, False, True, True, True)
    return Fp8Tensor(q, qs, R, K), Fp8Tensor(t, ts, K, R), part.sum(0)


def fp8_matmul(a, b: Fp8Tensor, bias: Optional[torch.Tensor] = None, act: Optional[str] = None,
               out_dtype=torch.bfloat16, aux: bool = False):
    """``act(a·bᵀ + bias)`` with block-scaled fp8 operands and fp32 accumulation.

    ``a``: an :class:`Fp8Tensor` [M, K], or a matrix / batch [..., K] in bf16, fp16 or fp32 that
    is quantised here with blocks 1 x 128.  ``b``: an Fp8Tensor [N, K] (a weight, or either side
    of a gradient product).  ``act``: None or ``"gelu_tanh"``.  ``out_dtype``: bf16 or fp32.
    ``aux=True`` also returns the value before ``act`` in bf16.

    It records no graph: an ``a`` or ``bias`` that requires a gradient is refused unless gradients
    are off (``quant.fp8_linear`` is the product under autograd)."""
    if not isinstance(b, Fp8Tensor):
        raise TypeError("fp8_matmul: b has to be an Fp8Tensor")
    if act not in (None, "gelu_tanh"):
        raise ValueError(f"fp8_matmul: act None or 'gelu_tanh', got {act!r}")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"fp8_matmul: out_dtype bf16 or fp32, got {out_dtype}")
    quantized = isinstance(a, Fp8Tensor)
    if torch.is_grad_enabled() and ((not quantized and a.requires_grad) or (bias is not None and bias.requires_grad)):
        raise RuntimeError("fp8_matmul has no gradient: use quant.fp8_linear, or torch.no_grad()")
    shape = a.shape
    if len(shape) == 0 or shape[-1] != b.cols:
        raise ValueError(f"fp8_matmul: a {tuple(shape)} against K = {b.cols}")
    if bias is not None and bias.shape != (b.rows,):
        raise ValueError(f"fp8_matmul: bias [{b.rows}], got {tuple(bias.shape)}")
    if not b.data.is_cuda or b.cols == 0:      # the reference; with K = 0 an empty sum: act(bias)
        if not quantized:
            a = fp8_quantize(a.reshape(a.shape[:-1].numel(), b.cols))
        out, pre = ref.fp8_matmul(a, b, bias, act, out_dtype)
    else:
        args = (b.data, b.scale, bias, 1 if act else 0, out_dtype == torch.float32, aux)
        if quantized:
            out, *pre = ext().fp8_gemm(a.data, a.scale, *args)
        elif a.dtype in _IN_TYPES:
            out, *pre = ext().fp8_linear(a, *args)
        else:
            raise TypeError(f"fp8_matmul: bf16, fp16 or fp32, got {a.dtype}")
        pre = pre[0] if aux else None
    if len(shape) != 2:
        out = out.view(*shape[:-1], b.rows)
        pre = None if pre is None else pre.view(*shape[:-1], b.rows)
    return (out, pre) if aux else out


def adamw_multi_(params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales=None, exp_avg_sq_scales=None, *, lr, beta1, beta2,
                 eps, weight_decay, step, grad_scale=1.0, seed=0):
    """In-place AdamW step on lists of contiguous tensors, all in one kernel per 480 tensors.

    Parameters and gradients: fp32 or bf16, each of one type through its list.  Moments: fp32,
    or in 8 bits when the scale lists are given: ``exp_avgs`` e4m3, ``exp_avg_sqs`` uint8 (top
    byte of a half without its sign), one uint8 power-of-two scale per 128 elements
    (:func:`adamw8_state` makes them).  8-bit moments are rounded stochastically with bits mixed
    from ``seed``, the tensor's place in the list and the element's index: pass another seed
    each step.  ``step`` counts from 1; ``grad_scale`` multiplies the gradients."""
    state8 = exp_avg_scales is not None or exp_avg_sq_scales is not None
    if state8 and (exp_avg_scales is None or exp_avg_sq_scales is None):
        raise ValueError("adamw_multi_: scales of both moments or of none")
    lists = [params, grads, exp_avgs, exp_avg_sqs] + ([exp_avg_scales, exp_avg_sq_scales] if state8 else [])
    if len({len(x) for x in lists}) != 1:
        raise ValueError("adamw_multi_: lists of different lengths")
    if step < 1:
        raise ValueError("adamw_multi_: step counts from 1")
    if not params:
        return
    if not params[0].is_cuda:
        return ref.adamw_multi_(params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, lr, beta1,
                                beta2, eps, weight_decay, step, grad_scale, seed)
    lists = [x if type(x) is list else list(x) for x in lists] + ([] if state8 else [[], []])
    ext().adamw_multi(*lists, float(lr), float(beta1), float(beta2), float(eps), float(weight_decay),
                      int(step), float(grad_scale), int(seed))


def adamw8_state(p: torch.Tensor):
    """Zero 8-bit moments of a tensor: (exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale)."""
    nb = -(-p.numel() // BLOCK)
    return (torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn),
            torch.zeros(p.shape, dtype=torch.uint8, device=p.device),
            torch.ones(nb, dtype=torch.uint8, device=p.device), torch.ones(nb, dtype=torch.uint8, device=p.device))


def adamw8_decode(exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale):
    """The fp32 moments that an 8-bit state stands for (PyTorch ops; for inspection, tests and
    conversion to fp32 moments)."""
    return ref.adamw8_decode(exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale)
