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


def _empty(rows: int, cols: int, device):
    kp = -(-cols // BLOCK) * BLOCK
    return (torch.empty(rows, kp, dtype=torch.float8_e4m3fn, device=device),
            torch.empty(-(-rows // 128), -(-cols // 512), 32, 4, 4, dtype=torch.uint8, device=device))


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
    x = x.detach()
    rows = cols = None
    if layout != "cols":
        rows = Fp8Tensor(*_empty(R, K, x.device), R, K, block_rows)
    if layout != "rows":
        cols = Fp8Tensor(*_empty(K, R, x.device), K, R, block_rows)
    a, b = rows, cols
    if K > 1 and x.stride(1) != 1:
        if R > 1 and x.stride(0) != 1:
            x = x.contiguous()
        else:                       # a transposed view: its rows are the columns of what is stored
            x, a, b = x.t(), cols, rows
    ext().fp8_quantize(x, None if a is None else a.data, None if a is None else a.scale,
                       None if b is None else b.data, None if b is None else b.scale, block_rows != 1)
    return (rows, cols) if layout == "both" else (rows if cols is None else cols)


def fp8_matmul(a, b: Fp8Tensor, bias: Optional[torch.Tensor] = None, act: Optional[str] = None,
               out_dtype=torch.bfloat16, aux: bool = False):
    """``act(a·bᵀ + bias)`` with block-scaled fp8 operands and fp32 accumulation.

    ``a``: an :class:`Fp8Tensor` [M, K], or a matrix / batch [..., K] in bf16, fp16 or fp32 that
    is quantised here with blocks 1 x 128.  ``b``: an Fp8Tensor [N, K] (a weight, or either side
    of a gradient product).  ``act``: None or ``"gelu_tanh"``.  ``out_dtype``: bf16 or fp32.
    ``aux=True`` also returns the value before ``act`` in bf16."""
    if not isinstance(b, Fp8Tensor):
        raise TypeError("fp8_matmul: b has to be an Fp8Tensor")
    if act not in (None, "gelu_tanh"):
        raise ValueError(f"fp8_matmul: act None or 'gelu_tanh', got {act!r}")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"fp8_matmul: out_dtype bf16 or fp32, got {out_dtype}")
    lead = None
    if not isinstance(a, Fp8Tensor):
        if a.dim() == 0 or a.shape[-1] != b.cols:
            raise ValueError(f"fp8_matmul: a {tuple(a.shape)} against K = {b.cols}")
        lead = a.shape[:-1]
        a = fp8_quantize(a if a.dim() == 2 else a.reshape(-1, a.shape[-1]))
    if a.cols != b.cols:
        raise ValueError(f"fp8_matmul: K differs: {a.cols} and {b.cols}")
    M, N = a.rows, b.rows
    if bias is not None and tuple(bias.shape) != (N,):
        raise ValueError(f"fp8_matmul: bias [{N}], got {tuple(bias.shape)}")
    if not a.data.is_cuda or a.cols == 0:      # an empty sum: act(bias)
        out, pre = ref.fp8_matmul(a, b, bias, act, out_dtype)
    else:
        out = torch.empty(M, N, dtype=out_dtype, device=a.data.device)
        pre = torch.empty(M, N, dtype=torch.bfloat16, device=a.data.device) if aux else None
        bb = None if bias is None else bias.detach().float().contiguous()
        ext().fp8_gemm(a.data, a.scale, b.data, b.scale, bb, out, 1 if act else 0, pre)
    if lead is not None and len(lead) != 1:
        out = out.view(*lead, N)
        pre = None if pre is None else pre.view(*lead, N)
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
    ext().adamw_multi(params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales if state8 else [],
                      exp_avg_sq_scales if state8 else [], float(lr), float(beta1), float(beta2), float(eps),
                      float(weight_decay), int(step), float(grad_scale), int(seed))


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
