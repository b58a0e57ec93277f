"""Gated feed-forward block (kernels: ``ops/csrc/gated_ffn.cu``): both projections, the activation and
the product in one kernel, then the down projection.

``models.functional.gated_ffn`` is the block under autograd.  CPU tensors run the PyTorch reference
(:mod:`.reference`); CUDA tensors run the kernels in bf16.
"""
from __future__ import annotations

import torch

from . import reference as ref
from ._ext import ext

ACTS = {"silu": 0, "gelu_tanh": 1}


def check_gated(x, w_gate, w_up, act, w_down=None, what="gated_linear"):
    """Raise for operands that do not fit each other."""
    if act not in ACTS:
        raise ValueError(f"{what}: act one of {tuple(ACTS)}, got {act!r}")
    if x.dim() == 0 or w_gate.dim() != 2 or w_up.shape != w_gate.shape or x.shape[-1] != w_gate.shape[1]:
        raise ValueError(f"{what}: x {tuple(x.shape)} against weights {tuple(w_gate.shape)} and {tuple(w_up.shape)}")
    ws = [w_gate, w_up]
    if w_down is not None:
        if w_down.dim() != 2 or w_down.shape[1] != w_gate.shape[0]:
            raise ValueError(f"{what}: down weight {tuple(w_down.shape)} against {w_gate.shape[0]} hidden features")
        ws.append(w_down)
    for t in [x] + ws:
        if not t.dtype.is_floating_point or t.device != x.device:
            raise TypeError(f"{what}: floating-point tensors on one device")


def matrix(t: torch.Tensor, columns: int = 8) -> torch.Tensor:
    """``t`` [rows, n] in bf16 as the kernels read it: rows at multiples of 16 bytes (a copy where they
    are not), zero columns up to a multiple of ``columns``."""
    t = t.to(torch.bfloat16)
    n = t.shape[1]
    if n % columns:
        return torch.nn.functional.pad(t, (0, -n % columns))
    if t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= n and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def hidden_rows(w: torch.Tensor) -> torch.Tensor:
    """A weight [F, K] as :func:`matrix`, with zero rows up to a multiple of 8."""
    w = matrix(w)
    return torch.nn.functional.pad(w, (0, 0, 0, -w.shape[0] % 8)) if w.shape[0] % 8 else w


def gated_linear(x, w_gate, w_up, act: str = "silu"):
    """``act(x W_gate^T) * (x W_up^T)``: x [..., K], weights [F, K] -> [..., F] (bf16 on the GPU).

    ``act``: "silu" or "gelu_tanh".  Sizes that are no multiples of 8 are padded in copies.  It records
    no graph: ``models.functional.gated_ffn`` is the block under autograd."""
    check_gated(x, w_gate, w_up, act)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, w_gate, w_up)):
        raise RuntimeError("gated_linear has no gradient: use models.functional.gated_ffn, or torch.no_grad()")
    if not x.is_cuda:
        return ref.gated_linear(x, w_gate, w_up, act)
    F, K = w_gate.shape
    lead = x.shape[:-1]
    if K == 0:
        return x.new_zeros(*lead, F, dtype=torch.bfloat16)
    h = ext().gated_linear_fwd(matrix(x.reshape(lead.numel(), K)), hidden_rows(w_gate), hidden_rows(w_up), ACTS[act],
                               False)[0]
    return h[:, :F].reshape(*lead, F)


def gated_ffn(x, w_gate, w_up, w_down, act: str = "silu"):
    """``(act(x W_gate^T) * (x W_up^T)) W_down^T``: x [..., K], W_gate and W_up [F, K], W_down [C, F] ->
    [..., C] (bf16 on the GPU).  It records no graph (see :func:`gated_linear`)."""
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad
                                    or w_down.requires_grad):
        raise RuntimeError("gated_ffn has no gradient here: use models.functional.gated_ffn, or torch.no_grad()")
    if x.is_cuda and act in ACTS:
        out = ext().gated_ffn_fwd(x, w_gate, w_up, w_down, ACTS[act], False)
        if out:
            return out[0]
    check_gated(x, w_gate, w_up, act, w_down, "gated_ffn")
    if not x.is_cuda:
        return ref.gated_ffn(x, w_gate, w_up, w_down, act)
    C, F = w_down.shape
    K = x.shape[-1]
    lead = x.shape[:-1]
    if 0 in (K, F, C, lead.numel()):
        return x.new_zeros(*lead, C, dtype=torch.bfloat16)
    # copies that fit; the down weight's too before the gate kernel, which the product starts behind
    parts = [matrix(x.reshape(lead.numel(), K)), hidden_rows(w_gate), hidden_rows(w_up), hidden_rows(w_down)]
    return ext().gated_ffn_fwd(*parts, ACTS[act], False)[0][:, :C].reshape(*lead, C)
