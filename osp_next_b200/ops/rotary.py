"""Rotary positions of q and k (kernel: ``ops/csrc/rotary.cu``).

Where :func:`osp_next_b200.ops.qk_norm_rope` rotates whole heads of a fused qkv behind a norm, this
is the rotation by itself, in the forms that language models use.  ``models.functional.rotary`` is the
form under autograd.  CPU tensors run the PyTorch reference (:mod:`.reference`).
"""
from __future__ import annotations

import math
from typing import Optional, Sequence

import torch

from . import reference as ref
from ._ext import ext

LAYOUTS = ("half", "interleaved")
_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def rotary_angles(dim: int, theta: float = 10000.0, scaling: Optional[dict] = None):
    """(angle of each of dim / 2 pairs per position in 64 bits, factor on cosine and sine).

    ``scaling`` for contexts longer than those of training:

    * ``{"type": "linear", "factor": s}``: positions divided by s
    * ``{"type": "ntk", "factor": s}``: theta s^(dim / (dim - 2)), so that the slowest pair turns s
      times slower and the fastest as before
    * ``{"type": "yarn", "factor": s, "original_len": L, "beta_fast": 32, "beta_slow": 1,
      "attention_factor": 0.1 ln s + 1}``: pairs of more than beta_fast turns within L are kept, those
      of less than beta_slow slowed by s, linear in the pair's number between; the factor multiplies
      cosines and sines"""
    if dim < 2 or dim % 2:
        raise ValueError(f"rotary: an even number of elements, got {dim}")
    if not theta > 0:
        raise ValueError(f"rotary: theta above 0, got {theta}")
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    if scaling is None:
        return theta ** (-i / dim), 1.0
    kind, rest = scaling.get("type"), {k: v for k, v in scaling.items() if k != "type"}
    s = float(rest.pop("factor", 1.0))
    if not s > 0:
        raise ValueError(f"rotary: a scaling factor above 0, got {s}")
    mult = 1.0
    if kind == "linear":
        f = theta ** (-i / dim) / s
    elif kind == "ntk":
        if dim < 4:
            raise ValueError("rotary: ntk scaling of 4 elements at least")
        f = (theta * s ** (dim / (dim - 2))) ** (-i / dim)
    elif kind == "yarn":
        L = float(rest.pop("original_len", 0))
        fast, slow = float(rest.pop("beta_fast", 32.0)), float(rest.pop("beta_slow", 1.0))
        mult = rest.pop("attention_factor", None)
        mult = (0.1 * math.log(s) + 1.0 if s > 1 else 1.0) if mult is None else float(mult)
        if not L > 0 or not fast >= slow > 0:
            raise ValueError("rotary: yarn scaling with original_len above 0 and beta_fast >= beta_slow > 0")

        def pair(turns):
            return dim * math.log(L / (turns * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dim - 1)
        f = theta ** (-i / dim)
        part = ((i / 2 - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        f = f * (1 - part) + f / s * part
    else:
        raise ValueError(f"rotary: scaling type linear, ntk or yarn, got {kind!r}")
    if rest:
        raise ValueError(f"rotary: unknown scaling keys {sorted(rest)}")
    return f, mult


def rotary_table(dim: int, positions: int, theta: float = 10000.0, scaling: Optional[dict] = None, device="cuda"):
    """fp32 [positions, dim / 2, 2]: cosine and sine of each pair's angle at each position, evaluated
    in 64 bits (see :func:`rotary_angles`).  Made once per model; :func:`rotary` reads it."""
    f, mult = rotary_angles(dim, theta, scaling)
    a = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * f.to(device)
    return torch.stack([a.cos(), a.sin()], -1).mul_(mult).float()


def rotary(q, k, pos, table, layout: str = "half", sections: Optional[Sequence[int]] = None, inverse: bool = False):
    """(q, k) rotated by their positions, in their own type (bf16, fp16 or fp32; fp32 arithmetic); k may
    be None, and is then returned as None.

    q [..., n, heads, D], k [..., n, key heads, D] (views of a fused projection among them).  ``table``
    fp32 [positions, R / 2, 2] (:func:`rotary_table`), R <= D <= 256: elements from R on are copied.
    ``layout``: pair i is elements (i, i + R / 2) ("half") or (2 i, 2 i + 1) ("interleaved").  ``pos``:
    whole numbers [n], or [n, axes] with ``sections``, the pairs of each axis (their sum R / 2; up to
    4 axes).  ``inverse`` turns back (the gradient).  A position outside the table makes its token NaN
    and is reported by ``check_device_errors`` on the GPU, and raises on the CPU.

    It records no graph: ``models.functional.rotary`` is the form under autograd."""
    if q.is_cuda and not (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)
                                                       or table.requires_grad)):
        try:
            # the kernel's own checks come first: a call of a few microseconds has no time for both
            if layout == "half" or layout == "interleaved":
                out = ext().rotary_apply(q, k, pos, table, () if sections is None else sections, layout == "half",
                                         inverse)
                return out[0], out[1] if k is not None else None
        except (RuntimeError, TypeError):
            check_rotary(q, k, pos, table, layout, sections)
            raise
    ts, pos, sections = check_rotary(q, k, pos, table, layout, sections)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (*ts, table)):
        raise RuntimeError("rotary has no gradient here: use models.functional.rotary, or torch.no_grad()")
    out = [ref.rotary(t, pos, table, layout, sections, inverse) for t in ts]
    return out[0], out[1] if k is not None else None


def check_rotary(q, k, pos, table, layout, sections):
    """Raise for arguments that do not fit each other; (tensors, pos [n, axes], sections)."""
    ts = [t for t in (q, k) if t is not None]
    if layout not in LAYOUTS:
        raise ValueError(f"rotary: layout one of {LAYOUTS}, got {layout!r}")
    if any(t.dim() < 3 for t in ts) or any(t.shape[:-2] != q.shape[:-2] or t.shape[-1] != q.shape[-1] for t in ts):
        raise ValueError(f"rotary: q and k [..., n, heads, head_dim], got {[tuple(t.shape) for t in ts]}")
    if any(t.dtype != q.dtype or t.device != q.device for t in ts) or table.device != q.device or pos.device != q.device:
        raise TypeError("rotary: q and k of one type, with pos and table on their device")
    if q.dtype not in _TYPES and q.is_cuda:
        raise TypeError(f"rotary: bf16, fp16 or fp32, got {q.dtype}")
    if table.dim() != 3 or table.shape[2] != 2 or table.dtype != torch.float32:
        raise ValueError(f"rotary: table fp32 [positions, pairs, 2], got {table.dtype} {tuple(table.shape)}")
    pairs, n, D = table.shape[1], q.shape[-3], q.shape[-1]
    if 2 * pairs > D or D > 256 or D % 2:
        raise ValueError(f"rotary: a table of {pairs} pairs for a head dim of {D} (even, at most 256)")
    if pos.dtype.is_floating_point or pos.dtype == torch.bool:
        raise TypeError(f"rotary: whole positions, got {pos.dtype}")
    axes = 1 if sections is None else len(sections)
    sections = [pairs] if sections is None else [int(s) for s in sections]
    if not 1 <= axes <= 4 or min(sections) < 0 or sum(sections) != pairs:
        raise ValueError(f"rotary: sections {sections} of up to 4 axes for {pairs} pairs")
    if pos.dim() == 1:
        pos = pos[:, None]
    if pos.shape != (n, axes):
        raise ValueError(f"rotary: pos [{n}] or [{n}, {axes}], got {tuple(pos.shape)}")
    return ts, pos, sections
