"""AdamW whose update is a fused sm_100a kernel.

Same update rule and hyper-parameters as ``torch.optim.AdamW`` (the reference's
optimizer, train_osp.py:303-311).  Works on plain tensors and on FSDP2 DTensor
parameters (it updates the local shard).  ``grad_scale`` folds the gradient
clipping factor into the same pass.  CPU tensors fall back to
``torch.optim.AdamW``'s math.

One launch per parameter shard by default; ``multi_tensor=True`` updates all of them in a
few launches (``ops.adamw_multi_``).  ``state_bits=8`` keeps both moments in 8 bits, a quarter
of the optimizer's memory (2.03 bytes per parameter for 8), and implies ``multi_tensor``.
Checkpoints hold fp32 moments either way, so a run can change ``state_bits`` on resume.

A step counts as an in-place change of each parameter (``_version``, through ``detach()``; ``.data``
would hide it), as with torch's optimizers: what was packed from the old weights is built anew.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import ops
from ..ops import reference as ref
from ..utils.weights import weights_changed


def _local(t):
    return t.to_local() if hasattr(t, "to_local") else t


def _like(local, p):
    """``local`` in the distributed layout of ``p`` (itself for a plain tensor)."""
    if not hasattr(p, "to_local"):
        return local
    from torch.distributed.tensor import DTensor
    return DTensor.from_local(local, p.device_mesh, p.placements, shape=p.shape, stride=p.stride())


_STATE8 = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")


class FusedAdamW(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits: int = 32,
                 multi_tensor: Optional[bool] = None, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits 8 or 32, got {state_bits}")
        if multi_tensor is None:
            multi_tensor = state_bits == 8
        if state_bits == 8 and not multi_tensor:
            raise ValueError("8-bit moments need multi_tensor")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self.grad_scale = 1.0
        self.state_bits = state_bits
        self.multi_tensor = multi_tensor
        self.seed = seed

    @torch.no_grad()
    def step(self, closure=None):
        loss = closure() if closure is not None else None
        for number, group in enumerate(self.param_groups):
            if self.multi_tensor:
                self._step_multi(number, group)
                continue
            b1, b2 = group["betas"]
            for p in group["params"]:
                if p.grad is None:
                    continue
                st = self.state[p]
                lp, lg = _local(p.detach()), _local(p.grad)
                if not st:
                    st["step"] = torch.tensor(0.0)
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                st["step"] += 1
                step = int(st["step"].item())
                m, v = _local(st["exp_avg"]), _local(st["exp_avg_sq"])
                if lp.is_cuda and lp.dtype == torch.float32 and lp.is_contiguous():
                    ops.adamw_(lp, lg.contiguous(), m, v, group["lr"], b1, b2, group["eps"], group["weight_decay"],
                               step, self.grad_scale)
                else:
                    g = lg.float() * self.grad_scale
                    lp.mul_(1 - group["lr"] * group["weight_decay"])
                    m.mul_(b1).add_(g, alpha=1 - b1)
                    v.mul_(b2).addcmul_(g, g, value=1 - b2)
                    bc1 = 1 - b1 ** step
                    bc2 = 1 - b2 ** step
                    denom = (v.sqrt() / (bc2 ** 0.5)).add_(group["eps"])
                    lp.addcdiv_(m, denom, value=-group["lr"] / bc1)
        weights_changed()
        return loss

    # ------------------------------------------------------------------ lists of tensors
    def _init_state(self, p):
        lp = _local(p.data)
        if self.state_bits == 8:
            return dict(zip(_STATE8, ops.adamw8_state(lp)))
        return {k: _like(torch.zeros(lp.shape, dtype=torch.float32, device=lp.device), p)
                for k in ("exp_avg", "exp_avg_sq")}

    def _step_multi(self, number, group):
        # parameters that share a step count, types and device go in one call
        sets = {}
        for p in group["params"]:
            if p.grad is None:
                continue
            st = self.state[p]
            if not st:
                st["step"] = torch.tensor(0.0)
                st.update(self._init_state(p))
            st["step"] += 1
            lp, lg = _local(p.detach()), _local(p.grad)
            if not lp.is_contiguous():
                raise ValueError("multi_tensor: parameters have to be contiguous")
            if lg.dtype not in (torch.float32, torch.bfloat16):
                lg = lg.float()
            lists = sets.setdefault((int(st["step"].item()), lp.dtype, lg.dtype, lp.device),
                                    [[] for _ in range(6 if self.state_bits == 8 else 4)])
            moments = [_local(st[k]) for k in (_STATE8 if self.state_bits == 8 else _STATE8[:2])]
            for dst, t in zip(lists, [lp, lg.contiguous(), *moments]):
                dst.append(t)
        b1, b2 = group["betas"]
        for i, ((step, *_), lists) in enumerate(sets.items()):
            # another seed for each step, parameter group and set
            seed = (self.seed + step * 0x9E3779B1 + number * 0x85EB + i * 0xCA6B) & 0x7FFFFFFF
            ops.adamw_multi_(*lists, lr=group["lr"], beta1=b1, beta2=b2, eps=group["eps"],
                             weight_decay=group["weight_decay"], step=step, grad_scale=self.grad_scale, seed=seed)

    # ------------------------------------------------------------------ checkpoints: fp32 moments
    def state_dict(self):
        sd = super().state_dict()
        if self.state_bits != 8:
            return sd
        order = [p for g in self.param_groups for p in g["params"]]
        state = {}
        for i, st in sd["state"].items():
            m, v = ops.adamw8_decode(*(st[k] for k in _STATE8))
            state[i] = {"step": st["step"], "exp_avg": _like(m, order[i]), "exp_avg_sq": _like(v, order[i])}
        return dict(sd, state=state)

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        if not self.multi_tensor:
            return
        # torch casts the state to the parameter's type; the moments of 16-bit parameters are taken
        # from the checkpoint again, as they were saved
        numbers = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(numbers, (p for g in self.param_groups for p in g["params"])):
            st = self.state.get(p, {})
            for k in ("exp_avg", "exp_avg_sq"):
                if k in st and st[k].dtype != torch.float32:
                    st[k] = state_dict["state"][i][k].to(device=st[k].device, dtype=torch.float32)
        if self.state_bits != 8:
            return
        for p, st in self.state.items():
            m, v = _local(st.pop("exp_avg")).float(), _local(st.pop("exp_avg_sq")).float()
            half = torch.full(m.shape, 0x80008000, dtype=torch.int64, device=m.device)    # to nearest
            for k, t in zip(("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"),
                            ref.adamw8_encode(m, v, half)):
                st[k] = t
