"""When to rebuild what is packed from weights (stacked q/k/v, folded LoRA factors, quantised copies).

A tensor's address and version tell of most changes.  They do not for the weights that FSDP
gathers: those are written without advancing the version, often into the same memory as the step
before.  So every optimizer step and every swap of averaged weights is counted as well.
"""
from __future__ import annotations

_CHANGES = [0]


def weights_changed():
    """To be called after the model's weights were written in place."""
    _CHANGES[0] += 1


def weights_key(tensors) -> tuple:
    """Equal for equal weights: what is packed from ``tensors`` holds while this stays the same."""
    return (_CHANGES[0],) + tuple((t.data_ptr(), t._version) for t in tensors if t is not None)
