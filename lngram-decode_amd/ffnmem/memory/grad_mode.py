"""What kind of derivative a call of a differentiable operator is asked for."""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad


def needs_grad(*tensors: Optional[Tensor]) -> bool:
    """Whether the call has to leave a node of the autograd graph.  Raises where a tensor carries a forward-mode
    tangent: the operators have no forward-mode derivative, and a kernel would drop it in silence."""
    if forward_ad._current_level >= 0:               # inside a dual level (or torch.func.jvp)
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("no forward-mode derivative: this operator is differentiable in reverse "
                                          "mode only")
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False
