"""What a transform of torch's has to be told, where an operator has no formula for it."""
from __future__ import annotations

import torch

from . import _lib


def refuse_tangents(name: str, *tensors) -> None:
    """An error for a tensor that carries a tangent of forward-mode differentiation, in whatever wrappers of torch.func: a registered operator
    without a formula drops it without a word where nothing requires a gradient, which counts as a tangent of zero."""
    wrapped, unwrap = torch._C._functorch.is_functorch_wrapped_tensor, torch._C._functorch.get_unwrapped
    for t in tensors:
        while t is not None:
            if _lib.host().has_tangent(t):
                raise NotImplementedError(f"{name} has no formula for forward mode differentiation")
            t = unwrap(t) if wrapped(t) else None
