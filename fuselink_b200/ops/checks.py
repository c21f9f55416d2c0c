"""Whether a tensor is one that a kernel may read in place of the framework's operations."""
from __future__ import annotations

import torch
import torch.nn as nn


def ordinary(t: torch.Tensor) -> bool:
    """Whether a kernel may read this tensor in place of the framework's operations: no subclass, and neither a function transform
    (vmap, grad, jvp), forward-mode differentiation, a dispatch mode nor tracing that has to see the operations."""
    # a batched gradient reaches the backward on a thread without the transform, and shows itself by having no memory
    return (type(t) in (torch.Tensor, nn.Parameter) and torch._C._has_storage(t) and not torch._C._are_functorch_transforms_active()
            and torch.autograd.forward_ad._current_level < 0 and torch._C._len_torch_dispatch_stack() == 0
            and not torch.jit.is_tracing() and not torch.compiler.is_compiling())
