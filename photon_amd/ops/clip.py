"""Norms over many tensors in one sweep, and clipping by the global norm.

Replaces the reference's composer ``algorithms.gradient_clipping`` (norm 1.0,
mpt-125m.yaml:65-68). One kernel sums the squares of all tensors in 64 bits,
whatever their lengths and types, a second makes each tensor's norm and the
global one, and a third scales every gradient by max_norm / (total + 1e-6)
where that is below 1; the norm never leaves the device.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import hip_ext, use_hip


def tensor_norms(tensors) -> tuple[torch.Tensor, torch.Tensor]:
    """(global L2 norm, [n] L2 norm of each) of fp32 and bf16 tensors on one
    device, as fp32 tensors there. The tensors stay as they are; no derivative
    passes through."""
    tensors = list(tensors)
    if not tensors:
        return torch.zeros(()), torch.zeros(0)
    if use_hip(tensors[0]):
        total, norms = hip_ext().tensor_norms([t.detach() for t in tensors])
        return total, norms
    squares = torch.stack([t.detach().double().square().sum() for t in tensors])
    return squares.sum().sqrt().float(), squares.sqrt().float()


@torch.no_grad()
def clip_grads_(grads, max_norm: float) -> tuple[torch.Tensor, torch.Tensor]:
    """Scale ``grads`` in place by min(1, max_norm / (total + 1e-6)).

    Returns (total, norms) as :func:`tensor_norms` does, of the gradients
    before clipping. The gradients are fp32 or bf16 (mixed lists too), dense
    or strided, on one device, and share no memory. Where the total is NaN, so
    is every gradient afterwards; where it is infinite, finite ones are zero."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"clip_grads_: max_norm must be >= 0, got {max_norm}")
    grads = list(grads)
    if not grads:
        return torch.zeros(()), torch.zeros(0)
    if use_hip(grads[0]):
        total, norms = hip_ext().clip_grads(grads, max_norm)
        return total, norms
    if not torch.is_inference_mode_enabled() and any(g.is_inference() for g in grads):
        raise RuntimeError("clip_grads_: a gradient was made in inference mode "
                           "and cannot be written outside of it")
    if forward_ad._current_level >= 0 and any(
            forward_ad.unpack_dual(g).tangent is not None for g in grads):
        raise NotImplementedError("clip_grads: forward-mode derivatives are not supported")
    total, norms = tensor_norms(grads)
    scale = max_norm / (total + 1e-6)
    if not scale >= 1.0:
        for g in grads:
            wide = g.double() if g.dtype == torch.float64 else g.float()
            g.copy_(wide * scale)
    return total, norms


def clip_grad_norm_(params, max_norm: float) -> torch.Tensor:
    """Clip the gradients of ``params`` in place; returns their global norm
    before clipping. A parameter listed twice counts once."""
    grads = {id(p): p.grad for p in params if p.grad is not None}
    if not grads:
        return torch.zeros(())
    return clip_grads_(grads.values(), max_norm)[0]
