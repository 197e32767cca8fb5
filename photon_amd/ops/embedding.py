"""Embedding lookup with scaling, and its gradient by sorted tokens.

    y[..., :]  = round(scale * table[ids, :])
    dtable[v]  = round(scale * sum of dy over the positions of token v)

The GPU path is a gather that scales and rounds on the way (under autocast it
writes the compute dtype directly, where ``nn.Embedding`` writes fp32 and a
second kernel rounds it), and a gradient that sorts the positions by token,
sums each token's rows in fp32 in a fixed order and writes every row of the
table once: the same inputs give the same bits. The CPU path is plain torch.
"""

from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd import forward_ad

from . import hip_ext, use_hip

_FLOATS = (torch.float32, torch.bfloat16)


def embedding(
    ids: torch.Tensor,
    table: torch.Tensor,
    scale: float = 1.0,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """Rows ``ids`` (int64 or int32, any shape) of ``table`` [V, D] (fp32 or
    bf16), times ``scale``, as ``out_dtype`` (default: the table's).

    Differentiable once in ``table``; on the GPU not in forward mode. An id
    outside [0, V) raises IndexError on the CPU; on the GPU, where looking
    would wait for the device, its row is NaN and it has no gradient."""
    out_dtype = out_dtype or table.dtype
    if use_hip(table):  # checks the same
        return hip_ext().embedding(ids, table, scale, out_dtype)
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"embedding: ids must be int64 or int32, got {ids.dtype}")
    if table.dim() != 2:
        raise ValueError(f"embedding: table must be [V, D], got {tuple(table.shape)}")
    if table.dtype == torch.bfloat16 and table.requires_grad \
            and torch.is_grad_enabled():
        table = table.float()  # torch adds the gradient up in the table's type
    y = F.embedding(ids, table)
    if scale != 1.0:
        y = y.to(torch.promote_types(y.dtype, torch.float32)) * scale
    return y.to(out_dtype)


def _kernel_sees(w: torch.Tensor) -> bool:
    """A plain table with whole rows, outside of forward mode, ``torch.func``
    transforms and tracing: none of them sees what a kernel does."""
    return (type(w) in (torch.Tensor, nn.Parameter)
            and (w.stride(1) == 1 or w.shape[1] <= 1)
            and forward_ad._current_level < 0
            and not torch._C._are_functorch_transforms_active()
            and not torch.jit.is_tracing()
            and not torch.compiler.is_compiling())


class FusedEmbedding(nn.Embedding):
    """``nn.Embedding`` whose rows come out scaled, and in the autocast dtype
    where autocast is on. ``impl="torch"`` keeps torch's lookup and gradient,
    which also serve where the kernel cannot (:func:`_kernel_sees`), but for
    second derivatives, which only ``impl="torch"`` has on a GPU."""

    def __init__(self, num_embeddings: int, embedding_dim: int,
                 scale: float = 1.0, impl: str = "fused", **kw):
        super().__init__(num_embeddings, embedding_dim, **kw)
        if self.padding_idx is not None or self.max_norm is not None \
                or self.scale_grad_by_freq or self.sparse:
            raise ValueError("FusedEmbedding: a dense table without padding "
                             "index, max_norm or frequency scaling")
        self.scale = float(scale)
        self.impl = impl

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        w = self.weight
        kind = w.device.type
        out_dtype = w.dtype
        if torch.is_autocast_enabled(kind):
            out_dtype = torch.get_autocast_dtype(kind)
        fused = self.impl == "fused" and w.dtype in _FLOATS \
            and out_dtype in _FLOATS and _kernel_sees(w)
        if fused:
            return embedding(ids, w, self.scale, out_dtype)
        y = F.embedding(ids, w)
        if self.scale != 1.0:
            y = y * self.scale
        return y.to(out_dtype)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, scale={self.scale}, impl={self.impl}"
