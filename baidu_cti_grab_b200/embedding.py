"""Embedding rows and the gradient of their table: what the RepEncoder's table needs to be trained.

The reference pools bags of ids from one shared table (nn.EmbeddingBag, models.py:14-34) and
is run for inference only; the pooled forward here is ``device_ops.rep_gather_pool`` and the
fused kernels around it.  ``embed`` looks rows up and scales them, with the table's gradient
by sorted ids.  ``bag_gradient`` is the gradient of sum-pooled bags (``rep_gather_pool``'s among
them): of all rows, or, for tables of which a batch touches a small part, ``SparseRows`` of
the touched rows alone, which ``grad_clip`` takes as they are.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
import torch.nn as nn

from . import device_ops


class SparseRows(NamedTuple):
    """Gradients of some rows of a table: the first ``count`` entries hold."""

    ids: torch.Tensor     # int64 [n], ascending
    rows: torch.Tensor    # [n, D]
    count: torch.Tensor   # int32 [1], on the device


def _padding_row(padding_idx: Optional[int], rows: int) -> Optional[int]:
    """padding_idx as a row of the table: one below 0 counts from its end, as torch's does."""
    if padding_idx is None:
        return None
    if not -rows <= padding_idx < max(rows, 1):
        raise ValueError(f"padding_idx must be a row of the table's {rows}, or count from its end")
    return padding_idx + rows if padding_idx < 0 else padding_idx


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale, ctx.padding_idx = table.shape[0], scale, padding_idx
        return device_ops.embed_rows(table, ids, scale=scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        ids, = ctx.saved_tensors
        return device_ops.embed_rows_backward(grad, ids, ctx.rows, scale=ctx.scale, padding_idx=ctx.padding_idx), None, None, None


def embed(table: torch.Tensor, ids: torch.Tensor, *, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """scale * table[ids] [*ids.shape, D], with the table's gradient; the row of padding_idx is looked up as it is and gets
    no gradient.  Ids are clamped to the table, as the RepEncoder clamps them; a padding_idx below 0 counts from its end."""
    padding_idx = _padding_row(padding_idx, table.shape[0])
    if torch.is_grad_enabled() and table.requires_grad:
        return _Embed.apply(table, ids, scale, padding_idx)
    return device_ops.embed_rows(table, ids, scale=scale)


def bag_gradient(grad: torch.Tensor, ids: torch.Tensor, bags: torch.Tensor, rows: int, *, scale: float = 1.0,
                 padding_idx: Optional[int] = 0, sparse: bool = False, out: Optional[torch.Tensor] = None):
    """The table's gradient of bags pooled by summing: grad [bags, D], ids [n], bags [bags + 1] offsets into them.

    Ids of padding_idx (row 0, as the RepEncoder has it) add nothing.  A tensor [rows, D], added to `out` where that is
    given, or SparseRows."""
    how = dict(bags=bags, scale=scale, padding_idx=_padding_row(padding_idx, rows))
    if not sparse:
        return device_ops.embed_rows_backward(grad, ids, rows, out=out, **how)
    if out is not None:
        raise ValueError("sparse rows are not added to an out")
    return SparseRows(*device_ops.embed_rows_backward_sparse(grad, ids, rows, **how))


class RowEmbedding(nn.Module):
    """A table [rows, width]; forward(ids) is ``embed`` with this module's scale and padding row."""

    def __init__(self, rows: int, width: int, *, scale: float = 1.0, padding_idx: Optional[int] = None, std: float = 0.02):
        super().__init__()
        self.scale, self.padding_idx = scale, _padding_row(padding_idx, rows)
        weight = torch.randn(rows, width) * std
        if padding_idx is not None:
            weight[self.padding_idx] = 0.0
        self.weight = nn.Parameter(weight)

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return embed(self.weight, ids, scale=self.scale, padding_idx=self.padding_idx)
