"""Low-rank adapters of many requests beside a projection that they share.

A projection whose weight is frozen (the RepEncoder's int8 Linear, a fused q/k/v
projection) serves users or scenarios that each have a small adapter: out = W x + bias +
scale_i B_i (A_i x).  ``AdapterBank`` holds the adapters of one projection, stacked, and adds
each token's own to the shared output in one call, whatever the order of the tokens:

    bank = AdapterBank.stack([(a0, b0, s0), (a1, b1, s1), ...])
    y = linear(x)                                  # shared: W8A8, bf16, ...
    bank(y, x, bank.per_token(user_adapter, user_offsets, n_items), out=y)
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch
import torch.nn as nn

from . import device_ops


class AdapterBank(nn.Module):
    """Adapters a [R, rank, K], b [R, N, rank] (buffers, one type) and scale fp32 [R]."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scale: Optional[torch.Tensor] = None):
        super().__init__()
        if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2] or a.dtype != b.dtype:
            raise ValueError("expected a [R, rank, K] and b [R, N, rank] of one type")
        scale = torch.ones(a.shape[0], device=a.device) if scale is None else scale
        if tuple(scale.shape) != (a.shape[0],):
            raise ValueError(f"scale must be [{a.shape[0]}]")
        self.register_buffer("a", a.detach().contiguous())
        self.register_buffer("b", b.detach().contiguous())
        self.register_buffer("scale", scale.detach().float().contiguous())

    @classmethod
    def stack(cls, adapters: Sequence[Tuple[torch.Tensor, torch.Tensor, float]]) -> "AdapterBank":
        """A bank of (a [rank, K], b [N, rank], scale) adapters; smaller ranks are filled up with zeros."""
        if not adapters:
            raise ValueError("no adapters")
        rank = max(a.shape[0] for a, _, _ in adapters)
        a = torch.stack([nn.functional.pad(a, (0, 0, 0, rank - a.shape[0])) for a, _, _ in adapters])
        b = torch.stack([nn.functional.pad(b, (0, rank - b.shape[1])) for _, b, _ in adapters])
        return cls(a, b, torch.tensor([float(s) for _, _, s in adapters], device=a.device))

    def _apply(self, fn, recurse=True):
        # module.to(bf16) also casts float buffers; the scales stay fp32
        scale = self.scale
        super()._apply(fn, recurse)
        if self.scale.dtype != torch.float32:
            self.scale = scale.to(self.scale.device)
        return self

    @staticmethod
    def per_token(request_adapter: torch.Tensor, offsets: torch.Tensor, n_tokens: int) -> torch.Tensor:
        """int32 [n_tokens]: each token's adapter, from its request's, request u being the tokens
        offsets[u] .. offsets[u + 1] - 1 (the batch's ``user_offsets``); -1 for tokens before the first
        and behind the last (a padded batch).  Nothing is read back."""
        token = torch.arange(n_tokens, dtype=offsets.dtype, device=offsets.device)
        request = torch.searchsorted(offsets[1:].contiguous(), token, right=True)
        who = nn.functional.pad(request_adapter.to(torch.int32), (0, 1), value=-1)[request]
        return who.masked_fill_(token < offsets[0], -1)

    def forward(self, y: torch.Tensor, x: torch.Tensor, adapter: torch.Tensor, out: Optional[torch.Tensor] = None):
        """y [..., N] plus each token's adapter of x [..., K]; adapter int32/int64 of the leading shape.
        No backward: with gradients enabled, tensors that ask for one are refused (call it under torch.no_grad())."""
        lead, N, K = y.shape[:-1], y.shape[-1], x.shape[-1]
        if out is not None and out.dim() != 2 and not out.is_contiguous():
            raise ValueError("out must be contiguous, or 2-D with contiguous rows")
        res = device_ops.low_rank_add(y.reshape(-1, N), x.reshape(-1, K), self.a, self.b, adapter.reshape(-1), self.scale,
                                      out=None if out is None else out.view(-1, N) if out.dim() != 2 else out)
        return res.view(*lead, N) if out is None else out
