"""Attention within packed users: the encoder's own attention over many users' items at once.

The reference packs users one behind the other and attends causally within each
(models.py:271-279), through a separate library or a dense [N, N] mask (models.py:258-265).
``segment_attention`` reads the user offsets on the device, needs neither the longest length
nor a mask, and has what encoders of longer histories use: fewer key/value heads than query
heads, a prefix that every query sees, scores capped by a tanh, a bias that falls with
distance, keys of other lengths than the queries' (a user's cached history under a few new
items); it is differentiable.  ``SegmentAttention`` is the module around it.
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from . import device_ops


class _SegmentAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets, k_offsets, how):
        out, lse = device_ops.segment_attention(q, k, v, offsets, k_offsets, want_lse=True, **how)
        ctx.save_for_backward(q, k, v, out, lse, offsets, k_offsets, how["prefix"], how["slopes"])
        ctx.how = {n: how[n] for n in ("causal", "cap", "scale")}
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        q, k, v, out, lse, offsets, k_offsets, prefix, slopes = ctx.saved_tensors
        grads = device_ops.segment_attention_backward(grad, q, k, v, out, lse, offsets, k_offsets, prefix=prefix,
                                                      slopes=slopes, **ctx.how)
        return (*grads, None, None, None)


def segment_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor,
                      k_offsets: Optional[torch.Tensor] = None, *, causal: bool = True,
                      prefix: Optional[torch.Tensor] = None, slopes: Optional[torch.Tensor] = None, cap: float = 0.0,
                      scale: Optional[float] = None) -> torch.Tensor:
    """device_ops.segment_attention with gradients for q, k and v (slopes are constants: one that asks for a gradient
    is refused)."""
    if slopes is not None and slopes.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("slopes get no gradient: give them detached")
    how = dict(causal=causal, prefix=prefix, slopes=slopes, cap=cap, scale=scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _SegmentAttention.apply(q, k, v, offsets, k_offsets, how)
    return device_ops.segment_attention(q, k, v, offsets, k_offsets, **how)[0]


class SegmentAttention(nn.Module):
    """Projections to queries, keys and values, ``segment_attention``, and the projection back.

    forward(x [N, d_model], offsets) attends within the users; forward(x, offsets, cache=(k, v, k_offsets)) reads the
    keys and values of ``keys_and_values`` instead, whose segments end with x's own items."""

    def __init__(self, d_model: int, n_heads: int, n_kv_heads: Optional[int] = None, *, head_dim: Optional[int] = None,
                 causal: bool = True, cap: float = 0.0, distance: bool = False, bias: bool = True):
        super().__init__()
        self.heads = n_heads
        self.kv_heads = n_heads if n_kv_heads is None else n_kv_heads
        if self.kv_heads < 1 or n_heads % self.kv_heads:
            raise ValueError("n_kv_heads must divide n_heads")
        if head_dim is None and d_model % n_heads:
            raise ValueError("n_heads must divide d_model where head_dim is not given")
        self.width = d_model // n_heads if head_dim is None else head_dim
        self.causal, self.cap = causal, cap
        self.qkv = nn.Linear(d_model, (n_heads + 2 * self.kv_heads) * self.width, bias=bias)
        self.out = nn.Linear(n_heads * self.width, d_model, bias=bias)
        slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / n_heads) for h in range(n_heads)]) if distance else None
        self.register_buffer("slopes", slopes, persistent=False)

    def _apply(self, fn, recurse=True):
        # module.to(bf16) also casts float buffers; the slopes are added to fp32 scores and stay fp32
        slopes = self.slopes
        super()._apply(fn, recurse)
        if slopes is not None and self.slopes.dtype != torch.float32:
            self.slopes = slopes.to(self.slopes.device)
        return self

    def _project(self, x: torch.Tensor):
        fused = self.qkv(x).view(x.shape[0], self.heads + 2 * self.kv_heads, self.width)
        return fused.split((self.heads, self.kv_heads, self.kv_heads), 1)

    def keys_and_values(self, x: torch.Tensor):
        """(k, v) [N, kv_heads, head_dim] of items, as a cache holds them."""
        _, k, v = self._project(x)
        return k.contiguous(), v.contiguous()

    def forward(self, x: torch.Tensor, offsets: torch.Tensor, *, prefix: Optional[torch.Tensor] = None, cache=None):
        q, k, v = self._project(x)
        k_offsets = None
        if cache is not None:
            k, v, k_offsets = cache
        o = segment_attention(q, k, v, offsets, k_offsets, causal=self.causal, prefix=prefix, slopes=self.slopes, cap=self.cap)
        return self.out(o.reshape(x.shape[0], self.heads * self.width))
