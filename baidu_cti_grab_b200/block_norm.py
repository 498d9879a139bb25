"""The seam between two blocks of the encoder: the norm after a block, its gate and residual
scale, and the norm before the next block, as one kernel in each direction.

The reference's TransformerEncoder adds a block's output to the stream and normalises the
sum for the next block as separate torch ops (models.py:208-249).  ``sandwich_norm`` does that
in one pass, with what deeper encoders need there: a norm of the block's output, a gate
(per channel, per row or per element) and a residual scale; it is differentiable.
``SandwichNorm`` is the module around it.
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from . import device_ops


class _SandwichNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, h, gate, post_weight, post_bias, pre_weight, pre_bias, how, eps):
        tensors = dict(post_weight=post_weight, post_bias=post_bias, gate=gate, pre_weight=pre_weight, pre_bias=pre_bias)
        y, z, stats = device_ops.sandwich_norm(x, h, want_stats=True, **tensors, **how, **eps)
        ctx.save_for_backward(x, h, gate, post_weight, post_bias, pre_weight, pre_bias, stats)
        ctx.how = how
        ctx.set_materialize_grads(False)
        return y, z

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y, grad_z):
        if grad_y is None and grad_z is None:
            return (None,) * 9
        x, h, gate, post_weight, post_bias, pre_weight, pre_bias, stats = ctx.saved_tensors
        grads = device_ops.sandwich_norm_backward(grad_y, grad_z, x, h, stats, post_weight=post_weight,
                                                  post_bias=post_bias, gate=gate, pre_weight=pre_weight,
                                                  pre_bias=pre_bias, **ctx.how)
        return (*grads, None, None)


def sandwich_norm(x: torch.Tensor, h: torch.Tensor, *, post: Optional[str] = None,
                  post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                  post_eps: float = 1e-5, gate: Optional[torch.Tensor] = None, gate_act: str = "none", scale: float = 1.0,
                  pre: Optional[str] = None, pre_weight: Optional[torch.Tensor] = None,
                  pre_bias: Optional[torch.Tensor] = None, pre_eps: float = 1e-5):
    """(y, z): y = x + scale * act(gate) * post(h), z = pre(y) (None without pre), with gradients for every
    tensor; see device_ops.sandwich_norm."""
    tensors = (x, h, gate, post_weight, post_bias, pre_weight, pre_bias)
    how = dict(post=post, gate_act=gate_act, scale=scale, pre=pre)
    eps = dict(post_eps=post_eps, pre_eps=pre_eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return _SandwichNorm.apply(*tensors, how, eps)
    y, z, _ = device_ops.sandwich_norm(x, h, gate=gate, post_weight=post_weight, post_bias=post_bias,
                                       pre_weight=pre_weight, pre_bias=pre_bias, **how, **eps)
    return y, z


class SandwichNorm(nn.Module):
    """The seam after one block: ``post`` norm of its output, gate, residual scale, ``pre`` norm of the next.

    ``channel_gate`` adds a learned gate per channel (initially ``gate_init``); a gate per row or
    element is given to forward instead.  forward(x, h, gate=None) returns (y, z)."""

    def __init__(self, width: int, *, post: Optional[str] = "layer", pre: Optional[str] = "layer", eps: float = 1e-5,
                 scale: float = 1.0, gate_act: str = "none", channel_gate: bool = False, gate_init: float = 1.0):
        super().__init__()
        self.post, self.pre, self.eps, self.scale, self.gate_act = post, pre, eps, scale, gate_act
        for name, kind in (("post", post), ("pre", pre)):
            self.register_parameter(name + "_weight", None if kind is None else nn.Parameter(torch.ones(width)))
            self.register_parameter(name + "_bias", nn.Parameter(torch.zeros(width)) if kind == "layer" else None)
        self.gate = nn.Parameter(torch.full((width,), float(gate_init))) if channel_gate else None

    def forward(self, x: torch.Tensor, h: torch.Tensor, gate: Optional[torch.Tensor] = None):
        if gate is not None and self.gate is not None:
            raise ValueError("this module has a gate of its own")
        return sandwich_norm(x, h, post=self.post, post_weight=self.post_weight, post_bias=self.post_bias,
                             post_eps=self.eps, gate=self.gate if gate is None else gate, gate_act=self.gate_act,
                             scale=self.scale, pre=self.pre, pre_weight=self.pre_weight, pre_bias=self.pre_bias,
                             pre_eps=self.eps)
