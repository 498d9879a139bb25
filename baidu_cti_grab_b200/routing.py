"""Routing to experts: the gate that stands before ``smoe.smoe_forward`` and
``device_ops.smoe_experts``.

The reference's gate (TopKGate, whose result SMoE.forward takes, models.py:131-178) is a
Linear, a softmax and a top-k.  ``route_topk`` is that choice as one kernel, with what
larger sets of experts need: sigmoid scores, a bias that balances the experts' load
without a loss, experts in groups, renormalised weights; it is differentiable.
``TopKRouter`` is a gate module around it: it returns (idx, score, probs) as the
reference's gate does, so an ``SMoE`` with ``moe.gate = TopKRouter(...)`` runs through
``smoe_forward`` unchanged.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
import torch.nn as nn

from . import device_ops


class Routing(NamedTuple):
    idx: torch.Tensor                # [T, k] experts by falling choice value
    score: torch.Tensor              # [T, k] weights of the chosen experts
    probs: Optional[torch.Tensor]    # [T, E] scores of all experts
    counts: Optional[torch.Tensor]   # int32 [E] how often each expert was chosen


class _RouteTopK(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, k, how, choice, wants):
        idx, score, probs, counts = device_ops.route_topk(logits, k, bias=bias, **how, **choice, **wants)
        ctx.save_for_backward(logits, idx)
        ctx.how = how
        ctx.mark_non_differentiable(*(t for t in (idx, counts) if t is not None))
        ctx.set_materialize_grads(False)
        return idx, score, probs, counts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, _idx, grad_score, grad_probs, _counts):
        if grad_score is None and grad_probs is None:
            return (None,) * 6
        logits, idx = ctx.saved_tensors
        grad = device_ops.route_topk_backward(logits, idx, grad_score, grad_probs, **ctx.how)
        return (grad,) + (None,) * 5


def route_topk(logits: torch.Tensor, k: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None,
               groups: int = 1, topk_groups: int = 1, group_top: int = 2, renormalize: bool = False,
               scale: float = 1.0, idx_dtype: torch.dtype = torch.int64, score_dtype: Optional[torch.dtype] = None,
               want_probs: bool = False, want_counts: bool = False) -> Routing:
    """device_ops.route_topk with gradients: score and probs carry the logits' (never the bias's)."""
    how = dict(score=score, renormalize=renormalize, scale=scale)
    choice = dict(groups=groups, topk_groups=topk_groups, group_top=group_top)
    wants = dict(idx_dtype=idx_dtype, score_dtype=score_dtype, want_probs=want_probs, want_counts=want_counts)
    if torch.is_grad_enabled() and logits.requires_grad:
        return Routing(*_RouteTopK.apply(logits, bias, k, how, choice, wants))
    return Routing(*device_ops.route_topk(logits, k, bias=bias, **how, **choice, **wants))


class TopKRouter(nn.Module):
    """A gate: Linear (``w_g``, as the reference's gate names it) and ``route_topk``.

    ``balance_bias`` (fp32 [E], a buffer, zeros at first) takes part in the choice when
    ``balanced``; ``update_balance(counts)`` moves it by ``step`` against the load, up for experts
    with fewer tokens than the mean and down for those with more."""

    def __init__(self, d_model: int, n_experts: int, k: int, *, score: str = "softmax", groups: int = 1,
                 topk_groups: int = 1, group_top: int = 2, renormalize: bool = False, scale: float = 1.0,
                 balanced: bool = False):
        super().__init__()
        self.w_g = nn.Linear(d_model, n_experts)
        self.k = k
        self.score = score
        self.groups, self.topk_groups, self.group_top = groups, topk_groups, group_top
        self.renormalize, self.scale = renormalize, scale
        self.balanced = balanced
        self.register_buffer("balance_bias", torch.zeros(n_experts, dtype=torch.float32) if balanced else None)

    def _apply(self, fn, recurse=True):
        # module.to(bf16) also casts float buffers; the bias is compared with fp32 scores and stays fp32
        bias = self.balance_bias
        super()._apply(fn, recurse)
        if bias is not None and self.balance_bias.dtype != torch.float32:
            self.balance_bias = bias.to(self.balance_bias.device)
        return self

    def route(self, x: torch.Tensor, want_probs: bool = True, want_counts: bool = False) -> Routing:
        """Routing of the rows of x [..., d_model], flattened to [T, d_model]."""
        logits = self.w_g(x.reshape(-1, x.shape[-1]))
        return route_topk(logits, self.k, score=self.score, bias=self.balance_bias, groups=self.groups,
                          topk_groups=self.topk_groups, group_top=self.group_top, renormalize=self.renormalize,
                          scale=self.scale, want_probs=want_probs, want_counts=want_counts)

    def forward(self, x: torch.Tensor):
        """(idx [..., k], score [..., k], probs [..., E]) of x [..., d_model], as the reference's gate."""
        r = self.route(x)
        lead = x.shape[:-1]
        return r.idx.view(*lead, self.k), r.score.view(*lead, self.k), r.probs.view(*lead, r.probs.shape[-1])

    @torch.no_grad()
    def update_balance(self, counts: torch.Tensor, step: float = 1e-3) -> None:
        if self.balance_bias is None:
            raise ValueError("this router has no balance bias (balanced=False)")
        load = counts.to(self.balance_bias.device, torch.float32)
        self.balance_bias.add_(torch.sign(load.mean() - load), alpha=step)
