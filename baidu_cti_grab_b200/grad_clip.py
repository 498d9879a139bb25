"""Clipping of a training step's gradients by their norm together, in two kernels and without waiting for the norm.

``clip_grad_norm`` is the call between backward and the optimiser: the gradients of some
parameters and, beside them, ``embedding.SparseRows`` of tables whose gradient is kept for
the touched rows alone.
"""

from __future__ import annotations

from typing import Iterable, Union

import torch

from . import device_ops
from .embedding import SparseRows


def _gradients(parameters, sparse):
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    return grads + [(s.rows, s.count) for s in sparse]


def clip_grad_norm(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, *,
                   sparse: Iterable[SparseRows] = (), scale: float = 1.0) -> torch.Tensor:
    """Clip the gradients of `parameters` (those that have one) and of `sparse` in place; returns their norm, fp32 [] on
    the device.  `scale` takes a loss scale back: it multiplies every gradient, and the norm is that of the products."""
    grads = _gradients(parameters, sparse)
    if not grads:
        return torch.zeros(())
    return device_ops.clip_grads(grads, max_norm, scale=scale)


def grad_norm(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], *, sparse: Iterable[SparseRows] = (),
              scale: float = 1.0) -> torch.Tensor:
    """The norm that clip_grad_norm would clip by."""
    grads = _gradients(parameters, sparse)
    if not grads:
        return torch.zeros(())
    return device_ops.grad_norm(grads, scale=scale)
