# SPDX-License-Identifier: MIT
"""Gradients that have no graph behind them: those that kernels compute."""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor


class _NoSecondGradient(torch.autograd.Function):
    @staticmethod
    def forward(ctx, operator: str, *grads: Tensor):
        ctx.operator = operator
        return tuple(g.view_as(g) for g in grads)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.operator} has no second derivatives here: its gradients cannot be differentiated")


def first_order(operator: str, grads: Tuple[Optional[Tensor], ...]) -> Tuple[Optional[Tensor], ...]:
    """`grads`, the result of an autograd backward. Where that backward is recorded
    (create_graph=True) they raise an error when they are differentiated; as constants they
    would drop their part of a second derivative without a word."""
    if not torch.is_grad_enabled():
        return grads
    some = iter(_NoSecondGradient.apply(operator, *(g.detach().requires_grad_(True) for g in grads if g is not None)))
    return tuple(g if g is None else next(some) for g in grads)
