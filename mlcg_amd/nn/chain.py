"""A sequence encoder for the beads of chains: embeddings that depend on where
in its chain a bead sits (no counterpart in the reference, whose embedding
layer knows a bead's type alone, mlcg/nn/schnet.py:419-440).

The encoder works on the chains, not on their positions: a table of
features, one row for every bead (site) of a set of molecules, which takes
the place of SchNet's embedding table (``ChainEmbedding``; ``atom_types`` then
holds the beads' sites).  A force-matching step differentiates through it once,
from the table's gradient, and a simulation evaluates it once
(``ChainEmbedding.as_embedding``).

``chain_attention``, ``group_norm_act`` and ``dropout_add`` are the operators
with their gradients, on the HIP kernels; like the rest of the package they
take GPU tensors only, and they are differentiable once.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import ops
from .mlp import init_xavier_uniform


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, buckets, chains, scale, keep, positions):
        out, lse = ops.chain_attention(q, k, v, table, buckets, chains, scale, keep, positions,
                                       want_lse=True)
        ctx.save_for_backward(q, k, v, table, out, lse, keep, positions)
        ctx.plan = (buckets, chains, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, table, out, lse, keep, positions = ctx.saved_tensors
        buckets, chains, scale = ctx.plan
        dq, dk, dv, dt = ops.chain_attention_backward(q, k, v, table, buckets, chains, out, lse,
                                                      grad, scale, keep, positions)
        return dq, dk, dv, dt, None, None, None, None, None


def _needs_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def chain_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor,
                    buckets: ops.RelativeBuckets, chains: ops.ChainLayout,
                    scale: Optional[float] = None, keep: Optional[torch.Tensor] = None,
                    positions: Optional[torch.Tensor] = None) -> torch.Tensor:
    """ops.chain_attention with gradients for q, k, v and table."""
    if not _needs_grad(q, k, v, table):
        return ops.chain_attention(q, k, v, table, buckets, chains, scale, keep, positions)[0]
    return _Attention.apply(q, k, v, table, buckets, chains, scale, keep, positions)


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, chains, eps, act):
        y, stats = ops.group_norm_act(x, weight, bias, groups, chains, eps, act)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.plan = (groups, chains, act)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, bias, stats = ctx.saved_tensors
        groups, chains, act = ctx.plan
        dx, dw, db = ops.group_norm_act_backward(x, weight, bias, groups, chains, stats, grad, act)
        return dx, dw, db, None, None, None, None


def group_norm_act(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, groups: int,
                   chains: ops.ChainLayout, eps: float = 1e-5, act: str = "none") -> torch.Tensor:
    """ops.group_norm_act with gradients for x, weight and bias."""
    if not _needs_grad(x, weight, bias):
        return ops.group_norm_act(x, weight, bias, groups, chains, eps, act)[0]
    return _GroupNorm.apply(x, weight, bias, groups, chains, eps, act)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, step):
        ctx.plan = (p, seed)
        if isinstance(step, torch.Tensor):
            ctx.save_for_backward(step)
        ctx.step = None if isinstance(step, torch.Tensor) else step
        return ops.dropout_add(x, p, seed, step, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        p, seed = ctx.plan
        dx = None
        if ctx.needs_input_grad[0]:
            step = ctx.saved_tensors[0] if ctx.step is None else ctx.step
            dx = ops.dropout_add(grad, p, seed, step)
        return dx, grad if ctx.needs_input_grad[1] else None, None, None, None


def dropout_add(x: torch.Tensor, p: float, seed: int, step,
                residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """ops.dropout_add with gradients for x and residual.  The backward pass
    draws the same mask again: a step that lives on the device must keep its
    value until then (changing it in between is an error)."""
    if not _needs_grad(x, residual):
        return ops.dropout_add(x, p, seed, step, residual)
    return _Dropout.apply(x, residual, p, seed, step)
