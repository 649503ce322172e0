"""A sequence encoder of linear cost for the beads of long chains (no
counterpart in the reference, as ChainEncoder).

In place of attention, whose cost goes with a chain's length squared, a layer
carries a state along the chain by the gated delta rule, in one direction or
half of the heads in each; the residual stream is added where it is normed
(``rms_norm_add``).  ``ChainDeltaEncoder`` takes ChainEncoder's place in a
``ChainEmbedding``.  A chain that grows goes on from its states, a bead at a time
(``step``).

``gated_delta``, ``rms_norm_add`` and ``scaled_embedding`` are the operators with
their gradients, on the HIP kernels; like the rest of the package they take GPU
tensors only, and they are differentiable once, in reverse mode.
"""

from __future__ import annotations

import math
from typing import List, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .. import ops
from .chain import CounterDropout, _needs_grad
from .mlp import init_xavier_uniform


def _once(backward):
    """once_differentiable's refusal of second derivatives, entered only where they
    are recorded: its wrapping takes about 5 us of a backward pass."""
    recorded = once_differentiable(backward)

    def either(ctx, *grads):
        return (recorded if torch.is_grad_enabled() else backward)(ctx, *grads)

    return either


class _GatedDelta(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, decay, beta, state, chains, scale, keep, reverse, normalize):
        args, scale, keep = ops._delta_args(q, k, v, decay, beta, chains, scale, keep)
        own = q.shape[2], v.shape[2]
        out, last, kept = ops._delta_forward(args, own, chains, scale, keep, state, reverse,
                                             normalize, True)
        q, qs, k, ks, v, vs, decay, beta, *dims = args
        ctx.save_for_backward(q, k, v, decay, beta, keep, kept)
        ctx.arrays = (dims, kept.shape, (q.stride(), k.stride(), v.stride()), (qs, ks, vs))
        ctx.plan = (own, chains, scale, reverse, normalize)
        ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    @_once
    def backward(ctx, grad, grad_last):
        if grad is None and grad_last is None:
            return (None,) * 11
        own, chains, scale, reverse, normalize = ctx.plan
        args, keep, kept = ops._delta_saved(ctx.saved_tensors, ctx.arrays, chains)
        if grad is None:
            v = args[4]
            grad = torch.zeros(*v.shape[:2], own[1], dtype=v.dtype, device=v.device)
        grads = ops._delta_backward(args, own, chains, kept, grad, grad_last, scale, keep, reverse,
                                    normalize, ctx.needs_input_grad[5])
        return (*grads, None, None, None, None, None)


def gated_delta(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, decay: torch.Tensor,
                beta: torch.Tensor, chains: ops.ChainLayout, scale: Optional[float] = None,
                keep: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
                reverse: bool = False, normalize: bool = True
                ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out, last) of ops.gated_delta with gradients for q, k, v, decay, beta and
    state."""
    if not _needs_grad(q, k, v, decay, beta, state):
        return ops.gated_delta(q, k, v, decay, beta, chains, scale, keep, state, reverse,
                               normalize)[:2]
    return _GatedDelta.apply(q, k, v, decay, beta, state, chains, scale, keep, reverse, normalize)


class _RMSNormAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, t, rstd = ops.rms_norm_add(x, residual, weight, eps)
        ctx.save_for_backward(t, weight, rstd)
        ctx.set_materialize_grads(False)
        return y, t

    @staticmethod
    @_once
    def backward(ctx, grad, grad_t):
        t, weight, rstd = ctx.saved_tensors
        if grad is None and grad_t is None:
            return None, None, None, None
        if grad is None:
            grad = torch.zeros(t.shape, dtype=weight.dtype, device=t.device)
        return (*ops._rms_backward(grad, grad_t, t, weight, rstd), None)


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        y, _, rstd = ops.rms_norm_add(x, None, weight, eps)
        ctx.save_for_backward(x, weight, rstd)
        return y

    @staticmethod
    @_once
    def backward(ctx, grad):
        x, weight, rstd = ctx.saved_tensors
        dx, _, dw = ops._rms_backward(grad, None, x, weight, rstd)
        return dx, dw, None


def rms_norm_add(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor,
                 eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, t) of ops.rms_norm_add with gradients for x, residual and weight; t
    is x itself without a residual."""
    if not _needs_grad(x, residual, weight):
        return ops.rms_norm_add(x, residual, weight, eps)[:2]
    if residual is None:
        return _RMSNorm.apply(x, weight, eps), x
    return _RMSNormAdd.apply(x, residual, weight, eps)


class _ScaledEmbedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, scale):
        ctx.save_for_backward(tokens)
        ctx.plan = (table.shape[0], scale)
        return ops.scaled_embedding(table, tokens, scale)

    @staticmethod
    @_once
    def backward(ctx, grad):
        tokens, = ctx.saved_tensors
        rows, scale = ctx.plan
        order = ops.token_order(tokens, rows)
        return ops.scaled_embedding_backward(grad, order, scale), None, None


def scaled_embedding(table: torch.Tensor, tokens: torch.Tensor, scale: float = 1.0
                     ) -> torch.Tensor:
    """ops.scaled_embedding with a gradient for the table, summed by sorted
    tokens."""
    if not _needs_grad(table):
        return ops.scaled_embedding(table, tokens, scale)
    return _ScaledEmbedding.apply(table, tokens, scale)


class RMSNormAdd(torch.nn.Module):
    """forward(x [N, width], residual=None) -> (norm of x + residual times a
    weight, x + residual): the first in x's type, the second in the residual's."""

    def __init__(self, width: int, eps: float = 1e-6):
        super().__init__()
        self.eps = eps
        self.weight = torch.nn.Parameter(torch.ones(width))

    def reset_parameters(self):
        torch.nn.init.ones_(self.weight)

    def forward(self, x, residual=None):
        return rms_norm_add(x, residual, self.weight.to(x.dtype), self.eps)


class ChainDelta(torch.nn.Module):
    """The gated delta rule along every chain: projections to queries, keys and
    values (``key_heads`` of the first two serve ``heads`` of the values), to the
    decay and to the strength of every bead and head, and back.  With
    ``bidirectional`` the second half of the heads goes through the chains from
    their last beads.

    forward(x [S, width], chains, keep=None) -> [S, width];
    step(x [B, width], state) -> [B, width], a bead each for B chains whose states
    (``new_state(B)`` at their beginning) it moves on, in one direction only."""

    def __init__(self, width: int, heads: int, key_heads: Optional[int] = None,
                 key_dim: Optional[int] = None, bidirectional: bool = True):
        super().__init__()
        key_heads = heads if key_heads is None else key_heads
        parts = 2 if bidirectional else 1
        if (width % heads != 0 or not 1 <= key_heads <= heads or heads % key_heads != 0
                or heads % parts != 0 or key_heads % parts != 0):
            raise ValueError(f"{width} channels cannot be split into {heads} heads with "
                             f"{key_heads} key heads, in {parts} direction(s)")
        self.heads, self.key_heads, self.parts = heads, key_heads, parts
        self.dim = width // heads
        self.key_dim = self.dim if key_dim is None else key_dim
        if not (1 <= self.dim <= ops.MAX_DELTA_DIM and 1 <= self.key_dim <= ops.MAX_DELTA_DIM):
            raise ValueError(f"heads have 1 .. {ops.MAX_DELTA_DIM} channels, got {self.dim} and "
                             f"{self.key_dim}")
        self.qkv = torch.nn.Linear(width, 2 * key_heads * self.key_dim + width)
        self.gates = torch.nn.Linear(width, 2 * heads)
        self.out = torch.nn.Linear(width, width)
        self.rate = torch.nn.Parameter(torch.empty(heads))  # log of the decay's factor
        self.reset_parameters()

    def reset_parameters(self):
        for m in (self.qkv, self.gates, self.out):
            init_xavier_uniform(m)
        # memories of about 3 to 700 beads
        with torch.no_grad():
            self.rate.copy_(torch.linspace(math.log(0.5), math.log(0.002), self.heads))

    def _project(self, x):
        n, kd = self.key_heads, self.key_dim
        q, k, v = self.qkv(x).split([n * kd, n * kd, self.heads * self.dim], 1)
        gates = self.gates(x).float()
        decay = -torch.nn.functional.softplus(gates[:, :self.heads]) * torch.exp(
            self.rate.float())
        beta = torch.sigmoid(gates[:, self.heads:])
        return (q.unflatten(1, (n, kd)), k.unflatten(1, (n, kd)),
                v.unflatten(1, (self.heads, self.dim)), decay, beta)

    def forward(self, x, chains, keep=None):
        q, k, v, decay, beta = self._project(x)
        n, h = self.key_heads // self.parts, self.heads // self.parts
        y = [gated_delta(q[:, i * n:(i + 1) * n], k[:, i * n:(i + 1) * n],
                         v[:, i * h:(i + 1) * h], decay[:, i * h:(i + 1) * h],
                         beta[:, i * h:(i + 1) * h], chains, keep=keep, reverse=i == 1)[0]
             for i in range(self.parts)]
        return self.out((y[0] if self.parts == 1 else torch.cat(y, 1)).flatten(1))

    def new_state(self, batch: int) -> torch.Tensor:
        return torch.zeros(batch, self.heads, self.key_dim, self.dim, dtype=torch.float32,
                           device=self.rate.device)

    @torch.no_grad()
    def step(self, x, state):
        if self.parts != 1:
            raise RuntimeError("a chain that is read from both ends cannot grow")
        y = ops.gated_delta_step(*self._project(x), state)
        return self.out(y.flatten(1))


class ChainDeltaLayer(torch.nn.Module):
    """A step of a residual stream t: x = delta(norm(t += x)), then
    x = lin(silu(lin(norm(t += x)))).  forward(x, t, chains, keep) -> (x, t), where
    x is still to be added (t is None before the first layer)."""

    def __init__(self, width: int, heads: int, key_heads: Optional[int] = None,
                 key_dim: Optional[int] = None, hidden: Optional[int] = None,
                 dropout: float = 0.0, seed: int = 0, bidirectional: bool = True):
        super().__init__()
        hidden = 2 * width if hidden is None else hidden
        self.norm1 = RMSNormAdd(width)
        self.delta = ChainDelta(width, heads, key_heads, key_dim, bidirectional)
        self.drop1 = CounterDropout(dropout, 2 * seed)
        self.norm2 = RMSNormAdd(width)
        self.lin1 = torch.nn.Linear(width, hidden)
        self.lin2 = torch.nn.Linear(hidden, width)
        self.drop2 = CounterDropout(dropout, 2 * seed + 1)
        self.reset_parameters()

    def reset_parameters(self):
        for m in (self.norm1, self.delta, self.norm2):
            m.reset_parameters()
        init_xavier_uniform(self.lin1)
        init_xavier_uniform(self.lin2)

    def _mlp(self, x, t):
        y, t = self.norm2(x, t)
        return self.lin2(torch.nn.functional.silu(self.lin1(y))), t

    def forward(self, x, t, chains, keep=None):
        y, t = self.norm1(x, t)
        x, t = self._mlp(self.drop1(self.delta(y, chains, keep)), t)
        return self.drop2(x), t

    @torch.no_grad()
    def step(self, x, t, state):
        y, t = self.norm1(x, t)
        return self._mlp(self.delta.step(y, state), t)


class ChainDeltaEncoder(torch.nn.Module):
    """ChainDeltaLayers in a row and a last norm: features [S, width] of the beads
    of all chains to features that depend on their place in the sequence, as
    ChainEncoder, at a cost that goes with the chains' lengths.  ``seed`` begins
    the layers' dropout streams.

    step(x [B, width], states): the features of one more bead for each of B chains,
    read in one direction (``bidirectional=False``); ``new_states(B)`` is where
    chains begin."""

    def __init__(self, width: int, layers: int, heads: int, seed: int = 0, **layer_options):
        super().__init__()
        if layers < 1:
            raise ValueError("At least one encoder layer must be specified")
        self.layers = torch.nn.ModuleList(
            ChainDeltaLayer(width, heads, seed=seed + i, **layer_options)
            for i in range(layers))
        self.norm = RMSNormAdd(width)

    def reset_parameters(self):
        for layer in self.layers:
            layer.reset_parameters()
        self.norm.reset_parameters()

    def forward(self, x, chains, keep=None, positions=None):
        if positions is not None:
            raise RuntimeError("ChainDeltaEncoder has no use for positions: the rule goes by the "
                               "beads' order")
        t = None
        for layer in self.layers:
            x, t = layer(x, t, chains, keep)
        return self.norm(x, t)[0]

    def new_states(self, batch: int) -> List[torch.Tensor]:
        return [layer.delta.new_state(batch) for layer in self.layers]

    @torch.no_grad()
    def step(self, x, states):
        t = None
        for layer, state in zip(self.layers, states):
            x, t = layer.step(x, t, state)
        return self.norm(x, t)[0]
