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
take GPU tensors only, and they are differentiable once, in reverse mode.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import ops
from .mlp import init_xavier_uniform


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, buckets, chains, scale, keep, positions):
        rest = None if q.dtype == torch.float32 else torch.empty(q.shape, dtype=q.dtype,
                                                                 device=q.device)
        out, lse = ops.chain_attention(q, k, v, table, buckets, chains, scale, keep, positions,
                                       want_lse=True, rest=rest)
        ctx.save_for_backward(q, k, v, table, out, lse, keep, positions, rest)
        ctx.plan = (buckets, chains, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, table, out, lse, keep, positions, rest = ctx.saved_tensors
        buckets, chains, scale = ctx.plan
        dq, dk, dv, dt = ops.chain_attention_backward(q, k, v, table, buckets, chains, out, lse,
                                                      grad, scale, keep, positions, rest)
        return dq, dk, dv, dt, None, None, None, None, None


def _needs_grad(*tensors) -> bool:
    """Whether a call goes through its autograd function: for a gradient, or to be
    refused there where a tangent asks for a forward-mode derivative."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return True
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


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


class ChainAttention(torch.nn.Module):
    """Attention of every bead to the present beads of its chain: a projection
    to queries, keys and values (``kv_heads`` of the latter serve ``heads``
    query heads), a learned bias by relative position, a projection back.

    forward(x [S, width], chains, keep=None, positions=None) -> [S, width].
    The bias table takes the type of the projection, under autocast 16 bits."""

    def __init__(self, width: int, heads: int, kv_heads: Optional[int] = None,
                 num_buckets: int = 32, reach: int = 128, kind: str = "log"):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if width % heads != 0 or not 1 <= kv_heads <= heads or heads % kv_heads != 0:
            raise ValueError(f"{width} channels cannot be split into {heads} heads with "
                             f"{kv_heads} key/value heads")
        self.heads, self.kv_heads, self.dim = heads, kv_heads, width // heads
        self.qkv = torch.nn.Linear(width, (heads + 2 * kv_heads) * self.dim)
        self.out = torch.nn.Linear(width, width)
        self.bias_table = torch.nn.Parameter(torch.zeros(num_buckets, heads))
        buckets = ops.relative_buckets(num_buckets, reach, kind, device="cpu")
        self.num_buckets, self.reach = num_buckets, reach
        for name in ("bucket_of", "order", "first"):
            self.register_buffer(name, getattr(buckets, name), persistent=False)
        self.reset_parameters()

    def reset_parameters(self):
        init_xavier_uniform(self.qkv)
        init_xavier_uniform(self.out)
        torch.nn.init.zeros_(self.bias_table)

    @property
    def buckets(self) -> ops.RelativeBuckets:
        return ops.RelativeBuckets(num_buckets=self.num_buckets, reach=self.reach,
                                   bucket_of=self.bucket_of, order=self.order, first=self.first)

    def forward(self, x, chains, keep=None, positions=None):
        h, kv, d = self.heads, self.kv_heads, self.dim
        qkv = self.qkv(x).view(-1, h + 2 * kv, d)
        y = chain_attention(qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:],
                            self.bias_table.to(qkv.dtype), self.buckets, chains, keep=keep,
                            positions=positions)
        return self.out(y.reshape(-1, h * d))


class GroupNormAct(torch.nn.Module):
    """Group norm of every chain with an affine map by channel and an
    activation: forward(x [S, width], chains) -> [S, width], in x's type."""

    def __init__(self, groups: int, width: int, act: str = "none", eps: float = 1e-5):
        super().__init__()
        if width % groups != 0 or act not in ops.CHAIN_ACTS:
            raise ValueError(f"GroupNormAct: {width} channels in {groups} groups, act {act!r}")
        self.groups, self.act, self.eps = groups, act, eps
        self.weight = torch.nn.Parameter(torch.ones(width))
        self.bias = torch.nn.Parameter(torch.zeros(width))

    def reset_parameters(self):
        torch.nn.init.ones_(self.weight)
        torch.nn.init.zeros_(self.bias)

    def forward(self, x, chains):
        return group_norm_act(x, self.weight.to(x.dtype), self.bias.to(x.dtype), self.groups,
                              chains, self.eps, self.act)


class CounterDropout(torch.nn.Module):
    """residual + dropout(x), the mask drawn from (seed, step) and never
    stored.  The step is a buffer that every training call moves on, on the
    device: a recorded training step draws a new mask on every replay, and a
    run resumed from a checkpoint goes on with the next one.  Modules of one
    model need seeds of their own.  In eval mode: residual + x.  x may be in 16
    bits beside an fp32 residual, as under autocast."""

    def __init__(self, p: float, seed: int):
        super().__init__()
        ops.dropout_threshold(p)
        self.p, self.seed = p, seed
        self.register_buffer("step", torch.zeros(1, dtype=torch.int64))

    def forward(self, x, residual=None):
        if not self.training or self.p == 0.0:
            return x if residual is None else residual + x
        # the backward pass reads the value that this call used
        step = self.step.add_(1).clone()
        if residual is not None:
            x = x.to(residual.dtype)
        return dropout_add(x, self.p, self.seed, step, residual)


class ChainEncoderLayer(torch.nn.Module):
    """x + drop(attention(norm(x))), then x + drop(lin(act(norm(lin(x)))))."""

    def __init__(self, width: int, heads: int, kv_heads: Optional[int] = None,
                 hidden: Optional[int] = None, norm_groups: int = 8, act: str = "silu",
                 dropout: float = 0.0, seed: int = 0, num_buckets: int = 32, reach: int = 128,
                 kind: str = "log"):
        super().__init__()
        hidden = 2 * width if hidden is None else hidden
        self.norm1 = GroupNormAct(norm_groups, width)
        self.attention = ChainAttention(width, heads, kv_heads, num_buckets, reach, kind)
        self.drop1 = CounterDropout(dropout, 2 * seed)
        self.lin1 = torch.nn.Linear(width, hidden)
        self.norm2 = GroupNormAct(norm_groups, hidden, act)
        self.lin2 = torch.nn.Linear(hidden, width)
        self.drop2 = CounterDropout(dropout, 2 * seed + 1)
        self.reset_parameters()

    def reset_parameters(self):
        for m in (self.norm1, self.attention, self.norm2):
            m.reset_parameters()
        init_xavier_uniform(self.lin1)
        init_xavier_uniform(self.lin2)

    def forward(self, x, chains, keep=None, positions=None):
        y = self.attention(self.norm1(x, chains), chains, keep, positions)
        x = self.drop1(y, residual=x)
        y = self.lin2(self.norm2(self.lin1(x), chains))
        return self.drop2(y, residual=x)


class ChainEncoder(torch.nn.Module):
    """ChainEncoderLayers in a row: features [S, width] of the beads of all
    chains to features that depend on their place in the sequence.  ``seed``
    begins the layers' dropout streams."""

    def __init__(self, width: int, layers: int, heads: int, seed: int = 0, **layer_options):
        super().__init__()
        if layers < 1:
            raise ValueError("At least one encoder layer must be specified")
        self.layers = torch.nn.ModuleList(
            ChainEncoderLayer(width, heads, seed=seed + i, **layer_options)
            for i in range(layers))

    def reset_parameters(self):
        for layer in self.layers:
            layer.reset_parameters()

    def forward(self, x, chains, keep=None, positions=None):
        for layer in self.layers:
            x = layer(x, chains, keep, positions)
        return x


class ChainEmbedding(torch.nn.Module):
    """An embedding layer for SchNet whose rows are the beads (sites) of given
    molecules in place of bead types: row s is the encoder's feature of site s
    in its chain, made from the embeddings of the sites' types.  A batch's
    ``atom_types`` then holds the sites (0 .. S - 1) its beads are.

    types [S]: the sites' bead types, chain after chain; lengths: the beads of
    every chain; keep [S] bool: sites without a resolved structure; positions
    [S]: residue numbers (the index in the chain by default).  encoder: a
    ChainEncoder or a ChainDeltaEncoder.  scale: a factor on the types' embeddings;
    given, the look-up and its gradient go by scaled_embedding, which sums the
    sites of a type in a fixed order (None: torch's look-up, no factor).

    The table is made anew in every forward pass, as training needs it;
    ``as_embedding()`` gives it as a plain Embedding for simulations."""

    scale: Optional[float] = None  # of modules that were saved before it was theirs

    def __init__(self, embedding_size: int, width: int, encoder: torch.nn.Module, types, lengths,
                 keep=None, positions=None, scale: Optional[float] = None):
        super().__init__()
        self.scale = None if scale is None else float(scale)
        self.weight = torch.nn.Parameter(torch.empty(embedding_size, width))
        self.encoder = encoder
        self.register_buffer("types", torch.as_tensor(types, dtype=torch.int64))
        self.register_buffer("keep", None if keep is None else
                             torch.as_tensor(keep, dtype=torch.bool))
        self.register_buffer("positions", None if positions is None else
                             torch.as_tensor(positions, dtype=torch.int32))
        self.lengths = tuple(int(n) for n in lengths)
        n = self.types.numel()
        if self.types.dim() != 1 or sum(self.lengths) != n or any(
                t is not None and tuple(t.shape) != (n,) for t in (self.keep, self.positions)):
            raise ValueError("types, keep and positions hold one value for every bead of the "
                             "chains")
        if n and not 0 <= int(self.types.min()) <= int(self.types.max()) < embedding_size:
            raise ValueError("a site's type lies outside the embedding table")
        torch.nn.init.normal_(self.weight)

    def reset_parameters(self):
        torch.nn.init.normal_(self.weight)
        self.encoder.reset_parameters()

    @property
    def chains(self) -> ops.ChainLayout:
        """The chains' layout, on the device of the weights."""
        made = self.__dict__.get("_layout")
        if made is None or made.device != self.weight.device:
            made = self.__dict__["_layout"] = ops.chain_layout(self.lengths, self.weight.device)
        return made

    def __getstate__(self):
        state = dict(self.__dict__)
        state.pop("_layout", None)  # of one device, and made again where it is needed
        return state

    def table(self) -> torch.Tensor:
        if self.scale is None:
            x = torch.nn.functional.embedding(self.types, self.weight)
        else:
            from .delta import scaled_embedding

            x = scaled_embedding(self.weight, self.types, self.scale)
        return self.encoder(x, self.chains, self.keep, self.positions)

    def forward(self, sites: torch.Tensor) -> torch.Tensor:
        return self.table().index_select(0, sites)

    @torch.no_grad()
    def as_embedding(self) -> torch.nn.Embedding:
        """The present table as a plain embedding layer (without dropout)."""
        modes = [(m, m.training) for m in self.modules()]
        try:
            return torch.nn.Embedding.from_pretrained(self.eval().table().detach().clone(),
                                                      freeze=False)
        finally:
            for m, training in modes:
                m.training = training
