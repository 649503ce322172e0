"""Host side of the sequence encoder: chain layouts, bucket tables, the
refusal of CPU tensors, and the float64 oracle against independent forms
(torch's own attention gradients, group norm, published Philox vectors)."""

import math

import numpy as np
import pytest
import torch

from mlcg_amd import nn, ops
from oracle import chain_ref as R


@pytest.mark.parametrize("lens", [[], [0], [1], [3, 0, 70, 33], [32, 64, 256, 257, 0, 1],
                                  [1000] * 3 + [5] * 40])
def test_chain_layout(lens):
    c = ops.chain_layout(lens, "cpu")
    assert c.lengths == tuple(lens) and c.n_beads == sum(lens) and c.n_chains == len(lens)
    assert c.ptr.tolist() == [0, *np.cumsum(lens).astype(int).tolist()]
    for rows in ops.CHAIN_TILE_ROWS:
        t = c.tiles[rows]
        assert t.shape == (sum(-(-n // rows) for n in lens), 4) and t.is_contiguous()
        seen = {}
        for i, (first, n, at, chain) in enumerate(t.tolist()):
            assert first == sum(lens[:chain]) and n == lens[chain] and at % rows == 0 and at < n
            if at == 0:
                assert c.first[rows][chain] == i
            else:  # a chain's tiles one after the other
                assert seen[chain] == (i - 1, at - rows)
            seen[chain] = (i, at)
        lengths = [n for _, n, _, _ in t.tolist()]
        assert lengths == sorted(lengths, reverse=True)  # the longest chains first
        for chain, n in enumerate(lens):
            assert n > 0 or c.first[rows][chain] == -1


def test_chain_layout_sources_and_refusals():
    a = ops.chain_layout(torch.tensor([4, 5]), "cpu")
    assert a.lengths == ops.chain_layout(np.array([4, 5], dtype=np.int32), "cpu").lengths
    for bad in ([-1], [1.5], [[1, 2]], torch.tensor([1.0]), torch.tensor([True]), [2 ** 31]):
        with pytest.raises(RuntimeError):
            ops.chain_layout(bad, "cpu")


@pytest.mark.parametrize("buckets,reach", [(2, 1), (8, 4), (16, 3), (32, 128), (47, 100),
                                           (64, 1024)])
def test_log_buckets(buckets, reach):
    t = ops.relative_bucket_table(buckets, reach, "log")
    side = buckets // 2
    assert len(t) == 2 * reach + 1 and t[reach] == 0
    back, ahead = t[reach::-1], t[reach + 1:]
    assert all(0 <= b < side for b in back) and all(side <= b < 2 * side for b in ahead)
    assert back == sorted(back) and ahead == sorted(ahead)
    assert [b + side for b in back[1:]] == ahead  # the same scheme both ways
    exact = max(1, side // 2)
    assert back[:exact] == list(range(exact))[:reach + 1]
    if reach > exact:
        assert back[-1] == side - 1


def test_bucket_tables_and_refusals():
    b = ops.relative_buckets(5, 2, "clip", device="cpu")
    assert b.bucket_of.tolist() == b.order.tolist() == [0, 1, 2, 3, 4]
    b = ops.relative_buckets(4, 2, [3, 0, 0, 1, 3], device="cpu")
    assert b.order.tolist() == [1, 2, 3, 0, 4] and b.first.tolist() == [0, 2, 3, 3, 5]
    for args in ((4, 2, "clip"), (1, 4, "log"), (8, 0, "log"), (8, 1025, "log"), (8, 4, "exp"),
                 (4, 2, [0, 1, 2, 3]), (4, 2, [0, 1, 2, 3, 4]), (4, 2, [0, 1, -1, 3, 3])):
        with pytest.raises(RuntimeError):
            ops.relative_buckets(*args, device="cpu")


def test_cpu_tensors_are_refused():
    c = ops.chain_layout([3], "cpu")
    b = ops.relative_buckets(8, 4, device="cpu")
    q, table = torch.zeros(3, 2, 16), torch.zeros(8, 2)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        nn.chain_attention(q, q, q, table, b, c)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        nn.group_norm_act(torch.zeros(3, 4), torch.ones(4), torch.ones(4), 2, c)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        nn.dropout_add(torch.zeros(4), 0.5, 1, 1)


def test_dropout_threshold():
    assert ops.dropout_threshold(0.0) == 0 and ops.dropout_threshold(0.5) == 32768
    assert ops.dropout_threshold(1.0 - 1e-9) == 65535
    for p in (1.0, -0.1, math.nan, "0.5"):
        with pytest.raises(RuntimeError):
            ops.dropout_threshold(p)


def test_philox_published_vectors():
    """The known-answer vectors that the generator's authors publish."""
    f = 0xFFFFFFFF
    assert R.philox4x32([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert R.philox4x32([f] * 4, [f] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert R.philox4x32([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344],
                        [0xA4093822, 0x299F31D0]) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420,
                                                      0x24126EA1]


def test_attention_oracle_against_autograd():
    g = torch.Generator().manual_seed(0)
    lens, heads, kv, dim = [7, 12], 4, 2, 5
    q = torch.randn(19, heads, dim, generator=g, dtype=torch.float64, requires_grad=True)
    k, v = (torch.randn(19, kv, dim, generator=g, dtype=torch.float64, requires_grad=True)
            for _ in range(2))
    bucket = ops.relative_bucket_table(8, 3, "log")
    table = torch.randn(8, heads, generator=g, dtype=torch.float64, requires_grad=True)
    keep = torch.rand(19, generator=g) < 0.7
    grad = torch.randn(19, heads, dim, generator=g, dtype=torch.float64)
    outs, at = [], 0
    for n in lens:
        r = slice(at, at + n)
        at += n
        d = (torch.arange(n)[None, :] - torch.arange(n)[:, None]).clamp(-3, 3) + 3
        bias = table[torch.tensor(bucket)[d]].permute(2, 0, 1)
        kk, vv = (t[r].repeat_interleave(heads // kv, 1).transpose(0, 1) for t in (k, v))
        logit = q[r].transpose(0, 1) @ kk.transpose(1, 2) / math.sqrt(dim) + bias
        logit = logit.masked_fill(~keep[r][None, None], -math.inf)
        outs.append((torch.softmax(logit, 2) @ vv).transpose(0, 1))
    out = torch.cat(outs)
    want = dict(zip(("q", "k", "v", "table"),
                    torch.autograd.grad(out, (q, k, v, table), grad)), out=out.detach())
    got, _ = R.attention(q, k, v, table, bucket, lens, keep=keep, grad=grad)
    for name, t in want.items():
        assert torch.allclose(got[name], t, rtol=1e-11, atol=1e-12), name


@pytest.mark.parametrize("act", ["none", "tanh", "ssp", "silu"])
def test_group_norm_oracle_against_autograd(act):
    g = torch.Generator().manual_seed(1)
    lens, width, groups = [5, 8], 12, 3
    x = torch.randn(13, width, generator=g, dtype=torch.float64, requires_grad=True)
    w, b = (torch.randn(width, generator=g, dtype=torch.float64, requires_grad=True)
            for _ in range(2))
    grad = torch.randn(13, width, generator=g, dtype=torch.float64)
    f = {"none": lambda z: z, "tanh": torch.tanh, "silu": torch.nn.functional.silu,
         "ssp": nn.ShiftedSoftplus()}[act]
    outs, at = [], 0
    for n in lens:
        t = x[at:at + n].t().reshape(1, width, n)  # torch's has the channels first
        at += n
        outs.append(f(torch.nn.functional.group_norm(t, groups, w, b))[0].t())
    out = torch.cat(outs)
    want = dict(zip(("x", "weight", "bias"), torch.autograd.grad(out, (x, w, b), grad)),
                out=out.detach())
    got = R.group_norm(x, w, b, groups, lens, act=act, grad=grad)
    for name, t in want.items():
        assert torch.allclose(got[name], t, rtol=1e-9, atol=1e-10), name
