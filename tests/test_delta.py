"""Host side of the encoder of linear cost: the float64 oracle against autograd,
the refusals that need no GPU, and what the modules take."""

import math

import pytest
import torch

from mlcg_amd import nn, ops
from oracle import delta_ref as R


def _autograd_delta(q, k, v, decay, beta, lengths, keep, state, reverse, normalize):
    """The rule with torch's operations, bead by bead."""
    group = v.shape[1] // q.shape[1]
    if normalize:
        q, k = (t / torch.sqrt((t * t).sum(2, keepdim=True) + R.EPS) for t in (q, k))
    q, k = (t.repeat_interleave(group, 1) for t in (q, k))
    rows, last, begin = {}, [], 0
    for b, n in enumerate(lengths):
        S = state[b]
        for t in sorted(range(begin, begin + n), reverse=reverse):
            if keep is None or keep[t]:
                S = torch.exp(decay[t])[:, None, None] * S
                u = beta[t][:, None] * (v[t] - torch.matmul(k[t].unsqueeze(1), S).squeeze(1))
                S = S + k[t].unsqueeze(2) * u.unsqueeze(1)
            rows[t] = torch.matmul(q[t].unsqueeze(1), S).squeeze(1) / math.sqrt(q.shape[2])
        last.append(S)
        begin += n
    return torch.stack([rows[t] for t in range(begin)]), torch.stack(last)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("normalize", [False, True])
def test_delta_oracle_against_autograd(normalize, reverse):
    g = torch.Generator().manual_seed(0)
    lens, heads, keys, dk, dv = [7, 0, 12], 4, 2, 5, 3

    def randn(*shape):
        return torch.randn(*shape, generator=g, dtype=torch.float64).requires_grad_(True)

    q, k, v = randn(19, keys, dk), randn(19, keys, dk), randn(19, heads, dv)
    decay = (-torch.rand(19, heads, generator=g, dtype=torch.float64)).requires_grad_(True)
    beta, state = randn(19, heads), randn(3, heads, dk, dv)
    keep = torch.rand(19, generator=g) < 0.7
    grad, grad_last = randn(19, heads, dv).detach(), randn(3, heads, dk, dv).detach()
    out, last = _autograd_delta(q, k, v, decay, beta, lens, keep, state, reverse, normalize)
    leaves = dict(q=q, k=k, v=v, decay=decay, beta=beta, state=state)
    want = dict(zip(leaves, torch.autograd.grad([out, last], list(leaves.values()),
                                                [grad, grad_last])), out=out, last=last)
    got = R.gated_delta(q, k, v, decay, beta, lens, None, keep, state, reverse, normalize, grad,
                        grad_last)
    for name, t in want.items():
        assert torch.allclose(got[name], t.detach(), rtol=1e-10, atol=1e-11), name


def test_rms_and_embedding_oracles_against_autograd():
    g = torch.Generator().manual_seed(1)
    x, r = (torch.randn(6, 11, generator=g, dtype=torch.float64).requires_grad_(True)
            for _ in range(2))
    w = torch.randn(11, generator=g, dtype=torch.float64).requires_grad_(True)
    gy, gt = (torch.randn(6, 11, generator=g, dtype=torch.float64) for _ in range(2))
    t = x + r
    y = t / torch.sqrt((t * t).mean(1, keepdim=True) + 1e-6) * w
    dx, dr, dw = torch.autograd.grad([y, t], [x, r, w], [gy, gt])
    got = R.rms_norm_add(x, r, w, grad=gy, grad_t=gt)
    assert torch.allclose(dx, dr)
    for a, b in ((got["y"], y), (got["t"], t), (got["x"], dx), (got["weight"], dw)):
        assert torch.allclose(a, b.detach(), rtol=1e-11, atol=1e-12)
    tokens = torch.randint(0, 6, (30,), generator=g)
    grad = torch.randn(30, 11, generator=g, dtype=torch.float64)
    out = 1.5 * torch.nn.functional.embedding(tokens, x)
    got = R.scaled_embedding(x, tokens, 1.5, grad)
    assert torch.allclose(got["out"], out.detach())
    assert torch.allclose(got["table"], torch.autograd.grad(out, x, grad)[0])


def test_cpu_tensors_are_refused():
    c = ops.chain_layout([3], "cpu")
    q, g = torch.zeros(3, 2, 16), torch.zeros(3, 2)
    calls = [lambda: nn.gated_delta(q, q, q, g, g, c),
             lambda: ops.gated_delta_step(q, q, q, g, g, torch.zeros(3, 2, 16, 16)),
             lambda: nn.rms_norm_add(torch.zeros(3, 4), None, torch.ones(4)),
             lambda: nn.rms_norm_add(torch.zeros(3, 4), torch.zeros(3, 4), torch.ones(4)),
             lambda: nn.scaled_embedding(torch.zeros(3, 4), torch.zeros(2, dtype=torch.int64)),
             lambda: ops.token_order(torch.zeros(2, dtype=torch.int64), 3),
             lambda: ops.scaled_embedding_backward(
                 torch.zeros(2, 4), ops.TokenOrder(torch.zeros(2, dtype=torch.int32),
                                                   torch.zeros(2, dtype=torch.int32), 3))]
    for f in calls:
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            f()


def test_step_has_no_gradients():
    q, g = torch.zeros(3, 2, 16), torch.zeros(3, 2)
    with pytest.raises(RuntimeError, match="no_grad"):
        ops.gated_delta_step(q.requires_grad_(True), q, q, g, g, torch.zeros(3, 2, 16, 16))


@pytest.mark.parametrize("lengths,chunks", [([1], 0), ([64, 0, 65, 700], 0), ([700, 3, 129], 4),
                                            ([64 * 8], 4), ([0, 0, 5], 3)])
def test_segments(monkeypatch, lengths, chunks):
    """Segments cover every chunk once, a chain's in order, its first and last
    marked."""
    monkeypatch.setattr(ops, "_delta_segment_tiles", lambda *a: chunks)
    c = ops.chain_layout(lengths, "cpu")
    plan = ops._delta_plan(c, 4)
    assert plan.split == (chunks > 0)
    segs, first = plan.segments.tolist(), plan.first.tolist()
    assert first[-1] == len(segs) and len(first) == 1 + sum(n > 0 for n in lengths)
    tiles = c.tiles[ops.DELTA_ROWS].tolist()
    seen = []
    for a, b in zip(first, first[1:]):
        chain = segs[a][0]
        assert segs[a][3] & 1 and segs[b - 1][3] & 2
        assert all(not s[3] & 1 for s in segs[a + 1:b]) and all(not s[3] & 2 for s in segs[a:b - 1])
        at = c.first[ops.DELTA_ROWS][chain]
        for s in segs[a:b]:
            assert s[0] == chain and s[1] == at and s[2] >= 1
            assert chunks == 0 or s[2] <= chunks
            seen += range(s[1], s[1] + s[2])
            at += s[2]
        assert all(tiles[t][3] == chain for t in range(segs[a][1], at))
    assert sorted(seen) == list(range(len(tiles)))


def test_modules_refuse():
    for args in ((30, 4), (32, 4, 3), (32, 3), (32, 2, 1), (32, 4, 0)):
        with pytest.raises(ValueError):
            nn.ChainDelta(*args)
    with pytest.raises(ValueError):
        nn.ChainDelta(256, 1, bidirectional=False)  # 256 channels a head
    with pytest.raises(ValueError):
        nn.ChainDelta(32, 2, key_dim=129)
    with pytest.raises(ValueError):
        nn.ChainDeltaEncoder(32, 0, 2)
    both = nn.ChainDelta(32, 2)
    with pytest.raises(RuntimeError, match="both ends"):
        both.step(torch.zeros(1, 32), both.new_state(1))
    enc = nn.ChainDeltaEncoder(32, 1, 2)
    with pytest.raises(RuntimeError, match="positions"):
        enc(torch.zeros(3, 32), ops.chain_layout([3], "cpu"), None,
            torch.zeros(3, dtype=torch.int32))


def test_embedding_without_a_factor_is_torchs():
    """ChainEmbedding's look-up with scale None, as it always was."""
    class Same(torch.nn.Module):
        def forward(self, x, chains, keep=None, positions=None):
            return x

    e = nn.ChainEmbedding(4, 8, Same(), [0, 1, 3, 1], (3, 1))
    assert torch.equal(e.table(), e.weight[torch.tensor([0, 1, 3, 1])])
    assert nn.ChainEmbedding(4, 8, Same(), [0, 1], (2,), scale=2).scale == 2.0
