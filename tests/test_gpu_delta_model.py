"""The encoder of linear cost as it is used: a run of its operators together, in
a ChainEmbedding before SchNet, under autocast, bead by bead, and recorded."""

import pytest
import torch

pytestmark = pytest.mark.gpu

LENS = [35, 1, 162, 20]


def _encoder(seed=3, **options):
    from mlcg_amd import nn

    torch.manual_seed(seed)
    enc = nn.ChainDeltaEncoder(64, 2, 4, **options)
    with torch.no_grad():
        for name, p in enc.named_parameters():
            if name.endswith("bias") or "norm" in name:
                p.add_(0.3 * torch.randn_like(p))
    return enc.cuda()


def _plain_rule(q, k, v, decay, beta, chains, keep=None, reverse=False, **_):
    """The rule with torch's operations in the arrays' type, all chains at once."""
    group = v.shape[1] // q.shape[1]
    q, k = (t / torch.sqrt((t * t).sum(2, keepdim=True) + 1e-6) for t in (q, k))
    q, k = (t.repeat_interleave(group, 1) for t in (q, k))
    rows, begin = [], 0
    for n in chains.lengths:
        S, out = v.new_zeros(v.shape[1], q.shape[2], v.shape[2]), {}
        for t in sorted(range(begin, begin + n), reverse=reverse):
            if keep is None or keep[t]:
                S = torch.exp(decay[t])[:, None, None] * S
                u = beta[t][:, None] * (v[t] - torch.matmul(k[t].unsqueeze(1), S).squeeze(1))
                S = S + k[t].unsqueeze(2) * u.unsqueeze(1)
            out[t] = torch.matmul(q[t].unsqueeze(1), S).squeeze(1) * q.shape[2] ** -0.5
        rows += [out[t] for t in range(begin, begin + n)]
        begin += n
    return torch.stack(rows), None


def _plain_norm(x, residual, weight, eps=1e-6):
    t = x if residual is None else x + residual
    return t / torch.sqrt((t * t).mean(1, keepdim=True) + eps) * weight, t


def _step(enc, x, grad, chains, keep=None):
    x = x.detach().requires_grad_(True)
    out = enc(x, chains, keep)
    return [out.detach(), *torch.autograd.grad(out, [x, *enc.parameters()], grad.to(out.dtype))]


@pytest.mark.parametrize("options", [{}, dict(bidirectional=False, key_heads=2, key_dim=24)])
def test_encoder_against_plain_operations(monkeypatch, options):
    """The whole encoder, forward and backward, against the same modules on the
    rule's plain form in float64 on the CPU.  fp32: some thirty operations follow
    each other, each to a few 2^-24: 1e-5 of a tensor's norm."""
    from mlcg_amd import nn, ops
    from mlcg_amd.nn import delta

    g = torch.Generator().manual_seed(0)
    enc = _encoder(**options)
    n = sum(LENS)
    x, grad = torch.randn(n, 64, generator=g), torch.randn(n, 64, generator=g)
    keep = torch.rand(n, generator=g) < 0.9
    got = _step(enc, x.cuda(), grad.cuda(), ops.chain_layout(LENS, "cuda"), keep.cuda())
    plain = nn.ChainDeltaEncoder(64, 2, 4, **options).double()
    plain.load_state_dict(enc.state_dict())
    monkeypatch.setattr(delta, "gated_delta", _plain_rule)
    monkeypatch.setattr(delta, "rms_norm_add", _plain_norm)
    # the gates are made in float32 by the module: here in float64
    monkeypatch.setattr(torch.Tensor, "float", lambda t: t)
    want = _step(plain, x.double(), grad.double(), ops.chain_layout(LENS, "cpu"), keep)
    for a, b in zip(got, want):
        d = float((a.cpu().double() - b).norm())
        assert d <= 1e-5 * float(b.norm()) + 1e-6, (tuple(a.shape), d, float(b.norm()))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dropout", [0.0, 0.2])
def test_autocast(dropout, dtype):
    """fp32 parameters under autocast: the 16-bit kernels run beside an fp32
    residual stream, the parameters' gradients are fp32.  About twenty roundings
    follow each other in two layers, forward and backward: 2^-8 sqrt(20) =
    1.7e-2 in the mean, of which some meet differences: 5e-2 (fp16: an eighth)."""
    from mlcg_amd import ops

    g = torch.Generator().manual_seed(1)
    n = sum(LENS)
    x, grad = torch.randn(n, 64, generator=g).cuda(), torch.randn(n, 64, generator=g).cuda()
    chains = ops.chain_layout(LENS, "cuda")
    want = _step(_encoder(dropout=dropout), x, grad, chains)
    with torch.autocast("cuda", dtype=dtype):
        got = _step(_encoder(dropout=dropout), x, grad, chains)
    assert all(t.dtype == torch.float32 for t in got[1:])
    for a, b in zip(got, want):
        d = float((a.double() - b.double()).norm())
        limit = 5e-2 if dtype == torch.bfloat16 else 5e-2 / 8
        assert d <= limit * float(b.double().norm()) + 1e-6, (tuple(a.shape), d)


def test_bead_by_bead():
    """A chain that grows: the features of every bead as the encoder gives them
    for the whole chain (fp32: as above, 1e-5 of the norm)."""
    from mlcg_amd import ops

    enc = _encoder(bidirectional=False).eval()
    x = torch.randn(3, 70, 64, device="cuda")
    with torch.no_grad():
        want = enc(x.flatten(0, 1), ops.chain_layout([70] * 3, "cuda")).view(3, 70, 64)
        states = enc.new_states(3)
        got = torch.stack([enc.step(x[:, t], states) for t in range(70)], 1)
    assert float((got - want).norm()) <= 1e-5 * float(want.norm())


def test_chain_embedding():
    """A ChainEmbedding on this encoder with a factor on the types' embeddings:
    the same as torch's look-up times the factor before the same encoder."""
    from mlcg_amd import nn

    torch.manual_seed(0)
    types = torch.randint(0, 8, (55,))
    enc = nn.ChainDeltaEncoder(128, 1, 4)
    a = nn.ChainEmbedding(8, 128, enc, types, (35, 20), scale=128 ** 0.5).cuda()
    sites = torch.randint(0, 55, (200,)).cuda()
    grad = torch.randn(200, 128, device="cuda")
    a(sites).backward(grad)
    got = [p.grad.clone() for p in a.parameters()]
    a.zero_grad()
    x = torch.nn.functional.embedding(types.cuda(), a.weight) * 128 ** 0.5
    out = a.encoder(x, a.chains, None, None).index_select(0, sites)
    assert float((out - a(sites)).norm()) <= 1e-6 * float(out.norm())
    out.backward(grad)
    for p, b in zip(a.parameters(), got):
        assert float((p.grad - b).norm()) <= 1e-5 * float(b.norm()) + 1e-6
    made = a.as_embedding()
    assert torch.equal(made.weight, a.table())
    # types that are loaded count, not those of an earlier call
    state = a.state_dict()
    state["types"] = (state["types"] + 1) % 8
    a.load_state_dict(state)
    a.zero_grad()
    a(sites).backward(grad)
    x = torch.nn.functional.embedding(a.types, a.weight.detach().requires_grad_(True))
    assert float((a.weight.grad - got[0]).norm()) > 1e-3 * float(got[0].norm())


def test_recorded_training_step():
    """Forward and backward of the encoder in one graph, replayed with other
    inputs between eager steps: the eager bits."""
    from mlcg_amd import ops

    enc = _encoder(dropout=0.0)
    chains = ops.chain_layout(LENS, "cuda")
    x, grad = torch.randn(sum(LENS), 64, device="cuda"), torch.randn(sum(LENS), 64, device="cuda")

    def work():
        leaf = x.detach().requires_grad_(True)
        out = enc(leaf, chains)
        return [out.detach(), *torch.autograd.grad(out, [leaf, *enc.parameters()], grad)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            work()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = work()
    torch.cuda.synchronize()
    for i in range(4):
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        want = work()
        for a, b in zip(outs, want):
            # the library's products may take another algorithm in a capture
            assert float((a - b).norm()) <= 1e-5 * float(b.norm()) + 1e-6, i


def test_training_moves_every_parameter():
    """A few steps on one batch: it runs, and no parameter is left without a
    gradient."""
    from mlcg_amd import ops

    enc = _encoder(dropout=0.1)
    chains = ops.chain_layout(LENS, "cuda")
    x, target = torch.randn(sum(LENS), 64, device="cuda"), torch.randn(sum(LENS), 64, device="cuda")
    opt = torch.optim.AdamW(enc.parameters(), lr=1e-3)
    before = [p.detach().clone() for p in enc.parameters()]
    for _ in range(3):
        opt.zero_grad()
        loss = (enc(x, chains) - target).square().mean()
        loss.backward()
        opt.step()
    assert bool(torch.isfinite(loss))
    for p, b in zip(enc.parameters(), before):
        assert bool(p.grad.any()) and not torch.equal(p.detach(), b)
