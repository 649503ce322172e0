"""The sequence encoder in use: ChainEncoder against a float64 model on the
CPU made of torch's own modules, ChainEmbedding as SchNet's embedding layer
against the same SchNet on a plain table, a recorded training step, and the
dropout's streams.

Tolerances: fp32 products of up to 256 terms in the linears and the
attention, two layers of them: 1e-5 of a tensor's largest element, as
elsewhere for fp32 against fp64 (gradients 1e-4)."""

import copy

import pytest
import torch

from tests.helpers import check, make_cfg, make_model

pytestmark = pytest.mark.gpu

LENS = [35, 1, 62, 20]


def _encoder(dropout=0.0, width=128, **more):
    from mlcg_amd import nn

    torch.manual_seed(3)
    enc = nn.ChainEncoder(width, 2, 4, kv_heads=2, num_buckets=16, reach=32, dropout=dropout,
                          **more)
    with torch.no_grad():
        for name, p in enc.named_parameters():
            if name.endswith("bias") or name.endswith("bias_table"):
                p.normal_(0.0, 0.3)
    return enc


def _reference(enc, x, lengths, keep, positions):
    """The encoder's formulas on torch's modules, chain by chain."""
    F = torch.nn.functional
    outs, at = [], 0
    for n in lengths:
        h = x[at:at + n]
        ok, pos = keep[at:at + n], positions[at:at + n].long()
        at += n
        for layer in enc.layers:
            a = layer.attention

            def norm(m, t):
                y = F.group_norm(t.t()[None], m.groups, m.weight, m.bias, m.eps)[0].t()
                return F.silu(y) if m.act == "silu" else y

            qkv = a.qkv(norm(layer.norm1, h)).view(n, -1, a.dim).transpose(0, 1)
            q, k, v = qkv.split([a.heads, a.kv_heads, a.kv_heads])
            k, v = (t.repeat_interleave(a.heads // a.kv_heads, 0) for t in (k, v))
            d = (pos[None, :] - pos[:, None]).clamp(-a.reach, a.reach) + a.reach
            bias = a.bias_table[a.bucket_of.long()[d]].permute(2, 0, 1)
            logit = (q @ k.transpose(1, 2)) * a.dim ** -0.5 + bias
            logit = logit.masked_fill(~ok[None, None, :], -torch.inf)
            y = (torch.softmax(logit, 2) @ v).transpose(0, 1).reshape(n, -1)
            h = h + a.out(y)
            h = h + layer.lin2(norm(layer.norm2, layer.lin1(h)))
        outs.append(h)
    return torch.cat(outs)


def test_encoder_against_float64():
    from mlcg_amd import ops

    enc = _encoder()
    s = sum(LENS)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(s, 128, generator=g)
    keep = torch.rand(s, generator=g) < 0.8
    keep[[0, 35, 36, 98]] = True  # a present bead in every chain
    positions = torch.cumsum((torch.rand(s, generator=g) < 0.5).int(), 0).to(torch.int32)
    grad = torch.randn(s, 128, generator=g)
    ref_enc = copy.deepcopy(enc).double()
    xr = x.double().requires_grad_(True)
    ref = _reference(ref_enc, xr, LENS, keep, positions)
    names = [n for n, _ in ref_enc.named_parameters()]
    ref_grads = torch.autograd.grad(ref, [xr, *ref_enc.parameters()], grad.double())
    enc = enc.cuda()
    xg = x.cuda().requires_grad_(True)
    out = enc(xg, ops.chain_layout(LENS, "cuda"), keep.cuda(), positions.cuda())
    check(out, ref.detach(), 1e-5, "encoder", atol_frac=1.0)
    grads = torch.autograd.grad(out, [xg, *enc.parameters()], grad.cuda())
    for name, a, b in zip(["x", *names], grads, ref_grads):
        check(a, b, 1e-4, name, atol_frac=1.0)


def _embedding(lengths, dropout=0.0):
    from mlcg_amd import nn

    g = torch.Generator().manual_seed(2)
    types = torch.randint(1, 21, (sum(lengths),), generator=g)
    emb = nn.ChainEmbedding(21, 128, _encoder(dropout), types, lengths)
    return emb


@pytest.mark.parametrize("lengths", [[35], [35, 100, 60]])
def test_schnet_on_a_chain_embedding(lengths):
    """Energies, forces and gradients of a SchNet whose table comes from the
    encoder equal those of the same SchNet on that table, chained through it."""
    from mlcg_amd import nn, synthetic
    from oracle import schnet_ref as R

    cfg = make_cfg(num_blocks=2, rc=20.0)
    model = make_model(cfg, R.random_state_dict(cfg, seed=1))
    model.embedding_layer = _embedding(lengths).cuda()
    assert model.fused_spec() is not None
    plain = copy.deepcopy(model)
    plain.embedding_layer = model.embedding_layer.as_embedding()
    data = synthetic.config2(n_frames=6).to_torch("cuda")
    n = data.pos.shape[0]
    data.atom_types = (torch.arange(n, device="cuda") % 35)  # the first chain's sites
    outs = []
    for m in (model, plain):
        d = nn.GradientsOut(m).train()(copy.copy(data))
        o = d.out["SchNet"]
        loss = torch.nn.functional.mse_loss(o["forces"], data.forces) + o["energy"].mean()
        loss.backward()
        outs.append((o["energy"].detach(), o["forces"].detach()))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    table_grad = plain.embedding_layer.weight.grad
    assert float(table_grad[:35].abs().max()) > 0.0
    emb = model.embedding_layer
    params = dict(emb.named_parameters())
    want = torch.autograd.grad(emb.table(), list(params.values()), table_grad)
    for (name, p), w in zip(params.items(), want):
        check(p.grad, w, 1e-6, name, atol_frac=1.0)
    sites = torch.tensor([3, 0, 3], device="cuda")
    assert torch.equal(emb(sites), emb.table()[sites])


def test_recorded_training_step():
    """A recorded forward and backward of the encoder with dropout: every
    replay draws the masks of its own step, as the eager module does."""
    enc = _encoder(dropout=0.2)
    from mlcg_amd import ops

    chains = ops.chain_layout(LENS, "cuda")
    g = torch.Generator().manual_seed(5)
    x = torch.randn(sum(LENS), 128, generator=g).cuda()
    grad = torch.randn(sum(LENS), 128, generator=g).cuda()
    enc = enc.cuda().train()
    eager = copy.deepcopy(enc)

    def step(m):
        out = m(x, chains)
        return [out.detach(), *torch.autograd.grad(out, list(m.parameters()), grad)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(enc)
    torch.cuda.current_stream().wait_stream(side)
    step(eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rec = step(enc)
    first = None
    for _ in range(4):
        x.copy_(torch.randn(x.shape, generator=g).cuda())
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(rec, step(eager)):
            check(a, b, 1e-6, "replay", atol_frac=1.0)
        torch.cuda.synchronize()
        assert first is None or not torch.equal(first, rec[0])
        first = rec[0].clone()
    assert int(enc.layers[0].drop1.step) == int(eager.layers[0].drop1.step) == 5


def test_dropout_module():
    from mlcg_amd import nn

    x = torch.randn(64, 32, device="cuda")
    a, b = nn.CounterDropout(0.5, 1).cuda().train(), nn.CounterDropout(0.5, 2).cuda().train()
    first, second, other = a(x), a(x), b(x)
    assert not torch.equal(first, second) and not torch.equal(first, other)
    again = nn.CounterDropout(0.5, 1).cuda()
    again.load_state_dict({"step": torch.ones(1, dtype=torch.int64)})
    assert torch.equal(again(x), second)  # a resumed run goes on with the next mask
    assert a.eval()(x) is x and torch.equal(a(x, residual=x), x + x)


def test_embedding_eval_and_copies():
    import pickle

    emb = _embedding([35, 20], dropout=0.3).cuda().train()
    plain = emb.as_embedding()
    assert emb.training and torch.equal(plain.weight.detach(), emb.eval().table().detach())
    twin = pickle.loads(pickle.dumps(emb))
    assert torch.equal(twin.table(), emb.table())
    assert torch.equal(copy.deepcopy(emb).table(), emb.table())
