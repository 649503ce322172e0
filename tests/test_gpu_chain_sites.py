"""SchNet on a ChainEmbedding of many sites: the table's gradient is summed in a
fixed order at every size of the table, by the native sweep, eager and
recorded."""

import copy

import pytest
import torch

from tests.helpers import make_cfg, make_model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,sites", [(1, 129), (17920, 268), (30000, 1000), (4097, 4097),
                                        (50000, 8191), (3000, 20000)])
def test_sums_by_site(rows, sites):
    """out[t] = the sum of t's rows against float64: compensated sums, a part of
    2^-23 of the terms' sizes, the same bits again; a site outside of the
    table is reported."""
    from mlcg_amd import ops

    print(f"sums by site {rows} {sites}", flush=True)
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, 128, generator=g).cuda()
    for types in (torch.arange(rows) % sites, torch.randint(0, sites, (rows,), generator=g),
                  torch.full((rows,), sites - 1)):
        types = types.cuda()
        out, bad = ops.site_sum(x, types, sites)
        want = torch.zeros(sites, 128, dtype=torch.float64, device="cuda")
        size = want.clone().index_add_(0, types, x.double().abs())
        want.index_add_(0, types, x.double())
        assert int(bad) == 0
        assert bool(((out.double() - want).abs() <= 2.0 ** -23 * size).all())
        assert torch.equal(ops.site_sum(x, types, sites)[0], out)
    types[0] = sites
    assert int(ops.site_sum(x, types, sites)[1]) == 1


def _model(lens):
    from mlcg_amd import nn
    from oracle import schnet_ref as R

    torch.manual_seed(3)
    cfg = make_cfg(num_blocks=2, rc=20.0)
    model = make_model(cfg, R.random_state_dict(cfg, seed=1))
    types = torch.randint(1, 21, (sum(lens),), generator=torch.Generator().manual_seed(2))
    enc = nn.ChainEncoder(128, 1, 4, num_buckets=16, reach=32, dropout=0.1, seed=5)
    model.embedding_layer = nn.ChainEmbedding(21, 128, enc, types, lens)
    return model.cuda().train()


def _data(sites):
    """Frames of 35 beads that are any of the sites."""
    from mlcg_amd import synthetic

    data = synthetic.config2(n_frames=24).to_torch("cuda")
    n = data.pos.shape[0]
    data.atom_types = torch.arange(n, device="cuda") % sites
    return data


def _step(model, data):
    from mlcg_amd import nn

    model.zero_grad(set_to_none=True)
    out = nn.GradientsOut(model)(copy.copy(data)).out["SchNet"]
    loss = torch.nn.functional.mse_loss(out["forces"], data.forces)
    loss.backward()
    return loss.detach(), [p.grad.clone() for p in model.parameters()]


def test_training_step_repeats():
    """The same bits from equal steps, and the native sweep's from the parts'."""
    from mlcg_amd.nn import _fused

    print("training step on 300 sites", flush=True)
    lens = [35] * 4 + [100, 60]
    first = _model(lens)
    data = _data(sum(lens))
    runs = []
    calls = []
    native = _fused.ops.energy_forces_grad

    def counted(*args):
        calls.append(1)
        return native(*args)

    _fused.ops.energy_forces_grad = counted
    try:
        for _ in range(3):
            runs.append(_step(copy.deepcopy(first), data))
    finally:
        _fused.ops.energy_forces_grad = native
    assert len(calls) == 3  # the native sweep serves this table, too
    saved, _fused._TMM_SIDE = _fused._TMM_SIDE, True
    try:
        runs.append(_step(copy.deepcopy(first), data))
    finally:
        _fused._TMM_SIDE = saved
    for loss, grads in runs[1:]:
        assert torch.equal(loss, runs[0][0])
        for a, b in zip(grads, runs[0][1]):
            assert torch.equal(a, b)


def test_recorded_step_equals_eager():
    """CapturedTrainStep on a ChainEmbedding with dropout: parameters bit for bit
    those of eager steps."""
    from mlcg_amd import nn
    from mlcg_amd.pl import CapturedTrainStep

    print("recorded step on 300 sites", flush=True)
    lens = [35] * 4 + [100, 60]
    runs = []
    for captured in (False, True):
        model = _model(lens)
        data = _data(sum(lens))
        g0 = model.build_graph(data)
        cap = int(g0.num_edges * 1.05) + 64
        model.graph_capacity = cap + (cap % 2)
        gm = nn.GradientsOut(model)
        opt = torch.optim.AdamW(model.parameters(), lr=1e-3, fused=True, capturable=True)

        def step(d):
            opt.zero_grad(set_to_none=True)
            out = gm(d)
            out.out.update(**out.out[model.name])
            loss = nn.ForceMSE()(out)
            loss.backward()
            opt.step()
            return loss

        params = []
        if captured:
            cs = CapturedTrainStep(step, data, model, opt, warmup=1)
            batch = _data(sum(lens))
            for _ in range(3):
                cs.step(batch)
                torch.cuda.synchronize()
                params.append([p.detach().clone() for p in model.parameters()])
            cs.check()
        else:
            step(data)
            for _ in range(3):
                step(data)
                params.append([p.detach().clone() for p in model.parameters()])
        runs.append(params)
    for a, b in zip(*runs):
        for x, y in zip(a, b):
            assert torch.equal(x, y)
