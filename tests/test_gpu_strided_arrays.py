"""Arrays with gaps or of another type, of which an operator makes copies: each copy
has its own room until the launch, so that the results are those of arrays without
gaps, bit for bit."""

import pytest
import torch
from test_gpu_basis import _pair_setup
from test_gpu_outnet import _params

pytestmark = pytest.mark.gpu


def _gaps(t):
    """The same values, every other element of an array."""
    if t is None:
        return None
    room = torch.full((*t.shape, 2), float("nan"), dtype=t.dtype, device=t.device)
    room[..., 0] = t
    return room[..., 0]


def _same(got, want):
    for a, b in zip(got, want):
        assert (a is None) == (b is None)
        assert a is None or torch.equal(a, b)


def test_langevin_masses_of_another_type():
    from mlcg_amd import ops

    g = torch.Generator(device="cuda").manual_seed(2)
    n = 1000
    pos, vel, forces, noise = (torch.randn(n, 3, device="cuda", generator=g) for _ in range(4))
    mass, ratio = (torch.rand(n, device="cuda", generator=g) + 0.5 for _ in range(2))
    results = []
    for how in (lambda t: t, lambda t: t.double(), _gaps, lambda t: _gaps(t.double())):
        p, v = pos.clone(), vel.clone()
        ops.langevin_baoa(p, v, forces, how(mass), how(ratio), 0.004, 0.9, 0.1, 7, noise=noise)
        ops.langevin_b(v, forces, how(mass), 0.004)
        results.append((p, v))
    for got in results[1:]:
        _same(got, results[0])


def test_output_network():
    from mlcg_amd import ops

    g = torch.Generator(device="cuda").manual_seed(3)
    W0, b0, w1, b1 = _params(64, 5, True, True)
    x, xdot = (torch.randn(50, 128, device="cuda", generator=g) for _ in range(2))
    tw, pw = (torch.randn(50, device="cuda", generator=g) for _ in range(2))
    want = ops.out_forward(x, W0, b0, w1, b1, 1, reverse=True)
    got = ops.out_forward(_gaps(x), _gaps(W0), _gaps(b0), _gaps(w1), _gaps(b1), 1, reverse=True)
    _same(got, want)
    _, oz, os_, _ = want
    a = (x, xdot, W0, w1, oz, os_)
    _same(ops.out_rev2(*map(_gaps, a), 1, _gaps(tw), _gaps(pw), True, True),
          ops.out_rev2(*a, 1, tw, pw, True, True))


def test_filters_and_gathers():
    from mlcg_amd import ops

    cfg, _, pos, graph, model, spec, _ = _pair_setup("gaussian")
    blk = model.fused_params().blocks[0]
    g = torch.Generator(device="cuda").manual_seed(4)
    cap, n, pairs = graph.pair_capacity, graph.num_nodes, graph.num_pairs
    Wbar, Wdbar = torch.zeros(2, cap, 128, device="cuda").unbind()
    for t in (Wbar, Wdbar):
        t[:pairs] = torch.randn(pairs, 128, device="cuda", generator=g)
    weights = (blk.W1, blk.b1, blk.W2)
    want = ops.filter_bwd(pos, graph, spec.filt, *weights, Wbar, Wdbar, pair_adjoints=True)
    _same(ops.filter_bwd(pos, graph, spec.filt, *weights, _gaps(Wbar), _gaps(Wdbar),
                         pair_adjoints=True), want)
    W, Wd, dist = ops.filter_fwd(pos, graph, spec.filt, *weights)
    _same(ops.rbf_param_grad(dist, graph, spec.filt, blk.W1, _gaps(want[3]), _gaps(want[4])),
          ops.rbf_param_grad(dist, graph, spec.filt, blk.W1, want[3], want[4]))

    g2, g1, y, yd = (torch.randn(n, 128, device="cuda", generator=g) for _ in range(4))
    u = torch.randn(n, 3, device="cuda", generator=g)
    dd = ops.pair_ddot(pos, dist, graph, u)
    assert torch.equal(ops.pair_ddot(pos, dist, graph, _gaps(u)), dd)
    _same(ops.filter_bwd_cfconv(pos, graph, spec.filt, *weights, _gaps(g2), _gaps(y), _gaps(g1),
                                _gaps(yd), dd),
          ops.filter_bwd_cfconv(pos, graph, spec.filt, *weights, g2, y, g1, yd, dd))
    _same(ops.cfconv_gather_rev2(_gaps(g2), _gaps(g1), _gaps(y), _gaps(yd), W, Wd, dd, graph),
          ops.cfconv_gather_rev2(g2, g1, y, yd, W, Wd, dd, graph))
    _same([ops.cfconv_gather_tangent(_gaps(yd), _gaps(y), W, Wd, dd, graph)],
          [ops.cfconv_gather_tangent(yd, y, W, Wd, dd, graph)])
    bars = torch.zeros(2, cap, device="cuda").unbind()
    _same([ops.cfconv_gather_bwd(_gaps(g1), _gaps(y), W, Wd, graph, bars[0])],
          [ops.cfconv_gather_bwd(g1, y, W, Wd, graph, bars[1])])
    assert torch.equal(*bars)
