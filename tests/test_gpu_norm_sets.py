"""Group norm over sets of chains: gradients summed over many chains, one long
chain among many short ones, more chains than a grid's second axis holds.
Against float64 (oracle/chain_ref.py); tolerances as in test_gpu_chain.py: fp32
sums, a few parts of the size of the largest element."""

import pytest
import torch

from oracle import chain_ref as R
from tests.test_gpu_chain import U, _randn, _within

pytestmark = pytest.mark.gpu


def _check_norm(x, lens, groups, act, out_tol=2e-6, grad_tol=4e-6):
    from mlcg_amd import nn, ops

    dtype, width = x.dtype, x.shape[1]
    w, b = _randn((width,), dtype, 2, 0.3) + 1.0, _randn((width,), dtype, 3, 0.3)
    grad = _randn(x.shape, dtype, 4)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    out = nn.group_norm_act(*leaves, groups, ops.chain_layout(lens, "cuda"), act=act)
    grads = torch.autograd.grad(out, leaves, grad)
    ref = R.group_norm(x, w, b, groups, lens, act=act, grad=grad)
    u = U[dtype] if dtype != torch.float32 else 0.0
    for n, got in (("out", out), *zip(("x", "weight", "bias"), grads)):
        tol = u * ref[n].abs() + (out_tol if n == "out" else grad_tol) * float(ref[n].abs().max())
        _within(got, ref[n], tol, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ["none", "silu"])
def test_gradients_over_many_chains(act, dtype):
    """More chains than workgroups: each adds the channels' sums of several."""
    print(f"many chains {act} {dtype}", flush=True)
    lens = [5 + (7 * i) % 9 for i in range(5000)]
    _check_norm(_randn((sum(lens), 32), dtype, 1) + 0.5, lens, 4, act)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_long_chain_among_many(dtype):
    """600 short chains and one of 50000 beads, whose first beads lie far from
    the others: its workgroups are many, and its deviations are taken from means
    of neighbours."""
    from mlcg_amd import _lib, ops

    print(f"one long chain {dtype}", flush=True)
    lens = [20] * 300 + [50000] + [35] * 300
    x = _randn((sum(lens), 64), dtype, 1)
    x[6000:6064] += 1000.0
    _check_norm(x, lens, 4, "none")
    chains = ops.chain_layout(lens, "cuda")
    assert _lib.load().mlcg_group_norm_workspace_floats(
        chains.tiles[256].shape[0], chains.n_chains, chains.whole.shape[0], chains.max_len, 64, 4,
        0) > 0


def test_more_chains_than_a_grid_axis():
    """70000 chains, most of them empty or short, and a long one."""
    print("70000 chains", flush=True)
    lens = [0] * 69600 + [3000] + [i % 7 for i in range(399)]
    _check_norm(_randn((sum(lens), 32), torch.float32, 1), lens, 4, "ssp")
