"""Host side of calls of the encoder of linear cost's operators: what the entry
points are handed, with the entry points themselves replaced."""

import pytest
import torch

from mlcg_amd import nn, ops


@pytest.fixture
def calls(monkeypatch):
    """(name, arguments) of the entry points that CPU tensors are handed to."""
    made = []
    monkeypatch.setattr(ops, "call", lambda name, *args, **_: made.append((name, args)))
    monkeypatch.setattr(ops, "require_device", lambda *tensors: None)
    monkeypatch.setattr(ops, "stream_handle", lambda device=None: 0)
    monkeypatch.setattr(ops, "_delta_floats", lambda *args: 64)
    return made


def _heads():
    """q, k and v [8, 2 or 4, 16] as views of one projection, decay and beta."""
    x = torch.randn(8, 2 * 2 * 16 + 4 * 16, requires_grad=True)
    q, k, v = x.split([32, 32, 64], 1)
    return (x, q.unflatten(1, (2, 16)), k.unflatten(1, (2, 16)), v.unflatten(1, (4, 16)),
            -torch.rand(8, 4), torch.rand(8, 4))


def _packed(t):
    return t.clone(memory_format=torch.contiguous_format)


def _turned(t):
    """The same values with the axes the other way round in memory."""
    order = tuple(range(t.dim()))[::-1]
    return t.permute(order).contiguous().permute(order)


def _shifted(t):
    """The same values from an address one element past an aligned one on."""
    room = torch.zeros(t.numel() + 1, dtype=t.dtype)
    return room[1:].view(t.shape).copy_(t)


@pytest.mark.parametrize("how", [_packed, _turned, _shifted])
def test_backward_takes_the_arrays_as_they_come_back(calls, how):
    """Autograd's hooks may give a saved array back with other strides than it had:
    those of the array that is read count."""
    x, *args = _heads()
    saved, given = [], []

    def unpack(i):
        given.append(how(saved[i]))
        return given[-1]

    def pack(t):
        saved.append(t.detach())
        return len(saved) - 1

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        out, _ = nn.gated_delta(*args, ops.chain_layout([5, 3], "cpu"))
    torch.autograd.grad(out, x, torch.ones_like(out))
    name, a = calls[-1]
    assert name == "mlcg_gated_delta_backward"
    arrays = {t.data_ptr(): t for t in given}
    for i, t in enumerate(args[:3]):
        assert a[2 * i + 1][1] >= 16 and a[2 * i + 1][0] >= t.shape[1] * 16
        if a[2 * i] in arrays:  # not copied again
            assert list(a[2 * i + 1]) == list(arrays[a[2 * i]].stride()[:2])
            assert arrays[a[2 * i]].stride(2) == 1
        else:
            assert list(a[2 * i + 1]) == [t.shape[1] * 16, 16]
    assert a[25] % 32 == 0 and a[26] == 64  # what the forward pass kept
    if how is not _turned:
        assert all(a[2 * i] in arrays for i in range(3))


@pytest.mark.parametrize("change", [lambda t: t[..., :8], lambda t: t.double(),
                                    lambda t: t.flatten()[:-1]])
def test_backward_refuses_other_arrays(calls, change):
    x, *args = _heads()
    saved = []
    for which in (0, 5):  # q; what the forward pass kept
        del saved[:]

        def pack(t):
            saved.append(t.detach())
            return len(saved) - 1

        with torch.autograd.graph.saved_tensors_hooks(
                pack, lambda i: change(saved[i]) if i == which else saved[i]):
            out, _ = nn.gated_delta(*args, ops.chain_layout([5, 3], "cpu"))
        with pytest.raises(RuntimeError):
            torch.autograd.grad(out, x, torch.ones_like(out), retain_graph=True)


def _step_args():
    _, q, k, v, decay, beta = _heads()
    return [q.detach(), k.detach(), v.detach(), decay, beta, torch.zeros(8, 4, 16, 16)]


@pytest.mark.parametrize("which", range(7))
def test_step_refuses_tangents(calls, which):
    """A forward-mode tangent is refused, not dropped: no_grad leaves that mode on."""
    args = _step_args()
    args.append(torch.zeros_like(args[5]))
    with torch.autograd.forward_ad.dual_level():
        args[which] = torch.autograd.forward_ad.make_dual(args[which],
                                                          torch.ones_like(args[which]))
        with torch.no_grad(), pytest.raises(RuntimeError, match="derivative"):
            ops.gated_delta_step(*args[:6], into=args[6])
        assert not calls
    with torch.no_grad():
        ops.gated_delta_step(*_step_args())
    assert len(calls) == 1


def test_module_step_refuses_tangents(calls):
    delta = nn.ChainDelta(32, 2, bidirectional=False)
    with torch.autograd.forward_ad.dual_level():
        x = torch.autograd.forward_ad.make_dual(torch.ones(3, 32), torch.ones(3, 32))
        with pytest.raises(RuntimeError, match="derivative"):
            delta.step(x, delta.new_state(3))


@pytest.mark.parametrize("own", [True, False])
def test_step_moves_the_version_of_what_it_writes(calls, own):
    """A state that a graph has saved cannot be written unseen."""
    args = _step_args()
    into = args[5] if own else torch.zeros_like(args[5])
    scale = torch.ones((), requires_grad=True)
    loss = (scale * into).sum()  # saves into
    before = [t._version for t in args]
    with torch.no_grad():
        ops.gated_delta_step(*args, into=None if own else into)
    assert [t._version for t in args[:5]] == before[:5]
    assert args[5]._version == before[5] + own
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        ops.gated_delta_step(*_step_args())


def test_step_into_a_leaf(calls):
    args = _step_args()
    into = torch.zeros_like(args[5]).requires_grad_(True)
    with pytest.raises(RuntimeError, match="no_grad"):
        ops.gated_delta_step(*args, into=into)
    assert not calls


def test_plan_is_not_made_inside_a_capture(monkeypatch, calls):
    """A plan is copied from the host: a first call inside a capture is refused before
    anything is recorded, later ones have it."""
    chains = ops.chain_layout([70, 3], "cpu")
    monkeypatch.setattr(ops, "_capturing", lambda device: True)
    _, q, k, v, decay, beta = _heads()
    with pytest.raises(RuntimeError, match="before the capture"):
        ops._delta_plan(chains, 4)
    monkeypatch.undo()
    plan = ops._delta_plan(chains, 4)
    monkeypatch.setattr(ops, "_capturing", lambda device: True)
    assert ops._delta_plan(chains, 4) is plan


def test_embedding_pickled_without_a_factor():
    """A ChainEmbedding saved whole before it had a factor is one without."""
    class Same(torch.nn.Module):
        def forward(self, x, chains, keep=None, positions=None):
            return x

    made = nn.ChainEmbedding(4, 8, Same(), [0, 1, 3, 1], (3, 1))
    state = made.__getstate__()
    state.pop("scale", None)
    old = nn.ChainEmbedding.__new__(nn.ChainEmbedding)
    old.__setstate__(state)
    assert torch.equal(old.table(), made.table())


def test_orders_that_token_order_did_not_make(calls):
    """The gradient reads the rows that an order names: arrays that cannot be one are
    refused."""
    order = ops.token_order(torch.tensor([1, 0, 1]), 2)
    grad = torch.zeros(3, 4)
    short, wide = order.index[:2], order.index.long()
    for keys, index, rows in ((order.keys, short, 2), (order.keys, wide, 2),
                              (order.keys.long(), order.index, 2),
                              (order.keys, order.index.new_zeros(3, 2)[:, 0], 2),
                              (order.keys, order.index, 0), (order.keys, order.index, 2 ** 30)):
        with pytest.raises(RuntimeError):
            ops.scaled_embedding_backward(grad, ops.TokenOrder(keys, index, rows))
    assert [name for name, _ in calls] == ["mlcg_token_order"]
    ops.scaled_embedding_backward(grad, order)


@pytest.mark.parametrize("lengths,heads,dk,best", [
    ([4099] * 2, 8, 64, 6), ([4099] * 2, 4, 128, 6), ([4099] * 8, 8, 64, 6), ([20000], 8, 128, 12),
    ([20000], 4, 32, 6), ([2000], 4, 32, 4), ([120001], 8, 64, 64), ([1000] * 64, 4, 32, 0),
    ([1000] * 16, 8, 64, 0), ([500], 4, 32, 0), ([35], 4, 32, 0), ([0, 0], 1, 1, 0)])
def test_segments_that_measured_best(lengths, heads, dk, best):
    """The choice is what was measured fastest (forward and backward together) or within
    2 % of it."""
    assert ops._delta_segment_tiles(ops.chain_layout(lengths, "cpu"), heads, dk) == best
