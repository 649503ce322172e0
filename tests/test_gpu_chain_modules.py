"""The sequence encoder's operators and modules beyond plain fp32 reverse mode."""

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu

LENS = [35, 1, 62, 20]


def test_forward_mode_is_refused():
    """A tangent must not get lost: none of the operators has a forward-mode
    derivative."""
    from mlcg_amd import nn, ops

    chains = ops.chain_layout([40], "cuda")
    buckets = ops.relative_buckets(8, 4)
    q = torch.randn(40, 2, 16, device="cuda")
    table = torch.zeros(8, 2, device="cuda")
    x, w = torch.randn(40, 32, device="cuda"), torch.ones(32, device="cuda")
    calls = [lambda t: nn.chain_attention(t.view(40, 2, 16), q, q, table, buckets, chains),
             lambda t: nn.group_norm_act(t.view(40, 32), w, w, 4, chains),
             lambda t: nn.dropout_add(t.view(40, 32), 0.5, 1, 1),
             lambda t: nn.dropout_add(x, 0.5, 1, 1, residual=t.view(40, 32))]
    for f in calls:
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(torch.randn(1280, device="cuda"),
                                        torch.randn(1280, device="cuda"))
            with pytest.raises((RuntimeError, NotImplementedError)):
                f(dual)
            with torch.no_grad():  # a plain call beside it still runs
                f(torch.randn(1280, device="cuda"))


def _encoder(dropout=0.0):
    from mlcg_amd import nn

    torch.manual_seed(3)
    enc = nn.ChainEncoder(128, 2, 4, kv_heads=2, num_buckets=16, reach=32, dropout=dropout)
    with torch.no_grad():
        for name, p in enc.named_parameters():
            if name.endswith("bias") or name.endswith("bias_table"):
                p.normal_(0.0, 0.3)
    return enc.cuda()


def _step(enc, x, grad):
    from mlcg_amd import ops

    x = x.detach().requires_grad_(True)
    out = enc(x, ops.chain_layout(LENS, "cuda"))
    return [out.detach(), *torch.autograd.grad(out, [x, *enc.parameters()], grad.to(out.dtype))]


def _close(got, want, relative):
    for a, b in zip(got, want):
        assert a.shape == b.shape
        d = float((a.double() - b.double()).norm())
        assert d <= relative * float(b.double().norm()) + 1e-6, (tuple(a.shape), d)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dropout", [0.0, 0.2])
def test_autocast(dropout, dtype):
    """fp32 parameters under autocast: the 16-bit kernels run, the parameters'
    gradients are fp32.  About twenty roundings of 2^-8 (2^-11) follow each
    other in two layers, forward and backward: 2^-8 sqrt(20) = 1.7e-2 in the
    mean, of which some meet differences: 5e-2 (2^-11: an eighth)."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(sum(LENS), 128, generator=g).cuda()
    grad = torch.randn(sum(LENS), 128, generator=g).cuda()
    want = _step(_encoder(dropout), x, grad)
    enc = _encoder(dropout)
    with torch.autocast("cuda", dtype=dtype):
        got = _step(enc, x, grad)
    assert got[0].dtype == torch.float32  # the residual stream
    assert all(t.dtype == torch.float32 for t in got[1:])
    _close(got, want, 5e-2 if dtype == torch.bfloat16 else 5e-2 / 8)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_16_bit_modules(dtype):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(sum(LENS), 128, generator=g).cuda().to(dtype)
    grad = torch.randn(sum(LENS), 128, generator=g).cuda().to(dtype)
    enc = _encoder().to(dtype)
    want = _step(_encoder().to(dtype).float(), x.float(), grad.float())
    got = _step(enc, x, grad)
    assert all(t.dtype == dtype for t in got)
    _close(got, want, 5e-2 if dtype == torch.bfloat16 else 5e-2 / 8)
