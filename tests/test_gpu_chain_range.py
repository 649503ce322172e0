"""The attention over chains where its numbers are large, small or absent:
biases that mask, common to a row or not, of the type's ends and infinite, and
the accuracy of what the gradients are formed from.  The bounds are those of
test_gpu_chain.py (the logits' roundings are of the products' size, whatever
the size of the biases that cancel) unless a test derives its own."""

import math

import pytest
import torch

from oracle import chain_ref as R
from tests.test_gpu_chain import TYPES, U, _attention_case, _check_attention

pytestmark = pytest.mark.gpu


def _masked_case(lens, heads, kv, dim, dtype, bias, seed=0):
    """A band of 8 beads of ordinary biases, `bias` beyond it."""
    q, k, v, table, b, chains, grad = _attention_case(lens, heads, kv, dim, dtype, seed=seed,
                                                      kind="clip", buckets=17, reach=8)
    table = table.clone()
    table[0] = table[-1] = bias
    return q, k, v, table, b, chains, grad


def _biases(dtype):
    info = torch.finfo(dtype)
    common = [-1e4, info.min, info.max, -math.inf]
    return common if dtype == torch.float16 else [*common, -1e8, -1e9, 1e9]


RANGE = [(t, b) for t in TYPES for b in _biases(t)]


@pytest.mark.parametrize("dtype,bias", RANGE)
@pytest.mark.parametrize("lens", [[40, 33], [300, 90], [300] * 12, [130] * 70])
def test_forward_of_masking_biases(lens, dtype, bias):
    """Keys beyond the band come before and after ordinary ones, and the bias is
    the same for all keys of some rows: it cancels, or leaves nothing."""
    from mlcg_amd import nn

    print(f"masking biases {lens[0]} {dtype} {bias}", flush=True)
    q, k, v, table, b, chains, _ = _masked_case(lens, 2, 1, 32, dtype, bias)
    s = sum(lens)
    keep = torch.ones(s, dtype=torch.bool)
    keep[:lens[0]] = False
    keep[lens[0] - 20:lens[0] - 3] = True
    pos = torch.cumsum((torch.rand(s, generator=torch.Generator().manual_seed(1)) < 0.4).int(),
                       0).to(torch.int32).cuda()
    u = U[dtype]
    parts = 64.0 if dtype == torch.float32 else 1.25
    for kp in (None, keep.cuda()):
        for ps in (None, pos):
            out = nn.chain_attention(q, k, v, table, b, chains, keep=kp, positions=ps)
            ref, size = R.attention(q, k, v, table, b.bucket_of, lens, None, kp, ps)
            floor = (4.0 * u if dtype == torch.float32 else 64 * 2.0 ** -24) * float(
                size["out"].max())
            d = (out.cpu().double() - ref["out"]).abs()
            bad = ~(d <= parts * u * size["out"] + floor + 2.0 ** -24)
            assert not bool(bad.any()), (
                f"{int(bad.sum())} of {bad.numel()} off, worst {float(d.max())}")


@pytest.mark.parametrize("dtype,bias", RANGE)
@pytest.mark.parametrize("lens,dim,scale", [([40, 33], 32, None), ([300, 90], 32, None),
                                            ([300, 90], 64, -0.2), ([300, 90], 128, None),
                                            ([300] * 12, 32, None), ([130] * 70, 24, None)])
def test_gradients_of_masking_biases(lens, dim, scale, dtype, bias):
    print(f"gradients, masking biases {lens[0]} {dim} {dtype} {bias}", flush=True)
    q, k, v, table, b, chains, grad = _masked_case(lens, 2, 1, dim, dtype, bias, seed=dim)
    s = sum(lens)
    keep = torch.ones(s, dtype=torch.bool)
    keep[:lens[0]] = False
    keep[lens[0] - 20:lens[0] - 3] = True
    pos = torch.cumsum((torch.rand(s, generator=torch.Generator().manual_seed(1)) < 0.4).int(),
                       0).to(torch.int32).cuda()
    for kp in (None, keep.cuda()):
        for ps in (None, pos):
            _check_attention(q, k, v, table, b, chains, grad, scale, kp, ps)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 5, 40])
def test_single_key_that_a_bias_takes_away(n, dtype):
    """One present key, which the bias of some offsets takes away: these rows
    are empty and give dv nothing; a logit that is no number stays one."""
    from mlcg_amd import nn, ops

    print(f"single key {n} {dtype}", flush=True)
    q, k, v, _, _, chains, grad = _attention_case([n, 3], 2, 1, 16, dtype)
    b = ops.relative_buckets(3, 1, "clip")
    table = torch.zeros(3, 2, dtype=dtype, device="cuda")
    table[0, 0] = table[1, 1] = -math.inf  # head 0 later rows, head 1 the key's own
    keep = torch.zeros(n + 3, dtype=torch.bool, device="cuda")
    keep[0] = True
    keep[n:] = True
    _check_attention(q, k, v, table, b, chains, grad, keep=keep)
    q = q.clone()
    q[n - 1, 0] = math.nan
    table = torch.zeros_like(table)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
    out = nn.chain_attention(*leaves, b, chains, keep=keep)
    dq, dk, dv, _ = torch.autograd.grad(out, leaves, grad)
    for t in (out[n - 1, 0], dq[n - 1, 0], dk[0, 0], dv[0, 0]):
        assert bool(torch.isnan(t).all())


def test_fp32_gradients_are_as_exact_as_their_logits():
    """P is off by the roundings of its logit, exp2 and the row's sum alone.  A
    model of these steps in 32 bits (1031 keys, 32 channels) gives P 2.2e-7,
    normwise; the sums of dk and dv over the 33 queries that have a gradient
    here add 2^-24 / sqrt(3) sqrt(33 / 2) = 1.4e-7: 2.6e-7, and twice that is
    allowed.  With the sums begun at the row's logarithm in place of 0 the
    same model gives 1.0e-6.  dq and out sum 1031 keys, two a step: 2^-24 /
    sqrt(3) sqrt(516 / 2) = 5.5e-7, with P's 6.0e-7."""
    from mlcg_amd import nn

    print("fp32 gradients", flush=True)
    lens = [1031] * 4
    q, k, v, table, b, chains, grad = _attention_case(lens, 4, 4, 32, torch.float32, seed=6)
    few = torch.zeros_like(grad)
    few[::32] = grad[::32]
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
    out = nn.chain_attention(*leaves, b, chains)
    got = dict(zip("qkv", torch.autograd.grad(out, leaves[:3], few)), out=out.detach())
    ref, _ = R.attention(q, k, v, table, b.bucket_of, lens, None, None, None, few)
    for name, bound in (("k", 5.2e-7), ("v", 5.2e-7), ("q", 1.2e-6), ("out", 1.2e-6)):
        d = (got[name].cpu().double() - ref[name]).norm() / ref[name].norm()
        print(name, float(d), flush=True)
        assert float(d) <= bound, (name, float(d))


def _normwise(got, ref, name, relative):
    """Relative roundings, and half a spacing of fp16's subnormal numbers."""
    d = float((got.detach().cpu().double() - ref).norm())
    bound = relative * float(ref.norm()) + 2.0 ** -25 * math.sqrt(ref.numel())
    assert d <= bound, f"{name}: {d / max(float(ref.norm()), 1e-300)} of its norm, bound " \
                       f"{bound / max(float(ref.norm()), 1e-300)}"


@pytest.mark.parametrize("lens", [[60, 45], [2000], [130] * 40])
@pytest.mark.parametrize("size", [1e-4, 1e-3, 1e2])
def test_fp16_gradients_of_any_size(size, lens):
    """Gradients of a loss that is scaled down or up: dS passes through 16 bits
    relative to its row, not to 1.  P, dS and the output each round by 2^-11 /
    sqrt(3) in the mean: 2^-11 for the three."""
    from mlcg_amd import nn

    print(f"fp16 gradients {lens[0]} {size}", flush=True)
    q, k, v, table, b, chains, grad = _attention_case(lens, 2, 1, 64, torch.float16, seed=8)
    grad = grad * size
    pos = torch.cumsum((torch.rand(sum(lens), generator=torch.Generator().manual_seed(1)) < 0.4)
                       .int(), 0).to(torch.int32).cuda()
    for ps in (None, pos):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
        out = nn.chain_attention(*leaves, b, chains, positions=ps)
        grads = torch.autograd.grad(out, leaves, grad)
        ref, _ = R.attention(q, k, v, table, b.bucket_of, lens, None, None, ps, grad)
        for name, got in zip(("q", "k", "v", "table"), grads):
            _normwise(got, ref[name], name, 2.0 ** -11)


def test_fp16_gradients_beyond_the_type_inside():
    """dS passes fp16's largest number, the gradients do not."""
    from mlcg_amd import nn

    print("fp16 gradients, large dS", flush=True)
    lens = [4, 70, 200]
    q, k, v, table, b, chains, grad = _attention_case(lens, 2, 1, 64, torch.float16, seed=9,
                                                      views=False)
    k, q = k * 0.01, q * 0.01
    v = v * 4.0
    grad = (grad * 2e4).clamp(-6e4, 6e4)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
    out = nn.chain_attention(*leaves, b, chains)
    grads = torch.autograd.grad(out, leaves, grad)
    ref, _ = R.attention(q, k, v, table, b.bucket_of, lens, None, None, None, grad)
    for name, got in zip(("q", "k"), grads):
        assert float(ref[name].abs().max()) < 6e4
        _normwise(got, ref[name], name, 2.0 ** -11)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_biases_that_no_pair_has(bad, dtype):
    """Table entries of offsets that occur in no chain do not matter, whatever they
    hold."""
    from mlcg_amd import nn

    print(f"unused biases {dtype} {bad}", flush=True)
    odd = torch.cat([2 * torch.arange(n) + 1 for n in (40, 35, 1, 200)]).to(torch.int32)
    for lens, ps, unused in (([40, 35], None, lambda d: abs(d) >= 40),
                             ([120, 7], None, lambda d: abs(d) >= 120),
                             ([40, 35, 1, 200], odd, lambda d: d % 2 == 1)):
        q, k, v, table, b, chains, grad = _attention_case(lens, 2, 1, 32, dtype, kind="clip",
                                                          buckets=257, reach=128)
        mask = torch.tensor([unused(d) for d in range(-128, 129)], device="cuda")
        outs = []
        for fill in (0.0, bad):
            t = table.clone()
            t[mask] = fill
            leaves = [x.detach().requires_grad_(True) for x in (q, k, v, t)]
            out = nn.chain_attention(*leaves, b, chains,
                                     positions=None if ps is None else ps.cuda())
            outs.append((out.detach(), *torch.autograd.grad(out, leaves, grad)))
        for x, y in zip(*outs):
            assert torch.equal(x, y)


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_table_gradient_of_a_long_chain(dtype, given):
    """As test_attention_table_gradient_of_a_long_chain, whose bound this is, in
    both 16-bit types and with sums along diagonals or by residue numbers: the
    table's gradient is off by its own rounding, u / sqrt(3) in the mean at most,
    and u / 16 for what comes before it."""
    from mlcg_amd import nn

    print(f"table gradient {dtype} {given}", flush=True)
    q, k, v, table, b, chains, grad = _attention_case([2000], 2, 2, 64, dtype, seed=4)
    pos = None
    if given:
        pos = torch.cumsum((torch.rand(2000, generator=torch.Generator().manual_seed(1)) < 0.4)
                           .int(), 0).to(torch.int32).cuda()
    leaf = table.clone().requires_grad_(True)
    got, = torch.autograd.grad(nn.chain_attention(q, k, v, leaf, b, chains, positions=pos), leaf,
                               grad)
    ref, _ = R.attention(q, k, v, table, b.bucket_of, chains.lengths, None, None, pos, grad)
    d = (got.cpu().double() - ref["table"]).norm() / ref["table"].norm()
    u = U[dtype]
    print(float(d) / u, flush=True)
    assert float(d) <= u / math.sqrt(3.0) + u / 16.0, float(d)
