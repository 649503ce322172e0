"""The sequence encoder's operators (ops.chain_attention, group_norm_act,
dropout_add and their gradients) against float64 (oracle/chain_ref.py).

Tolerances.  With u the unit roundoff of the arrays' type (2^-24, 2^-11,
2^-8), an attention output rounds once itself and its terms once (P, dS, and
delta through the rounded output): at most u times the sizes that the oracle
gives, each rounding 1 part, 1.25 covering the products of two of them and
the fp32 sums under 16 bits.  In fp32 the roundings are those of the logits (a
sum of up to 128 products, then the exponential's argument: about
2^-24 (8 + 2 |l|) relative in P with |l| up to ~20 here) and of sums over up
to 700 terms: 64 parts.  Group norm: fp32 sums (a few parts of the size of the
largest element, 2e-6), outputs rounded once.  fp16 values below 2^-14 round
by 2^-25 absolutely, in dS too: a term for the sums over it.
"""

import math

import pytest
import torch

from oracle import chain_ref as R

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
U = {t: torch.finfo(t).eps / 2 for t in TYPES}  # 2^-24, 2^-11, 2^-8


def _randn(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def _within(got, ref, bound, name):
    d = (got.detach().cpu().double() - ref).abs()
    bad = ~(d <= bound)
    assert not bool(bad.any()), (
        f"{name}: {int(bad.sum())} of {bad.numel()} off, worst "
        f"{float((d / bound.clamp_min(1e-300)).max()):.3f} of the bound")


def _attention_case(lengths, heads, kv, dim, dtype, seed=0, kind="log", buckets=32, reach=128,
                    keep=None, positions=None, views=True):
    from mlcg_amd import ops

    s = sum(lengths)
    if views:  # slices of one projection
        qkv = _randn((s, heads + 2 * kv, dim), dtype, seed)
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    else:
        q, k, v = (_randn((s, n, dim), dtype, seed + i)
                   for i, n in enumerate((heads, kv, kv)))
    b = ops.relative_buckets(buckets, reach, kind)
    table = _randn((b.num_buckets, heads), dtype, seed + 7, 0.5)
    grad = _randn((s, heads, dim), dtype, seed + 8)
    chains = ops.chain_layout(lengths, "cuda")
    return q, k, v, table, b, chains, grad


def _check_attention(q, k, v, table, b, chains, grad, scale=None, keep=None, positions=None):
    from mlcg_amd import nn

    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
    out = nn.chain_attention(*leaves, b, chains, scale, keep, positions)
    grads = torch.autograd.grad(out, leaves, grad)
    alone = nn.chain_attention(q, k, v, table, b, chains, scale, keep, positions)
    assert torch.equal(out.detach(), alone) or bool(torch.isnan(alone).any())
    ref, size = R.attention(q, k, v, table, b.bucket_of, chains.lengths, scale, keep, positions,
                            grad)
    u = U[q.dtype]
    parts = 64.0 if q.dtype == torch.float32 else 1.25
    group = q.shape[1] // k.shape[1]
    # 2^-25 absolute roundings of fp16: one term for each bead of the chain
    tiny = 2.0 ** -25 * (4.0 * chains.max_len * group + 4.0) if q.dtype == torch.float16 else 0.0
    for name, got in (("out", out), *zip(("q", "k", "v", "table"), grads)):
        t = tiny * (chains.n_beads if name == "table" else 1.0)
        floor = u * 1e-3 * float(size[name].abs().max()) if size[name].numel() else 0.0
        if q.dtype != torch.float32:  # fp32 arithmetic under 16-bit values
            floor += 64 * 2.0 ** -24 * (float(size[name].max()) if size[name].numel() else 0.0)
        else:
            floor *= 1e3 * 4.0
        assert got.shape == ref[name].shape and got.dtype == q.dtype
        _within(got, ref[name], parts * u * size[name] + t + floor, name)
    return out, grads


LENGTHS = {
    "one": [1],
    "ones": [1, 1, 1, 2, 1],
    "gaps": [0, 5, 0, 0, 33, 0],
    "short": [35, 10, 7, 31, 32],
    "tiles": [63, 64, 65, 127, 128, 129, 1],
    "long": [700, 3, 257],
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", sorted(LENGTHS))
def test_attention_lengths(lengths, dtype):
    print(f"attention {lengths} {dtype}", flush=True)
    _check_attention(*_attention_case(LENGTHS[lengths], 2, 2, 32, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 5, 16, 20, 24, 33, 48, 64, 96, 100, 128])
def test_attention_head_dims(dim, dtype):
    print(f"attention dim {dim} {dtype}", flush=True)
    _check_attention(*_attention_case([70, 1, 33], 3, 1, dim, dtype, seed=dim))


@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 4), (4, 2), (6, 1), (8, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_shared_heads(heads, kv, dtype):
    print(f"attention heads {heads}/{kv} {dtype}", flush=True)
    _check_attention(*_attention_case([90, 140], heads, kv, 16, dtype, seed=heads))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [16, 40, 64])
def test_attention_few_long_chains(dim, dtype):
    """The keys of a tile in four parts: absent beads (whole parts of them, too)
    and residue numbers, a reach that takes the most LDS, unaligned rows."""
    from mlcg_amd import nn

    print(f"attention few long {dim} {dtype}", flush=True)
    lens = [611, 258]
    q, k, v, table, b, chains, grad = _attention_case(lens, 2, 1, dim, dtype, seed=dim,
                                                      reach=1024)
    g = torch.Generator().manual_seed(dim)
    keep = torch.rand(sum(lens), generator=g) < 0.8
    keep[64:330] = False
    keep[611:] = False
    keep[700] = True
    pos = torch.cumsum((torch.rand(sum(lens), generator=g) < 0.4).int(), 0).to(torch.int32)
    for kp, ps in ((None, None), (keep.cuda(), None), (keep.cuda(), pos.cuda())):
        _check_attention(q, k, v, table, b, chains, grad, keep=kp, positions=ps)
    odd = torch.empty(sum(lens), 4, dim + 1, dtype=dtype, device="cuda")[:, :, :dim]
    odd[:, :2], odd[:, 2:3], odd[:, 3:] = q, k, v
    a = nn.chain_attention(q, k, v, table, b, chains, keep=keep.cuda())
    o = nn.chain_attention(odd[:, :2], odd[:, 2:3], odd[:, 3:], table, b, chains,
                           keep=keep.cuda())
    assert torch.equal(a, o)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("chains_of_130", [20, 40, 50])
def test_attention_many_middling_chains(chains_of_130, dtype):
    """Workgroup counts on both sides of the compute units and of half as many
    again, where the shapes change."""
    print(f"attention middling {chains_of_130} {dtype}", flush=True)
    _check_attention(*_attention_case([130] * chains_of_130, 4, 2, 16, dtype,
                                      seed=chains_of_130))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("reach", [192, 193, 512, 513, 768, 769, 1024])
def test_attention_reach(reach, dim, dtype):
    """A reach that leaves little room beside the tiles, at every shape of the
    backward pass, positions given or not."""
    print(f"attention reach {reach} {dim} {dtype}", flush=True)
    for lens in ([33, 20], [60], [300], [130] * 40):
        q, k, v, table, b, chains, grad = _attention_case(lens, 4, 4, dim, dtype, seed=reach,
                                                          reach=reach)
        pos = 3 * torch.arange(sum(lens), dtype=torch.int32, device="cuda")
        for ps in (None, pos):
            _check_attention(q, k, v, table, b, chains, grad, positions=ps)


def test_attention_table_gradient_of_a_long_chain():
    """The table's gradient sums dS of millions of pairs, which nearly cancel:
    it is off by its own rounding alone, at most u / sqrt(3) in the mean over a
    binade, and by what the 32-bit sums leave (u / 16)."""
    print("attention table gradient", flush=True)
    q, k, v, table, b, chains, grad = _attention_case([2000], 2, 2, 64, torch.bfloat16, seed=4)
    leaf = table.clone().requires_grad_(True)
    from mlcg_amd import nn

    got, = torch.autograd.grad(nn.chain_attention(q, k, v, leaf, b, chains), leaf, grad)
    ref, _ = R.attention(q, k, v, table, b.bucket_of, chains.lengths, None, None, None, grad)
    d = (got.cpu().double() - ref["table"]).norm() / ref["table"].norm()
    u = U[torch.bfloat16]
    assert float(d) <= u / math.sqrt(3.0) + u / 16.0, float(d)


@pytest.mark.parametrize("kind,buckets,reach", [
    ("clip", 3, 1), ("clip", 65, 32), ("clip", 257, 128), ("log", 2, 5), ("log", 47, 100),
    ("log", 32, 1024), ("log", 16, 3)])
def test_attention_buckets(kind, buckets, reach):
    print(f"attention buckets {kind} {buckets} {reach}", flush=True)
    for dtype in (torch.float32, torch.bfloat16):
        _check_attention(*_attention_case([300, 20], 2, 2, 32, dtype, seed=reach, kind=kind,
                                          buckets=buckets, reach=reach))


def test_attention_own_bucket_table():
    from mlcg_amd import ops

    q, k, v, _, _, chains, grad = _attention_case([150], 2, 2, 16, torch.float32)
    b = ops.relative_buckets(5, 4, [4, 0, 0, 2, 1, 1, 2, 0, 4])  # bucket 3 is not used
    table = _randn((5, 2), torch.float32, 3)
    _, grads = _check_attention(q, k, v, table, b, chains, grad)
    assert float(grads[3][3].abs().max()) == 0.0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", ["short", "long", "gaps", "tiles"])
def test_attention_absent_beads(lengths, dtype):
    """Absent beads with NaN and infinities in their keys and values, a chain
    without any present bead, one with a single one."""
    from mlcg_amd import nn

    print(f"attention keep {lengths} {dtype}", flush=True)
    lens = LENGTHS[lengths]
    q, k, v, table, b, chains, grad = _attention_case(lens, 4, 2, 32, dtype, seed=3)
    g = torch.Generator().manual_seed(5)
    keep = torch.rand(sum(lens), generator=g) < 0.6
    ends = [0]
    for n in lens:
        ends.append(ends[-1] + n)
    big = max(range(len(lens)), key=lambda i: lens[i])
    other = next(i for i in range(len(lens)) if i != big and lens[i] > 0)
    keep[ends[other]:ends[other + 1]] = False
    keep[ends[big]:ends[big + 1] - 1] |= torch.rand(lens[big] - 1, generator=g) < 0.3
    keep = keep.cuda()
    _check_attention(q, k, v, table, b, chains, grad, keep=keep)
    clean = nn.chain_attention(q, k, v, table, b, chains, keep=keep)
    k2, v2 = k.clone(), v.clone()
    k2[~keep] = math.nan
    v2[~keep] = math.inf
    leaves = [t.detach().requires_grad_(True) for t in (q, k2, v2, table)]
    dirty = nn.chain_attention(*leaves, b, chains, keep=keep)
    assert torch.equal(clean, dirty.detach())
    for gr in torch.autograd.grad(dirty, leaves, grad):
        assert bool(torch.isfinite(gr).all())
    assert float(clean[ends[other]:ends[other + 1]].abs().max()) == 0.0
    # one present key in the largest chain: its value, and no gradient but dv
    keep[ends[big]:ends[big + 1]] = False
    keep[ends[big] + 1 if lens[big] > 1 else ends[big]] = True
    out, _ = _check_attention(q, k, v, table, b, chains, grad, keep=keep)
    one = v[ends[big] + 1].repeat_interleave(2, 0)
    assert torch.equal(out.detach()[ends[big]:ends[big + 1]],
                       one.expand(lens[big], -1, -1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_positions(dtype):
    """Residue numbers: several beads to one, gaps, decreasing ones, and the
    ends of the type, whose differences do not fit it."""
    lens = [200, 70, 40]
    q, k, v, table, b, chains, grad = _attention_case(lens, 2, 1, 32, dtype, kind="clip",
                                                      buckets=65, reach=32)
    g = torch.Generator().manual_seed(1)
    a = torch.cumsum((torch.rand(200, generator=g) < 0.3).long()
                     + 40 * (torch.rand(200, generator=g) < 0.02).long(), 0)
    c = torch.randint(-20, 20, (70,), generator=g)
    d = torch.where(torch.rand(40, generator=g) < 0.5, -2 ** 31, 2 ** 31 - 1)
    pos = torch.cat([a, c, d]).to(torch.int32).cuda()
    print(f"attention positions {dtype}", flush=True)
    _check_attention(q, k, v, table, b, chains, grad, positions=pos)
    # far apart throughout: every pair at the reach or at zero
    far = (torch.arange(310) * 1000).to(torch.int32).cuda()
    _check_attention(q, k, v, table, b, chains, grad, positions=far)


def test_attention_single_key_has_no_gradient():
    """A bead alone in its chain: softmax over one key is constant."""
    from mlcg_amd import nn

    for dtype in TYPES:
        q, k, v, table, b, chains, grad = _attention_case([1] * 40, 2, 2, 24, dtype)
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
        out = nn.chain_attention(*leaves, b, chains)
        dq, dk, dv, dt = torch.autograd.grad(out, leaves, grad)
        assert torch.equal(out.detach(), v) and torch.equal(dv, grad)
        for z in (dq, dk, dt):
            assert float(z.abs().max()) == 0.0


def test_attention_large_logits_and_scale():
    """Logits of hundreds: the running maximum keeps the exponentials in range.
    The values are exact powers of two, so that the logits are."""
    from mlcg_amd import ops

    s = 300
    q = torch.full((s, 1, 8), 16.0, device="cuda")
    k = torch.zeros(s, 1, 8, device="cuda")
    k[:, 0, 0] = torch.arange(s, device="cuda").float() - 150.0
    v = _randn((s, 1, 8), torch.float32, 1)
    b = ops.relative_buckets(3, 1, "clip")
    table = torch.zeros(3, 1, device="cuda")
    chains = ops.chain_layout([s], "cuda")
    _check_attention(q, k, v, table, b, chains, _randn((s, 1, 8), torch.float32, 2), scale=1.0)
    _check_attention(q, k, v, table, b, chains, _randn((s, 1, 8), torch.float32, 2), scale=0.0)


def test_attention_layouts():
    """Heads first in memory, a last axis that is not contiguous, rows that
    begin at an odd element: the same values bit for bit."""
    from mlcg_amd import nn

    for dtype in TYPES:
        q, k, v, table, b, chains, grad = _attention_case([90, 45], 2, 2, 32, dtype, views=False)
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
        out = nn.chain_attention(*leaves, b, chains)
        ref = [out.detach(), *torch.autograd.grad(out, leaves, grad)]

        def heads_first(t):
            return t.transpose(0, 1).contiguous().transpose(0, 1)

        def last_strided(t):
            return t.transpose(1, 2).contiguous().transpose(1, 2)

        def odd(t):
            flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
            flat[1:] = t.reshape(-1)
            return flat[1:].view(t.shape)

        for form in (heads_first, last_strided, odd):
            leaves = [form(t).detach().requires_grad_(True) for t in (q, k, v)]
            leaves.append(table.detach().requires_grad_(True))
            out = nn.chain_attention(*leaves, b, chains)
            got = [out.detach(), *torch.autograd.grad(out, leaves, form(grad))]
            for x, y in zip(got, ref):
                assert torch.equal(x, y), form.__name__


def test_attention_differences():
    """The gradient along a random direction against central differences of
    the float32 operator: (f(x + h d) - f(x - h d)) / 2h with h = 2^-6 has a
    truncation error of h^2 / 6 f''' (about 1e-4 here) and a rounding error of
    2^-24 |f| sqrt(n) / h (about 1e-4): 2e-3 of the derivatives' scale."""
    from mlcg_amd import nn

    q, k, v, table, b, chains, grad = _attention_case([60, 140], 2, 1, 16, torch.float32, seed=4)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
    grads = torch.autograd.grad(nn.chain_attention(*leaves, b, chains), leaves, grad)
    h = 2.0 ** -6
    for i, t in enumerate((q, k, v, table)):
        d = _randn(t.shape, torch.float32, 20 + i)
        d /= d.norm()
        f = []
        for sign in (h, -h):
            args = [x + sign * d if j == i else x for j, x in enumerate((q, k, v, table))]
            f.append(float((nn.chain_attention(*args, b, chains).double() * grad).sum()))
        got = float((grads[i].double() * d).sum())
        scale = float(grads[i].double().norm())
        assert abs((f[0] - f[1]) / (2 * h) - got) <= 2e-3 * max(scale, 1.0)


def test_attention_repeats_and_streams():
    """The same bits on every call and on another stream; a recorded graph's
    replays equal the eager call."""
    from mlcg_amd import ops

    q, k, v, table, b, chains, grad = _attention_case([400, 35, 129], 4, 2, 32, torch.bfloat16)

    def call():
        out, lse = ops.chain_attention(q, k, v, table, b, chains, want_lse=True)
        return (out, *ops.chain_attention_backward(q, k, v, table, b, chains, out, lse, grad))

    ref = call()
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(call(), ref))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, ref))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rec = call()
    for i in range(4):
        q.copy_(_randn(q.shape, q.dtype, 50 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(rec, call()))
        torch.cuda.synchronize()


NORMS = {
    "one": ([1], 8, 4),
    "single_values": ([1, 1], 6, 6),
    "gaps": ([0, 3, 0, 40], 128, 8),
    "ragged": ([35, 80, 27, 1, 63], 128, 32),
    "odd": ([19, 44], 129, 3),
    "odd_one": ([300], 77, 1),
    "wide": ([70, 5], 1024, 4),
    "wide_odd": ([40], 1023, 11),
    "by_channel": ([150, 31], 64, 64),
    "long": ([2500, 3], 96, 3),
    "longer": ([9000], 128, 1),
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["none", "tanh", "ssp", "silu"])
@pytest.mark.parametrize("name", sorted(NORMS))
def test_group_norm(name, act, dtype):
    from mlcg_amd import nn, ops

    lens, width, groups = NORMS[name]
    print(f"group norm {name} {act} {dtype}", flush=True)
    s = sum(lens)
    x = _randn((s, width), dtype, 1) + 3.0
    w = _randn((width,), dtype, 2, 0.3) + 1.0
    b = _randn((width,), dtype, 3, 0.3)
    grad = _randn((s, width), dtype, 4)
    chains = ops.chain_layout(lens, "cuda")
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    out = nn.group_norm_act(*leaves, groups, chains, act=act)
    grads = torch.autograd.grad(out, leaves, grad)
    assert torch.equal(out.detach(), nn.group_norm_act(x, w, b, groups, chains, act=act))
    ref = R.group_norm(x, w, b, groups, lens, act=act, grad=grad)
    u = U[dtype] if dtype != torch.float32 else 0.0
    for n, got in (("out", out), *zip(("x", "weight", "bias"), grads)):
        assert got.dtype == dtype and got.shape == ref[n].shape
        # a group of few values with a small variance enlarges the deviations'
        # rounding (2^-24 of x, up to 6) by up to 1 / sqrt(eps)
        few = 2.0 ** -24 * 6 / math.sqrt(1e-5) if min(lens, default=1) * width // groups < 8 else 0
        tol = u * ref[n].abs() + (2e-6 + few) * float(ref[n].abs().max()) + 1e-6
        if dtype == torch.float16:
            tol = tol + 2.0 ** -24
        _within(got, ref[n], tol, f"{n}")


def test_group_norm_far_from_zero():
    """Values whose mean is 1000 times their spread: the variance comes from
    deviations, not from a difference of squares (which would lose all but one
    digit).  x itself is known to 2^-24 1000 = 6e-5 of its spread."""
    from mlcg_amd import nn, ops

    lens = [3000, 50]
    x = _randn((3050, 64), torch.float32, 9) + 1000.0
    w, b = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    got = nn.group_norm_act(x, w, b, 4, ops.chain_layout(lens, "cuda"))
    ref = R.group_norm(x, w, b, 4, lens)["out"]
    _within(got, ref, torch.full_like(ref, 2e-4), "out")


def test_group_norm_constant_rows():
    """No variance: the bias and no gradient but the bias's."""
    from mlcg_amd import nn, ops

    x = torch.full((40, 32), 5.0, device="cuda", requires_grad=True)
    w = _randn((32,), torch.float32, 1).requires_grad_(True)
    b = _randn((32,), torch.float32, 2).requires_grad_(True)
    out = nn.group_norm_act(x, w, b, 4, ops.chain_layout([33, 7], "cuda"))
    assert torch.equal(out.detach(), b.detach().expand(40, 32))
    gw, gb = torch.autograd.grad(out.sum(), (w, b))
    assert float(gw.abs().max()) == 0.0 and torch.equal(gb, torch.full_like(gb, 40.0))


def test_group_norm_strides_repeats_streams():
    from mlcg_amd import ops

    lens = [100, 7, 330]
    for width in (64, 63):
        big = _randn((437, 200), torch.float32, 1)
        w, b = _randn((width,), torch.float32, 2), _randn((width,), torch.float32, 3)
        chains = ops.chain_layout(lens, "cuda")
        grad = _randn((437, width), torch.float32, 4)
        groups = width // 9 if width % 9 == 0 else 8
        ref = None
        for x in (big[:, :width].contiguous(), big[:, :width],
                  big[:, :width].t().contiguous().t()):
            y, stats = ops.group_norm_act(x, w, b, groups, chains, act="silu")
            got = (y, *ops.group_norm_act_backward(x, w, b, groups, chains, stats, grad,
                                                   "silu"))
            ref = ref or got
            assert all(torch.equal(p, q) for p, q in zip(got, ref))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y, stats = ops.group_norm_act(x, w, b, groups, chains, act="silu")
            got = (y, *ops.group_norm_act_backward(x, w, b, groups, chains, stats, grad,
                                                   "silu"))
        side.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, ref))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 64, 1001, 20000])
def test_dropout(n, dtype):
    """The kept elements exactly, their values to one rounding, the gradient
    with the same mask."""
    from mlcg_amd import nn

    seed, step = 0x123456789ABCDEF1, (7 << 32) + 5
    for p in (0.0, 0.1, 0.5, 0.99, 1.0 - 2.0 ** -16):
        print(f"dropout {n} {p} {dtype}", flush=True)
        x = _randn((n,), dtype, n) + 4.0
        r = _randn((n,), dtype, n + 1)
        g = _randn((n,), dtype, n + 2)
        kept, scale = R.dropout_kept(n, p, seed, step)
        xa, ra = x.clone().requires_grad_(True), r.clone().requires_grad_(True)
        for how in (step, torch.tensor([step], device="cuda")):
            out = nn.dropout_add(xa, p, seed, how, residual=ra)
            gx, gr = torch.autograd.grad(out, (xa, ra), g)
            ref = torch.where(kept, x.cpu().double() * scale, 0.0)
            want = ref + r.cpu().double()
            # fp32: scale, product and sum round once each
            u = max(U[dtype], 3 * 2.0 ** -24)
            big = float(U[torch.float32]) * 3 * (ref.abs() + r.cpu().double().abs())
            inside = want.abs() < (60000 if dtype == torch.float16 else 1e38)
            d = (out.detach().cpu().double() - want).abs()
            assert bool((d <= 1.01 * u * want.abs() + big)[inside].all())
            gref = torch.where(kept, g.cpu().double() * scale, 0.0)
            inside = gref.abs() < (60000 if dtype == torch.float16 else 1e38)
            assert bool(((gx.cpu().double() - gref).abs()
                         <= 1.01 * u * gref.abs() + 2.0 ** -25)[inside].all())
            assert torch.equal(gr, g)
            plain = nn.dropout_add(x, p, seed, how)
            assert torch.equal(plain.cpu() != 0, kept & (x.cpu() != 0))


def test_dropout_drops_whatever_stands_there():
    from mlcg_amd import ops

    x = torch.full((4096,), math.nan, device="cuda")
    kept, _ = R.dropout_kept(4096, 0.5, 3, 1)
    y = ops.dropout_add(x, 0.5, 3, 1, torch.ones(4096, device="cuda"))
    assert torch.equal(torch.isnan(y).cpu(), kept)
    assert bool((y.cpu()[~kept] == 1.0).all())


def test_dropout_layouts_and_graph():
    """Views that do not begin at a multiple of 16 bytes or are transposed; a
    recorded graph draws a new mask whenever its step moves on."""
    from mlcg_amd import ops

    x = _randn((257, 33), torch.float32, 1)
    ref = ops.dropout_add(x, 0.3, 11, 4, x)
    flat = torch.empty(x.numel() + 1, device="cuda")
    flat[1:] = x.reshape(-1)
    off = flat[1:].view(x.shape)
    assert torch.equal(ops.dropout_add(off, 0.3, 11, 4, off), ref)
    t = x.t().contiguous().t()
    assert torch.equal(ops.dropout_add(t, 0.3, 11, 4, t), ref)
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    ops.dropout_add(x, 0.3, 11, step)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.add_(1)
        rec = ops.dropout_add(x, 0.3, 11, step)
    seen = []
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(rec, ops.dropout_add(x, 0.3, 11, int(step.item())))
        seen.append(rec.clone())
    assert not any(torch.equal(a, c) for a, c in zip(seen, seen[1:]))


def test_offsets_past_32_bits():
    """Rows so far apart that their offsets pass 2^31 elements give what
    contiguous ones give, and so do rows past 2^31 elements of a long x."""
    from mlcg_amd import nn, ops

    print("offsets past 32 bits: views", flush=True)
    lens = [500, 90, 1]
    s = sum(lens)
    q, k, v, table, b, chains, grad = _attention_case(lens, 2, 1, 64, torch.bfloat16, views=False)
    far = torch.empty(s, 2 ** 22 - 8, dtype=torch.bfloat16, device="cuda")  # 5 GB
    assert far.stride(0) * (s - 1) > 2 ** 31
    wide = far[:, :256].unflatten(1, (4, 64))
    wide[:, :2], wide[:, 2:3], wide[:, 3:] = q, k, v
    near = [q, k, v]
    apart = [wide[:, :2], wide[:, 2:3], wide[:, 3:]]
    outs = []
    for args in (near, apart):
        leaves = [t.detach().requires_grad_(True) for t in args]
        out = nn.chain_attention(*leaves, table, b, chains)
        outs.append((out.detach(), *torch.autograd.grad(out, leaves, grad)))
    for x, y in zip(*outs):
        assert torch.equal(x, y)
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    x = _randn((s, 128), torch.bfloat16, 5)
    far[:, 300 * 8:300 * 8 + 128] = x
    y0, st0 = ops.group_norm_act(x, w, w, 8, chains)
    y1, st1 = ops.group_norm_act(far[:, 300 * 8:300 * 8 + 128], w, w, 8, chains)
    assert torch.equal(y0, y1) and torch.equal(st0, st1)
    del far, wide, apart
    print("offsets past 32 bits: a long x", flush=True)
    n, c = 2 ** 23 + 256, 256
    x = torch.empty(n, c, dtype=torch.bfloat16, device="cuda").normal_()
    assert x.numel() > 2 ** 31
    lens = [256] * (n // 256)
    chains = ops.chain_layout(lens, "cuda")
    w = torch.ones(c, dtype=torch.bfloat16, device="cuda")
    y, st = ops.group_norm_act(x, w, w, 8, chains)
    dx, _, _ = ops.group_norm_act_backward(x, w, w, 8, chains, st, y)
    last = ops.chain_layout([256] * 512, "cuda")
    rows = slice(n - 512 * 256, n)
    y1, st1 = ops.group_norm_act(x[rows], w, w, 8, last)
    dx1, _, _ = ops.group_norm_act_backward(x[rows], w, w, 8, last, st1, y1)
    assert torch.equal(y[rows], y1) and torch.equal(dx[rows], dx1)
    del y, dx
    z = ops.dropout_add(x, 0.5, 11, 3).view(-1)
    e = 2 ** 31 + 8
    kept, scale = R.dropout_kept(4096, 0.5, 11, 3, first=e)
    want = torch.where(kept, x.view(-1)[e:e + 4096].cpu() * scale, 0.0)  # scale 2: exact
    assert torch.equal(z[e:e + 4096].cpu(), want)


def test_empty_inputs():
    from mlcg_amd import nn, ops

    for lens in ([], [0], [0, 0, 0]):
        chains = ops.chain_layout(lens, "cuda")
        b = ops.relative_buckets(8, 4)
        q = torch.empty(0, 2, 16, device="cuda", requires_grad=True)
        table = torch.ones(8, 2, device="cuda", requires_grad=True)
        out = nn.chain_attention(q, q, q, table, b, chains)
        gq, gt = torch.autograd.grad(out, (q, table), torch.empty_like(out))
        assert out.shape == gq.shape == (0, 2, 16) and float(gt.abs().max()) == 0.0
        x = torch.empty(0, 8, device="cuda", requires_grad=True)
        w = torch.ones(8, device="cuda", requires_grad=True)
        y = nn.group_norm_act(x, w, w, 2, chains)
        gx, gw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
        assert y.shape == gx.shape == (0, 8) and float(gw.abs().max()) == 0.0
    assert ops.dropout_add(torch.empty(0, device="cuda"), 0.5, 1, 1).numel() == 0


def test_refusals():
    from mlcg_amd import nn, ops

    chains = ops.chain_layout([4, 6], "cuda")
    b = ops.relative_buckets(8, 4)
    q = torch.zeros(10, 4, 16, device="cuda")
    k = torch.zeros(10, 2, 16, device="cuda")
    table = torch.zeros(8, 4, device="cuda")
    bad = [
        (dict(q=q[:9]), "q must be"),
        (dict(k=k[:, :, :8]), "k and v must be"),
        (dict(k=torch.zeros(10, 3, 16, device="cuda"),
              v=torch.zeros(10, 3, 16, device="cuda")), "cannot share"),
        (dict(v=k.half()), "v must be"),
        (dict(q=q.double(), k=k.double(), v=k.double(), table=table.double()), "float32, float16"),
        (dict(table=table[:7]), "table must be"),
        (dict(table=table.half()), "table must be"),
        (dict(keep=torch.ones(10, device="cuda")), "keep must be"),
        (dict(keep=torch.ones(9, dtype=torch.bool, device="cuda")), "keep must be"),
        (dict(positions=torch.zeros(10, dtype=torch.int64, device="cuda")), "positions must be"),
        (dict(q=q.cpu()), "ROCm GPU"),
        (dict(chains=ops.chain_layout([4, 6], "cpu")), "ChainLayout"),
        (dict(chains=[4, 6]), "ChainLayout"),
        (dict(q=torch.zeros(10, 4, 129, device="cuda"), k=torch.zeros(10, 2, 129, device="cuda"),
              v=torch.zeros(10, 2, 129, device="cuda")), "head dimension"),
    ]
    for change, match in bad:
        args = dict(dict(q=q, k=k, v=k, table=table, buckets=b, chains=chains), **change)
        with pytest.raises(RuntimeError, match=match):
            nn.chain_attention(**args)
    h = torch.float16
    for rest in (q.to(h)[:9], q, q.to(h).transpose(0, 1)):
        with pytest.raises(RuntimeError, match="rest must"):
            ops.chain_attention(q.to(h), k.to(h), k.to(h), table.to(h), b, chains, rest=rest)
    x = torch.zeros(10, 12, device="cuda")
    w = torch.zeros(12, device="cuda")
    for args, match in (((x, w, w, 5, chains), "equal groups"), ((x[:9], w, w, 3, chains), "x must"),
                        ((x, w[:11], w, 3, chains), "weight must"),
                        ((x, w, w.half(), 3, chains), "bias must"),
                        ((torch.zeros(10, 1025, device="cuda"), w, w, 1, chains), "channels"),
                        ((x, w, w, 3, chains, 1e-5, "relu"), "act must")):
        with pytest.raises(RuntimeError, match=match):
            nn.group_norm_act(*args)
    for args, match in (((x, 1.0, 1, 1), "probability"), ((x, -0.1, 1, 1), "probability"),
                        ((x, 0.5, -1, 1), "seed"), ((x, 0.5, 1, -1), "step"),
                        ((x, 0.5, 1, torch.zeros(2, dtype=torch.int64, device="cuda")), "step"),
                        ((x, 0.5, 1, 1, x[:9]), "residual"), ((x.double(), 0.5, 1, 1), "float32")):
        with pytest.raises(RuntimeError, match=match):
            nn.dropout_add(*args)
    with pytest.raises(RuntimeError):  # differentiable once
        qq = q.clone().requires_grad_(True)
        out = nn.chain_attention(qq, k, k, table, b, chains)
        (g,) = torch.autograd.grad(out.sum(), qq, create_graph=True)
        g.sum().backward()
