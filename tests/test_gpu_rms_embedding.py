"""RMS norm with the residual's addition and the scaled embedding, with their
gradients, against float64 (oracle/delta_ref.py).

Tolerances, with u half a step of the output's type: one rounding of the output, u
|value|; fp32 sums over up to 8192 channels in a tree and lanes' chains (a few
parts of 2^-24: 32 of the row's largest value).  The gradient of x is a difference
of two terms, dy w rstd and hat sum(dy w hat) rstd / C, that cancel for one
channel but for eps: 32 parts of the largest of the first.  The backward pass takes t as it
was stored, u' = half a step of its type: 2 u' more where the oracle has the sum
itself.  Sums over rows (the weight's, the table's gradient): 2^-24 sqrt(terms)
at most of the sum of sizes, here 8 of it.
"""

import pytest
import torch

from oracle import delta_ref as R

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
U = {t: torch.finfo(t).eps / 2 for t in TYPES}
E = 2.0 ** -24


def _within(got, ref, bound, name):
    d = (got.detach().cpu().double() - ref).abs()
    assert got.shape == ref.shape, name
    assert bool((d <= bound).all()), (name, float((d / bound.clamp_min(1e-300)).max()))


def _rms_case(n, width, dtype, rtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, width, generator=g).to(dtype).cuda()
    r = gt = None
    if rtype is not None:
        r = (2 * torch.randn(n, width, generator=g)).to(rtype).cuda()
        gt = torch.randn(n, width, generator=g).to(rtype).cuda()
    w = (1 + 0.3 * torch.randn(width, generator=g)).to(dtype).cuda()
    return x, r, w, torch.randn(n, width, generator=g).to(dtype).cuda(), gt


def _rms_run(x, r, w, gy, gt):
    from mlcg_amd import nn

    leaves = [t.detach().requires_grad_(True) for t in (x, r, w) if t is not None]
    y, t = nn.rms_norm_add(leaves[0], None if r is None else leaves[1], leaves[-1])
    if r is None:
        grads = torch.autograd.grad(y, leaves, gy)
    else:
        grads = torch.autograd.grad([y, t], leaves, [gy, gt])
    return y.detach(), t.detach(), grads


def _rms_check(x, r, w, gy, gt):
    y, t, grads = _rms_run(x, r, w, gy, gt)
    ref = R.rms_norm_add(x, r, w, grad=gy, grad_t=gt, stored=t)
    u = U[x.dtype]
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0

    f8 = (x if r is None else x.double() + r.double()).cpu().double()
    rstd = 1.0 / torch.sqrt((f8 * f8).mean(1, keepdim=True) + 1e-6)
    terms = (gy.cpu().double() * w.cpu().double() * rstd).abs().max(1, keepdim=True).values

    def bound(name, u):
        v = ref[name].abs()
        size = v.max(1, keepdim=True).values
        return u * v + 32 * E * (size + terms if name == "x" else size) + tiny

    _within(y, ref["y"], bound("y", u), "y")
    if r is None:
        assert torch.equal(t, x)
    else:
        ut = U[r.dtype]
        assert t.dtype == r.dtype
        _within(t, ref["t"], ut * ref["t"].abs() + tiny, "t")
        assert grads[1].dtype == r.dtype
        _within(grads[1], ref["x"], bound("x", ut), "residual")
    assert y.dtype == grads[0].dtype == grads[-1].dtype == x.dtype
    _within(grads[0], ref["x"], bound("x", u), "x")
    # sum of sizes: |dy| |hat|
    size = (gy.cpu().double().abs() * (ref["y"] / w.cpu().double()).abs()).sum(0)
    _within(grads[-1], ref["weight"], u * ref["weight"].abs() + 8 * E * size
            + 2 * E * size + tiny, "weight")


KINDS = [(torch.float32, None), (torch.float32, torch.float32), (torch.float16, torch.float16),
         (torch.float16, torch.float32), (torch.bfloat16, None), (torch.bfloat16, torch.bfloat16),
         (torch.bfloat16, torch.float32)]


@pytest.mark.parametrize("dtype,rtype", KINDS)
@pytest.mark.parametrize("n,width", [(1, 1), (1, 128), (3, 7), (35, 64), (100, 77), (1000, 129),
                                     (33, 512), (70, 1000), (5, 2048), (9, 2049), (3, 8192),
                                     (3, 8191)])
def test_rms(n, width, dtype, rtype):
    print(f"rms {n} {width} {dtype} {rtype}", flush=True)
    _rms_check(*_rms_case(n, width, dtype, rtype, seed=width))


def test_rms_many_rows():
    """More rows than a pass of the backward's workgroups takes, and a rest."""
    for width in (16, 128, 300):
        _rms_check(*_rms_case(70001, width, torch.bfloat16, torch.float32))


def test_rms_strides():
    from mlcg_amd import ops

    for dtype in TYPES:
        x, r, w, gy, gt = _rms_case(50, 96, dtype, torch.float32)
        want = ops.rms_norm_add(x, r, w)
        wide = torch.full((50, 200), float("nan"), dtype=dtype, device="cuda")
        wide[:, 3:99] = x
        rows = torch.full((50, 101), float("nan"), device="cuda")
        rows[:, 1:97] = r
        for a, b in ((wide[:, 3:99], rows[:, 1:97]), (x.t().contiguous().t(), r)):
            for got, ref in zip(ops.rms_norm_add(a, b, w), want):
                assert torch.equal(got, ref)
        one = r[:1].expand(50, 96)  # one row for all
        for got, ref in zip(ops.rms_norm_add(x, one, w), ops.rms_norm_add(x, one.contiguous(), w)):
            assert torch.equal(got, ref)
        assert all(t.shape[0] == 0 for t in ops.rms_norm_add(x[:0], r[:0], w))


def test_rms_sizes_of_values():
    """Rows of zeros, rows whose squares pass fp16's range, one row's NaN."""
    from mlcg_amd import ops

    x, r, w, gy, gt = _rms_case(6, 128, torch.float16, torch.float16)
    x[0], r[0] = 0.0, 0.0
    x[1], r[1] = 3e4, 1e4
    _rms_check(x, r, w, gy, gt)
    x[3, 5] = float("nan")
    y, t, _ = ops.rms_norm_add(x, r, w)
    assert bool(torch.isnan(y[3]).all())
    assert bool(torch.isfinite(y[[0, 1, 2, 4, 5]]).all())


def test_rms_outputs_alone():
    """A gradient of one of the two outputs; broadcast gradients."""
    from mlcg_amd import nn

    x, r, w, gy, gt = _rms_case(40, 64, torch.float32, torch.float32)
    for which in (0, 1):
        leaves = [t.detach().requires_grad_(True) for t in (x, r, w)]
        out = nn.rms_norm_add(*leaves)
        got = torch.autograd.grad(out[which], leaves, (gy, gt)[which])
        z = [gy * 0, gt * 0]
        z[which] = (gy, gt)[which]
        for a, b in zip(got, _rms_run(x, r, w, *z)[2]):
            assert torch.equal(a, b)
    leaves = [t.detach().requires_grad_(True) for t in (x, r, w)]
    sum(t.sum() for t in nn.rms_norm_add(*leaves)).backward()
    for a, b in zip(leaves, _rms_run(x, r, w, torch.ones_like(gy), torch.ones_like(gt))[2]):
        assert torch.equal(a.grad, b)


def test_rms_against_differences():
    """fp32, steps of 2^-6: as in the gated delta rule's test."""
    from mlcg_amd import nn

    x, r, w, gy, gt = _rms_case(20, 33, torch.float32, torch.float32)
    grads = _rms_run(x, r, w, gy, gt)[2]

    def value(a, b, c):
        y, t = nn.rms_norm_add(a, b, c)
        return float((y.double() * gy.double()).sum() + (t.double() * gt.double()).sum())

    g = torch.Generator().manual_seed(1)
    for i, grad in enumerate(grads):
        way = torch.randn(grad.shape, generator=g).cuda()
        way *= 2.0 ** -6 / way.norm()
        up, down = [x, r, w], [x, r, w]
        up[i], down[i] = up[i] + way, down[i] - way
        slope, want = value(*up) - value(*down), 2 * float((grad.double() * way.double()).sum())
        assert abs(slope - want) <= 2e-3 * 2.0 ** -5 * float(grad.norm()) + 2e-5


def test_rms_refusals():
    from mlcg_amd import nn, ops

    x, r, w, gy, gt = _rms_case(6, 32, torch.bfloat16, torch.float32)
    for args in ((x, r[:5], w), (x, r.half(), w), (x, r, w.float()), (x, r, w[:31]), (x[0], None, w),
                 (x, r.cpu(), w), (x.double(), None, w.double()), (x, r, w.cpu()),
                 (torch.zeros(2, 8193, device="cuda"), None, torch.zeros(8193, device="cuda"))):
        with pytest.raises(RuntimeError):
            nn.rms_norm_add(*args)
    y, t, rstd = ops.rms_norm_add(x, r, w)
    for args in ((gy, gt.bfloat16(), t, w, rstd), (gy, gt, t, w, rstd[:5]), (gy[:5], gt, t, w, rstd),
                 (gy, gt, t.half(), w, rstd)):
        with pytest.raises(RuntimeError):
            ops.rms_norm_add_backward(*args)


# ---------------------------------------------------------------------------

def _embed_check(rows, tokens, width, dtype, scale=2.5, seed=0):
    from mlcg_amd import nn, ops

    g = torch.Generator().manual_seed(seed)
    table = torch.randn(rows, width, generator=g).to(dtype).cuda().requires_grad_(True)
    grad = torch.randn(tokens.shape[0], width, generator=g).to(dtype).cuda()
    out = nn.scaled_embedding(table, tokens, scale)
    dt, = torch.autograd.grad(out, table, grad)
    ref = R.scaled_embedding(table, tokens, scale, grad)
    u = U[dtype]
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    _within(out, ref["out"], u * ref["out"].abs() + E * ref["out"].abs() + tiny, "out")
    _within(dt, ref["table"], u * ref["table"].abs() + 8 * E * ref["size"] + tiny, "table")
    order = ops.token_order(tokens, rows)
    key = torch.where((tokens < 0) | (tokens >= rows), rows, tokens)
    keys, index = torch.sort(key, stable=True)
    assert torch.equal(order.keys.long(), keys) and torch.equal(order.index.long(), index)
    again, = torch.autograd.grad(nn.scaled_embedding(table, tokens, scale), table, grad)
    assert torch.equal(dt, again)
    return out, dt


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,width", [
    (1, 1, 1), (1, 500, 77), (25, 1000, 128), (20, 50001, 33), (255, 2047, 8), (256, 2049, 16),
    (257, 4096, 24), (300, 20000, 96), (65535, 3000, 64), (65536, 3000, 64), (70000, 5000, 256),
    (3000, 30000, 600), (5, 100, 8192), (7, 300, 1025)])
def test_embedding(rows, n, width, dtype):
    print(f"embedding {rows} {n} {width} {dtype}", flush=True)
    g = torch.Generator().manual_seed(n)
    _embed_check(rows, torch.randint(0, rows, (n,), generator=g).cuda(), width, dtype, seed=rows)


@pytest.mark.parametrize("n", [0, 1, 31, 32, 33, 64, 2048, 2049])
def test_embedding_runs(n):
    """Tokens in order, all the same, and runs that begin and end at slabs."""
    _embed_check(3, torch.zeros(n, dtype=torch.int64, device="cuda"), 40, torch.float32)
    _embed_check(9, torch.arange(n, device="cuda") // 32 % 9, 40, torch.float32)
    _embed_check(n + 1, torch.arange(n, device="cuda").flip(0), 40, torch.float32)
    _embed_check(70, (torch.arange(n, device="cuda") + 16) // 32, 40, torch.float32)


def test_embedding_of_other_tokens():
    """Tokens outside the table: zeros, no part of a gradient, and a flag."""
    from mlcg_amd import ops

    ops.numerics_flags(clear=True)
    tokens = torch.tensor([0, 5, -1, 4, 2 ** 40, 5, -2 ** 50, 1], device="cuda")
    with torch.no_grad():
        ops.scaled_embedding(torch.ones(5, 4, device="cuda"), tokens % 5)
    assert int(ops.numerics_flags(clear=False)[0]) == 0
    out, _ = _embed_check(5, tokens, 20, torch.float32)
    assert not bool(out[[1, 2, 4, 5, 6]].any())
    with pytest.raises(Exception):
        ops.check_numerics()
    ops.numerics_flags(clear=True)


def test_embedding_values():
    """A row's NaN stays with its token."""
    from mlcg_amd import ops

    tokens = torch.arange(200, device="cuda") % 5
    grad = torch.ones(200, 16, device="cuda")
    grad[7] = float("nan")
    dt = ops.scaled_embedding_backward(grad, ops.token_order(tokens, 6))
    assert bool(torch.isnan(dt[2]).all()) and not bool(dt[5].any())
    assert torch.equal(dt[[0, 1, 3, 4]], torch.full((4, 16), 40.0, device="cuda"))


def test_embedding_refusals():
    from mlcg_amd import nn, ops

    table, tokens = torch.zeros(5, 8, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    for args in ((table, tokens.int()), (table, tokens[None]), (table, tokens.cpu()),
                 (table.double(), tokens), (table[0], tokens), (table[:0], tokens),
                 (torch.zeros(2, 8193, device="cuda"), tokens)):
        with pytest.raises(RuntimeError):
            nn.scaled_embedding(*args)
    order = ops.token_order(tokens, 5)
    for grad in (torch.zeros(3, 8, device="cuda"), torch.zeros(4, 8), torch.zeros(4, device="cuda"),
                 torch.zeros(4, 8, device="cuda").double()):
        with pytest.raises(RuntimeError):
            ops.scaled_embedding_backward(grad, order)
    for rows in (0, 2 ** 30):
        with pytest.raises(RuntimeError):
            ops.token_order(tokens, rows)


def test_recorded_and_replayed():
    from mlcg_amd import ops

    x, r, w, gy, gt = _rms_case(300, 96, torch.bfloat16, torch.float32)
    table = torch.randn(300, 96, device="cuda").bfloat16()
    tokens = torch.randint(0, 300, (300,), device="cuda")

    def work():
        e = ops.scaled_embedding(table, tokens, 3.0)
        y, t, rstd = ops.rms_norm_add(e, r, w)
        dx, dr, dw = ops.rms_norm_add_backward(gy, gt, t, w, rstd)
        order = ops.token_order(tokens, 300)
        return [e, y, t, dx, dr, dw, order.keys, order.index,
                ops.scaled_embedding_backward(dx, order, 3.0)]

    work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = work()
    torch.cuda.synchronize()
    for i in range(4):
        tokens.copy_(torch.randint(0, 300 if i % 2 else 3, (300,), device="cuda"))
        table.copy_(torch.randn(300, 96, device="cuda"))
        graph.replay()
        want = work()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), i


def test_other_derivatives_are_refused():
    from torch.autograd import forward_ad

    from mlcg_amd import nn

    tokens = torch.arange(6, device="cuda") % 4
    w = torch.ones(16, device="cuda")
    calls = [lambda t: nn.rms_norm_add(t, None, w)[0], lambda t: nn.rms_norm_add(w[None], t[:1], w)[0],
             lambda t: nn.rms_norm_add(t, t * 2, w)[1], lambda t: nn.scaled_embedding(t, tokens, 2.0)]
    for f in calls:
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(torch.randn(4, 16, device="cuda"),
                                        torch.randn(4, 16, device="cuda"))
            with pytest.raises((RuntimeError, NotImplementedError)):
                f(dual)
        leaf = torch.randn(4, 16, device="cuda", requires_grad=True)
        out = f(leaf)
        (d,) = torch.autograd.grad(out, leaf, torch.ones_like(out), create_graph=True,
                                   allow_unused=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(d.sum(), leaf)


def test_gradients_of_other_layouts():
    """Gradients that autograd hands on as one number for all, or as a transpose."""
    from mlcg_amd import nn

    x, r, w, gy, gt = _rms_case(33, 40, torch.bfloat16, torch.float32)
    table = torch.randn(5, 40, device="cuda")
    tokens = torch.arange(33, device="cuda") % 5
    for turn in (lambda g: torch.ones((), dtype=g.dtype, device="cuda").expand_as(g),
                 lambda g: g.t().contiguous().t()):
        grads = []
        for how in (turn, lambda g: turn(g).contiguous()):
            leaf = [t.detach().requires_grad_(True) for t in (x, r, w, table)]
            y, t = nn.rms_norm_add(*leaf[:3])
            e = nn.scaled_embedding(leaf[3], tokens, 3.0)
            grads.append(torch.autograd.grad([y, t, e], leaf, [how(gy), how(gt), how(gt)]))
        for a, b in zip(*grads):
            assert torch.equal(a, b)


def test_elements_past_31_bits():
    """Rows whose elements lie past 2^31: their results are those of the rows alone
    (of a row nothing depends on the others but the weight's gradient)."""
    from mlcg_amd import ops

    n, width = 2 ** 22 + 21, 512
    x = torch.ones(n, width, dtype=torch.bfloat16, device="cuda")
    last = slice(n - 21, n)
    x[last].normal_()
    w = torch.randn(width, device="cuda").bfloat16()
    y, _, rstd = ops.rms_norm_add(x, None, w)
    want = ops.rms_norm_add(x[last], None, w)
    assert torch.equal(y[last], want[0]) and torch.equal(rstd[last], want[2])
    dx = ops.rms_norm_add_backward(y, None, x, w, rstd)[0]
    assert torch.equal(dx[last], ops.rms_norm_add_backward(y[last], None, x[last], w,
                                                           rstd[last])[0])
    del y, dx, rstd
    tokens = torch.zeros(n, dtype=torch.int64, device="cuda")
    tokens[last] = torch.arange(21, device="cuda") + 1
    table = torch.randn(22, width, device="cuda").bfloat16()
    out = ops.scaled_embedding(table, tokens, 2.0)
    assert torch.equal(out[last], 2 * table[1:])
    dt = ops.scaled_embedding_backward(x, ops.token_order(tokens, 22), 2.0)
    assert torch.equal(dt[1:], 2 * x[last])
    assert torch.equal(dt[0].float(), torch.full((width,), 2.0 ** 23, device="cuda"))
    # a table whose rows lie past 2^31
    del out, dt
    tokens = torch.tensor([n - 1, 3, n - 21, n - 1], device="cuda")
    assert torch.equal(ops.scaled_embedding(x, tokens, 0.5), 0.5 * x[tokens])
    dt = ops.scaled_embedding_backward(x[:4].contiguous(), ops.token_order(tokens, n), 1.0)
    assert torch.equal(dt[n - 1], x[0] + x[3]) and torch.equal(dt[n - 21], x[2])
    assert not bool(dt[4:n - 21].any()) and not bool(dt[n - 20:n - 1].any())


def test_two_streams_at_once():
    from mlcg_amd import nn

    cases = [_rms_case(20000, 128, torch.float32, torch.float32, seed) for seed in (0, 1)]
    tokens = [torch.randint(0, 9, (20000,), device="cuda") for _ in cases]

    def work(c, tok):
        x, r, w, gy, gt = c
        leaf = [t.detach().requires_grad_(True) for t in (x, r, w, x[:9])]
        outs = [*nn.rms_norm_add(*leaf[:3]), nn.scaled_embedding(leaf[3], tok, 2.0)]
        return [*outs, *torch.autograd.grad(outs, leaf, [gy, gt, gy])]

    want = [work(c, t) for c, t in zip(cases, tokens)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for s, c, t in zip(streams, cases, tokens):
            with torch.cuda.stream(s):
                got.append(work(c, t))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for p, q in zip(a, b):
                assert torch.equal(p, q)
