"""The gated delta rule (ops.gated_delta, its gradients and its step) against
float64 bead by bead (oracle/delta_ref.py).

Tolerances.  With u half a step of the arrays' type (2^-24, 2^-11, 2^-8) an output
in it is rounded once: u |value|.  Inside, operands of the products are held to
p = 2^-17 (16-bit arrays) or 2^-24 (fp32).  A value passes through five products,
each with two operands that are rounded (10 p), whose sums have up to 64 + 128
terms (fp32 additions, 2^-24 sqrt(192) at least in the mean, below 14 p), and
where 1 + A is inverted the errors of up to four blocks add up (4 x 10 p): 64 p
of the size of the terms, which is the largest value of the tensor.  A decay's
gradient is the sum of D S over the state, of terms of both signs: of the
largest sum of their sizes, |D| |S| <= |D|_F |S|_F.  A longer chain adds nothing: the
state forgets.  A gradient through the length of q or k is r (d - u (u.d)): two terms of
size r |d| that cancel (for one channel but for the small addend), each off by the
64 p that d itself is: of r |d|, where that is the larger.  fp16 values below 2^-14 round by 2^-25 absolutely.
"""

import pytest
import torch

from oracle import delta_ref as R

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
U = {t: torch.finfo(t).eps / 2 for t in TYPES}  # 2^-24, 2^-11, 2^-8
P = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -17, torch.bfloat16: 2.0 ** -17}


def _case(lengths, heads, keys, dk, dv, dtype, seed=0, keep=False, state=False, views=True):
    from mlcg_amd import ops

    g = torch.Generator().manual_seed(seed)
    n = sum(lengths)
    if views:  # slices of one projection
        x = torch.randn(n, 2 * keys * dk + heads * dv, generator=g).to(dtype).cuda()
        q, k, v = x.split([keys * dk, keys * dk, heads * dv], 1)
        q, k, v = q.unflatten(1, (keys, dk)), k.unflatten(1, (keys, dk)), v.unflatten(
            1, (heads, dv))
    else:
        q, k, v = (torch.randn(n, h, d, generator=g).to(dtype).cuda()
                   for h, d in ((keys, dk), (keys, dk), (heads, dv)))
    c = dict(q=q, k=k, v=v,
             decay=(-torch.exp(-6 * torch.rand(n, heads, generator=g))).cuda(),
             beta=torch.rand(n, heads, generator=g).cuda(),
             chains=ops.chain_layout(lengths, "cuda"),
             keep=(torch.rand(n, generator=g) < 0.8).cuda() if keep else None,
             state=torch.randn(len(lengths), heads, dk, dv, generator=g).cuda() if state else None,
             reverse=False, normalize=True, scale=None)
    c["grad"] = torch.randn(n, heads, dv, generator=g).to(dtype).cuda()
    c["grad_last"] = torch.randn(len(lengths), heads, dk, dv, generator=g).cuda()
    return c


def _run(c, grads=True):
    """{name: value} of the operator, and with grads of its gradients."""
    from mlcg_amd import nn

    names = [n for n in ("q", "k", "v", "decay", "beta", "state") if c[n] is not None]
    leaf = {n: c[n].detach().requires_grad_(grads) for n in names}
    out, last = nn.gated_delta(leaf["q"], leaf["k"], leaf["v"], leaf["decay"], leaf["beta"],
                               c["chains"], c["scale"], c["keep"], leaf.get("state"),
                               c["reverse"], c["normalize"])
    got = {"out": out.detach(), "last": last.detach()}
    if grads:
        got.update(zip(names, torch.autograd.grad([out, last], list(leaf.values()),
                                                  [c["grad"], c["grad_last"]])))
    return got


def _oracle(c):
    return R.gated_delta(c["q"], c["k"], c["v"], c["decay"], c["beta"], c["chains"].lengths,
                         c["scale"], c["keep"], c["state"], c["reverse"], c["normalize"],
                         c["grad"], c["grad_last"])


def _within(got, ref, name, u, p, size=None, tiny=0.0):
    got = got.cpu().double()
    assert got.shape == ref.shape, name
    if ref.numel() == 0:
        return
    bound = u * ref.abs() + 64 * p * (float(ref.abs().max()) if size is None else size) + tiny
    d = (got - ref).abs()
    assert bool((d <= bound).all()), (
        f"{name}: {int((~(d <= bound)).sum())} of {d.numel()} off, worst "
        f"{float((d / bound).max()):.3f} of the bound, {float(d.max()):.3e}")


def _check(c, got=None, ref=None):
    got = _run(c) if got is None else got
    ref = _oracle(c) if ref is None else ref
    dtype = c["q"].dtype
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for name, t in got.items():
        size = None
        if name == "decay":  # |D|_F |S|_F, D and S at most as large as at the chains' ends
            size = max([1.0] + [float(x.flatten(2).norm(dim=2).max()) for x in
                                (ref["last"], c["grad_last"].cpu().double())]) ** 2
            size = max(size, float(ref["decay"].abs().max()))
        elif name in ("q", "k"):
            size = max(float(ref[name].abs().max()) if t.numel() else 0.0, ref[name + "_size"])
        own = t.dtype == dtype
        _within(t, ref[name], name, U[dtype] if own else 2.0 ** -24, P[dtype], size,
                tiny if own else 0.0)
    return got


LENGTHS = {
    "one": [1],
    "ones": [1, 1, 1, 2, 1],
    "gaps": [0, 5, 0, 0, 33, 0],
    "short": [35, 10, 7, 31, 32],
    "chunks": [63, 64, 65, 127, 128, 129, 1],
    "long": [700, 3, 257],
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", sorted(LENGTHS))
def test_lengths(lengths, dtype):
    print(f"delta {lengths} {dtype}", flush=True)
    _check(_case(LENGTHS[lengths], 2, 2, 32, 32, dtype, state=True))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dk,dv", [(1, 1), (5, 16), (16, 5), (24, 40), (32, 128), (33, 17),
                                   (64, 64), (96, 100), (127, 33), (128, 128)])
def test_head_dims(dk, dv, dtype):
    print(f"delta dims {dk} {dv} {dtype}", flush=True)
    _check(_case([70, 1, 33], 3, 1, dk, dv, dtype, seed=dk))


@pytest.mark.parametrize("heads,keys", [(1, 1), (4, 4), (4, 2), (6, 1), (8, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shared_heads(heads, keys, dtype):
    print(f"delta heads {heads}/{keys} {dtype}", flush=True)
    _check(_case([90, 140], heads, keys, 16, 16, dtype, seed=heads, keep=True))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("keep", [False, True])
def test_options(keep, normalize, reverse, dtype):
    print(f"delta options {keep} {normalize} {reverse} {dtype}", flush=True)
    c = _case([129, 0, 40, 64], 2, 1, 32, 48, dtype, keep=keep, state=True)
    c["reverse"], c["normalize"] = reverse, normalize
    if not normalize:  # |k|^2 beta < 2, so that the state does not grow
        c["q"], c["k"] = c["q"] / 8, c["k"] / 8
        c["scale"] = -0.7
    _check(c)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("chunks", [1, 2, 3])
def test_segments(monkeypatch, chunks, dtype):
    """A long chain in segments that run at the same time, against the same rule
    and against one segment."""
    from mlcg_amd import ops

    print(f"delta segments {chunks} {dtype}", flush=True)
    c = _case([700, 64, 1, 0, 330], 4, 2, 40, 72, dtype, keep=True, state=True)
    c["reverse"] = chunks == 2
    monkeypatch.setattr(ops, "_delta_segment_tiles", lambda *a: chunks)
    a = _check(c)
    for name, t in _run(c).items():
        assert torch.equal(t, a[name]), name


@pytest.mark.parametrize("dtype", TYPES)
def test_wide_segments(monkeypatch, dtype):
    from mlcg_amd import ops

    print(f"delta wide segments {dtype}", flush=True)
    monkeypatch.setattr(ops, "_delta_segment_tiles", lambda *a: 2)
    for dk, dv in ((128, 128), (64, 64), (16, 16)):
        _check(_case([400], 1, 1, dk, dv, dtype, state=True))


@pytest.mark.parametrize("dtype", TYPES)
def test_absent_beads(dtype):
    """Whatever an absent bead's rows hold; a chain without any bead; its
    gradients are exact zeros."""
    c = _case([100, 70, 64], 2, 2, 32, 32, dtype, keep=True, state=True)
    c["keep"][100:170] = False
    off = ~c["keep"]
    c = {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in c.items()}
    plain = _run(c)
    c["k"][off], c["v"][off] = float("nan"), float("inf")
    c["decay"][off], c["beta"][off] = float("nan"), float("inf")
    got = _run(c)
    for name, t in plain.items():
        assert torch.equal(t, got[name]), name
    for name in ("k", "v", "decay", "beta"):
        assert not bool(got[name][off].any()), name
    assert torch.equal(got["last"][1], c["state"][1])
    clean = dict(c, k=c["k"].masked_fill(off[:, None, None], 0.0),
                 v=c["v"].masked_fill(off[:, None, None], 0.0),
                 decay=c["decay"].masked_fill(off[:, None], 0.0),
                 beta=c["beta"].masked_fill(off[:, None], 0.0))
    _check(clean, got=got)


def test_chains_do_not_meet():
    """A chain's NaN stays in it, and rows behind the last one are left alone."""
    c = _case([70, 64, 30], 2, 2, 32, 32, torch.float32, state=True, views=False)
    plain = _run(c)
    for name in ("q", "k", "v", "decay", "beta", "grad"):
        c[name][70:134] = float("nan")
    got = _run(c)
    for name in ("out", "q", "k", "v", "decay", "beta"):
        assert torch.equal(plain[name][:70], got[name][:70]), name
        assert torch.equal(plain[name][134:], got[name][134:]), name
    for name in ("last", "state"):
        assert torch.equal(plain[name][[0, 2]], got[name][[0, 2]]), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decays(dtype):
    """Factors from 1 to 0, and none left of one in the middle of a chunk: what
    follows does not feel how much was forgotten before.  Sums of 64 logarithms
    of up to 256 in fp32 alone would be off by 2^-11."""
    c = _case([200, 64], 2, 2, 32, 32, dtype, state=True)
    d = c["decay"]
    d[3], d[40], d[41], d[90], d[130] = 0.0, float("-inf"), -1e30, -200.0, -103.5
    d[64:90, 0] = -40.0
    d[10:30, 1] = -300.0
    got = _check(c)
    assert not bool(got["decay"][40].any()) and not bool(got["decay"][41].any())
    assert bool(torch.isfinite(got["state"]).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_keys(dtype):
    """Every key the same and beta 1: 1 + A is all ones below its diagonal, the
    products of whose powers have no digits left; each bead replaces the one
    before.  beta of 0 writes nothing and has a gradient."""
    c = _case([150], 2, 1, 32, 32, dtype)
    c["k"][:] = c["k"][:1].clone()
    c["beta"][:] = 1.0
    c["beta"][70:75] = 0.0
    c["decay"][:] = -1e-3
    got = _check(c)
    assert bool(got["beta"][72].any())


def test_zero_rows():
    """Keys and queries of zero, which have no direction: the small addend gives
    them zeros."""
    c = _case([70], 2, 2, 16, 16, torch.float32)
    c["k"][5:9], c["q"][7:11] = 0.0, 0.0
    got = _check(c)
    assert not bool(got["out"][7:11].any())


@pytest.mark.parametrize("scale", [2.0 ** -18, 2.0 ** 8])
def test_fp16_gradients_of_any_size(scale):
    """Gradients near fp16's smallest and largest numbers keep their digits inside:
    fp32's outputs are the scaled ones."""
    c = _case([150, 20], 2, 2, 32, 32, torch.float16)
    c["grad_last"] *= 0.0
    big = _run(c)
    c["grad"] = (c["grad"].float() * scale).to(torch.float16)
    c2 = dict(c)
    got = _run(c2)
    ref = _oracle(c2)
    for name in ("decay", "beta"):
        d = (got[name].cpu().double() - ref[name]).abs().max()
        assert float(d) <= 64 * 2.0 ** -17 * float(ref[name].abs().max()) * 32, name
    assert float(big["beta"].abs().max()) > 0


def test_strides_and_alignment():
    from mlcg_amd import nn

    for dtype in TYPES:
        c = _case([90, 33], 4, 4, 32, 32, dtype, views=False)
        want = _run(c)
        odd = {}
        for name in ("q", "k", "v"):
            t = c[name]
            room = torch.full((t.shape[0] + 1, 5, 33), float("nan"), dtype=dtype, device="cuda")
            room[1:, :4, 1:] = t
            odd[name] = room[1:, :4, 1:]  # rows that begin at odd elements
        got = _run(dict(c, **odd))
        for name, t in want.items():
            assert torch.equal(t, got[name]), name
        turned = {name: c[name].permute(2, 0, 1).contiguous().permute(1, 2, 0)
                  for name in ("q", "k", "v")}
        got = _run(dict(c, **turned))
        for name, t in want.items():
            assert torch.equal(t, got[name]), name
        # one row's values for all heads, and gates as one head's views
        one = c["k"][:, :1].expand(-1, 4, -1)
        a = nn.gated_delta(c["q"], one, c["v"], c["decay"][:, :1].expand(-1, 4), c["beta"],
                           c["chains"])[0]
        b = nn.gated_delta(c["q"], one.contiguous(), c["v"],
                           c["decay"][:, :1].expand(-1, 4).contiguous(), c["beta"], c["chains"])[0]
        assert torch.equal(a, b)


def test_gradients_against_differences():
    """Central differences of the kernel's own outputs in fp32: with steps of 2^-6
    the curvature's part is 2^-12 relative, the outputs' rounding 2^-24 64 / 2^-6
    of the summed output."""
    from mlcg_amd import nn

    c = _case([70, 5], 2, 1, 8, 8, torch.float32, state=True, keep=True)
    got = _run(c)

    def value(d):
        out, last = nn.gated_delta(d["q"], d["k"], d["v"], d["decay"], d["beta"], c["chains"],
                                   keep=c["keep"], state=d["state"])
        return float((out.double() * c["grad"].double()).sum()
                     + (last.double() * c["grad_last"].double()).sum())

    g = torch.Generator().manual_seed(3)
    h = 2.0 ** -6
    for name in ("q", "k", "v", "decay", "beta", "state"):
        way = torch.randn(c[name].shape, generator=g).cuda()
        way /= way.norm()
        up, down = dict(c), dict(c)
        up[name], down[name] = c[name] + h * way, c[name] - h * way
        slope = (value(up) - value(down)) / (2 * h)
        want = float((got[name].double() * way.double()).sum())
        size = float(got[name].norm())
        assert abs(slope - want) <= 2e-3 * size + 1e-3, (name, slope, want, size)


def test_outputs_alone():
    """A gradient of one of the two outputs, of some of the inputs."""
    from mlcg_amd import nn

    c = _case([70, 64], 2, 2, 16, 32, torch.float32)
    for which in (0, 1):
        v = c["v"].detach().requires_grad_(True)
        state = torch.zeros(2, 2, 16, 32, device="cuda", requires_grad=True)
        o = nn.gated_delta(c["q"], c["k"], v, c["decay"], c["beta"], c["chains"], state=state)
        grad = (c["grad"], c["grad_last"])[which]
        dv, ds = torch.autograd.grad(o[which], [v, state], grad)
        z = {"grad": c["grad"] * 0, "grad_last": c["grad_last"] * 0}
        z[("grad", "grad_last")[which]] = grad
        full = _run(dict(c, state=state.detach(), **z))
        assert torch.equal(dv, full["v"]) and torch.equal(ds, full["state"])


def test_without_beads():
    c = _case([0, 0], 2, 2, 16, 16, torch.float32, state=True)
    got = _run(c)
    assert torch.equal(got["last"], c["state"]) and torch.equal(got["state"], c["grad_last"])
    assert got["q"].shape == (0, 2, 16) and got["out"].shape == (0, 2, 16)
    c = _case([0, 3, 0], 2, 2, 16, 16, torch.float32)
    got = _run(c)
    assert not bool(got["last"][[0, 2]].any())
    _check(c, got=got)


def test_equal_calls_give_equal_bits():
    for dtype in TYPES:
        c = _case([300, 64, 7], 4, 2, 64, 64, dtype, keep=True, state=True)
        first = _run(c)
        assert torch.equal(first["out"], _run(c, grads=False)["out"])
        for _ in range(3):
            for name, t in _run(c).items():
                assert torch.equal(t, first[name]), name


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,heads,keys,dk,dv", [
    (1, 1, 1, 1, 1), (3, 4, 2, 32, 32), (5, 2, 1, 128, 128), (2, 1, 1, 7, 33), (2, 2, 2, 128, 127),
    (70, 3, 3, 64, 20), (1, 1, 1, 128, 1), (2, 2, 1, 16, 4)])
def test_step(batch, heads, keys, dk, dv, dtype):
    from mlcg_amd import ops

    print(f"step {batch} {heads}/{keys} {dk} {dv} {dtype}", flush=True)
    c = _case([1] * batch, heads, keys, dk, dv, dtype, state=True)
    for normalize in (True, False):
        ref = R.gated_delta(c["q"], c["k"], c["v"], c["decay"], c["beta"], [1] * batch,
                            state=c["state"], normalize=normalize)
        args = [c[n] for n in ("q", "k", "v", "decay", "beta")]
        into = torch.full_like(c["state"], float("nan"))
        out = ops.gated_delta_step(*args, c["state"], normalize=normalize, into=into)
        size = float(c["k"].float().norm(dim=2).max()) ** 2 if not normalize else 1.0
        for got, want, u in ((out, ref["out"], U[dtype]), (into, ref["last"], 2.0 ** -24)):
            tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
            _within(got, want, "step", u, 2.0 ** -24 * max(1.0, size), tiny=tiny)
        state = c["state"].clone()
        assert torch.equal(out, ops.gated_delta_step(*args, state, normalize=normalize))
        assert torch.equal(state, into)


def test_steps_make_a_chain():
    """A chain by single beads, against the same beads in chunks: roundings of
    either, 64 p of the largest value each."""
    from mlcg_amd import ops

    n, dtype = 130, torch.bfloat16
    c = _case([n, n, n], 4, 2, 32, 40, dtype, state=True)
    out, last, _ = ops.gated_delta(c["q"], c["k"], c["v"], c["decay"], c["beta"], c["chains"],
                                   state=c["state"])
    state, rows = c["state"].clone(), torch.arange(3, device="cuda") * n
    got = [ops.gated_delta_step(*[c[x][rows + t] for x in ("q", "k", "v", "decay", "beta")], state)
           for t in range(n)]
    got = torch.stack(got, 1).flatten(0, 1)
    _within(got, out.cpu().double(), "out", 2 * U[dtype], 2 * P[dtype])
    _within(state, last.cpu().double(), "last", 0.0, 2 * P[dtype])


def test_refusals():
    from mlcg_amd import nn, ops

    c = _case([5, 3], 4, 2, 16, 16, torch.float32, state=True)
    good = {n: c[n] for n in ("q", "k", "v", "decay", "beta", "chains", "keep", "state")}
    bad = dict(
        q=[c["q"][:, :, :8], c["q"][:7], c["q"].half(), c["q"].double(), c["q"][:, 0]],
        k=[c["k"].half(), c["k"][:, :1]],
        v=[c["v"][:, :3], c["v"][:7], c["v"].half(), c["v"].cpu()],
        decay=[c["decay"].half(), c["decay"][:, :2], c["decay"][:7], c["decay"].cpu()],
        beta=[c["beta"].double(), c["beta"][:, :2]],
        chains=[ops.chain_layout([5, 3], "cpu"), ops.chain_layout([5, 4], "cuda"), [5, 3]],
        keep=[torch.ones(7, dtype=torch.bool, device="cuda"), torch.ones(8, device="cuda"),
              torch.ones(8, dtype=torch.bool)],
        state=[c["state"][:1], c["state"].half(), c["state"].cpu()])
    for name, values in bad.items():
        for value in values:
            with pytest.raises(RuntimeError):
                nn.gated_delta(**dict(good, **{name: value}))
    wide = torch.zeros(8, 1, 129, device="cuda")
    with pytest.raises(RuntimeError):
        nn.gated_delta(wide, wide, wide, c["decay"][:, :1], c["beta"][:, :1], c["chains"])
    args = [c[n] for n in ("q", "k", "v", "decay", "beta")]
    state = torch.zeros(8, 4, 16, 16, device="cuda")
    for s, into in ((state[:7], None), (state.half(), None), (state.cpu(), None),
                    (torch.zeros(8, 4, 16, 32, device="cuda")[..., ::2], None),
                    (state, state[:7]), (state, state.double())):
        with pytest.raises(RuntimeError):
            ops.gated_delta_step(*args, s, into=into)
    room = torch.zeros(9, 4, 16, 16, device="cuda")
    with pytest.raises(RuntimeError, match="overlap"):
        ops.gated_delta_step(*args, room[:8], into=room[1:])
    out, last, kept = ops.gated_delta(*args, c["chains"], train=False)
    with pytest.raises(RuntimeError, match="kept"):
        ops.gated_delta_backward(*args, c["chains"], kept, c["grad"])


def test_recorded_and_replayed():
    """Forward, backward and step in one graph, replayed with other inputs between
    eager calls of the same sizes; two graphs do not share workspaces."""
    from mlcg_amd import ops

    c = _case([200, 64, 5], 4, 2, 32, 32, torch.bfloat16, keep=True, state=True)
    s = torch.randn(8, 4, 32, 32, device="cuda")
    args = [c[n] for n in ("q", "k", "v", "decay", "beta")]

    def work():
        out, last, kept = ops.gated_delta(*args, c["chains"], keep=c["keep"], state=c["state"],
                                          train=True)
        grads = ops.gated_delta_backward(*args, c["chains"], kept, c["grad"], c["grad_last"],
                                         keep=c["keep"], want_state=True)
        into = torch.empty_like(s)
        o = ops.gated_delta_step(*[t[:8] for t in args], s, into=into)
        return [out, last, *grads, o, into]

    work()
    graphs = []
    for _ in range(2):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs = work()
        graphs.append((graph, outs))
    torch.cuda.synchronize()
    for i in range(4):
        c["q"].copy_(torch.randn_like(c["q"]))
        c["decay"].mul_(0.9)
        for graph, _ in graphs:
            graph.replay()
        want = work()
        torch.cuda.synchronize()
        for _, outs in graphs:
            for a, b in zip(outs, want):
                assert torch.equal(a, b), i


def test_other_stream():
    c = _case([300, 64], 4, 4, 32, 32, torch.float32, state=True)
    want = _run(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(c)
    side.synchronize()
    for name, t in want.items():
        assert torch.equal(t, got[name]), name


def test_other_derivatives_are_refused():
    from torch.autograd import forward_ad

    from mlcg_amd import nn, ops

    c = _case([5, 3], 4, 2, 16, 16, torch.float32, state=True, views=False)
    names = ("q", "k", "v", "decay", "beta", "state")
    for name in names:
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(c[name].clone(), torch.ones_like(c[name]))
            args = dict({n: c[n] for n in names}, **{name: dual})
            with pytest.raises((RuntimeError, NotImplementedError)):
                nn.gated_delta(chains=c["chains"], **args)
        args = dict({n: c[n] for n in names}, **{name: c[name].clone().requires_grad_(True)})
        out = nn.gated_delta(chains=c["chains"], **args)[0]
        (d,) = torch.autograd.grad(out, args[name], torch.ones_like(out), create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(d.sum(), args[name])
        with pytest.raises(RuntimeError, match="no gradients"):
            ops.gated_delta_step(*[t[:8] for t in list(args.values())[:5]],
                                 torch.zeros(8, 4, 16, 16, device="cuda",
                                             requires_grad=name == "state"))


@pytest.mark.parametrize("dtype", TYPES)
def test_states_that_grow(dtype):
    """Decays above zero: the rule as it is written, over one chunk."""
    c = _case([64, 17], 2, 1, 32, 32, dtype, state=True)
    c["decay"] = c["decay"].abs() / 8
    _check(c)


def test_elements_past_31_bits():
    """Values, outputs, gradients and operands that lie past 2^31 elements: the last
    chain's are those that it has alone."""
    from mlcg_amd import ops

    length, chains, heads = 101, 2600, 64  # 262600 beads x 64 heads x 128 > 2^31
    n, g = length * chains, torch.Generator(device="cuda").manual_seed(3)
    q, k = (torch.randn(n, 1, 32, device="cuda", generator=g).bfloat16() for _ in range(2))
    v = torch.randn(n, heads, 128, device="cuda", dtype=torch.bfloat16, generator=g)
    decay = -torch.rand(n, heads, device="cuda", generator=g)
    beta = torch.rand(n, heads, device="cuda", generator=g)
    results = []
    for at, count in ((slice(0, n), chains), (slice(n - length, n), 1)):
        args = [t[at] for t in (q, k, v, decay, beta)]
        lay = ops.chain_layout([length] * count, "cuda")
        out, last, kept = ops.gated_delta(*args, lay, train=True)
        grads = ops.gated_delta_backward(*args, lay, kept, args[2], last)
        results.append([t[-length:].clone() for t in (out, *grads[:5])] + [last[-1:].clone()])
        del out, last, kept, grads
    for name, a, b in zip(("out", "q", "k", "v", "decay", "beta", "last"), *results):
        assert torch.equal(a, b), name


def test_two_streams_at_once():
    cases = [_case([300, 64, 1], 4, 2, 32, 32, torch.bfloat16, seed, state=True)
             for seed in (0, 1)]
    want = [_run(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(_run(c))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for name in b:
                assert torch.equal(a[name], b[name]), name


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,keys,d", [(4, 4, 16), (4, 2, 64), (2, 1, 128)])
def test_sixteen_bit_arrays_keep_their_digits(monkeypatch, heads, keys, d, dtype):
    """16-bit arrays are exact in one or two pieces, and what is computed from them
    has three: states and the gates' gradients, which are fp32, are as far off as those
    of fp32 arrays (p = 2^-24), the other outputs by their own rounding more."""
    monkeypatch.setitem(P, dtype, 2.0 ** -24)
    _check(_case([130, 64, 7], heads, keys, d, d, dtype, state=True))
