"""The operators of the encoder of linear cost: what they are measured on,
their plain forms and their values in 64 bits.

  delta  the gated delta rule along every chain.  A head's state S, Dk x Dv,
         goes from bead to bead,
             S <- e^g S,  S <- S + beta k (v - S^T k)^T,  o = scale S^T q,
         forwards or from the last bead to the first; q and k may be brought to
         length one (x / sqrt(x.x + 1e-6)) before.  Beads that `keep` marks as
         absent leave the state as it is.  `keys` heads of q and k serve
         `heads` of v, the decay g and beta.  With `state` a chain begins at a
         given state and its last one is an output too.
  step   one more bead of every chain: the rule above on states held in memory
  rms    t = x + residual, y = t / sqrt(mean t^2 + 1e-6) weight, over the
         channels of a row; x may be in 16 bits beside a residual in 32
  embed  rows of a table by token, times a factor

``train`` asks for the gradients of every input too.
"""

import math

import numpy as np
import torch

own = False

EPS = 1e-6


# ---------------------------------------------------------------------------
# cases

def _delta(name, chains, beads, heads, keys, dk, dv, dtype, train, **more):
    case = dict(name=name, kind="delta", chains=chains, beads=beads, ragged=False, heads=heads,
                keys=keys, dk=dk, dv=dv, dtype=dtype, train=train, normalize=True, keep=False,
                state=False, reverse=False)
    case.update(more)
    return case


def _step(name, chains, heads, keys, dk, dv, dtype):
    return dict(name=name, kind="step", chains=chains, heads=heads, keys=keys, dk=dk, dv=dv,
                dtype=dtype, normalize=True, train=False)


def _rms(name, rows, width, dtype, residual, train):
    return dict(name=name, kind="rms", rows=rows, width=width, dtype=dtype, residual=residual,
                train=train)


def _embed(name, rows, tokens, width, dtype, train, skewed=False):
    return dict(name=name, kind="embed", rows=rows, tokens=tokens, width=width, dtype=dtype,
                train=train, skewed=skewed)


def listed():
    return [
        # one chain of 35 beads before a simulation of it: the smallest call
        _delta("delta_infer_1x35_f32", 1, 35, 4, 4, 32, 32, "float32", False),
        # the molecules of a data set in the type that force fields are
        # trained in, some of their beads unresolved
        _delta("delta_train_48x268_f32", 48, 268, 8, 8, 16, 16, "float32", True, ragged=True,
               keep=True),
        # a batch of many short chains in 16 bits, from their last bead
        _delta("delta_train_512x100_bf16", 512, 100, 4, 4, 32, 32, "bfloat16", True, ragged=True,
               reverse=True),
        # two large proteins, two heads on each key head
        _delta("delta_train_2x4099_bf16", 2, 4099, 8, 4, 64, 64, "bfloat16", True),
        # a very large complex in one piece, its state kept for what follows
        _delta("delta_infer_1x120001_bf16", 1, 120001, 8, 8, 64, 64, "bfloat16", False,
               state=True),
        # chains that grow, a bead each at a time: few, and many with wide heads
        _step("step_16_f32", 16, 4, 4, 32, 32, "float32"),
        _step("step_1024_bf16", 1024, 8, 4, 64, 128, "bfloat16"),
        # the features of one small protein
        _rms("rms_infer_35x128_f32", 35, 128, "float32", "float32", False),
        # the beads of the benchmark's training batch
        _rms("rms_train_17920x128_f32", 17920, 128, "float32", "float32", True),
        # a large batch in 16 bits beside a residual stream in 32
        _rms("rms_train_262144x512_bf16", 262144, 512, "bfloat16", "float32", True),
        # bead types of the benchmark's training batch
        _embed("embed_train_17920x128_f32", 25, 17920, 128, "float32", True, skewed=True),
        # words of three residues of a large batch
        _embed("embed_train_548864x256_bf16", 8000, 548864, 256, "bfloat16", True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["delta", "delta", "delta", "step", "rms", "embed"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    train = rng.random() < 0.6
    if kind in ("delta", "step"):
        dk, dv = rng.choice([16, 24, 32, 48, 64, 128]), rng.choice([16, 32, 40, 64, 128])
        heads = rng.choice([1, 2, 4, 6, 8])
        keys = rng.choice([h for h in (1, 2, heads) if heads % h == 0])
    if kind == "delta":
        size = heads * max(dk, 32) * max(dv, 32)
        most = (2 * 4099 if train else 120001) * 8 * 64 * 64 // size
        beads = _log_int(rng, 1, min(4099 if train else 60000, most))
        chains = _log_int(rng, 1, max(1, min(512, most // beads)))
        case = _delta("", chains, beads, heads, keys, dk, dv, dtype, train,
                      ragged=rng.random() < 0.6, normalize=rng.random() < 0.8,
                      keep=rng.random() < 0.4, state=rng.random() < 0.4,
                      reverse=rng.random() < 0.4)
    elif kind == "step":
        most = 1024 * 8 * 64 * 128 // (heads * dk * dv)
        case = _step("", _log_int(rng, 1, min(4096, most)), heads, keys, dk, dv, dtype)
        case["normalize"] = rng.random() < 0.8
    elif kind == "rms":
        width = rng.choice([64, 77, 96, 128, 129, 256, 320, 512, 1000, 2048])
        residual = rng.choice(["none", dtype, "float32"])
        case = _rms("", _log_int(rng, 1, 262144 * 512 // width // 2), width, dtype, residual,
                    train)
    else:
        width = rng.choice([64, 77, 96, 128, 129, 256, 320])
        case = _embed("", _log_int(rng, 1, 100000), _log_int(rng, 1, 548864 * 64 // width),
                      width, dtype, train, rng.random() < 0.5)
    del case["name"]
    return case


def _lengths(case):
    """The chains' lengths: the same for every seed (shapes go by the case)."""
    chains, beads = case["chains"], case["beads"]
    if not case["ragged"]:
        return np.full(chains, beads, dtype=np.int64)
    rng = np.random.default_rng([chains, beads])
    lens = rng.integers(max(1, beads // 8), beads + 1, chains)
    lens[rng.integers(0, chains)] = beads
    return lens


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] in ("delta", "step"):
        state = 4 * case["chains"] * case["heads"] * case["dk"] * case["dv"]
        s = case["chains"] if case["kind"] == "step" else int(_lengths(case).sum())
        qk, v = 2 * s * case["keys"] * case["dk"], s * case["heads"] * case["dv"]
        gates = 2 * s * case["heads"]
        products = s * case["heads"] * case["dk"] * case["dv"]
        total = size * (qk + 2 * v) + 4 * gates  # q, k, v, out; decay, beta
        if case["kind"] == "step" or case["state"]:
            total += 2 * state
        if case["train"]:  # grad out; grads of q, k, v, decay and beta
            total += size * (qk + 2 * v) + 4 * gates + (2 * state if case["state"] else 0)
        if case["kind"] == "delta" and case["keep"]:
            total += s
        return {"bytes": total, "flops": (18 if case["train"] else 6) * products}
    if case["kind"] == "rms":
        n = case["rows"] * case["width"]
        rsize = size if case["residual"] == "none" else (
            4 if case["residual"] == "float32" else 2)
        total = n * 2 * size + case["width"] * size  # x, y, weight
        if case["residual"] != "none":
            total += n * 2 * rsize  # residual, t
        if case["train"]:  # grads of y and of t; of x, of the residual, of the weight
            total += n * 2 * size + case["width"] * size
            if case["residual"] != "none":
                total += n * 2 * rsize
        return {"bytes": total, "flops": n * (12 if case["train"] else 5)}
    n, table = case["tokens"] * case["width"], case["rows"] * case["width"]
    total = size * (n + min(n, table)) + 8 * case["tokens"]
    if case["train"]:
        total += size * (n + table)
    return {"bytes": total, "flops": n * (2 if case["train"] else 1)}


# ---------------------------------------------------------------------------
# inputs

def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _inputs(case, seed):
    """The arrays of a case: made from the seed alone, for run and exact."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng([seed, 13])
    dtype = getattr(torch, case["dtype"])
    out = {}
    if case["kind"] in ("delta", "step"):
        s = case["chains"] if case["kind"] == "step" else int(_lengths(case).sum())
        h, kh, dk, dv = case["heads"], case["keys"], case["dk"], case["dv"]
        # one projection's output, as the encoder has it: q, k and v are views
        qkv = _randn(gen, (s, 2 * kh * dk + h * dv), dtype)
        if not case["normalize"]:
            qkv[:, :2 * kh * dk] *= dk ** -0.5
        out["q"] = qkv[:, :kh * dk].unflatten(1, (kh, dk))
        out["k"] = qkv[:, kh * dk:2 * kh * dk].unflatten(1, (kh, dk))
        out["v"] = qkv[:, 2 * kh * dk:].unflatten(1, (h, dv))
        # memories of two to a thousand beads; keys longer than one by chance
        # (not brought to one) are written in part, so that no state grows
        rate = torch.rand((s, h), generator=gen, device="cuda") * math.log(512.0)
        out["decay"] = -0.5 * torch.exp(-rate)
        out["beta"] = torch.sigmoid(torch.randn((s, h), generator=gen, device="cuda"))
        if not case["normalize"]:
            out["beta"] *= 0.5
        out["grad"] = _randn(gen, (s, h, dv), dtype)
        out["state"] = out["grad_state"] = out["keep"] = None
        if case["kind"] == "step" or case["state"]:
            shape = (case["chains"], h, dk, dv)
            out["state"] = _randn(gen, shape, torch.float32, dk ** -0.5)
            out["grad_state"] = _randn(gen, shape, torch.float32, dk ** -0.5)
        if case["kind"] == "delta" and case["keep"]:
            out["keep"] = torch.from_numpy(rng.random(s) < 0.9).cuda()
    elif case["kind"] == "rms":
        shape = (case["rows"], case["width"])
        out["x"] = _randn(gen, shape, dtype)
        out["residual"] = out["grad_t"] = None
        if case["residual"] != "none":
            rtype = getattr(torch, case["residual"])
            out["residual"] = _randn(gen, shape, rtype, 2.0)
            out["grad_t"] = _randn(gen, shape, rtype)
        out["weight"] = _randn(gen, shape[1:], dtype, 0.2) + 1
        out["grad"] = _randn(gen, shape, dtype)
    else:
        rows, n = case["rows"], case["tokens"]
        out["table"] = _randn(gen, (rows, case["width"]), dtype)
        if case["skewed"]:  # some tokens are common, most are rare
            tokens = np.minimum(rng.zipf(1.3, n) - 1, rng.integers(0, rows, n))
        else:
            tokens = rng.integers(0, rows, n)
        out["tokens"] = torch.from_numpy(tokens.astype(np.int64)).cuda()
        out["scale"] = math.sqrt(case["width"])
        out["grad"] = _randn(gen, (n, case["width"]), dtype)
    return out


LEAVES = {"delta": ("q", "k", "v", "decay", "beta", "state"),
          "rms": ("x", "residual", "weight"), "embed": ("table",)}


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if case["kind"] == "delta":
        lens = _lengths(case)
        if own:
            from mlcg_amd import ops
            state["chains"] = ops.chain_layout(lens, device="cuda")
        else:  # where each chain's beads lie in a rectangle of whole chunks
            state["pad"], state["valid"] = _rectangle(case, CHUNK)
    elif case["kind"] == "step":
        state["next"] = torch.empty_like(state["state"])
    if own and case["train"]:
        for name in LEAVES[case["kind"]]:
            if state[name] is not None:
                state[name] = state[name].detach().requires_grad_(True)
    return state


def _rectangle(case, multiple):
    """Bead indices [chains, columns] in the order of the rule, and whether a
    column is a bead."""
    lens = _lengths(case)
    at = np.concatenate([[0], np.cumsum(lens)[:-1]])[:, None]
    col = np.arange(-(-int(lens.max()) // multiple) * multiple)[None, :]
    valid = col < lens[:, None]
    bead = at + (lens[:, None] - 1 - col if case["reverse"] else col)
    return (torch.from_numpy(np.where(valid, bead, 0)).cuda(), torch.from_numpy(valid).cuda())


# ---------------------------------------------------------------------------
# the framework's operators

def _run_own(state):
    from mlcg_amd import nn, ops

    case = state["case"]
    if case["kind"] == "step":
        out = ops.gated_delta_step(state["q"], state["k"], state["v"], state["decay"],
                                   state["beta"], state["state"], normalize=case["normalize"],
                                   into=state["next"])
        return {"out": out, "state": state["next"]}
    if case["kind"] == "delta":
        out, last = nn.gated_delta(state["q"], state["k"], state["v"], state["decay"],
                                   state["beta"], state["chains"], keep=state["keep"],
                                   state=state["state"], reverse=case["reverse"],
                                   normalize=case["normalize"])
        result, cotangents = {"out": out}, [state["grad"]]
        if case["state"]:
            result["state"] = last
            cotangents.append(state["grad_state"])
    elif case["kind"] == "rms":
        y, t = nn.rms_norm_add(state["x"], state["residual"], state["weight"], eps=EPS)
        result, cotangents = {"out": y}, [state["grad"]]
        if state["residual"] is not None:
            result["t"] = t
            cotangents.append(state["grad_t"])
    else:
        out = nn.scaled_embedding(state["table"], state["tokens"], state["scale"])
        result, cotangents = {"out": out}, [state["grad"]]
    if case["train"]:
        wanted = [n for n in LEAVES[case["kind"]] if state[n] is not None]
        grads = torch.autograd.grad(list(result.values()), [state[n] for n in wanted], cotangents)
        result = {name: t.detach() for name, t in result.items()}
        result.update(("grad_" + n, g) for n, g in zip(wanted, grads))
    return result


# ---------------------------------------------------------------------------
# their plain forms

CHUNK = 64


def _unit(t):
    return t / torch.sqrt((t * t).sum(-1, keepdim=True) + EPS)


def _by_chunk(t):
    """[chains, columns, H, ...] -> [chains, H, chunks, CHUNK, ...]"""
    n, columns, h = t.shape[:3]
    t = t.reshape(n, columns // CHUNK, CHUNK, h, *t.shape[3:])
    return t.permute(0, 3, 1, 2, *range(4, t.dim()))


def _plain_delta(state):
    """The rule in chunks of 64 beads.  Inside a chunk, with G the sum of g up
    to a bead and A_ts = beta_t e^(G_t - G_s) k_t.k_s for s < t,
    (1 + A) u = beta (v - e^G S^T k) gives what the beads add to the state."""
    case, valid, pad = state["case"], state["valid"], state["pad"]
    names = [n for n in LEAVES["delta"] if state[n] is not None]
    leaf = {n: state[n].detach().requires_grad_(case["train"]) for n in names}
    group = case["heads"] // case["keys"]
    present = valid if state["keep"] is None else valid & state["keep"][pad]

    def rows(name, mask):
        t = leaf[name].float()[pad]
        return t.masked_fill(~mask.reshape(*mask.shape, *[1] * (t.dim() - 2)), 0.0)

    with torch.set_grad_enabled(case["train"]):
        q, k, v = rows("q", valid), rows("k", present), rows("v", present)
        if case["normalize"]:
            q, k = _unit(q), _unit(k)
        q, k = (_by_chunk(t.repeat_interleave(group, 2)) for t in (q, k))
        v, g, beta = (_by_chunk(t) for t in (v, rows("decay", present), rows("beta", present)))
        total = g.double().cumsum(3)
        gap = total[..., :, None] - total[..., None, :]
        lower = torch.ones(CHUNK, CHUNK, device=q.device).tril().bool()
        e = torch.exp(gap.masked_fill(~lower, -math.inf)).float()
        a = (torch.matmul(k, k.transpose(3, 4)) * e).tril(-1) * beta[..., None]
        eye = torch.eye(CHUNK, device=q.device)
        with torch.no_grad():  # the inverse, row by row
            inv = eye.expand_as(a).clone()
            for i in range(1, CHUNK):
                inv[..., i, :i] = -torch.matmul(a[..., i:i + 1, :i], inv[..., :i, :i])[..., 0, :]
        inv = 2.0 * inv - torch.matmul(inv, torch.matmul(eye + a, inv))  # and its derivative
        scores = torch.matmul(q, k.transpose(3, 4)) * e
        first = torch.exp(total).float()[..., None]
        rest = torch.exp(total[..., -1:] - total).float()[..., None]
        own_u = torch.matmul(inv, beta[..., None] * v)
        from_s = torch.matmul(inv, beta[..., None] * first * k)
        q_first, k_rest = q * first, (k * rest).transpose(3, 4)
        if "state" in leaf:
            s = leaf["state"]
        else:
            s = q.new_zeros(case["chains"], case["heads"], case["dk"], case["dv"])
        outs = []
        for c in range(q.shape[2]):
            u = own_u[:, :, c] - torch.matmul(from_s[:, :, c], s)
            outs.append(torch.matmul(q_first[:, :, c], s) + torch.matmul(scores[:, :, c], u))
            s = first[:, :, c, -1:] * s + torch.matmul(k_rest[:, :, c], u)
        out = torch.cat(outs, 2).transpose(1, 2)[valid] * case["dk"] ** -0.5
        # where the rectangle's beads stand in the packed array
        out = out.new_zeros(out.shape).index_copy(0, pad[valid], out)
    result, cotangents = {"out": out}, [state["grad"].float()]
    if case["state"]:
        result["state"] = s
        cotangents.append(state["grad_state"])
    if case["train"]:
        grads = torch.autograd.grad(list(result.values()), [leaf[n] for n in names], cotangents)
        result.update(("grad_" + n, t) for n, t in zip(names, grads))
    result["out"] = result["out"].to(state["q"].dtype)
    return {name: t.detach() for name, t in result.items()}


def _plain_step(state):
    case = state["case"]
    group = case["heads"] // case["keys"]
    q, k = state["q"].float(), state["k"].float()
    if case["normalize"]:
        q, k = _unit(q), _unit(k)
    q, k = (t.repeat_interleave(group, 1).unsqueeze(3) for t in (q, k))
    s = state["state"] * torch.exp(state["decay"])[..., None, None]
    error = state["v"].float() - (s * k).sum(2)
    s = s + k * (state["beta"][..., None] * error).unsqueeze(2)
    out = (s * q).sum(2) * case["dk"] ** -0.5
    return {"out": out.to(state["q"].dtype), "state": s}


def _plain_rms(state):
    x, residual, dtype = state["x"], state["residual"], state["x"].dtype
    t = x.float() if residual is None else x.float() + residual.float()
    rstd = 1.0 / torch.sqrt((t * t).sum(1, keepdim=True) / t.shape[1] + EPS)
    hat, w = t * rstd, state["weight"].float()
    result = {"out": (hat * w).to(dtype)}
    if residual is not None:
        result["t"] = t.to(residual.dtype)
    if not state["case"]["train"]:
        return result
    g = state["grad"].float()
    dhat = g * w
    dt = (dhat - hat * ((dhat * hat).sum(1, keepdim=True) / t.shape[1])) * rstd
    if residual is not None:
        dt = dt + state["grad_t"].float()
    result["grad_x"] = dt.to(dtype)
    if residual is not None:
        result["grad_residual"] = dt.to(residual.dtype)
    result["grad_weight"] = (g * hat).sum(0).to(dtype)
    return result


def _plain_embed(state):
    table, tokens = state["table"], state["tokens"]
    result = {"out": (table.float()[tokens] * state["scale"]).to(table.dtype)}
    if state["case"]["train"]:
        total = torch.zeros(table.shape, dtype=torch.float64, device=table.device)
        total.index_add_(0, tokens, state["grad"].double())
        result["grad_table"] = (total * state["scale"]).to(table.dtype)
    return result


def run(state):
    if own:
        return _run_own(state)
    return {"delta": _plain_delta, "step": _plain_step, "rms": _plain_rms,
            "embed": _plain_embed}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# their values in 64 bits

def _exact_delta(case, a):
    """Bead by bead, for all chains and heads at once."""
    f8 = torch.float64
    group = case["heads"] // case["keys"]
    if case["kind"] == "step":
        at = torch.arange(case["chains"], device="cuda")[:, None]
        valid = torch.ones_like(at, dtype=torch.bool)
        train = False
    else:
        at, valid = _rectangle(case, 1)
        train = case["train"]
    names = [n for n in LEAVES["delta"] if a[n] is not None]
    leaf = {n: a[n].to(f8).requires_grad_(train) for n in names}
    with torch.set_grad_enabled(train):
        q, k = leaf["q"], leaf["k"]
        if case["normalize"]:
            q, k = (t * (t.square().sum(2, keepdim=True) + EPS).rsqrt() for t in (q, k))
        there = valid if a["keep"] is None else valid & a["keep"][at]
        # [columns, chains, heads, ...], zeros where the state stays as it is
        there = there.t()[:, :, None]
        at_t = at.t()
        none = torch.zeros((), dtype=f8, device="cuda")
        k = torch.where(there[..., None], k[at_t], none).repeat_interleave(group, 2)
        v = torch.where(there[..., None], leaf["v"][at_t], none)
        keep = torch.exp(torch.where(there, leaf["decay"][at_t], none))
        beta = torch.where(there, leaf["beta"][at_t], none)
        q = q[at_t].repeat_interleave(group, 2) * case["dk"] ** -0.5
        if "state" in leaf:
            s = leaf["state"]
        else:
            s = torch.zeros(case["chains"], case["heads"], case["dk"], case["dv"], dtype=f8,
                            device="cuda")
        outs = []
        # one column's factors at a time; slices of all of them are costly to
        # differentiate, unbind is not
        for qc, kc, vc, ac, bc in zip(q.unbind(0), k.unbind(0), v.unbind(0),
                                      keep.unbind(0), beta.unbind(0)):
            s = s * ac[..., None, None]
            read = torch.matmul(kc.unsqueeze(2), s).squeeze(2)
            s = s + kc.unsqueeze(3) * (bc[..., None] * (vc - read)).unsqueeze(2)
            outs.append(torch.matmul(qc.unsqueeze(2), s).squeeze(2))
        o = torch.stack(outs, 1)[valid]
        out = torch.zeros_like(leaf["v"]).index_copy(0, at[valid], o)
    result = {"out": out}
    if case["kind"] == "step" or case["state"]:
        result["state"] = s
    if train:
        cotangents = [a["grad"].to(f8)] + ([a["grad_state"].to(f8)] if case["state"] else [])
        grads = torch.autograd.grad(list(result.values()), [leaf[n] for n in names], cotangents)
        result.update(("grad_" + n, t) for n, t in zip(names, grads))
    return {name: t.detach() for name, t in result.items()}


def _exact_rms(case, a):
    f8 = torch.float64
    leaf = {n: a[n].to(f8).requires_grad_(case["train"])
            for n in LEAVES["rms"] if a[n] is not None}
    with torch.set_grad_enabled(case["train"]):
        t = leaf["x"] if "residual" not in leaf else leaf["x"] + leaf["residual"]
        y = t * (t.square().mean(1, keepdim=True) + EPS).rsqrt() * leaf["weight"]
    result, cotangents = {"out": y}, [a["grad"].to(f8)]
    if "residual" in leaf:
        result["t"] = t
        cotangents.append(a["grad_t"].to(f8))
    if case["train"]:
        grads = torch.autograd.grad(list(result.values()), list(leaf.values()), cotangents)
        result.update(("grad_" + n, g) for n, g in zip(leaf, grads))
    return {name: t.detach() for name, t in result.items()}


def _exact_embed(case, a):
    tokens = a["tokens"]
    result = {"out": a["table"].double().index_select(0, tokens) * a["scale"]}
    if case["train"]:
        order = torch.argsort(tokens)
        ends = torch.searchsorted(tokens[order], torch.arange(case["rows"], device="cuda"),
                                  right=True)
        running = torch.cumsum(a["grad"].double()[order], 0)
        running = torch.cat([running.new_zeros(1, running.shape[1]), running])[ends]
        before = torch.cat([running.new_zeros(1, running.shape[1]), running[:-1]])
        result["grad_table"] = (running - before) * a["scale"]
    return result


def exact(case, seed):
    a = _inputs(case, seed)
    if case["kind"] in ("delta", "step"):
        return _exact_delta(case, a)
    return {"rms": _exact_rms, "embed": _exact_embed}[case["kind"]](case, a)
