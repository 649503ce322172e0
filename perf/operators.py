"""The sequence encoder's operators: what they are measured on, their plain
forms and their values in 64 bits.

Beads of all chains lie one after the other ([S, ...], channels last); the
lengths of the chains say where each one ends.

  attn   attention of every bead to the beads of its own chain.  The logits
         are  scale q.k + table[bucket(clip(pos_k - pos_q, -R, R)), head],
         pos the bead's index in its chain or its residue number; a bead
         that `keep` marks as absent is no key (a chain without any present
         bead gives zeros).  `kv` key/value heads serve `heads` query heads.
  norm   group norm of a chain (statistics over its beads and the channels of
         a group, biased variance), an affine map by channel, an activation
  drop   dropout and a residual sum: y = residual + x keep / (1 - p'), the
         mask from Philox4x32-10 with the key `seed` and the counter
         (element // 8, step); element e takes bits 16 (e % 8) ... of the 128
         and is kept where they are at least t = round(65536 p), p' = t / 65536

``train`` asks for the gradients of every input too.
"""

import math

import numpy as np
import torch

own = False

SPECIES = 20  # bead types, and residues' kinds


# ---------------------------------------------------------------------------
# cases

def _attn(name, chains, beads, heads, dim, dtype, train, **more):
    case = dict(name=name, kind="attn", chains=chains, beads=beads, ragged=False, heads=heads,
                kv=heads, dim=dim, dtype=dtype, train=train, buckets=32, reach=128, log=True,
                keep=False, residues=False)
    case.update(more)
    return case


def _norm(name, chains, beads, width, groups, dtype, act, train, ragged=False):
    return dict(name=name, kind="norm", chains=chains, beads=beads, ragged=ragged, width=width,
                groups=groups, dtype=dtype, act=act, train=train)


def _drop(name, rows, width, dtype, p, train, residual=True):
    return dict(name=name, kind="drop", rows=rows, width=width, dtype=dtype, p=p, train=train,
                residual=residual)


def listed():
    return [
        # one chain of 35 beads before a simulation of it: the smallest call
        _attn("attn_infer_1x35_f32", 1, 35, 4, 32, "float32", False),
        # the molecules of a data set, several beads to a residue, in the
        # type that force fields are trained in
        _attn("attn_train_48x268_f32", 48, 268, 8, 16, "float32", True, ragged=True,
              residues=True, buckets=65, reach=32, log=False),
        # a batch of many short chains in 16 bits
        _attn("attn_train_512x100_bf16", 512, 100, 4, 32, "bfloat16", True, ragged=True),
        # a few large proteins in 32 bits: bound by the products
        _attn("attn_train_4x1031_f32", 4, 1031, 4, 32, "float32", True),
        # one large complex with unresolved beads, shared key/value heads
        _attn("attn_infer_1x8191_bf16", 1, 8191, 8, 64, "bfloat16", False, kv=2, keep=True),
        # two of half its size in training
        _attn("attn_train_2x4099_bf16", 2, 4099, 8, 64, "bfloat16", True, keep=True),
        # the features of one small protein
        _norm("norm_infer_1x35_f32", 1, 35, 128, 8, "float32", "tanh", False),
        # an ordinary batch of several molecules
        _norm("norm_train_192x80_f32", 192, 80, 128, 8, "float32", "ssp", True, ragged=True),
        # a large batch of the benchmark's 268-bead protein
        _norm("norm_train_2048x268_bf16", 2048, 268, 128, 32, "bfloat16", "silu", True,
              ragged=True),
        # one very long chain: few statistics, each over many beads
        _norm("norm_train_1x120001_f32", 1, 120001, 256, 8, "float32", "none", True),
        # the beads of the benchmark's training batch
        _drop("drop_train_17920x128_f32", 17920, 128, "float32", 0.1, True),
        # a large batch in 16 bits
        _drop("drop_train_548864x128_bf16", 548864, 128, "bfloat16", 0.2, True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "norm", "norm", "drop"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    train = rng.random() < 0.65
    if kind == "attn":
        dim = rng.choice([16, 24, 32, 48, 64, 128])
        heads = rng.choice([1, 2, 4, 6, 8])
        if heads * dim > 512:
            heads = 4
        beads = _log_int(rng, 1, 4099 if train else 8191)
        pairs = (2 * 4099 ** 2 if train else 8191 ** 2) * 512
        chains = _log_int(rng, 1, max(1, min(512, pairs // (beads ** 2 * heads * max(dim, 64)),
                                             200000 // beads)))
        case = _attn("", chains, beads, heads, dim, dtype, train, ragged=rng.random() < 0.6)
        case["kv"] = rng.choice([h for h in (1, 2, heads) if heads % h == 0])
        case["log"] = rng.random() < 0.6
        case["reach"] = rng.choice([16, 32, 100, 128])
        case["buckets"] = rng.choice([16, 32, 47]) if case["log"] else 2 * case["reach"] + 1
        case["keep"] = rng.random() < 0.4
        case["residues"] = rng.random() < 0.3
    elif kind == "norm":
        width = rng.choice([64, 96, 128, 129, 256, 320])
        groups = rng.choice([g for g in (1, 3, 4, 8, 32, width) if width % g == 0])
        rows = _log_int(rng, 1, 120001 * 256 // width)
        chains = _log_int(rng, 1, min(2048, rows))
        case = _norm("", chains, max(1, rows // chains), width, groups, dtype,
                     rng.choice(["none", "tanh", "ssp", "silu"]), train, rng.random() < 0.6)
    else:
        width = rng.choice([64, 96, 128, 129, 256, 77])
        most = 548864 * (64 if dtype == "float32" else 128) // width
        case = _drop("", _log_int(rng, 1, most), width, dtype,
                     rng.choice([0.0, 0.05, 0.1, 0.25, 0.5]), train, rng.random() < 0.7)
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
    if case["kind"] == "attn":
        lens = _lengths(case)
        s, pairs = int(lens.sum()), int((lens * lens).sum())
        row = case["heads"] * case["dim"]
        q, kv = s * row, s * case["kv"] * case["dim"]
        table = case["buckets"] * case["heads"]
        read, products = 2 * q + 2 * kv + table, 2  # q, k, v, table; out
        if case["train"]:
            read, products = read + 2 * q + 2 * kv + table, 7  # grad out; dq, dk, dv, dtable
        more = s * (int(case["keep"]) + 4 * int(case["residues"]))
        return {"bytes": size * read + more, "flops": 2 * products * pairs * row}
    if case["kind"] == "norm":
        n = int(_lengths(case).sum()) * case["width"]
        return {"bytes": size * (n * (4 if case["train"] else 2)
                                 + case["width"] * (4 if case["train"] else 2)),
                "flops": n * (20 if case["train"] else 8)}
    n = case["rows"] * case["width"]
    return {"bytes": size * n * (2 + int(case["residual"]) + (2 if case["train"] else 0)),
            "flops": n * (20 if case["train"] else 10)}


# ---------------------------------------------------------------------------
# inputs

def _bucket_of(buckets, reach, log):
    """bucket_of[d + reach]: the bucket of every clipped offset d.  Clipped
    offsets have one each; in the logarithmic scheme half of the buckets
    serve each direction, a half of these the offsets below their number and
    the rest larger ones in equal ratios, up to `reach`."""
    d = np.arange(-reach, reach + 1)
    if not log:
        return (d + reach).astype(np.int64)
    side = buckets // 2
    near = max(1, side // 2)
    out = []
    for v in d:
        a = abs(int(v))
        if a >= near:
            ratio = math.log(a / near) / math.log(reach / near) if reach > near else 1.0
            a = min(side - 1, near + int(ratio * (side - near) + 1e-9))
        out.append(min(a, side - 1) + (side if v > 0 else 0))
    return np.asarray(out, dtype=np.int64)


def _residues(lens, rng):
    """Residue numbers of beads in chains: one to five beads a residue, with
    numbers left out where a loop is not resolved."""
    out = []
    for n in lens:
        step = (rng.random(n) < 0.4).astype(np.int64)
        step += (rng.random(n) < 0.01) * 7
        out.append(np.cumsum(step))
    return np.concatenate(out)


def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _inputs(case, seed):
    """The arrays of a case: made from the seed alone, for run and exact."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng([seed, 11])
    dtype = getattr(torch, case["dtype"])
    out = {}
    if case["kind"] == "attn":
        lens = _lengths(case)
        s, h, kv, d = int(lens.sum()), case["heads"], case["kv"], case["dim"]
        # one projection's output, as the encoder has it: q, k and v are views
        qkv = _randn(gen, (s, h + 2 * kv, d), dtype)
        out["q"], out["k"], out["v"] = qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:]
        out["table"] = _randn(gen, (case["buckets"], h), dtype, 0.5)
        out["grad"] = _randn(gen, (s, h, d), dtype)
        out["keep"] = out["residues"] = None
        if case["keep"]:
            out["keep"] = torch.from_numpy(rng.random(s) < 0.9).cuda()
        if case["residues"]:
            out["residues"] = torch.from_numpy(_residues(lens, rng)).to(torch.int32).cuda()
    elif case["kind"] == "norm":
        s, c = int(_lengths(case).sum()), case["width"]
        # features of beads by type: types differ in offset and spread
        types = torch.from_numpy(rng.integers(0, SPECIES, s)).cuda()
        x = torch.randn((s, c), generator=gen, device="cuda")
        x += torch.randn((SPECIES, c), generator=gen, device="cuda").index_select(0, types)
        out["x"] = x.to(dtype)
        out["weight"] = _randn(gen, (c,), dtype, 0.2) + 1
        out["bias"] = _randn(gen, (c,), dtype, 0.2)
        out["grad"] = _randn(gen, (s, c), dtype)
    else:
        shape = (case["rows"], case["width"])
        out["x"] = _randn(gen, shape, dtype)
        out["residual"] = _randn(gen, shape, dtype) if case["residual"] else None
        out["grad"] = _randn(gen, shape, dtype)
        out["seed"] = int(rng.integers(0, 1 << 62))
        out["step"] = torch.tensor([int(rng.integers(0, 1 << 40))], device="cuda")
    return out


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if case["kind"] != "drop":
        lens = _lengths(case)
        if own:
            from mlcg_amd import ops
            state["chains"] = ops.chain_layout(lens, device="cuda")
        else:  # where each chain's beads lie in a rectangle, and back
            at = np.concatenate([[0], np.cumsum(lens)[:-1]])
            col = np.arange(int(lens.max()))
            valid = col[None, :] < lens[:, None]
            state["pad"] = torch.from_numpy(np.where(valid, at[:, None] + col, 0)).cuda()
            state["valid"] = torch.from_numpy(valid).cuda()
            state["count"] = torch.from_numpy(lens).cuda()
    if case["kind"] == "attn":
        if own:
            from mlcg_amd import ops
            state["buckets"] = ops.relative_buckets(
                case["buckets"], case["reach"], "log" if case["log"] else "clip", device="cuda")
        else:
            state["buckets"] = torch.from_numpy(
                _bucket_of(case["buckets"], case["reach"], case["log"])).cuda()
    if own and case["train"]:
        for name in ("q", "k", "v", "table", "x", "weight", "bias", "residual"):
            if state.get(name) is not None:
                state[name] = state[name].detach().requires_grad_(True)
    return state


# ---------------------------------------------------------------------------
# the framework's operators

def _run_own(state):
    from mlcg_amd import nn

    case, names = state["case"], ("x", "residual")
    if case["kind"] == "attn":
        names = ("q", "k", "v", "table")
        out = nn.chain_attention(state["q"], state["k"], state["v"], state["table"],
                                 state["buckets"], state["chains"], keep=state["keep"],
                                 positions=state["residues"])
    elif case["kind"] == "norm":
        names = ("x", "weight", "bias")
        out = nn.group_norm_act(state["x"], state["weight"], state["bias"], case["groups"],
                                state["chains"], act=case["act"])
    else:
        out = nn.dropout_add(state["x"], case["p"], state["seed"], state["step"],
                             residual=state["residual"])
    result = {"out": out}
    if case["train"]:
        wanted = [n for n in names if state[n] is not None]
        grads = torch.autograd.grad(out, [state[n] for n in wanted], state["grad"])
        result["out"] = out.detach()
        result.update(("grad_" + n, g) for n, g in zip(wanted, grads))
    return result


# ---------------------------------------------------------------------------
# their plain forms

def _pad(state, t):
    """[S, ...] -> [chains, longest, ...] in 32 bits, zero past each end."""
    p = t.float().index_select(0, state["pad"].reshape(-1))
    p = p.reshape(*state["valid"].shape, *t.shape[1:])
    return p * state["valid"].reshape(*state["valid"].shape, *[1] * (t.dim() - 1))


def _plain_attn(state):
    case, valid = state["case"], state["valid"]
    dtype, h, kv = state["q"].dtype, case["heads"], case["kv"]
    n, length = valid.shape
    scale = 1.0 / math.sqrt(case["dim"])

    def heads(t, by):  # [S, by, D] -> [n, h, L, D]
        p = _pad(state, t).transpose(1, 2)
        return p.repeat_interleave(h // by, 1) if by != h else p

    present = valid
    if state["keep"] is not None:
        present = valid & state["keep"][state["pad"]]
    q = heads(state["q"], h)
    k = heads(state["k"], kv).masked_fill(~present[:, None, :, None], 0.0)
    v = heads(state["v"], kv).masked_fill(~present[:, None, :, None], 0.0)
    if state["residues"] is not None:
        pos = state["residues"].long()[state["pad"]]
    else:
        pos = torch.arange(length, device=valid.device)[None, :]
    offset = (pos[:, None, :] - pos[:, :, None]).clamp(-case["reach"], case["reach"])
    offset += case["reach"]
    by_offset = state["table"].float()[state["buckets"]]  # [2 reach + 1, h]
    logits = torch.matmul(q, k.transpose(2, 3)).mul_(scale)
    logits += by_offset.t()[:, offset].transpose(0, 1)
    logits.masked_fill_(~present[:, None, None, :], -math.inf)
    top = logits.amax(3, keepdim=True)
    p = logits.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = p.sum(3, keepdim=True)
    p = p.div_(total.masked_fill(total == 0.0, 1.0))
    o = torch.matmul(p, v)

    def packed(t):  # [n, h, L, D] -> [S, h, D]
        return t.transpose(1, 2)[valid].to(dtype)

    result = {"out": packed(o)}
    if not case["train"]:
        return result
    g = heads(state["grad"], h)
    dv = torch.matmul(p.transpose(2, 3), g)
    ds = torch.matmul(g, v.transpose(2, 3))
    ds = ds.sub_((p * ds).sum(3, keepdim=True)).mul_(p)  # 0 for a row of one key
    dq = torch.matmul(ds, k).mul_(scale)
    dk = torch.matmul(ds.transpose(2, 3), q).mul_(scale)
    shared = (n, kv, h // kv, length, case["dim"])
    by_row = torch.zeros(n, h, length, 2 * case["reach"] + 1, device=ds.device)
    by_row.scatter_add_(3, offset[:, None].expand(n, h, length, length), ds)
    dtable = torch.zeros(case["buckets"], h, device=ds.device)
    dtable.index_add_(0, state["buckets"], by_row.sum((0, 2)).t().contiguous())
    result.update(grad_q=packed(dq), grad_k=packed(dk.reshape(shared).sum(2)),
                  grad_v=packed(dv.reshape(shared).sum(2)), grad_table=dtable.to(dtype))
    return result


def _act(z, act):
    """The activation and its derivative."""
    if act == "tanh":
        y = torch.tanh(z)
        return y, 1.0 - y * y
    s = 1.0 / (1.0 + torch.exp(-z))
    if act == "silu":
        return z * s, s * (1.0 + z * (1.0 - s))
    if act == "ssp":
        return z.clamp_min(0.0) + torch.log1p(torch.exp(-z.abs())) - math.log(2.0), s
    return z, torch.ones_like(z)


def _plain_norm(state):
    case, valid, dtype = state["case"], state["valid"], state["x"].dtype
    n, length = valid.shape
    groups, width = case["groups"], case["width"]
    split = (n, length, groups, width // groups)
    inside = valid[:, :, None, None]
    count = (state["count"] * (width // groups)).reshape(n, 1, 1, 1).float()
    x = _pad(state, state["x"]).reshape(split)
    mean = x.sum((1, 3), keepdim=True) / count
    centred = (x - mean) * inside
    rstd = 1.0 / torch.sqrt(centred.square().sum((1, 3), keepdim=True) / count + 1e-5)
    hat = centred * rstd
    weight = state["weight"].float().reshape(split[2:])
    z = hat * weight + state["bias"].float().reshape(split[2:])
    y, slope = _act(z, case["act"])
    result = {"out": y.reshape(n, length, width)[valid].to(dtype)}
    if not case["train"]:
        return result
    dz = _pad(state, state["grad"]).reshape(split) * slope
    dhat = dz * weight
    dx = dhat - dhat.sum((1, 3), keepdim=True) / count
    dx = (dx - hat * ((dhat * hat).sum((1, 3), keepdim=True) / count)) * rstd
    result.update(grad_x=dx.reshape(n, length, width)[valid].to(dtype),
                  grad_weight=(dz * hat).sum((0, 1)).reshape(width).to(dtype),
                  grad_bias=dz.sum((0, 1)).reshape(width).to(dtype))
    return result


def _philox(counter, step, seed):
    """The four 32-bit words of every counter, as int64 arrays: products of
    two words wrap in 64 bits, and their upper halves are masked."""
    low = 0xFFFFFFFF
    c = [counter & low, counter >> 32, (step & low).expand_as(counter),
         ((step >> 32) & low).expand_as(counter)]
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):  # the generator's ten rounds
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & low) ^ c[1] ^ k0, b & low, ((a >> 32) & low) ^ c[3] ^ k1, a & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return c


def _plain_drop(state):
    case, x = state["case"], state["x"]
    t = int(round(case["p"] * 65536))
    counter = torch.arange((x.numel() + 7) // 8, device=x.device)
    words = torch.stack(_philox(counter, state["step"], state["seed"]), 1)
    halves = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:x.numel()]
    factor = (halves >= t).float().mul_(65536.0 / (65536 - t)).reshape(x.shape)
    y = x.float() * factor
    if state["residual"] is not None:
        y += state["residual"].float()
    result = {"out": y.to(x.dtype)}
    if case["train"]:
        result["grad_x"] = (state["grad"].float() * factor).to(x.dtype)
        if state["residual"] is not None:
            result["grad_residual"] = state["grad"]
    return result


def run(state):
    if own:
        return _run_own(state)
    return {"attn": _plain_attn, "norm": _plain_norm, "drop": _plain_drop}[
        state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# their values in 64 bits, one chain and one head at a time

def _exact_attn(case, a):
    f8 = torch.float64
    lens, h, group = _lengths(case), case["heads"], case["heads"] // case["kv"]
    reach, scale = case["reach"], case["dim"] ** -0.5
    bucket = torch.from_numpy(_bucket_of(case["buckets"], reach, case["log"])).cuda()
    q, k, v, g = (a[n].to(f8) for n in ("q", "k", "v", "grad"))
    table = a["table"].to(f8)
    out, dq = torch.zeros_like(q), torch.zeros_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    dtable = torch.zeros_like(table)
    start = 0
    for n in lens.tolist():
        rows = slice(start, start + n)
        start += n
        pos = (a["residues"][rows].long() if a["residues"] is not None
               else torch.arange(n, device="cuda"))
        cell = bucket[(pos.unsqueeze(0) - pos.unsqueeze(1)).clamp(-reach, reach) + reach]
        absent = None if a["keep"] is None else ~a["keep"][rows]
        for head in range(h):
            kk, vv = k[rows, head // group], v[rows, head // group]
            logit = q[rows, head] @ kk.t() * scale + table[:, head][cell]
            if absent is not None:
                logit[:, absent] = -math.inf
            lse = torch.logsumexp(logit, 1, keepdim=True)
            prob = torch.where(lse == -math.inf, 0.0, torch.exp(logit - lse))
            out[rows, head] = prob @ vv
            if case["train"]:
                go = g[rows, head]
                dp = go @ vv.t()
                ds = prob * (dp - (prob * dp).sum(1, keepdim=True))
                dq[rows, head] = ds @ kk * scale
                dk[rows, head // group] += ds.t() @ q[rows, head] * scale
                dv[rows, head // group] += prob.t() @ go
                dtable[:, head] += torch.bincount(cell.reshape(-1), ds.reshape(-1),
                                                  case["buckets"])
    result = {"out": out}
    if case["train"]:
        result.update(grad_q=dq, grad_k=dk, grad_v=dv, grad_table=dtable)
    return result


def _exact_norm(case, a):
    x, g, weight, bias = (a[n].double() for n in ("x", "grad", "weight", "bias"))
    s, width = x.shape
    groups, per = case["groups"], case["width"] // case["groups"]
    out, dx = torch.empty_like(x), torch.empty_like(x)
    dweight, dbias = torch.zeros_like(weight), torch.zeros_like(bias)
    start = 0
    for n in _lengths(case).tolist():
        rows = slice(start, start + n)
        start += n
        t = x[rows].reshape(n, groups, per)
        var, mean = torch.var_mean(t, (0, 2), correction=0, keepdim=True)
        inv = (var + 1e-5).rsqrt()
        hat = ((t - mean) * inv).reshape(n, width)
        z = (hat * weight + bias).requires_grad_(True)
        with torch.enable_grad():
            y = {"tanh": torch.tanh, "silu": torch.nn.functional.silu,
                 "ssp": lambda u: torch.logaddexp(u, torch.zeros_like(u)) - math.log(2.0),
                 "none": lambda u: u * 1.0}[case["act"]](z)
            (dz,) = torch.autograd.grad(y, z, g[rows])
        out[rows] = y.detach()
        dweight += (dz * hat).sum(0)
        dbias += dz.sum(0)
        e, hg = (dz * weight).reshape(n, groups, per), hat.reshape(n, groups, per)
        e = e - e.mean((0, 2), keepdim=True) - hg * (e * hg).mean((0, 2), keepdim=True)
        dx[rows] = (e * inv).reshape(n, width)
    result = {"out": out}
    if case["train"]:
        result.update(grad_x=dx, grad_weight=dweight, grad_bias=dbias)
    return result


def _exact_drop(case, a):
    shape = tuple(a["x"].shape)
    n = shape[0] * shape[1]
    step, seed = int(a["step"].item()), a["seed"]
    word = np.uint64(0xFFFFFFFF)
    half = np.uint64(32)
    i = np.arange(-(-n // 8), dtype=np.uint64)
    x0, x1 = i & word, i >> half
    x2 = np.full_like(i, step % 2 ** 32)
    x3 = np.full_like(i, step // 2 ** 32)
    for r in range(10):
        key0 = np.uint64((seed + r * 0x9E3779B9) % 2 ** 32)
        key1 = np.uint64((seed // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32)
        m0, m1 = x0 * np.uint64(0xD2511F53), x2 * np.uint64(0xCD9E8D57)
        x0, x1, x2, x3 = (m1 >> half) ^ x1 ^ key0, m1 & word, (m0 >> half) ^ x3 ^ key1, m0 & word
    bits = np.stack([x0, x1, x2, x3], 1).astype("<u4").view("<u2").reshape(-1)[:n]
    t = int(round(case["p"] * 65536))
    kept = torch.from_numpy((bits >= t).reshape(shape)).cuda()
    scale = 65536.0 / (65536 - t)
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    out = torch.where(kept, a["x"].double() * scale, zero)
    if a["residual"] is not None:
        out = out + a["residual"].double()
    result = {"out": out}
    if case["train"]:
        result["grad_x"] = torch.where(kept, a["grad"].double() * scale, zero)
        if a["residual"] is not None:
            result["grad_residual"] = a["grad"].double()
    return result


def exact(case, seed):
    a = _inputs(case, seed)
    return {"attn": _exact_attn, "norm": _exact_norm, "drop": _exact_drop}[case["kind"]](case, a)
