"""The operators of the encoder of linear cost in float64 on the CPU, from their
formulas: the gated delta rule bead by bead, with gradients written out, and the
sizes of the terms that rounding errors scale with."""

import torch

EPS = 1e-6


def _unit(x):
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) + EPS)


def _unit_grad(x, grad):
    """The gradient of x from that of x / sqrt(x.x + EPS)."""
    r = 1.0 / torch.sqrt((x * x).sum(-1, keepdim=True) + EPS)
    u = x * r
    return r * (grad - u * (u * grad).sum(-1, keepdim=True))


def gated_delta(q, k, v, decay, beta, lengths, scale=None, keep=None, state=None, reverse=False,
                normalize=True, grad=None, grad_last=None):
    """{"out", "last", and with grad "q", "k", "v", "decay", "beta", "state"}, and
    as "q_size" and "k_size" the largest term r |gradient of the unit vector| that
    the gradient through the lengths of q and k is a difference of."""
    def f8(t):
        return None if t is None else t.detach().cpu().double()

    q, k, v, decay, beta, state, grad, grad_last = map(
        f8, (q, k, v, decay, beta, state, grad, grad_last))
    keep = None if keep is None else keep.detach().cpu()
    group = v.shape[1] // q.shape[1]
    heads, dk, dv = v.shape[1], q.shape[2], v.shape[2]
    scale = dk ** -0.5 if scale is None else scale
    out = torch.zeros_like(v)
    last = torch.zeros(len(lengths), heads, dk, dv, dtype=torch.float64)
    if state is not None:
        last += state
    g = {n: torch.zeros_like(t) for n, t in
         (("q", q), ("k", k), ("v", v), ("decay", decay), ("beta", beta), ("state", last))}
    sizes = {"q_size": 0.0, "k_size": 0.0}

    def through_length(name, x, d):
        if not normalize:
            return d
        r = 1.0 / torch.sqrt((x * x).sum(-1, keepdim=True) + EPS)
        sizes[name] = max(sizes[name], float((r * d.norm(dim=-1, keepdim=True)).max()))
        return _unit_grad(x, d)

    if grad_last is not None:
        g["state"] += grad_last
    begin = 0
    for b, n in enumerate(lengths):
        beads = range(begin, begin + n)
        begin += n
        if reverse:
            beads = reversed(beads)
        beads = list(beads)
        S, seen = last[b].clone(), []
        for t in beads:
            qq, kk = (x[t].repeat_interleave(group, 0) for x in (q, k))
            if normalize:
                qq, kk = _unit(qq), _unit(kk)
            here = keep is None or bool(keep[t])
            before = S
            if here:
                a = torch.exp(decay[t])[:, None, None]
                d = torch.where(a == 0.0, 0.0, a * S)
                y = v[t] - (d * kk[:, :, None]).sum(1)
                S = d + kk[:, :, None] * (beta[t][:, None] * y)[:, None]
                seen.append((t, qq, kk, before, d, y, S))
            else:
                seen.append((t, qq, None, before, None, None, S))
            out[t] = scale * (S * qq[:, :, None]).sum(1)
        last[b] = S
        if grad is None:
            continue
        D = g["state"][b].clone()
        for t, qq, kk, before, d, y, S in reversed(seen):
            go = grad[t]
            dq = scale * (S * go[:, None]).sum(2)
            D = D + scale * qq[:, :, None] * go[:, None]
            dq = through_length("q_size", q[t].repeat_interleave(group, 0), dq)
            g["q"][t] = dq.reshape(-1, group, dk).sum(1)
            if kk is None:
                continue
            r = (D * kk[:, :, None]).sum(1)  # D^T k
            dk_ = (D * (beta[t][:, None] * y)[:, None]).sum(2)
            dy = beta[t][:, None] * r
            g["beta"][t] = (r * y).sum(1)
            g["v"][t] = dy
            dk_ = dk_ - (d * dy[:, None]).sum(2)
            dk_ = through_length("k_size", k[t].repeat_interleave(group, 0), dk_)
            g["k"][t] = dk_.reshape(-1, group, dk).sum(1)
            D = D - kk[:, :, None] * dy[:, None]
            g["decay"][t] = (D * d).sum((1, 2))
            a = torch.exp(decay[t])[:, None, None]
            D = torch.where(a == 0.0, 0.0, a * D)
        g["state"][b] = D
    result = {"out": out, "last": last}
    if grad is not None:
        result.update(g, **sizes)
    return result


def rms_norm_add(x, residual, weight, eps=EPS, grad=None, grad_t=None, stored=None):
    """{"y", "t", and with grad "x", "weight"}; the gradients are those at
    `stored` (t as it was rounded) where that is given."""
    x, weight = x.detach().cpu().double(), weight.detach().cpu().double()
    t = x if residual is None else x + residual.detach().cpu().double()
    rstd = 1.0 / torch.sqrt((t * t).mean(1, keepdim=True) + eps)
    result = {"y": t * rstd * weight, "t": t}
    if grad is not None:
        grad = grad.detach().cpu().double()
        if stored is not None:
            t = stored.detach().cpu().double()
        hat = t * rstd
        d = grad * weight
        dx = rstd * (d - hat * (d * hat).mean(1, keepdim=True))
        if grad_t is not None:
            dx = dx + grad_t.detach().cpu().double()
        result.update(x=dx, weight=(grad * hat).sum(0))
    return result


def scaled_embedding(table, tokens, scale, grad=None):
    table, tokens = table.detach().cpu().double(), tokens.cpu()
    ok = (tokens >= 0) & (tokens < table.shape[0])
    out = torch.where(ok[:, None], scale * table[tokens.clamp(0, table.shape[0] - 1)], 0.0)
    result = {"out": out}
    if grad is not None:
        g = torch.zeros_like(table)
        g.index_add_(0, tokens[ok], grad.detach().cpu().double()[ok])
        result["table"] = scale * g
        size = torch.zeros_like(table)
        size.index_add_(0, tokens[ok], grad.detach().cpu().double()[ok].abs())
        result["size"] = abs(scale) * size
    return result
