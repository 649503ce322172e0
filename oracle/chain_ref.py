"""The sequence encoder's operators in float64 on the CPU, from their
formulas, one chain and one head at a time, with the sizes of the terms that
their rounding errors scale with."""

import math

import numpy as np
import torch


def attention(q, k, v, table, bucket_of, lengths, scale=None, keep=None, positions=None,
              grad=None):
    """{"out", and with grad "q", "k", "v", "table"} and, under the same names,
    the sizes of the terms that a rounding of the probabilities, of dS and of
    the output (each by one part) moves the values by."""
    q, k, v, table = (t.detach().cpu().double() for t in (q, k, v, table))
    grad = None if grad is None else grad.detach().cpu().double()
    bucket = torch.as_tensor(bucket_of, dtype=torch.int64).cpu()
    reach = (bucket.numel() - 1) // 2
    heads, kv = q.shape[1], k.shape[1]
    scale = q.shape[2] ** -0.5 if scale is None else scale
    val = {n: torch.zeros_like(t) for n, t in
           (("out", q), ("q", q), ("k", k), ("v", v), ("table", table))}
    size = {n: torch.zeros_like(t) for n, t in val.items()}
    begin = 0
    for n in lengths:
        r = slice(begin, begin + n)
        begin += n
        if n == 0:
            continue
        pos = torch.arange(n) if positions is None else positions[r].detach().cpu().long()
        cell = bucket[(pos[None, :] - pos[:, None]).clamp(-reach, reach) + reach]
        ok = torch.ones(n, dtype=torch.bool) if keep is None else keep[r].detach().cpu()
        for h in range(heads):
            s = h * kv // heads
            # an absent bead is no key, whatever its rows hold
            kk = torch.where(ok[:, None], k[r, s], 0.0)
            vv = torch.where(ok[:, None], v[r, s], 0.0)
            logit = (q[r, h] @ kk.T) * scale + table[cell, h]
            logit = logit.masked_fill(~ok[None, :], -math.inf)
            # a row that nothing is left of (no key, or biases of -inf alone) is 0
            empty = (logit == -math.inf).all(1, keepdim=True)
            p = torch.softmax(logit.masked_fill(empty, 0.0), 1).masked_fill(empty, 0.0)
            o = p @ vv
            val["out"][r, h] = o
            size["out"][r, h] = o.abs() + p @ vv.abs()
            if grad is None:
                continue
            g = grad[r, h]
            dp = g @ vv.T
            ds = p * (dp - (p * dp).sum(1, keepdim=True))
            # delta is formed from the rounded output
            e = p * (g.abs() * o.abs()).sum(1, keepdim=True)
            val["q"][r, h] = ds @ kk * scale
            size["q"][r, h] = (ds.abs() + e) @ kk.abs() * abs(scale)
            val["k"][r, s] += ds.T @ q[r, h] * scale
            size["k"][r, s] += (ds.abs() + e).T @ q[r, h].abs() * abs(scale)
            val["v"][r, s] += p.T @ g
            size["v"][r, s] += p.T @ g.abs()
            flat = cell.reshape(-1).numpy()
            val["table"][:, h] += torch.from_numpy(
                np.bincount(flat, ds.reshape(-1).numpy(), table.shape[0]))
            size["table"][:, h] += torch.from_numpy(
                np.bincount(flat, e.reshape(-1).numpy(), table.shape[0]))
    if grad is None:
        return {"out": val["out"]}, {"out": size["out"]}
    for n in ("q", "k", "v", "table"):
        size[n] += val[n].abs()
    return val, size


ACTS = {
    "none": (lambda z: z, torch.ones_like),
    "tanh": (torch.tanh, lambda z: 1.0 - torch.tanh(z) ** 2),
    "ssp": (lambda z: torch.logaddexp(z, torch.zeros_like(z)) - math.log(2.0), torch.sigmoid),
    "silu": (lambda z: z * torch.sigmoid(z),
             lambda z: torch.sigmoid(z) * (1.0 + z * (1.0 - torch.sigmoid(z)))),
}


def group_norm(x, weight, bias, groups, lengths, eps=1e-5, act="none", grad=None):
    """{"out", and with grad "x", "weight", "bias"}."""
    x, weight, bias = (t.detach().cpu().double() for t in (x, weight, bias))
    grad = None if grad is None else grad.detach().cpu().double()
    value, slope = ACTS[act]
    width = x.shape[1]
    out = {"out": torch.zeros_like(x), "x": torch.zeros_like(x),
           "weight": torch.zeros_like(weight), "bias": torch.zeros_like(bias)}
    begin = 0
    for n in lengths:
        r = slice(begin, begin + n)
        begin += n
        if n == 0:
            continue
        split = (n, groups, width // groups)
        t = x[r].reshape(split)
        mean = t.mean((0, 2), keepdim=True)
        inv = ((t - mean).square().mean((0, 2), keepdim=True) + eps).rsqrt()
        hat = ((t - mean) * inv).reshape(n, width)
        z = hat * weight + bias
        out["out"][r] = value(z)
        if grad is None:
            continue
        dz = grad[r] * slope(z)
        out["weight"] += (dz * hat).sum(0)
        out["bias"] += dz.sum(0)
        d, hg = (dz * weight).reshape(split), hat.reshape(split)
        d = d - d.mean((0, 2), keepdim=True) - hg * (d * hg).mean((0, 2), keepdim=True)
        out["x"][r] = (d * inv).reshape(n, width)
    return out if grad is not None else {"out": out["out"]}


def philox4x32(counter, key, rounds=10):
    """The four words of Philox4x32 for a 128-bit counter and a 64-bit key
    (four and two 32-bit words; Salmon, Moraes, Dror, Shaw, SC 2011)."""
    x, (k0, k1) = list(counter), key
    for _ in range(rounds):
        a, b = 0xD2511F53 * x[0], 0xCD9E8D57 * x[2]
        x = [(b >> 32) ^ x[1] ^ k0, b & 0xFFFFFFFF, (a >> 32) ^ x[3] ^ k1, a & 0xFFFFFFFF]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return x


def dropout_kept(n, p, seed, step, first=0):
    """[n] bool: which of the elements from `first` (a multiple of 8) on
    dropout_add keeps, in Python integers."""
    t = min(65535, int(round(65536 * p)))
    kept = []
    for c in range(first // 8, first // 8 + (n + 7) // 8):
        words = philox4x32([c & 0xFFFFFFFF, c >> 32, step & 0xFFFFFFFF, step >> 32],
                           [seed & 0xFFFFFFFF, seed >> 32])
        for w in words:
            kept += [(w & 0xFFFF) >= t, (w >> 16) >= t]
    return torch.tensor(kept[:n], dtype=torch.bool), 65536.0 / (65536 - t)
