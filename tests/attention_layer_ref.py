"""The attention half of a layer in 64 bits, from checkpoint tensors one by one, with a bound on what roundings may change."""
from __future__ import annotations

import math

import torch

U = 2.0 ** -8  # half a step of bf16, relative to the value
PREFIX = "model.layers.3.self_attn"


def checkpoint(heads, kv, d, hidden, *, bias, sinks, seed=0):
    """Tensors under checkpoint names, bf16.  Each row of the q, k and v weights adds three columns of x up (signs, no factors), each
    row of the output's takes one column, biases are eighths: with x in eighths up to 3/4, q, k and v are exact in bf16, and what a
    mistake changes is not lost in a worst-case bound over long sums."""
    g = torch.Generator().manual_seed(seed)
    t = {}
    for n, rows, cols, terms in (("q", heads * d, hidden, 3), ("k", kv * d, hidden, 3), ("v", kv * d, hidden, 3), ("o", hidden, heads * d, 1)):
        at = torch.rand(rows, cols, generator=g).argsort(1)[:, :terms]
        sign = torch.randint(0, 2, (rows, terms), generator=g) * 2.0 - 1
        t[f"{PREFIX}.{n}_proj.weight"] = torch.zeros(rows, cols).scatter_(1, at, sign).bfloat16()
        if bias:
            t[f"{PREFIX}.{n}_proj.bias"] = (torch.randint(-4, 5, (rows,), generator=g) / 8).bfloat16()
    if sinks:
        t[f"{PREFIX}.sinks"] = torch.randn(heads, generator=g).bfloat16()
    return t


def tokens(n, hidden, seed):
    return (torch.randint(-6, 7, (n, hidden), generator=torch.Generator().manual_seed(seed)) / 8).bfloat16()


def linear(x, dx, t, name):
    """x W^T + b of x known to dx, and how far a bf16 product of it may be off: one or two roundings, none where the sum is exact."""
    w = t[f"{PREFIX}.{name}_proj.weight"].double()
    b = t.get(f"{PREFIX}.{name}_proj.bias")
    p = x @ w.T
    y = p if b is None else p + b.double()
    off = dx @ w.abs().T
    if not dx.any() and torch.equal(y.bfloat16().double(), y) and torch.equal(p.bfloat16().double(), p):
        return y, off
    off = off + (w.shape[1] + 4) * 2.0 ** -23 * ((x.abs() + dx) @ w.abs().T)
    return y, (off + U * p.abs()) * (1 + U) + U * y.abs()


def rotated(x, dx, cos, sin):
    """The halves of a head's row turned against each other; one rounding."""
    a, b = x.chunk(2, -1)
    da, db = dx.chunk(2, -1)
    c, s = cos.double()[:, None], sin.double()[:, None]
    y = torch.cat([a * c - b * s, b * c + a * s], -1)
    dy = torch.cat([da * c.abs() + db * s.abs(), db * c.abs() + da * s.abs()], -1)
    return y, (dy + 2.0 ** -22 * (y.abs() + dy)) * (1 + U) + U * y.abs()


def layer(x, t, cos, sin, heads, kv, d, window=0, scale=None):
    """One sequence x [T, hidden] (bf16) from position 0: (y [T, hidden], bound).

    Scores off by e_ij = scale (|dq| |k| + |q| |dk| + |dq| |dk|) and an fp32 sum change each weight by a factor of at most
    exp(2 max_j e_ij); beside it the numerators' rounding (u) and exponentials (7.5e-5 + 2^-20, in numerator and denominator); then
    the values' own error, and the output's rounding."""
    T, scale = x.shape[0], d ** -0.5 if scale is None else scale
    x = x.double()
    q, k, v = ((a.view(T, -1, d), b.view(T, -1, d)) for a, b in (linear(x, torch.zeros_like(x), t, n) for n in "qkv"))
    q, k = rotated(*q, cos[:T], sin[:T]), rotated(*k, cos[:T], sin[:T])
    g = heads // kv
    (q, dq), (k, dk), (v, dv) = q, *((a.repeat_interleave(g, 1), b.repeat_interleave(g, 1)) for a, b in (k, v))
    s = torch.einsum("ihd,jhd->hij", q, k) * scale
    e = (torch.einsum("ihd,jhd->hij", dq, k.abs() + dk) + torch.einsum("ihd,jhd->hij", q.abs(), dk)
         + (d + 4) * 2.0 ** -23 * torch.einsum("ihd,jhd->hij", q.abs() + dq, k.abs() + dk)) * scale
    pos = torch.arange(T)
    see = pos[None, :] <= pos[:, None]
    if window > 0:
        see &= pos[None, :] > pos[:, None] - window
    s = s.masked_fill(~see, -math.inf)
    sinks = t.get(f"{PREFIX}.sinks")
    full = s if sinks is None else torch.cat([s, sinks.double().view(heads, 1, 1).expand(heads, T, 1)], 2)
    p = torch.exp(s - torch.logsumexp(full, 2, keepdim=True))
    o = torch.einsum("hij,jhd->ihd", p, v)
    grow = torch.exp(2 * e.masked_fill(~see, 0).amax(2)).T[..., None]  # [T, heads, 1]
    rel = grow * (1 + U + 2 * (7.5e-5 + 2.0 ** -20) + 4 * T * 2.0 ** -24) - 1
    do = rel * torch.einsum("hij,jhd->ihd", p, v.abs() + dv) + torch.einsum("hij,jhd->ihd", p, dv)
    do = do * (1 + U) + U * o.abs()
    return linear(o.reshape(T, -1), do.reshape(T, -1), t, "o")


def tables(n, d):
    ang = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    return ang.cos().float(), ang.sin().float()
