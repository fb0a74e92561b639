"""Plain 64-bit attention, rotary embedding and error bounds for the attention tests."""
from __future__ import annotations

import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative to the value


def attention(q, k, v, pos, scale, window=0, sinks=None):
    """q [n, H, D] at positions pos [n], over k, v [m, Hkv, D], float64.

    Returns (out [n, H, D], lse [n, H], bound [n, H, D]): how far a correct kernel may be off.  With u half a
    step of the element type, a numerator p_ij is rounded once (u), the exponential is good to 7.5e-5 (bf16) or
    2.6e-6 (f16) plus 2^-20, and an error d of the score changes it by d: d <= (D + 4) 2^-23 sum_e |q_e k_e| scale for an
    fp32 sum of D products.  All of it is relative to sum_j p_ij |v_j| / l, and the denominator has the last two again; the
    output is rounded once more (u |o|).  f16 numerators below 2^-14 are rounded to 2^-25 at worst.
    """
    dt = q.dtype
    u = U[dt]
    q, k, v = q.double(), k.double(), v.double()
    n, H, D = q.shape
    m, g = k.shape[0], H // k.shape[1]
    kk, vv = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    s = torch.einsum("nhd,mhd->nhm", q, kk) * scale
    mag = torch.einsum("nhd,mhd->nhm", q.abs(), kk.abs()) * scale
    key = torch.arange(m, device=q.device)
    see = key[None] <= pos[:, None]
    if window > 0:
        see = see & (key[None] > pos[:, None] - window)
    see = see[:, None].expand(n, H, m)
    s = s.masked_fill(~see, -math.inf)
    full = s if sinks is None else torch.cat([s, sinks.double().view(1, H, 1).expand(n, H, 1)], 2)
    lse = torch.logsumexp(full, 2) if full.shape[2] else torch.full((n, H), -math.inf, dtype=torch.float64, device=q.device)
    p = torch.exp(s - lse[..., None].nan_to_num(neginf=0.0)) if m else s
    p = torch.where(see, p, torch.zeros_like(p))
    out = torch.einsum("nhm,mhd->nhd", p, vv)
    weight = torch.einsum("nhm,mhd->nhd", p, vv.abs())
    d = (D + 4) * 2.0 ** -23 * (mag.masked_fill(~see, 0).amax(2) if m else torch.zeros(n, H, device=q.device))
    e = (7.5e-5 if dt == torch.bfloat16 else 2.6e-6) + 2.0 ** -20
    rel = u + 2 * (e + d) + 4 * m * 2.0 ** -24
    bound = u * out.abs() + rel[..., None] * weight + 1e-9
    if dt == torch.float16:
        bound = bound + 2.0 ** -24 + (2.0 ** -25 * m * vv.abs().amax() if m else 0)
    return out, lse, bound


def assert_close(got, want, bound, what=""):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / bound).nan_to_num(nan=1e30).max()):.3g} x the bound"


def assert_lse(got, want, what=""):
    """fp32 log-sum-exp: the error of a sum of exponentials good to 1e-4 each, and of fp32 at the value."""
    empty = want == -math.inf
    assert torch.equal(got == -math.inf, empty), f"{what}: lse of empty rows"
    err = (got.double() - want).abs()[~empty]
    assert (err <= 3e-4 + 2.0 ** -21 * want[~empty].abs()).all(), f"{what}: lse off by {float(err.max()):.3g}"


def rotate(x, cos, sin):
    a, b = x.double().chunk(2, -1)
    c, s = cos.double()[:, None], sin.double()[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def paged(seq_k, seq_v, page_size, extra=2, seed=0, fill=float("nan")):
    """Pools and a table for sequences' keys and values ([n_i, Hkv, D] each); everything unused holds `fill`."""
    dev, (hkv, d), dt = seq_k[0].device, seq_k[0].shape[1:], seq_k[0].dtype
    need = [-(-t.shape[0] // page_size) for t in seq_k]
    total = sum(need) + extra
    ids = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    kp = torch.full((total, hkv, page_size, d), fill, dtype=dt, device=dev)
    vp = kp.clone()
    table = torch.full((len(seq_k), max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for i, (k, v) in enumerate(zip(seq_k, seq_v)):
        for j in range(need[i]):
            page = ids[at]
            at += 1
            table[i, j] = page
            part_k, part_v = k[j * page_size:(j + 1) * page_size], v[j * page_size:(j + 1) * page_size]
            kp[page, :, :part_k.shape[0]] = part_k.transpose(0, 1)
            vp[page, :, :part_v.shape[0]] = part_v.transpose(0, 1)
    return kp, vp, table.to(dev)
