"""64-bit references of the grouped and paged attention, with elementwise error
bounds of the kernels' roundings.

u is half a step of the 16-bit type. Rounding the softmax weights to it moves
o = sum w v / sum w by at most u (sum p |v| + |o|), rounding the result by u |o|;
rounding ds and p moves dq, dk by u sum |ds| |k|, u sum |ds| |q|, and dv by
u sum p |dO|, their own rounding adds u of the result, and delta = dO . o carries
o's error before its rounding (and u^2 of what is left of it). SLACK covers fp32
sums, scores and exponentials, relative to the sums of magnitudes. floor() is what
a weight or a result loses where it falls below the normal numbers: weights below
2^-126 leave the exponential as 0 and bf16 has no smaller normal number, so each
of them, and of the products and results made of them, is off by at most 2^-126 of
what it weighs (a ds of 1e-55 is 0); an fp16 weight, relative to a maximum that is
at most its row's, is rounded to a multiple of 2^-24, so by at most 2^-25.
"""
import math

import torch

SLACK = 2.0 ** -13


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def floor(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126


def attend(q, k, v, seen, scale):
    """o and its error bound (without u) for q (R, N), k and v (L, N), seen (R, L), all 64-bit."""
    s = torch.where(seen, (q @ k.T) * scale, -math.inf)
    top = s.amax(1, keepdim=True) if s.shape[1] else s.new_full((s.shape[0], 1), -math.inf)
    p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    den = p.sum(1, keepdim=True)
    p = p / torch.where(den == 0, 1.0, den)
    o = p @ v
    return o, p, p @ v.abs()


def packed(q, k, v, lens, scale, dout=None):
    """Reference of grouped_attn_varlen: {name: (value, tolerance)} of o and, with
    dout, of dq, dk, dv. Inputs on any device; computed in 64 bits there."""
    u, f = half_step(q.dtype), floor(q.dtype)
    q, k, v = (t.detach().double() for t in (q, k, v))
    G = q.shape[1] // k.shape[1]
    out = {n: [torch.zeros_like(t), torch.zeros_like(t)] for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    t0 = 0
    for L in lens:
        r = slice(t0, t0 + L)
        t0 += L
        if L == 0:
            continue
        seen = torch.tril(torch.ones(L, L, dtype=torch.bool, device=q.device))
        for h in range(q.shape[1]):
            g = h // G
            qh, kh, vh = q[r, h], k[r, g], v[r, g]
            o, p, mag = attend(qh, kh, vh, seen, scale)
            out["o"][0][r, h] = o
            out["o"][1][r, h] = u * (2 * o.abs() + mag) + SLACK * mag + f * (1 + vh.abs().sum(0))
            if dout is None:
                continue
            d = dout[r, h].double()
            dp = d @ vh.T
            ds = p * (dp - (d * o).sum(1, keepdim=True))
            # delta's error: o's before its rounding, and what is left of o in u bits.
            e = (d.abs() * ((u + SLACK) * (mag + o.abs()) + u * u * o.abs())).sum(1, keepdim=True)
            size = p * ((d.abs() @ vh.abs().T) + (d.abs() * mag).sum(1, keepdim=True))  # of the terms of ds
            eds = u * ds.abs() + p * e + SLACK * size
            eds += torch.where(seen, f * (1 + d.abs() @ vh.abs().T + (d.abs() * mag).sum(1, keepdim=True)), 0.0)
            dq, dk = scale * (ds @ kh), scale * (ds.T @ qh)
            out["dq"][0][r, h] = dq
            out["dq"][1][r, h] = u * dq.abs() + scale * (eds @ kh.abs()) + f
            out["dk"][0][r, g] += dk
            out["dk"][1][r, g] += scale * (eds.T @ qh.abs())
            out["dv"][0][r, g] += p.T @ d
            out["dv"][1][r, g] += (u + SLACK) * (p.T @ d.abs()) + f * d.abs().sum(0)
    for n in ("dk", "dv"):
        out[n][1] += u * out[n][0].abs() + f
    return {n: tuple(x) for n, x in out.items()}


def assert_within(name, got, ref):
    want, tol = (t.to(got.device) for t in ref)
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{name}: NaN in other places"
    bad = ~((got - want).abs() <= tol) & (got != want) & ~torch.isnan(want)
    if bool(bad.any()):
        worst = torch.where(bad, (got - want).abs() / tol, 0.0)
        at = tuple(int(x) for x in torch.unravel_index(worst.argmax(), worst.shape))
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} outside, worst at {at}: "
                             f"{float(got[at])} for {float(want[at])} +- {float(tol[at])}")


def cache_rows(cache, s, pool):
    """The rows (length, Hkv, N) of sequence s."""
    L = int(cache.lengths[s])
    ids = cache.table[s, : -(-L // cache.page)].long()
    return pool[ids].transpose(1, 2).reshape(-1, pool.shape[1], pool.shape[3])[:L]


def step(q, cache, mask, scale):
    """Reference of tree_attn: (value, tolerance) for q (S, n, Hq, N)."""
    S, n, Hq, N = q.shape
    u, f, H = half_step(q.dtype), floor(q.dtype), cache.k.shape[1]
    G = Hq // H
    o, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for s in range(S):
        k, v = (cache_rows(cache, s, pool).double().cpu() for pool in (cache.k, cache.v))
        L = k.shape[0]
        m = torch.tril(torch.ones(n, n, dtype=torch.bool)) if mask is None else (mask[s] if mask.dim() == 3 else mask).cpu()
        rel = torch.arange(L) - (L - n)
        seen = torch.where(rel < 0, torch.tensor(True), m[:, rel.clamp(min=0)]) if L else torch.zeros(n, 0, dtype=torch.bool)
        for h in range(Hq):
            value, _, mag = attend(q[s, :, h].double().cpu(), k[:, h // G], v[:, h // G], seen, scale)
            o[s, :, h] = value
            tol[s, :, h] = u * (2 * value.abs() + mag) + SLACK * mag + f * (1 + v[:, h // G].abs().sum(0))
    return o, tol
