"""Attention over packed sequences and over a paged cache, and rotary positions with several axes, in
64 bits on the CPU from their definitions (the forms that the GPU operators are tested against)."""
from __future__ import annotations

import math

import torch


def _bounds(cu, total):
    b = [0] + [min(max(int(c), 0), total) for c in cu] + [total]
    return list(zip(b[:-1], b[1:]))  # tokens of no sequence first and last


def _visible(lq, lk, causal):
    see = torch.ones(lq, lk, dtype=torch.bool)
    return see.tril(lk - lq) if causal else see


def _weights(q, k, scale, see):
    """softmax(scale q k^T) over the visible keys (zeros for a row that sees none) and its lse."""
    s = (q @ k.t() * scale).masked_fill(~see, -math.inf)
    lse = torch.logsumexp(s, 1) if s.shape[1] else torch.full((s.shape[0],), -math.inf, dtype=s.dtype)
    p = torch.where(see, torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[:, None]), 0.0)
    return p, lse


def packed_attention(q, k, v, cu_q, cu_k, causal=False, scale=None, do=None):
    """q [Tq, Hq, D], k, v [Tk, Hk, D] of any float type. Returns a dict of 64-bit tensors: o, lse, and
    with ``do`` also dq, dk, dv; besides, for error bounds, the sums of magnitudes that the roundings of
    16-bit weights act on: ``o_mag`` = P|V|, ``dv_mag`` = P^T|dO|, ``dq_mag``/``dk_mag`` (|dS| and P |o||dO|
    weighted by |K|/|Q|), and ``s_mag`` = the largest scale |q||k| of a row."""
    q, k, v = q.double(), k.double(), v.double()
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    tq, hq, d = q.shape
    tk, hk, _ = k.shape
    out = {"o": torch.zeros_like(q), "o_mag": torch.zeros_like(q), "lse": torch.full((tq, hq), -math.inf, dtype=torch.float64),
           "s_mag": torch.zeros(tq, hq, dtype=torch.float64)}
    if do is not None:
        do = do.double()
        for n, t in (("dq", q), ("dk", k), ("dv", v)):
            out[n], out[n + "_mag"] = torch.zeros_like(t), torch.zeros_like(t)
    for i, ((a, b), (c, e)) in enumerate(zip(_bounds(cu_q, tq), _bounds(cu_k, tk))):
        if i == 0 or i == len(cu_q) or b <= a or e <= c:
            continue
        see = _visible(b - a, e - c, causal)
        for h in range(hq):
            j = h // (hq // hk)
            qi, ki, vi = q[a:b, h], k[c:e, j], v[c:e, j]
            # what a masked place holds has no part in the result
            p, lse = _weights(qi, ki, scale, see)
            o = p @ vi
            out["o"][a:b, h], out["lse"][a:b, h] = o, lse
            out["o_mag"][a:b, h] = p @ vi.abs()
            out["s_mag"][a:b, h] = (qi.abs() @ ki.abs().t() * scale).amax(1)
            if do is None:
                continue
            g = do[a:b, h]
            dp = g @ vi.t()
            delta = (o * g).sum(1, keepdim=True)
            ds = p * (dp - delta)
            dmag = p * (dp.abs() + (o.abs() * g.abs()).sum(1, keepdim=True))
            out["dq"][a:b, h] = scale * ds @ ki
            out["dq_mag"][a:b, h] = scale * dmag @ ki.abs()
            out["dk"][c:e, j] += scale * ds.t() @ qi
            out["dk_mag"][c:e, j] += scale * dmag.t() @ qi.abs()
            out["dv"][c:e, j] += p.t() @ g
            out["dv_mag"][c:e, j] += p.t() @ g.abs()
    return out


def paged_attention(q, k_cache, v_cache, table, lens, scale=None, causal=True):
    """q [B, N, Hq, D], caches [pages, page, Hk, D], table [B, W], lens [B] -> (o, lse, o_mag, s_mag) in 64 bits.
    Table entries outside the pool hold keys that nobody sees; query i sees keys below lens - N + 1 + i."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    bsz, new, hq, d = q.shape
    pool, page, hk, _ = k_cache.shape
    o = torch.zeros(q.shape, dtype=torch.float64)
    mag, s_mag = torch.zeros_like(o), torch.zeros(bsz, new, hq, dtype=torch.float64)
    lse = torch.full((bsz, new, hq), -math.inf, dtype=torch.float64)
    for b in range(bsz):
        n = min(max(int(lens[b]), 0), table.shape[1] * page)
        at = torch.arange(n)
        pg = table[b].long()[at // page] if n else at
        ok = (pg >= 0) & (pg < pool)
        pg = pg.clamp(0, max(pool - 1, 0))
        see = _visible(new, n, causal) & ok[None]
        for h in range(hq):
            j = h // (hq // hk)
            k, v = k_cache[pg, at % page, j].double(), v_cache[pg, at % page, j].double()
            k, v = torch.where(ok[:, None], k, 0.0), torch.where(ok[:, None], v, 0.0)
            p, lse[b, :, h] = _weights(q[b, :, h].double(), k, scale, see)
            o[b, :, h], mag[b, :, h] = p @ v, p @ v.abs()
            if n:
                s_mag[b, :, h] = (q[b, :, h].double().abs() @ k.abs().t() * scale).amax(1)
    return o, lse, mag, s_mag


def rotary_axes(x, positions, axis_dims, bases, sign=1.0):
    """x [..., H, D], positions [..., A] -> 64-bit turned x."""
    x, pos = x.double(), positions.double()
    y, at = x.clone(), 0
    for a, n in enumerate(axis_dims):
        for i in range(n // 2):
            t = sign * pos[..., a] * bases[a] ** (-2.0 * i / n)
            c, s = t.cos()[..., None], t.sin()[..., None]
            u, w = x[..., at + i], x[..., at + n // 2 + i]
            y[..., at + i], y[..., at + n // 2 + i] = u * c - w * s, w * c + u * s
        at += n
    return y
