"""A paged key-value cache in 64 bits on the CPU, from the definitions: what an append writes, in 16 or 4 bits, and what
a read returns. Slots are found one by one."""
from __future__ import annotations

import torch

FP4 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
NAN = 255  # a scale that is not a number


def fp4_scales(top):
    """Biased exponents for the largest magnitudes ``top`` (64 bits) of 32 values: the largest comes to (3.5, 7]."""
    mantissa, exponent = torch.frexp(top.double())  # mantissa in [1/2, 1): 7 / 8 is 7 units of 2^(exponent - 3)
    e = (exponent - 3 + (mantissa > 0.875) + 127).clamp_min(0)
    e = torch.where(top == 0, 0, e)
    return torch.where(top < float("inf"), e, NAN).to(torch.uint8)


def fp4_codes(y):
    """Codes (0 to 15) of values in units: the nearest, of two as near the one with an even code."""
    d = (y.abs()[..., None] - FP4).abs()
    best = d.amin(-1, keepdim=True)
    near = d == best
    even = near & (torch.arange(8) % 2 == 0)
    code = torch.where(even.any(-1), even.to(torch.uint8).argmax(-1), near.to(torch.uint8).argmax(-1))
    return (code + 8 * torch.signbit(y)).to(torch.uint8)


def fp4_encode(x):
    """x [..., D] -> (codes [..., D / 2], scales [..., D / 32]) as they lie in memory."""
    x = x.double().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    top = torch.where(x.isnan().any(-1), float("nan"), top)
    scales = fp4_scales(top)
    y = torch.where((scales == NAN)[..., None], 0.0, x * torch.pow(2.0, 127.0 - scales.double())[..., None])
    c = fp4_codes(y).flatten(-2)
    return c[..., 0::2] + 16 * c[..., 1::2], scales


def fp4_decode(codes, scales):
    """64-bit values."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    v = torch.where(c >= 8, -FP4[c & 7], FP4[c & 7])
    unit = torch.where(scales == NAN, float("nan"), torch.pow(2.0, scales.double() - 127.0))
    return v * unit.repeat_interleave(32, -1)


def token_slots(lens, table, page, pages, count=None, cu=None, tokens=None):
    """[(page, slot) or None] of each new token: ``count`` of each sequence, or packed by ``cu``."""
    out = []
    if cu is None:
        of = [(b, i, count) for b in range(len(lens)) for i in range(count)]
    else:
        of = [None] * tokens
        for b in range(len(cu) - 1):
            for t in range(max(int(cu[b]), 0), min(int(cu[b + 1]), tokens)):
                of[t] = (b, t - int(cu[b]), int(cu[b + 1]) - int(cu[b]))
    for item in of:
        at = None
        if item is not None:
            b, i, n = item
            key = int(lens[b]) - n + i
            if 0 <= key < table.shape[1] * page and 0 <= int(table[b, key // page]) < pages:
                at = (int(table[b, key // page]), key % page)
        out.append(at)
    return out


def read_slots(cu, table, page, pages, tokens):
    """[(page, slot) or None] of each packed row."""
    out = [None] * tokens
    for b in range(len(cu) - 1):
        for t in range(max(int(cu[b]), 0), min(int(cu[b + 1]), tokens)):
            key = t - int(cu[b])
            if key < table.shape[1] * page and 0 <= int(table[b, key // page]) < pages:
                out[t] = (int(table[b, key // page]), key % page)
    return out
