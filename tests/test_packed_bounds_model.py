"""CPU model of how the packed attention passes find their tiles, lists of tiles and parts from the bounds on the
device (pk_find_tile, pk_order and pk_token of csrc/gw_packed.h; dq_work, dkv_work and the joins of
csrc/packed_attn_bwd.hip), step by step as the kernels do: whatever the bounds hold, every row, key, list entry and part
lies within its tensor, list or workspace; where they are in order, every row of every sequence is computed once. No GPU
work."""
import random

import pytest

TILE, STAT, CLASSES = 128, 16, 128


def bound(cu, n, t, i):
    if i <= 0:
        return 0
    if i > n + 1:
        return t
    return min(max(cu[i - 1], 0), t)


def span(cu, n, t, i):
    a = bound(cu, n, t, i)
    return a, max(0, bound(cu, n, t, i + 1) - a)


def find_tile(cu, n, t, g, bm, slot):
    """The search with 64 probes at a time: (sequence, start, length, tile)."""
    first = lambda i: bound(cu, n, t, i) * g // bm + i  # noqa: E731
    lo, cnt = 0, n + 2
    while cnt > 1:
        step = (cnt + 63) >> 6
        below = [lane for lane in range(64) if lane * step < cnt and first(lo + lane * step) <= slot]
        top = below[-1] if below else 0
        lo, cnt = lo + top * step, min(step, cnt - top * step)
    start, length = span(cu, n, t, lo)
    return lo, start, length, slot - first(lo)


def order(cu, t, other, t_other, n, g, bm, slots):
    """The list's (sequence, tile) entries, as many as it has room for."""
    tiles = [(i, x) for i in range(n + 2) for x in range((span(cu, n, t, i)[1] * g + bm - 1) // bm)]
    random.Random(1).shuffle(tiles)  # their order in the list is no part of this
    return [tiles[s] if s < len(tiles) else (0, -1) for s in range(slots)]


def token(cu, n, t, x):
    lo, hi = 0, n + 2
    while hi - lo > 1:
        mid = (lo + hi) >> 1
        lo, hi = (mid, hi) if bound(cu, n, t, mid) <= x else (lo, mid)
    return lo, *span(cu, n, t, lo)


def parts(work, split, per):
    return min(split, max(1, int((work + per - 1) / per))) if split > 1 else 1


def div(a, b):
    return int(a / b)  # towards zero, as on the device


def dq_work(causal, g, length, lk, x):
    last = div(min((x + 1) * TILE, length * g) - 1, g)
    keys = min(last + lk - length, lk - 1) + 1 if causal else lk
    return (keys + 63) >> 6 if keys > 0 else 0


def dkv_work(causal, g, length, lq, x):
    first = max(0, x * TILE - (length - lq)) >> 6 if causal else 0
    return max(0, ((lq + 63) >> 6) - first) * g


def check(cu_q, cu_k, tq, tk, g, causal, split, per, ordered):
    n = len(cu_q) - 1
    seen_rows, seen_keys = [0] * (tq * g), [0] * tk
    # dQ: rows (token, head of the group) in tiles of 128, found by search and by the list.
    for listed in (False, True):
        slots = tq * g // TILE + n + 2
        entries = order(cu_q, tq, cu_k, tk, n, g, TILE, slots)
        for slot in range(slots):
            if listed:
                seq, tile = entries[slot]
                start, length = span(cu_q, n, tq, seq)
            else:
                seq, start, length, tile = find_tile(cu_q, n, tq, g, TILE, slot)
                assert tile >= 0
            assert 0 <= seq <= n + 1
            rows = length * g
            if tile < 0 or tile >= (rows + TILE - 1) // TILE:
                continue
            k0, lk = span(cu_k, n, tk, seq) if 1 <= seq <= n else (0, 0)
            assert 0 <= start <= start + length <= tq and 0 <= k0 <= k0 + lk <= tk
            work = dq_work(causal, g, length, lk, tile)
            p = parts(work, split, per)
            assert 1 <= p <= split and 0 <= work <= (lk + 63) // 64
            if listed:
                for r in range(tile * TILE, min(tile * TILE + TILE, rows)):
                    seen_rows[start * g + r] += 1
    # dK/dV: keys in tiles of 128.
    for listed in (False, True):
        slots = tk // TILE + n + 2
        entries = order(cu_k, tk, cu_q, tq, n, 1, TILE, slots)
        for slot in range(slots):
            if listed:
                seq, tile = entries[slot]
                start, length = span(cu_k, n, tk, seq)
            else:
                seq, start, length, tile = find_tile(cu_k, n, tk, 1, TILE, slot)
            assert 0 <= seq <= n + 1
            if tile < 0 or tile * TILE >= length:
                continue
            q0, lq = span(cu_q, n, tq, seq) if 1 <= seq <= n else (0, 0)
            assert 0 <= start <= start + length <= tk and 0 <= q0 <= q0 + lq <= tq
            work = dkv_work(causal, g, length, lq, tile)
            p = parts(work, split, per)
            share = (work + p - 1) // p
            for part in range(p):
                t0 = min(part * share, work)
                total = min(share, work - t0)
                if total:  # tiles of 64 queries, head by head of the group
                    first = max(0, tile * TILE - (length - lq)) >> 6 if causal else 0
                    around = ((lq + 63) >> 6) - first
                    for x in range(t0, t0 + total):
                        assert 0 <= x // around < g and 64 * (first + x % around) < lq
            assert 1 <= p <= split
            if listed:
                for key in range(tile * TILE, min(tile * TILE + TILE, length)):
                    seen_keys[start + key] += 1
    # Statistics: tiles of 16 tokens.
    stats = [0] * tq
    for slot in range(tq // STAT + n + 2):
        seq, start, length, tile = find_tile(cu_q, n, tq, 1, STAT, slot)
        assert tile >= 0
        for x in range(tile * STAT, min(tile * STAT + STAT, length)):
            stats[start + x] += 1
    # The joins: each row's sequence, and its parts.
    for cu, other, t, t_other, keys in ((cu_q, cu_k, tq, tk, False), (cu_k, cu_q, tk, tq, True)):
        for x in range(t):
            seq, start, length = token(cu, n, t, x)
            assert 0 <= seq <= n + 1 and 0 <= start <= x
            lo = span(other, n, t_other, seq)[1] if 1 <= seq <= n else 0
            at = x - start
            for h in range(1 if keys else g):
                work = dkv_work(causal, g, length, lo, at // TILE) if keys else \
                    dq_work(causal, g, length, lo, (at * g + h) // TILE)
                assert 1 <= parts(work, split, per) <= split
    if ordered:
        assert set(seen_rows) <= {1} and set(seen_keys) <= {1} and set(stats) <= {1}


@pytest.mark.parametrize("seed", range(8))
def test_every_index_is_in_range(seed):
    rng = random.Random(seed)
    for _ in range(12):
        n, g = rng.choice([0, 1, 2, 5, 70, 200]), rng.choice([1, 2, 3, 8])
        tq, tk = rng.randint(0, 900), rng.randint(0, 900)
        ordered = rng.random() < 0.3
        if ordered:
            cu_q, cu_k = (sorted(rng.randint(0, t) for _ in range(n + 1)) for t in (tq, tk))
        else:
            wild = lambda t: rng.choice([rng.randint(0, t), rng.randint(-5, t + 5), -2 ** 31, 2 ** 31 - 1, t])  # noqa: E731
            cu_q, cu_k = ([wild(t) for _ in range(n + 1)] for t in (tq, tk))
        check(cu_q, cu_k, tq, tk, g, rng.random() < 0.5, rng.choice([1, 2, 16]), rng.choice([8, 20, 64]), ordered)
