"""Paged attention over a cache in 4 bits (gw_paged_attn_fp4_fwd) against the 64-bit oracle on the values that the codes
stand for.

Tolerance: a weight enters its product as two bf16 terms, off by at most 2^-8 of 2^-8 / 2, so below 2^-17 of itself; the
output is rounded once, u = eps / 2. Values and q enter exactly: a score is off by the fp32 sums of its products, 2 D 2^-24
of its magnitudes (twice that for q in two terms); the other fp32 sums add less than 2^-18."""
import math

import pytest
import torch

from geoweave_amd.custom_flash_attn.packed_flash_attn import packed_flash_attn_inference_func
from geoweave_amd.custom_flash_attn.paged_flash_attn import paged_flash_attn_inference_func
from geoweave_amd.custom_flash_attn.paged_kv_cache import (FP4Cache, fp4_paged_cache, paged_kv_append_func,
                                                           paged_kv_read_func)
from oracle.packed_attention import paged_attention
from oracle.paged_kv import fp4_decode, fp4_encode

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def make(lens, new, hq, hk, d, page, dtype, seed=0, spare=3, width=2, gain=1.5, unit=126, spread=2):
    """(q, (codes, scales) of k and of v, table, lens) on the CPU."""
    g = torch.Generator().manual_seed(seed)
    pages = [-(-n // page) for n in lens]
    pool = sum(pages) + spare
    order = torch.randperm(pool, generator=g)
    table = torch.full((len(lens), max(pages + [0]) + width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n].to(torch.int32)
        at += n
    q = (torch.randn(len(lens), new, hq, d, generator=g) * gain).to(dtype)
    kv = []
    for _ in range(2):
        codes, _ = fp4_encode(torch.randn(64, 32, generator=g))
        codes = codes.flatten()[torch.randint(0, codes.numel(), (pool, page, hk, d // 2), generator=g)]
        kv.append((codes, (unit + torch.randint(-spread, spread + 1, (pool, page, hk, d // 32), generator=g)).to(torch.uint8)))
    return q, *kv, table, torch.tensor(lens, dtype=torch.int32)


def on_gpu(kept, dev):
    """An FP4Cache with the layout of fp4_paged_cache."""
    c = fp4_paged_cache(*kept[0].shape[:3], kept[0].shape[3] * 2, device=dev)
    for x, y in zip(c, kept):
        x.copy_(y)
    return c


def run(args, dev, **kw):
    q, k, v, table, lens = args
    return paged_flash_attn_inference_func(q.to(dev), on_gpu(k, dev), on_gpu(v, dev), table.to(dev), lens.to(dev),
                                           return_lse=True, **kw)


def reference(args, **kw):
    q, k, v, table, lens = args
    return paged_attention(q, fp4_decode(*k), fp4_decode(*v), table, lens, **kw)


def check(got, lse, ref, args):
    o, want_lse, mag, s_mag = ref
    dtype, d = args[0].dtype, args[0].shape[-1]
    u = torch.finfo(dtype).eps / 2
    s = (2 if dtype == HF else 1) * 2 * d * 2.0 ** -24 * s_mag
    lim = 1.01 * u * o.abs() + (2.0 ** -17 + 4 * s[..., None] + 2.0 ** -18) * mag + (2.0 ** -24 if dtype == HF else 2.0 ** -60)
    err = (got.double().cpu() - o).abs()
    assert torch.isfinite(got).all()
    assert (err <= lim).all(), float((err / lim).max())
    a = lse.double().cpu()
    assert torch.equal(a == -math.inf, want_lse == -math.inf)
    on = want_lse != -math.inf
    assert ((a - want_lse)[on].abs() <= (s + 2.0 ** -18 * (1 + s_mag))[on]).all()


LENS = {
    "one key": [1],
    "edges": [1, 0, 15, 16, 17, 31, 32, 33, 63, 64, 65, 255, 256, 257, 600],
    "ragged": [4000, 3, 700, 1, 129],
    "long": [20011],
}


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,hq,hk", [(64, 2, 2), (128, 8, 1), (64, 6, 2), (128, 3, 3), (64, 16, 1)])
@pytest.mark.parametrize("new,page,causal", [(1, 16, True), (1, 100, True), (5, 64, True), (7, 1, False), (9, 7, True)])
@pytest.mark.parametrize("lens", list(LENS))
def test_values(gpu_device, dtype, d, hq, hk, new, page, causal, lens):
    args = make(LENS[lens], new, hq, hk, d, page, dtype)
    o, lse = run(args, gpu_device, causal=causal)
    check(o, lse, reference(args, causal=causal), args)
    again, lse2 = run(args, gpu_device, causal=causal)
    assert torch.equal(o, again) and torch.equal(lse, lse2), "the same inputs give the same bits"


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,hq,hk", [(64, 2, 2), (128, 4, 1)])
@pytest.mark.parametrize("new,lens", [(200, [200, 900]), (700, [1100, 650])])
def test_many_new_tokens(gpu_device, dtype, d, hq, hk, new, lens):
    args = make(lens, new, hq, hk, d, 32, dtype, 40)
    o, lse = run(args, gpu_device)
    check(o, lse, reference(args), args)


@pytest.mark.parametrize("d,hq,hk,new", [(64, 16, 16, 1), (128, 24, 12, 2), (64, 32, 16, 40), (128, 16, 8, 17)])
def test_units_of_many_blocks(gpu_device, d, hq, hk, new):
    """Units of more than four blocks that end one row tile, take others whole and begin another."""
    lens = [3000, 65, 64, 1, 0, 2500, 700, 128, 4100, 17, 17, 333]
    args = make(lens, new, hq, hk, d, 16, BF, 50)
    o, lse = run(args, gpu_device)
    check(o, lse, reference(args), args)


def test_more_key_heads_than_units(gpu_device):
    """1,100 key heads: one unit takes all row tiles of a head."""
    args = make([70, 0, 300, 64, 5], 3, 1100, 1100, 64, 16, HF, 51)
    o, lse = run(args, gpu_device)
    pick = [0, 1, 550, 1099]
    some = (args[0][:, :, pick], *(tuple(t[:, :, pick] for t in c) for c in args[1:3]), *args[3:])
    check(o[:, :, pick], lse[:, :, pick], reference(some), some)


def test_many_sequences_without_a_split(gpu_device):
    lens = torch.randint(0, 90, (4200,), generator=torch.Generator().manual_seed(1)).tolist()
    args = make(lens, 1, 2, 1, 64, 32, BF)
    o, lse = run(args, gpu_device)
    check(o, lse, reference(args), args)


def test_more_sequences_than_one_scan_round(gpu_device):
    lens = torch.randint(0, 200, (150,), generator=torch.Generator().manual_seed(2)).tolist()
    lens[70] = 9000
    args = make(lens, 3, 8, 1, 128, 48, HF)
    o, lse = run(args, gpu_device)
    check(o, lse, reference(args), args)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("gain,unit,spread", [(1e-3, 126, 2), (30.0, 122, 2), (1.5, 126, 12), (1e-30, 180, 3), (1e4, 113, 3),
                                              (2.0 ** -20, 137, 2)])
def test_ranges(gpu_device, dtype, d, gain, unit, spread):
    """Small and large queries, kept rows whose powers of two differ widely."""
    if dtype == HF and gain == 1e-30:
        gain, unit = 2.0 ** -24, 150  # subnormal
    args = make([300, 77], 2, 4, 2, d, 16, dtype, 21, gain=gain, unit=unit, spread=spread)
    args[2][1].fill_(126)
    ref = reference(args)
    o, lse = run(args, gpu_device)
    check(o, lse, ref, args)


def test_a_row_of_one_large_query_dim(gpu_device):
    """One dim of 32 a million times the others: these keep their part."""
    args = make([500], 1, 2, 1, 64, 16, BF, 22, gain=1.0)
    args[0][..., 5] = 2.0 ** 14
    args[1][0][..., 2] &= 0x0F  # dim 5 of the keys: 0
    ref = reference(args)
    o, lse = run(args, gpu_device)
    check(o, lse, ref, args)
    args[0][..., 5] = 0.0
    assert (ref[0] - reference(args)[0]).abs().max() == 0  # they are all that counts


@pytest.mark.parametrize("scale", [1e-30, 0.01, 3.0])
def test_scales(gpu_device, scale):
    args = make([700, 30], 3, 4, 2, 64, 16, HF, 23)
    o, lse = run(args, gpu_device, softmax_scale=scale)
    check(o, lse, reference(args, scale=scale), args)


@pytest.mark.parametrize("page,d", [(24, 64), (32, 64), (32, 128)])
def test_unused_slots_and_pages_outside_the_pool(gpu_device, page, d):
    """Scales that are not numbers wherever no key lies, page numbers outside the pool in the middle and at the end."""
    args = make([300, 77, 500, 40], 4, 4, 2, d, page, BF, 3)
    q, k, v, table, lens = args
    used = torch.zeros(k[0].shape[:2], dtype=torch.bool)
    gone = [(0, 2), (0, 299 // page), (2, 0), (2, 5), (3, 0), (3, 1)]
    for (b, p), bad in zip(gone, (-1, 10 ** 6, k[0].shape[0], -2 ** 31, -5, 2 ** 31 - 1)):
        table[b, p] = bad
    for b, n in enumerate(lens.tolist()):
        for j in range(n):
            if 0 <= table[b, j // page] < k[0].shape[0]:
                used[table[b, j // page], j % page] = True
    assert not used.all()
    k[1][~used], v[1][~used] = 255, 255
    o, lse = run(args, gpu_device)
    for kept in (k, v):  # the oracle's own 0 * NaN
        kept[1][~used] = 100
    check(o, lse, reference(args), args)
    assert (o[3] == 0).all() and (lse[3] == -math.inf).all()


@pytest.mark.parametrize("d,hk,new", [(64, 2, 6), (128, 1, 6), (64, 1, 9)])
@pytest.mark.parametrize("n", [40, 1003])
def test_what_a_new_token_does_not_see(gpu_device, d, hk, new, n):
    """32 values that are not numbers, of the newest tokens, reach the tokens that see them, in their dims, and no other."""
    args = make([n, 20], new, 4, hk, d, 16, HF, 8)
    q, k, v, table, lens = args
    clean, lse = run(args, gpu_device)
    j = n - 3  # seen by the last three new tokens
    page, slot, a = int(table[0, j // 16]), j % 16, new - 3
    v[1][page, slot, :, 1] = 255
    o, lse2 = run(args, gpu_device)
    assert torch.equal(clean[0, :a], o[0, :a]) and torch.equal(clean[1], o[1]) and torch.equal(lse, lse2)
    assert torch.equal(clean[0, :, :, :32], o[0, :, :, :32]) and torch.equal(clean[0, :, :, 64:], o[0, :, :, 64:])
    assert o[0, a:, :, 32:64].isnan().all()
    v[1][page, slot, :, 1] = 126
    k[1][page, slot, :, 1] = 255
    o, lse2 = run(args, gpu_device)
    assert torch.equal(clean[0, :a], o[0, :a]) and torch.equal(clean[1], o[1]) and torch.equal(lse[0, :a], lse2[0, :a])
    assert o[0, a:].isnan().all() and lse2[0, a:].isnan().all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_queries_that_are_not_finite(gpu_device, dtype, value):
    args = make([100, 60, 0], 3, 12, 2, 64, 16, dtype, 9)
    clean, lse = run(args, gpu_device)
    args[0][0, 1, 4, 40] = value
    args[0][2, 1, 4, 40] = value  # it sees no key
    o, lse2 = run(args, gpu_device)
    assert o[0, 1, 4].isnan().all() and lse2[0, 1, 4].isnan()
    hit = torch.zeros(o.shape[:3], dtype=torch.bool)
    hit[0, 1, 4] = True
    assert torch.equal(o[~hit], clean[~hit]) and torch.equal(lse2[~hit], lse[~hit])


def test_lengths_outside_the_table(gpu_device):
    args = list(make([60, 60, 60], 2, 2, 2, 64, 20, HF, 4, width=0))
    args[4] = torch.tensor([-3, 61, 2 ** 31 - 1], dtype=torch.int32)
    o, lse = run(args, gpu_device)
    check(o, lse, reference(args), args)


def test_layouts(gpu_device):
    dev = gpu_device
    q, k, v, table, lens = make([333, 50], 1, 8, 2, 64, 16, BF, 5)
    want, _ = run((q, k, v, table, lens), dev)
    q, table, lens = q.to(dev), table.to(dev), lens.to(dev)
    slot_major = [FP4Cache(*(t.to(dev) for t in c)) for c in (k, v)]
    got, _ = paged_flash_attn_inference_func(q, *slot_major, table, lens)
    assert torch.equal(want[:], got)
    both = [torch.stack([k[i], v[i]], 1).to(dev) for i in range(2)]  # k and v of a page together
    got, _ = paged_flash_attn_inference_func(q[:, 0], *(FP4Cache(both[0][:, i], both[1][:, i]) for i in range(2)),
                                             table[:, :30].t().contiguous().t(), lens)
    assert torch.equal(want[:, 0], got)
    wide = torch.cat([q, q], -1)[..., 3:67]
    wide.copy_(q)
    got, _ = paged_flash_attn_inference_func(wide, on_gpu(k, dev), slot_major[1], table, lens)
    assert torch.equal(want, got)


def test_single_entries_and_empty_pools(gpu_device):
    dev = gpu_device
    args = make([30], 1, 1, 1, 64, 32, HF, 9, spare=0, width=0)
    want, _ = run(args, dev)
    q, table, lens = (args[i].to(dev) for i in (0, 3, 4))
    kv = [FP4Cache(c[0].to(dev).as_strided((1, 32, 1, 32), (7, 32, 9, 1)), c[1].to(dev).as_strided((1, 32, 1, 2), (5, 2, 3, 1)))
          for c in args[1:3]]
    got, _ = paged_flash_attn_inference_func(q, *kv, table, lens)
    assert torch.equal(want, got)
    none = fp4_paged_cache(0, 32, 1, 64, device=dev)
    for tab in (table, table[:, :0]):
        o, lse = paged_flash_attn_inference_func(q, none, none, tab, lens, return_lse=True)
        assert (o == 0).all() and (lse == -math.inf).all()
    e, _ = paged_flash_attn_inference_func(q[:0], *kv, table[:0], lens[:0])
    assert e.shape == (0, 1, 1, 64)


def test_offsets_past_32_bits(gpu_device):
    """Pages 2^27 bytes apart: the last begins more than 2^32 bytes behind the first."""
    dev, pages, page = gpu_device, 40, 64
    q, k, v, table, lens = make([pages * page - 7], 1, 4, 1, 64, page, BF, 12, spare=0)
    near = [on_gpu(c, dev) for c in (k, v)]
    room = torch.empty((pages - 1) * (1 << 27) + page * 32, device=dev, dtype=torch.uint8)
    far = FP4Cache(room.as_strided((pages, page, 1, 32), (1 << 27, 32, 32, 1)), near[0].scales)
    far.codes.copy_(near[0].codes)
    rest = (table.to(dev), lens.to(dev))
    want, _ = paged_flash_attn_inference_func(q.to(dev), *near, *rest)
    got, _ = paged_flash_attn_inference_func(q.to(dev), far, near[1], *rest)
    assert torch.equal(want, got)
    far.codes.copy_(near[1].codes)
    got, _ = paged_flash_attn_inference_func(q.to(dev), near[0], FP4Cache(far.codes, near[1].scales), *rest)
    assert torch.equal(want, got)


def test_replays_follow_table_and_lengths(gpu_device):
    dev = gpu_device
    q, k, v, table, lens = make([900, 20, 333], 1, 4, 4, 64, 16, HF, 6)
    q, table, lens = q.to(dev), table.to(dev), lens.to(dev)
    k, v = on_gpu(k, dev), on_gpu(v, dev)
    paged_flash_attn_inference_func(q, k, v, table, lens)
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, _ = paged_flash_attn_inference_func(q, k, v, table, lens)
    for new in ([900, 20, 333], [1, 0, 2], [640, 32, 100], [900, 21, 333]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize(dev)
        assert torch.equal(o, paged_flash_attn_inference_func(q, k, v, table, lens)[0]), new


def test_a_row_alone(gpu_device):
    """A row's bits depend on its query and what it sees: not on the other rows of its tile, nor on later keys."""
    dev = gpu_device
    q, k, v, table, lens = make([777, 300], 6, 4, 1, 64, 16, BF, 14)
    k, v, table = on_gpu(k, dev), on_gpu(v, dev), table.to(dev)
    o, lse = paged_flash_attn_inference_func(q.to(dev), k, v, table, lens.to(dev), return_lse=True)
    loud = q.clone()
    loud[:, 1:] *= 40
    o2, lse2 = paged_flash_attn_inference_func(loud.to(dev), k, v, table, lens.to(dev), return_lse=True)
    assert torch.equal(o[:, 0], o2[:, 0]) and torch.equal(lse[:, 0], lse2[:, 0])


def test_two_streams_and_two_graphs(gpu_device):
    """Calls under way at once, and captured ones replayed in turn, have workspaces of their own."""
    dev = gpu_device
    calls = []
    for seed, (lens, hq, hk, d) in enumerate([([9000, 4000, 31], 8, 2, 64), ([12000, 500], 4, 4, 128)]):
        q, k, v, table, n = make(lens, 2, hq, hk, d, 16, BF, 60 + seed)
        args = (q.to(dev), on_gpu(k, dev), on_gpu(v, dev), table.to(dev), n.to(dev))
        calls.append(lambda args=args: paged_flash_attn_inference_func(*args)[0])
    want = [call() for call in calls]
    torch.cuda.synchronize(dev)
    streams, got = [torch.cuda.Stream(dev) for _ in calls], [[], []]
    for _ in range(5):
        for i, (s, call) in enumerate(zip(streams, calls)):
            with torch.cuda.stream(s):
                got[i].append(call())
    torch.cuda.synchronize(dev)
    for outs, ref in zip(got, want):
        assert all(torch.equal(o, ref) for o in outs)
    graphs = []
    for call in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    for _ in range(3):
        for (graph, out), call, ref in zip(graphs, calls, want):
            graph.replay()
            torch.cuda.synchronize(dev)
            assert torch.equal(out, ref) and torch.equal(call(), ref)


@pytest.mark.parametrize("dtype,d,hq,hk", [(BF, 64, 4, 4), (HF, 128, 8, 2)])
def test_a_stream_of_steps(gpu_device, dtype, d, hq, hk):
    """The run as it is used: whole scenes written into 4 bits and attended to as packed rows read back, then steps that
    append a few tokens and attend over all, each against the oracle on what the cache then holds."""
    dev, g, page = gpu_device, torch.Generator().manual_seed(15), 32
    lens = [200, 45, 0]
    pool = 24
    table = torch.randperm(pool, generator=g).to(torch.int32).view(3, 8)
    cache = [fp4_paged_cache(pool, page, hk, d, device=dev) for _ in range(2)]
    dims = (16, 24, 24) if d == 64 else (32, 48, 48)

    def tokens(*lead):
        y = torch.randn(*lead, (hq + 2 * hk) * d, generator=g).to(dtype).to(dev).unflatten(-1, (-1, d))
        pos = torch.randint(0, 40, (*lead, 3), generator=g).to(torch.int32).to(dev)
        return y[..., :hq, :], y[..., hq:hq + hk, :], y[..., hq + hk:, :], pos

    q, k, v, pos = tokens(sum(lens))
    cu = torch.tensor([0, 200, 245, 245], dtype=torch.int32, device=dev)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    q = paged_kv_append_func(k, v, *cache, table.to(dev), n, q=q, positions=pos, axis_dims=dims, cu_seqlens=cu)
    kr, vr = paged_kv_read_func(*cache, table.to(dev), cu, sum(lens), dtype=dtype)
    o, lse = packed_flash_attn_inference_func(q, kr, vr, cu, return_lse=True)
    for b, a, e in ((0, 0, 200), (1, 200, 245)):  # the same over the pages
        one, lse1 = paged_flash_attn_inference_func(q[None, a:e], *cache, table[b:b + 1].to(dev), n[b:b + 1], causal=False,
                                                    return_lse=True)
        kept = [tuple(t.cpu() for t in c) for c in cache]
        args = (q[None, a:e].cpu(), *kept, table[b:b + 1], n[b:b + 1].cpu())
        ref = reference(args, causal=False)
        check(one, lse1, ref, args)
        assert ((o[a:e].double().cpu() - ref[0][0]).abs() <= 2.0 ** -8 * (ref[0][0].abs() + 1.5 * ref[2][0])).all()
    for step in range(3):
        new = (1, 5, 1)[step]
        n += new
        q, k, v, pos = tokens(3, new)
        q = paged_kv_append_func(k, v, *cache, table.to(dev), n, q=q, positions=pos, axis_dims=dims)
        o, lse = paged_flash_attn_inference_func(q, *cache, table.to(dev), n, return_lse=True)
        args = (q.cpu(), *(tuple(t.cpu() for t in c) for c in cache), table, n.cpu())
        check(o, lse, reference(args), args)
