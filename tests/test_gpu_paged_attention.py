"""Paged attention (gw_paged_attn_fwd) against the 64-bit oracle.

Tolerance: the weights are rounded once to the 16-bit type before the product with V (their sum is
not) and the output once, so with u = eps / 2 |error| <= u (|o| + P|V|); the fp32 sums of a score's D products
change a weight by at most 2 D 2^-24 of the score's magnitudes, the other fp32 sums add less than 2^-18."""
import math

import pytest
import torch

from geoweave_amd.custom_flash_attn.packed_flash_attn import packed_flash_attn_inference_func
from geoweave_amd.custom_flash_attn.paged_flash_attn import paged_flash_attn_inference_func
from oracle.packed_attention import paged_attention

pytestmark = pytest.mark.gpu


def make(lens, new, hq, hk, d, page, dtype, seed=0, spare=3, width=2, gain=1.5):
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
    k, v = (torch.randn(pool, page, hk, d, generator=g).to(dtype) for _ in range(2))
    return q, k, v, table, torch.tensor(lens, dtype=torch.int32)


def run(args, dev, **kw):
    return paged_flash_attn_inference_func(*(t.to(dev) for t in args), return_lse=True, **kw)


def check(got, lse, ref, dtype, d):
    o, want_lse, mag, s_mag = ref
    u = torch.finfo(dtype).eps / 2
    s = 2 * d * 2.0 ** -24 * float(s_mag.max()) + 2.0 ** -18
    lim = 1.01 * u * o.abs() + (u + 4 * s) * mag + (2.0 ** -20 if dtype == torch.float16 else 2.0 ** -60)
    err = (got.double().cpu() - o).abs()
    assert torch.isfinite(got).all()
    assert (err <= lim).all(), float((err / lim).max())
    a = lse.double().cpu()
    assert torch.equal(a == -math.inf, want_lse == -math.inf)
    on = want_lse != -math.inf
    assert ((a - want_lse)[on].abs() <= 2.0 ** -17 * (1 + s_mag[on])).all()


LENS = {
    "one key": [1],
    "edges": [1, 0, 15, 16, 17, 31, 32, 33, 127, 128, 129, 300],
    "ragged": [4000, 3, 700, 1, 129],
    "long": [20011],
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,hk", [(64, 2, 2), (128, 8, 1), (64, 6, 2), (128, 3, 3)])
@pytest.mark.parametrize("new,page,causal", [(1, 16, True), (1, 100, True), (5, 64, True), (7, 1, False), (9, 7, True)])
@pytest.mark.parametrize("lens", list(LENS))
def test_values(gpu_device, dtype, d, hq, hk, new, page, causal, lens):
    args = make(LENS[lens], new, hq, hk, d, page, dtype)
    o, lse = run(args, gpu_device, causal=causal)
    check(o, lse, paged_attention(*args, causal=causal), dtype, d)
    again, lse2 = run(args, gpu_device, causal=causal)
    assert torch.equal(o, again) and torch.equal(lse, lse2), "the same inputs give the same bits"


def test_many_sequences_without_a_split(gpu_device):
    lens = torch.randint(0, 90, (4200,), generator=torch.Generator().manual_seed(1)).tolist()
    args = make(lens, 1, 2, 1, 64, 32, torch.bfloat16)
    o, lse = run(args, gpu_device)
    check(o, lse, paged_attention(*args), torch.bfloat16, 64)


def test_more_sequences_than_one_scan_round(gpu_device):
    lens = torch.randint(0, 200, (150,), generator=torch.Generator().manual_seed(2)).tolist()
    lens[70] = 9000
    args = make(lens, 3, 4, 2, 128, 48, torch.float16)
    o, lse = run(args, gpu_device)
    check(o, lse, paged_attention(*args), torch.float16, 128)


def test_pages_that_several_sequences_share(gpu_device):
    """A prefix that sequences have in common, and a page that one sequence names twice."""
    args = list(make([200, 330, 96, 2000], 2, 4, 2, 64, 16, torch.bfloat16, 5))
    table = args[3]
    table[1, :6] = table[0, :6]
    table[2, :6] = table[0, :6]
    table[3, 40:80] = table[3, 0:40]
    o, lse = run(args, gpu_device)
    check(o, lse, paged_attention(*args), torch.bfloat16, 64)


def test_unused_slots_and_pages_outside_the_pool(gpu_device):
    """inf and NaN wherever no key lies, page numbers outside the pool in the middle and at the end."""
    args = list(make([300, 77, 500, 40], 4, 4, 2, 64, 24, torch.bfloat16, 3))
    q, k, v, table, lens = args
    used = torch.zeros(k.shape[:2], dtype=torch.bool)
    for b, n in enumerate(lens.tolist()):
        for j in range(n):
            used[table[b, j // 24], j % 24] = True
    k[~used], v[~used] = math.nan, math.inf
    gone = [(0, 2), (0, 12), (2, 0), (2, 5), (3, 0), (3, 1)]
    for (b, p), bad in zip(gone, (-1, 10 ** 6, k.shape[0], -2 ** 31, -5, 2 ** 31 - 1)):
        k[table[b, p]], v[table[b, p]] = math.nan, math.nan
        table[b, p] = bad
    k[0, :, :], v[0, :, :] = (k[0], v[0]) if used[0].any() else (math.nan, math.nan)
    o, lse = run(args, gpu_device)
    check(o, lse, paged_attention(*args), torch.bfloat16, 64)
    assert (o[3] == 0).all() and (lse[3] == -math.inf).all()


@pytest.mark.parametrize("d,hk", [(64, 2), (128, 1)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("n", [40, 1003])
def test_what_a_new_token_does_not_see(gpu_device, d, hk, value, n):
    """inf and NaN in the newest tokens' keys and values reach the tokens that see them and no other."""
    q, k, v, table, lens = make([n, 20], 6, 4, hk, d, 16, torch.float16, 8)
    clean, lse = run((q, k, v, table, lens), gpu_device)
    ref = paged_attention(q, k, v, table, lens)
    j = n - 3  # seen by new tokens 3, 4 and 5
    page, slot = int(table[0, j // 16]), j % 16
    v[page, slot, :, 7] = value
    o, lse2 = run((q, k, v, table, lens), gpu_device)
    assert torch.equal(clean[0, :3], o[0, :3]) and torch.equal(clean[1], o[1]) and torch.equal(lse, lse2)
    assert torch.equal(clean[0, :, :, :7], o[0, :, :, :7]) and torch.equal(clean[0, :, :, 8:], o[0, :, :, 8:])
    got = o[0, 3:, :, 7]
    assert (got == value).all() if value == value else got.isnan().all()
    k[page, slot] = value
    # the rows of a tile raise their running reference together: within the bounds, not the same bits
    o, lse2 = run((q, k, v, table, lens), gpu_device)
    check(o[:1, :3], lse2[:1, :3], tuple(t[:1, :3] for t in ref), torch.float16, d)
    check(o[1:], lse2[1:], tuple(t[1:] for t in ref), torch.float16, d)


def test_lengths_outside_the_table(gpu_device):
    args = list(make([60, 60, 60], 2, 2, 2, 64, 20, torch.float16, 4, width=0))
    args[4] = torch.tensor([-3, 61, 2 ** 31 - 1], dtype=torch.int32)
    o, lse = run(args, gpu_device)
    check(o, lse, paged_attention(*args), torch.float16, 64)


def test_layouts(gpu_device):
    dev = gpu_device
    q, k, v, table, lens = (t.to(dev) for t in make([333, 50], 1, 8, 2, 64, 16, torch.bfloat16, 5))
    want, _ = paged_flash_attn_inference_func(q, k, v, table, lens)
    both = torch.stack([k, v], 1)  # [pages, 2, page, Hk, D]
    got, _ = paged_flash_attn_inference_func(q, both[:, 0], both[:, 1], table, lens)
    assert torch.equal(want, got)
    heads_first = k.transpose(1, 2).contiguous().transpose(1, 2)  # [pages, Hk, page, D] in memory
    got, _ = paged_flash_attn_inference_func(q[:, 0], heads_first, v, table[:, :30].t().contiguous().t(), lens)
    assert torch.equal(want[:, 0], got)
    wide = torch.cat([q, q], -1)[..., 3:67]
    wide.copy_(q)
    got, _ = paged_flash_attn_inference_func(wide, k, v, table, lens)
    assert torch.equal(want, got)


def test_single_entries_and_empty_pools(gpu_device):
    dev = gpu_device
    q, k, v, table, lens = (t.to(dev) for t in make([30], 1, 1, 1, 64, 32, torch.float16, 9, spare=0, width=0))
    want, _ = paged_flash_attn_inference_func(q, k, v, table, lens)
    y = torch.zeros(2, 67, device=dev, dtype=torch.float16)
    y[1, 3:] = q.view(-1)
    odd = y[1:, 3:].as_strided((1, 1, 1, 64), (67, 5, 3, 1), 67 + 3)  # one entry in all dims but the last
    one = k.as_strided((1, 32, 1, 64), (7, 64, 9, 1))
    got, _ = paged_flash_attn_inference_func(odd, one, v, table, lens)
    assert torch.equal(want, got)
    none = k[:0]
    for tab in (table, table[:, :0]):
        o, lse = paged_flash_attn_inference_func(q, none, none, tab, lens, return_lse=True)
        assert (o == 0).all() and (lse == -math.inf).all()
    e, _ = paged_flash_attn_inference_func(q[:0], k, v, table[:0], lens[:0])
    assert e.shape == (0, 1, 1, 64)


def test_offsets_past_32_bits(gpu_device):
    """Pages 2^26 elements apart: the last begins more than 2^32 bytes behind the first."""
    dev, pages, page, d = gpu_device, 40, 64, 64
    room = torch.empty((pages - 1) * (1 << 26) + page * d, device=dev, dtype=torch.bfloat16)
    far = room.as_strided((pages, page, 1, d), (1 << 26, d, d, 1))
    near = torch.randn(pages, page, 1, d, device=dev, dtype=torch.bfloat16)
    far.copy_(near)
    table = torch.randperm(pages, device=dev).to(torch.int32)[None]
    lens = torch.tensor([pages * page - 7], dtype=torch.int32, device=dev)
    q = torch.randn(1, 4, d, device=dev, dtype=torch.bfloat16)
    want, _ = paged_flash_attn_inference_func(q, near, near, table, lens)
    got, _ = paged_flash_attn_inference_func(q, far, far, table, lens)
    assert torch.equal(want, got)


def test_replays_follow_table_and_lengths(gpu_device):
    dev = gpu_device
    q, k, v, table, lens = (t.to(dev) for t in make([900, 20, 333], 1, 4, 4, 64, 16, torch.float16, 6))
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


def test_agrees_with_packed_attention_over_the_same_keys(gpu_device):
    """The run as it is used: a prompt's attention, then new tokens over the cache that it left."""
    dev, page = gpu_device, 32
    lens = [200, 45]
    q, k, v, table, n = (t.to(dev) for t in make(lens, 3, 4, 2, 64, page, torch.bfloat16, 7))
    rows = [(table[b, torch.arange(m, device=dev) // page].long(), torch.arange(m, device=dev) % page) for b, m in enumerate(lens)]
    ks, vs = (torch.cat([c[p, s] for p, s in rows]) for c in (k, v))
    cu_k = torch.tensor([0, 200, 245], dtype=torch.int32, device=dev)
    cu_q = torch.tensor([0, 3, 6], dtype=torch.int32, device=dev)
    packed, plse = packed_flash_attn_inference_func(q.reshape(6, 4, 64), ks, vs, cu_q, cu_k, causal=True, return_lse=True)
    paged, lse = paged_flash_attn_inference_func(q, k, v, table, n, return_lse=True)
    ref = paged_attention(*(t.cpu() for t in (q, k, v, table, n)))
    check(paged, lse, ref, torch.bfloat16, 64)
    check(packed.view(2, 3, 4, 64), plse.view(2, 3, 4), ref, torch.bfloat16, 64)
