"""gw_paged_kv_append and gw_paged_kv_read against the 64-bit oracle.

Tolerances. The angles are formed in 64 bits and their cosines and sines rounded once to fp32, the two products and
their sum once each: a turned value is off by at most 2 * 2^-24 (|x1| + |x2|) + 2^-24 |y|, below ``near`` = 4 * 2^-24
(|x1| + |x2|), and by half a step, u |y|, in 16 bits. In 4 bits the codes of v, which is not turned, are the oracle's bit
by bit; a code of k lies between those of the exact value less and plus ``near``, and so does a power of two."""
import math

import pytest
import torch

from geoweave_amd.custom_flash_attn.paged_kv_cache import (FP4Cache, fp4_paged_cache, paged_kv_append_func,
                                                           paged_kv_read_func)
from geoweave_amd.rotary import rotary_axes_qk_func
from oracle.packed_attention import rotary_axes
from oracle.paged_kv import fp4_codes, fp4_decode, fp4_encode, fp4_scales, read_slots, token_slots

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def tables(lens, page, g, spare=3, width=2):
    pages = [-(-max(n, 0) // page) for n in lens]
    pool = sum(pages) + spare
    order = torch.randperm(pool, generator=g)
    table = torch.full((len(lens), max(pages + [0]) + width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n].to(torch.int32)
        at += n
    return table, pool


def caches(fp4, pool, page, hk, d, dtype, g, dev):
    """(CPU copies, GPU caches) of old contents."""
    if not fp4:
        old = [torch.randn(pool, page, hk, d, generator=g).to(dtype) for _ in range(2)]
        return [(o,) for o in old], [o.to(dev) for o in old]
    old, new = [], []
    for _ in range(2):
        c = fp4_paged_cache(pool, page, hk, d, device=dev)
        o = (torch.randint(0, 256, c.codes.shape, generator=g).to(torch.uint8),
             torch.randint(100, 140, c.scales.shape, generator=g).to(torch.uint8))
        for x, y in zip(c, o):
            x.copy_(y)
        old.append(o)
        new.append(c)
    return old, new


def parts(cache):
    return tuple(t.cpu() for t in cache) if isinstance(cache, FP4Cache) else (cache.cpu(),)


def turned(x, pos, dims, bases):
    """(64-bit turned x, near)."""
    if dims is None:
        return x.double(), torch.zeros(x.shape, dtype=torch.float64)
    y = rotary_axes(x, pos, dims, bases)
    mag = x.double().abs()
    at = 0
    for n in dims:
        pair = mag[..., at:at + n // 2] + mag[..., at + n // 2:at + n]
        mag[..., at:at + n] = torch.cat([pair, pair], -1)
        at += n
    mag[..., at:] = 0
    return y, 4 * 2.0 ** -24 * mag


def check16(got, y, near, dtype):
    u = torch.finfo(dtype).eps / 2
    lim = near + u * (y.abs() + near) + (2.0 ** -25 if dtype == HF else 0.0)
    assert ((got.double() - y).abs() <= lim).all()


def check4(codes, scales, y, near):
    """Codes [T, H, D / 2], scales [T, H, D / 32] of y [T, H, D], each value off by at most near."""
    groups = lambda t: t.unflatten(-1, (-1, 32))  # noqa: E731
    a = groups(y.abs())
    low, high = (fp4_scales((a + s * groups(near)).amax(-1)) for s in (-1, 1))
    assert ((scales >= low) & (scales <= high)).all()
    unit = torch.pow(2.0, 127.0 - scales.double())[..., None]
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    least, most = (groups(y) + s * groups(near) for s in (-1, 1))
    order = lambda c: torch.where(c >= 8, -(c.int() & 7), c.int() & 7)  # noqa: E731
    got = order(groups(code))
    assert ((got >= order(fp4_codes(least * unit))) & (got <= order(fp4_codes(most * unit)))).all()


def check_append(dev, fp4, dtype, hq, hk, d, page, lens, dims=None, bases=None, count=None, cu=None, tokens=None, far=64,
                 pos_type=torch.int32, seed=0, table=None, edit=None):
    g = torch.Generator().manual_seed(seed)
    made, pool = tables(lens, page, g)
    table = made if table is None else table
    old, new = caches(fp4, pool, page, hk, d, dtype, g, dev)
    lead = (len(lens), count) if cu is None else (tokens,)
    t = math.prod(lead)
    y = torch.randn(t, (hq + 2 * hk) * d, generator=g).to(dtype)
    if edit:
        edit(y)
    pos = torch.stack([torch.randint(0, far, lead, generator=g) for _ in dims], -1).to(pos_type) if dims else None
    on = y.to(dev)
    q, k, v = (on[:, a * d:b * d].view(*lead, b - a, d) for a, b in ((0, hq), (hq, hq + hk), (hq + hk, hq + 2 * hk)))
    out = paged_kv_append_func(k, v, *new, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                               q=q if hq else None, positions=None if pos is None else pos.to(dev), axis_dims=dims,
                               bases=100.0 if bases is None else bases,
                               cu_seqlens=None if cu is None else torch.tensor(cu, dtype=torch.int32, device=dev))
    torch.cuda.synchronize(dev)
    flat = None if pos is None else pos.view(t, -1)
    base = [100.0] * len(dims or ()) if bases is None else bases
    qy, kx, vx = (y[:, a * d:b * d].view(t, b - a, d) for a, b in ((0, hq), (hq, hq + hk), (hq + hk, hq + 2 * hk)))
    if hq:
        assert out.is_contiguous() and out.shape == q.shape
        check16(out.cpu().view(t, hq, d), *turned(qy, flat, dims, base), dtype)
    else:
        assert out is None
    slots = token_slots(lens, table, page, pool, count, cu, tokens)
    live = [i for i, s in enumerate(slots) if s is not None]
    at = tuple(torch.tensor([slots[i][x] for i in live], dtype=torch.long) for x in (0, 1))
    ky, near = turned(kx, flat, dims, base)
    for was, cache, x, tol, is_k in ((old[0], new[0], ky, near, True), (old[1], new[1], vx.double(), None, False)):
        now = parts(cache)
        if fp4:
            if is_k:
                check4(now[0][at], now[1][at], x[live], tol[live])
            else:
                for a, b in zip(now, fp4_encode(x[live])):
                    assert torch.equal(a[at], b)
        elif is_k:
            check16(now[0][at], x[live], tol[live], dtype)
        else:
            assert torch.equal(now[0][at].view(torch.int16), vx[live].view(torch.int16))
        for a, b in zip(was, now):  # every other slot as it was
            a, b = (z.contiguous().view(torch.uint8).clone() for z in (a, b))
            a[at] = b[at] = 0
            assert torch.equal(a, b)
    return new


AXES = [(None, None), ((64,), (100.0,)), ((16, 24, 24), (100.0, 100.0, 50.0)), ((18, 14, 20), (100.0, 10000.0, 3.0)),
        ((4, 0, 2, 8, 10, 12, 6, 6), (100.0,) * 8), ((32, 32), (10000.0, 100.0))]


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,hq,hk", [(64, 4, 2), (128, 3, 3), (64, 0, 1), (128, 8, 1), (64, 17, 5)])
@pytest.mark.parametrize("axes", range(len(AXES)))
def test_values(gpu_device, fp4, dtype, d, hq, hk, axes):
    dims, bases = AXES[axes]
    check_append(gpu_device, fp4, dtype, hq, hk, d, 16, [5, 33, 16, 100], dims, bases, count=5, seed=axes)


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("lens,count,page", [([1], 1, 64), ([700], 700, 100), ([300, 299, 5], 2, 1), ([40] * 3, 40, 300),
                                             ([2000 + i for i in range(70)], 1, 16)])
def test_sizes(gpu_device, fp4, lens, count, page):
    check_append(gpu_device, fp4, BF, 4, 2, 64, page, lens, (16, 24, 24), None, count=count)


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("cu,tokens", [([0, 3, 3, 10, 41], 41), ([2, 2, 7, 9, 9], 13), ([0, 0, 0, 0, 0], 4), ([0, 37, 37, 37, 41], 41)])
def test_packed_bounds(gpu_device, fp4, cu, tokens):
    """Empty sequences, and tokens before the first and behind the last bound."""
    check_append(gpu_device, fp4, BF, 2, 2, 128, 24, [50, 20, 7, 64], (64, 64), None, cu=cu, tokens=tokens)


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("d,hq,hk", [(64, 1, 2), (128, 2, 1)])
def test_many_tokens(gpu_device, fp4, d, hq, hk):
    """Eight tokens to a workgroup, the last of them with fewer, sequences that end inside one."""
    check_append(gpu_device, fp4, BF, hq, hk, d, 40, [5000, 3300, 90], (d,), None, cu=[0, 5000, 8197, 8261], tokens=8263)


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_many_heads(gpu_device, fp4, d):
    """More heads than a workgroup takes of one token."""
    check_append(gpu_device, fp4, HF, 300, 70, d, 8, [9, 20], (16, 24), None, count=3)
    dev, g = gpu_device, torch.Generator().manual_seed(17)
    table, pool = tables([9, 20], 8, g)
    old, new = caches(fp4, pool, 8, 170, d, HF, g, dev)
    k, v = paged_kv_read_func(*new, table.to(dev), torch.tensor([0, 9, 29], dtype=torch.int32, device=dev), 29, dtype=HF)
    for was, got in zip(old, (k, v)):
        rows = fp4_decode(*was).float().to(HF) if fp4 else was[0]
        want = torch.stack([rows[s] for s in read_slots([0, 9, 29], table, 8, pool, 29)])
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("n", [1, 63, 64, 65, 200, 4200])
def test_packed_many_sequences(gpu_device, n):
    g = torch.Generator().manual_seed(n)
    counts = torch.randint(0, 4, (n,), generator=g).tolist()
    lens = [c + int(x) for c, x in zip(counts, torch.randint(0, 30, (n,), generator=g))]
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    check_append(gpu_device, True, BF, 1, 1, 64, 8, lens, (32, 32), None, cu=cu, tokens=cu[-1] + 3)


@pytest.mark.parametrize("fp4", [False, True])
def test_tokens_without_a_slot(gpu_device, fp4):
    """Lengths below the new tokens' number and behind the table, pages outside the pool."""
    dev, g = gpu_device, torch.Generator().manual_seed(5)
    table, pool2 = tables([60, 16, 64, 16, 64, 64, 64], 16, g, width=0)
    lens = [60, 2, 200, -4, 2 ** 31 - 1, 64, 34]
    table[0, 3], table[5, 3], table[6, 1] = -1, 10 ** 6, pool2
    old, new = caches(fp4, pool2, 16, 2, 64, BF, g, dev)
    k, v = (torch.randn(7, 5, 2, 64, generator=g).to(BF) for _ in range(2))
    paged_kv_append_func(k.to(dev), v.to(dev), *new, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev))
    slots = token_slots(lens, table, 16, pool2, 5)
    assert sum(s is not None for s in slots) == 4
    for was, cache, x in ((old[0], new[0], k), (old[1], new[1], v)):
        want = [t.clone() for t in was]
        enc = fp4_encode(x) if fp4 else (x,)
        for i, s in enumerate(slots):
            if s is not None:
                for w, e in zip(want, enc):
                    w[s] = e.flatten(0, 1)[i]
        for w, got in zip(want, parts(cache)):
            assert torch.equal(w.contiguous().view(torch.uint8), got.contiguous().view(torch.uint8))


@pytest.mark.parametrize("dtype", [BF, HF])
def test_four_bits_of_special_values(gpu_device, dtype):
    """Rows of zeros, of one value, at the powers' borders, tiny, huge, and with inf and NaN."""
    top = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # the smallest subnormal
    values = [0.0, -0.0, 1.0, 7.0, 7.03125, 3.5, 3.515625, 6.0, 5.0, 2.5, 1.75, 0.75, 0.25, -5.0, -0.25, top, -top / 2, tiny,
              7 * tiny, 1e-4, math.inf, -math.inf, math.nan]
    g = torch.Generator().manual_seed(0)

    def edit(y):
        rows = y.view(-1, 32)
        for i, x in enumerate(values):
            rows[2 * i].mul_(min(max(abs(x), tiny * 100), 1e4) / 4 if math.isfinite(x) else 1.0)
            if math.isfinite(x):
                rows[2 * i].clamp_(-abs(x), abs(x))
            rows[2 * i, int(torch.randint(0, 32, (1,), generator=g))] = x
            rows[2 * i + 1] = x
        rows[2 * len(values), :] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4)
        rows[2 * len(values) + 1, :] = -rows[2 * len(values)]

    # v alone is checked bit by bit; k = v without positions
    n = 40
    y = torch.randn(n, 64, generator=g).to(dtype)
    edit(y)
    dev = gpu_device
    cache = [fp4_paged_cache(3, 16, 1, 64, device=dev) for _ in range(2)]
    table = torch.tensor([[1, 2, 0]], dtype=torch.int32, device=dev)
    x = y.view(n, 1, 64).to(dev)
    paged_kv_append_func(x, x, *cache, table, torch.tensor([n], dtype=torch.int32, device=dev),
                         cu_seqlens=torch.tensor([0, n], dtype=torch.int32, device=dev))
    codes, scales = fp4_encode(y.view(n, 1, 64))
    at = torch.tensor([1] * 16 + [2] * 16 + [0] * 8), torch.arange(n) % 16
    for c in cache:
        got = parts(c)
        assert torch.equal(got[1][at], scales)
        assert torch.equal(got[0][at], codes)
    assert (scales == 255).sum() >= 6 and (scales == 0).sum() >= 1
    k, v = paged_kv_read_func(*cache, table, torch.tensor([0, n], dtype=torch.int32, device=dev), n, dtype=dtype)
    want = fp4_decode(codes, scales)
    want = want.float().to(dtype)  # exact in bf16; fp16: one rounding
    assert torch.equal(k.cpu().isnan(), want.isnan()) and torch.equal(k.cpu().nan_to_num(1.0), want.nan_to_num(1.0))
    assert torch.equal(k.view(torch.int16), v.view(torch.int16))


@pytest.mark.parametrize("pos_type,far", [(torch.int64, 10 ** 6), (torch.float32, 1000), (torch.int32, 10 ** 6)])
def test_positions(gpu_device, pos_type, far):
    check_append(gpu_device, False, HF, 2, 1, 64, 16, [40, 9], (32, 32), (10000.0, 100.0), count=9, far=far, pos_type=pos_type)


def test_agrees_with_the_rotation_of_its_own(gpu_device):
    """The same angles: a value differs from rotary_axes_qk_func's by one rounding of the type at most."""
    dev, g = gpu_device, torch.Generator().manual_seed(3)
    q, k = torch.randn(50, 4, 64, generator=g).to(BF).to(dev), torch.randn(50, 2, 64, generator=g).to(BF).to(dev)
    pos = torch.randint(0, 40, (50, 3), generator=g).to(torch.int32).to(dev)
    kc, vc = (torch.zeros(4, 16, 2, 64, dtype=BF, device=dev) for _ in range(2))
    table = torch.arange(4, dtype=torch.int32, device=dev)[None]
    out = paged_kv_append_func(k, k, kc, vc, table, torch.tensor([50], dtype=torch.int32, device=dev), q=q, positions=pos,
                               axis_dims=(16, 24, 24), cu_seqlens=torch.tensor([0, 50], dtype=torch.int32, device=dev))
    want = rotary_axes_qk_func(q, k, pos, (16, 24, 24))
    for a, b in ((out, want[0]), (kc.view(64, 2, 64)[:50], want[1])):
        # Both round, by at most half a step (2^-8 of the value) each, values that differ by less than 2^-22 of |x1| + |x2|
        # <= 12: two such values on the two sides of a middle end a whole step, 2 * 2^-8, apart.
        assert ((a.float() - b.float()).abs() <= 2 * 2.0 ** -8 * b.float().abs() * 1.01 + 2.0 ** -18).all()


@pytest.mark.parametrize("fp4", [False, True])
def test_one_token_form_layouts_and_copies(gpu_device, fp4):
    """[B, H, D] is [B, 1, H, D]; slot-major codes, pages of both caches in one tensor, tables and lengths that are
    views, and rows of tokens that have to be copied give the same bits."""
    dev, g = gpu_device, torch.Generator().manual_seed(7)
    lens = [33, 64, 5]
    table, pool = tables(lens, 16, g)
    k, v, q = (torch.randn(3, 1, h, 64, generator=g).to(BF).to(dev) for h in (2, 2, 4))
    pos = torch.randint(0, 40, (3, 1, 2), generator=g).to(torch.int32).to(dev)
    lens = torch.tensor(lens, dtype=torch.int32, device=dev)
    table = table.to(dev)

    def empty(slot_major=False):
        if not fp4:
            if slot_major:
                both = torch.zeros(pool, 2, 2, 16, 64, dtype=BF, device=dev)
                return [both[:, i].transpose(1, 2) for i in range(2)]
            return [torch.zeros(pool, 16, 2, 64, dtype=BF, device=dev) for _ in range(2)]
        if slot_major:
            both = [torch.zeros(pool, 2, 16, 2, w, dtype=torch.uint8, device=dev) for w in (32, 2)]
            return [FP4Cache(both[0][:, i], both[1][:, i]) for i in range(2)]
        return [fp4_paged_cache(pool, 16, 2, 64, device=dev) for _ in range(2)]

    first, want = empty(), None
    want = paged_kv_append_func(k, v, *first, table, lens, q=q, positions=pos, axis_dims=(32, 32))
    wide = torch.zeros(3, 1, 2, 67, dtype=BF, device=dev)[..., 3:]
    wide.copy_(k)
    columns = torch.zeros(3, 2 * table.shape[1], dtype=torch.int32, device=dev)
    columns[:, ::2] = table
    spread = torch.zeros(6, dtype=torch.int32, device=dev)
    spread[::2] = lens
    for args, other in (((k[:, 0], v[:, 0]), dict(q=q[:, 0], positions=pos[:, 0])),
                        ((wide, v.transpose(2, 3).contiguous().transpose(2, 3)), dict(q=q, positions=pos.expand(3, 1, 2)))):
        cache = empty(True)
        out = paged_kv_append_func(*args, *cache, columns[:, ::2], spread[::2], axis_dims=(32, 32), **other)
        assert torch.equal(out.view(want.shape), want)
        for a, b in zip(first, cache):
            assert all(torch.equal(x, y) for x, y in zip(parts(a), parts(b)))


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,hk", [(64, 1), (64, 5), (128, 2)])
@pytest.mark.parametrize("cu,more", [([0, 1], 0), ([0, 100, 100, 133, 140], 5), ([3, 50, 51], 0), ([0, 6000, 8205], 2)])
def test_read(gpu_device, fp4, dtype, d, hk, cu, more):
    dev, g = gpu_device, torch.Generator().manual_seed(11)
    lens = [b - a for a, b in zip(cu[:-1], cu[1:])]
    page = 24
    table, pool = tables(lens, page, g)
    if len(lens) > 1:
        table[0, 1] = -7
    old, new = caches(fp4, pool, page, hk, d, dtype, g, dev)
    n = cu[-1] + more
    k, v = paged_kv_read_func(*new, table.to(dev), torch.tensor(cu, dtype=torch.int32, device=dev), n, dtype=dtype)
    assert k.shape == v.shape == (n, hk, d) and k.dtype == v.dtype == dtype and k.is_contiguous() and v.is_contiguous()
    slots = read_slots(cu, table, page, pool, n)
    for was, got in zip(old, (k, v)):
        rows = fp4_decode(*was).float().to(dtype) if fp4 else was[0]
        want = torch.stack([rows[s] if s is not None else torch.zeros(hk, d, dtype=dtype) for s in slots])
        assert torch.equal(got.cpu(), want)


def test_bounds_longer_than_the_table_and_out_of_order(gpu_device):
    dev = gpu_device
    cache = [torch.ones(2, 8, 1, 64, dtype=BF, device=dev) for _ in range(2)]
    table = torch.tensor([[0, 1]], dtype=torch.int32, device=dev)
    k, _ = paged_kv_read_func(*cache, table, torch.tensor([0, 40], dtype=torch.int32, device=dev), 40)
    assert (k[:16] == 1).all() and (k[16:] == 0).all()
    for cu in ([30, 2], [-5, 10], [0, 2 ** 31 - 1], [-2 ** 31, 2 ** 31 - 1]):
        b = torch.tensor(cu, dtype=torch.int32, device=dev)
        paged_kv_read_func(*cache, table, b, 20)
        x = torch.ones(20, 1, 64, dtype=BF, device=dev)
        paged_kv_append_func(x, x, *cache, table, torch.tensor([16], dtype=torch.int32, device=dev), cu_seqlens=b)
    torch.cuda.synchronize(dev)


def test_empty_calls(gpu_device):
    dev = gpu_device
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    for cache in ([torch.zeros(0, 16, 2, 64, dtype=BF, device=dev)] * 2, [fp4_paged_cache(0, 16, 2, 64, device=dev)] * 2):
        x = torch.ones(2, 2, 64, dtype=BF, device=dev)
        q = paged_kv_append_func(x, x, *cache, ints(0, 0)[:, None], ints(1, 1), q=x)  # no pages: nothing written
        assert torch.equal(q, x)
        assert paged_kv_append_func(x[:0], x[:0], *cache, ints()[:, None].expand(0, 3), ints()) is None
        q = paged_kv_append_func(x, x, *cache, ints()[:, None].expand(0, 3), ints(), q=x, cu_seqlens=ints(0))
        assert torch.equal(q, x)
        k, v = paged_kv_read_func(*cache, ints(0)[:, None], ints(0, 3), 4)
        assert (k == 0).all() and (v == 0).all()
        assert paged_kv_read_func(*cache, ints(0)[:, None], ints(0, 0), 0)[0].shape == (0, 2, 64)


def test_offsets_past_32_bits(gpu_device):
    """Pages 2^27 bytes apart: the last begins more than 2^32 bytes behind the first."""
    dev, pages, page = gpu_device, 40, 16
    room = torch.empty((pages - 1) * (1 << 27) + page * 32, device=dev, dtype=torch.uint8)
    far = [FP4Cache(room.as_strided((pages, page, 1, 32), (1 << 27, 32, 32, 1)),
                    torch.zeros(pages, page, 1, 2, device=dev, dtype=torch.uint8)),
           fp4_paged_cache(pages, page, 1, 64, device=dev)]
    near = [fp4_paged_cache(pages, page, 1, 64, device=dev) for _ in range(2)]
    n = pages * page
    x = torch.randn(n, 1, 64, device=dev, dtype=BF)
    table = torch.randperm(pages, device=dev).to(torch.int32)[None]
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    for c in (far, near):
        paged_kv_append_func(x, x, *c, table, cu[1:], cu_seqlens=cu)
    assert torch.equal(far[0].codes, near[0].codes) and torch.equal(far[0].scales, near[0].scales)
    assert torch.equal(paged_kv_read_func(*far, table, cu, n)[0], paged_kv_read_func(*near, table, cu, n)[0])


@pytest.mark.parametrize("fp4", [False, True])
def test_replays_follow_positions_table_and_lengths(gpu_device, fp4):
    dev, g = gpu_device, torch.Generator().manual_seed(13)
    table, pool = tables([90, 40], 16, g)
    table = table.to(dev)
    lens = torch.tensor([90, 40], dtype=torch.int32, device=dev)
    k, v, q = (torch.randn(2, 3, h, 64, generator=g).to(BF).to(dev) for h in (2, 2, 4))
    pos = torch.randint(0, 40, (2, 3, 2), generator=g).to(torch.int32).to(dev)
    cu = torch.tensor([0, 90, 130], dtype=torch.int32, device=dev)

    def fresh():
        if fp4:
            return [fp4_paged_cache(pool, 16, 2, 64, device=dev) for _ in range(2)]
        return [torch.zeros(pool, 16, 2, 64, dtype=BF, device=dev) for _ in range(2)]

    def step(cache):
        out = paged_kv_append_func(k, v, *cache, table, lens, q=q, positions=pos, axis_dims=(32, 32))
        return out, *paged_kv_read_func(*cache, table, cu, 130)

    kept, eager = fresh(), fresh()
    step(kept)
    for c in kept:
        for t in (c if fp4 else (c,)):
            t.zero_()
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(kept)
    for i, new in enumerate(([90, 40], [20, 3], [50, 1], [64, 17])):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        pos.add_(1)
        k.copy_(torch.randn(k.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize(dev)
        want = step(eager)
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i
    for a, b in zip(kept, eager):
        assert all(torch.equal(x, y) for x, y in zip(parts(a), parts(b)))


def test_a_stream_of_its_own(gpu_device):
    dev, g = gpu_device, torch.Generator().manual_seed(14)
    k = torch.randn(4000, 4, 64, generator=g).to(BF).to(dev)
    table = torch.arange(250, dtype=torch.int32, device=dev)[None]
    cu = torch.tensor([0, 4000], dtype=torch.int32, device=dev)
    pos = torch.randint(0, 60, (4000, 1), generator=g).to(torch.int32).to(dev)
    want, got = ([fp4_paged_cache(250, 16, 4, 64, device=dev) for _ in range(2)] for _ in range(2))
    paged_kv_append_func(k, k, *want, table, cu[1:], positions=pos, axis_dims=(64,), cu_seqlens=cu)
    ref = paged_kv_read_func(*want, table, cu, 4000)
    torch.cuda.synchronize(dev)
    side = torch.cuda.Stream(dev)
    with torch.cuda.stream(side):
        late = torch.zeros_like(k)
        for _ in range(20):
            late = late + 0.0
        late.copy_(k)
        paged_kv_append_func(late, late, *got, table, cu[1:], positions=pos, axis_dims=(64,), cu_seqlens=cu)
        out = paged_kv_read_func(*got, table, cu, 4000)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, out))
