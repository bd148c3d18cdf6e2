"""Kept values of V from 2^128 on (scales of 253 and more), which bf16 has no finite number for: they are inf, in the rows that
see their key and in no other."""
import math

import pytest
import torch

from geoweave_amd.custom_flash_attn.paged_flash_attn import paged_flash_attn_inference_func
from geoweave_amd.custom_flash_attn.paged_kv_cache import FP4Cache, fp4_paged_cache, paged_kv_append_func, paged_kv_read_func
from oracle.packed_attention import paged_attention
from oracle.paged_kv import fp4_decode
from test_gpu_paged_attention_fp4 import make, run

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("d,hk,page", [(64, 2, 16), (64, 2, 100), (128, 1, 16), (128, 1, 100)])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("new,n", [(3, 40), (6, 1003), (9, 5000)])
@pytest.mark.parametrize("scale", [253, 254])
@pytest.mark.parametrize("back", [2, 3, 30])
def test_rows_that_see_them_and_rows_that_do_not(gpu_device, d, hk, page, dtype, new, n, scale, back):
    """One key's 32 values of a large power, of every code. Queries are 0, so that all n weights are 1 and a finite value's
    product stays below 2^128. Bits of what does not see them: as with values of a usual power."""
    args = make([n, 20], new, 4, hk, d, page, dtype, 81)
    q, k, v, table, _ = args
    q.zero_()
    j = max(n - back, 0)
    at = int(table[0, j // page]), j % page
    v[0][at][:, 16:32] = torch.tensor([c + 16 * ((c + 5) % 16) for c in range(16)], dtype=torch.uint8)
    clean, clean_lse = run(args, gpu_device)
    v[1][at][:, 1] = scale
    o, lse = run(args, gpu_device)
    sees = torch.arange(new) + n - new >= j
    assert sees.any()
    assert torch.equal(lse, clean_lse) and torch.equal(o[1], clean[1])
    assert torch.equal(o[0, ~sees], clean[0, ~sees]), "rows that do not see the key"
    assert torch.equal(o[0, :, :, :32], clean[0, :, :, :32]) and torch.equal(o[0, :, :, 64:], clean[0, :, :, 64:])
    big = fp4_decode(*(t[at] for t in v))[:, 32:64]  # [hk, 32]
    inf = big.abs() >= 2.0 ** 128
    assert inf.any() and not inf.all()
    kept = fp4_decode(*v)
    kept[at][:, 32:64] = torch.where(inf, 0.0, big)
    want, _, mag, _ = paged_attention(q, fp4_decode(*k), kept, *args[3:])
    got, want, mag = (t[0, sees][:, :, 32:64].double().cpu() for t in (o, want, mag))
    heads = torch.arange(4) // (4 // hk)
    big, inf = big[heads][None].expand(want.shape), inf[heads][None].expand(want.shape)
    assert torch.equal(got[inf], torch.sign(big[inf]) * math.inf)
    # weights of 1, sums in 32 bits, one rounding (which fp16 may not have a number for)
    want, mag, got = want[~inf], mag[~inf], got[~inf]
    over = want.abs() > torch.finfo(dtype).max
    assert torch.equal(got[over], torch.sign(want[over]) * math.inf)
    lim = 1.01 * torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -17 * mag + 2.0 ** -24
    assert ((got - want).abs() <= lim)[~over].all()


@pytest.mark.parametrize("d,hq,hk,page", [(64, 4, 2, 16), (64, 4, 1, 40), (128, 8, 1, 32), (128, 2, 2, 7)])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("scale", [253, 254])
def test_signs_and_both_signs(gpu_device, d, hq, hk, page, dtype, scale):
    """Usual weights: a row is inf of the sign that it sees, and NaN where it sees both."""
    new, n = 8, 300
    args = make([n], new, hq, hk, d, page, dtype, 82)
    _, _, v, table, _ = args
    for j, code in ((n - 2, 0xFF), (n - 5, 0x77), (n - 40, 0x00)):  # -inf, inf, zeros of a large power
        at = int(table[0, j // page]), j % page
        v[0][at][:, :16] = code
    clean, clean_lse = run(args, gpu_device)
    for j in (n - 2, n - 5, n - 40):
        v[1][int(table[0, j // page]), j % page, :, 0] = scale
    o, lse = run(args, gpu_device)
    assert torch.equal(lse, clean_lse) and torch.equal(o[..., 32:], clean[..., 32:])
    assert torch.equal(o[0, :3], clean[0, :3])
    assert (o[0, 3:6, :, :32] == math.inf).all() and o[0, 6:, :, :32].isnan().all()


def test_a_new_token_of_the_largest_values(gpu_device):
    """As an append writes them: finite bf16 values above 3.5 * 2^126 are kept as 4 * 2^126."""
    dev, n, new = gpu_device, 200, 5
    g = torch.Generator().manual_seed(83)
    k, v = (torch.randn(1, n, 2, 64, generator=g).to(BF).to(dev) for _ in range(2))
    q = torch.randn(1, new, 4, 64, generator=g).to(BF).to(dev)
    table = torch.randperm(13, generator=g).to(torch.int32)[None].to(dev)
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    outs = []
    for value in (1.0, torch.finfo(BF).max):
        v[0, n - 2, :, 7] = value
        cache = [fp4_paged_cache(13, 16, 2, 64, device=dev) for _ in range(2)]
        paged_kv_append_func(k, v, *cache, table, lens)
        outs.append(paged_flash_attn_inference_func(q, *cache, table, lens, return_lse=True))
    at = int(table[0, (n - 2) // 16]), (n - 2) % 16
    assert (cache[1].scales[at][:, 0] == 253).all() and (cache[1].codes[at][:, 3] >> 4 == 6).all()
    (a, lse_a), (b, lse_b) = outs
    assert torch.equal(lse_a, lse_b) and torch.equal(a[0, :3], b[0, :3])
    assert (b[0, 3:, :, 7] == math.inf).all()
    # the other dims of the 32 are kept as zeros beside it
    assert torch.isfinite(b[..., :7]).all() and torch.isfinite(b[..., 8:]).all()
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    rows = paged_kv_read_func(*cache, table, cu, n)[1]
    assert (rows[n - 2, :, 7] == math.inf).all() and torch.isfinite(rows[:n - 2]).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("scale", [1, 64, 126, 140, 141, 252, 253, 254])
def test_values_read_back(gpu_device, dtype, scale):
    """Every code, infinities told apart from the largest finite value."""
    dev = gpu_device
    c = torch.arange(16, dtype=torch.uint8)
    codes = (c[None] + 16 * c[:, None]).view(1, 8, 1, 32)
    scales = torch.full((1, 8, 1, 2), scale, dtype=torch.uint8)
    cache = FP4Cache(codes.to(dev), scales.to(dev))
    rows, _ = paged_kv_read_func(cache, cache, torch.zeros(1, 1, dtype=torch.int32, device=dev),
                                 torch.tensor([0, 8], dtype=torch.int32, device=dev), 8, dtype=dtype)
    want = fp4_decode(codes, scales)[0].to(dtype)
    assert torch.equal(rows.cpu(), want)
    assert want.isinf().any() == (scale >= (253 if dtype == BF else 141))
