"""Dense layers on streams: new tokens written into paged caches of 16 and 4 bits and attending to all kept ones."""
import pytest
import torch

from geoweave_amd import aggregator as agg
from geoweave_amd.custom_flash_attn.paged_flash_attn import paged_flash_attn_inference_func
from geoweave_amd.custom_flash_attn.paged_kv_cache import fp4_paged_cache, paged_kv_read_func

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _layer(qk_norm=True, rope=100.0, block=False, dim=256, heads=4):
    torch.manual_seed(0)
    m = agg.Block(dim, heads, 2.0, qk_norm, rope, init_values=0.5) if block else agg.DenseAttention(dim, heads, qk_norm, rope)
    return m.cuda().to(BF)


def _pages(b, width, g):
    return torch.randperm(b * width, generator=g).to(torch.int32).view(b, width).cuda()


def _near(got, want, roundings):
    """Two bf16 runs that round at different places: each of ``roundings`` steps by 2^-8 / sqrt(3) of the 2-norm of what it
    rounds, independent in the two."""
    assert torch.isfinite(got).all()
    off = float((got.float() - want.float()).norm() / want.float().norm())
    assert off <= (2 * roundings) ** 0.5 * 2.0 ** -8 / 3 ** 0.5, off


@pytest.mark.parametrize("qk_norm,axes", [(True, (16, 24, 24)), (False, None), (True, None), (False, (32, 32))])
def test_steps_are_the_whole_sequence(gpu_device, qk_norm, axes):
    """A causal layer on a sequence at once, and token by token and in blocks over a cache. Roundings of a run: projection,
    norm, rotation, weights, o, output projection."""
    g = torch.Generator().manual_seed(1)
    m = _layer(qk_norm)
    x = torch.randn(2, 150, 256, generator=g).to(BF).cuda()
    pos = torch.randint(0, 40, (2, 150, len(axes)), generator=g).to(torch.int32).cuda() if axes else None
    table, page = _pages(2, 6, g), 32
    k, v = (torch.zeros(12, page, 4, 64, dtype=BF, device="cuda") for _ in range(2))
    lens, outs = torch.zeros(2, dtype=torch.int32, device="cuda"), []
    for a, b in ((0, 100), (100, 101), (101, 102), (102, 107), (107, 150)):
        lens.fill_(b)
        outs.append(m.forward_cached(x[:, a:b], k, v, table, lens, None if pos is None else pos[:, a:b], axes, causal=True))
    got = torch.cat(outs, 1)
    for i in range(2):
        want = m.forward_train(x[i], None if pos is None else pos[i], None, axes, causal=True)
        _near(got[i], want.detach(), 6)


@pytest.mark.parametrize("new", [3, 300])
@pytest.mark.parametrize("lengths", [False, True])
def test_four_bits(gpu_device, new, lengths):
    """The layer's output is the attention over what the cache holds, and the cache's error its own: normal rows kept in 4
    bits are off by 0.112 of their rms."""
    g = torch.Generator().manual_seed(2)
    m = _layer()
    page, width = 16, 50
    table = _pages(2, width, g)
    cache = [fp4_paged_cache(2 * width, page, 4, 64, device="cuda") for _ in range(2)]
    full = [torch.zeros(2 * width, page, 4, 64, dtype=BF, device="cuda") for _ in range(2)]
    lens = [400, 77]
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for b, length in enumerate(lens):  # earlier tokens, sequence by sequence
        x = torch.randn(1, length, 256, generator=g).to(BF).cuda()
        for c in (cache, full):
            m.forward_cached(x, *c, table[b:b + 1], n[b:b + 1])
    n += new
    lens = [length + new for length in lens]
    x = torch.randn(2, new, 256, generator=g).to(BF).cuda()
    got = m.forward_cached(x, *cache, table, n, lengths=lens if lengths else None)
    m.forward_cached(x, *full, table, n)
    cu = torch.tensor([0, lens[0], sum(lens)], dtype=torch.int32, device="cuda")
    kept, exact = paged_kv_read_func(*cache, table, cu, sum(lens)), paged_kv_read_func(*full, table, cu, sum(lens))
    for a, b in zip(kept, exact):
        off = float((a.float() - b.float()).norm() / b.float().norm())
        assert 0.09 <= off <= 0.13, off  # 0.112 for normal rows; these are nearly
    # the same attention over a 16-bit cache of the kept values, which 16 bits hold exactly
    q = m.q_norm(m.qkv(x).view(2, new, 3, 4, 64)[:, :, 0]).to(BF)
    for c, rows in zip(full, kept):
        for b in range(2):
            at = torch.arange(lens[b], device="cuda")
            c[table[b].long()[at // page], at % page] = rows[int(cu[b]):int(cu[b + 1])]
    o, _ = paged_flash_attn_inference_func(q, *full, table, n, causal=False)
    _near(got, m.proj(o.reshape(2, new, 256)).detach(), 3)  # weights, o, projection


def test_block_and_refusals(gpu_device):
    g = torch.Generator().manual_seed(3)
    m = _layer(block=True)
    x = torch.randn(1, 40, 256, generator=g).to(BF).cuda()
    table = _pages(1, 4, g)
    k, v = (torch.zeros(4, 16, 4, 64, dtype=BF, device="cuda") for _ in range(2))
    n = torch.tensor([40], dtype=torch.int32, device="cuda")
    got = m.forward_cached(x, k, v, table, n)
    want, _ = m(x)
    _near(got, want.detach(), 14)  # a block's roundings: see test_gpu_packed_layers.py
    with pytest.raises(ValueError, match="lengths"):
        m.forward_cached(x, k, v, table, n, lengths=[40, 40])
    sparse = agg.Block(256, 4, 2.0, True, 100.0, sparse=True).cuda().to(BF)
    with pytest.raises(NotImplementedError, match="cache"):
        sparse.forward_cached(x, k, v, table, n)
