"""Dense layers on streams whose kept keys are read back as packed rows: the same results as over the pages and as of whole
sequences, in every order, type and grouping."""
import pytest
import torch

from geoweave_amd import aggregator as agg
from geoweave_amd.custom_flash_attn.paged_kv_cache import fp4_paged_cache

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture
def reads(monkeypatch):
    """Attention always takes the keys read back where lengths are given; the rows of each reading."""
    monkeypatch.setattr(agg.DenseAttention, "READ_BACK_FROM", ((-1, 0), (-1, 0)))
    rows, read = [], agg.paged_kv_read_func
    monkeypatch.setattr(agg, "paged_kv_read_func", lambda *a, **kw: rows.append(a[4]) or read(*a, **kw))
    return rows


def layer(dtype, qk_norm=True, rope=100.0, dim=256, heads=4):
    torch.manual_seed(0)
    return agg.DenseAttention(dim, heads, qk_norm, rope).cuda().to(dtype)


def caches(fp4, pages, page, heads, d, dtype):
    if fp4:
        return [fp4_paged_cache(pages, page, heads, d, device="cuda") for _ in range(2)]
    return [torch.zeros(pages, page, heads, d, dtype=dtype, device="cuda") for _ in range(2)]


def test_fp16_over_four_bits_stays_on_its_pages(gpu_device, reads):
    """Values near fp16's largest, kept as 65,536, of both signs: their mean is a number of fp16."""
    m = layer(HF, qk_norm=False)
    for p in m.parameters():
        torch.nn.init.zeros_(p)
    with torch.no_grad():
        m.qkv.weight[512:, 0] = torch.finfo(HF).max
        m.proj.weight.copy_(torch.eye(256))
    x = torch.zeros(1, 320, 256, dtype=HF, device="cuda")
    x[0, :, 0] = torch.tensor([1.0, -1.0, 1.0, -1.0, -1.0]).repeat(64)
    cache = caches(True, 20, 16, 4, 64, HF)
    table, n = torch.arange(20, dtype=torch.int32, device="cuda")[None], torch.tensor([320], dtype=torch.int32, device="cuda")
    got = m.forward_cached(x, *cache, table, n, lengths=[320])
    assert not reads
    # 64 more of one sign, of 320: -65,536 / 5, rounded once to fp16
    assert torch.equal(got, torch.full_like(got, -65536.0 / 5))
