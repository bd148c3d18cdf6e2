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


def near(got, want, roundings):
    """Two runs that round at different places: each of ``roundings`` steps by eps / 2 / sqrt(3) of the 2-norm of what it rounds,
    independent in the two."""
    assert torch.isfinite(got).all()
    off = float((got.float() - want.float()).norm() / want.float().norm())
    assert off <= (2 * roundings) ** 0.5 * torch.finfo(got.dtype).eps / 2 / 3 ** 0.5, off


@pytest.mark.parametrize("fp4,dtype", [(False, BF), (False, HF), (True, BF)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim,axes", [(256, (16, 24, 24)), (512, None)])
@pytest.mark.parametrize("new,earlier", [(130, (900, 20)), (400, (1100, 0)), (1, (300, 64)), (257, (31, 1000))])
def test_as_over_pages(gpu_device, reads, fp4, dtype, causal, dim, axes, new, earlier):
    """New tokens behind earlier ones of sequences of different lengths. Roundings that differ: the weights', the output's, the
    projection's."""
    g = torch.Generator().manual_seed(1)
    heads = dim // 64
    m = layer(dtype, dim=dim, heads=heads)
    page, width = 32, 50
    table = torch.randperm(2 * width, generator=g).to(torch.int32).view(2, width).cuda()
    cache = caches(fp4, 2 * width, page, heads, 64, dtype)
    turn = lambda b, n: None if axes is None else torch.randint(0, 40, (b, n, 3), generator=g).to(torch.int32).cuda()  # noqa: E731
    n = torch.tensor(earlier, dtype=torch.int32, device="cuda")
    for b, length in enumerate(earlier):
        if length:
            x = torch.randn(1, length, dim, generator=g).to(dtype).cuda()
            m.forward_cached(x, *cache, table[b:b + 1], n[b:b + 1], turn(1, length), axes)
    n += new
    lengths = [length + new for length in earlier]
    x, pos = torch.randn(2, new, dim, generator=g).to(dtype).cuda(), turn(2, new)
    pages = m.forward_cached(x, *cache, table, n, pos, axes, causal=causal)
    assert not reads
    got = m.forward_cached(x, *cache, table, n, pos, axes, causal=causal, lengths=lengths)
    assert reads == [sum(lengths)]
    near(got, pages, 3)
    # every row, not the norm of all alone: a row that saw one key too many or too few would differ by far more
    off = (got.float() - pages.float()).norm(dim=-1) / pages.float().norm(dim=-1)
    assert off.max() <= 8 * torch.finfo(dtype).eps, float(off.max())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("qk_norm,axes", [(True, (16, 24, 24)), (False, None), (False, (32, 32))])
def test_steps_are_the_whole_sequence(gpu_device, reads, dtype, qk_norm, axes):
    """A causal layer on a sequence at once, and in blocks whose keys are read back. Roundings: projection, norm, rotation,
    weights, o, output projection."""
    g = torch.Generator().manual_seed(2)
    m = layer(dtype, qk_norm)
    total = 800
    x = torch.randn(2, total, 256, generator=g).to(dtype).cuda()
    pos = torch.randint(0, 40, (2, total, len(axes)), generator=g).to(torch.int32).cuda() if axes else None
    page = 48
    table = torch.randperm(34, generator=g).to(torch.int32).view(2, 17).cuda()
    k, v = caches(False, 34, page, 4, 64, dtype)
    lens, outs = torch.zeros(2, dtype=torch.int32, device="cuda"), []
    blocks = ((0, 100), (100, 400), (400, 401), (401, 800))
    for a, b in blocks:
        lens.fill_(b)
        outs.append(m.forward_cached(x[:, a:b], k, v, table, lens, None if pos is None else pos[:, a:b], axes, causal=True,
                                     lengths=[b, b]))
    assert reads == [2 * b for _, b in blocks]
    got = torch.cat(outs, 1)
    for i in range(2):
        want = m.forward_train(x[i], None if pos is None else pos[i], None, axes, causal=True)
        near(got[i], want.detach(), 6)


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("limit,want", [(10 ** 9, [1700]), (700, [700, 640, 360]), (400, [300, 400, 360]), (350, [300, 350, 10])])
def test_groups_of_sequences(gpu_device, reads, monkeypatch, fp4, limit, want):
    """What is read back at a time is bounded; a sequence beyond the bound stays on its pages."""
    g = torch.Generator().manual_seed(3)
    m = layer(BF)
    lengths, new, page, width = [300, 400, 640, 350, 10], 10, 16, 40
    table = torch.randperm(5 * width, generator=g).to(torch.int32).view(5, width).cuda()
    cache = caches(fp4, 5 * width, page, 4, 64, BF)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for b, length in enumerate(lengths):
        x = torch.randn(1, length, 256, generator=g).to(BF).cuda()
        m.forward_cached(x, *cache, table[b:b + 1], n[b:b + 1])
    x = torch.randn(5, new, 256, generator=g).to(BF).cuda()
    pages = m.forward_cached(x, *cache, table, n)
    monkeypatch.setattr(agg.DenseAttention, "READ_BACK_BYTES", limit * 4 * 256)
    got = m.forward_cached(x, *cache, table, n, lengths=lengths)
    assert reads == want
    near(got, pages, 3)


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


@pytest.mark.parametrize("limit", [10 ** 9, 400, 0])
def test_sequences_of_no_keys(gpu_device, reads, monkeypatch, limit):
    """Beside others, in a group of their own, and behind one that stays on its pages."""
    g = torch.Generator().manual_seed(4)
    m = layer(BF)
    lengths = [0, 640, 0, 0, 30]
    table = torch.randperm(200, generator=g).to(torch.int32).view(5, 40).cuda()
    cache = caches(False, 200, 16, 4, 64, BF)
    for c in cache:
        c.copy_(torch.randn(c.shape, generator=g))
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    x = torch.randn(5, 10, 256, generator=g).to(BF).cuda()
    pages = m.forward_cached(x, *cache, table, n)
    monkeypatch.setattr(agg.DenseAttention, "READ_BACK_BYTES", limit * 4 * 256)
    got = m.forward_cached(x, *cache, table, n, lengths=lengths)
    assert sum(reads) == {10 ** 9: 670, 400: 30, 0: 0}[limit]
    near(got, pages, 3)
    assert torch.equal(got[[0, 2, 3]], m.proj.bias.detach().expand(3, 10, 256))
