"""CPU checks of how a dense layer on streams chooses between the pages of its cache and their keys read back."""
import pytest
import torch

from geoweave_amd import aggregator as agg
from geoweave_amd.custom_flash_attn.paged_kv_cache import fp4_paged_cache

BF, HF = torch.bfloat16, torch.float16


def test_groups_cover_the_sequences_in_order():
    g = torch.Generator().manual_seed(0)
    for _ in range(200):
        lengths = torch.randint(0, 60, (int(torch.randint(0, 12, (1,), generator=g)),), generator=g).tolist()
        limit = int(torch.randint(0, 120, (1,), generator=g))
        groups = agg._groups(lengths, limit)
        assert [i for a, b in groups for i in range(a, b)] == list(range(len(lengths)))
        for i, (a, b) in enumerate(groups):
            assert b > a and (sum(lengths[a:b]) <= limit or b == a + 1)
            # no two could have been taken together
            assert i == 0 or sum(lengths[groups[i - 1][0]:groups[i - 1][1]]) + lengths[a] > limit


@pytest.mark.parametrize("fp4,least,work", [(False, 80, 2.5e9), (True, 300, 4e9)])
def test_borders(fp4, least, work):
    m = agg.DenseAttention(1024, 16, False, None)
    cache = fp4_paged_cache(1, 16, 16, 64) if fp4 else torch.zeros(1, 16, 16, 64, dtype=BF)
    for new in (least - 1, least, least + 1, 400, 1374):
        keys = int(work / 1024 / max(new - least, 1))
        assert not m._reads_back(new, [keys], cache, BF)
        assert not m._reads_back(new, [1, 2], cache, BF)
        assert m._reads_back(new, [keys // 2, keys - keys // 2 + 1], cache, BF) == (new > least)
        assert not m._reads_back(new, [], cache, BF)


def test_fp16_does_not_hold_what_four_bits_keep():
    m = agg.DenseAttention(1024, 16, False, None)
    lengths = [100000] * 4
    assert not m._reads_back(1374, lengths, fp4_paged_cache(1, 16, 16, 64), HF)
    assert m._reads_back(1374, lengths, fp4_paged_cache(1, 16, 16, 64), BF)
    assert m._reads_back(1374, lengths, torch.zeros(1, 16, 16, 64, dtype=HF), HF)
