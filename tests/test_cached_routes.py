"""CPU checks of how a dense layer on streams chooses between the pages of its cache and their keys read back."""
import pytest
import torch

from geoweave_amd import aggregator as agg
from geoweave_amd.custom_flash_attn.paged_kv_cache import fp4_paged_cache

BF = torch.bfloat16


@pytest.mark.parametrize("fp4,least,work", [(False, 80, 2.5e9), (True, 300, 4e9)])
def test_borders(fp4, least, work):
    m = agg.DenseAttention(1024, 16, False, None)
    cache = fp4_paged_cache(1, 16, 16, 64) if fp4 else torch.zeros(1, 16, 16, 64, dtype=BF)
    for new in (least - 1, least, least + 1, 400, 1374):
        keys = int(work / 1024 / max(new - least, 1))
        assert not m._reads_back(new, [keys], cache)
        assert not m._reads_back(new, [1, 2], cache)
        assert m._reads_back(new, [keys // 2, keys - keys // 2 + 1], cache) == (new > least)
        assert not m._reads_back(new, [], cache)
