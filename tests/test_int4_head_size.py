"""Head sizes that the operators over a cache in 4 bits do not take are refused before anything is allocated."""

import pytest
import torch

from pagedserve_amd.cache.manager import CacheGroupSpec, CacheManager


def _manager(head_dim):
    return CacheManager([CacheGroupSpec((0,), 1, head_dim)], 2, 8, 1, torch.bfloat16, "cpu", cache_format="int4")


def test_heads_of_more_than_256_dimensions():
    assert _manager(256).key_pools[0].shape == (1, 2, 1, 8, 144)
    with pytest.raises(ValueError, match="up to 256 dimensions, not 320"):
        _manager(320)
