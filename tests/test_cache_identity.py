"""What the native steps and the captured graphs keep of a cache has to change with the
cache, on the CPU: addresses alone do not tell two caches apart, since a smaller pool may
be carved from the start of a freed one."""

import pytest
import torch

from mu_b200.core.cache import PagedKVCache
from mu_b200.core.config import MuConfig
from mu_b200.models.base import MuModelBase

FP8 = torch.float8_e4m3fn
KINDS = [torch.bfloat16, FP8]


def _cache(blocks, dtype, bs=16, heads=2, d=64, layers=2):
    return PagedKVCache(layers, heads, d, bs, blocks, dtype, "cpu", MuConfig(enabled=False))


def _at(cache, other):
    """`cache` moved to the start of `other`'s memory."""
    for name in ("block_pool", "scales"):
        t, o = getattr(cache, name), getattr(other, name)
        if t is not None:
            setattr(cache, name, o.view(-1)[: t.numel()].view(t.shape))
    return cache


@pytest.mark.parametrize("dtype", KINDS)
def test_key_tells_pools_at_one_address_apart(dtype):
    a = _cache(12, dtype)
    key = MuModelBase.cache_key(a)
    assert key == MuModelBase.cache_key(_at(_cache(12, dtype), a))
    for other in (_cache(8, dtype), _cache(8, dtype, bs=8)):
        b = _at(other, a)
        assert b.block_pool.data_ptr() == a.block_pool.data_ptr()
        assert MuModelBase.cache_key(b) != key
