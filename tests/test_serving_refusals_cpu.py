"""Refusals of the serving-step operators that need no GPU."""

import ctypes

import pytest
import torch

from ultrametric import SharedPrefixCache, build_paged_tables, paged_kv_write, release_paged_requests, ultrametric_prefix_decode
from ultrametric import _native as nat


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_prefix_beyond_the_pool():
    cache = SharedPrefixCache(2, 1, 16, 8, 1, 1, 2, 2, 8, device="cpu")
    for n in (33, 100):
        with pytest.raises(ValueError, match="pages"):
            cache.plan_prefix(n)
        assert cache.prefix_tokens == 0
    with pytest.raises(RuntimeError, match="no CPU fallback"):  # fits: only the device is missing
        cache.plan_prefix(32)
    assert cache.prefix_tokens == 0
