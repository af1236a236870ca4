"""GPU checks of the serving-step operators at the edges of their arguments."""

import pytest
import torch

from oracle import serving_oracle as so
from ultrametric import SharedPrefixCache, build_paged_tables, paged_kv_write
from ultrametric import _native as nat

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def test_prefix_is_set_before_any_request():
    cache = SharedPrefixCache(8, 1, 16, 64, 1, 1, 2, 4, 4, device=DEV)
    cache.plan(_i32([3, 0]), 3)
    with pytest.raises(ValueError, match="before any request"):
        cache.plan_prefix(20)
    assert cache.prefix_tokens == 0 and int(cache.prefix_len) == 0 and int(cache.num_free) == 7
    t = cache.plan(_i32([1, 2]), 3)
    assert t.positions.tolist() == [3, 0, 1]
    assert nat.read_device_status(reset=True) == 0


def test_a_prefix_that_fills_the_pool():
    cache = SharedPrefixCache(3, 1, 16, 64, 1, 1, 2, 4, 9, device=DEV)
    with pytest.raises(ValueError, match="pages"):
        cache.plan_prefix(49)
    t = cache.plan_prefix(48)  # the refusal left the cache as it was
    assert t.slot_mapping.ge(0).all() and int(cache.prefix_len) == 48 and int(cache.num_free) == 0
    assert nat.read_device_status(reset=True) == 0
