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


def test_positions_stay_in_32_bits():
    top = 2 ** 31 - 1

    def build(ctx, new, base):
        bt = torch.full((len(ctx), 4), -7, dtype=torch.int32, device=DEV)
        t = build_paged_tables(_i32(ctx), _i32(new), bt, _i32(list(range(20))), _i32([20]), page_size=16,
                               num_tokens=sum(new), position_base=base)
        assert t.positions.min() >= 0
        return t, nat.read_device_status(reset=True)
    # the last position is the largest that 32 bits hold
    t, status = build([0, 5, 0], [3, 0, 6], top - 5)
    assert status == 0 and t.positions.tolist() == [top - 5 + i for i in (0, 1, 2, 0, 1, 2, 3, 4, 5)]
    assert t.context_lens.tolist() == [3, 5, 6] and t.slot_mapping.ge(0).all()
    # one more is refused, like any request that does not fit; idle requests are not
    t, status = build([0, 5, 0, 16], [3, 0, 7, 0], top - 5)
    assert status == 2 and t.context_lens.tolist() == [3, 5, 0, 16] and t.num_free.tolist() == [19]
    assert t.slot_mapping[:3].ge(0).all() and t.slot_mapping[3:].eq(-1).all()


@pytest.mark.parametrize("T", [40, 3000])
def test_write_takes_routes_across_slots_past_the_cache(T):
    """A row whose slot lies past the cache is skipped, also between the rows of one page."""
    torch.manual_seed(T)
    Hkv, D, page, H, TD = 2, 64, 16, 4, 3
    P = -(-T // page)
    slots = torch.arange(T, device=DEV)
    gone = torch.rand(T, device=DEV) < 0.4
    slots = torch.where(gone, P * page + slots, slots)
    k, v = torch.randn(T, Hkv, D, device=DEV), torch.randn(T, Hkv, D, device=DEV)
    kc, vc = torch.zeros(P, Hkv, page, D, device=DEV), torch.zeros(P, Hkv, page, D, device=DEV)
    routes = torch.randint(0, 1000, (T, H, TD), device=DEV, dtype=torch.int32)
    router = torch.full((P, H, TD), -1, dtype=torch.int32, device=DEV)
    want = [x.cpu().clone() for x in (kc, vc, router)]
    so.write_rows(k.cpu(), v.cpu(), slots.cpu(), want[0], want[1], routes.cpu(), want[2])
    for _ in range(5):
        paged_kv_write(k, v, slots, kc, vc, routes=routes, router_indices=router)
        assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1]) and torch.equal(router.cpu(), want[2])
    assert nat.read_device_status(reset=True) == 2


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
