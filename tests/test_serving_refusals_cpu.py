"""Refusals of the serving-step operators that need no GPU."""

import ctypes

import pytest
import torch

from ultrametric import SharedPrefixCache, build_paged_tables, paged_kv_write, release_paged_requests, ultrametric_prefix_decode
from ultrametric import _native as nat


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


class OnDevice(torch.Tensor):
    """A host tensor that says it lies on a GPU."""

    is_cuda = property(lambda self: True)

    def get_device(self):
        return self.index


def on(index, t):
    t = t.as_subclass(OnDevice)
    t.index = index
    return t


def _calls(a, b):
    """The four operators with their first tensor on GPU a and the others on GPU b."""
    k, c = torch.zeros(5, 2, 8), torch.zeros(3, 2, 4, 8)
    return {
        "build_paged_tables": lambda: build_paged_tables(
            on(a, _i32(3)), on(b, _i32(3)), on(b, _i32(3, 4)), on(b, _i32(9)), on(b, _i32(1)), page_size=4, num_tokens=2),
        "release_paged_requests": lambda: release_paged_requests(
            on(a, torch.zeros(3, dtype=torch.bool)), on(b, _i32(3)), on(b, _i32(3, 4)), on(b, _i32(9)), on(b, _i32(1)),
            page_size=4),
        "paged_kv_write": lambda: paged_kv_write(on(a, k), on(b, k), on(b, torch.zeros(5, dtype=torch.int64)), on(b, c),
                                                 on(b, c)),
        "ultrametric_prefix_decode": lambda: ultrametric_prefix_decode(
            on(a, torch.zeros(2, 4, 8)), on(b, c), on(b, c), on(b, _i32(2)), on(b, _i32(1)), on(b, _i32(2, 3)),
            on(b, _i32(2)), on(b, _i32(3, 4, 2)), on(b, _i32(2, 4, 2)), 1),
    }


@pytest.mark.parametrize("name", list(_calls(0, 0)))
def test_tensors_of_another_device(name, monkeypatch):
    def no_launch(*a):
        raise AssertionError("the library was called")
    monkeypatch.setattr(nat, "lib", no_launch)
    monkeypatch.setattr(nat, "current_device", lambda: 0)
    for a, b in ((0, 1), (1, 0)):
        with pytest.raises(ValueError, match="one device"):
            _calls(a, b)[name]()
    with pytest.raises(ValueError, match="current device"):
        _calls(1, 1)[name]()


def test_prefix_beyond_the_pool():
    cache = SharedPrefixCache(2, 1, 16, 8, 1, 1, 2, 2, 8, device="cpu")
    for n in (33, 100):
        with pytest.raises(ValueError, match="pages"):
            cache.plan_prefix(n)
        assert cache.prefix_tokens == 0
    with pytest.raises(RuntimeError, match="no CPU fallback"):  # fits: only the device is missing
        cache.plan_prefix(32)
    assert cache.prefix_tokens == 0


def test_broadcast_outputs():
    k, c, s = torch.zeros(5, 2, 8), torch.zeros(3, 2, 4, 8), torch.zeros(5, dtype=torch.int64)
    wide = torch.zeros(3, 1, 4, 8).expand(3, 2, 4, 8)
    routes, router = _i32(5, 4, 2), _i32(1, 4, 2).expand(3, 4, 2)
    for args, kw in (((k, k, s, wide, c), {}), ((k, k, s, c, wide), {}),
                     ((k, k, s, c, c), dict(routes=routes, router_indices=router))):
        with pytest.raises(ValueError, match="written in place"):
            paged_kv_write(*args, **kw)
    with pytest.raises(ValueError, match="written in place"):
        build_paged_tables(_i32(3), _i32(3), _i32(1, 4).expand(3, 4), _i32(9), _i32(1), page_size=4, num_tokens=2)
    # a dimension of one may have any stride
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        build_paged_tables(_i32(1), _i32(1), _i32(4).as_strided((1, 4), (0, 1)), _i32(9), _i32(1), page_size=4, num_tokens=2)


def test_decode_workspace_alignment():
    lib = nat.lib()
    st, buf = (ctypes.c_int64 * 4)(1, 1, 1, 1), ctypes.create_string_buffer(4096)
    at = -(-ctypes.addressof(buf) // 256) * 256

    def decode(ws):
        p = at
        return lib.sa_ultrametric_prefix_decode(
            nat.SA_F16, 2, 4, 2, 16, 4, 6, p, st, p, st, p, st, p, 2, 8, None, p, st, 3, p, p, nat.SA_I32, st, p, nat.SA_I32,
            st, 3, 1, 0, 0, p, st, None, ws, 1 << 40, None)
    for off in (1, 4, 16, 128):
        assert decode(at + off) == nat.SA_EINVAL and b"256-byte aligned" in lib.sa_last_error()
