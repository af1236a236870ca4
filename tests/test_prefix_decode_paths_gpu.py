"""Which kernels a shared-prefix decode runs on: the width of the tables, which is a capacity, does not
move a 16-bit batch off the tensor cores until the sizes that the kernel counts in 32 bits are reached;
past them the CUDA-core path gives the same result.  Kernel names are read from the torch profiler."""

import pytest
import torch
from torch.profiler import ProfilerActivity, profile

from test_prefix_decode_gpu import call, check, make

pytestmark = pytest.mark.gpu


def run(t, n, depth, local=0, sink=False):
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as prof:
        got = call(t, n, depth, local, sink)
        torch.cuda.synchronize()
    names = [e.name for e in prof.events() if e.device_type == torch.autograd.DeviceType.CUDA]
    tensor, general = (any(k in x for x in names) for k in ("prefix_sm100_kernel", "prefix_split_kernel"))
    assert tensor != general, names
    return got, tensor


def widen(t, key, width):
    x = t[key]
    wide = torch.full((*x.shape[:-1], width), 10 ** 8, dtype=torch.int32)  # past the lengths: not read
    wide[..., :x.shape[-1]] = x
    t[key] = wide


@pytest.mark.parametrize("depth", [0, 1])
@pytest.mark.parametrize("key,width", [("bt", 8192), ("pp", 9000)])
def test_wide_tables_stay_on_the_tensor_cores(key, width, depth):
    """256 requests, 8 KV heads, pages of 16: tables for 131072 tokens, lists for a prefix of 144000."""
    t, n = make(256, 8, 8, 64, 16, 100, [13 * i % 70 for i in range(256)], seed=depth)
    widen(t, key, width)
    got, tensor = run(t, n, depth, 1, True)
    assert tensor
    check(t, n, depth, 1, True, got=got)


@pytest.mark.parametrize("depth", [0, 2])
@pytest.mark.parametrize("width,fast", [(10000, True), (32767, False)])
def test_both_sides_of_the_limit(width, fast, depth):
    """Pages of 65536 rows; 32767 of them are 512 x 32767 key tiles for each of 16 (request, KV head)
    pairs, 4.0e9 when weighted: past 2^31."""
    t, n = make(2, 8, 8, 8, 65536, 70, [65600, 300], seed=3)
    widen(t, "bt", width)
    got, tensor = run(t, n, depth, 1, False)
    assert tensor == fast
    check(t, n, depth, 1, False, got=got)


def test_a_cache_without_pages():
    t, _ = make(3, 4, 2, 64, 16, 0, [0, 0, 0], seed=1)
    for key in ("kc", "vc", "ri"):
        t[key] = t[key][:0].contiguous()
    for depth in (0, 1):
        out, lse = call(t, 0, depth, 1, True)
        assert (out == 0).all() and torch.isneginf(lse).all()
