"""GPU checks of the serving step end to end: ``SharedPrefixCache`` over admissions, decode steps
and releases against plain-integer bookkeeping and the 64-bit decode oracle (bounds of
``test_prefix_decode_gpu.py``), eagerly and replayed from a CUDA graph."""

import pytest
import torch

from oracle import serving_oracle as so
from ultrametric import SharedPrefixCache
from ultrametric import _native as nat

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _check(cache, layer, q, qri, out, depth, dense):
    """dense: per request the (k, v, route of page) it should hold."""
    ref, _, w = so.prefix_decode(q.cpu(), cache.k_cache[layer].cpu(), cache.v_cache[layer].cpu(), cache.prefix_table[0].cpu(),
                                 int(cache.prefix_len), cache.block_tables.cpu(), cache.context_lens.cpu(),
                                 cache.router[layer].cpu(), qri.cpu(), depth, 1, True)
    vmax = float(cache.v_cache.abs().max())
    over = (out.double().cpu() - ref).abs() - 2.0 ** -8 * (w + ref.abs()) - 1e-5 * vmax
    assert over.max() <= 0
    page = cache.page_size
    for b, (k, v) in dense.items():
        n = int(cache.context_lens[b])
        assert n == k.shape[0]
        rows = torch.arange(n)
        ids = cache.block_tables[b].cpu().long()[rows // page]
        assert torch.equal(cache.k_cache[layer].cpu()[ids, :, rows % page], k)
        assert torch.equal(cache.v_cache[layer].cpu()[ids, :, rows % page], v)


@pytest.mark.parametrize("H,Hkv,D,page", [(8, 2, 128, 64), (6, 3, 64, 16), (4, 4, 80, 8)])
def test_serving_loop(H, Hkv, D, page):
    g = torch.Generator().manual_seed(H * D)
    TD, R, layers, n = 3, 5, 2, 3 * page + 5
    cache = SharedPrefixCache(60, Hkv, page, D, H, TD, R, 9, 6, num_layers=layers, device=DEV)
    dense = [{b: (torch.zeros(0, Hkv, D).bfloat16(), torch.zeros(0, Hkv, D).bfloat16()) for b in range(R)}
             for _ in range(layers)]

    def rows(T):
        return (torch.randn(T, Hkv, D, generator=g).bfloat16(), torch.randn(T, Hkv, D, generator=g).bfloat16(),
                torch.randint(0, 2, (T, H, TD), generator=g, dtype=torch.int32))

    t = cache.plan_prefix(n)
    assert t.positions.tolist() == list(range(n))
    for layer in range(layers):
        k, v, r = rows(n)
        cache.write(layer, k.to(DEV), v.to(DEV), t, r.to(DEV))
    steps = [[17, 0, page, 2 * page + 3, 1], [1] * R, [1, 1, 1, 0, 0], [0, 40, 0, 0, 7], [1] * R]
    finish = {2: [False, False, True, True, False]}
    for i, new in enumerate(steps):
        T = sum(new)
        t = cache.plan(torch.tensor(new, dtype=torch.int32, device=DEV), T + 3)
        assert t.slot_mapping[T:].tolist() == [-1] * 3
        for layer in range(layers):
            k, v, r = rows(T + 3)
            cache.write(layer, k.to(DEV), v.to(DEV), t, r.to(DEV))
            at = 0
            for b in range(R):
                d = dense[layer][b]
                dense[layer][b] = (torch.cat([d[0], k[at:at + new[b]]]), torch.cat([d[1], v[at:at + new[b]]]))
                at += new[b]
            q = torch.randn(R, H, D, generator=g).bfloat16().to(DEV)
            qri = torch.randint(0, 2, (R, H, TD), generator=g, dtype=torch.int32).to(DEV)
            for depth in (0, 1):
                _check(cache, layer, q, qri, cache.decode(layer, q, qri, depth), depth, dense[layer])
        if i in finish:
            cache.finish(torch.tensor(finish[i], device=DEV))
            for layer in range(layers):
                for b, f in enumerate(finish[i]):
                    if f:
                        dense[layer][b] = tuple(x[:0] for x in dense[layer][b])
    # every page is in exactly one place
    used = cache.prefix_table[0, :-(-n // page)].tolist()
    for b in range(R):
        used += cache.block_tables[b, :-(-int(cache.context_lens[b]) // page)].tolist()
    free = cache.free_pages[:int(cache.num_free)].tolist()
    assert sorted(used + free) == list(range(60))
    assert nat.read_device_status(reset=True) == 0


def test_decode_step_replays_in_a_graph():
    g = torch.Generator().manual_seed(2)
    H, Hkv, D, page, TD, R, n = 8, 2, 128, 16, 2, 4, 100
    cache = SharedPrefixCache(80, Hkv, page, D, H, TD, R, 8, 8, device=DEV)
    t = cache.plan_prefix(n)
    kv = torch.randn(2, n, Hkv, D, generator=g).bfloat16().to(DEV)
    cache.write(0, kv[0], kv[1], t, torch.randint(0, 2, (n, H, TD), generator=g, dtype=torch.int32).to(DEV))
    k, v = torch.zeros(R, Hkv, D, dtype=torch.bfloat16, device=DEV), torch.zeros(R, Hkv, D, dtype=torch.bfloat16, device=DEV)
    q, ones = torch.zeros(R, H, D, dtype=torch.bfloat16, device=DEV), torch.ones(R, dtype=torch.int32, device=DEV)
    r, qri = (torch.zeros(R, H, TD, dtype=torch.int32, device=DEV) for _ in range(2))

    def step():
        tables = cache.plan(ones, R)
        cache.write(0, k, v, tables, r)
        return cache.decode(0, q, qri, 1)
    dense = {b: (torch.zeros(0, Hkv, D).bfloat16(), torch.zeros(0, Hkv, D).bfloat16()) for b in range(R)}

    def feed():
        for x, hi in ((r, 2), (qri, 2)):
            x.copy_(torch.randint(0, hi, x.shape, generator=g, dtype=torch.int32))
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, generator=g).bfloat16())
        for b in range(R):
            dense[b] = (torch.cat([dense[b][0], k[b:b + 1].cpu()]), torch.cat([dense[b][1], v[b:b + 1].cpu()]))
    feed()
    out = step()  # once outside: modules load before the capture
    _check(cache, 0, q, qri, out, 1, dense)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(2 * page):
        feed()
        graph.replay()
        if i % 7 == 0:
            torch.cuda.synchronize()
            _check(cache, 0, q, qri, out, 1, dense)
    assert cache.context_lens.tolist() == [2 * page + 1] * R
    assert nat.read_device_status(reset=True) == 0


def test_refusals():
    cache = SharedPrefixCache(8, 1, 16, 64, 1, 1, 2, 2, 2, device=DEV)
    with pytest.raises(ValueError, match="does not fit"):
        cache.plan_prefix(33)
    cache.plan_prefix(20)
    with pytest.raises(ValueError, match="already holds"):
        cache.plan_prefix(5)
    # more tokens than pages: refused on the device, the cache stays as it was
    t = cache.plan(torch.tensor([33, 10], dtype=torch.int32, device=DEV), 43)
    assert t.slot_mapping[:33].eq(-1).all() and t.slot_mapping[33:].ge(0).all()
    assert cache.context_lens.tolist() == [0, 10]
    assert nat.read_device_status(reset=True) == 2
