"""GPU checks of the step's tables, releases and ragged writes: every integer and every copied byte
equals the plain-integer / row-by-row oracle's."""

import random

import pytest
import torch

from oracle import serving_oracle as so
from ultrametric import _native as nat
from ultrametric import build_paged_tables, paged_kv_write, release_paged_requests

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _state(rng, B, page, ctx_hi, L, spare, zero=0.2):
    ctx = [0 if rng.random() < zero else rng.randint(0, ctx_hi) for _ in range(B)]
    have = [-(-c // page) for c in ctx]
    total = sum(have) + spare
    ids = list(range(total))
    rng.shuffle(ids)
    table = [[-7] * L for _ in range(B)]
    at = 0
    for b in range(B):
        table[b][:have[b]] = ids[at:at + have[b]]
        at += have[b]
    return ctx, table, ids[at:]


def _check(ctx, new, table, free, page, rows, base=0, num_free=None, status=None, bt=None):
    nf = len(free) if num_free is None else num_free
    bt = _i32(table) if bt is None else bt
    want = [list(r) for r in table]
    slots, rids, pos, cu, ctx_out, nf_out, refused = so.build_tables(ctx, new, want, free, nf, page, rows, base)
    before = (_i32(ctx), _i32(new), _i32(free), _i32([nf]))
    for _ in range(2):  # a call leaves its inputs but the new entries, so it can be repeated
        got = build_paged_tables(before[0], before[1], bt, before[2], before[3], page_size=page, num_tokens=rows,
                                 position_base=base)
    assert got.slot_mapping.tolist() == slots
    assert got.request_ids.tolist() == rids
    assert got.positions.tolist() == pos
    assert got.cu_new_lens.tolist() == cu
    assert got.context_lens.tolist() == ctx_out
    assert got.num_free.tolist() == [nf_out]
    assert bt.tolist() == want
    assert before[2].tolist() == free and before[0].tolist() == ctx
    expect = (2 if refused else 0) if status is None else status
    assert nat.read_device_status(reset=True) == expect
    return got


@pytest.mark.parametrize("B,page,ctx_hi,new_hi,pad", [
    (1, 16, 0, 1, 0), (1, 64, 100, 300, 5), (7, 1, 9, 4, 3), (64, 64, 4000, 1, 0), (33, 24, 500, 90, 7),
    (256, 16, 300, 40, 1), (257, 128, 1000, 3, 0), (700, 32, 200, 9, 2), (5, 16, 70, 9000, 0)])
def test_tables_match_plain_integers(B, page, ctx_hi, new_hi, pad):
    rng = random.Random(B * 31 + page)
    L = -(-(ctx_hi + new_hi) // page)
    new = [0 if rng.random() < 0.3 else rng.randint(0, new_hi) for _ in range(B)]
    ctx, table, free = _state(rng, B, page, ctx_hi, L, spare=sum(-(-n // page) + 1 for n in new))
    _check(ctx, new, table, free, page, sum(new) + pad, base=rng.choice([0, 11]))


def test_more_requests_than_one_block_of_shared_memory():
    rng = random.Random(5)
    B = 9000
    new = [rng.randint(0, 2) for _ in range(B)]
    ctx, table, free = _state(rng, B, 16, 40, 4, spare=B)
    _check(ctx, new, table, free, 16, sum(new))


def test_no_requests_and_no_tokens():
    t = build_paged_tables(_i32([]), _i32([]), _i32([]).view(0, 4), _i32([3, 4]), _i32([2]), page_size=16, num_tokens=5)
    assert t.slot_mapping.tolist() == [-1] * 5 and t.request_ids.tolist() == [-1] * 5
    assert t.cu_new_lens.tolist() == [0] and t.num_free.tolist() == [2]
    _check([5, 0], [0, 0], [[9], [-7]], [1], 16, 0)


def test_refused_requests_change_nothing():
    # out of pages at request 1: it and the later ones that need pages are refused, request 3 needs none
    _check([0, 10, 0, 3, 0], [16, 40, 5, 4, 0], [[-7] * 8 for _ in range(1)] + [[4] + [-7] * 7, [-7] * 8, [5] + [-7] * 7, [-7] * 8],
           [0, 1, 2], 16, 65)
    # more pages than the table holds; negative lengths; rows past num_tokens
    _check([30, 0], [3, 4], [[7, 8], [-7, -7]], [0, 1, 2], 16, 7)
    _check([-1, 4, 0], [3, -2, 6], [[-7], [3], [-7]], [0, 1], 16, 20)
    _check([0, 0, 0], [4, 4, 4], [[-7], [-7], [-7]], [0, 1, 2], 16, 9)
    # a height past the stack's capacity is cut to it
    _check([0], [4], [[-7]], [6, 5], 16, 4, num_free=9, status=2)


def test_strided_table_and_other_stream():
    rng = random.Random(8)
    ctx, table, free = _state(rng, 20, 16, 100, 9, spare=60)
    wide = torch.full((20, 30), -7, dtype=torch.int32, device=DEV)
    bt = wide[:, 3:30:3]
    bt.copy_(_i32(table))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _check(ctx, [7] * 20, table, free, 16, 140, bt=bt)


@pytest.mark.parametrize("B", [1, 40, 300])
def test_release_then_build(B):
    rng = random.Random(B)
    page, L = 16, 12
    ctx, table, free = _state(rng, B, page, 150, L, spare=30)
    finished = [rng.random() < 0.4 for _ in range(B)]
    cap = len(free) + sum(-(-c // page) for c in ctx)
    stack = free + [-1] * (cap - len(free))
    want = list(stack)
    ctx_w, top = so.release(finished, ctx, table, want, len(free), page)
    fp = _i32(stack)
    c2, nf = release_paged_requests(torch.tensor(finished, device=DEV), _i32(ctx), _i32(table), fp, _i32([len(free)]),
                                    page_size=page)
    assert c2.tolist() == ctx_w and nf.tolist() == [top] and fp.tolist() == want
    assert nat.read_device_status(reset=True) == 0
    new = [rng.randint(0, 20) for _ in range(B)]
    _check(ctx_w, new, table, want, page, sum(new), num_free=top, status=None)


def test_release_past_the_stack_keeps_the_pages():
    fp = _i32([9, -1])
    c, nf = release_paged_requests(torch.tensor([True, True, True], device=DEV), _i32([16, 20, 0]),
                                   _i32([[1, 0], [2, 3], [0, 0]]), fp, _i32([1]), page_size=16)
    assert c.tolist() == [0, 20, 0] and nf.tolist() == [2] and fp.tolist() == [9, 1]
    assert nat.read_device_status(reset=True) == 2


def _randn(shape, dtype):
    return torch.randn(*shape, device=DEV).to(dtype)


@pytest.mark.parametrize("T,Hkv,D,page,dtype,idt", [
    (1, 1, 8, 1, torch.float16, torch.int32), (5, 8, 128, 64, torch.bfloat16, torch.int32),
    (333, 3, 80, 16, torch.float32, torch.int64), (200, 2, 20, 24, torch.float16, torch.int32),
    (77, 5, 7, 16, torch.bfloat16, torch.int64), (1000, 8, 64, 32, torch.bfloat16, None), (3, 1, 1, 4, torch.float32, None)])
@pytest.mark.parametrize("packed", [False, True])
def test_write_matches_rows(T, Hkv, D, page, dtype, idt, packed):
    torch.manual_seed(T)
    P, H, TD = -(-T // page) + 9, Hkv * 2, 3
    perm = torch.randperm(P * page, device=DEV)[:T]
    slots = perm.sort().values if T % 2 else perm  # runs, or rows anywhere
    slots = slots.clone()
    if T > 4:
        slots[1], slots[T - 1] = -1, -1
    kv = _randn((T, 2 * Hkv, D), dtype)
    k, v = (kv[:, :Hkv], kv[:, Hkv:]) if packed else (kv[:, :Hkv].contiguous(), kv[:, Hkv:].contiguous())
    kc, vc = _randn((P, Hkv, page, D), dtype), _randn((P, Hkv, page, D), dtype)
    if packed:  # a cache laid out token-major
        kc = kc.transpose(1, 2).contiguous().transpose(1, 2)
    routes = router = None
    if idt is not None and T % 2:
        routes = torch.randint(0, 9, (T, H, TD), device=DEV).to(idt)
        router = torch.full((P, H, TD), -1, dtype=torch.int64 if idt == torch.int32 else torch.int32, device=DEV)
    want = [x.cpu().clone() if x is not None else None for x in (kc, vc, router)]
    so.write_rows(k.cpu(), v.cpu(), slots.cpu(), want[0], want[1], None if routes is None else routes.cpu(), want[2])
    paged_kv_write(k, v, slots, kc, vc, routes=routes, router_indices=router)
    assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])
    assert router is None or torch.equal(router.cpu(), want[2])
    assert nat.read_device_status(reset=True) == 0


def test_write_skips_slots_past_the_cache():
    k = torch.ones(3, 1, 8, device=DEV)
    kc, vc = torch.zeros(2, 1, 4, 8, device=DEV), torch.zeros(2, 1, 4, 8, device=DEV)
    paged_kv_write(k, k, torch.tensor([8, 7, 1 << 40], device=DEV), kc, vc)
    assert kc[1, 0, 3].eq(1).all() and kc.sum() == 8 and vc.sum() == 8
    assert nat.read_device_status(reset=True) == 2
    paged_kv_write(k[:0], k[:0], torch.zeros(0, dtype=torch.int64, device=DEV), kc, vc)


def test_write_past_32_bit_offsets():
    page, Hkv, D = 64, 8, 128
    P = 2 ** 32 // (page * Hkv * D * 2) + 40  # the last rows lie past 2^32 bytes and 2^31 elements
    kc = torch.empty(P, Hkv, page, D, dtype=torch.bfloat16, device=DEV)
    k = torch.randn(2, Hkv, D, device=DEV).bfloat16()
    slots = torch.tensor([P * page - 1, (P - 9) * page + 3], device=DEV)
    paged_kv_write(k, k, slots, kc, kc)
    assert torch.equal(kc[P - 1, :, page - 1], k[0]) and torch.equal(kc[P - 9, :, 3], k[1])
    assert nat.read_device_status(reset=True) == 0


@pytest.mark.parametrize("T,live,Hkv,D,dtype", [(5000, 4700, 1, 64, torch.bfloat16), (9000, 40, 2, 80, torch.float32),
                                                (2400, 2399, 3, 20, torch.float16), (700, 1, 1, 8, torch.float32)])
def test_write_small_rows_with_gaps_and_padding(T, live, Hkv, D, dtype):
    torch.manual_seed(T)
    page, H, TD = 16, 4, 2
    P = -(-T // page) + 3
    slots = torch.randperm((P - 1) * page, device=DEV)[:T].sort().values
    slots[torch.rand(T, device=DEV) < 0.2] = -1
    slots[live - 1] = slots.max() + 1
    slots[live:] = -1
    k, v = _randn((T, Hkv, D), dtype), _randn((T, Hkv, D), dtype)
    kc, vc = torch.zeros(P, Hkv, page, D, dtype=dtype, device=DEV), torch.zeros(P, Hkv, page, D, dtype=dtype, device=DEV)
    routes = torch.randint(0, 9, (T, H, TD), device=DEV, dtype=torch.int32)
    router = torch.full((P, H, TD), -1, dtype=torch.int32, device=DEV)
    want = [x.cpu().clone() for x in (kc, vc, router)]
    so.write_rows(k.cpu(), v.cpu(), slots.cpu(), want[0], want[1], routes.cpu(), want[2])
    paged_kv_write(k, v, slots, kc, vc, routes=routes, router_indices=router)
    assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1]) and torch.equal(router.cpu(), want[2])
    assert nat.read_device_status(reset=True) == 0
