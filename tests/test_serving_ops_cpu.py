"""Refusals of the serving-step operators and CPU checks of their oracle (no GPU, no launch)."""

import ctypes

import pytest
import torch

from oracle import decode_oracle as dor
from oracle import serving_oracle as so
from ultrametric import _native as nat
from ultrametric import build_paged_tables, paged_kv_write, release_paged_requests, ultrametric_prefix_decode


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_tables_refusals():
    ok = (_i32(3), _i32(3), _i32(3, 4), _i32(9), _i32(1))

    def call(i=None, bad=None, page_size=16, num_tokens=4, position_base=0):
        a = list(ok)
        if i is not None:
            a[i] = bad
        return build_paged_tables(*a, page_size=page_size, num_tokens=num_tokens, position_base=position_base)
    for i, bad in [(0, _i32(3, 1)), (0, torch.zeros(3, dtype=torch.int64)), (1, _i32(2)), (2, _i32(2, 4)), (2, _i32(3)),
                   (3, torch.zeros(9)), (3, _i32(18)[::2]), (4, _i32(2))]:
        with pytest.raises(ValueError):
            call(i, bad)
    for kw in (dict(page_size=0), dict(num_tokens=-1), dict(position_base=-1)):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        call()
    with pytest.raises(ValueError, match="finished"):
        release_paged_requests(_i32(3), *(ok[i] for i in (0, 2, 3, 4)), page_size=16)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        release_paged_requests(torch.zeros(3, dtype=torch.bool), *(ok[i] for i in (0, 2, 3, 4)), page_size=16)


def test_write_refusals():
    k, c, s = torch.zeros(5, 2, 8), torch.zeros(3, 2, 4, 8), torch.zeros(5, dtype=torch.int64)
    for a, kw, msg in [
        ((k[0], k[0], s, c, c), {}, "must be"), ((k, k[:4], s, c, c), {}, "must be"),
        ((k, k, s, c[..., :4], c[..., :4]), {}, "k_cache"), ((k, k, s, c, c[:2]), {}, "k_cache"),
        ((k.half(), k, s, c, c), {}, "dtype"), ((k, k, s.int(), c, c), {}, "slot_mapping"),
        ((k, k, s[:3], c, c), {}, "slot_mapping"), ((k, k, s, c, c), dict(routes=_i32(5, 4, 2)), "go together"),
        ((k, k, s, c, c), dict(routes=_i32(5, 4, 2), router_indices=_i32(3, 4, 3)), "routes must be"),
        ((k, k, s, c.transpose(2, 3).contiguous().transpose(2, 3), c), {}, "contiguous"),
    ]:
        with pytest.raises(ValueError, match=msg):
            paged_kv_write(*a, **kw)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged_kv_write(k, k, s, c, c)


def test_prefix_decode_refusals():
    q, c = torch.zeros(2, 4, 16), torch.zeros(6, 2, 4, 16)
    base = dict(q=q, k_cache=c, v_cache=c, prefix_pages=_i32(2), prefix_len=7, block_tables=_i32(2, 3),
                context_lens=_i32(2), router_indices=_i32(6, 4, 3), q_router_indices=_i32(2, 4, 3), req_depth=1)
    for kw, msg in [
        (dict(q=q[0]), "q must be"), (dict(k_cache=c[0]), "k_cache"), (dict(k_cache=c[:, :1]), "k_cache"),
        (dict(q=torch.zeros(2, 3, 16)), "heads"), (dict(q=q.half()), "dtype"), (dict(prefix_pages=_i32(2, 1)), "prefix_pages"),
        (dict(block_tables=_i32(3, 3)), "block_tables"), (dict(context_lens=_i32(3)), "context_lens"),
        (dict(router_indices=_i32(5, 4, 3)), "router_indices"), (dict(q_router_indices=_i32(2, 4, 2)), "router_indices"),
        (dict(req_depth=4), "req_depth"), (dict(req_depth=-1), "req_depth"), (dict(local_blocks=-1), "local_blocks"),
        (dict(prefix_len=9), "prefix_len"), (dict(prefix_len=-1), "prefix_len"),
        (dict(prefix_len=torch.tensor([1.0])), "prefix_len"),
    ]:
        with pytest.raises(ValueError, match=msg):
            ultrametric_prefix_decode(**dict(base, **kw))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ultrametric_prefix_decode(**base)


def test_library_refusals_without_launch():
    lib = nat.lib()
    st = (ctypes.c_int64 * 4)(1, 1, 1, 1)
    assert lib.sa_paged_build_tables(-1, 1, 1, 0, *[None] * 3, st, None, 0, None, 0, *[None] * 7) == nat.SA_EINVAL
    assert lib.sa_paged_build_tables(2, 1, 1, 0, *[None] * 3, st, None, 0, None, 0, *[None] * 7) == nat.SA_EINVAL
    assert b"null" in lib.sa_last_error()
    assert lib.sa_paged_build_tables(1 << 20, 1, 1, 0, *[None] * 3, st, None, 0, None, 0, *[None] * 7) == nat.SA_EUNSUPPORTED
    assert lib.sa_paged_release(1, 1, 0, *[None] * 3, st, None, 0, *[None] * 4) == nat.SA_EINVAL

    def write(dtype=nat.SA_F16, T=1, Hkv=1, D=8, page=4, ptr=None):
        return lib.sa_paged_kv_write(dtype, T, Hkv, D, page, 2, ptr, st, ptr, st, ptr, ptr, st, ptr, st, None, 0, None, 0,
                                     0, None, 0, None, None)
    assert write(D=0) == nat.SA_EINVAL and write(page=0) == nat.SA_EINVAL and write() == nat.SA_EINVAL
    assert write(dtype=nat.SA_I32) == nat.SA_EUNSUPPORTED and write(T=0) == nat.SA_OK

    def decode(dtype=nat.SA_F16, B=2, H=4, Hkv=2, D=16, page=4, Lp=2, plen=8, TD=3, r=1, local=0):
        return lib.sa_ultrametric_prefix_decode(dtype, B, H, Hkv, D, page, 6, None, st, None, st, None, st, None, Lp, plen,
                                                None, None, st, 3, None, None, nat.SA_I32, st, None, nat.SA_I32, st, TD, r,
                                                local, 0, None, st, None, None, 0, None)
    assert decode(B=0) == nat.SA_OK
    for kw in (dict(B=-1), dict(H=3), dict(plen=9), dict(plen=-1), dict(r=4), dict(r=-1), dict(local=-1), dict(TD=0), {}):
        assert decode(**kw) == nat.SA_EINVAL, kw
    assert decode(dtype=7) == nat.SA_EUNSUPPORTED and decode(D=257) == nat.SA_EUNSUPPORTED
    size = lib.sa_ultrametric_prefix_decode_workspace_bytes
    assert size(nat.SA_BF16, 0, 4, 2, 64, 16, 4, 4) == 0 and size(nat.SA_BF16, 4, 4, 2, 64, 16, 0, 4) > 0


def test_oracle_agrees_with_the_routed_decode_oracle():
    g = torch.Generator().manual_seed(1)
    B, H, Hkv, D, page, n = 4, 4, 2, 16, 8, 24
    ctx = torch.tensor([0, 5, 8, 30], dtype=torch.int32)
    perm = torch.randperm(24, generator=g).to(torch.int32)
    pp, bt = perm[:3], perm[3:19].view(B, 4)
    kc, vc = (torch.randn(24, Hkv, page, D, generator=g) for _ in range(2))
    q = torch.randn(B, H, D, generator=g)
    ri = torch.randint(0, 2, (24, H, 2), generator=g, dtype=torch.int32)
    qri = torch.randint(0, 2, (B, H, 2), generator=g, dtype=torch.int32)
    for r, local, sink in ((0, 0, False), (1, 1, True), (2, 3, False)):
        out, lse, _ = so.prefix_decode(q, kc, vc, pp, n, bt, ctx, ri, qri, r, local, sink)
        joined = torch.cat([pp[None].expand(B, -1), bt], 1)
        ref = dor.ultrametric_decode_reference(q, kc, vc, joined, ctx + n, ri, qri, r, local_blocks=local, sink_block=sink,
                                               compute_dtype=torch.float64)
        assert (out - ref.double()).abs().max() < 1e-6
        assert torch.equal(torch.isinf(lse), (out == 0).all(-1))
