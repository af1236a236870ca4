"""GPU checks of the shared-prefix decode against a 64-bit oracle over the joined page list.

Error bound per element, with u the unit roundoff of the type (2^-8 bf16, 2^-11 fp16): the
probabilities are rounded once to the type before they meet V (relative u each, so at most
u * sum p |v|) and the result once (u * |out|); 1e-5 * max|v| covers the 32-bit arithmetic.  fp32: the
norm-wise 1e-5 of the other operators.  The LSE carries no rounding to 16 bits: 1e-4 absolute covers
D = 128 products summed in 32 bits (128 * 2^-23 * sum |q k| / sqrt(D), about 2e-5 here) and the
exponentials."""

import pytest
import torch

from helpers import assert_fp32_close, lse_close
from oracle import serving_oracle as so
from ultrametric import _native as nat
from ultrametric import ultrametric_decode, ultrametric_prefix_decode

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(B, H, Hkv, D, page, prefix, own, dtype=torch.bfloat16, TD=3, arity=2, seed=0, idt=torch.int32):
    """own: own tokens of each request (a list)."""
    g = torch.Generator().manual_seed(seed)
    Lp, L = -(-prefix // page), max(1, -(-max(own) // page))
    P = Lp + B * L + 3
    perm = torch.randperm(P, generator=g).to(torch.int32)
    t = dict(q=torch.randn(B, H, D, generator=g).to(dtype), kc=torch.randn(P, Hkv, page, D, generator=g).to(dtype),
             vc=torch.randn(P, Hkv, page, D, generator=g).to(dtype), pp=perm[:Lp].clone(),
             bt=perm[Lp:Lp + B * L].view(B, L).clone(), ctx=torch.tensor(own, dtype=torch.int32),
             ri=torch.randint(0, arity, (P, H, TD), generator=g).to(idt),
             qri=torch.randint(0, arity, (B, H, TD), generator=g).to(idt))
    return t, prefix


def call(t, prefix, depth, local=0, sink=False, **kw):
    d = {k: v.to(DEV) for k, v in t.items()}
    plen = prefix.to(DEV) if isinstance(prefix, torch.Tensor) else prefix
    return ultrametric_prefix_decode(d["q"], d["kc"], d["vc"], d["pp"], plen, d["bt"], d["ctx"], d["ri"], d["qri"], depth,
                                     local_blocks=local, sink_block=sink, return_lse=True, **kw)


def check(t, prefix, depth, local=0, sink=False, got=None, status=0):
    out, lse = call(t, prefix, depth, local, sink) if got is None else got
    ref, rlse, w = so.prefix_decode(t["q"], t["kc"], t["vc"], t["pp"], prefix, t["bt"], t["ctx"], t["ri"], t["qri"],
                                    depth, local, sink)
    o = out.double().cpu()
    assert out.dtype == t["q"].dtype and torch.isfinite(o).all()
    if t["q"].dtype == torch.float32:
        assert_fp32_close(out, ref, "prefix decode")
    else:
        vmax = t["vc"].double().nan_to_num(0, 0, 0).abs().max()
        over = (o - ref).abs() - U[t["q"].dtype] * (w + ref.abs()) - 1e-5 * vmax
        assert over.max() <= 0, f"{over.max():.3e} over the bound at {(over == over.max()).nonzero()[0].tolist()}"
    lse_close(lse, rlse, 1e-4)
    empty = torch.isinf(rlse)
    assert (o[empty] == 0).all()
    assert nat.read_device_status(reset=True) == status


SHAPES = [  # B, H, Hkv, D, page, prefix, own
    (1, 1, 1, 64, 16, 1, [0]),
    (1, 4, 1, 128, 64, 64, [1]),
    (3, 8, 2, 64, 16, 203, [0, 9, 40]),
    (2, 4, 4, 128, 32, 0, [33, 1]),
    (5, 6, 3, 80, 8, 77, [3, 0, 16, 17, 64]),
    (4, 8, 1, 96, 24, 500, [1, 25, 120, 130]),
    (9, 16, 2, 128, 128, 300, [0, 1, 127, 128, 129, 256, 5, 60, 64]),
    (3, 4, 2, 128, 192, 700, [400, 1, 193]),
    (40, 8, 2, 128, 64, 1000, [7 * i % 150 for i in range(40)]),
    (70, 8, 2, 64, 64, 777, [11 * i % 90 for i in range(70)]),
    (130, 8, 1, 64, 32, 250, [i % 50 for i in range(130)]),
    (3, 40, 2, 64, 16, 130, [5, 0, 70]),
    (2, 8, 8, 8, 40, 90, [0, 41]),
]


@pytest.mark.parametrize("shape", SHAPES, ids=[f"B{s[0]}H{s[1]}-{s[2]}D{s[3]}p{s[4]}n{s[5]}" for s in SHAPES])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("depth,local,sink", [(0, 0, False), (1, 1, True), (3, 0, False)])
def test_matches_oracle(shape, dtype, depth, local, sink):
    t, n = make(*shape, dtype=dtype, seed=sum(shape[:6]))
    check(t, n, depth, local, sink)


@pytest.mark.parametrize("D,page,dtype", [(20, 16, torch.float16), (7, 5, torch.bfloat16), (256, 16, torch.bfloat16),
                                          (200, 12, torch.float32), (128, 20, torch.bfloat16)])
def test_general_path_shapes(D, page, dtype):
    t, n = make(3, 6, 2, D, page, 333, [0, 50, 9], dtype=dtype, seed=D)
    check(t, n, 1, 2, True)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float32, 64)])
@pytest.mark.parametrize("local", [1, 3, 50])
def test_local_pages_reach_into_the_prefix(dtype, D, local):
    t, n = make(4, 4, 2, D, 16, 90, [0, 5, 17, 40], dtype=dtype, TD=2, arity=7, seed=local)
    check(t, n, 2, local, False)
    check(t, n, 2, local, True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_attend_nothing(dtype):
    t, n = make(6, 4, 2, 128, 16, 300, [0, 0, 20, 64, 1, 300], dtype=dtype, seed=3)
    t["qri"][1] = 5  # matches no page
    t["qri"][3, 2] = 5
    check(t, n, 2)
    t["ctx"][:] = 0
    check(t, 0, 0)
    check(t, 0, 1, 4, True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
def test_values_in_masked_places_do_not_spread(dtype, poison):
    t, n = make(5, 8, 2, 64, 16, 200, [0, 30, 7, 100, 16], dtype=dtype, TD=2, seed=11)
    used = torch.zeros(t["kc"].shape[0], 16, dtype=torch.bool)
    for ids, m in [(t["pp"], n)] + [(t["bt"][b], int(t["ctx"][b])) for b in range(5)]:
        for j in range(m):
            used[ids[j // 16].long(), j % 16] = True
    for c in ("kc", "vc"):  # rows past every length and unlisted pages
        t[c][(~used)[:, None].expand(-1, 2, -1)] = poison
    check(t, n, 1, 1, True)
    # a prefix page that only some rows attend: it must reach those alone
    page = int(t["pp"][3])
    for c in ("vc", "kc"):
        t[c][page, 1, 4] = poison
        out, lse = call(t, n, 1)
        hit = (t["ri"][page, :, 0][None] == t["qri"][:, :, 0]) & (torch.arange(8) >= 4)[None]
        assert hit.any() and not hit[:, 4:].all()
        keep = ~hit
        s = {k: v.clone() for k, v in t.items()}
        s["kc"][page, 1, 4] = 0
        s["vc"][page, 1, 4] = 0
        ref, rlse, w = so.prefix_decode(s["q"], s["kc"], s["vc"], s["pp"], n, s["bt"], s["ctx"], s["ri"], s["qri"], 1)
        o = out.double().cpu()
        assert torch.isfinite(o[keep]).all()
        u = U.get(dtype, 1e-6)
        assert ((o - ref).abs() - u * (w + ref.abs()) - 5e-5)[keep].max() <= 0
        lse_close(lse.cpu()[keep], rlse[keep], 1e-4)
        if c == "vc":
            assert not torch.isfinite(o[hit]).all(-1).any()


def test_equals_the_routed_decode_over_joined_tables():
    t, n = make(17, 16, 4, 128, 64, 512, [i * 13 % 200 for i in range(17)], seed=4)
    out, _ = call(t, n, 2, 1, True)
    joined = torch.cat([t["pp"][None].expand(17, -1), t["bt"]], 1)
    d = {k: v.to(DEV) for k, v in t.items()}
    ref = ultrametric_decode(d["q"], d["kc"], d["vc"], joined.to(DEV), (t["ctx"] + n).to(DEV), d["ri"], d["qri"], 2,
                             local_blocks=1, sink_block=True)
    # both round their probabilities and results to bf16: twice the bound of one, |out| <= max |v|
    assert (out.float() - ref.float()).abs().max() <= 2 * 2.0 ** -8 * 2 * float(t["vc"].abs().max())
    check(t, n, 2, 1, True, got=call(t, n, 2, 1, True))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_and_tied_scores(dtype):
    t, n = make(20, 8, 2, 128, 16, 400, [3 * i for i in range(20)], dtype=dtype, seed=6)
    t["q"] = t["q"] * 30  # sharp rows, maxima that rise along the keys
    if dtype == torch.float32:
        # scores of some hundreds: 2^-23 of them is the error of the exponent, so the norm-wise bound scales
        out, _ = call(t, n, 0)
        ref, _, _ = so.prefix_decode(t["q"], t["kc"], t["vc"], t["pp"], n, t["bt"], t["ctx"], t["ri"], t["qri"], 0)
        assert (out.double().cpu() - ref).norm() <= 300 * 2.0 ** -20 * ref.norm()
    else:
        out, lse = call(t, n, 0)
        ref, rlse, w = so.prefix_decode(t["q"], t["kc"], t["vc"], t["pp"], n, t["bt"], t["ctx"], t["ri"], t["qri"], 0)
        # the scores' own 32-bit error (|s| up to 400, 128 products) moves a weight by up to 2e-3 relative
        assert ((out.double().cpu() - ref).abs() - (2.0 ** -8 + 4e-3) * (w + ref.abs()) - 1e-4).max() <= 0
    t["kc"][:] = t["kc"][:1]  # every key alike
    check(t, n, 0)


def test_layouts_dtypes_and_streams():
    t, n = make(6, 8, 2, 128, 32, 270, [0, 5, 33, 64, 90, 31], seed=9)
    want = call(t, n, 1, 1, True)
    d = {k: v.to(DEV) for k, v in t.items()}
    B, H, D = t["q"].shape
    packed = torch.zeros(B, H + 4, D, dtype=torch.bfloat16, device=DEV)
    packed[:, 2:2 + H] = d["q"]
    token_major = [d[c].transpose(1, 2).contiguous().transpose(1, 2) for c in ("kc", "vc")]
    wide_bt = torch.zeros(B, 2 * d["bt"].shape[1], dtype=torch.int64, device=DEV)
    wide_bt[:, ::2] = d["bt"]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ultrametric_prefix_decode(packed[:, 2:2 + H], *token_major, d["pp"].long(), torch.tensor([n], dtype=torch.int32, device=DEV),
                                        wide_bt[:, ::2], d["ctx"].long(), d["ri"].long(), d["qri"].transpose(1, 2).contiguous().transpose(1, 2),
                                        1, local_blocks=1, sink_block=True, return_lse=True)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # caches and queries that are not 16-byte aligned take the general path
    pad = torch.zeros(d["kc"].numel() + 1, dtype=torch.bfloat16, device=DEV)[1:].view(d["kc"].shape)
    pad.copy_(d["kc"])
    odd = ultrametric_prefix_decode(d["q"], pad, d["vc"], d["pp"], n, d["bt"], d["ctx"], d["ri"], d["qri"], 1, local_blocks=1,
                                    sink_block=True, return_lse=True)
    check(t, n, 1, 1, True, got=odd)
    check(t, n, 1, 1, True, got=want)


def test_repeats_bit_for_bit_and_replays_in_a_graph():
    t, n = make(33, 16, 4, 128, 64, 1500, [i * 29 % 300 for i in range(33)], seed=2)
    d = {k: v.to(DEV) for k, v in t.items()}
    plen = torch.tensor([n], dtype=torch.int32, device=DEV)

    def go():
        return ultrametric_prefix_decode(d["q"], d["kc"], d["vc"], d["pp"], plen, d["bt"], d["ctx"], d["ri"], d["qri"], 1,
                                         return_lse=True)
    a = go()
    b = go()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c = go()
    plen.fill_(700)  # lengths are read on the device at replay
    d["ctx"].copy_(t["ctx"].flip(0))
    g.replay()
    torch.cuda.synchronize()
    t2 = dict(t, ctx=t["ctx"].flip(0))
    check(t2, 700, 1, got=c)


def test_pages_outside_the_pool_are_skipped_and_flagged():
    for dtype in (torch.bfloat16, torch.float32):
        t, n = make(3, 4, 2, 64, 16, 100, [20, 0, 50], dtype=dtype, seed=1)
        t["pp"][2] = 10 ** 6
        t["bt"][2, 1] = -3
        check(t, n, 0, status=2)


def test_pool_past_32_bit_offsets():
    B, H, Hkv, D, page, n = 3, 8, 8, 128, 64, 130
    t, _ = make(B, H, Hkv, D, page, n, [70, 0, 9], seed=5)
    P0 = t["kc"].shape[0]
    P = 2 ** 32 // (page * Hkv * D * 2) + P0
    d = {k: v.to(DEV) for k, v in t.items()}
    big = torch.empty(P, Hkv, page, D, dtype=torch.bfloat16, device=DEV)
    ri = torch.zeros(P, H, 3, dtype=torch.int32, device=DEV)
    off = P - P0
    outs = []
    for c in ("kc", "vc"):
        big[off:] = d[c]
        outs.append(big)
        if c == "kc":
            big = torch.empty_like(big)
    ri[off:] = d["ri"]
    got = ultrametric_prefix_decode(d["q"], outs[0], outs[1], d["pp"] + off, n, d["bt"] + off, d["ctx"], ri, d["qri"], 1,
                                    return_lse=True)
    check(t, n, 1, got=got)


def test_broadcast_and_unaligned_inputs():
    t, n = make(5, 8, 2, 128, 16, 130, [0, 5, 33, 17, 64], seed=12)
    t["q"] = t["q"][:1].expand(5, -1, -1).contiguous()
    for c in ("kc", "vc"):
        t[c] = t[c][:, :1].expand(-1, 2, -1, -1).contiguous()
    d = {k: v.to(DEV) for k, v in t.items()}
    rest = (d["pp"], n, d["bt"], d["ctx"], d["ri"], d["qri"], 1)
    heads = [d[c][:, :1].contiguous().expand(-1, 2, -1, -1) for c in ("kc", "vc")]  # one head for both: stride 0
    qb = d["q"][:1].expand(5, -1, -1)
    odd = torch.zeros(d["q"].numel() + 1, dtype=torch.bfloat16, device=DEV)[1:].view(d["q"].shape)
    odd.copy_(d["q"])
    for q, kc, vc in ((qb, d["kc"], d["vc"]), (odd, d["kc"], d["vc"]), (d["q"], *heads), (qb, *heads)):
        check(t, n, 1, got=ultrametric_prefix_decode(q, kc, vc, *rest, return_lse=True))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("depth", [0, 1])
def test_no_own_table_and_no_prefix_list(dtype, depth):
    t, n = make(19, 8, 2, 64, 16, 210, [0] * 19, dtype=dtype, seed=13)
    t["bt"] = t["bt"][:, :0].contiguous()
    check(t, n, depth, 1, True)  # the prefix alone, without a column of own pages
    t["pp"] = t["pp"][:0].contiguous()
    check(t, 0, depth, 1, True)  # nothing at all
    t, _ = make(19, 8, 2, 64, 16, 0, [5 * i for i in range(19)], dtype=dtype, seed=14)
    check(t, 0, depth)  # own pages alone


@pytest.mark.parametrize("B,H,Hkv,D,page,prefix,hi", [
    (60, 9, 3, 64, 16, 300, 40),    # groups of 3: 126 of a tile's 128 rows
    (41, 35, 5, 128, 32, 700, 70),  # 7
    (9, 34, 2, 96, 64, 260, 200),   # 17: own items in the 128-row form
    (5, 132, 2, 64, 16, 333, 90),   # 66: one request per row tile
    (3, 128, 1, 128, 64, 500, 130),
    (17, 256, 16, 64, 128, 900, 300),
    (300, 4, 4, 128, 64, 128, 3),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("depth", [0, 1])
def test_group_sizes(B, H, Hkv, D, page, prefix, hi, dtype, depth):
    t, n = make(B, H, Hkv, D, page, prefix, [(i * 37 + 5) % (hi + 1) for i in range(B)], dtype=dtype, seed=B)
    check(t, n, depth, depth, bool(depth))
