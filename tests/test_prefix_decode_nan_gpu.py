"""GPU checks of the shared-prefix decode on scores that are not numbers.

A row that attends a key whose score is NaN has a NaN result and a NaN LSE, whichever form its keys
are computed in: the 16-column form (groups of up to 16 heads over own pages, batches of up to 16
rows over the prefix), the 128-row form, or the CUDA cores.  Every other row keeps the bounds of
``test_prefix_decode_gpu.py``."""

import pytest
import torch

from helpers import lse_close
from oracle import serving_oracle as so
from test_prefix_decode_gpu import U, call, make
from ultrametric import _native as nat

pytestmark = pytest.mark.gpu
NAN = float("nan")
# heads per KV head: 16-column form, 128-row form
GROUPS = [4, 16, 24]
TYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])


def check_nan(t, prefix, depth, local=0, sink=False):
    """Rows (b, h) whose result is NaN by the definition; returns their mask."""
    out, lse = call(t, prefix, depth, local, sink)
    ref, rlse, w = so.prefix_decode(t["q"], t["kc"], t["vc"], t["pp"], prefix, t["bt"], t["ctx"], t["ri"], t["qri"],
                                    depth, local, sink)
    o, bad = out.double().cpu(), torch.isnan(rlse)
    assert torch.equal(torch.isnan(lse.cpu()), bad), "LSE: rows with NaN"
    assert torch.equal(torch.isnan(o).all(-1), bad) and torch.isfinite(o[~bad]).all(), "output: rows with NaN"
    vmax = t["vc"].double().abs().max()
    u = U.get(t["q"].dtype, 2.0 ** -20)
    over = ((o - ref).abs() - u * (w + ref.abs()) - 1e-5 * vmax)[~bad]
    assert over.numel() == 0 or over.max() <= 0, f"{over.max():.3e} over the bound"
    lse_close(lse.cpu()[~bad], rlse[~bad], 1e-4)
    assert nat.read_device_status(reset=True) == 0
    return bad


@TYPES
@pytest.mark.parametrize("G", GROUPS)
@pytest.mark.parametrize("prefix", [0, 5, 200])
def test_only_own_token_is_nan(dtype, G, prefix):
    t, n = make(5, 2 * G, 2, 64, 16, prefix, [1, 1, 40, 1, 0], dtype=dtype, seed=G)
    t["kc"][t["bt"][1, 0], 1, 0] = NAN  # request 1, the second KV head
    bad = check_nan(t, n, 0)
    assert bad[1, G:].all() and bad.sum() == G


@TYPES
@pytest.mark.parametrize("G", GROUPS)
@pytest.mark.parametrize("page,own", [(16, [3, 60, 1]), (48, [30, 100, 96]), (24, [200, 500, 7]), (64, [64, 127, 300])])
def test_nan_query_without_a_prefix(dtype, G, page, own):
    t, n = make(3, 2 * G, 2, 128, page, 0, own, dtype=dtype, seed=page + G)
    t["q"][0, 1] = NAN           # every column
    t["q"][1, G, 5] = NAN        # one column makes every score NaN
    t["q"][2, 2 * G - 1] = NAN
    bad = check_nan(t, n, 0)
    assert bad.sum() == 3


@TYPES
@pytest.mark.parametrize("B,G", [(1, 4), (2, 8), (4, 4), (3, 24), (40, 4)])
def test_nan_query_over_the_prefix(dtype, B, G):
    t, n = make(B, 2 * G, 2, 64, 24, 333, [5 * i % 31 for i in range(B)], dtype=dtype, seed=B)
    t["q"][B - 1, G] = NAN
    assert check_nan(t, n, 0).sum() == 1


@TYPES
@pytest.mark.parametrize("B,G", [(1, 8), (2, 4), (3, 5), (2, 16), (9, 4)])
def test_routed_pages_of_nan(dtype, B, G):
    """Rows whose only attended pages hold NaN keys, beside rows that attend others as well."""
    H = 2 * G
    t, n = make(B, H, 2, 128, 16, 170, [21 + i for i in range(B)], dtype=dtype, TD=1, arity=2, seed=G)
    t["ri"][:] = 0
    t["qri"][:] = 0
    page, own = int(t["pp"][4]), int(t["bt"][0, 1])
    t["ri"][page], t["ri"][own] = 1, 2
    t["qri"][0, 1::2] = 1       # these heads attend the prefix's page 4 alone
    t["qri"][B - 1, 0] = 2      # own page 1 of request 0 alone, or, in another request, nothing
    t["kc"][page, 1] = NAN
    t["kc"][own, 0] = NAN
    bad = check_nan(t, n, 1)
    assert bad[0, 1::2][torch.arange(1, H, 2) >= G].all() and not bad[0, 1:G:2].any()
    assert bool(bad[B - 1, 0]) == (B == 1)
    # one NaN key of the page: it reaches those that attend the page, as before
    t["kc"][page, 1, 1:] = 0.5
    check_nan(t, n, 1, 1, True)


@TYPES
@pytest.mark.parametrize("G", [4, 24])
@pytest.mark.parametrize("lo,hi", [(0, 16), (0, 128), (128, 256), (250, 300)])
def test_nan_in_one_tile_of_several(dtype, G, lo, hi):
    t, n = make(2, G, 1, 64, 16, 0, [300, 299], dtype=dtype, seed=lo + hi)
    pos = torch.arange(lo, min(hi, 299))
    t["kc"][t["bt"][1].long()[pos // 16], 0, pos % 16] = NAN
    bad = check_nan(t, n, 0)
    assert bad[1].all() and not bad[0].any()
