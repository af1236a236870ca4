"""Routed paged decode of a batch whose requests share a long prefix, the prefix computed once.

``ultrametric_decode`` (``kernel_decode.py``; sparse-ai's ``src/ultrametric/kernel_decode.py:
188-247``) reads every request's pages by itself, so a prefix that many requests share -- a system
prompt, a document that is asked about, several samples of one prompt -- is streamed once per
request.  ``ultrametric_prefix_decode`` takes the prefix's pages apart from the requests' own:
the query rows of all requests meet the prefix's keys in one product per KV head, each request
meets its own pages, and the parts are joined by log-sum-exp.  Routing, sink and local pages act
on the joined page list, as if the prefix's pages stood first in every block table.
"""

from __future__ import annotations

import functools
from typing import Union

import torch

from . import _native as nat


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(code, B, H, Hkv, D, page, Lp, L, device_index):
    return max(256, int(nat.lib().sa_ultrametric_prefix_decode_workspace_bytes(code, B, H, Hkv, D, page, Lp, L)))


def _rows_load(q: torch.Tensor) -> bool:
    """Whether q's rows can be loaded where they are: 16-byte aligned, no broadcast dimension.  (Copying
    a few rows costs a launch; the path that reads any layout takes many times the time.)"""
    if q.data_ptr() % 16:
        return False
    if q.is_contiguous():
        return True
    a, b, c = q.stride()
    unit = 16 // q.element_size()
    return c == 1 and a > 0 and b > 0 and a % unit == 0 and b % unit == 0


def ultrametric_prefix_decode(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    prefix_pages: torch.Tensor,
    prefix_len: Union[int, torch.Tensor],
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    router_indices: torch.Tensor,
    q_router_indices: torch.Tensor,
    req_depth: int,
    local_blocks: int = 0,
    sink_block: bool = False,
    return_lse: bool = False,
):
    """Decode one token per request against a shared prefix and the request's own pages.

    q (B, H, D); k_cache, v_cache (num_pages, Hkv, page_size, D), H % Hkv == 0; prefix_pages (Lp,)
    int32; ``prefix_len`` tokens of them are valid (an int, or one int32 on the device, which is
    not read back); block_tables (B, L) int32 and context_lens (B,): each request's own pages and
    own tokens (0: the prefix alone).  router_indices (num_pages, H, TD), q_router_indices
    (B, H, TD), req_depth, local_blocks and sink_block as in ``ultrametric_decode``, over the
    prefix's pages followed by the request's own; req_depth 0 attends every page.

    Returns (B, H, D) in q.dtype, and with ``return_lse`` the (B, H) fp32 natural-log LSE; a row
    that attends nothing gets zeros and -inf.  fp32, fp16 or bf16; head_dim up to 256.
    fp16/bf16 with head_dim a multiple of 8 up to 128 and a page size that is a multiple of 8 run
    on the tensor cores, the rest on the CUDA cores, as do tables wider than about 1.8e10 tokens x KV
    heads over all requests.  All tensors lie on the current device."""
    if q.dim() != 3:
        raise ValueError(f"q must be (B, H, D), got {tuple(q.shape)}")
    B, H, D = q.shape
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError(f"k_cache/v_cache must be (num_pages, Hkv, page_size, D); got "
                         f"{tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    P, Hkv, page, d2 = k_cache.shape
    if d2 != D or Hkv == 0 or H % Hkv:
        raise ValueError("cache head_dim / heads incompatible with q")
    dtype = q.dtype
    if not (k_cache.dtype is dtype and v_cache.dtype is dtype):
        raise ValueError("q, k_cache, v_cache must share dtype")
    rows, L = block_tables.shape if block_tables.dim() == 2 else (-1, 0)
    if rows != B or prefix_pages.dim() != 1 or context_lens.dim() != 1 or context_lens.shape[0] != B:
        raise ValueError(f"expected prefix_pages (Lp,), block_tables ({B}, L) and context_lens ({B},); got "
                         f"{tuple(prefix_pages.shape)}, {tuple(block_tables.shape)}, {tuple(context_lens.shape)}")
    Lp = prefix_pages.shape[0]
    TD = q_router_indices.shape[2] if q_router_indices.dim() == 3 else 0
    if TD < 1 or q_router_indices.shape != (B, H, TD) or router_indices.shape != (P, H, TD):
        raise ValueError(f"router_indices must be ({P}, {H}, TD) and q_router_indices ({B}, {H}, TD); got "
                         f"{tuple(router_indices.shape)}, {tuple(q_router_indices.shape)}")
    req_depth, local_blocks = int(req_depth), int(local_blocks)
    if not 0 <= req_depth <= TD:
        raise ValueError(f"req_depth must be in [0, {TD}], got {req_depth}")
    if local_blocks < 0:
        raise ValueError(f"local_blocks must be >= 0, got {local_blocks}")
    plen_dev = None
    if isinstance(prefix_len, torch.Tensor):
        if prefix_len.dtype is not torch.int32 or prefix_len.numel() != 1:
            raise ValueError(f"prefix_len must be an int or one int32, got {prefix_len.dtype} {tuple(prefix_len.shape)}")
        plen_dev, plen = prefix_len, 0
    else:
        plen = int(prefix_len)
        if not 0 <= plen <= Lp * page:
            raise ValueError(f"prefix_len {plen} does not fit {Lp} pages of {page}")
    nat.require_one_device("ultrametric_prefix_decode", q, k_cache, v_cache, prefix_pages, plen_dev, block_tables,
                           context_lens, router_indices, q_router_indices)
    code = nat.float_code(dtype)
    i32, i64 = torch.int32, torch.int64
    pp = (prefix_pages if prefix_pages.dtype is i32 else prefix_pages.to(i32)).contiguous()
    bt = block_tables if block_tables.dtype is i32 else block_tables.to(i32)
    ctx = (context_lens if context_lens.dtype is i32 else context_lens.to(i32)).contiguous()
    ri = router_indices if router_indices.dtype in (i32, i64) else router_indices.to(i64)
    qri = q_router_indices if q_router_indices.dtype in (i32, i64) else q_router_indices.to(i64)
    kc = k_cache if k_cache.stride()[3] == 1 else k_cache.contiguous()
    vc = v_cache if v_cache.stride()[3] == 1 else v_cache.contiguous()
    qq = q if _rows_load(q) else q.clone(memory_format=torch.contiguous_format)
    out = torch.empty_like(qq, memory_format=torch.contiguous_format)
    lse = q.new_empty((B, H), dtype=torch.float32) if return_lse else None
    ws_bytes = _workspace_bytes(code, B, H, Hkv, D, page, Lp, L, q.get_device())
    ws = q.new_empty(ws_bytes, dtype=torch.uint8)
    st, ptr = nat.cached_strides, nat.ptr
    nat.check(nat.lib().sa_ultrametric_prefix_decode(
        code, B, H, Hkv, D, page, P, qq.data_ptr(), st(qq), kc.data_ptr(), st(kc), vc.data_ptr(), st(vc), pp.data_ptr(), Lp,
        plen, ptr(plen_dev), bt.data_ptr(), st(bt), L, ctx.data_ptr(), ri.data_ptr(), nat.int_code(ri.dtype), st(ri),
        qri.data_ptr(), nat.int_code(qri.dtype), st(qri), TD, req_depth, local_blocks, int(bool(sink_block)),
        out.data_ptr(), st(out), ptr(lse), ws.data_ptr(), ws_bytes, nat.raw_stream(q)), "ultrametric_prefix_decode")
    return (out, lse) if return_lse else out
