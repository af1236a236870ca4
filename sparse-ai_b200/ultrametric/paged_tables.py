"""Page allocation, slot maps and ragged K/V writes of a serving step, on the device.

``PagedKVCache`` (``paged.py``) keeps its page allocator on the host and writes one prompt or one
token per request at a time.  These operators do the same work for a whole ragged step from
device tensors alone -- request lengths in, tables and slots out -- with no host synchronisation,
so a step's bookkeeping can follow the previous step's sampling on the device or be captured in a
CUDA graph:

* ``build_paged_tables``     -> ``sa_paged_build_tables``: pages for the step's new tokens from a
  stack of free pages, the slot of every new token, positions, row ranges, new lengths;
* ``release_paged_requests`` -> ``sa_paged_release``: finished requests' pages back on the stack;
* ``paged_kv_write``         -> ``sa_paged_kv_write``: K/V rows (and the touched pages' routing
  vectors) into the cache by the slot map.

sparse-ai has no counterpart: its paged decode (``src/ultrametric/kernel_decode.py:188-247``)
reads such a cache and nothing there writes one.  CUDA tensors of the current device only.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _native as nat


class PagedTables(NamedTuple):
    """What ``build_paged_tables`` returns, besides the entries it adds to ``block_tables``.

    slot_mapping:  (num_tokens,) int64, page * page_size + row; -1: no slot.
    request_ids:   (num_tokens,) int32, the row's request; -1 past the last token.
    positions:     (num_tokens,) int32, the token's position in its request; 0 past the last.
    cu_new_lens:   (B + 1,) int32, request b's rows are [cu[b], cu[b + 1]).
    context_lens:  (B,) int32, lengths after the step.
    num_free:      (1,) int32, height of the free stack after the step.
    """

    slot_mapping: torch.Tensor
    request_ids: torch.Tensor
    positions: torch.Tensor
    cu_new_lens: torch.Tensor
    context_lens: torch.Tensor
    num_free: torch.Tensor


def _check_written(name, t):
    """Refuse a broadcast tensor that the kernels write: its elements share addresses."""
    st = t.stride()
    if 0 in st and any(s == 0 and n > 1 for s, n in zip(st, t.shape)):
        raise ValueError(f"{name} is written in place and must not be broadcast; got strides {tuple(st)} for "
                         f"{tuple(t.shape)}")


def _tables_args(context_lens, block_tables, free_pages, num_free, page_size, per_request):
    """(B, L) of checked arguments; ``per_request`` = (name, tensor, dtype) beside the lengths."""
    i32 = torch.int32
    if context_lens.dim() != 1 or block_tables.dim() != 2 or free_pages.dim() != 1:
        raise ValueError("context_lens and free_pages must be 1-d and block_tables 2-d; got "
                         f"{tuple(context_lens.shape)}, {tuple(free_pages.shape)}, {tuple(block_tables.shape)}")
    (B,), (rows, L) = shape, _ = context_lens.shape, block_tables.shape
    name, t, dtype = per_request
    if not (context_lens.dtype is i32 and block_tables.dtype is i32 and free_pages.dtype is i32) or rows != B:
        raise ValueError(f"context_lens, block_tables and free_pages must be int32 of shapes ({B},), ({B}, L) and (F,); got "
                         + ", ".join(f"{x.dtype} {tuple(x.shape)}" for x in (context_lens, block_tables, free_pages)))
    if t.dtype is not dtype or t.shape != shape:
        raise ValueError(f"{name} must be {dtype} of shape ({B},), got {t.dtype} {tuple(t.shape)}")
    if num_free.dtype is not i32 or num_free.numel() != 1:
        raise ValueError(f"num_free must be one int32, got {num_free.dtype} {tuple(num_free.shape)}")
    if not free_pages.is_contiguous():
        raise ValueError("free_pages must be contiguous")
    if page_size < 1:
        raise ValueError(f"page_size must be >= 1, got {page_size}")
    return B, L


def build_paged_tables(
    context_lens: torch.Tensor,
    new_lens: torch.Tensor,
    block_tables: torch.Tensor,
    free_pages: torch.Tensor,
    num_free: torch.Tensor,
    *,
    page_size: int,
    num_tokens: int,
    position_base: int = 0,
) -> PagedTables:
    """Pages and slots for ``new_lens[b]`` more tokens of each request.

    context_lens, new_lens  (B,) int32: tokens held, tokens to add (0 for idle requests).
    block_tables            (B, L) int32, physical page per logical page; the new pages' entries
                            are written in place, the others are left as they are.
    free_pages, num_free    (F,) and (1,) int32: a stack of free pages, taken from its top in
                            request order.  Neither is changed: the new height is returned.
    num_tokens              rows of the flat token batch (a host number: the sum of ``new_lens``,
                            or more to keep one shape from step to step).
    position_base           added to the positions (the length of a shared prefix).

    A request that does not fit (negative length, more than L pages, rows past ``num_tokens``,
    positions past 2^31 - 1, or no pages left) is refused: its rows get slot -1, its length and
    table stay, and the device status gets bit 2.  Requests after one that found no pages are
    refused too if they need any.
    Nothing is read back to the host."""
    page_size, T, position_base = int(page_size), int(num_tokens), int(position_base)
    B, L = _tables_args(context_lens, block_tables, free_pages, num_free, page_size,
                        ("new_lens", new_lens, torch.int32))
    if T < 0:
        raise ValueError(f"num_tokens must be >= 0, got {num_tokens}")
    if position_base < 0:
        raise ValueError(f"position_base must be >= 0, got {position_base}")
    _check_written("block_tables", block_tables)
    nat.require_one_device("build_paged_tables", context_lens, new_lens, block_tables, free_pages, num_free)
    ctx, new = context_lens.contiguous(), new_lens.contiguous()
    slots = ctx.new_empty(T, dtype=torch.int64)
    # the int32 results share one allocation, those by token on 16-byte boundaries
    pad = -T % 4
    buf = ctx.new_empty(2 * (T + pad) + 2 * B + 2)
    rid, _, pos, _, cu, ctx_out, free_out = buf.unsafe_split_with_sizes((T, pad, T, pad, B + 1, B, 1))
    p0 = buf.data_ptr()
    p1 = p0 + 8 * (T + pad)
    nat.check(nat.lib().sa_paged_build_tables(
        B, L, page_size, T, ctx.data_ptr(), new.data_ptr(), block_tables.data_ptr(),
        nat.cached_strides(block_tables), free_pages.data_ptr(), free_pages.shape[0], num_free.data_ptr(),
        position_base, slots.data_ptr(), p0, p0 + 4 * (T + pad), p1, p1 + 4 * (B + 1), p1 + 4 * (2 * B + 1),
        nat.raw_stream(ctx)), "build_paged_tables")
    return PagedTables(slots, rid, pos, cu, ctx_out, free_out)


def release_paged_requests(
    finished: torch.Tensor,
    context_lens: torch.Tensor,
    block_tables: torch.Tensor,
    free_pages: torch.Tensor,
    num_free: torch.Tensor,
    *,
    page_size: int,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Push the pages of every request with ``finished[b]`` ((B,) bool) back on the stack, in
    request order; returns the new (context_lens, num_free).  ``free_pages`` is written above its
    old height; the block tables are left as they are."""
    page_size = int(page_size)
    B, L = _tables_args(context_lens, block_tables, free_pages, num_free, page_size,
                        ("finished", finished, torch.bool))
    nat.require_one_device("release_paged_requests", finished, context_lens, block_tables, free_pages, num_free)
    ctx, done = context_lens.contiguous(), finished.contiguous()
    out_ctx, out_free = torch.empty_like(ctx), ctx.new_empty(1)
    nat.check(nat.lib().sa_paged_release(
        B, L, page_size, done.data_ptr(), ctx.data_ptr(), block_tables.data_ptr(), nat.cached_strides(block_tables),
        free_pages.data_ptr(), free_pages.shape[0], num_free.data_ptr(), out_ctx.data_ptr(), out_free.data_ptr(),
        nat.raw_stream(ctx)), "release_paged_requests")
    return out_ctx, out_free


def paged_kv_write(
    k: torch.Tensor,
    v: torch.Tensor,
    slot_mapping: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    *,
    routes: Optional[torch.Tensor] = None,
    router_indices: Optional[torch.Tensor] = None,
) -> None:
    """Write T tokens' K/V rows into the paged caches, in place.

    k, v            (T, Hkv, D), any strides with D contiguous (slices of a packed projection).
    slot_mapping    (T,) int64 as ``build_paged_tables`` makes it: distinct, -1 to skip a row.
    k_cache, v_cache  (P, Hkv, page_size, D) of k's dtype.
    routes, router_indices  optional (T, H, TD) and (P, H, TD) int32 or int64: a page that receives
                    tokens takes the routing vector of the last of them, as one append per token
                    would leave it (the rows of a page stand together in the batch)."""
    if k.dim() != 3 or v.shape != k.shape:
        raise ValueError(f"k and v must be (T, Hkv, D); got {tuple(k.shape)}, {tuple(v.shape)}")
    T, Hkv, D = k.shape
    P, h2, page, d2 = k_cache.shape if k_cache.dim() == 4 else (0, -1, 0, -1)
    if h2 != Hkv or d2 != D or v_cache.shape != k_cache.shape:
        raise ValueError(f"k_cache/v_cache must be (num_pages, {Hkv}, page_size, {D}); got "
                         f"{tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    dtype = k.dtype
    if not (v.dtype is dtype and k_cache.dtype is dtype and v_cache.dtype is dtype):
        raise ValueError("k, v, k_cache, v_cache must share dtype")
    if slot_mapping.dtype is not torch.int64 or slot_mapping.dim() != 1 or slot_mapping.shape[0] != T:
        raise ValueError(f"slot_mapping must be int64 of shape {(T,)}, got {slot_mapping.dtype} "
                         f"{tuple(slot_mapping.shape)}")
    if (routes is None) != (router_indices is None):
        raise ValueError("routes and router_indices go together")
    H = TD = 0
    if routes is not None:
        t2, H, TD = routes.shape if routes.dim() == 3 else (-1, 0, 0)
        if t2 != T or router_indices.shape != (P, H, TD):
            raise ValueError(f"routes must be (T, H, TD) and router_indices (num_pages, H, TD); got "
                             f"{tuple(routes.shape)}, {tuple(router_indices.shape)}")
        _check_written("router_indices", router_indices)
    kst, vst, kcs, vcs = k.stride(), v.stride(), k_cache.stride(), v_cache.stride()
    if kcs[3] != 1 or vcs[3] != 1:
        raise ValueError("the caches' head_dim must be contiguous")
    _check_written("k_cache", k_cache)
    _check_written("v_cache", v_cache)
    nat.require_one_device("paged_kv_write", k, v, slot_mapping, k_cache, v_cache, routes, router_indices)
    code = nat.float_code(dtype)
    kk = k if kst[2] == 1 else k.contiguous()
    vv = v if vst[2] == 1 else v.contiguous()
    slots = slot_mapping.contiguous()
    st = nat.cached_strides
    if routes is None:
        r_args = (None, 0, None, 0, 0, None, 0, None)
    else:
        r_args = (routes.data_ptr(), nat.int_code(routes.dtype), st(routes), H, TD, router_indices.data_ptr(),
                  nat.int_code(router_indices.dtype), st(router_indices))
    nat.check(nat.lib().sa_paged_kv_write(
        code, T, Hkv, D, page, P, kk.data_ptr(), st(kk), vv.data_ptr(), st(vv), slots.data_ptr(), k_cache.data_ptr(),
        st(k_cache), v_cache.data_ptr(), st(v_cache), *r_args, nat.raw_stream(k_cache)), "paged_kv_write")
