"""A paged, routed K/V cache for a batch of requests on one shared prefix, kept on the device.

``PagedKVCache`` (``paged.py``) allocates pages on the host and reads each request by itself.
``SharedPrefixCache`` keeps the allocator's state in device tensors (a stack of free pages, block
tables, lengths) and the prefix in pages of its own, and runs a serving step as four calls, none
of which reads anything back:

    tables = cache.plan(new_lens, num_tokens)       # pages, slots and positions of the new tokens
    for layer in range(num_layers):                 # q, k, v from tables.positions and the tokens
        cache.write(layer, k, v, tables, routes)    # ragged K/V rows and page routes
        out = cache.decode(layer, q, q_routes, req_depth)   # one query per request slot
    cache.finish(finished)                          # finished requests' pages go back

so a decode step (``plan`` with ``new_lens`` of ones, ``write``, ``decode``) can be captured in a CUDA
graph and replayed.  Routing vectors are per page, as in ``kernel_decode.py:79`` of sparse-ai's
``src/ultrametric``.
"""

from __future__ import annotations

from typing import Optional

import torch

from .kernel_prefix_decode import ultrametric_prefix_decode
from .paged_tables import PagedTables, build_paged_tables, paged_kv_write, release_paged_requests


class SharedPrefixCache:
    """Pools (num_layers, num_pages, Hkv, page_size, D) for K and V, page routes (num_layers,
    num_pages, H, TD), block tables (max_requests, max_pages_per_request), lengths, and the
    prefix's pages.  A request is a row of the block table; idle rows have length 0."""

    def __init__(self, num_pages: int, num_kv_heads: int, page_size: int, head_dim: int, num_heads: int,
                 tree_depth: int, max_requests: int, max_pages_per_request: int, max_prefix_pages: int,
                 num_layers: int = 1, dtype=torch.bfloat16, device="cuda"):
        self.page_size, self.num_layers, self.num_pages = int(page_size), int(num_layers), int(num_pages)
        shape = (num_layers, num_pages, num_kv_heads, page_size, head_dim)
        self.k_cache = torch.zeros(shape, dtype=dtype, device=device)
        self.v_cache = torch.zeros(shape, dtype=dtype, device=device)
        self.router = torch.zeros((num_layers, num_pages, num_heads, tree_depth), dtype=torch.int32, device=device)
        i32 = dict(dtype=torch.int32, device=device)
        self.block_tables = torch.zeros((max_requests, max_pages_per_request), **i32)
        self.context_lens = torch.zeros(max_requests, **i32)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, **i32)  # the top of the stack is page 0
        self.num_free = torch.tensor([num_pages], **i32)
        self.prefix_table = torch.zeros((1, max_prefix_pages), **i32)
        self.prefix_len = torch.zeros(1, **i32)  # read by the decode on the device
        self._prefix_tokens = 0                  # the same number for positions
        self._planned = False                    # requests may hold pages

    @property
    def prefix_tokens(self) -> int:
        return self._prefix_tokens

    def plan_prefix(self, num_tokens: int) -> PagedTables:
        """Pages for a prefix of ``num_tokens``; its K/V rows are then written, layer by layer, with
        ``write``.  The cache holds one prefix, set before any request: the positions of a request's
        tokens count from its end, and the whole pool is free for it."""
        if self._prefix_tokens:
            raise ValueError("the cache already holds a prefix")
        if self._planned:
            raise ValueError("the prefix must be set before any request is planned")
        if not 0 < num_tokens <= self.prefix_table.shape[1] * self.page_size:
            raise ValueError(f"a prefix of {num_tokens} tokens does not fit {self.prefix_table.shape[1]} pages of "
                             f"{self.page_size}")
        if num_tokens > self.num_pages * self.page_size:
            raise ValueError(f"a prefix of {num_tokens} tokens does not fit the cache's {self.num_pages} pages of "
                             f"{self.page_size}")
        n = torch.full((1,), int(num_tokens), dtype=torch.int32, device=self.prefix_len.device)
        t = build_paged_tables(self.prefix_len, n, self.prefix_table, self.free_pages, self.num_free,
                               page_size=self.page_size, num_tokens=int(num_tokens))
        self.prefix_len.copy_(t.context_lens)
        self.num_free.copy_(t.num_free)
        self._prefix_tokens = int(num_tokens)
        return t

    def plan(self, new_lens: torch.Tensor, num_tokens: int) -> PagedTables:
        """Pages and slots for ``new_lens[b]`` more tokens of each request slot (see
        ``build_paged_tables``); lengths and the free stack move on.  Positions count from the
        prefix's end."""
        t = build_paged_tables(self.context_lens, new_lens, self.block_tables, self.free_pages, self.num_free,
                               page_size=self.page_size, num_tokens=num_tokens, position_base=self._prefix_tokens)
        self._planned = True
        self.context_lens.copy_(t.context_lens)
        self.num_free.copy_(t.num_free)
        return t

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, tables: PagedTables,
              routes: Optional[torch.Tensor] = None) -> None:
        """The planned tokens' K/V rows (T, Hkv, D) of one layer; ``routes`` (T, H, TD): each page takes
        the routing vector of its last new token."""
        paged_kv_write(k, v, tables.slot_mapping, self.k_cache[layer], self.v_cache[layer], routes=routes,
                       router_indices=self.router[layer] if routes is not None else None)

    def decode(self, layer: int, q: torch.Tensor, q_routes: torch.Tensor, req_depth: int, local_blocks: int = 1,
               sink_block: bool = True, return_lse: bool = False):
        """``ultrametric_prefix_decode`` of one query per request slot, q (max_requests, H, D)."""
        return ultrametric_prefix_decode(q, self.k_cache[layer], self.v_cache[layer], self.prefix_table[0],
                                         self.prefix_len, self.block_tables, self.context_lens, self.router[layer],
                                         q_routes, req_depth, local_blocks=local_blocks, sink_block=sink_block,
                                         return_lse=return_lse)

    def finish(self, finished: torch.Tensor) -> None:
        """Free the pages of every request slot with ``finished[b]`` (bool)."""
        ctx, nf = release_paged_requests(finished, self.context_lens, self.block_tables, self.free_pages, self.num_free,
                                         page_size=self.page_size)
        self.context_lens.copy_(ctx)
        self.num_free.copy_(nf)
