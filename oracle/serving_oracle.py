"""CPU restatement of the serving-step operators: tables and slots in plain integers, ragged
writes row by row, and the shared-prefix decode in 64 bits, one (request, head) at a time over
the joined page list (the page rule of ``src/ultrametric/kernel_decode.py:79-89``)."""

from __future__ import annotations

import math

import torch


def build_tables(ctx, new, table, free, num_free, page, rows, base=0):
    """Lists of ints (``table``: list of lists, changed in place).  Returns slots, request ids,
    positions, cu, new lengths, new stack height, refused requests."""
    B, L = len(ctx), len(table[0]) if table else 0
    num_free = max(0, min(num_free, len(free)))
    slots, rids, pos = [-1] * rows, [-1] * rows, [0] * rows
    cu, ctx_out, refused = [0], list(ctx), []
    taken_sum, used = 0, 0
    for b in range(B):
        n = max(new[b], 0)
        cu.append(cu[-1] + n)
        old = -(-max(ctx[b], 0) // page)
        total = -(-(max(ctx[b], 0) + n) // page)
        ok = ctx[b] >= 0 and new[b] >= 0 and total <= L and cu[-1] <= rows
        need = total - old if ok else 0
        taken_sum += need
        fits = ok and (need == 0 or taken_sum <= num_free)
        if fits:
            for j in range(need):
                table[b][old + j] = free[num_free - 1 - (taken_sum - need + j)]
            ctx_out[b] = ctx[b] + n
            used = max(used, taken_sum if need else 0)
        else:
            refused.append(b)
        for i in range(n):
            t = cu[b] + i
            if t >= rows:
                break
            p = max(ctx[b], 0) + i
            rids[t], pos[t] = b, base + p
            if fits:
                slots[t] = table[b][p // page] * page + p % page
    return slots, rids, pos, cu, ctx_out, num_free - used, refused


def release(finished, ctx, table, free, num_free, page):
    """``free`` (a list of the stack's whole capacity) is changed in place."""
    ctx_out, top = list(ctx), num_free
    pushed = 0
    for b, done in enumerate(finished):
        if not done:
            continue
        pages = -(-max(ctx[b], 0) // page)
        if ctx[b] < 0 or pages > len(table[b]):
            continue
        pushed += pages
        if pages and num_free + pushed > len(free):
            continue
        for j in range(pages):
            free[num_free + pushed - pages + j] = table[b][j]
        top = num_free + pushed if pages else top
        ctx_out[b] = 0
    return ctx_out, top


def write_rows(k, v, slots, k_cache, v_cache, routes=None, router=None):
    page = k_cache.shape[2]
    for t, s in enumerate(slots.tolist()):
        if s < 0 or s >= k_cache.shape[0] * page:
            continue
        k_cache[s // page, :, s % page] = k[t]
        v_cache[s // page, :, s % page] = v[t]
        if routes is not None:
            router[s // page] = routes[t]


def prefix_decode(q, k_cache, v_cache, prefix_pages, prefix_len, block_tables, ctx, router, q_router, depth,
                  local_blocks=0, sink_block=False):
    """64-bit result: out, lse and weight = sum p |v| (for error bounds), each attended token a key."""
    B, H, D = q.shape
    P, Hkv, page, _ = k_cache.shape
    out, lse = torch.zeros(B, H, D, dtype=torch.float64), torch.full((B, H), -math.inf, dtype=torch.float64)
    weight = torch.zeros_like(out)
    for b in range(B):
        pages, valid = [], []
        for ids, n in ((prefix_pages.tolist(), int(prefix_len)), (block_tables[b].tolist(), int(ctx[b]))):
            n = max(0, min(n, len(ids) * page))
            for i in range(-(-n // page)):
                pages.append(ids[i])
                valid.append(min(page, n - i * page))
        for h in range(H):
            g = h // (H // Hkv)
            ks, vs = [], []
            for i, (ph, n) in enumerate(zip(pages, valid)):
                if not 0 <= ph < P:
                    continue
                hit = bool((router[ph, h, :depth] == q_router[b, h, :depth]).all())
                if hit or (sink_block and i == 0) or i >= len(pages) - local_blocks:
                    ks.append(k_cache[ph, g, :n].double())
                    vs.append(v_cache[ph, g, :n].double())
            if not ks:
                continue
            kk, vv = torch.cat(ks), torch.cat(vs)
            z = kk @ q[b, h].double() / math.sqrt(D)
            lse[b, h] = torch.logsumexp(z, 0)
            w = torch.softmax(z, 0)
            out[b, h], weight[b, h] = w @ vv, w @ vv.abs()
    return out, lse, weight
