"""The serving-step operators on a paged, routed K/V cache, as they are timed and compared.

Three operators, in the order in which a serving step calls them:

* ``tables``: block tables and slot map of a ragged batch of new tokens, from request lengths
  (``build_paged_tables``), once per step;
* ``write``: the new tokens' K/V rows scattered into the cache by the slot map, with the touched
  pages' routing vectors (``paged_kv_write``), once per layer and step;
* ``prefix``: routed decode of a batch whose requests share a long prefix
  (``ultrametric_prefix_decode``), once per layer and step.

Each case is run either in its plain form (elementary torch operations, 32-bit arithmetic,
rounded once) or, with ``own`` set, through the package's public entry points.
"""

import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _package():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparse-ai_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import ultrametric

    return ultrametric


# ----------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------
def _tables(name, requests, tokens, page, ctx_hi, pad):
    """requests: rows of the block table; tokens: new tokens of the step over all of them;
    pad: rows of the flat batch past the last token; ctx_hi: longest context before the step."""
    return dict(name=name, op="tables", requests=requests, tokens=tokens, page=page, ctx_hi=ctx_hi, pad=pad)


def _write(name, tokens, kv_heads, head_dim, page, dtype, heads, levels, run, pad):
    """run: new tokens per request (consecutive rows of its pages); levels: routing levels, 0
    for a cache without routes; pad: rows with slot -1 at the end."""
    return dict(name=name, op="write", tokens=tokens, kv_heads=kv_heads, head_dim=head_dim, page=page,
                dtype=dtype, heads=heads, levels=levels, run=run, pad=pad)


def _prefix(name, requests, heads, kv_heads, head_dim, dtype, page, prefix, own_lo, own_hi, depth, local, sink,
            lse=False):
    """prefix: shared tokens; own_lo..own_hi: each request's own tokens; depth: routing levels
    that must agree (0: every page is attended)."""
    return dict(name=name, op="prefix", requests=requests, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                dtype=dtype, page=page, prefix=prefix, own_lo=own_lo, own_hi=own_hi, depth=depth, local=local,
                sink=sink, lse=lse)


def listed():
    return [
        # one decode step of a 64-request batch: a token each
        _tables("tables_step", 64, 61, 64, 32768, 3),
        # a step that admits many ragged prompts beside running requests
        _tables("tables_prompts", 256, 120001, 16, 8192, 1000),
        # the writes of a decode step: one token per request, with the tail pages' routes
        _write("write_step", 64, 8, 128, 64, "bf16", 32, 6, 1, 0),
        # a batch of ragged prompts, padded to a fixed number of rows
        _write("write_prompts", 32768, 8, 128, 64, "bf16", 32, 6, 1477, 500),
        # 32-bit cache of a small model with an odd number of heads and a short page
        _write("write_small_model", 3001, 3, 80, 16, "fp32", 12, 0, 211, 5),
        # an interactive session: two requests on a short prompt, latency alone
        _prefix("prefix_pair", 2, 8, 2, 64, "fp16", 16, 203, 0, 9, 0, 0, False),
        # chat serving under one system prompt that ends inside a page
        _prefix("prefix_chat", 32, 32, 8, 128, "bf16", 64, 4133, 1, 512, 0, 0, False),
        # the routed decode batch (64 requests, depth 4, sink and newest page) with most of each
        # context shared
        _prefix("prefix_routed", 64, 32, 8, 128, "bf16", 64, 24576, 64, 4096, 4, 1, True, True),
        # many samples drawn over one long document: the largest batch
        _prefix("prefix_wide", 256, 32, 8, 128, "bf16", 64, 32768, 1, 768, 0, 0, False),
        # one KV head for 16 query heads, short pages, an odd batch
        _prefix("prefix_one_kv_head", 23, 16, 1, 128, "fp16", 32, 9001, 0, 300, 1, 1, True),
        # 32-bit cache with heads of 80
        _prefix("prefix_fp32", 5, 12, 12, 80, "fp32", 16, 1000, 0, 100, 1, 0, True, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "write", "prefix", "prefix"])
    if op == "tables":
        c = _tables("", _log(rng, 1, 700), 0, rng.choice([16, 32, 64, 128]), _log(rng, 16, 32768), rng.randrange(0, 300))
        c["tokens"] = max(1, min(120000, c["requests"] * _log(rng, 1, 2000)))
    elif op == "write":
        run = _log(rng, 1, 4000)
        c = _write("", max(run, _log(rng, 1, 32000)), rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 80, 96, 128]),
                   rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "fp16", "fp32"]), 0, rng.choice([0, 4, 6]), run,
                   rng.randrange(0, 64))
        c["heads"] = c["kv_heads"] * rng.choice([1, 2, 4])
        if c["dtype"] == "fp32":
            c["tokens"] = max(run, c["tokens"] // 2)
    else:
        kv = rng.choice([1, 2, 4, 8])
        own_hi = _log(rng, 1, 1500)
        c = _prefix("", _log(rng, 1, 256), kv * rng.choice([1, 2, 4, 8]), kv, rng.choice([64, 80, 96, 128, 128]),
                    rng.choice(["bf16", "bf16", "fp16"]), rng.choice([16, 32, 64, 128]), _log(rng, 1, 32000),
                    rng.randrange(0, own_hi + 1), own_hi, rng.choice([0, 0, 1, 2, 4]), rng.randrange(0, 3),
                    rng.random() < 0.5, rng.random() < 0.3)
        if rng.random() < 0.1:  # a 32-bit cache serves small batches
            c.update(dtype="fp32", requests=min(c["requests"], 8), prefix=min(c["prefix"], 2000), own_hi=min(own_hi, 200),
                     own_lo=min(c["own_lo"], own_hi, 200))
        # no dearer than the largest listed batch
        most = 256 * 32 * 33000
        while c["requests"] * c["heads"] * (c["prefix"] + c["own_hi"]) > most:
            c["requests"] = (c["requests"] + 1) // 2
    del c["name"]
    return c


# ----------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------
def _ragged(rng, n, total):
    """n lengths that sum to total, none above 8 times the mean, about a tenth of them 0 where
    there is a choice."""
    if n >= total:
        at = set(rng.sample(range(n), total))
        return [int(i in at) for i in range(n)]
    w = [0.0 if rng.random() < 0.1 else rng.uniform(0.1, 2.0) for _ in range(n)]
    s = sum(w)
    if s == 0.0:
        w, s = [1.0] * n, float(n)
    lens = [int(total * x / s) for x in w]
    for i in range(total - sum(lens)):
        lens[i] += 1
    return lens


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    c = case
    if c["op"] == "tables":
        B, p = c["requests"], c["page"]
        new = _ragged(rng, B, c["tokens"])
        ctx = [0 if rng.random() < 0.2 else rng.randrange(0, c["ctx_hi"] + 1) for _ in range(B)]
        have = [-(-x // p) for x in ctx]
        need = [-(-(x + n) // p) - h for x, n, h in zip(ctx, new, have)]
        width = -(-(c["ctx_hi"] + 8 * -(-c["tokens"] // B)) // p)
        total = sum(have) + sum(need) + 17
        perm = torch.randperm(total, generator=gen, device=DEV).to(torch.int32)
        off = [0] * B
        run_ = 0
        for i in range(B):
            off[i] = run_
            run_ += have[i]
        col = torch.arange(width, device=DEV)
        inside = col[None] < _i32(have)[:, None]
        at = torch.where(inside, _i32(off)[:, None] + col[None], 0)
        bt = torch.where(inside, perm[at], 0).to(torch.int32).contiguous()
        free = torch.zeros(total, dtype=torch.int32, device=DEV)
        free[: total - run_] = perm[run_:]
        return dict(c, ctx=_i32(ctx), new=_i32(new), bt=bt, free=free, num_free=_i32([total - run_]),
                    rows=c["tokens"] + c["pad"])
    dt = _DT[c["dtype"]]
    Hkv, D, p, H = c["kv_heads"], c["head_dim"], c["page"], c["heads"]
    if c["op"] == "write":
        T, run_ = c["tokens"], c["run"]
        slots, next_page = [], 0
        pages = -(-T // run_) * (-(-run_ // p) + 1) + 3
        order = torch.randperm(pages, generator=gen, device=DEV).tolist()
        left = T
        while left:
            n = min(run_, left)
            pos = rng.randrange(0, p)  # where the request's tail page stood
            for _ in range(-(-(pos + n) // p)):
                take = min(p - pos, n)
                slots.extend(range(order[next_page] * p + pos, order[next_page] * p + pos + take))
                next_page, pos, n, left = next_page + 1, 0, n - take, left - take
        slots += [-1] * c["pad"]
        R = T + c["pad"]
        # K and V rows are slices of the projection's packed output, as a model's layer has them
        kv = torch.randn(R, 2 * Hkv, D, generator=gen, device=DEV, dtype=torch.float32).to(dt)
        s = dict(c, k=kv[:, :Hkv], v=kv[:, Hkv:], slots=torch.tensor(slots, dtype=torch.int64, device=DEV),
                 kc=torch.zeros(pages, Hkv, p, D, device=DEV, dtype=dt), vc=torch.zeros(pages, Hkv, p, D, device=DEV, dtype=dt),
                 routes=None, router=None)
        if c["levels"]:
            s["routes"] = torch.randint(0, 2, (R, H, c["levels"]), generator=gen, device=DEV, dtype=torch.int32)
            s["router"] = torch.zeros(pages, H, c["levels"], device=DEV, dtype=torch.int32)
        return s
    B, Lp = c["requests"], -(-c["prefix"] // p)
    ctx = [rng.randint(c["own_lo"], c["own_hi"]) for _ in range(B)]
    width = max(1, -(-c["own_hi"] // p))
    pages = Lp + B * width + 2
    perm = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    kc = torch.randn(pages, Hkv, p, D, generator=gen, device=DEV, dtype=dt if dt != torch.float32 else None)
    vc = torch.randn(pages, Hkv, p, D, generator=gen, device=DEV, dtype=dt if dt != torch.float32 else None)
    TD = max(1, c["depth"] + 2)
    # the query rows are a slice of the projection's packed output
    q = torch.randn(B, H + 2 * Hkv, D, generator=gen, device=DEV).to(dt)[:, :H]
    return dict(c, q=q, kc=kc, vc=vc, prefix_pages=perm[:Lp].contiguous(), bt=perm[Lp:Lp + B * width].view(B, width).contiguous(),
                ctx=_i32(ctx), ri=torch.randint(0, 2, (pages, H, TD), generator=gen, device=DEV, dtype=torch.int32),
                qri=torch.randint(0, 2, (B, H, TD), generator=gen, device=DEV, dtype=torch.int32))


# ----------------------------------------------------------------------------------------
# plain forms
# ----------------------------------------------------------------------------------------
def _plain_tables(s):
    p, rows = s["page"], s["rows"]
    ctx, new, bt, free, nf = s["ctx"].long(), s["new"].long(), s["bt"], s["free"], s["num_free"].long()
    B, L = bt.shape
    cu = torch.zeros(B + 1, dtype=torch.int64, device=DEV)
    cu[1:] = torch.cumsum(new, 0)
    old, tot = (ctx + p - 1) // p, (ctx + new + p - 1) // p
    ok = (tot <= L) & (cu[1:] <= rows)
    need = torch.where(ok, tot - old, 0)
    incl = torch.cumsum(need, 0)
    fits = ok & ((need == 0) | (incl <= nf))
    first = incl - need
    col = torch.arange(L, device=DEV)[None]
    fresh = (col >= old[:, None]) & (col < tot[:, None]) & fits[:, None]
    taken = torch.clamp(nf - 1 - (first[:, None] + col - old[:, None]), 0, free.numel() - 1)
    table = torch.where(fresh, free[taken], bt)
    t = torch.arange(rows, device=DEV)
    live = t < cu[B]
    rid = torch.clamp(torch.searchsorted(cu[1:], t, right=True), max=B - 1)
    pos = ctx[rid] + t - cu[rid]
    page = table[rid, torch.clamp(pos // p, max=L - 1)].long()
    slots = torch.where(live & fits[rid], page * p + pos % p, -1)
    used = torch.where(fits & (need > 0), incl, 0).max()
    return dict(block_tables=table, slot_mapping=slots, request_ids=torch.where(live, rid, -1).int(),
                positions=torch.where(live, pos, 0).int(), cu_new_lens=cu.int(),
                context_lens=torch.where(fits, ctx + new, ctx).int(), num_free=(nf - used).int())


def _plain_write(s):
    p, n = s["page"], s["tokens"]  # the rows past n have no slot
    slots = s["slots"][:n]
    page, off = slots // p, slots % p
    s["kc"][page, :, off] = s["k"][:n]
    s["vc"][page, :, off] = s["v"][:n]
    if s["routes"] is None:
        return dict(k_cache=s["kc"], v_cache=s["vc"])
    # every token of a page writes the routes of the page's last one
    at = torch.arange(n, device=DEV)
    last = torch.ones(n, dtype=torch.bool, device=DEV)
    last[:-1] = page[1:] != page[:-1]
    upto = torch.where(last, at, n).flip(0).cummin(0).values.flip(0)
    s["router"][page] = s["routes"][upto]
    return dict(k_cache=s["kc"], v_cache=s["vc"], router=s["router"])


def _plain_prefix(s):
    q, p, r = s["q"], s["page"], s["depth"]
    B, H, D = q.shape
    Hkv = s["kv_heads"]
    G, Lp, Lo = H // Hkv, s["prefix_pages"].numel(), s["bt"].shape[1]
    scale = 1.0 / math.sqrt(D)
    pp, bt = s["prefix_pages"].long(), s["bt"].long()
    qg = q.float().reshape(B, Hkv, G, D)
    own_pages = (s["ctx"] + p - 1) // p
    total = Lp + own_pages  # logical pages of each request
    # attended pages of (request, head): prefix (B, Lp, H), own (B, Lo, H)
    want = s["qri"][:, None, :, :r]
    lp, lo = torch.arange(Lp, device=DEV), Lp + torch.arange(Lo, device=DEV)
    on_p = (s["ri"][pp][None, :, :, :r] == want).all(-1)
    on_o = (s["ri"][bt][:, :, :, :r] == want).all(-1)
    on_p = on_p | (lp[None] >= total[:, None] - s["local"])[..., None]
    on_o = on_o | (lo[None] >= total[:, None] - s["local"])[..., None]
    if s["sink"]:
        on_p = on_p | (lp == 0)[None, :, None]
        on_o = on_o | (lo == 0)[None, :, None]
    tok_p = torch.arange(Lp * p, device=DEV) < s["prefix"]
    tok_o = torch.arange(Lo * p, device=DEV)[None] < s["ctx"][:, None]
    see_p = on_p.transpose(1, 2).repeat_interleave(p, 2) & tok_p  # (B, H, Lp * p)
    see_o = on_o.transpose(1, 2).repeat_interleave(p, 2) & tok_o[:, None]
    # the prefix once for all requests, per KV head
    kp = s["kc"][pp].float().transpose(0, 1).reshape(Hkv, Lp * p, D)
    vp = s["vc"][pp].float().transpose(0, 1).reshape(Hkv, Lp * p, D)
    rows = qg.transpose(0, 1).reshape(Hkv, B * G, D)
    sp = torch.matmul(rows, kp.transpose(1, 2)).view(Hkv, B, G, Lp * p).transpose(0, 1).reshape(B, H, Lp * p) * scale
    ko = s["kc"][bt].float().transpose(1, 2).reshape(B, Hkv, Lo * p, D)
    vo = s["vc"][bt].float().transpose(1, 2).reshape(B, Hkv, Lo * p, D)
    so = torch.matmul(qg, ko.transpose(2, 3)).reshape(B, H, Lo * p) * scale
    sp = torch.where(see_p, sp, -math.inf)
    so = torch.where(see_o, so, -math.inf)
    m = torch.maximum(sp.amax(-1), so.amax(-1))
    ref = torch.where(m == -math.inf, 0.0, m)[..., None]
    sp, so = torch.exp(sp - ref), torch.exp(so - ref)
    total_w = sp.sum(-1) + so.sum(-1)
    acc = torch.matmul(sp.view(B, Hkv, G, Lp * p).transpose(0, 1).reshape(Hkv, B * G, Lp * p), vp)
    acc = acc.view(Hkv, B, G, D).transpose(0, 1) + torch.matmul(so.view(B, Hkv, G, Lo * p), vo)
    out = acc.reshape(B, H, D) / torch.where(total_w == 0, 1.0, total_w)[..., None]
    lse = m + torch.log(total_w)
    return (out.to(q.dtype), lse) if s["lse"] else out.to(q.dtype)


def run(state):
    s = state
    if s["op"] == "tables":
        if not own:
            return _plain_tables(s)
        t = _package().build_paged_tables(s["ctx"], s["new"], s["bt"], s["free"], s["num_free"], page_size=s["page"],
                                          num_tokens=s["rows"])
        return dict(t._asdict(), block_tables=s["bt"])
    if s["op"] == "write":
        if not own:
            return _plain_write(s)
        _package().paged_kv_write(s["k"], s["v"], s["slots"], s["kc"], s["vc"], routes=s["routes"], router_indices=s["router"])
        out = dict(k_cache=s["kc"], v_cache=s["vc"])
        return out if s["routes"] is None else dict(out, router=s["router"])
    if not own:
        return _plain_prefix(s)
    return _package().ultrametric_prefix_decode(
        s["q"], s["kc"], s["vc"], s["prefix_pages"], s["prefix"], s["bt"], s["ctx"], s["ri"], s["qri"], s["depth"],
        local_blocks=s["local"], sink_block=s["sink"], return_lse=s["lse"])


# ----------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "tables":
        rows, B = c["tokens"] + c["pad"], c["requests"]
        fresh = c["tokens"] / c["page"]
        # lengths in and out, pages taken and listed, tail entries; slot, request and position per row
        return {"bytes": B * 20 + fresh * 8 + B * 4 + rows * 16, "flops": 0}
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "write":
        row = c["kv_heads"] * c["head_dim"] * size
        runs = -(-c["tokens"] // c["run"])
        pages = runs * (1 + (c["run"] - 1) / c["page"])
        return {"bytes": c["tokens"] * 4 * row + (c["tokens"] + c["pad"]) * 8 + pages * 2 * 4 * c["heads"] * c["levels"],
                "flops": 0}
    B, H, Hkv, D, r = c["requests"], c["heads"], c["kv_heads"], c["head_dim"], c["depth"]
    G, own_mean, hit = H // Hkv, (c["own_lo"] + c["own_hi"]) / 2, 0.5 ** r
    forced = min(own_mean, c["local"] * c["page"]) if r else 0
    seen = 1 - (1 - hit) ** (B * G)  # share of the prefix that some row of a KV head attends
    seen_own = 1 - (1 - hit) ** G
    pages = -(-c["prefix"] // c["page"]) + B * (own_mean / c["page"] + 0.5)
    kv = 2 * D * size * Hkv
    tokens = c["prefix"] * hit + min(own_mean, own_mean * hit + forced)
    return {"bytes": c["prefix"] * seen * kv + B * min(own_mean, own_mean * seen_own + forced) * kv
            + 2 * B * H * D * size + pages * (4 + H * r * 4) + B * H * r * 4,
            "flops": 4 * D * H * B * tokens}


# ----------------------------------------------------------------------------------------
# the definition in 64 bits
# ----------------------------------------------------------------------------------------
def exact(case, seed):
    """Decode, request by request: its pages in order, each page's tokens, a softmax over the
    attended ones.  Writes, by rows of the flattened pool.  Tables are whole numbers."""
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    if case["op"] == "write":
        rows = s["slots"][s["slots"] >= 0]
        want = {"k_cache": (s["kc"], s["k"]), "v_cache": (s["vc"], s["v"])}
        for name in want:
            pages, heads, p, D = want[name][0].shape
            flat = torch.zeros(pages * p, heads, D, dtype=torch.float64, device=DEV)
            flat.index_copy_(0, rows, want[name][1][:rows.numel()].double())
            want[name] = flat.view(pages, p, heads, D).permute(0, 2, 1, 3)
        return want if s["routes"] is None else dict(want, router=None)
    B, H, D = s["q"].shape
    p, r, G = s["page"], s["depth"], H // s["kv_heads"]
    Lp = s["prefix_pages"].numel()
    out = torch.zeros(B, H, D, dtype=torch.float64, device=DEV)
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device=DEV)
    head_kv = torch.arange(H, device=DEV) // G
    lens = s["ctx"].tolist()
    kp = s["kc"][s["prefix_pages"].long()].double().permute(1, 0, 2, 3).reshape(s["kv_heads"], Lp * p, D)[:, :s["prefix"]]
    vp = s["vc"][s["prefix_pages"].long()].double().permute(1, 0, 2, 3).reshape(s["kv_heads"], Lp * p, D)[:, :s["prefix"]]
    for b in range(B):
        n_own = -(-lens[b] // p)
        own_ids = s["bt"][b, :n_own].long()
        ids = torch.cat([s["prefix_pages"].long(), own_ids])
        n = ids.numel()
        if n == 0:
            continue
        page_on = torch.ones(H, n, dtype=torch.bool, device=DEV)
        for level in range(r):
            page_on &= (s["ri"][ids][:, :, level] == s["qri"][b, :, level][None]).T
        if s["local"] > 0:
            page_on[:, max(0, n - s["local"]):] = True
        if s["sink"]:
            page_on[:, 0] = True
        k = torch.cat([kp, s["kc"][own_ids].double().permute(1, 0, 2, 3).reshape(s["kv_heads"], n_own * p, D)[:, :lens[b]]], 1)
        v = torch.cat([vp, s["vc"][own_ids].double().permute(1, 0, 2, 3).reshape(s["kv_heads"], n_own * p, D)[:, :lens[b]]], 1)
        page_of_token = torch.cat([torch.arange(s["prefix"], device=DEV) // p, Lp + torch.arange(lens[b], device=DEV) // p])
        for g in range(s["kv_heads"]):
            mine = (head_kv == g).nonzero().flatten()
            z = s["q"][b, mine].double() @ k[g].T / math.sqrt(D)
            z = z.masked_fill(~page_on[mine][:, page_of_token], -math.inf)
            lse[b, mine] = torch.logsumexp(z, 1)
            w = torch.softmax(z, 1)
            w = torch.where(torch.isnan(w), 0.0, w)
            out[b, mine] = w @ v[g]
    return (out, lse) if s["lse"] else out
