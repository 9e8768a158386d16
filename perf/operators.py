"""Measured cases of the operators that serve several requests over one prompt.

Five operators of ``oscar_new_b200.kernels``, each with its plain form (elementary torch
operations in 32 bits, rounded once at the end):

* ``qk_norm_rope``: root-mean-square norm of every query and key head and the position
  rotation of its first dimensions;
* ``fork_requests``: a request's cache pages forked for another request (shared full pages,
  private first and partial last page);
* ``resize_requests``: requests admitted, grown and released on the page pool;
* ``compact_pages``: live pages moved to the lowest page numbers;
* ``decode_attention`` with a shared prefix: one decode / verify step of a batch whose
  requests share long prefixes, on the INT2 history and the BF16 window of the paged cache.

Cache format: a page holds ``block`` tokens.  In the K stripe a token slot of a KV head has
160 bytes: 64 bytes of 2-bit key codes (four to a byte, lowest bits first), fp16 scale and
zero, then the same 68 bytes for the value; the element is bf16(code * scale + zero).  The V
stripe of a request's first page holds its BF16 window: ``sink`` tokens and a ring of
``recent + query`` tokens, [index, K / V, head, 256].  Tables are in 128-token blocks.
"""

import math

import torch

own = False

DEV = "cuda"
DIM = 256


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------


def listed():
    return [
        # a decode step of one request: latency
        dict(name="norm rope decode 1", op="norm_rope", tokens=1, q_heads=24, kv_heads=4, rotary=64, interleaved=False,
             gated=True, offset=1.0, weight="bf16", table="fp32", positions=32768),
        # a verify step of 32 requests x 4 tokens, full rotary width in adjacent pairs, plain fp32 weights
        dict(name="norm rope verify 128", op="norm_rope", tokens=128, q_heads=8, kv_heads=1, rotary=256,
             interleaved=True, gated=False, offset=0.0, weight="fp32", table="bf16", positions=262144),
        # a prefill chunk, queries interleaved with the gate of the output in one projection
        dict(name="norm rope prefill 16384", op="norm_rope", tokens=16384, q_heads=24, kv_heads=4, rotary=64,
             interleaved=False, gated=True, offset=1.0, weight="bf16", table="fp32", positions=32768),
        # one more answer to a medium prompt on a one-head rank
        dict(name="fork 1 to 1", op="fork", parents=1, children=1, tokens=4099, kv_heads=1, block=768, sink=64,
             recent=256, query=4),
        # parallel sampling: 60 answers over four long prompts
        dict(name="fork 4 to 60", op="fork", parents=4, children=60, tokens=32635, kv_heads=4, block=768, sink=64,
             recent=256, query=4),
        # a decode step's growth: 64 requests, a few of which need a page
        dict(name="resize grow 64", op="resize", requests=64, tokens=4000, grow=1, release=0, block=768, kv_heads=4),
        # a busy server: 192 of 512 requests end, others grow by a prefill chunk
        dict(name="resize turnover 512", op="resize", requests=512, tokens=8192, grow=2048, release=192, block=768,
             kv_heads=4),
        # a few holes left by short requests
        dict(name="compact few", op="compact", requests=8, tokens=2500, share=0, free=2, kv_heads=1, block=768,
             sink=64, recent=256, query=1),
        # half of a large pool freed, prefixes shared among the rest
        dict(name="compact half", op="compact", requests=64, tokens=6000, share=16, free=32, kv_heads=4, block=768,
             sink=64, recent=256, query=4),
        # four answers over a short prompt, 8 query heads on one KV head: latency
        dict(name="shared decode 4 x 2k", op="shared", requests=4, groups=1, prefix=2048, suffix=160, query=1,
             q_heads=8, kv_heads=1, block=768, sink=64, recent=256),
        # verify steps (4 tokens) of 24 requests over three prompts of different lengths
        dict(name="shared verify 24 x 12k", op="shared", requests=24, groups=3, prefix=12345, suffix=700, query=4,
             q_heads=24, kv_heads=4, block=768, sink=4, recent=128),
        # 64 answers over one 32K prompt
        dict(name="shared decode 64 x 32k", op="shared", requests=64, groups=1, prefix=32635, suffix=512, query=1,
             q_heads=24, kv_heads=4, block=768, sink=4, recent=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rope", "fork", "resize", "compact", "shared", "shared"])
    hq, h = rng.choice([(24, 4), (8, 1), (6, 1), (12, 2)])
    if op == "norm_rope":
        return dict(op=op, tokens=_log(rng, 1, 16000), q_heads=hq, kv_heads=h, rotary=rng.choice([32, 64, 128, 256]),
                    interleaved=rng.random() < 0.5, gated=rng.random() < 0.5, offset=rng.choice([0.0, 1.0]),
                    weight=rng.choice(["bf16", "fp32"]), table=rng.choice(["bf16", "fp32"]),
                    positions=_log(rng, 64, 262144))
    if op == "fork":
        return dict(op=op, parents=rng.randint(1, 4), children=_log(rng, 1, 48), tokens=_log(rng, 1, 24000), kv_heads=h,
                    block=rng.choice([768, 1024]), sink=rng.choice([4, 64]), recent=rng.choice([128, 256]),
                    query=rng.choice([1, 4]))
    if op == "resize":
        n = _log(rng, 8, 512)
        return dict(op=op, requests=n, tokens=_log(rng, 1, 8192), grow=_log(rng, 1, 2048),
                    release=rng.randint(0, n // 2), block=rng.choice([128, 768, 1024]), kv_heads=h)
    if op == "compact":
        n = rng.randint(2, 64)
        return dict(op=op, requests=n, tokens=_log(rng, 1, 5000), share=rng.randint(0, n // 3),
                    free=rng.randint(1, n // 2), kv_heads=h, block=rng.choice([768, 1024]), sink=rng.choice([4, 64]),
                    recent=rng.choice([128, 256]), query=rng.choice([1, 4]))
    n = rng.randint(2, 40)
    return dict(op=op, requests=n, groups=rng.randint(1, max(1, n // 3)), prefix=_log(rng, 1, 16000),
                suffix=_log(rng, 1, 700), query=rng.choice([1, 1, 2, 4]), q_heads=hq, kv_heads=h,
                block=rng.choice([768, 1024]), sink=rng.choice([4, 64]), recent=rng.choice([128, 256]))


# ---------------------------------------------------------------------------------------
# sizes that a case's numbers imply (the same for every seed)
# ---------------------------------------------------------------------------------------


def _lengths(count, longest):
    """`count` ragged lengths of at most `longest`, the first of them that long."""
    return [max(1, longest - (i * 7919) % max(1, longest // 3)) for i in range(count)]


def _window_tokens(c):
    return c["sink"] + c["recent"] + c["query"]


def _pages(tokens, block):
    return -(-tokens // block)


def _shared_sizes(c):
    """Group of each request, prefix length of each group, sequence length of each request."""
    base, more = divmod(c["requests"], c["groups"])
    sizes = [base + (i < more) for i in range(c["groups"])]
    of = [g for g, s in enumerate(sizes) for _ in range(s)]
    prefix = _lengths(c["groups"], c["prefix"])
    own_tokens = [(i * 7919 + 13) % c["suffix"] for i in range(c["requests"])]
    seq = [prefix[g] + t + c["query"] for g, t in zip(of, own_tokens)]
    return of, prefix, seq


def work(case):
    c, op = case, case["op"]
    if op == "norm_rope":
        rows = c["tokens"] * (c["q_heads"] + c["kv_heads"])
        wide = {"bf16": 2, "fp32": 4}
        used = min(c["tokens"], c["positions"]) * c["rotary"] * wide[c["table"]]
        return {"bytes": rows * DIM * 4 + c["tokens"] * 8 + 2 * DIM * wide[c["weight"]] + used,
                "flops": rows * (4 * DIM + 3 * c["rotary"])}
    if op == "fork":
        lens = _lengths(c["parents"], c["tokens"])
        slot, window = c["kv_heads"] * 160, _window_tokens(c) * c["kv_heads"] * 1024
        read = write = 0
        for i, n in enumerate(lens):
            first, last = min(n, c["block"]), n % c["block"] if n > c["block"] else 0
            part = (first + last) * slot + window
            kids = c["children"] // c["parents"] + (i < c["children"] % c["parents"])
            read += part if kids else 0
            write += kids * part
        columns = _pages(c["tokens"], c["block"]) * (c["block"] // 128)
        return {"bytes": read + write + c["children"] * columns * 8, "flops": 0}
    if op == "resize":
        columns = c["block"] // 128
        freed = sum(_pages(n, c["block"]) for n in _lengths(c["requests"], c["tokens"])[: c["release"]])
        kept = c["requests"] - c["release"]
        return {"bytes": freed * (columns * 8 + 8) + kept * (16 + _pages(c["grow"], c["block"]) * (columns * 4 + 8))
                + _resize_pool(c) * 4, "flops": 0}
    if op == "compact":
        lens, gone = _compact_sizes(c)
        slot, window = c["kv_heads"] * 160, _window_tokens(c) * c["kv_heads"] * 1024
        live = sum(1 + max(0, _pages(n, c["block"]) - 1) for i, n in enumerate(lens) if i not in gone)
        total = sum(_pages(n, c["block"]) for n in lens)
        moved = live * (total - live) / max(1, total)  # pages expected above the live count, at random places
        kept = [n for i, n in enumerate(lens) if i not in gone]
        held = sum(n for n in kept) * slot + len(kept) * window
        return {"bytes": 2 * moved * held / max(1, live) + 8 * total, "flops": 0}
    of, prefix, seq = _shared_sizes(c)
    q, hq, h, g = c["query"], c["q_heads"], c["kv_heads"], c["q_heads"] // c["kv_heads"]
    shared = own_history = raw = 0
    rows_flops = 0
    for k, p in enumerate(prefix):
        members = [s for s, o in zip(seq, of) if o == k]
        top = max(0, min([p] + [s - q - c["recent"] for s in members]) - c["sink"])
        shared += top
        for s in members:
            hist = max(0, s - q - c["recent"] - c["sink"])
            own_history += hist - top
            raw += s - hist
            rows_flops += 4 * q * hq * DIM * s
    return {"bytes": (shared + own_history) * h * 136 + raw * h * 1024 + 3 * c["requests"] * q * hq * 512
            + 3 * c["requests"] * q * h * 1024 + DIM * DIM * 2,
            "flops": rows_flops + 2 * c["requests"] * q * hq * DIM * DIM}


def _resize_pool(c):
    lens = _lengths(c["requests"], c["tokens"])
    return 2 + sum(_pages(n, c["block"]) for n in lens) + c["requests"] * _pages(c["grow"], c["block"])


def _compact_sizes(c):
    lens = _lengths(c["requests"], c["tokens"])
    return lens, set(range(0, 2 * c["free"], 2)) if 2 * c["free"] <= c["requests"] else set(range(c["free"]))


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, device=DEV, generator=gen)


def _int(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _slots(gen, tokens, heads):
    """Packed 160-byte slots of Gaussian vectors clipped and quantised to two bits."""
    out = torch.zeros(tokens, heads, 160, dtype=torch.uint8, device=DEV)
    for at in (0, 68):
        x = _randn(gen, tokens, heads, DIM)
        top = 1.8 + 0.1 * _randn(gen, tokens, heads, 1)
        zero = (-top + 0.05 * _randn(gen, tokens, heads, 1)).half()
        scale = (2 * top / 3).half()
        code = ((x - zero.float()) / scale.float() + 0.5).floor().clamp(0, 3).to(torch.uint8).view(tokens, heads, 64, 4)
        out[..., at: at + 64] = code[..., 0] | code[..., 1] << 2 | code[..., 2] << 4 | code[..., 3] << 6
        out[..., at + 64: at + 68] = torch.cat((scale, zero), -1).view(torch.uint8)
    return out


def _cache(pages, c):
    """[2, blocks, 128, H, 256] bf16 K and V stripes of `pages` pages, zero."""
    return torch.zeros(2, pages * (c["block"] // 128), 128, c["kv_heads"], DIM, dtype=torch.bfloat16, device=DEV)


def _history(cache, c):
    """[pages, block, H, 160] bytes of the K stripe."""
    h = c["kv_heads"]
    flat = cache[0].view(torch.uint8).view(-1, c["block"] * h * 512)
    return flat[:, : c["block"] * h * 160].unflatten(1, (c["block"], h, 160))


def _window(cache, c):
    """[pages, window tokens, 2, H, 256] bf16 of the V stripe."""
    h, w = c["kv_heads"], _window_tokens(c)
    return cache[1].view(-1, c["block"] * h * DIM)[:, : w * 2 * h * DIM].unflatten(1, (w, 2, h, DIM))


def _fill(gen, cache, c):
    """Every slot and window row of the cache with what a server would hold there."""
    hist, win = _history(cache, c), _window(cache, c)
    step = max(1, 65536 // c["block"])
    for a in range(0, hist.shape[0], step):
        part = hist[a: a + step]
        part.copy_(_slots(gen, part.shape[0] * c["block"], c["kv_heads"]).view(part.shape))
        win[a: a + step] = _randn(gen, *win[a: a + step].shape).bfloat16()


def _table(pages_of, columns, block):
    """int32 [rows, columns] of 128-token blocks from each row's page numbers."""
    per = block // 128
    t = torch.zeros(len(pages_of), columns, dtype=torch.int32)
    for i, pages in enumerate(pages_of):
        if pages:
            t[i, : len(pages) * per] = (torch.tensor(pages)[:, None] * per + torch.arange(per)).flatten().int()
    return t


def _pool_state(pages_of, lens, total, columns, block):
    """Reference counts (page 0 is never handed out), block tables and lengths."""
    refs = torch.zeros(total, dtype=torch.int32)
    refs[0] = 1
    for pages in pages_of:
        refs.index_add_(0, torch.tensor(pages, dtype=torch.int64), torch.ones(len(pages), dtype=torch.int32))
    return [refs.to(DEV), _table(pages_of, columns, block).to(DEV), _int(lens)]


def _layout(c):
    from dataclasses import replace

    from oscar_new_b200.config import OscarConfig
    from oscar_new_b200.layout import CacheLayout

    cfg = replace(OscarConfig(), sink_tokens=c.get("sink", 4), recent_tokens=c.get("recent", 64),
                  speculative_tokens=c.get("query", 1) - 1)
    return CacheLayout(c["block"], kv_heads=c["kv_heads"], config=cfg)


def _with_pool(state, c):
    """The framework's handles over the same pool: kept by a server for its whole life."""
    from oscar_new_b200.pages import PagePool

    refs, table, lens = state["pool"]
    pool = PagePool(refs.shape[0], table.shape[0], table.shape[1], _layout(c), DEV)
    pool.refcounts.copy_(refs)
    pool.block_tables.copy_(table)
    pool.seq_lens.copy_(lens)
    state["handle"], state["start"] = pool, pool.state.clone()
    if "cache" in state:
        state["views"] = pool.layout.tensor_views(state["cache"])
    return state


def prepare(case, seed):
    c, gen = case, _gen(seed)
    perm = torch.Generator().manual_seed(seed)
    if c["op"] == "norm_rope":
        n, hq, h = c["tokens"], c["q_heads"], c["kv_heads"]
        wide = 2 * DIM if c["gated"] else DIM
        fused = _randn(gen, n, hq * wide + 2 * h * DIM)
        fused = (fused * (1 + 4 * torch.rand(n, 1, device=DEV, generator=gen))).bfloat16()
        kind = {"bf16": torch.bfloat16, "fp32": torch.float32}
        centre = 1.0 - c["offset"]
        angle = torch.arange(c["positions"], dtype=torch.float64, device=DEV)[:, None] * torch.exp(
            -math.log(1e6) * torch.arange(0, c["rotary"], 2, dtype=torch.float64, device=DEV) / c["rotary"])
        return dict(c=c, query=fused[:, : hq * wide].unflatten(1, (hq, wide))[..., :DIM],
                    key=fused[:, hq * wide: hq * wide + h * DIM].unflatten(1, (h, DIM)),
                    q_weight=(centre + 0.1 * _randn(gen, DIM)).to(kind[c["weight"]]),
                    k_weight=(centre + 0.1 * _randn(gen, DIM)).to(kind[c["weight"]]),
                    positions=torch.randint(0, c["positions"], (n,), device=DEV, generator=gen),
                    table=torch.cat((angle.cos(), angle.sin()), 1).to(kind[c["table"]]))
    if c["op"] == "fork":
        lens = _lengths(c["parents"], c["tokens"])
        need = [_pages(n, c["block"]) for n in lens]
        total = 1 + sum(need) + 2 * c["children"] + 8
        order = (torch.randperm(total - 1, generator=perm) + 1).tolist()
        rows, at = [], 0
        for k in need:
            rows.append(order[at: at + k])
            at += k
        rows += [[] for _ in range(c["children"])]
        columns = max(need) * (c["block"] // 128)
        cache = _cache(total, c)
        _fill(gen, cache, c)
        state = dict(c=c, pool=_pool_state(rows, lens + [0] * c["children"], total, columns, c["block"]), cache=cache,
                     parents=_int([i % c["parents"] for i in range(c["children"])]),
                     children=_int([c["parents"] + i for i in range(c["children"])]))
        return _with_pool(state, c) if own else state
    if c["op"] == "resize":
        lens, total = _lengths(c["requests"], c["tokens"]), _resize_pool(c)
        order = (torch.randperm(total - 1, generator=perm) + 1).tolist()
        rows, at = [], 0
        for n in lens:
            rows.append(order[at: at + _pages(n, c["block"])])
            at += len(rows[-1])
        columns = _pages(c["tokens"] + c["grow"], c["block"]) * (c["block"] // 128)
        who = torch.randperm(c["requests"], generator=perm).tolist()
        gone = set(who[: c["release"]])
        state = dict(c=c, pool=_pool_state(rows, lens, total, columns, c["block"]), rows=_int(who),
                     lens=_int([0 if r in gone else lens[r] + c["grow"] for r in who]))
        return _with_pool(state, dict(c, sink=4, recent=32, query=1)) if own else state
    if c["op"] == "compact":
        lens, gone = _compact_sizes(c)
        total = 1 + sum(_pages(n, c["block"]) for n in lens)
        order = (torch.randperm(total - 1, generator=perm) + 1).tolist()
        rows, at = [], 0
        for i, n in enumerate(lens):
            rows.append(order[at: at + _pages(n, c["block"])])
            at += len(rows[-1])
            if i and i <= c["share"]:  # interior pages of a forked request belong to the one before it
                common = min(len(rows[i]), len(rows[i - 1])) - 1
                if common > 1:
                    rows[i][1:common] = rows[i - 1][1:common]
        rows = [[] if i in gone else r for i, r in enumerate(rows)]
        lens = [0 if i in gone else n for i, n in enumerate(lens)]
        columns = max(len(r) for r in rows) * (c["block"] // 128)
        cache = _cache(total, c)
        _fill(gen, cache, c)
        state = dict(c=c, pool=_pool_state(rows, lens, total, columns, c["block"]), cache=cache)
        return _with_pool(state, c) if own else state
    return _prepare_shared(c, gen, perm)


def _prepare_shared(c, gen, perm):
    of, prefix, seq = _shared_sizes(c)
    block, h, hq, q, r = c["block"], c["kv_heads"], c["q_heads"], c["query"], c["requests"]
    rows, free = [], 1
    for i, (g, s) in enumerate(zip(of, seq)):  # full interior pages of the prefix are the first member's
        first = of.index(g)
        pages = []
        for k in range(_pages(s, block)):
            if i != first and 0 < k < prefix[g] // block:
                pages.append(rows[first][k])
            else:
                pages.append(free)
                free += 1
        rows.append(pages)
    order = [0] + (torch.randperm(free - 1, generator=perm) + 1).tolist()
    rows = [[order[p] for p in pages] for pages in rows]
    table = _table(rows, max(len(p) for p in rows) * (block // 128), block)
    cache = _cache(free, c)
    hist, win = _history(cache, c), _window(cache, c)
    common = [_slots(gen, p, h) for p in prefix]
    for i, (g, s) in enumerate(zip(of, seq)):
        pages = torch.tensor(rows[i], device=DEV)
        pos = torch.arange(s, device=DEV)
        p = prefix[g]
        if i != of.index(g):  # shared pages are already filled
            pos = pos[(pos < block) | (pos >= max(1, p // block) * block)]
        data = torch.cat((common[g][pos[pos < p]], _slots(gen, int((pos >= p).sum()), h)))
        hist[pages[pos // block], pos % block] = data
        win[pages[0]] = _randn(gen, *win.shape[1:]).bfloat16()
    n = r * q
    rotation = torch.linalg.qr(_randn(gen, DIM, DIM).double())[0].float()
    state = dict(c=c, cache=cache, table=table.to(DEV), seq_lens=_int(seq), starts=_int(list(range(0, n + 1, q))),
                 counts=_int([r, n]), groups=_int(of), prefix=_int([prefix[g] for g in of]),
                 query=(_randn(gen, n, hq, DIM) * (1 + torch.rand(1, hq, 1, device=DEV, generator=gen))).bfloat16(),
                 key=_randn(gen, n, h, DIM).bfloat16(), value=_randn(gen, n, h, DIM).bfloat16(),
                 rv=rotation.bfloat16())
    state["qrot"] = (state["query"].float() @ rotation).bfloat16()
    # one task (request, first query) per request: a step of at most four queries
    state["tasks"] = torch.stack((torch.arange(r, device=DEV), torch.zeros(r, dtype=torch.int64, device=DEV)), 1).int()
    state["task_count"] = _int([r])
    if own:
        from types import SimpleNamespace

        from oscar_new_b200.config import decode_split_cap

        layout = _layout(c)
        state["layout"], state["views"] = layout, layout.tensor_views(cache)
        state["splits"] = min(16, decode_split_cap(r, h, q, n, hq))
        state["meta"] = SimpleNamespace(query_start_loc=state["starts"], seq_lens=state["seq_lens"],
                                        block_tables=state["table"], counts=state["counts"], tasks=state["tasks"],
                                        task_count=state["task_count"], num_reqs=r, max_num_reqs=r, max_query_len=q)
    return state


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------


def run(state):
    op = state["c"]["op"]
    if own:
        return _own(state, op)
    return {"norm_rope": _plain_norm_rope, "fork": _plain_fork, "resize": _plain_resize, "compact": _plain_compact,
            "shared": _plain_shared}[op](state)


def _own(s, op):
    from oscar_new_b200 import kernels

    c = s["c"]
    if op == "norm_rope":
        return kernels.qk_norm_rope(s["query"], s["key"], s["q_weight"], s["k_weight"], s["positions"], s["table"],
                                    eps=1e-6, weight_offset=c["offset"], interleaved=c["interleaved"])
    if op == "shared":
        out = torch.empty(s["query"].shape[0], c["q_heads"] * DIM, dtype=torch.bfloat16, device=DEV)
        history, window = s["views"]
        shared = kernels.prepare_shared_prefix(s["meta"], s["groups"], s["prefix"], s["layout"], c["q_heads"])
        kernels.decode_attention(s["qrot"], s["query"], s["key"], s["value"], history, window, s["meta"], s["layout"],
                                 1 / 16, s["splits"], s["rv"], out, shared=shared)
        return out, s["cache"][1].view(torch.int16)
    pool = s["handle"]
    pool.state.copy_(s["start"])  # every pass starts from the same pool
    if op == "resize":
        done = kernels.resize_requests(pool, s["rows"], s["lens"])
        return pool.refcounts, pool.block_tables, pool.seq_lens, done
    history, window = s["views"]
    if op == "fork":
        done = kernels.fork_requests(pool, s["parents"], s["children"], history, window)
        return pool.refcounts, pool.block_tables, pool.seq_lens, done, s["cache"].view(torch.int16)
    summary, moved_to = kernels.compact_pages(pool, history, window)
    return pool.refcounts, pool.block_tables, pool.seq_lens, summary, moved_to, s["cache"].view(torch.int16)


def _plain_norm_rope(s):
    c, half = s["c"], s["c"]["rotary"] // 2
    cos, sin = s["table"][s["positions"]].float()[:, None].split(half, -1)

    def rows(x, w):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (w.float() + c["offset"])
        a, b = (x[..., 0: 2 * half: 2], x[..., 1: 2 * half: 2]) if c["interleaved"] else (x[..., :half],
                                                                                            x[..., half: 2 * half])
        turned = (a * cos - b * sin, b * cos + a * sin)
        turned = torch.stack(turned, -1).flatten(-2) if c["interleaved"] else torch.cat(turned, -1)
        return torch.cat((turned, x[..., 2 * half:]), -1).bfloat16()

    return rows(s["query"], s["q_weight"]), rows(s["key"], s["k_weight"])


def _copy_pages(s, src, dst, tokens, window):
    """The first `tokens` slots of pages src to pages dst, and the window where asked."""
    c = s["c"]
    hist, win = _history(s["cache"], c), _window(s["cache"], c)
    used = torch.arange(c["block"], device=DEV)[None, :] < tokens[:, None]
    hist[dst] = torch.where(used[..., None, None], hist[src], hist[dst])
    win[dst[window]] = win[src[window]]


def _block_rows(pages, per):
    """Table columns of page numbers [rows, pages]; no page (0) is all zeros."""
    blocks = pages[..., None] * per + torch.arange(per, device=DEV)
    return torch.where(pages[..., None] > 0, blocks, 0).flatten(1).int()


def _plain_fork(s):
    c, block, per = s["c"], s["c"]["block"], s["c"]["block"] // 128
    refs, table, lens = (x.clone() for x in s["pool"])
    parents, children = s["parents"].long(), s["children"].long()
    n = lens[parents].long()
    count = (n + block - 1) // block
    partial = (n % block != 0) & (count > 1)
    need = 1 + partial.long()
    upto = need.cumsum(0)
    free = (refs == 0).nonzero().flatten()
    ok = upto <= free.numel()
    first, last = free[upto - need], free[(upto - 1).clamp(max=free.numel() - 1)]
    pages = (table[parents][:, ::per] // per).long()
    kept = torch.arange(pages.shape[1], device=DEV)[None, :]
    shared = (kept > 0) & (kept < (count - partial.long())[:, None]) & ok[:, None]
    new = torch.where(kept == 0, first[:, None], pages)
    new = torch.where(partial[:, None] & (kept == count[:, None] - 1), last[:, None], new)
    new = torch.where(kept < count[:, None], new, 0)
    refs.index_add_(0, pages[shared], torch.ones_like(pages[shared], dtype=torch.int32))
    refs[first[ok]] = 1
    refs[last[ok & partial]] = 1
    table[children[ok]] = _block_rows(new, per)[ok]
    lens[children[ok]] = n[ok].int()
    tail = ok & partial
    src = torch.cat((pages[ok, 0], pages[tail, count[tail] - 1]))
    tokens = torch.cat((n.clamp(max=block)[ok], (n % block)[tail]))
    window = torch.arange(src.numel(), device=DEV) < ok.sum()
    _copy_pages(s, src, torch.cat((first[ok], last[tail])), tokens, window)
    return refs, table, lens, ok.int(), s["cache"].view(torch.int16)


def _plain_resize(s):
    block, per = s["c"]["block"], s["c"]["block"] // 128
    refs, table, lens = (x.clone() for x in s["pool"])
    rows, want = s["rows"].long(), s["lens"].long()
    pages = (table[:, ::per] // per).long()
    had = (lens[rows].long() + block - 1) // block
    column = torch.arange(pages.shape[1], device=DEV)[None, :]
    gone = (want == 0)[:, None] & (column < had[:, None])
    refs.index_add_(0, pages[rows][gone], torch.full_like(pages[rows][gone], -1, dtype=torch.int32))
    need = ((want + block - 1) // block - had).clamp(min=0)
    upto = need.cumsum(0)
    free = (refs == 0).nonzero().flatten()
    ok = (need == 0) | (upto <= free.numel())
    fresh = (column >= had[:, None]) & (column < (had + need)[:, None]) & ok[:, None]
    at = ((upto - need)[:, None] + column - had[:, None])[fresh]
    new = pages[rows]
    new[fresh] = free[at]
    new[gone] = 0
    refs[free[at]] = 1
    table[rows] = _block_rows(new, per)
    lens[rows] = torch.where(ok, want, lens[rows].long()).int()
    return refs, table, lens, ok.int()


def _plain_compact(s):
    c, block, per = s["c"], s["c"]["block"], s["c"]["block"] // 128
    refs, table, lens = (x.clone() for x in s["pool"])
    total = refs.numel()
    number = torch.arange(total, device=DEV)
    live = (refs > 0) & (number > 0)
    count = live.sum()
    holes, movers = ((~live) & (number > 0) & (number <= count)).nonzero().flatten(), (live & (number > count)).nonzero()
    movers = movers.flatten()
    to = torch.where(live | (number == 0), number, -1)
    to[movers] = holes
    pages = (table[:, ::per] // per).long()
    column = torch.arange(pages.shape[1], device=DEV)[None, :]
    held = column < ((lens.long() + block - 1) // block)[:, None]
    tokens = (lens.long()[:, None] - column * block).clamp(max=block)
    used = torch.zeros(total, dtype=torch.int64, device=DEV).scatter_reduce(0, pages[held], tokens[held], "amax")
    owner = torch.zeros(total, dtype=torch.bool, device=DEV)
    owner[pages[:, 0][lens > 0]] = True
    _copy_pages(s, movers, holes, used[movers], owner[movers])
    moved = refs.clone()
    moved[movers] = 0
    moved[holes] = refs[movers]
    table = _block_rows(torch.where(held, to[pages], 0), per)
    summary = torch.stack((count, torch.tensor(movers.numel(), device=DEV))).int()
    return moved, table, lens, summary, to.int(), s["cache"].view(torch.int16)


def _levels(slots, at):
    """fp32 elements [..., 256] of the key (at = 0) or value (68) of packed slots."""
    codes = torch.stack([(slots[..., at: at + 64] >> k) & 3 for k in (0, 2, 4, 6)], -1).flatten(-2).float()
    scale, zero = slots[..., at + 64: at + 68].contiguous().view(torch.float16).float().split(1, -1)
    return (codes * scale + zero).bfloat16().float()


def _plain_shared(s):
    c, block, per = s["c"], s["c"]["block"], s["c"]["block"] // 128
    r, q, h, sink, recent = c["requests"], c["query"], c["kv_heads"], c["sink"], c["recent"]
    g = c["q_heads"] // h
    hist, win = _history(s["cache"], c), _window(s["cache"], c)
    pages = (s["table"][:, ::per] // per).long()
    before = s["seq_lens"].long() - q
    low = before.clamp(max=sink)
    begin = torch.maximum(low, before - recent)
    of = s["groups"].long()
    firsts = (of[:, None] == torch.arange(c["groups"], device=DEV)).int().argmax(0)
    slot = torch.arange(r, device=DEV) - firsts[of]
    end = torch.full((c["groups"],), 1 << 30, device=DEV).scatter_reduce(0, of, torch.minimum(begin, s["prefix"].long()), "amin")
    scale = 1 / 16
    qr = s["qrot"].float().view(r, q, h, g, DIM) * scale
    qo = s["query"].float().view(r, q, h, g, DIM) * scale
    # the prefix of each group, once
    pos = torch.arange(c["prefix"], device=DEV)
    lead = pages[firsts]
    packed = hist[lead[:, (pos // block).clamp(max=lead.shape[1] - 1)], pos % block]
    most = -(-r // c["groups"])
    padded = torch.zeros(c["groups"], most, q, h, g, DIM, device=DEV)
    padded[of, slot] = qr
    score = torch.einsum("amqhgd,aphd->amqhgp", padded, _levels(packed, 0))
    inside = (pos >= sink) & (pos < end[:, None])
    score = torch.where(inside[:, None, None, None, None, :], score, -math.inf)
    # what each request has for itself
    place = end[of].clamp(min=sink)[:, None] + torch.arange(c["suffix"] + recent + 2, device=DEV)
    tail = hist[pages.gather(1, (place // block).clamp(max=pages.shape[1] - 1)), place % block]
    part = torch.einsum("rqhgd,rphd->rqhgp", qr, _levels(tail, 0))
    inside = (place >= low[:, None]) & (place < begin[:, None])
    part = torch.where(inside[:, None, None, None, :], part, -math.inf)
    # window: sink, then the ring's recent tokens; current tokens
    at = torch.cat((torch.arange(sink, device=DEV).expand(r, sink), begin[:, None] + torch.arange(recent, device=DEV)), 1)
    inside = torch.cat((torch.arange(sink, device=DEV) < low[:, None], at[:, sink:] < before[:, None]), 1)
    index = torch.where(at < sink, at, sink + at % (recent + q))
    rows = win[pages[:, :1], index].float()
    now = s["key"].float().view(r, q, 1, h, DIM), s["value"].float().view(r, q, 1, h, DIM)
    keys = torch.cat((rows[:, :, 0], now[0][:, :, 0]), 1)
    values = torch.cat((rows[:, :, 1], now[1][:, :, 0]), 1)
    raw = torch.einsum("rqhgd,rphd->rqhgp", qo, keys)
    causal = torch.arange(q, device=DEV)[:, None] >= torch.arange(q, device=DEV)
    inside = torch.cat((inside[:, None].expand(r, q, sink + recent), causal.expand(r, q, q)), -1)
    raw = torch.where(inside[:, :, None, None, :], raw, -math.inf)
    own_score = torch.cat((part, raw), -1)
    top = torch.maximum(own_score.amax(-1), score[of, slot].amax(-1))
    spread = torch.zeros_like(padded[..., 0])
    spread[of, slot] = top
    score = torch.exp(score - spread[..., None])
    part, raw = torch.exp(part - top[..., None]), torch.exp(raw - top[..., None])
    total = score.sum(-1)[of, slot] + part.sum(-1) + raw.sum(-1)
    rotated = torch.einsum("amqhgp,aphd->amqhgd", score, _levels(packed, 68))[of, slot]
    # slots that no key was written to carry no weight, whatever they hold
    tail_v = torch.where(((place >= low[:, None]) & (place < begin[:, None]))[..., None, None], _levels(tail, 68), 0.0)
    rotated = rotated + torch.einsum("rqhgp,rphd->rqhgd", part, tail_v)
    out = rotated @ s["rv"].float().T + torch.einsum("rqhgp,rphd->rqhgd", raw, values)
    out = (out / total[..., None]).bfloat16().view(r * q, c["q_heads"] * DIM)
    # the current tokens into the window (a ring index belongs to its latest position)
    spot = before[:, None] + torch.arange(q, device=DEV)
    index = torch.where(spot < sink, spot, sink + spot % (recent + q))
    win[pages[:, :1], index] = torch.stack((now[0][:, :, 0], now[1][:, :, 0]), 2).bfloat16()
    return out, s["cache"][1].view(torch.int16)


# ---------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------


def exact(case, seed):
    if case["op"] == "norm_rope":
        return _exact_norm_rope(prepare(case, seed))
    if case["op"] == "shared":
        return _exact_shared(prepare(case, seed)), None
    return None  # whole numbers and copies


def _exact_norm_rope(s):
    c, rotary = s["c"], s["c"]["rotary"]
    table = s["table"].double()[s["positions"]]
    i = torch.arange(rotary, device=DEV)
    pair = i // 2 if c["interleaved"] else i % (rotary // 2)
    first = i % 2 == 0 if c["interleaved"] else i < rotary // 2
    other = torch.where(first, i + 1, i - 1) if c["interleaved"] else (i + rotary // 2) % rotary
    cos = table[:, pair][:, None]
    sin = (table[:, rotary // 2 + pair] * torch.where(first, -1.0, 1.0).double())[:, None]
    out = []
    for x, w in ((s["query"], s["q_weight"]), (s["key"], s["k_weight"])):
        y = x.double()
        y = y / (y.pow(2).sum(-1, keepdim=True) / DIM + 1e-6).sqrt() * (w.double() + c["offset"])
        z = y.clone()
        z[..., :rotary] = y[..., :rotary] * cos + y[..., other] * sin
        out.append(z)
    return tuple(out)


def _exact_shared(s):
    """Request by request over its own table, without any sharing."""
    c = s["c"]
    block, h, q, sink, recent = c["block"], c["kv_heads"], c["query"], c["sink"], c["recent"]
    hist, win, rv = _history(s["cache"], c), _window(s["cache"], c), s["rv"].double()
    group = c["q_heads"] // h

    def elements(rows, at):
        byte = rows[..., at: at + 64].to(torch.int32)
        code = (byte[..., None] >> torch.tensor([0, 2, 4, 6], device=DEV)) & 3
        pair = rows[..., at + 64: at + 68].contiguous().view(torch.float16).double()
        value = code.flatten(-2).double() * pair[..., :1] + pair[..., 1:]
        return value.float().bfloat16().double()

    out = []
    for r in range(c["requests"]):
        length = int(s["seq_lens"][r])
        before = length - q
        low = min(sink, before)
        begin = max(low, before - recent)
        pos = torch.arange(low, begin, device=DEV)
        blocks = s["table"][r].long()
        place = blocks[pos // 128] * 128 + pos % 128
        rows = hist[place // block, place % block]
        owner = int(blocks[0]) // (block // 128)
        held = list(range(low)) + list(range(begin, before))
        held = torch.tensor([p if p < sink else sink + p % (recent + q) for p in held], dtype=torch.long, device=DEV)
        mine = slice(r * q, r * q + q)
        key = torch.cat((win[owner, held, 0].double(), s["key"][mine].double()))
        value = torch.cat((win[owner, held, 1].double(), s["value"][mine].double()))
        a = s["qrot"][mine].double().view(q, h, group, DIM) / 16
        b = s["query"][mine].double().view(q, h, group, DIM) / 16
        far = torch.einsum("qhgd,phd->qhgp", a, elements(rows, 0))
        near = torch.einsum("qhgd,phd->qhgp", b, key)
        later = torch.arange(q, device=DEV)[None, :] > torch.arange(q, device=DEV)[:, None]
        near[..., held.numel():].masked_fill_(later[:, None, None, :], -math.inf)
        weight = torch.softmax(torch.cat((far, near), -1), -1)
        o = torch.einsum("qhgp,phd->qhgd", weight[..., : pos.numel()], elements(rows, 68)) @ rv.T
        out.append(o + torch.einsum("qhgp,phd->qhgd", weight[..., pos.numel():], value))
    return torch.cat(out).reshape(c["requests"] * q, c["q_heads"] * DIM)
