"""Decode attention with shared prefixes against the definition in 64 bits, request by
request over its own table.

Tolerances.  Against the exact result an output element is off by the final bf16 rounding
(2^-8 |y|) and, through the inverse rotation, by the bf16 rounding of the softmax weights of
the shared and the BF16 tokens (2^-8 of each weight) and, for a request's own history, by
weights in fp16 (2^-11) and values that are not rounded to bf16 levels (2^-8 of each value):
|error| <= 2^-8 |y| + 1.2 * 2^-8 (sum_t w_t |v_t| |Rv|) with 20 % left for fp32 sums.  In the
norm those roundings are independent, each about 2^-8 / sqrt(6) = 1.6e-3 of the norm at
most: three of them stay below 3.5e-3."""

import math
import random
from types import SimpleNamespace

import pytest
import torch

from oscar_new_b200 import _lib, kernels
from oscar_new_b200.layout import CacheLayout
from oscar_new_b200.pages import PagePool
from oscar_new_b200.synthetic import cache_stripes, rotation
from tests.helpers import make_config

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def slots(gen, tokens, heads, amp=1.0):
    out = torch.zeros(tokens, heads, 160, dtype=torch.uint8, device=DEV)
    for at in (0, 68):
        out[..., at:at + 64] = torch.randint(0, 256, (tokens, heads, 64), device=DEV, generator=gen).to(torch.uint8)
        scale = amp * (0.4 + torch.rand(tokens, heads, 1, device=DEV, generator=gen))
        zero = amp * (-1.5 + 0.6 * torch.rand(tokens, heads, 1, device=DEV, generator=gen))
        out[..., at + 64:at + 68] = torch.cat((scale, zero), -1).half().view(torch.uint8)
    return out


class Batch:
    """A step of requests in groups (label, prefix length of each request) over one cache
    whose unused bytes are NaN scales.  seq = tokens with the current ones."""

    def __init__(self, labels, prefix, seq, query, hq, h, cfg, block=768, seed=0, pages=None, amp=1.0, max_reqs=None,
                 q_amp=1.0):
        self.layout = lay = CacheLayout(block, kv_heads=h, config=cfg)
        self.labels, self.prefix, self.seq, self.query_lens, self.hq, self.h = labels, prefix, seq, query, hq, h
        gen = torch.Generator(device=DEV).manual_seed(seed)
        rng = random.Random(seed)
        rows, number = [], 0
        first = {}
        for i, (g, s) in enumerate(zip(labels, seq)):
            lead = first.setdefault(g, i) if g >= 0 else i
            row = []
            for k in range(max(1, -(-s // block))):
                if lead != i and 0 < k < min(prefix[i], prefix[lead]) // block:
                    row.append(rows[lead][k])
                else:
                    row.append(number)
                    number += 1
            rows.append(row)
        total = pages or number + 3
        names = rng.sample(range(1, total), number)
        if pages:  # some pages far out
            names[0], names[-1] = total - 1, total - 2
        rows = [[names[p] for p in row] for row in rows]
        r, n = max_reqs or len(seq), sum(query)
        table = torch.zeros(r, max(len(x) for x in rows) * lay.blocks_per_page, dtype=torch.int32)
        for i, row in enumerate(rows):
            table[i, :len(row) * lay.blocks_per_page] = torch.tensor(
                [p * lay.blocks_per_page + j for p in row for j in range(lay.blocks_per_page)])
        self.cache = cache_stripes(total, block, h, DEV, sentinel=0xFF) if not pages else torch.empty(
            2, total * lay.blocks_per_page, 128, h, 256, dtype=torch.bfloat16, device=DEV)
        self.history, self.window = lay.tensor_views(self.cache)
        hist = self.history.view(total, -1)[:, :lay.history_page_bytes].unflatten(1, (block, h, 160))
        win = self.window.view(total, -1)[:, :lay.window_page_bytes // 2].unflatten(1, (-1, 2, h, 256))
        for name in set(p for row in rows for p in row):
            self.history.view(total, -1)[name] = 0xFF
        common = {g: slots(gen, prefix[first[g]], h, amp) for g in set(labels) if g >= 0}
        for i, (g, s) in enumerate(zip(labels, seq)):
            p = min(prefix[i], prefix[first[g]], s) if g >= 0 else 0
            data = torch.cat((common[g][:p] if p else slots(gen, 0, h), slots(gen, s - p, h, amp)))
            at, pages_of = torch.arange(s, device=DEV), torch.tensor(rows[i], device=DEV)
            mine = torch.ones(s, dtype=torch.bool, device=DEV)
            if g >= 0 and first[g] != i:
                mine = (at < block) | (at >= max(1, min(prefix[i], prefix[first[g]]) // block) * block)
            hist[pages_of[at[mine] // block], at[mine] % block] = data[mine]
            win[pages_of[0]] = torch.randn(win.shape[1:], device=DEV, generator=gen).bfloat16()
        self.hist, self.win, self.rows = hist, win, rows
        starts = [0]
        for q in query:
            starts.append(starts[-1] + q)
        tile = cfg.queries_per_tile
        tasks = [(i, o) for i, q in enumerate(query) for o in range(0, q, tile)]
        pad = [0] * (r - len(seq))
        self.meta = SimpleNamespace(query_start_loc=ints(starts + [n] * len(pad)), seq_lens=ints(list(seq) + pad),
                                    block_tables=table.to(DEV), counts=ints([len(seq), n]), num_reqs=len(seq),
                                    max_num_reqs=r, max_query_len=max(query),
                                    tasks=ints(tasks + [(-1, -1)] * (n - len(tasks))), task_count=ints([len(tasks)]))
        self.groups, self.lens = ints(list(labels) + [-1] * len(pad)), ints(list(prefix) + pad)
        self.q = (q_amp * torch.randn(n, hq, 256, device=DEV, generator=gen)).bfloat16()
        self.k = torch.randn(n, h, 256, device=DEV, generator=gen).bfloat16()
        self.v = torch.randn(n, h, 256, device=DEV, generator=gen).bfloat16()
        self.rv = rotation(2).bfloat16().to(DEV)
        self.qrot = (self.q.float() @ rotation(1).to(DEV)).bfloat16()

    def run(self, shared=True, splits=8, out=None, store_window=False, **kw):
        out = torch.empty(self.q.shape[0], self.hq * 256, dtype=torch.bfloat16, device=DEV) if out is None else out
        plan = kernels.prepare_shared_prefix(self.meta, self.groups, self.lens, self.layout, self.hq) if shared is True else shared
        kernels.decode_attention(self.qrot, self.q, self.k, self.v, self.history, self.window, self.meta, self.layout, 1 / 16,
                                 splits, self.rv, out, store_window=store_window, shared=plan or None, **kw)
        self.plan = plan
        return out.view(-1, self.hq, 256)

    def exact(self):
        """(output, weighted size) in 64 bits; the size is sum_t w_t |v_t| through |Rv|."""
        cfg, block, h = self.layout.config, self.layout.physical_block_tokens, self.h
        rv, outs, sizes, t0 = self.rv.double(), [], [], 0

        def elements(x, at):
            code = (x[..., at:at + 64].int()[..., None] >> torch.tensor([0, 2, 4, 6], device=DEV)) & 3
            sz = x[..., at + 64:at + 68].contiguous().view(torch.float16).double()
            return (code.flatten(-2) * sz[..., :1] + sz[..., 1:]).float().bfloat16().double()

        for i, (s, nq) in enumerate(zip(self.seq, self.query_lens)):
            before = s - nq
            low = min(cfg.sink_tokens, before)
            begin = max(low, before - cfg.recent_tokens)
            pages = torch.tensor(self.rows[i], device=DEV)
            pos = torch.arange(low, begin, device=DEV)
            x = self.hist[pages[pos // block], pos % block]
            held = [p if p < cfg.sink_tokens else cfg.sink_tokens + p % cfg.ring_tokens
                    for p in list(range(low)) + list(range(begin, before))]
            w = self.win[self.rows[i][0], torch.tensor(held, dtype=torch.long, device=DEV)].double()
            cur = slice(t0, t0 + nq)
            t0 += nq
            key, value = torch.cat((w[:, 0], self.k[cur].double())), torch.cat((w[:, 1], self.v[cur].double()))
            a = self.qrot[cur].double().view(nq, h, self.hq // h, 256) / 16
            b = self.q[cur].double().view(nq, h, self.hq // h, 256) / 16
            far = torch.einsum("qhgd,phd->qhgp", a, elements(x, 0))
            near = torch.einsum("qhgd,phd->qhgp", b, key)
            later = torch.arange(nq, device=DEV)[None] > torch.arange(nq, device=DEV)[:, None]
            near[..., len(held):].masked_fill_(later[:, None, None], -math.inf)
            p = torch.softmax(torch.cat((far, near), -1), -1)
            ph, pr, vh = p[..., :len(pos)], p[..., len(pos):], elements(x, 68)
            o = torch.einsum("qhgp,phd->qhgd", ph, vh) @ rv.T + torch.einsum("qhgp,phd->qhgd", pr, value)
            size = torch.einsum("qhgp,phd->qhgd", ph, vh.abs()) @ rv.abs().T + torch.einsum("qhgp,phd->qhgd", pr, value.abs())
            outs.append(o.reshape(nq, self.hq, 256))
            sizes.append(size.reshape(nq, self.hq, 256))
        return torch.cat(outs), torch.cat(sizes)

    def check(self, got):
        y, size = self.exact()
        err = (got.double() - y).abs()
        bound = 2**-8 * y.abs() + 1.2 * 2**-8 * size
        assert bool((err <= bound).all()), float((err - bound).max())
        rel = float((got.double() - y).norm() / y.norm())
        assert rel < 3.5e-3, rel
        assert kernels.read_status(DEV) == 0
        return rel

    def plan_words(self):
        """The plan as the kernels read it: items, end and used splits per request."""
        head = self.plan.plan.tolist()
        up = (self.plan.max_reqs + 3) // 4 * 4
        n = head[0]
        items = [head[8 + 2 * up + 8 * i:8 + 2 * up + 8 * i + 8] for i in range(n)]
        return items, head[8:8 + self.plan.max_reqs], head[8 + up:8 + up + self.plan.max_reqs]


def simple(members, prefix, extra, query, hq, h, **kw):
    seq = [prefix + extra(i) + query for i in range(members)]
    cfg = kw.pop("cfg", None) or make_config(4, 64, mtp=query - 1)
    return Batch([0] * members, [prefix] * members, seq, [query] * members, hq, h, cfg, **kw)


@pytest.mark.parametrize("members,prefix,query,hq,h", [
    (2, 200, 1, 8, 1), (2, 64, 1, 6, 1), (3, 65, 1, 8, 1), (4, 2048, 1, 8, 1), (5, 1000, 4, 24, 4), (21, 777, 1, 24, 4),
    (22, 640, 1, 12, 2), (64, 1537, 1, 6, 1), (33, 1300, 4, 8, 1), (2, 5000, 1, 1, 1), (7, 900, 2, 35, 5),
])
def test_one_group(cuda_lib, members, prefix, query, hq, h):
    b = simple(members, prefix, lambda i: (i * 37) % 150, query, hq, h, seed=members + prefix)
    b.check(b.run())
    items, ends, used = b.plan_words()
    limit = min(prefix, min(s - query for s in b.seq) - 64)
    assert ends[:members] == [limit if limit > 4 else 0] * members
    tiles = {(it[1], it[7]): (it[4], it[5]) for it in items}
    assert len(tiles) == len(items) and (not items or used[:members] == [max(s for _, s in tiles) + 1] * members)
    for row0 in {r for r, _ in tiles}:  # every row tile covers every history tile once
        spans = sorted(v for (r, _), v in tiles.items() if r == row0)
        assert spans[0][0] == 0 and spans[-1][1] == -(-limit // 64) and all(a[1] == c[0] for a, c in zip(spans, spans[1:]))


def test_groups_of_all_kinds_in_one_step(cuda_lib):
    """Two groups, loners, a labelled request alone, a group whose prefix is inside the sink,
    one shorter than the recent window, members without tokens in the step."""
    labels = [3, 3, 3, -1, 0, 5, 5, 5, 5, -1, 9, 9, 2, 2]
    prefix = [1500, 1500, 1500, 0, 700, 3000, 3000, 3000, 3000, 0, 3, 3, 40, 40]
    seq = [1600, 1510, 1502, 900, 800, 3001, 3300, 3064, 3100, 5, 500, 300, 90, 41]
    query = [1, 4, 2, 1, 1, 1, 0, 3, 1, 1, 4, 1, 1, 1]
    b = Batch(labels, prefix, seq, query, 24, 4, make_config(4, 64, mtp=3), seed=1, max_reqs=17)
    out = b.run(store_window=False)
    b.check(out)
    _, ends, used = b.plan_words()
    # ends: the shortest start of an active member's recent window bounds the prefix
    assert ends[:3] == [min(1500, 1600 - 1 - 64, 1510 - 4 - 64, 1502 - 2 - 64)] * 3
    assert ends[5:9] == [3000 - 64] * 4 and ends[3] == ends[4] == ends[9] == 0
    assert ends[10:14] == [0] * 4 and used[3] == used[4] == 0 and min(used[:3]) > 0
    plain = b.run(shared=False)
    rel = float((out.float() - plain.float()).norm() / plain.float().norm())
    assert rel < 5e-3, rel


def test_prefixes_of_unequal_lengths_use_the_shortest(cuda_lib):
    b = Batch([1, 1, 1], [2000, 1290, 2000], [2300, 2300, 2100], [1, 1, 1], 8, 1, make_config(4, 64), seed=2)
    # request 1 shares fewer tokens: the rest of the group's prefix is attended per request
    b.check(b.run())
    assert b.plan_words()[1][:3] == [1290] * 3


def test_interrupted_labels_are_separate_groups(cuda_lib):
    b = Batch([1, 1, -1, 1, 1], [900] * 5, [1000, 1001, 990, 1002, 1003], [1] * 5, 8, 1, make_config(4, 64), seed=3)
    b.check(b.run())
    items, ends, _ = b.plan_words()
    assert ends[:5] == [900, 900, 0, 900, 900] and {it[3] for it in items} == {0, 3}


@pytest.mark.parametrize("sink,recent,block", [(0, 0, 128), (64, 256, 768), (100, 32, 384), (4, 128, 1024)])
def test_windows_and_pages(cuda_lib, sink, recent, block):
    b = simple(6, 1111, lambda i: 17 * i, 1, 6, 1, cfg=make_config(sink, recent), block=block, seed=block)
    b.check(b.run())


def test_peaked_and_large_scores(cuda_lib):
    """Scores of hundreds: one token takes nearly all the weight, rows re-base often."""
    b = simple(8, 1500, lambda i: 9 * i, 1, 8, 1, seed=5, q_amp=12.0, amp=2.0)
    b.check(b.run())


def test_more_items_than_sms(cuda_lib):
    b = simple(80, 700, lambda i: i, 16, 24, 4, seed=6, cfg=make_config(4, 64, mtp=15))
    assert len(b.plan_words()[0] if b.run() is not None else []) * 4 > 148
    b.check(b.run())


def test_prefill_of_many_suffixes(cuda_lib):
    """Long suffixes: hundreds of query tokens per request on one prefix."""
    b = Batch([0] * 3, [1500] * 3, [1900, 1763, 1600], [300, 163, 1], 6, 1, make_config(4, 64), seed=7)
    b.check(b.run(splits=1))


def test_pages_beyond_32_bits(cuda_lib):
    b = simple(3, 1700, lambda i: i, 1, 24, 4, seed=8, pages=1500)
    assert max(max(r) for r in b.rows) * b.layout.stripe_page_bytes > 2**31
    b.check(b.run())


def test_non_finite_queries_stay_in_their_rows(cuda_lib):
    b = simple(4, 500, lambda i: i, 1, 8, 1, seed=9)
    clean = b.run().clone()
    b.qrot[1, 3, 5] = float("nan")
    b.qrot[2, 0, 7] = float("inf")
    out = b.run()
    assert torch.isnan(out[1, 3]).all() and not torch.isfinite(out[2, 0]).all()
    keep = torch.ones(4, 8, dtype=torch.bool, device=DEV)
    keep[1, 3] = keep[2, 0] = False
    assert torch.equal(out[keep], clean[keep])


def test_same_results_every_time_and_on_another_stream(cuda_lib):
    b = simple(24, 3000, lambda i: 11 * i, 1, 24, 4, seed=10)
    first = b.run().clone()
    for _ in range(3):
        assert torch.equal(b.run(), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = b.run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, first)


def test_replays_follow_new_groups(cuda_lib):
    b = simple(8, 1400, lambda i: 5 * i, 1, 8, 1, seed=11, max_reqs=10)
    plan = kernels.SharedPrefix(10, 8, 8, b.layout, DEV)
    out = torch.empty(8, 8 * 256, dtype=torch.bfloat16, device=DEV)

    def step():
        kernels.prepare_shared_prefix(b.meta, b.groups, b.lens, b.layout, 8, shared=plan)
        b.run(shared=plan, out=out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for groups, lens in (([0] * 8, [1400] * 8), ([-1] * 8, [0] * 8), ([1, 1, 1, -1, 4, 4, 4, 4], [1300, 1200, 1400, 5] + [900] * 4)):
        b.groups.copy_(ints(groups + [-1, -1]))
        b.lens.copy_(ints(lens + [0, 0]))
        out.fill_(7.0)
        graph.replay()
        b.check(out.view(8, 8, 256))


def test_empty_step_and_dummy_counts(cuda_lib):
    b = simple(4, 500, lambda i: i, 1, 8, 1, seed=12)
    b.meta.counts.zero_()
    b.meta.task_count.zero_()
    b.run()
    torch.cuda.synchronize()
    items, ends, used = b.plan_words()
    assert items == [] and not any(ends) and not any(used) and kernels.read_status(DEV) == 0


def test_plan_too_small_for_a_step_falls_back(cuda_lib):
    b = simple(4, 900, lambda i: i, 1, 8, 1, seed=13)
    plan = kernels.SharedPrefix(4, 4, 8, b.layout, DEV)
    plan.items = 1  # the step below needs one row tile: fits; two groups do not
    b.groups.copy_(ints([0, 0, 1, 1]))
    kernels.prepare_shared_prefix(b.meta, b.groups, b.lens, b.layout, 8, shared=plan)
    b.check(b.run(shared=plan))
    assert b.plan_words()[0] == [] and not any(b.plan_words()[1])


def test_withheld_tile_times_out_and_the_context_lives(cuda_lib):
    b = simple(4, 2048, lambda i: i, 1, 8, 1, seed=14)
    want = b.run().clone()
    lib = _lib.lib()
    try:
        lib.oscar_test_set_wait_fault(0, 2000)  # a split here may be a single tile
        b.run()
        assert kernels.read_status(DEV) == 4
    finally:
        lib.oscar_test_set_wait_fault(-1, 0)
    assert torch.equal(b.run(), want) and kernels.read_status(DEV) == 0


def test_refusals(cuda_lib):
    b = simple(4, 500, lambda i: i, 1, 8, 1, seed=15)
    b.run()
    plan = b.plan
    with pytest.raises(ValueError, match="other heads"):
        kernels.prepare_shared_prefix(b.meta, b.groups, b.lens, b.layout, 4, shared=plan)
    with pytest.raises(ValueError, match="entry per request"):
        kernels.prepare_shared_prefix(b.meta, b.groups.long(), b.lens, b.layout, 8)
    with pytest.raises(ValueError, match="entry per request"):
        kernels.prepare_shared_prefix(b.meta, b.groups, b.lens[:3], b.layout, 8)
    out = torch.empty(4, 8 * 256, dtype=torch.bfloat16, device=DEV)
    args = (b.qrot, b.q, b.k, b.v, b.history, b.window, b.meta, b.layout)
    with pytest.raises(ValueError, match="positive softmax scale"):
        kernels.decode_attention(*args, 0.0, 8, b.rv, out, shared=plan)
    with pytest.raises(ValueError, match="contiguous bf16"):
        kernels.decode_attention(*args, 1 / 16, 8, b.rv, out[:, ::2], shared=plan)
    with pytest.raises(ValueError, match="whole contiguous pages"):
        kernels.decode_attention(b.qrot, b.q, b.k, b.v, b.history[:-160], b.window, b.meta, b.layout, 1 / 16, 8, b.rv,
                                 out, shared=plan)


def test_plans_of_other_steps_reach_nothing_outside(cuda_lib):
    """An unfilled plan shares nothing; a plan of a larger step, or of fewer requests than the
    device counts say, stays inside this step's buffers."""
    b = simple(6, 1300, lambda i: i, 1, 8, 1, seed=16)
    want = b.run(shared=False).clone()
    blank = kernels.SharedPrefix(6, 6, 8, b.layout, DEV)
    got = b.run(shared=blank)
    assert float((got.float() - want.float()).norm() / want.float().norm()) < 5e-3
    small = simple(3, 500, lambda i: i, 1, 8, 1, seed=17)
    stale = kernels.prepare_shared_prefix(b.meta, b.groups, b.lens, b.layout, 8)
    scratch = kernels.DecodeScratch(4, 8, 8 + stale.splits, DEV)
    guard = scratch.partials[3].fill_(3.0)
    small.run(shared=stale, scratch=scratch)  # its rows mean nothing, the memory behind them does
    torch.cuda.synchronize()
    assert bool((guard == 3.0).all()) and kernels.read_status(DEV) == 0
    # the first three requests are planned, the others go their own way
    b.meta.num_reqs = 3
    few = kernels.prepare_shared_prefix(b.meta, b.groups[:3], b.lens[:3], b.layout, 8)
    b.meta.num_reqs = 3
    b.check(b.run(shared=few))
    assert few.max_reqs == 3


def test_scratch_of_another_device_is_refused(cuda_lib):
    b = simple(4, 500, lambda i: i, 1, 8, 1, seed=19)
    plan = kernels.prepare_shared_prefix(b.meta, b.groups, b.lens, b.layout, 8)
    with pytest.raises((ValueError, RuntimeError), match="devices|CUDA device only"):
        b.run(shared=plan, scratch=kernels.DecodeScratch(4, 8, 8 + plan.splits, "cpu"))


@pytest.mark.parametrize("active", [1, 3, 7])
def test_padded_step(cuda_lib, active):
    """Requests behind the device counts take no part: their rows get what the step without
    sharing gives them, and the others' rows are those of a step of their own."""
    b = simple(8, 900, lambda i: 20 * i, 1, 8, 1, seed=20)
    b.meta.counts.copy_(torch.tensor([active, active], dtype=torch.int32))
    b.meta.task_count.fill_(active)
    got, plain = b.run().clone(), b.run(shared=False)
    want = b.exact()[0][:active]
    # the bound that check() puts on a whole step
    assert float((got[:active].double() - want).norm() / want.norm()) < 3.5e-3
    assert torch.equal(got[active:], plain[active:]) and kernels.read_status(DEV) == 0


def test_rotation_by_rows_columns_and_strides(cuda_lib):
    b = simple(5, 700, lambda i: i, 4, 24, 4, seed=21)
    want = b.run().clone()
    b.rv = b.rv.t().contiguous().t()
    assert b.rv.stride() == (1, 256) and torch.equal(b.run(), want)
    wide = torch.zeros(256, 512, dtype=torch.bfloat16, device=DEV)
    wide[:, ::2] = b.rv
    b.rv = wide[:, ::2]
    assert torch.equal(b.run(), want)


def set_queries(b, query):
    """New query lengths of the batch's requests in the same device buffers (n unchanged)."""
    starts = [0]
    for q in query:
        starts.append(starts[-1] + q)
    assert starts[-1] == b.q.shape[0] and len(query) == len(b.seq)
    tile = b.layout.config.queries_per_tile
    tasks = [(i, o) for i, q in enumerate(query) for o in range(0, q, tile)]
    b.meta.query_start_loc.copy_(ints(starts))
    b.meta.tasks.copy_(ints(tasks + [(-1, -1)] * (b.meta.tasks.shape[0] - len(tasks))))
    b.meta.task_count.fill_(len(tasks))
    b.query_lens = list(query)


@pytest.mark.parametrize("sharing", [True, False])
@pytest.mark.parametrize("most", [4, 1, 3])
def test_replays_follow_new_query_lengths(cuda_lib, sharing, most):
    """A captured step holds for runs of up to the ``max_query_len`` it was captured with;
    queries of longer ones come back as NaN with the status word set, never as old scratch."""
    b = simple(8, 1400, lambda i: 5 * i, 1, 8, 1, seed=22, cfg=make_config(4, 64, mtp=3))
    b.meta.max_query_len = most
    plan = kernels.SharedPrefix(8, 8, 8, b.layout, DEV) if sharing else False
    out = torch.empty(8, 8 * 256, dtype=torch.bfloat16, device=DEV)

    def step():
        if sharing:
            kernels.prepare_shared_prefix(b.meta, b.groups, b.lens, b.layout, 8, shared=plan)
        b.run(shared=plan, out=out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for query in ([1] * 8, [4, 4] + [0] * 6, [2, 0, 3, 1, 0, 2, 0, 0], [1] * 8):
        set_queries(b, query)
        out.fill_(7.0)
        kernels.read_status(DEV)
        graph.replay()
        past = torch.tensor([i >= most for q in query for i in range(q)], device=DEV)
        got = out.view(8, 8, 256)
        assert kernels.read_status(DEV) == (1 if bool(past.any()) else 0)
        assert bool(torch.isnan(got[past]).all())
        y, size = b.exact()
        err, bound = (got.double() - y).abs(), 2**-8 * y.abs() + 1.2 * 2**-8 * size
        assert bool((err <= bound)[~past].all())


def test_partials_of_runs_longer_than_the_launch(cuda_lib):
    b = simple(2, 300, lambda i: i, 4, 8, 1, seed=23, cfg=make_config(4, 64, mtp=3))
    whole, lse = kernels.attention_partials(b.q, b.k, b.v, b.history, b.window, b.meta, b.layout, 1 / 16, 1, True)
    assert kernels.read_status(DEV) == 0
    b.meta.max_query_len = 2
    part, short = kernels.attention_partials(b.q, b.k, b.v, b.history, b.window, b.meta, b.layout, 1 / 16, 1, True)
    assert kernels.read_status(DEV) == 1
    keep = torch.tensor([0, 1, 4, 5], device=DEV)
    assert torch.equal(part[keep], whole[keep]) and torch.equal(short[keep], lse[keep])
    assert bool(torch.isnan(short[keep + 2]).all())


@pytest.mark.parametrize("name", ["query_start_loc", "seq_lens", "counts", "tasks", "task_count", "block_tables"])
def test_metadata_on_the_host_is_refused(cuda_lib, name):
    b = simple(4, 500, lambda i: i, 1, 8, 1, seed=26)
    b.run()
    kept, here = b.plan, getattr(b.meta, name)
    setattr(b.meta, name, here.cpu())
    with pytest.raises(RuntimeError, match="CUDA device only"):
        b.run(shared=kept)
    if name in ("query_start_loc", "seq_lens", "counts", "block_tables"):
        with pytest.raises(RuntimeError, match="CUDA device only"):
            kernels.prepare_shared_prefix(b.meta, b.groups, b.lens, b.layout, 8)
    setattr(b.meta, name, here)
    b.check(b.run())


def test_step_without_requests(cuda_lib):
    b = simple(4, 500, lambda i: i, 1, 8, 1, seed=27)
    empty = ints([])
    b.meta.num_reqs = b.meta.max_query_len = 0
    b.meta.counts.zero_()
    b.meta.task_count.zero_()
    plan = kernels.prepare_shared_prefix(b.meta, empty, empty, b.layout, 8)
    for name in ("qrot", "q", "k", "v"):
        setattr(b, name, getattr(b, name)[:0])
    assert b.run(shared=plan).shape == (0, 8, 256)
    assert kernels.read_status(DEV) == 0


@pytest.mark.parametrize("sharing", [True, False])
def test_windows_of_requests_behind_many_without_tokens(cuda_lib, sharing):
    """More requests than tokens: the windows of the last ones are stored too."""
    query = [0] * 9 + [1, 0, 2]
    b = Batch([0] * 12, [500] * 12, [600 + i for i in range(12)], query, 8, 1, make_config(4, 64, mtp=3), seed=25)
    before = b.win.clone()
    b.run(shared=sharing, store_window=True)
    torch.cuda.synchronize()
    want, t = before.clone(), 0
    for i, q in enumerate(query):
        for pos in range(b.seq[i] - q, b.seq[i]):
            at = pos if pos < 4 else 4 + pos % b.layout.config.ring_tokens
            want[b.rows[i][0], at, 0], want[b.rows[i][0], at, 1] = b.k[t], b.v[t]
            t += 1
    assert torch.equal(b.win.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("max_reqs", [300, 2100])
def test_more_requests_than_the_plan_kernel_has_threads(cuda_lib, max_reqs):
    """Groups on both sides of the 256th request; at 2100 requests the plan kernel needs more
    than the default 48 KB of shared memory."""
    labels = [0] * 100 + [1] * 90 + [-1] * 30 + [2] * 60 + [3] * 20
    prefix = [300] * 100 + [200] * 90 + [0] * 30 + [500] * 60 + [150] * 20
    seq = [p + 80 + i % 7 for i, p in enumerate(prefix)]
    b = Batch(labels, prefix, seq, [1] * 300, 6, 1, make_config(4, 64), block=256, seed=24, max_reqs=max_reqs)
    b.check(b.run(splits=4))
    items, ends, used = b.plan_words()
    assert ends[:300] == prefix and not any(ends[300:]) and not any(used[300:])
    rows = {it[0]: 0 for it in items}
    assert sorted(rows) == [0, 100, 220, 280]
    spans = sorted((it[0], it[1], it[4], it[5]) for it in items)
    for tok0, members, p in ((0, 100, 300), (100, 90, 200), (220, 60, 500), (280, 20, 150)):
        for row0 in range(0, 6 * members, 128):
            mine = [s[2:] for s in spans if s[:2] == (tok0, row0)]
            assert mine[0][0] == 0 and mine[-1][1] == -(-p // 64) and all(x[1] == y[0] for x, y in zip(mine, mine[1:]))
    assert len({(it[0], it[1], it[7]) for it in items}) == len(items)


def test_plan_of_the_most_requests(cuda_lib):
    """8192 requests, the plan's limit: pairs of them share, one token each."""
    n = 8192
    lay = CacheLayout(256, kv_heads=1, config=make_config(4, 64))
    meta = SimpleNamespace(query_start_loc=torch.arange(n + 1, dtype=torch.int32, device=DEV),
                           seq_lens=torch.full((n,), 400, dtype=torch.int32, device=DEV),
                           block_tables=torch.zeros(n, 4, dtype=torch.int32, device=DEV), counts=ints([n, n]), num_reqs=n,
                           max_num_reqs=n, max_query_len=1)
    groups, lens = torch.arange(n, dtype=torch.int32, device=DEV) // 2, ints([130] * n)
    plan = kernels.prepare_shared_prefix(meta, groups, lens, lay, 6)
    words = plan.plan.cpu()
    items = words[8 + 2 * n:8 + 2 * n + 8 * int(words[0])].view(-1, 8)
    assert int(words[0]) >= n // 2 and bool((words[8:8 + n] == 130).all())
    used = words[8 + n:8 + 2 * n]
    assert torch.equal(torch.bincount(items[:, 0].long() // 2, minlength=n // 2), used[::2].long())
    assert torch.equal(used[::2], used[1::2]) and bool((items[:, 2] == 12).all()) and bool((items[:, 6] == 130).all())
    assert torch.equal(items[:, 3], items[:, 0])


@pytest.mark.parametrize("members,prefix,query,hq,h", [(3, 700, 1, 64, 1), (4, 600, 1, 16, 16), (5, 800, 4, 16, 1)])
def test_head_layouts_at_the_ends(cuda_lib, members, prefix, query, hq, h):
    b = simple(members, prefix, lambda i: 40 * i, query, hq, h, seed=30 + hq + h)
    b.check(b.run())
    assert min(b.plan_words()[1][:members]) > 4


@pytest.mark.parametrize("parts,own", [(63, 1), (1, 63), (32, 64)])
def test_most_and_fewest_splits(cuda_lib, parts, own):
    b = simple(3, 6000, lambda i: 2500 * i, 1, 8, 1, seed=31)
    plan = kernels.SharedPrefix(3, 3, 8, b.layout, DEV, splits=parts)
    kernels.prepare_shared_prefix(b.meta, b.groups, b.lens, b.layout, 8, shared=plan)
    b.check(b.run(shared=plan, splits=own))
    assert b.plan_words()[2][:3] == [max(it[7] for it in b.plan_words()[0]) + 1] * 3 and max(b.plan_words()[2]) <= parts


def test_two_steps_at_once_on_two_streams(cuda_lib):
    """Own plans, scratch and outputs; the library's side stream is common to both."""
    steps = [simple(12, 2000 + 300 * i, lambda j: 7 * j, 1, 24, 4, seed=32 + i) for i in range(2)]
    want = [b.run().clone() for b in steps]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for i, (b, stream) in enumerate(zip(steps, streams)):
            with torch.cuda.stream(stream):
                got[i].append(b.run())
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i]) and kernels.read_status(DEV) == 0
