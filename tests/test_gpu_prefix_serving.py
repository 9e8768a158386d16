"""The operators of prefix sharing as a server uses them together: norm and rotation, page
pool, rotate_store, fork, decode with a shared prefix, release, compaction, growth.  The
same requests run beside it without any sharing (own pages, plain decode_attention).

Tolerance: both sides round the output once more than the shared path (bf16, 1.7e-3 of the
norm each) and the softmax weights of the bf16 / fp16 operands; independent roundings of at
most 1.7e-3, 6 of them between the two sides: 4.2e-3, with 20 % for fp32 sums 5e-3."""

import math
from types import SimpleNamespace

import pytest
import torch

from oscar_new_b200 import kernels
from oscar_new_b200.layout import CacheLayout
from oscar_new_b200.pages import PagePool
from oscar_new_b200.synthetic import cache_stripes, rotation
from tests.helpers import make_config

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Server:
    def __init__(self, layout, pages, rows, tokens):
        self.layout = layout
        columns = -(-tokens // layout.physical_block_tokens) * layout.blocks_per_page
        self.pool = PagePool(pages, rows, columns, layout, DEV)
        self.history, self.window = layout.tensor_views(
            cache_stripes(pages, layout.physical_block_tokens, layout.kv_heads, DEV, sentinel=0xFF))
        self.rk, self.rv = (rotation(i).bfloat16().to(DEV) for i in (1, 2))

    def meta(self, rows, query):
        """Step metadata of `query` new tokens for each of `rows` (already counted in the pool)."""
        table, lens = self.pool.block_tables[rows].contiguous(), self.pool.seq_lens[rows].contiguous()
        r, n, tile = len(rows), len(rows) * query, self.layout.config.queries_per_tile
        tasks = [(i, o) for i in range(r) for o in range(0, query, tile)]
        pos = (lens.long()[:, None] - query + torch.arange(query, device=DEV))
        slots = table.long().gather(1, pos // 128) * 128 + pos % 128
        return SimpleNamespace(query_start_loc=ints(list(range(0, n + 1, query))), seq_lens=lens, block_tables=table,
                               counts=ints([r, n]), num_reqs=r, max_num_reqs=r, max_query_len=query, tasks=ints(tasks),
                               task_count=ints([len(tasks)]), slot_mapping=slots.flatten()), pos.flatten()

    def step(self, rows, q, k, v, norm, groups=None, prefix=None):
        """New tokens of `rows` ([rows, query, heads, 256]) through norm + rotation, store and attention."""
        query, hq = q.shape[1], q.shape[2]
        done = kernels.resize_requests(self.pool, ints(rows), self.pool.seq_lens[rows] + query)
        assert done.tolist() == [1] * len(rows)
        meta, pos = self.meta(rows, query)
        q, k = kernels.qk_norm_rope(q.flatten(0, 1), k.flatten(0, 1), *norm, pos, self.table)
        v = v.flatten(0, 1)
        qrot = kernels.rotate_store(k, v, self.rk, self.rv, self.history, meta.slot_mapping, meta.counts, self.layout,
                                    query=q)
        out = torch.empty(q.shape[0], hq * 256, dtype=torch.bfloat16, device=DEV)
        shared = None
        if groups is not None:
            shared = kernels.prepare_shared_prefix(meta, ints(groups), ints(prefix), self.layout, hq)
        kernels.decode_attention(qrot, q, k, v, self.history, self.window, meta, self.layout, 1 / 16, 1 if query > 16 else 8,
                                 self.rv, out, shared=shared)
        return out.view(len(rows), query, hq, 256)


def close(a, b):
    rel = float((a.float() - b.float()).norm() / b.float().norm())
    assert rel < 5e-3, rel


@pytest.mark.parametrize("hq,h,prompt,query,block,sink,recent", [
    (6, 1, 1000, 1, 768, 4, 64), (12, 2, 1536, 2, 768, 64, 256), (24, 4, 700, 4, 256, 4, 32)])
def test_one_prompt_many_answers(cuda_lib, hq, h, prompt, query, block, sink, recent):
    layout = CacheLayout(block, kv_heads=h, config=make_config(sink, recent, mtp=query - 1))
    shared, alone = (Server(layout, 60, 8, prompt + 600) for _ in range(2))
    angle = torch.arange(prompt + 600, dtype=torch.float64, device=DEV)[:, None] * torch.exp(
        -math.log(1e6) * torch.arange(0, 64, 2, dtype=torch.float64, device=DEV) / 64)
    shared.table = alone.table = torch.cat((angle.cos(), angle.sin()), 1).float()
    gen = torch.Generator(device=DEV).manual_seed(prompt)
    norm = [(1 + 0.1 * torch.randn(256, device=DEV, generator=gen)).bfloat16() for _ in range(2)]

    def tokens(rows, count):
        return [torch.randn(rows, count, heads, 256, device=DEV, generator=gen).bfloat16() for heads in (hq, h, h)]

    # the prompt: one row of the shared server, five rows of the other
    q, k, v = tokens(1, prompt)
    first = shared.step([2], q, k, v, norm)
    for r in range(5):
        close(first, alone.step([r], q, k, v, norm))
    result = kernels.fork_requests(shared.pool, ints([2] * 4), ints([0, 1, 3, 4]), shared.history, shared.window)
    assert result.tolist() == [1] * 4
    full = prompt // block
    if full > 1:  # pages 1 .. full - 1 are held by all five
        assert int((shared.pool.refcounts == 5).sum()) == full - 1
    rows = [0, 1, 2, 3, 4]
    for step in range(4):
        q, k, v = tokens(len(rows), query)
        got = shared.step(rows, q, k, v, norm, groups=[7] * len(rows), prefix=[prompt] * len(rows))
        close(got, alone.step(rows, q, k, v, norm))
        if step == 1:  # the parent and another answer end, the pages move
            for s in (shared, alone):
                assert kernels.resize_requests(s.pool, ints([2, 4]), ints([0, 0])).tolist() == [1, 1]
            summary, _ = kernels.compact_pages(shared.pool, shared.history, shared.window)
            live = int((shared.pool.refcounts[1:] > 0).sum())
            assert summary[0] == live and bool((shared.pool.refcounts[1:live + 1] > 0).all())
            rows = [0, 1, 3]
    # a long continuation of one answer and a short one of the others, sharing on
    for s in (shared, alone):
        extra = torch.Generator(device=DEV).manual_seed(5)
        qkv = [torch.randn(1, 200, heads, 256, device=DEV, generator=extra).bfloat16() for heads in (hq, h, h)]
        s.last = s.step([1], *qkv, norm)
    close(shared.last, alone.last)
    q, k, v = tokens(3, query)
    close(shared.step([0, 1, 3], q, k, v, norm, groups=[1, 1, 1], prefix=[prompt] * 3),
          alone.step([0, 1, 3], q, k, v, norm))
    assert kernels.read_status(DEV) == 0


@pytest.mark.parametrize("prompt", [700, 766, 1023])
def test_forks_behind_rejected_drafts(cuda_lib, prompt):
    """Verify steps whose drafts are partly rejected: lengths in the pool stay at what was
    reserved, the kept ones are the host's; a fork waits until no whole page of the reserved
    length lies behind the kept tokens."""
    block, hq, h, query = 256, 8, 1, 4
    layout = CacheLayout(block, kv_heads=h, config=make_config(4, 64, mtp=query - 1))
    shared, alone = (Server(layout, 40, 4, prompt + 200) for _ in range(2))
    angle = torch.arange(prompt + 200, dtype=torch.float64, device=DEV)[:, None] * torch.exp(
        -math.log(1e6) * torch.arange(0, 64, 2, dtype=torch.float64, device=DEV) / 64)
    shared.table = alone.table = torch.cat((angle.cos(), angle.sin()), 1).float()
    gen = torch.Generator(device=DEV).manual_seed(prompt)
    norm = [(1 + 0.1 * torch.randn(256, device=DEV, generator=gen)).bfloat16() for _ in range(2)]

    def tokens(rows, count):
        return [torch.randn(rows, count, heads, 256, device=DEV, generator=gen).bfloat16() for heads in (hq, h, h)]

    def verify(s, rows, kept, qkv, prefix=None):
        """One step at the kept lengths; the pool's own go no further than they must."""
        have = s.pool.seq_lens[rows].tolist()
        lens = [max(a, b + query) for a, b in zip(have, kept)]
        assert kernels.resize_requests(s.pool, ints(rows), ints(lens)).tolist() == [1] * len(rows)
        meta, _ = s.meta(rows, query)
        meta.seq_lens = ints([k + query for k in kept])
        pos = (meta.seq_lens.long()[:, None] - query + torch.arange(query, device=DEV))
        meta.slot_mapping = (meta.block_tables.long().gather(1, pos // 128) * 128 + pos % 128).flatten()
        q, k, v = (x.flatten(0, 1) for x in qkv)
        q, k = kernels.qk_norm_rope(q, k, *norm, pos.flatten(), s.table)
        qrot = kernels.rotate_store(k, v, s.rk, s.rv, s.history, meta.slot_mapping, meta.counts, layout, query=q)
        out = torch.empty(q.shape[0], hq * 256, dtype=torch.bfloat16, device=DEV)
        plan = None
        if prefix is not None:
            plan = kernels.prepare_shared_prefix(meta, ints([0] * len(rows)), ints([prefix] * len(rows)), layout, hq)
        kernels.decode_attention(qrot, q, k, v, s.history, s.window, meta, layout, 1 / 16, 8, s.rv, out, shared=plan)
        return out.view(len(rows), query, hq, 256)

    q, k, v = tokens(1, prompt)
    shared.step([0], q, k, v, norm)
    for r in range(3):
        alone.step([r], q, k, v, norm)
    kept, waited = prompt, 0
    while True:
        qkv = tokens(1, query)
        close(verify(shared, [0], [kept], qkv), verify(alone, [0, 1, 2], [kept] * 3, [x.repeat(3, 1, 1, 1) for x in qkv])[:1])
        kept += 1  # three drafts rejected
        reserved = int(shared.pool.seq_lens[0])
        if kept >= reserved // block * block:
            break
        waited += 1
    assert reserved == kept + 3 and waited == (0 if prompt == 700 else 1 if prompt == 766 else 0)
    assert kernels.fork_requests(shared.pool, ints([0, 0]), ints([1, 2]), shared.history, shared.window).tolist() == [1, 1]
    at = [kept] * 3
    for accepted in ([1, 4, 2], [3, 1, 4], [4, 4, 1], [2, 3, 3]):
        qkv = tokens(3, query)
        close(verify(shared, [0, 1, 2], at, qkv, prefix=kept), verify(alone, [0, 1, 2], at, qkv))
        at = [a + b for a, b in zip(at, accepted)]
    assert kernels.read_status(DEV) == 0
