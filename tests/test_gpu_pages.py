"""Page pool operators against the plain model: state, results and every byte of the cache
are equal."""

import random

import numpy as np
import pytest
import torch

from oscar_new_b200 import kernels
from oscar_new_b200.layout import CacheLayout
from oscar_new_b200.pages import PagePool
from oscar_new_b200.synthetic import cache_stripes
from tests.helpers import make_config
from tests.pool_model import PoolModel

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Pair:
    """A pool and its model over one cache."""

    def __init__(self, pages, rows, tokens, layout, seed=0):
        columns = -(-tokens // layout.physical_block_tokens) * layout.blocks_per_page
        self.pool, self.model = PagePool(pages, rows, columns, layout, DEV), PoolModel(pages, rows, columns, layout)
        cache = cache_stripes(pages, layout.physical_block_tokens, layout.kv_heads, DEV)
        g = torch.Generator(device=DEV).manual_seed(seed)
        cache.view(torch.int16).random_(generator=g)
        self.history, self.window = layout.tensor_views(cache)
        self.h = self.history.cpu().numpy().copy()
        self.w = self.window.view(torch.uint8).cpu().numpy().copy()

    def ints(self, x):
        return torch.tensor(x, dtype=torch.int32, device=DEV)

    def resize(self, rows, lens):
        got = kernels.resize_requests(self.pool, self.ints(rows), self.ints(lens))
        assert got.tolist() == self.model.resize(rows, lens)
        self.state()

    def fork(self, parents, children):
        got = kernels.fork_requests(self.pool, self.ints(parents), self.ints(children), self.history, self.window)
        want, copies = self.model.fork(parents, children)
        assert got.tolist() == want
        self.model.copy(self.h, self.w, copies)
        self.state()
        self.bytes()

    def compact(self):
        summary, to = kernels.compact_pages(self.pool, self.history, self.window)
        live, want, copies = self.model.compact()
        assert summary.tolist() == [live, len(copies)] and to.tolist() == want
        self.model.copy(self.h, self.w, copies)
        self.state()
        self.bytes()

    def state(self):
        assert self.pool.refcounts.tolist() == self.model.refs and self.pool.seq_lens.tolist() == self.model.lens
        assert np.array_equal(self.pool.block_tables.cpu().numpy(), self.model.table())

    def bytes(self):
        assert np.array_equal(self.history.cpu().numpy(), self.h)
        assert np.array_equal(self.window.view(torch.uint8).cpu().numpy(), self.w)


@pytest.mark.parametrize("block,heads,sink,recent,mtp", [(768, 4, 64, 256, 3), (128, 1, 0, 8, 0), (256, 3, 4, 64, 0)])
def test_random_steps(cuda_lib, block, heads, sink, recent, mtp):
    layout = CacheLayout(block, kv_heads=heads, config=make_config(sink, recent, mtp))
    p, rng = Pair(23, 9, 5 * block, layout), random.Random(block)
    for step in range(40):
        kind = rng.random()
        k = rng.randint(1, 9)
        rows = [rng.randint(-1, 9) for _ in range(k)]
        if kind < 0.5:
            p.resize(rows, [rng.choice([0, rng.randint(1, 5 * block + 3), block * rng.randint(1, 5), 1, -7])
                            for _ in range(k)])
        elif kind < 0.85:
            p.fork([rng.randint(-1, 9) for _ in range(k)], rows)
        else:
            p.compact()


@pytest.mark.parametrize("tokens", [1, 127, 767, 768, 769, 1536, 1537, 3000])
def test_fork_lengths_around_the_page_edges(cuda_lib, tokens):
    layout = CacheLayout(768, kv_heads=2, config=make_config(4, 64))
    p = Pair(40, 8, 3500, layout, seed=tokens)
    p.resize([5, 2], [tokens, 900])
    p.fork([5, 5, 2, 5], [0, 1, 3, 7])
    p.fork([0, 7], [4, 6])  # forks of forks
    p.resize([5, 0], [0, min(tokens + 800, 3500)])  # the first parent ends, its children live on
    p.compact()


def test_pages_run_out_in_list_order(cuda_lib):
    layout = CacheLayout(256, kv_heads=1, config=make_config(4, 64))
    p = Pair(8, 6, 2048, layout)
    p.resize([0, 1, 2, 3], [600, 512, 600, 1])  # 3 + 2 + 3 pages of 7: the last two entries fail
    assert p.pool.seq_lens.tolist() == [600, 512, 0, 0, 0, 0]
    p.fork([0, 1, 0], [2, 3, 4])  # two pages left: one fork of 0
    p.resize([0, 4], [0, 256])  # the released pages serve the same call
    p.resize([1, 1, 2], [512, 0, 601])  # no page needed; the second naming of row 1 is refused


def test_many_rows_and_pages(cuda_lib):
    """More list entries than one block's threads and more pages than one scan step."""
    layout = CacheLayout(128, kv_heads=1, config=make_config(0, 4))
    rng = random.Random(1)
    p = Pair(9000, 2500, 640, layout)
    order = list(range(2500))
    rng.shuffle(order)
    p.resize(order, [rng.randint(1, 640) if r < 2000 else 0 for r in order])
    p.fork([rng.randint(0, 2100) for _ in range(600)], [rng.randint(1990, 2499) for _ in range(600)])
    p.resize(order[:1700], [0] * 1700)
    p.compact()
    p.resize(list(range(2500)), [640] * 2500)


def test_captured_steps_replay_on_new_lists(cuda_lib):
    layout = CacheLayout(256, kv_heads=2, config=make_config(4, 64))
    p = Pair(30, 6, 2048, layout)
    a, b = p.ints([0, 0]), p.ints([1, 2])
    r, n = p.ints([0, 3]), p.ints([700, 300])
    kernels.resize_requests(p.pool, p.ints([]), p.ints([]))  # nothing to do
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grown = kernels.resize_requests(p.pool, r, n)
        forked = kernels.fork_requests(p.pool, a, b, p.history, p.window)
        summary, to = kernels.compact_pages(p.pool, p.history, p.window)
    for lists in (([0, 3], [700, 300], [0, 0], [1, 2]), ([1, 2], [0, 900], [3, 0], [4, 1]), ([0, 5], [0, 1], [0, 5], [1, 0])):
        for t, v in zip((r, n, a, b), lists):
            t.copy_(p.ints(v))
        graph.replay()
        want = p.model.resize(lists[0], lists[1])
        wanted, copies = p.model.fork(lists[2], lists[3])
        p.model.copy(p.h, p.w, copies)
        live, where, copies = p.model.compact()
        p.model.copy(p.h, p.w, copies)
        assert grown.tolist() == want and forked.tolist() == wanted
        assert summary.tolist() == [live, len(copies)] and to.tolist() == where
        p.state()
        p.bytes()


def test_caches_of_several_layers_repeat_a_call_from_one_state(cuda_lib):
    layout = CacheLayout(768, 2, config=make_config(4, 64))
    p = Pair(30, 6, 5000, layout, seed=9)
    p.resize([0, 3], [4100, 900])
    layers = [(p.history.clone(), p.window.clone()) for _ in range(2)]
    for call in (lambda h, w: kernels.fork_requests(p.pool, p.ints([0, 3, 0]), p.ints([1, 2, 5]), h, w),
                 lambda h, w: kernels.compact_pages(p.pool, h, w)[0]):
        before, seen = p.pool.state.clone(), []
        for h, w in layers:
            p.pool.state.copy_(before)
            seen.append((call(h, w), p.pool.state.clone()))
        assert all(torch.equal(x, y) for x, y in zip(*seen)) and not torch.equal(seen[0][1], before)
        assert torch.equal(layers[0][0], layers[1][0])
        assert torch.equal(layers[0][1].view(torch.int16), layers[1][1].view(torch.int16))
        kernels.resize_requests(p.pool, p.ints([0]), p.ints([0]))  # holes for the second call
    assert not torch.equal(layers[0][0], p.history)


@pytest.mark.parametrize("pages", [1, 2, 3])
def test_pools_of_very_few_pages(cuda_lib, pages):
    layout = CacheLayout(256, kv_heads=1, config=make_config(4, 64))
    p = Pair(pages, 3, 512, layout)
    p.compact()  # nothing lives
    p.resize([1, 0], [200, 300])
    p.compact()
    p.resize([1], [0])
    p.compact()
    p.resize([2, 0], [100, 512])
    p.fork([2, 2], [0, 1])
    p.compact()


def test_compaction_takes_pages_along_that_only_a_count_holds(cuda_lib):
    """A host that keeps a prompt's pages by their counts alone (no row) finds the whole pages,
    slots and windows, at their new numbers."""
    layout = CacheLayout(256, kv_heads=2, config=make_config(4, 64))
    p = Pair(20, 5, 2048, layout, seed=4)
    p.resize([0, 1, 2], [1000, 700, 300])
    kept = p.model.pages[1]
    p.pool.refcounts[kept] += 1
    kernels.resize_requests(p.pool, p.ints([1, 0]), p.ints([0, 0]))
    before = p.history.view(20, -1)[kept].clone(), p.window.view(20, -1)[kept].clone().view(torch.int16)
    summary, to = kernels.compact_pages(p.pool, p.history, p.window)
    assert summary.tolist() == [5, 5 - len([x for x in kept if x <= 5])] and p.pool.refcounts.tolist() == [1] * 6 + [0] * 14
    now = to[kept].long()
    hist, win = p.history.view(20, -1)[now], p.window.view(20, -1)[now].view(torch.int16)
    size = layout.history_page_bytes
    assert torch.equal(hist[:, :size], before[0][:, :size])
    assert torch.equal(win[:, :layout.window_page_bytes // 2], before[1][:, :layout.window_page_bytes // 2])


def test_rows_of_nearly_two_to_the_31_tokens(cuda_lib):
    layout = CacheLayout(1 << 21, kv_heads=1, config=make_config(4, 64))
    pool, model = PagePool(1100, 1, 1 << 24, layout, DEV), PoolModel(1100, 1, 1 << 24, layout)
    i = lambda x: torch.tensor([x], dtype=torch.int32, device=DEV)  # noqa: E731
    for tokens in (2**31 - 1 - 2**21, 2**31 - 1, 0):
        assert kernels.resize_requests(pool, i(0), i(tokens)).tolist() == model.resize([0], [tokens])
        assert pool.seq_lens.tolist() == model.lens and pool.refcounts.tolist() == model.refs
        assert np.array_equal(pool.block_tables.cpu().numpy(), model.table())


@pytest.mark.parametrize("block,columns,pages", [(128, 300, 900), (384, 600, 500)])
def test_long_rows(cuda_lib, block, columns, pages):
    """Rows of more pages than a warp has lanes and of more table words than a block has
    threads, through every operator."""
    layout = CacheLayout(block, kv_heads=1, config=make_config(0, 16))
    p, rng = Pair(pages, 7, columns * 128, layout, seed=columns), random.Random(columns)
    long = columns * 128
    p.resize([0, 1, 2], [long, long - 129, 40 * block + 1])
    p.fork([0, 1, 1], [3, 4, 5])
    p.resize([1, 0, 6, 2], [0, 0, long // 2, 70 * block])
    p.compact()
    p.fork([3, 6, 2], [0, 1, 1])
    for _ in range(8):
        rows = rng.sample(range(7), 4)
        p.resize(rows, [rng.choice([0, rng.randint(1, long), long]) for _ in rows])
        p.fork([rng.randint(0, 6) for _ in range(3)], [rng.randint(0, 6) for _ in range(3)])
        if rng.random() < 0.5:
            p.compact()


def test_lists_that_are_views_of_the_pool(cuda_lib):
    """Every row takes its neighbour's length: the list is the pool's own length vector, and
    counts as it was before the call."""
    layout = CacheLayout(256, kv_heads=1, config=make_config(4, 64))
    p = Pair(4000, 1400, 512, layout)
    for spread in (0, 300):
        p.resize(list(range(1400)), [0] * 1400)
        p.resize(list(range(1400)), [100 + spread * (i < 700) - i // 14 for i in range(1400)])
        rows, lens = list(range(1, 1400)), p.pool.seq_lens.tolist()[:1399]
        got = kernels.resize_requests(p.pool, p.ints(rows), p.pool.seq_lens[:1399])
        assert got.tolist() == p.model.resize(rows, lens)
        p.state()


def test_pages_beyond_32_bits(cuda_lib):
    """Fork and compaction of pages more than 2^31 bytes into the stripes."""
    layout = CacheLayout(768, kv_heads=4, config=make_config(64, 256, 3))
    pages, size = 1500, layout.stripe_page_bytes
    assert 1400 * size > 2**31
    pool = PagePool(pages, 4, 24, layout, DEV)
    history = torch.zeros(pages * size, dtype=torch.uint8, device=DEV)
    window = torch.zeros(pages * size // 2, dtype=torch.bfloat16, device=DEV)
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    pool.refcounts[1:1400] = 1  # all low pages are held by someone
    assert kernels.resize_requests(pool, i(2), i(1000)).tolist() == [1]
    assert pool.block_tables[2, :12:6].tolist() == [1400 * 6, 1401 * 6]
    g = torch.Generator(device=DEV).manual_seed(1)
    h, w = history.view(pages, -1), window.view(torch.int16).view(pages, -1)
    h[1400:1402] = torch.randint(0, 256, (2, size), dtype=torch.uint8, device=DEV, generator=g)
    w[1400] = torch.randint(-2**15, 2**15, (size // 2,), dtype=torch.int16, device=DEV, generator=g)
    used = [768 * 4 * 160, 232 * 4 * 160]
    first, last, win = h[1400, :used[0]].clone(), h[1401, :used[1]].clone(), w[1400, :layout.window_page_bytes // 2].clone()
    assert kernels.fork_requests(pool, i(2), i(0), history, window).tolist() == [1]
    assert torch.equal(h[1402, :used[0]], first) and torch.equal(h[1403, :used[1]], last)
    assert torch.equal(w[1402, :win.numel()], win) and not h[1403, used[1]:].any() and not w[1403].any()
    pool.refcounts[1:1400] = 0
    kernels.resize_requests(pool, i(2), i(0))
    summary, to = kernels.compact_pages(pool, history, window)
    assert summary.tolist() == [2, 2] and to[1402:1404].tolist() == [1, 2]
    assert torch.equal(h[1, :used[0]], first) and torch.equal(h[2, :used[1]], last) and torch.equal(w[1, :win.numel()], win)
    assert pool.block_tables[0, :12:6].tolist() == [6, 12]
