"""Page pool on the CPU: arena layout, host checks, refusals of the C entry points, and the
plain model the GPU tests compare with."""

import random

import pytest
import torch

from oscar_new_b200 import _lib, kernels
from oscar_new_b200.layout import CacheLayout
from oscar_new_b200.pages import PagePool
from tests.helpers import make_config
from tests.pool_model import PoolModel

LAYOUT = CacheLayout(768, kv_heads=2, config=make_config(4, 64))


def test_arena_holds_state_and_workspace_apart():
    off = kernels.page_pool_layout(11, 5, 12)
    assert (off["refcounts"], off["lens"], off["table"], off["state"]) == (0, 12, 20, 80)
    # head 8, claim 8, remap / used / list 12 each, jobs 4 x max(2 x 5, 11)
    assert off["words"] == 80 + 8 + 8 + 36 + 44
    pool = PagePool(11, 5, 12, LAYOUT, "cpu")
    assert pool.refcounts.tolist() == [1] + [0] * 10 and pool.block_tables.shape == (5, 12)
    assert pool.row_tokens == 12 * 128 and pool.state.numel() == 80
    pool.block_tables.fill_(3)
    pool.seq_lens.fill_(4)
    assert pool.refcounts.tolist() == [1] + [0] * 10 and int(pool.state.sum()) == 1 + 180 + 20


@pytest.mark.parametrize("size", [(0, 1, 6), (1, 0, 6), (1, 1, 0), (4, 4, 7)])
def test_empty_pools_and_partial_page_columns_are_refused(size):
    with pytest.raises(ValueError):
        PagePool(*size, LAYOUT, "cpu")


def test_host_checks():
    pool = PagePool(4, 3, 6, LAYOUT, "cpu")
    history = torch.zeros(4 * LAYOUT.stripe_page_bytes, dtype=torch.uint8)
    window = torch.zeros(2 * LAYOUT.stripe_page_bytes, dtype=torch.bfloat16)
    rows = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA device only"):
        kernels.fork_requests(pool, rows, rows, history, window)
    with pytest.raises(RuntimeError, match="CUDA device only"):
        kernels.resize_requests(pool, rows, rows)
    with pytest.raises(RuntimeError, match="CUDA device only"):
        kernels.compact_pages(pool, history, window)
    for bad in (rows.long(), rows[None], torch.zeros(1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="row lists"):
            kernels.resize_requests(pool, rows, bad)
    with pytest.raises(ValueError, match="4 entries for a pool of 3 rows"):
        kernels.resize_requests(pool, *[torch.zeros(4, dtype=torch.int32)] * 2)
    with pytest.raises(ValueError, match="smaller than the pool"):
        kernels.compact_pages(pool, history[:-1], window)
    with pytest.raises(ValueError, match="smaller than the pool"):
        kernels.fork_requests(pool, rows, rows, history, window[:-1])
    for h, w in ((history.view(torch.int8), window), (history, window.view(torch.int16)), (history[::2], window)):
        with pytest.raises(ValueError, match="contiguous uint8 history"):
            kernels.compact_pages(pool, h, w)


def test_c_entries_refuse_before_any_launch():
    lib, p = _lib.lib(), 1 << 20  # never dereferenced
    geo = kernels.geometry(LAYOUT, 2, 6)
    assert lib.oscar_fork_requests(p, 4, 3, 6, p, p, 4, p, p, geo, p, None) == 1  # more pairs than rows
    assert lib.oscar_fork_requests(p, 4, 3, 6, p, p, -1, p, p, geo, p, None) == 1
    assert lib.oscar_fork_requests(p, 4, 3, 6, None, p, 1, p, p, geo, p, None) == 1
    assert lib.oscar_fork_requests(p, 4, 3, 6, p, p, 1, None, p, geo, p, None) == 1
    assert lib.oscar_fork_requests(p, 4, 3, 6, p, p, 1, p, p + 8, geo, p, None) == 1
    assert lib.oscar_fork_requests(p, 4, 3, 6, p, p, 0, p, p, geo, p, None) == 0
    assert lib.oscar_resize_requests(p + 4, 4, 3, 6, 768, p, p, 1, p, None) == 1
    assert lib.oscar_resize_requests(p, 0, 3, 6, 768, p, p, 1, p, None) == 1
    assert lib.oscar_resize_requests(p, 4, 3, 6, 100, p, p, 1, p, None) == 1
    assert lib.oscar_resize_requests(p, 4, 3, 6, 0, p, p, 1, p, None) == 1
    assert lib.oscar_resize_requests(p, 4, 3, 6, 768, p, None, 1, p, None) == 1
    assert lib.oscar_resize_requests(p, 4, 3, 6, 768, p, p, 0, None, None) == 0
    assert lib.oscar_compact_pages(p, 4, 3, 6, p, p, geo, None, p, None) == 1
    assert lib.oscar_compact_pages(p, 1 << 25, 3, 6, p, p, geo, p, p, None) == 1
    off = torch.zeros(5, dtype=torch.int64)
    assert lib.oscar_page_pool_layout(4, 3, 0, off.data_ptr()) == 1
    assert lib.oscar_page_pool_layout(4, 3, 6, None) == 1


def test_model_keeps_its_own_rules():
    rng = random.Random(0)
    m = PoolModel(12, 6, 24, LAYOUT)
    for _ in range(300):
        if rng.random() < 0.5:
            k = rng.randint(1, 4)
            m.resize([rng.randint(0, 5) for _ in range(k)], [rng.choice([0, rng.randint(1, 3000)]) for _ in range(k)])
        else:
            k = rng.randint(1, 3)
            m.fork([rng.randint(0, 5) for _ in range(k)], [rng.randint(0, 5) for _ in range(k)])
        if rng.random() < 0.2:
            live, to, _ = m.compact()
            assert sorted({p for row in m.pages for p in row}) == list(range(1, live + 1))
        counts = [0] * 12
        for row, n in zip(m.pages, m.lens):
            assert len(row) == -(-n // 768) and 0 not in row
            for p in row:
                counts[p] += 1
        assert counts[1:] == m.refs[1:]
        for row, n in zip(m.pages, m.lens):  # first and partial last pages are private
            assert not row or m.refs[row[0]] == 1 and (n % 768 == 0 or m.refs[row[-1]] == 1)


def test_tables_whose_pages_pass_32_bits_are_refused():
    off = torch.zeros(5, dtype=torch.int64)
    layout = _lib.lib().oscar_page_pool_layout
    assert layout(4, 1 << 20, 2047, off.data_ptr()) == 0 and layout(4, 127, 1 << 24, off.data_ptr()) == 0
    assert layout(4, 1 << 20, 2048, off.data_ptr()) == 1 and layout(4, 128, 1 << 24, off.data_ptr()) == 1
