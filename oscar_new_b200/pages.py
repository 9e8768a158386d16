"""Device page pool of the paged OSCAR cache.

One int32 arena on the device holds, per pool: a reference count per physical page, the
length in tokens of every request row, the block table the attention kernels read
(128-token kernel blocks), and the workspace of the page operators.  Rules:

* page 0 is never handed out (the null page of block tables);
* a row of ``L`` tokens holds ``ceil(L / block_tokens)`` pages, in order, its first page
  owning the request's BF16 window; table entries past them are 0;
* full pages may be shared between rows (their count is the number of rows that hold
  them); a row's first page and its partial last page are its own.  A host may raise the
  counts of a row's pages by one to keep them when the row is released (a prompt to come
  back to): compaction takes such pages along whole and ``moved_to`` says where;
* fresh pages are the free pages of the lowest numbers.

``kernels.resize_requests`` admits, grows and releases rows, ``kernels.fork_requests``
forks them copy-on-write and ``kernels.compact_pages`` moves live pages to the lowest
numbers.  A row's length counts what is reserved for it.  Where a verify step's drafts are
rejected it stays ahead of the tokens that are kept: the host passes the kept lengths to the
attention and asks the next step for the longer of its need and the present length (a
shorter one is refused).  Such a row may be forked once no whole page of its length lies
behind the kept tokens, ``kept >= length // block_tokens * block_tokens``, a step or two
later; before that both rows would write one shared page.

The operators change the pool (and the cache) in stream order and share the arena's
workspace: calls on one pool must be ordered, on one stream or by events.
"""

from __future__ import annotations

import torch

from . import kernels
from .layout import CacheLayout


class PagePool:
    """``num_pages`` pages for ``max_reqs`` request rows of ``columns`` kernel blocks."""

    def __init__(self, num_pages: int, max_reqs: int, columns: int, layout: CacheLayout, device):
        if num_pages < 1 or max_reqs < 1 or columns < 1 or columns % layout.blocks_per_page:
            raise ValueError("a pool needs pages, rows and whole pages of table columns")
        off = kernels.page_pool_layout(num_pages, max_reqs, columns)
        self.num_pages, self.max_reqs, self.columns, self.layout = num_pages, max_reqs, columns, layout
        self.arena = torch.zeros(off["words"], dtype=torch.int32, device=device)
        #: reference counts, lengths and table as one tensor (a snapshot is its clone)
        self.state = self.arena[: off["state"]]
        self.refcounts = self.arena[:num_pages]
        self.seq_lens = self.arena[off["lens"]: off["lens"] + max_reqs]
        self.block_tables = self.arena[off["table"]: off["table"] + max_reqs * columns].view(max_reqs, columns)
        self.refcounts[0] = 1
        self.geometry = kernels.geometry(layout, layout.kv_heads, columns)

    @property
    def device(self):
        return self.arena.device

    @property
    def row_tokens(self) -> int:
        """Most tokens a row can hold."""
        return self.columns * self.layout.kernel_block_tokens

    def check_stripes(self, history, window):
        """The flat cache views of ``CacheLayout.tensor_views`` hold at least the pool's pages."""
        size = self.num_pages * self.layout.stripe_page_bytes
        if history.dtype != torch.uint8 or window.dtype != torch.bfloat16 or not (
                history.is_contiguous() and window.is_contiguous()):
            raise ValueError("the cache views are contiguous uint8 history and bf16 window stripes")
        if history.numel() < size or 2 * window.numel() < size:
            raise ValueError(f"the cache stripes are smaller than the pool's {self.num_pages} pages")
