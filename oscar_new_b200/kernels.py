"""OSCAR INT2 KV-cache operators on B200, behind the reference's operator names.

Each function keeps the name, argument order and meaning of the reference's
``oscar_ascend/kernels.py`` (Triton-Ascend) and calls the sm_100a CUDA library through
its C ABI.  There is deliberately no CPU fallback: tensors must live on a CUDA device
and the library must be built, otherwise the call raises.

Fused entry points that the reference does not have (``rotate_store``,
``decode_attention``) implement the same arithmetic in fewer launches; the backend
uses them.
"""

from __future__ import annotations

import contextlib
import ctypes as C
import functools
import os

import torch

from . import _lib
from .config import attention_programs, quantile_weight_f32

LOG2E = 1.4426950408889634

# Device status words (one int32 per device).  Kernels with bounded device waits store
# 4 (device wait timeout) into their device's word when a wait gives up; the library
# never clears it.  With OSCAR_CHECK_STATUS=1 every such call synchronises and raises
# on a nonzero word (debug mode); otherwise `read_status` reports it on demand.
_STATUS_WORDS: dict = {}
_CHECK_STATUS = os.environ.get("OSCAR_CHECK_STATUS", "0") not in ("", "0")


def status_word(device) -> torch.Tensor:
    """The int32[1] device status word that this module passes to ``device``'s launches."""
    device = torch.device(device)
    index = device.index if device.index is not None else torch.cuda.current_device()
    word = _STATUS_WORDS.get(index)
    if word is None:
        word = torch.zeros(1, dtype=torch.int32, device=f"cuda:{index}")
        _STATUS_WORDS[index] = word
    return word


def read_status(device=None, clear: bool = True) -> int:
    """Synchronise ``device`` and return its status word (0 = no device wait gave up)."""
    word = status_word(device if device is not None else torch.device("cuda"))
    torch.cuda.synchronize(word.device)
    value = int(word.item())
    if clear and value:
        word.zero_()
    return value


def _status(t: torch.Tensor):
    word = _STATUS_WORDS.get(t.get_device())
    return (status_word(t.device) if word is None else word).data_ptr()


def _checked(name: str, t: torch.Tensor):
    """Debug mode: a launch whose device wait gave up raises instead of leaving stale outputs."""
    if _CHECK_STATUS:
        value = read_status(t.device)
        if value:
            raise RuntimeError(f"{name} failed on the device: {_lib.STATUS.get(value, value)}")


def _stream(t: torch.Tensor):
    # the raw handle of torch.cuda.current_stream(t.device), without building a Stream
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _ptr(t):
    return None if t is None else t.data_ptr()


def _require_cuda(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError("OSCAR kernels run on a CUDA device only (no CPU fallback)")


def _rows(x: torch.Tensor):
    """[n, h, 256] bf16 view with unit inner stride and 16-byte aligned rows."""
    if x.dtype != torch.bfloat16 or x.ndim != 3 or x.shape[-1] != 256:
        raise ValueError(f"expected bf16 [n, h, 256], got {tuple(x.shape)} {x.dtype}")
    if x.stride(2) != 1 or x.stride(0) % 8 or x.stride(1) % 8 or x.data_ptr() % 16:
        x = x.contiguous()
    return x


def geometry(layout, hq: int, table_stride: int) -> _lib.Geometry:
    cfg = layout.config
    if hq % layout.kv_heads:
        raise ValueError("query heads must be a multiple of KV heads")
    return _lib.Geometry(
        kv_heads=layout.kv_heads,
        group=hq // layout.kv_heads,
        head_dim=cfg.head_dim,
        block_tokens=layout.physical_block_tokens,
        kernel_block=layout.kernel_block_tokens,
        slot_bytes=cfg.slot_bytes,
        vector_bytes=cfg.vector_bytes,
        sink=cfg.sink_tokens,
        recent=cfg.recent_tokens,
        ring=cfg.ring_tokens,
        table_stride=table_stride,
        query_tile=cfg.queries_per_tile,
        page_bytes=layout.stripe_page_bytes,
    )


def clip_params(cfg, kind: str) -> _lib.Clip:
    """torch.quantile semantics (fp32 rank/weight) or fixed max-abs factor."""
    ratio = cfg.k_clip_ratio if kind == "k" else cfg.v_clip_ratio
    factor = cfg.k_clip_factor if kind == "k" else cfg.v_clip_factor
    if cfg.clip_mode == "factor":
        return _lib.Clip(enabled=1, mode=1, asc_lo=0, asc_hi=0, weight=0.0, factor=factor)
    if not ratio:
        return _lib.Clip(enabled=0, mode=0, asc_lo=0, asc_hi=0, weight=0.0, factor=1.0)
    lo, hi, w = quantile_weight_f32(ratio, cfg.head_dim)
    return _lib.Clip(enabled=1, mode=0, asc_lo=lo, asc_hi=hi, weight=w, factor=1.0)


def _rotation(r: torch.Tensor):
    if r.dtype != torch.bfloat16 or r.shape != (256, 256):
        raise ValueError("rotation must be bf16 [256, 256]")
    s0, s1 = r.stride()
    if not ((s1 == 1 and s0 % 8 == 0) or (s0 == 1 and s1 % 8 == 0)) or r.data_ptr() % 16:
        r = r.contiguous()
    return r


# ----------------------------------------------------------------------------
# reference operators (oscar_ascend/kernels.py)
# ----------------------------------------------------------------------------


def rotate(x: torch.Tensor, rotation: torch.Tensor) -> torch.Tensor:
    """``bf16(x) @ bf16(R)`` with fp32 accumulation -> bf16 (reference kernels.py:51-66)."""
    _require_cuda(x, rotation)
    n, h, d = x.shape
    out = torch.empty((n, h, d), device=x.device, dtype=torch.bfloat16)
    if n == 0:
        return out
    x = _rows(x)
    r = _rotation(rotation)
    _lib.call("oscar_rotate", x.data_ptr(), n, h, x.stride(0), x.stride(1), x.stride(2), r.data_ptr(),
              r.stride(0), r.stride(1), out.data_ptr(), _stream(x))
    return out


def store_int2(key_rot, value_rot, history, slots, counts, layout):
    """Clip + INT2 pack + masked scatter (reference kernels.py:175-202)."""
    _require_cuda(key_rot, value_rot, history, slots, counts)
    cfg = layout.config
    n = key_rot.shape[0]
    kr, vr = key_rot.contiguous(), value_rot.contiguous()
    geo = geometry(layout, layout.kv_heads, 1)
    _lib.call("oscar_store_int2", kr.data_ptr(), vr.data_ptr(), n, history.data_ptr(), slots.data_ptr(),
              counts.data_ptr(), geo, clip_params(cfg, "k"), clip_params(cfg, "v"), _stream(history))


def rotate_store(key, value, rk, rv, history, slots, counts, layout, query=None, debug_rotated=False):
    """Fused ``rotate(K,Rk)``, ``rotate(V,Rv)``, ``store_int2`` and optionally
    ``rotate(Q,Rk)`` in one launch.  Returns ``qrot`` (or None) and, with
    ``debug_rotated``, the bf16 rotated K/V rows that were quantised."""
    _require_cuda(key, value, rk, rv, history, slots, counts, query)
    cfg = layout.config
    n = key.shape[0]
    key, value = _rows(key), _rows(value)
    rk, rv = rk.contiguous(), rv.contiguous()
    qrot = kout = vout = None
    qargs = (None, 0, 0, 0, None)
    if query is not None:
        query = _rows(query)
        qrot = torch.empty(query.shape, device=query.device, dtype=torch.bfloat16)
        qargs = (query.data_ptr(), query.stride(0), query.stride(1), query.shape[1], qrot.data_ptr())
    if debug_rotated:
        kout = torch.empty((n, layout.kv_heads, 256), device=key.device, dtype=torch.bfloat16)
        vout = torch.empty_like(kout)
    geo = geometry(layout, layout.kv_heads, 1)
    _lib.call("oscar_rotate_store", key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(),
              value.stride(0), value.stride(1), n, rk.data_ptr(), rv.data_ptr(), history.data_ptr(),
              slots.data_ptr(), counts.data_ptr(), geo, clip_params(cfg, "k"), clip_params(cfg, "v"),
              *qargs, _ptr(kout), _ptr(vout), _status(key), _stream(key))
    _checked("oscar_rotate_store", key)
    if debug_rotated:
        return qrot, kout, vout
    return qrot


def prepare_tasks(qstarts, counts, tasks, task_count, max_reqs, query_tile, num_reqs=None, source_table=None,
                  table=None, copy_columns=0):
    """Compact (request, query offset) task table (reference kernels.py:262-287)."""
    _require_cuda(qstarts, counts, tasks, task_count, source_table, table)
    copy = source_table is not None and table is not None and copy_columns > 0
    if copy and source_table.stride(1) != 1:
        source_table = source_table.contiguous()
    _lib.call("oscar_prepare_tasks", qstarts.data_ptr(), counts.data_ptr(), tasks.data_ptr(),
              task_count.data_ptr(), tasks.shape[0], max_reqs, query_tile,
              source_table.data_ptr() if copy else None, source_table.stride(0) if copy else 0,
              table.data_ptr() if copy else None, table.stride(0) if copy else 0, copy_columns if copy else 0,
              _stream(counts))


def step_arena_layout(max_reqs: int, columns: int, task_capacity: int) -> dict:
    """Word offsets of the fixed per-step metadata arena (host-only call, no device)."""
    off = (C.c_int64 * 5)()
    _lib.call("oscar_step_arena_layout", max_reqs, columns, task_capacity, C.addressof(off))
    return dict(zip(("qstarts", "seq_lens", "table", "tasks", "words"), (int(x) for x in off)))


def stage_step_metadata(arena, slot_out, max_reqs, columns, task_capacity, query_tile, num_reqs=0, num_tokens=0,
                        qstarts=None, seq_lens=None, table=None, slots=None, copy_columns=0):
    """Stage one step's metadata into the fixed arena in one launch (counts, query starts,
    sequence lengths, reachable block-table columns, slot mapping, task table).  No
    sources and zero requests / tokens stage a dummy step: counts and task count 0,
    nothing else."""
    _require_cuda(arena, slot_out, qstarts, seq_lens, table, slots)
    if arena.dtype != torch.int32 or slot_out.dtype != torch.int64:
        raise ValueError("the arena is int32 and the slot buffer int64")
    if qstarts is not None:
        qstarts = qstarts.to(torch.int32)
    if not num_reqs:
        seq_lens = table = None
    if seq_lens is not None:
        seq_lens = seq_lens.to(torch.int32)
    if table is None or not copy_columns:
        table, copy_columns = None, 0
    elif table.dtype != torch.int32 or table.stride(1) != 1:
        table = table.to(torch.int32).contiguous()
    slots = slots.to(torch.int64) if num_tokens else None
    _lib.call("oscar_stage_step_metadata", _ptr(qstarts), _ptr(seq_lens), _ptr(table),
              0 if table is None else table.stride(0), _ptr(slots), num_reqs, num_tokens, copy_columns, query_tile,
              arena.data_ptr(), max_reqs, columns, task_capacity, slot_out.data_ptr(), slot_out.shape[0],
              _stream(arena))


def prefill_attention(query, key, value, query_start_loc, num_reqs: int, max_query_len: int, scale: float,
                      out=None):
    """Causal attention of a first prefill over the current tokens only (tcgen05 kernel):
    query [n, Hq, 256], key / value [n, Hkv, 256] bf16, device query starts
    [num_reqs + 1]; returns / fills out [n, Hq, 256] bf16."""
    _require_cuda(query, key, value, query_start_loc, out)
    n, hq, d = query.shape
    if out is None:
        out = torch.empty((n, hq, d), dtype=torch.bfloat16, device=query.device)
    if n == 0 or num_reqs == 0:
        return out
    query, key, value = _rows(query), _rows(key), _rows(value)
    _lib.call("oscar_prefill_attention", query.data_ptr(), query.stride(0), query.stride(1), key.data_ptr(),
              key.stride(0), key.stride(1), value.data_ptr(), value.stride(0), value.stride(1),
              query_start_loc.data_ptr(), num_reqs, max_query_len, n, hq, key.shape[1], float(scale), out.data_ptr(),
              out.stride(0), out.stride(1), _status(out), _stream(query))
    return out


_HERE = contextlib.nullcontext()


def _dense(t: torch.Tensor):
    return t if t.is_contiguous() else t.contiguous()



def _same_device(*tensors):
    """All on one CUDA device (None: skipped, but not the first); returns the context that
    makes it current if it is not."""
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != index:
            _require_cuda(*tensors)
            raise ValueError(f"tensors on several devices: {sorted({str(t.device) for t in tensors if t is not None})}")
    if index < 0:
        _require_cuda(*tensors)
    return _HERE if index == torch.cuda.current_device() else torch.cuda.device(index)


def _output_rows(out, like):
    """``out`` (or a new tensor) as the bf16 rows a kernel writes for ``like``."""
    if out is None:
        return like.new_empty(like.shape)
    if out.dtype != torch.bfloat16 or out.shape != like.shape:
        raise ValueError(f"expected a bf16 output of shape {tuple(like.shape)}, got {tuple(out.shape)} {out.dtype}")
    if out.stride(2) != 1 or out.stride(0) % 8 or out.stride(1) % 8 or out.data_ptr() % 16:
        raise ValueError("output rows must be 16-byte aligned with unit inner stride")
    n, h, _ = out.shape
    step = sorted((stride, size) for stride, size in ((out.stride(0), n), (out.stride(1), h)) if size > 1)
    width = 256
    for stride, size in step:
        if stride < width:
            raise ValueError("output rows overlap each other")
        width = stride * (size - 1) + width
    return out


def _rows_apart(a, b) -> bool:
    """Whether two [n, h, 256] row sets cannot share memory: apart altogether, or columns of
    one fused [n, width] buffer that do not meet."""
    def span(t):
        n, h, _ = t.shape
        return t.data_ptr(), t.data_ptr() + 2 * ((n - 1) * t.stride(0) + (h - 1) * t.stride(1) + 256)

    (a0, a1), (b0, b1) = span(a), span(b)
    if a1 <= b0 or b1 <= a0:
        return True
    step = 2 * a.stride(0)
    if a.shape[0] != b.shape[0] or step != 2 * b.stride(0) or step <= 0:
        return False
    wide = [2 * ((t.shape[1] - 1) * t.stride(1) + 256) for t in (a, b)]
    gap = (b0 - a0) % step
    return max(wide) <= step and gap >= wide[0] and gap + wide[1] <= step


def qk_norm_rope(query, key, q_weight, k_weight, positions, cos_sin, eps=1e-6, weight_offset=0.0, interleaved=False,
                 counts=None, query_out=None, key_out=None):
    """Norm of every query and key head and the rotation of its position, in one pass.

    query [n, Hq, 256] and key [n, Hkv, 256] bf16, any strides with unit inner stride (views
    of a fused projection); weights [256] and the table cos_sin [positions, rotary]
    (cosines, then sines) fp32 or bf16; positions int64 or int32 [n].
    ``y = x * rsqrt(mean(x^2) + eps) * (w + weight_offset)``, then the first ``rotary`` dims
    turn: pairs (i, i + rotary/2), or (2i, 2i+1) with ``interleaved``; none for a table of
    no columns, whatever the positions.  fp32 inside (a row's sum of squares has to fit:
    elements up to about 2^59).
    Outputs are new tensors, or ``query_out`` / ``key_out``: an output may be its own input,
    and must otherwise not overlap the other rows.  ``counts`` (device [requests, active
    tokens]) leaves the tokens behind the active ones as they were.  A token whose position
    is not in the table stays unwritten and raises the status word (``read_status`` = 1).
    Returns (query_out, key_out)."""
    for t, name in ((query, "query"), (key, "key")):
        if t.ndim != 3 or t.dtype != torch.bfloat16 or t.shape[2] != 256:
            raise ValueError(f"{name}: expected bf16 [n, heads, 256], got {tuple(t.shape)} {t.dtype}")
    n = query.shape[0]
    if key.shape[0] != n or positions.shape != (n,):
        raise ValueError("query, key and positions must have the same tokens")
    if q_weight.shape != (256,) or k_weight.shape != (256,) or q_weight.dtype != k_weight.dtype:
        raise ValueError("norm weights are [256], both of one type")
    if cos_sin.ndim != 2 or cos_sin.shape[1] % 16 or cos_sin.shape[1] > 256:
        raise ValueError("the cos / sin table is [positions, rotary], rotary a multiple of 16 up to 256")
    for t, name in ((q_weight, "weights"), (cos_sin, "table")):
        if t.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"{name} must be fp32 or bf16, got {t.dtype}")
    if positions.dtype not in (torch.int64, torch.int32):
        raise ValueError("positions must be int64 or int32")
    if counts is not None and (counts.dtype != torch.int32 or counts.numel() < 2):
        raise ValueError("counts are int32 [requests, active tokens]")
    if not float(eps) >= 0.0:
        raise ValueError("eps must not be negative")
    counts = None if counts is None else _dense(counts)
    qo, ko = _output_rows(query_out, query), _output_rows(key_out, key)
    if query_out is not None or key_out is not None:
        # the same rows: strides of dims of one element do not matter
        same = [o.data_ptr() == i.data_ptr() and all(a == b for a, b, size in zip(o.stride(), i.stride(), o.shape) if size > 1)
                for o, i in ((qo, query), (ko, key))]
        pairs = [(qo, ko), (qo, key), (ko, query)] + [p for p, s in zip(((qo, query), (ko, key)), same) if not s]
        if not all(0 in a.shape or 0 in b.shape or _rows_apart(a, b) for a, b in pairs):
            raise ValueError("an output overlaps rows other than its own input's")
    device = _same_device(query, key, q_weight, k_weight, positions, cos_sin, counts, query_out, key_out)
    if n == 0:
        return qo, ko
    query, key = _rows(query), _rows(key)
    aligned = [t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)
               for t in (q_weight, k_weight, cos_sin, positions)]
    with device:
        _lib.call("oscar_qk_norm_rope", query.data_ptr(), query.stride(0), query.stride(1), key.data_ptr(),
                  key.stride(0), key.stride(1), n, query.shape[1], key.shape[1], aligned[0].data_ptr(),
                  aligned[1].data_ptr(), int(q_weight.dtype == torch.float32), float(weight_offset), float(eps),
                  aligned[3].data_ptr(), int(positions.dtype == torch.int64), aligned[2].data_ptr(),
                  int(cos_sin.dtype == torch.float32), cos_sin.shape[0], cos_sin.shape[1], int(bool(interleaved)),
                  _ptr(counts), qo.data_ptr(), qo.stride(0), qo.stride(1), ko.data_ptr(), ko.stride(0), ko.stride(1),
                  _status(query), _stream(query))
    _checked("oscar_qk_norm_rope", query)
    return qo, ko


# ----------------------------------------------------------------------------
# page pool (``pages.PagePool``)
# ----------------------------------------------------------------------------


def page_pool_layout(num_pages: int, max_reqs: int, columns: int) -> dict:
    """Word offsets of a page pool's arena (host-only call, no device)."""
    off = (C.c_int64 * 5)()
    _lib.call("oscar_page_pool_layout", num_pages, max_reqs, columns, C.addressof(off))
    return dict(zip(("refcounts", "lens", "table", "state", "words"), (int(x) for x in off)))


def _pool_list(pool, *lists):
    """int32 device lists of one length, at most one entry per row of the pool."""
    for t in lists:
        if t.dtype != torch.int32 or t.ndim != 1 or t.shape != lists[0].shape:
            raise ValueError("row lists are int32 [count], all of one length")
    if lists[0].shape[0] > pool.max_reqs:
        raise ValueError(f"{lists[0].shape[0]} entries for a pool of {pool.max_reqs} rows")
    # a view of the pool's own state counts as it is before the call
    first = pool.arena.data_ptr()
    last = first + 4 * pool.arena.numel()
    return [t.clone() if first <= t.data_ptr() < last else _dense(t) for t in lists]


def fork_requests(pool, parents, children, history, window):
    """Fork rows of a page pool copy-on-write: row ``children[i]`` gets the tokens of row
    ``parents[i]`` (int32 device lists).

    Full pages but the first are shared; the first page's used slots and BF16 window and a
    partial last page's used slots are copied to fresh pages of the cache (``history`` /
    ``window``, the flat views of ``CacheLayout.tensor_views``).  Returns int32 [count]: 1
    forked; 0 the free pages ran out at this pair or before; -1 not a valid pair (an empty
    or unknown parent, a child that holds tokens or that an earlier pair names).  A parent
    whose last tokens were rejected drafts waits until ``kept >= length // block_tokens *
    block_tokens`` (``pages``)."""
    pool.check_stripes(history, window)
    parents, children = _pool_list(pool, parents, children)
    device = _same_device(pool.arena, parents, children, history, window)
    result = parents.new_empty(parents.shape)
    with device:
        _lib.call("oscar_fork_requests", pool.arena.data_ptr(), pool.num_pages, pool.max_reqs, pool.columns,
                  parents.data_ptr(), children.data_ptr(), parents.shape[0], history.data_ptr(), window.data_ptr(),
                  pool.geometry, result.data_ptr(), _stream(parents))
    return result


def resize_requests(pool, rows, lens):
    """Admit, grow and release rows of a page pool: row ``rows[i]`` gets ``lens[i]`` tokens
    (int32 device lists), 0 to release it.

    Releases come before growth, so their pages serve the same call.  Returns int32
    [count]: 1 done; 0 the free pages ran out at this entry or before (the row is
    unchanged); -1 refused (row or length out of range, a shorter length other than 0, a
    row that an earlier entry names).  Rejected draft tokens stay reserved (``pages``)."""
    rows, lens = _pool_list(pool, rows, lens)
    device = _same_device(pool.arena, rows, lens)
    result = rows.new_empty(rows.shape)
    with device:
        _lib.call("oscar_resize_requests", pool.arena.data_ptr(), pool.num_pages, pool.max_reqs, pool.columns,
                  pool.layout.physical_block_tokens, rows.data_ptr(), lens.data_ptr(), rows.shape[0],
                  result.data_ptr(), _stream(rows))
    return result


def compact_pages(pool, history, window):
    """Move a pool's live pages onto the lowest page numbers (1 .. live), with the slots and
    windows they hold (all of them, for a page that only its count holds); counts and table
    follow.  Returns (summary int32 [live pages, moved pages], moved_to int32 [num_pages]:
    each page's new number, -1 for a free page)."""
    pool.check_stripes(history, window)
    device = _same_device(pool.arena, history, window)
    summary, moved_to = pool.arena.new_empty(2), pool.arena.new_empty(pool.num_pages)
    with device:
        _lib.call("oscar_compact_pages", pool.arena.data_ptr(), pool.num_pages, pool.max_reqs, pool.columns,
                  history.data_ptr(), window.data_ptr(), pool.geometry, summary.data_ptr(), moved_to.data_ptr(),
                  _stream(summary))
    return summary, moved_to


def _meta_common(meta, layout, hq):
    geo = geometry(layout, hq, meta.block_tables.stride(0))
    if meta.block_tables.stride(1) != 1:
        raise ValueError("block table rows must be contiguous")
    # Launch only the query-row tiles this step can use: a task never holds more than
    # min(queries_per_tile, max_query_len) queries (host scheduler value, no device read).
    # The raw kernel checks that on the device: queries past it become NaN, status word 1.
    max_q = getattr(meta, "max_query_len", None)
    if isinstance(max_q, int) and max_q > 0:
        geo.query_tile = min(geo.query_tile, max_q)
    return geo


def attention_partials(query, key, value, history, window, meta, layout, scale, splits, raw):
    """Split-KV attention partials (reference kernels.py:439-482)."""
    _require_cuda(query, key, value, history, window)
    n, hq, d = query.shape
    partials = torch.empty((n, hq, splits, d), dtype=torch.float32, device=query.device)
    lse = torch.empty((n, hq, splits), dtype=torch.float32, device=query.device)
    if n == 0:
        return partials, lse
    query = _rows(query)
    key, value = _rows(key), _rows(value)
    geo = _meta_common(meta, layout, hq)
    programs = attention_programs(n, meta.max_num_reqs, layout.config.queries_per_tile)
    _lib.call("oscar_attention_partials", query.data_ptr(), query.stride(0), query.stride(1), key.data_ptr(),
              key.stride(0), key.stride(1), value.data_ptr(), value.stride(0), value.stride(1),
              history.data_ptr(), window.data_ptr(), meta.query_start_loc.data_ptr(), meta.seq_lens.data_ptr(),
              meta.block_tables.data_ptr(), meta.counts.data_ptr(), meta.tasks.data_ptr(),
              meta.task_count.data_ptr(), min(programs, meta.tasks.shape[0]), n, partials.data_ptr(),
              lse.data_ptr(), geo, float(scale), int(splits), int(bool(raw)), _status(query), _stream(query))
    _checked("oscar_attention_partials", query)
    return partials, lse


def merge_splits(partials, lse, counts):
    """LSE merge of split partials (reference kernels.py:506-511)."""
    _require_cuda(partials, lse, counts)
    n, hq, splits, d = partials.shape
    out = torch.empty((n, hq, d), dtype=torch.bfloat16, device=partials.device)
    logsum = torch.empty((n, hq), dtype=torch.float32, device=partials.device)
    if n:
        _lib.call("oscar_merge_splits", partials.contiguous().data_ptr(), lse.contiguous().data_ptr(), n, hq, splits,
                  counts.data_ptr(), out.data_ptr(), logsum.data_ptr(), _stream(partials))
    return out, logsum


def merge_paths(history_out, history_lse, raw_partials, raw_lse, counts, output):
    """LSE merge of the history and raw paths into ``output`` (reference kernels.py:530-541)."""
    _require_cuda(history_out, history_lse, raw_partials, raw_lse, counts, output)
    n, hq, d = history_out.shape
    if n == 0:
        return
    if not output.is_contiguous():
        raise ValueError("output must be contiguous")
    a = history_out.contiguous()
    b = raw_partials.contiguous()
    lb = raw_lse.contiguous()
    b_stride = b.shape[2] * d if b.ndim == 4 else d
    lb_stride = lb.shape[2] if lb.ndim == 3 else 1
    _lib.call("oscar_merge_paths", a.data_ptr(), history_lse.contiguous().data_ptr(), b.data_ptr(), b_stride,
              lb.data_ptr(), lb_stride, n, hq, counts.data_ptr(), output.data_ptr(), _stream(a))


def store_windows(key, value, window, meta, layout):
    """Write current BF16 K/V into the sink/ring window (reference kernels.py:598-620)."""
    _require_cuda(key, value, window)
    key, value = _rows(key), _rows(value)
    geo = _meta_common(meta, layout, layout.kv_heads)
    programs = min(key.shape[0], meta.max_num_reqs)
    _lib.call("oscar_store_windows", key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(),
              value.stride(0), value.stride(1), window.data_ptr(), meta.query_start_loc.data_ptr(),
              meta.seq_lens.data_ptr(), meta.block_tables.data_ptr(), meta.counts.data_ptr(), programs, geo,
              _stream(key))


def dequant_inverse_rotate(history, slots, rk, rv, layout):
    """Diagnostic finite tile only (reference kernels.py:651-672)."""
    _require_cuda(history, slots, rk, rv)
    n, h = slots.numel(), layout.kv_heads
    if n > 4096:
        raise ValueError("diagnostic dequant is limited to 4096 tokens; use fused attention")
    k = torch.empty((n, h, 256), device=history.device, dtype=torch.bfloat16)
    v = torch.empty_like(k)
    geo = geometry(layout, h, 1)
    _lib.call("oscar_unpack", history.data_ptr(), slots.contiguous().data_ptr(), n, geo, k.data_ptr(),
              v.data_ptr(), _stream(history))
    return rotate(k, rk.T), rotate(v, rv.T)


# ----------------------------------------------------------------------------
# fused decode step
# ----------------------------------------------------------------------------


class DecodeScratch:
    """Caller-owned split scratch: fp32 partials [n, Hq, splits+1, 256] and lse.  A step
    with a shared prefix takes ``splits`` = its own splits + the plan's."""

    def __init__(self, max_tokens: int, hq: int, splits: int, device):
        self.splits = splits
        self.partials = torch.empty((max_tokens, hq, splits + 1, 256), dtype=torch.float32, device=device)
        self.lse = torch.empty((max_tokens, hq, splits + 1), dtype=torch.float32, device=device)


@functools.lru_cache(maxsize=256)
def _shared_sizes(max_reqs: int, max_tokens: int, hq: int, kv_heads: int):
    """(work items, int32 words) of a shared-prefix plan (host-only call, no device)."""
    sizes = (C.c_int64 * 2)()
    _lib.call("oscar_shared_prefix_layout", max_reqs, max_tokens, hq, kv_heads, C.addressof(sizes))
    return int(sizes[0]), int(sizes[1])


class SharedPrefix:
    """Device plan of steps whose requests share prefixes (``prepare_shared_prefix``): for
    steps of at most ``max_reqs`` requests and ``max_tokens`` tokens.  ``splits``: most parts
    a group's history is cut into; the default fills the GPU for one group while the split
    scratch stays under ``scratch_bytes``."""

    def __init__(self, max_reqs: int, max_tokens: int, hq: int, layout, device, splits: int | None = None,
                 scratch_bytes: int = 256 << 20, _blank: bool = True):
        if splits is None:
            fit = scratch_bytes // max(max_tokens * hq * 256 * 4, 1)
            splits = max(1, min(48, -(-148 // layout.kv_heads), fit))
        if not 1 <= splits <= 63:
            raise ValueError("a shared prefix is cut into 1 to 63 splits")
        self.items, words = _shared_sizes(max_reqs, max_tokens, hq, layout.kv_heads)
        self.max_reqs, self.max_tokens, self.splits, self.hq, self.layout = max_reqs, max_tokens, splits, hq, layout
        # a plan that was never filled shares nothing
        self.plan = (torch.zeros if _blank else torch.empty)(words, dtype=torch.int32, device=device)
        self._geometries: dict = {}

    def geometry(self, table_stride: int, query_tile: int):
        # one struct per form, never changed: threads may call with the same plan
        geo = self._geometries.get((table_stride, query_tile))
        if geo is None:
            geo = geometry(self.layout, self.hq, table_stride)
            geo.query_tile = query_tile
            self._geometries[table_stride, query_tile] = geo
        return geo


def prepare_shared_prefix(meta, groups, prefix_lens, layout, hq, shared=None):
    """Plan one step of requests that share prefixes; once per step, for all its layers.

    groups, prefix_lens: int32 device tensors [requests].  Consecutive requests with the
    same label >= 0 form a group whose first ``prefix_lens`` tokens (the shortest counts)
    hold the same history, as after ``fork_requests``; -1: not in a group.  ``shared`` is a
    ``SharedPrefix`` to fill again (needed for graph capture of changing steps; in stream
    order, behind the steps that read it), else a new one.  Labels, lengths and query
    lengths may change from replay to replay, the last up to the ``meta.max_query_len`` that
    ``decode_attention`` was captured with.  Returns it, for
    ``decode_attention(..., shared=)``."""
    if groups.dtype != torch.int32 or prefix_lens.dtype != torch.int32 or groups.ndim != 1 or prefix_lens.ndim != 1:
        raise ValueError("groups and prefix_lens must be int32 with an entry per request")
    reqs = min(groups.shape[0], prefix_lens.shape[0], meta.max_num_reqs)
    if reqs < meta.num_reqs:
        raise ValueError("groups and prefix_lens must be int32 with an entry per request")
    if shared is None:
        tokens = getattr(meta, "num_actual_tokens", None) or meta.num_reqs * max(1, meta.max_query_len)
        shared = SharedPrefix(max(reqs, 1), tokens, hq, layout, groups.device, _blank=reqs == 0)
    elif shared.hq != hq or shared.max_reqs < meta.num_reqs or shared.layout != layout:
        raise ValueError("the plan was made for other heads, another layout or fewer requests")
    elif reqs < shared.max_reqs:
        raise ValueError(f"groups and prefix_lens must have the plan's {shared.max_reqs} entries")
    for name, size in (("query_start_loc", meta.num_reqs + 1), ("seq_lens", meta.num_reqs), ("counts", 2)):
        t = getattr(meta, name)
        if t.dtype != torch.int32 or t.ndim != 1 or not t.is_contiguous() or t.shape[0] < size:
            raise ValueError(f"{name} must be a contiguous int32 vector of {size} entries or more, "
                             f"got {tuple(t.shape)} {t.dtype}")
    table = meta.block_tables
    device = _same_device(groups, prefix_lens, shared.plan, meta.query_start_loc, meta.seq_lens, meta.counts, table)
    if reqs == 0:  # a new plan of an empty step: it shares nothing as it is
        return shared
    groups, prefix_lens = _dense(groups), _dense(prefix_lens)
    with device:
        _lib.call("oscar_prepare_shared_prefix", meta.query_start_loc.data_ptr(), meta.seq_lens.data_ptr(),
                  meta.counts.data_ptr(), groups.data_ptr(), prefix_lens.data_ptr(), shared.max_reqs, shared.items,
                  shared.splits, shared.geometry(table.stride(0), layout.config.queries_per_tile),
                  shared.plan.data_ptr(), _stream(groups))
    return shared


def _decode_shared(qrot, query, key, value, history, window, meta, layout, scale, splits, rv, output, scratch,
                   store_window, shared):
    """``decode_attention`` of a step with a plan."""
    n, hq, _ = query.shape
    if shared.hq != hq or shared.max_reqs < meta.num_reqs or shared.layout != layout:
        raise ValueError("the plan was made for other heads, another layout or fewer requests")
    if not scale > 0:
        raise ValueError("a shared prefix needs a positive softmax scale")
    if history.dtype != torch.uint8 or history.numel() % layout.stripe_page_bytes or not history.is_contiguous():
        raise ValueError("the history view must be whole contiguous pages of bytes")
    if window.dtype != torch.bfloat16 or not window.is_contiguous() or 2 * window.numel() < history.numel():
        raise ValueError("the window view must be the contiguous bf16 stripe beside the history")
    if output.dtype != torch.bfloat16 or not output.is_contiguous() or output.numel() != query.numel():
        raise ValueError("output must be contiguous bf16 [n, Hq * 256]")
    if qrot.shape != query.shape or qrot.dtype != torch.bfloat16 or rv.shape != (256, 256) or rv.dtype != torch.bfloat16:
        raise ValueError("qrot must be bf16 like the query, and rv a bf16 [256, 256] rotation")
    if key.shape != (n, layout.kv_heads, 256) or value.shape != key.shape:
        raise ValueError("key and value must be [n, KV heads, 256]")
    table = meta.block_tables
    if table.stride(1) != 1 or table.shape[0] < meta.num_reqs:
        raise ValueError("the block table must have a contiguous row per request")
    device = _same_device(qrot, query, key, value, history, window, rv, output, shared.plan, table,
                          meta.query_start_loc, meta.seq_lens, meta.counts, meta.tasks, meta.task_count,
                          None if scratch is None else scratch.partials)
    if n == 0:
        return output
    splits = min(int(splits), 64 - shared.splits)
    if splits < 1:
        raise ValueError("a step needs at least one split")
    slots = splits + shared.splits + 1
    if scratch is None or scratch.partials.shape[0] < n or scratch.splits != slots - 1 or scratch.partials.shape[1] != hq:
        rows = n * hq * slots
        buffer = torch.empty(rows * 257, dtype=torch.float32, device=query.device)
        partials = buffer.data_ptr()
        lse = partials + rows * 1024
    else:
        partials, lse = scratch.partials.data_ptr(), scratch.lse.data_ptr()
    query, key, value = _rows(query), _rows(key), _rows(value)
    qrot = _dense(qrot)
    columns = rv.stride() == (1, 256)  # a transposed rotation, as it lies
    rv = rv if columns else _dense(rv)
    tile = layout.config.queries_per_tile
    max_q = getattr(meta, "max_query_len", None)
    programs = min(attention_programs(n, meta.max_num_reqs, tile), meta.tasks.shape[0])
    if isinstance(max_q, int) and 0 < max_q < tile:
        tile = max_q
    with device:
        _lib.call("oscar_decode_attention_shared", qrot.data_ptr(), query.data_ptr(), query.stride(0), query.stride(1),
                  key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(), value.stride(0), value.stride(1),
                  history.data_ptr(), history.numel() // layout.stripe_page_bytes, window.data_ptr(),
                  meta.query_start_loc.data_ptr(), meta.seq_lens.data_ptr(), table.data_ptr(), table.shape[0],
                  meta.counts.data_ptr(), meta.tasks.data_ptr(), meta.task_count.data_ptr(), programs, n, rv.data_ptr(),
                  int(columns), shared.plan.data_ptr(), shared.max_reqs, shared.items, shared.splits, partials, lse,
                  output.data_ptr(), shared.geometry(table.stride(0), tile), float(scale), splits,
                  min(n, meta.max_num_reqs) if store_window else 0, _status(query), _stream(query))
    _checked("oscar_decode_attention_shared", query)
    return output


def decode_attention(qrot, query, key, value, history, window, meta, layout, scale, splits, rv, output, scratch=None,
                     store_window=True, shared=None):
    """History + raw attention, split merge, inverse V rotation, path merge and the
    window store of one decode / MTP-verify step (reference backend.py:195-226).

    ``shared`` (``prepare_shared_prefix``): the history that groups of requests share is
    attended once per group, and only the rest per request; ``splits`` is then at most
    64 - shared.splits (more is cut to that).

    ``meta.max_query_len`` bounds the queries per request, in every replay of a captured
    step too: capture with the most that a replay will have.  Rows of queries past it come
    back as NaN and set the status word (``read_status`` = 1)."""
    if shared is not None:
        return _decode_shared(qrot, query, key, value, history, window, meta, layout, scale, splits, rv, output, scratch,
                              store_window, shared)
    _require_cuda(qrot, query, key, value, history, window, rv, output)
    n, hq, _ = query.shape
    if n == 0:
        return output
    if scratch is None or scratch.partials.shape[0] < n or scratch.splits != splits:
        scratch = DecodeScratch(n, hq, splits, query.device)
    query, key, value = _rows(query), _rows(key), _rows(value)
    qrot = qrot.contiguous()
    rv = rv.contiguous()
    geo = _meta_common(meta, layout, hq)
    programs = min(attention_programs(n, meta.max_num_reqs, layout.config.queries_per_tile), meta.tasks.shape[0])
    window_programs = min(n, meta.max_num_reqs) if store_window else 0
    _lib.call("oscar_decode_attention", qrot.data_ptr(), query.data_ptr(), query.stride(0), query.stride(1),
              key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(), value.stride(0), value.stride(1),
              history.data_ptr(), window.data_ptr(), meta.query_start_loc.data_ptr(), meta.seq_lens.data_ptr(),
              meta.block_tables.data_ptr(), meta.counts.data_ptr(), meta.tasks.data_ptr(),
              meta.task_count.data_ptr(), programs, n, rv.data_ptr(), scratch.partials.data_ptr(),
              scratch.lse.data_ptr(), output.data_ptr(), geo, float(scale), int(splits), window_programs,
              _status(query), _stream(query))
    _checked("oscar_decode_attention", query)
    return output
