"""Shared-prefix decode on the CPU: plan sizes and the refusals of the wrappers and the C
entry points, all before any device work."""

from types import SimpleNamespace

import pytest
import torch

from oscar_new_b200 import _lib, kernels
from oscar_new_b200.layout import CacheLayout
from tests.helpers import make_config

LAYOUT = CacheLayout(768, kv_heads=4, config=make_config(4, 64))


def meta(reqs=3, query=1):
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    return SimpleNamespace(query_start_loc=i(reqs + 1), seq_lens=i(reqs), block_tables=i(reqs, 12), counts=i(2),
                           tasks=i(reqs, 2), task_count=i(1), num_reqs=reqs, max_num_reqs=reqs, max_query_len=query)


def test_plan_sizes_hold_every_row_tile():
    # 64 requests x 6 rows a KV head: 3 tiles and 32 groups at most, 4 waves of splits over 4 heads
    plan = kernels.SharedPrefix(64, 64, 24, LAYOUT, "cpu")
    assert plan.items == 64 * 6 // 128 + 32 + 1 + 148
    assert plan.plan.numel() == 8 + 2 * 64 + 8 * plan.items and not plan.plan.any()
    assert plan.splits == 37 and kernels.SharedPrefix(4, 4, 8, CacheLayout(768, 1), "cpu").splits == 48
    # the split scratch bounds the splits of a long step
    assert kernels.SharedPrefix(4, 4096, 24, LAYOUT, "cpu").splits == (256 << 20) // (4096 * 24 * 1024)
    assert kernels.SharedPrefix(4, 1 << 20, 24, LAYOUT, "cpu").splits == 1


@pytest.mark.parametrize("splits", [0, 64, -3])
def test_split_counts_out_of_range_are_refused(splits):
    with pytest.raises(ValueError, match="1 to 63"):
        kernels.SharedPrefix(4, 4, 24, LAYOUT, "cpu", splits=splits)


def test_bad_plan_sizes_are_refused():
    for reqs, tokens, hq, h in ((0, 4, 8, 1), (8193, 4, 8, 1), (4, -1, 8, 1), (4, 4, 9, 2), (4, 4, 0, 1)):
        sizes = torch.zeros(2, dtype=torch.int64)
        assert _lib.lib().oscar_shared_prefix_layout(reqs, tokens, hq, h, sizes.data_ptr()) == 1
    assert _lib.lib().oscar_shared_prefix_layout(4, 4, 8, 1, None) == 1


def test_prepare_refuses():
    ok = torch.zeros(3, dtype=torch.int32)
    for groups, lens in ((ok.long(), ok), (ok, ok.float()), (ok[:2], ok), (ok, ok[None])):
        with pytest.raises(ValueError, match="entry per request"):
            kernels.prepare_shared_prefix(meta(), groups, lens, LAYOUT, 24)
    with pytest.raises(RuntimeError, match="CUDA device only"):
        kernels.prepare_shared_prefix(meta(), ok, ok, LAYOUT, 24)
    plan = kernels.SharedPrefix(3, 3, 24, LAYOUT, "cpu")
    with pytest.raises(ValueError, match="other heads"):
        kernels.prepare_shared_prefix(meta(), ok, ok, LAYOUT, 12, shared=plan)
    with pytest.raises(ValueError, match="another layout"):
        kernels.prepare_shared_prefix(meta(), ok, ok, CacheLayout(1024, 4, config=LAYOUT.config), 24, shared=plan)
    big = kernels.SharedPrefix(5, 5, 24, LAYOUT, "cpu")
    with pytest.raises(ValueError, match="the plan's 5 entries"):
        kernels.prepare_shared_prefix(meta(), ok, ok, LAYOUT, 24, shared=big)
    with pytest.raises(ValueError, match="fewer requests"):
        kernels.prepare_shared_prefix(meta(5), torch.zeros(5, dtype=torch.int32), torch.zeros(5, dtype=torch.int32), LAYOUT,
                                      24, shared=plan)


def decode_args(n=3, hq=24):
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    pages = 2 * LAYOUT.stripe_page_bytes
    return dict(qrot=b(n, hq, 256), query=b(n, hq, 256), key=b(n, 4, 256), value=b(n, 4, 256),
                history=torch.zeros(pages, dtype=torch.uint8), window=b(pages // 2), meta=meta(n), layout=LAYOUT, scale=0.1,
                splits=8, rv=b(256, 256), output=b(n, hq * 256), shared=kernels.SharedPrefix(n, n, hq, LAYOUT, "cpu"))


@pytest.mark.parametrize("change,text", [
    (dict(scale=0.0), "positive softmax scale"),
    (dict(scale=-1.0), "positive softmax scale"),
    (dict(scale=float("nan")), "positive softmax scale"),
    (dict(history=torch.zeros(100, dtype=torch.uint8)), "whole contiguous pages"),
    (dict(output=torch.zeros(3, 24 * 256)), "contiguous bf16"),
    (dict(output=torch.zeros(3, 24 * 255, dtype=torch.bfloat16)), "contiguous bf16"),
    (dict(qrot=torch.zeros(2, 24, 256, dtype=torch.bfloat16)), "qrot must be bf16"),
    (dict(qrot=torch.zeros(3, 24, 256)), "qrot must be bf16"),
    (dict(rv=torch.zeros(256, 128, dtype=torch.bfloat16)), "qrot must be bf16"),
    (dict(key=torch.zeros(3, 2, 256, dtype=torch.bfloat16)), "KV heads"),
    (dict(value=torch.zeros(2, 4, 256, dtype=torch.bfloat16)), "KV heads"),
    (dict(shared=kernels.SharedPrefix(2, 3, 24, LAYOUT, "cpu")), "fewer requests"),
    (dict(shared=kernels.SharedPrefix(3, 3, 12, LAYOUT, "cpu")), "other heads"),
])
def test_decode_refuses(change, text):
    with pytest.raises(ValueError, match=text):
        kernels.decode_attention(**{**decode_args(), **change})


def test_decode_on_the_host_is_refused():
    with pytest.raises(RuntimeError, match="CUDA device only"):
        kernels.decode_attention(**decode_args())


def test_c_entries_refuse_before_any_launch():
    lib, p = _lib.lib(), 1 << 20  # never dereferenced
    geo = kernels.geometry(LAYOUT, 24, 12)
    prep = lambda **k: lib.oscar_prepare_shared_prefix(*{**dict(q=p, s=p, c=p, g=p, l=p, r=3, i=10, n=8, geo=geo, plan=p,  # noqa: E731
                                                               st=None), **k}.values())
    for bad in (dict(q=None), dict(s=None), dict(c=None), dict(g=None), dict(l=None), dict(r=0), dict(r=8193), dict(i=0),
                dict(n=0), dict(n=64), dict(plan=None), dict(plan=p + 4)):
        assert prep(**bad) == 1, bad
    names = dict(qrot=p, q=p, qs0=6144, qs1=256, k=p, ks0=1024, ks1=256, v=p, vs0=1024, vs1=256, hist=p, pages=4, win=p,
                 qst=p, seq=p, tab=p, rows=3, counts=p, tasks=p, tc=p, nt=3, n=3, rv=p, rvc=0, plan=p, reqs=3, items=10, ps=8,
                 part=p, lse=p, out=p, geo=geo, scale=0.1, splits=8, wp=3, status=None, stream=None)
    call = lambda **k: lib.oscar_decode_attention_shared(*{**names, **k}.values())  # noqa: E731
    for bad in (dict(plan=None), dict(reqs=0), dict(items=0), dict(ps=0), dict(ps=64), dict(pages=0), dict(pages=1 << 31),
                dict(scale=0.0), dict(scale=-0.5), dict(rows=0), dict(splits=57), dict(splits=0), dict(n=-1), dict(qrot=None),
                dict(qrot=p + 8), dict(qs0=6140), dict(hist=None), dict(part=None), dict(out=p + 2), dict(wp=-1)):
        assert call(**bad) == 1, bad
    assert call(n=0) == 0


@pytest.mark.parametrize("name", ["query_start_loc", "seq_lens", "counts"])
def test_metadata_that_the_plan_would_misread_is_refused(name):
    ok = torch.zeros(3, dtype=torch.int32)
    for bad in (lambda t: t.long(), lambda t: torch.stack((t, t), 1)[:, 0], lambda t: t[None]):
        m = meta()
        setattr(m, name, bad(getattr(m, name)))
        with pytest.raises(ValueError, match=name):
            kernels.prepare_shared_prefix(m, ok, ok, LAYOUT, 24)


def test_a_plan_used_by_two_callers_keeps_their_geometries_apart():
    plan = kernels.SharedPrefix(3, 3, 24, LAYOUT, "cpu")
    four, one, wide = plan.geometry(12, 4), plan.geometry(12, 1), plan.geometry(24, 4)
    assert (four.query_tile, one.query_tile, wide.query_tile) == (4, 1, 4)
    assert (four.table_stride, one.table_stride, wide.table_stride) == (12, 12, 24)


@pytest.mark.parametrize("window", [
    torch.zeros(LAYOUT.stripe_page_bytes - 8, dtype=torch.bfloat16), torch.zeros(LAYOUT.stripe_page_bytes, dtype=torch.float16),
    torch.zeros(2 * LAYOUT.stripe_page_bytes, dtype=torch.bfloat16)[::2]])
def test_windows_other_than_the_caches_are_refused(window):
    with pytest.raises(ValueError, match="window view"):
        kernels.decode_attention(**{**decode_args(), "window": window})


def test_a_history_of_another_type_is_refused():
    with pytest.raises(ValueError, match="whole contiguous pages"):
        kernels.decode_attention(**{**decode_args(), "history": torch.zeros(LAYOUT.stripe_page_bytes, dtype=torch.bfloat16)})


@pytest.mark.parametrize("name,rows", [("query_start_loc", 3), ("seq_lens", 2), ("counts", 1)])
def test_metadata_of_fewer_requests_is_refused_by_the_plan(name, rows):
    ok, m = torch.zeros(3, dtype=torch.int32), meta()
    setattr(m, name, getattr(m, name)[:rows])
    with pytest.raises(ValueError, match=name):
        kernels.prepare_shared_prefix(m, ok, ok, LAYOUT, 24)


def test_block_tables_of_fewer_requests_are_refused():
    a = decode_args()
    a["meta"].block_tables = a["meta"].block_tables[:2]
    with pytest.raises(ValueError, match="block table"):
        kernels.decode_attention(**a)
