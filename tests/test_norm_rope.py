"""Refusals of ``kernels.qk_norm_rope``, on the CPU: host checks of the wrapper and of the
C entry point, all before any device work."""

import pytest
import torch

from oscar_new_b200 import _lib, kernels


def args(n=3, hq=4, h=2, rotary=64):
    return dict(query=torch.zeros(n, hq, 256, dtype=torch.bfloat16), key=torch.zeros(n, h, 256, dtype=torch.bfloat16),
                q_weight=torch.ones(256), k_weight=torch.ones(256), positions=torch.zeros(n, dtype=torch.int64),
                cos_sin=torch.zeros(8, rotary))


@pytest.mark.parametrize("change,text", [
    (dict(query=torch.zeros(3, 4, 128, dtype=torch.bfloat16)), "query: expected bf16"),
    (dict(key=torch.zeros(3, 2, 256)), "key: expected bf16"),
    (dict(key=torch.zeros(2, 2, 256, dtype=torch.bfloat16)), "same tokens"),
    (dict(positions=torch.zeros(4, dtype=torch.int64)), "same tokens"),
    (dict(positions=torch.zeros(3, dtype=torch.int16)), "int64 or int32"),
    (dict(q_weight=torch.ones(256, dtype=torch.bfloat16)), "both of one type"),
    (dict(k_weight=torch.ones(128)), "both of one type"),
    (dict(cos_sin=torch.zeros(8, 40)), "multiple of 16"),
    (dict(cos_sin=torch.zeros(8, 272)), "multiple of 16"),
    (dict(cos_sin=torch.zeros(8, 64, dtype=torch.float16)), "table must be fp32 or bf16"),
    (dict(q_weight=torch.ones(256).half(), k_weight=torch.ones(256).half()), "weights must be fp32 or bf16"),
    (dict(counts=torch.zeros(2, dtype=torch.int64)), "counts are int32"),
    (dict(counts=torch.zeros(1, dtype=torch.int32)), "counts are int32"),
    (dict(eps=-1e-6), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(query_out=torch.zeros(3, 4, 256)), "bf16 output"),
    (dict(key_out=torch.zeros(3, 3, 256, dtype=torch.bfloat16)), "bf16 output"),
    (dict(key_out=torch.zeros(3, 2, 260, dtype=torch.bfloat16)[..., :256]), "16-byte aligned"),
    (dict(key_out=torch.zeros(1, 1, 256, dtype=torch.bfloat16).expand(3, 2, 256)), "overlap each other"),
    (dict(key_out=torch.zeros(1024, dtype=torch.bfloat16).as_strided((3, 2, 256), (256, 256, 1))), "overlap each other"),
    (dict(key_out=torch.zeros(1536, dtype=torch.bfloat16).as_strided((3, 2, 256), (512, 128, 1))), "overlap each other"),
])
def test_bad_arguments_are_refused(change, text):
    with pytest.raises(ValueError, match=text):
        kernels.qk_norm_rope(**{**args(), **change})


def test_host_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA device only"):
        kernels.qk_norm_rope(**args())


def test_outputs_over_other_rows_are_refused():
    fused = torch.zeros(3, 6 * 256, dtype=torch.bfloat16)
    a = args()
    a["query"], a["key"] = fused[:, :1024].unflatten(1, (4, 256)), fused[:, 1024:].unflatten(1, (2, 256))
    # in place: reaches the device check, so the overlap rules let it pass
    with pytest.raises(RuntimeError, match="CUDA device only"):
        kernels.qk_norm_rope(**a, query_out=a["query"], key_out=a["key"])
    with pytest.raises(RuntimeError, match="CUDA device only"):
        kernels.qk_norm_rope(**a, key_out=a["key"])
    for bad in (dict(query_out=fused[:, 256:1280].unflatten(1, (4, 256))),  # shifted over itself and the key
                dict(key_out=fused[:, :512].unflatten(1, (2, 256))),  # over the query
                dict(key_out=fused.view(-1)[512:512 + 3 * 512].view(3, 2, 256)),
                dict(query_out=torch.zeros(3, 4, 256, dtype=torch.bfloat16), key_out=fused[:, 512:1024].unflatten(1, (2, 256)))):
        with pytest.raises(ValueError, match="overlaps rows"):
            kernels.qk_norm_rope(**a, **bad)
    both = torch.zeros(3, 4, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="overlaps rows"):  # the two outputs over each other
        kernels.qk_norm_rope(**a, query_out=both, key_out=both[:, :2])


def test_c_entry_refuses_before_any_launch():
    h = _lib.lib()
    p = 1 << 20  # never dereferenced

    def call(**kw):
        a = dict(q=p, qs0=1024, qs1=256, k=p, ks0=512, ks1=256, n=3, hq=4, hkv=2, qw=p, kw=p, wf=1, off=0.0, eps=1e-6,
                 pos=p, p64=1, tab=p, tf=1, mp=8, rot=64, il=0, counts=None, qo=p, qos0=1024, qos1=256, ko=p,
                 kos0=512, kos1=256)
        a.update(kw)
        return h.oscar_qk_norm_rope(*a.values(), None, None)

    for bad in (dict(n=-1), dict(hq=-1), dict(rot=24), dict(rot=272), dict(rot=-16), dict(eps=-1.0), dict(pos=None),
                dict(tab=None), dict(q=None), dict(qo=None), dict(k=None), dict(ko=None), dict(qw=None),
                dict(q=p + 2), dict(ko=p + 8), dict(qs0=1020), dict(kos1=4), dict(mp=-1), dict(tab=p + 4)):
        assert call(**bad) == 1, bad
    assert call(n=0) == 0


def test_one_token_in_place_under_another_stride():
    """A dim of one element has no stride that matters: the rows are the input's own."""
    fused = torch.zeros(2, 6 * 256, dtype=torch.bfloat16)
    flat, a = fused.view(-1), args(n=1)
    a["query"], a["key"] = fused[:, :1024].unflatten(1, (4, 256))[:1], fused[:, 1024:].unflatten(1, (2, 256))[:1]
    q, k = flat[:1024].view(1, 4, 256), flat[1024:1536].view(1, 2, 256)
    assert q.stride() != a["query"].stride() and k.stride() != a["key"].stride()
    with pytest.raises(RuntimeError, match="CUDA device only"):
        kernels.qk_norm_rope(**a, query_out=q, key_out=k)
    with pytest.raises(ValueError, match="overlaps rows"):
        kernels.qk_norm_rope(**a, query_out=q, key_out=flat[512:1024].view(1, 2, 256))
