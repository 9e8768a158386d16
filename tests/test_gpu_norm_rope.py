"""``kernels.qk_norm_rope`` against the formula in 64 bits.

Tolerance: the arithmetic is fp32 (about a dozen roundings of 2^-24 each, relative to the
larger of the pair's two products) and the result is rounded once to bf16 (half a step,
2^-8 relative at most): |error| <= 2^-8 |y| + 2^-19 max(|a|, |b|) over the element's pair."""

import math

import pytest
import torch

from oscar_new_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"


def table(positions, rotary, dtype=torch.float32):
    f = torch.exp(-math.log(1e6) * torch.arange(0, rotary, 2, dtype=torch.float64) / max(rotary, 1))
    a = torch.arange(positions, dtype=torch.float64)[:, None] * f
    return torch.cat((a.cos(), a.sin()), 1).to(dtype).to(DEV)


def formula(x, w, offset, eps, rows, rotary, interleaved):
    """(y, magnitude of the element's pair) in 64 bits; rows = table rows of the tokens."""
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (w.double() + offset)
    z, size = y.clone(), y.abs()
    half = rotary // 2
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = rows[:, i, None].double(), rows[:, half + i, None].double()
        z[..., a] = y[..., a] * c - y[..., b] * s
        z[..., b] = y[..., b] * c + y[..., a] * s
        size[..., a] = size[..., b] = torch.maximum(y[..., a].abs(), y[..., b].abs())
    return z, size


def check(got, want):
    y, size = want
    nan = torch.isnan(y)
    assert torch.equal(torch.isnan(got), nan)
    err = (got.double() - y).abs()[~nan]
    bound = (y.abs() * 2**-8 + size * 2**-19)[~nan]
    assert bool((err <= bound).all()), float((err - bound).max())


@pytest.mark.parametrize("n,hq,h,rotary,interleaved,wt,tt,gated", [
    (1, 24, 4, 64, False, torch.bfloat16, torch.float32, True),
    (1, 1, 1, 16, False, torch.float32, torch.bfloat16, False),
    (7, 6, 1, 256, False, torch.float32, torch.float32, False),
    (33, 8, 1, 256, True, torch.bfloat16, torch.bfloat16, False),
    (64, 3, 5, 48, True, torch.float32, torch.float32, True),
    (129, 24, 4, 128, False, torch.bfloat16, torch.bfloat16, True),
    (257, 5, 0, 32, False, torch.float32, torch.float32, False),
    (5, 9, 2, 0, False, torch.float32, torch.float32, False),
    (2000, 24, 4, 64, True, torch.bfloat16, torch.float32, True),
])
def test_matches_the_formula(cuda_lib, n, hq, h, rotary, interleaved, wt, tt, gated):
    g = torch.Generator().manual_seed(n + rotary)
    wide = 512 if gated else 256
    fused = (torch.randn(n, hq * wide + h * 256, generator=g) * 10 ** (4 * torch.rand(n, 1, generator=g) - 2))
    fused = fused.bfloat16().to(DEV)
    q = fused[:, :hq * wide].unflatten(1, (hq, wide))[..., :256]
    k = fused[:, hq * wide:].unflatten(1, (h, 256)) if h else torch.zeros(n, 0, 256, dtype=torch.bfloat16, device=DEV)
    qw, kw = ((0.1 * torch.randn(256, generator=g)).to(wt).to(DEV) for _ in range(2))
    tab = table(500, rotary, tt) if rotary else torch.zeros(500, 0, device=DEV)
    pos = torch.randint(0, 500, (n,), generator=g).to(DEV)
    pos[0], pos[-1] = 499, 0
    before = fused.clone()
    for p in (pos, pos.int()):
        qo, ko = kernels.qk_norm_rope(q, k, qw, kw, p, tab, eps=1e-6, weight_offset=1.0, interleaved=interleaved)
        check(qo, formula(q, qw, 1.0, 1e-6, tab[pos], rotary, interleaved))
        check(ko, formula(k, kw, 1.0, 1e-6, tab[pos], rotary, interleaved))
    assert torch.equal(fused, before) and kernels.read_status(DEV) == 0


def test_in_place_rows_of_a_fused_buffer(cuda_lib):
    g = torch.Generator().manual_seed(1)
    fused = torch.randn(70, 4 * 512 + 4 * 256, generator=g).bfloat16().to(DEV)
    tab, pos = table(100, 64), torch.arange(70, device=DEV)
    w = torch.ones(256, device=DEV)
    views = lambda t: (t[:, :2048].unflatten(1, (4, 512))[..., :256], t[:, 2048:2560].unflatten(1, (2, 256)))  # noqa: E731
    want = kernels.qk_norm_rope(*views(fused), w, w, pos, tab)
    mine = fused.clone()
    q, k = views(mine)
    kernels.qk_norm_rope(q, k, w, w, pos, tab, query_out=q, key_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    rest = mine[:, :2048].unflatten(1, (4, 512))[..., 256:]
    assert torch.equal(rest, fused[:, :2048].unflatten(1, (4, 512))[..., 256:]) and torch.equal(mine[:, 2560:], fused[:, 2560:])


def test_odd_layouts_and_types_of_views(cuda_lib):
    g = torch.Generator().manual_seed(2)
    base = torch.randn(9, 3, 260, generator=g).bfloat16().to(DEV)
    q, k = base[..., 1:257], base[:, :1, 4:260].transpose(0, 1).contiguous().transpose(0, 1)
    w = torch.randn(512, generator=g).to(DEV)
    tab = table(64, 32, torch.bfloat16)
    wide = torch.zeros(64, 40, dtype=torch.bfloat16, device=DEV)
    wide[:, 3:35] = tab
    pos = torch.arange(18, device=DEV)[::2]
    qo, ko = kernels.qk_norm_rope(q, k, w[::2], w[1::2], pos, wide[:, 3:35], weight_offset=-0.5, interleaved=True)
    check(qo, formula(q, w[::2], -0.5, 1e-6, tab[pos], 32, True))
    check(ko, formula(k, w[1::2], -0.5, 1e-6, tab[pos], 32, True))


def test_zero_rows_large_rows_and_non_finite_rows(cuda_lib):
    q = torch.zeros(5, 2, 256, dtype=torch.bfloat16)
    q[1], q[2] = 2.0**50, 2.0**-70
    q[3, 0, 7], q[4, 1, 200] = float("nan"), float("inf")
    q[0, 1, 0] = 1.0
    q = q.to(DEV)
    w = torch.ones(256, device=DEV)
    tab, pos = table(8, 64), torch.arange(5, device=DEV)
    qo, ko = kernels.qk_norm_rope(q, q[:, :1], w, w, pos, tab, eps=1e-6)
    assert torch.equal(qo[0, 0], torch.zeros_like(qo[0, 0]))  # eps keeps the empty row finite
    check(qo[:3], formula(q[:3], w, 0.0, 1e-6, tab[pos[:3]], 64, False))
    # a non-finite element spoils its own row only
    assert torch.isnan(qo[3, 0]).all() and torch.isfinite(qo[3, 1]).all() and torch.isnan(ko[3, 0]).all()
    assert torch.isfinite(qo[4, 0]).all() and not torch.isfinite(qo[4, 1]).all()


def test_padding_and_positions_outside_the_table(cuda_lib):
    g = torch.Generator().manual_seed(3)
    q = torch.randn(6, 4, 256, generator=g).bfloat16().to(DEV)
    k = q[:, :2].contiguous()
    w, tab = torch.ones(256, device=DEV), table(10, 64)
    pos = torch.tensor([0, 9, 10, -1, 3, 1 << 40], device=DEV)
    qo, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    counts = torch.tensor([2, 5], dtype=torch.int32, device=DEV)
    kernels.read_status(DEV)
    kernels.qk_norm_rope(q, k, w, w, pos, tab, counts=counts, query_out=qo, key_out=ko)
    assert kernels.read_status(DEV) == 1 and kernels.read_status(DEV) == 0
    for t in (0, 1, 4):
        check(qo[t:t + 1], formula(q[t:t + 1], w, 0.0, 1e-6, tab[pos[t:t + 1]], 64, False))
    for t in (2, 3, 5):
        assert bool((qo[t] == 7).all()) and bool((ko[t] == 7).all())
    empty = kernels.qk_norm_rope(q[:0], k[:0], w, w, pos[:0], tab)
    assert empty[0].shape == (0, 4, 256) and empty[1].shape == (0, 2, 256)
    counts[1] = 0
    qo.fill_(7.0)
    kernels.qk_norm_rope(q, k, w, w, pos, tab, counts=counts, query_out=qo, key_out=ko)
    assert bool((qo == 7).all()) and kernels.read_status(DEV) == 0


def test_captured_replays_follow_their_inputs(cuda_lib):
    g = torch.Generator().manual_seed(4)
    q, k = torch.zeros(16, 4, 256, dtype=torch.bfloat16, device=DEV), torch.zeros(16, 1, 256, dtype=torch.bfloat16, device=DEV)
    w, tab, pos = torch.ones(256, device=DEV), table(128, 128), torch.zeros(16, dtype=torch.int64, device=DEV)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        kernels.qk_norm_rope(q, k, w, w, pos, tab)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qo, ko = kernels.qk_norm_rope(q, k, w, w, pos, tab)
    for seed in range(2):
        q.copy_(torch.randn(q.shape, generator=g))
        k.copy_(torch.randn(k.shape, generator=g))
        pos.copy_(torch.randint(0, 128, (16,), generator=g))
        graph.replay()
        check(qo, formula(q, w, 0.0, 1e-6, tab[pos], 128, False))
        check(ko, formula(k, w, 0.0, 1e-6, tab[pos], 128, False))


def test_strided_counts(cuda_lib):
    q = torch.randn(6, 4, 256, generator=torch.Generator().manual_seed(5)).bfloat16().to(DEV)
    k = q[:, :2].contiguous()
    w, tab = torch.ones(256, device=DEV), table(10, 64)
    pos = torch.arange(6, device=DEV)
    qo, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    counts = torch.tensor([2, 6, 3, 6], dtype=torch.int32, device=DEV)[::2]  # 3 active tokens
    kernels.qk_norm_rope(q, k, w, w, pos, tab, counts=counts, query_out=qo, key_out=ko)
    assert bool((qo[3:] == 7).all()) and not bool((qo[2] == 7).any())


@pytest.mark.parametrize("rows", [0, 3])
def test_no_rotation_takes_any_position(cuda_lib, rows):
    """rotary 0: norms alone, no table row is looked up."""
    g = torch.Generator().manual_seed(6)
    q = torch.randn(7, 4, 256, generator=g).bfloat16().to(DEV)
    k = torch.randn(7, 2, 256, generator=g).bfloat16().to(DEV)
    w, tab = torch.randn(256, generator=g).to(DEV), torch.zeros(rows, 0, device=DEV)
    pos = torch.tensor([0, 2, 3, -1, 1 << 40, 5, 1], device=DEV)
    kernels.read_status(DEV)
    for interleaved in (False, True):
        qo, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
        kernels.qk_norm_rope(q, k, w, w, pos, tab, interleaved=interleaved, query_out=qo, key_out=ko)
        assert kernels.read_status(DEV) == 0
        check(qo, formula(q, w, 0.0, 1e-6, tab, 0, interleaved))
        check(ko, formula(k, w, 0.0, 1e-6, tab, 0, interleaved))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("value", [float("inf"), -float("inf")])
def test_infinities_reach_what_the_formula_says(cuda_lib, interleaved, value):
    """An infinity makes the row's scale 0: its own dim is NaN, and the partner it turns with;
    dims that do not turn have no partner."""
    rotary, g = 64, torch.Generator().manual_seed(7)
    at = [0, 5, 37, 63, 64, 68, 100, 131, 200, 255]
    q = torch.randn(len(at), 3, 256, generator=g).bfloat16()
    for t, d in enumerate(at):
        q[t, 1, d] = value
    q = q.to(DEV)
    w, tab, pos = torch.randn(256, generator=g).to(DEV), table(40, rotary), torch.arange(1, len(at) + 1, device=DEV)
    qo, ko = kernels.qk_norm_rope(q, q[:, 1:2], w, w, pos, tab, interleaved=interleaved)
    check(qo, formula(q, w, 0.0, 1e-6, tab[pos], rotary, interleaved))
    check(ko, formula(q[:, 1:2], w, 0.0, 1e-6, tab[pos], rotary, interleaved))
    for t, d in enumerate(at):
        assert int(torch.isnan(qo[t, 1]).sum()) == (2 if d < rotary else 1)


def test_rows_beyond_32_bits(cuda_lib):
    n, hq = 360000, 24
    assert n * hq * 256 > 2**31
    q = torch.empty(n, hq, 256, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(n, 1, 256, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(8)
    some = torch.tensor([0, 1, 174762, 174763, 349525, 349526, n - 2, n - 1], device=DEV)
    q[some] = torch.randn(len(some), hq, 256, device=DEV, generator=g).bfloat16()
    k[some] = torch.randn(len(some), 1, 256, device=DEV, generator=g).bfloat16()
    w, tab, pos = torch.ones(256, device=DEV), table(1000, 64), torch.arange(n, device=DEV) % 1000
    qo, ko = kernels.qk_norm_rope(q, k, w, w, pos, tab)
    check(qo[some], formula(q[some], w, 0.0, 1e-6, tab[pos[some]], 64, False))
    check(ko[some], formula(k[some], w, 0.0, 1e-6, tab[pos[some]], 64, False))
