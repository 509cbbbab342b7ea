"""Tree attention where scores move the running maximum, against the plain
restatement in 64 bits."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import running_max as M
from test_paged_gpu import Case

pytestmark = pytest.mark.gpu
F = np.float32


def _set_scores(c, r, scores):
    """Raw scores of request ``r``'s positions, exactly: three parts of each in
    three columns of K, against ones in q."""
    page = c.k.shape[2]
    rest = torch.from_numpy(np.asarray(scores, dtype=np.float64))
    for col in range(3):
        part = rest.to(c.k.dtype)
        rest = rest - part.double()
        for b in range(-(-len(scores) // page)):
            rows = part[b * page:(b + 1) * page]
            c.k[c.table[r][b], :, :len(rows), col] = rows
    assert (rest == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("nodes", [1, 7, 14, 40])
def test_scores_at_the_headroom(cuda_device, dtype, D, nodes):
    """120 requests whose maximum rises several times, each time by a score
    that lies within a few roundings of the headroom."""
    R = 120
    scale = F(F(1 / np.sqrt(D)) * M.LOG2E)
    rng = np.random.default_rng(D + nodes)
    c = Case(D + nodes, [1100 + int(x) for x in rng.integers(0, 200, R)],
             [nodes if r % 8 == 0 else 1 for r in range(R)], 4, 1, D, 16, dtype)
    c.k[:] = 0
    c.q[:] = 0
    c.q[:, :, :3] = 1
    # fp16 holds 24 bits in three parts from 2^-2 up (its steps end at 2^-24)
    for r in range(R):
        n = c.ctx[r] + c.cu[r + 1] - c.cu[r]
        s0 = F(rng.uniform(1, 100))
        scores = (s0 - rng.uniform(2, 20, n) * 4).astype(F)
        scores = np.where(np.abs(scores) < 1, F(1), scores)
        scores[int(rng.integers(0, 100))] = s0
        for at in (150, 300, 450, 700, 1000):
            w = M.split_window(s0, scale) if rng.random() < 0.6 else None
            s0 = M.at_headroom(s0, scale, int(rng.integers(-2, 3))) if w is None else w
            scores[at + int(rng.integers(0, 60))] = s0
        _set_scores(c, r, scores)
    out, lse = c.run(out_dtype=torch.float32)
    c.check(out, lse)


@pytest.mark.parametrize("dtype,top", [(torch.bfloat16, 50), (torch.float16, 8)])
@pytest.mark.parametrize("nodes", [1, 3, 12, 40, 70])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_any_finite_size(cuda_device, dtype, top, nodes, sign):
    """Scores whose rounding is more than the headroom, up to 2^100: the
    position with the largest one has all the weight (two have half each)."""
    exps = [e for e in (4, 8, 12, 14, 17, 30, 50) if e <= top]
    R, n_ctx, D = len(exps), 900, 64
    c = Case(nodes, [n_ctx] * R, [nodes] * R, 4, 1, D, 16, dtype)
    c.mask[:] = False
    c.k[:] = 0
    c.q[:] = 0
    rng = np.random.default_rng(nodes)
    best = []
    for r, e in enumerate(exps):
        c.q[c.cu[r]:c.cu[r + 1], :, 0] = sign * 2.0 ** e
        a = rng.integers(1, 100, n_ctx)
        first, second = 37 + 40 * r, 700
        a[first], a[second] = (100, 100) if sign > 0 else (0, 0)
        best.append((first, second))
        page = c.k.shape[2]
        for b in range(-(-n_ctx // page)):
            rows = torch.from_numpy(a[b * page:(b + 1) * page]).to(dtype) * 2.0 ** e
            c.k[c.table[r][b], :, :len(rows), 0] = rows
    out, lse = c.run(out_dtype=torch.float32)
    assert torch.isfinite(out).all()
    for r, (x, y) in enumerate(best):
        gap = 4.0 ** exps[r] / math.sqrt(D)        # to every other position
        assert gap > 30
        page = c.v.shape[2]
        v = [c.v[c.table[r][p // page], 0, p % page].double() for p in (x, y)]
        want = (v[0] + v[1]) / 2
        got = out[c.cu[r]:c.cu[r + 1]].cpu().double()
        # two weights of 16 bits each; n weights of at most e^-gap beside them
        room = (v[0].abs() + v[1].abs()) * 2.0 ** -15 + n_ctx * 5 * math.exp(-gap)
        assert ((got - want).abs() <= room).all()
        wl = (100 * 4.0 ** exps[r] / math.sqrt(D) if sign > 0 else 0.0) + math.log(2)
        room = abs(wl) * 2.0 ** -21 + n_ctx * math.exp(-gap) + 2.0 ** -20
        assert ((lse[c.cu[r]:c.cu[r + 1]].cpu().double() - wl).abs() <= room).all()
    from halo_b200 import _lib as L
    assert L.device_error() == 0


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("D", [64, 128])
def test_maxima_that_rise_often(cuda_device, seed, D):
    """Contexts whose scores grow with the position, several rises a segment."""
    rng = np.random.default_rng(seed)
    nodes = [int(x) for x in rng.integers(1, 17, 40)]
    c = Case(seed, [int(x) for x in rng.integers(100, 2500, 40)], nodes, 4, 1, D, 16,
             torch.float16 if seed % 2 else torch.bfloat16)
    page = c.k.shape[2]
    for r, row in enumerate(c.table):
        n = -(-(c.ctx[r] + nodes[r]) // page)
        for b in range(n):
            c.k[row[b], :, :, 0] = c.k[row[b], :, :, 0] * 0.2 + 40.0 * (b + 1) / n
    c.q[:, :, 0] = 2.0 + rng.random()
    out, lse = c.run(out_dtype=torch.float32)
    c.check(out, lse)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nodes", [1, 7, 14, 20, 40])
def test_many_small_weights_beside_a_large_one(cuda_device, dtype, nodes):
    """One position 25.1 log2 units above 300000 equal ones whose V is 1 where
    its own is 0: their share, 0.8 % together, has to come out whole."""
    from halo_b200 import ops
    n, H, H_kv, D, page = 300_000, 32, 8, 64, 64
    dev = torch.device("cuda")
    n_pages = -(-(n + nodes) // page)
    k = torch.zeros(n_pages, H_kv, page, D, dtype=dtype, device=dev)
    v = torch.ones_like(k)
    table = torch.randperm(n_pages, generator=torch.Generator().manual_seed(1)).int()
    k[table[0], :, 5, 0] = 139.0
    v[table[0], :, 5] = 0
    q = torch.zeros(nodes, H, D, dtype=dtype, device=dev)
    q[:, :, 0] = 1
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)      # noqa: E731
    out, lse = ops.tree_attention(q, k, v, table[None].to(dev), i32([n]), i32([0, nodes]),
                                  torch.zeros(nodes, nodes, dtype=torch.bool, device=dev),
                                  out_dtype=torch.float32)
    w = math.exp(-139 / math.sqrt(D))                      # 2^-25.07 of the large one
    mass = (n - 1) * w
    want = mass / (1 + mass)
    # a weight is off by 2^-32 of the largest (fp16) and by 2^-16 of itself, an
    # exponential by 2^-21, sums of n keys as oracle.paged.allowed has them
    room = n * 2.0 ** -32 + mass * (2.0 ** -16 + 2.0 ** -20) + 2 * want * (n / 8 + 64) * 2.0 ** -23
    assert float((out.double() - want).abs().max()) <= room
    assert float((lse.double() - (139 / math.sqrt(D) + math.log1p(mass))).abs().max()) <= 1e-5


@pytest.mark.parametrize("nodes", [1, 5, 14, 20, 40, 70])
@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.float16),
                                     (128, torch.bfloat16), (64, torch.float16)])
@pytest.mark.parametrize("ctx", [130, 2000, 40000])
def test_infinities_of_the_context(cuda_device, nodes, D, dtype, ctx):
    """An infinity that a node sees is its column's value wherever it lies and
    however small its weight, as one of a drafted row is; other columns are as
    they were."""
    c = Case(ctx + nodes, [ctx, 70], [nodes, 2], 4, 1, D, 16, dtype)
    page = 16

    def put(r, pos, col, x):
        c.v[c.table[r][pos // page], 0, pos % page, col] = x
    low = ctx // 2                           # a position whose weight ends as zero
    c.k[c.table[0][low // page], 0, low % page] = 0
    c.k[c.table[0][low // page], 0, low % page, 1] = -300
    c.q[:, :, 1] = 60.0
    c.k[:, :, :, 1].clamp_(max=1)
    bad = {0: math.inf, 3: -math.inf, 5: math.nan, 31: math.nan, 40: math.inf, D - 1: -math.inf}
    spots = {0: [(0, math.inf)], 3: [(ctx - 1, -math.inf)], 5: [(127, math.nan)],
             31: [(2, math.inf), (ctx - 3, -math.inf)], 40: [(low, math.inf)],
             D - 1: [(at, -math.inf) for at in range(1, ctx, 7)]}
    for col, at in spots.items():
        for pos, x in at:
            put(0, pos, col, x)
    out, lse = c.run(out_dtype=torch.float32)
    half, _ = c.run()
    for o in (out.cpu(), half.float().cpu()):
        for col, x in bad.items():
            got = o[:nodes, :, col]
            assert torch.isnan(got).all() if math.isnan(x) else (got == x).all(), col
        for col in spots:
            assert torch.isfinite(o[nodes:]).all()
    for col, at in spots.items():            # the oracle's other columns
        for pos, _ in at:
            put(0, pos, col, 0.0)
        out[:nodes, :, col] = 0
    keep = [x for x in range(D) if x not in spots]
    c.v[:, :, :, list(spots)] = 0
    out[:, :, list(spots)] = 0
    assert torch.isfinite(out).all() and len(keep) == D - len(spots)
    c.check(out, lse)


def test_accepting_an_infinity_keeps_the_answer(cuda_device):
    """A node's infinity gives the same output drafted and accepted."""
    from test_paged_gpu import _i32, _small_cache
    cache = _small_cache(12)
    got = cache.extend(_i32([2, 0]), 2)
    k = torch.ones(2, 1, 64, dtype=torch.bfloat16, device="cuda")
    v = k.clone()
    v[0, 0, 9] = math.inf
    q = torch.rand(2, 4, 64, device="cuda").bfloat16()
    mask = torch.ones(2, 2, dtype=torch.bool, device="cuda")
    cache.write(0, k, v, got)
    drafted = cache.attend(0, q, got, mask)[0][1]
    cache.accept(None, _i32([1, 0]))
    got = cache.extend(_i32([1, 0]), 1)
    cache.write(0, k[1:], v[1:], got)
    accepted = cache.attend(0, q[1:], got, mask[1:, :1])[0][0]
    assert (drafted[:, 9] == math.inf).all()
    assert torch.equal(drafted, accepted)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nodes", [2, 30])
@pytest.mark.parametrize("scale", [1e-40, 1e-38, 1e-30, 1e-6])
def test_scales_that_leave_a_mean(cuda_device, dtype, nodes, scale):
    """Weights that are all one: the headroom of a raw score may be infinite."""
    c = Case(nodes, [700, 50], [nodes, 1], 4, 1, 64, 16, dtype)
    out, lse = c.run(out_dtype=torch.float32, scale=scale)
    c.check(out, lse, scale=scale)


@pytest.mark.parametrize("nodes", [3, 30])
def test_infinities_everywhere(cuda_device, nodes):
    """Every column of a long context holds infinities: no wait runs out."""
    from halo_b200 import _lib as L
    c = Case(nodes, [100000], [nodes], 4, 1, 128, 64, torch.bfloat16)
    c.v[c.table[0][::3]] = math.inf
    out, lse = c.run(out_dtype=torch.float32)
    assert (out == math.inf).all() and torch.isfinite(lse).all() and L.device_error() == 0


@pytest.mark.parametrize("nodes", [1, 6, 16, 33])
@pytest.mark.parametrize("want_lse", [True, False])
def test_infinities_of_many_requests(cuda_device, nodes, want_lse):
    """Segments that one CTA finishes by itself, every third request with
    infinities in some columns and every seventh with K that is NaN as well."""
    R, D, page = 330, 64, 16
    rng = np.random.default_rng(nodes)
    ctx = [int(x) for x in rng.integers(1, 500, R)]
    c = Case(nodes, ctx, [nodes if r % 5 else 1 for r in range(R)], 4, 1, D, page, torch.bfloat16)
    keep_v, keep_k = c.v.clone(), c.k.clone()
    bad, dead = list(range(0, R, 3)), list(range(0, R, 21))
    for r in bad:
        pos = int(rng.integers(0, ctx[r]))
        c.v[c.table[r][pos // page], 0, pos % page, 7] = math.inf
        c.v[c.table[r][0], 0, 0, 8] = -math.inf
    for r in dead:
        c.k[c.table[r][0], 0, 0, 3] = math.nan
    out, lse = c.run(out_dtype=torch.float32, want_lse=want_lse)
    assert (lse is not None) == want_lse
    out = out.cpu()
    for r in bad:
        rows = slice(c.cu[r], c.cu[r + 1])
        if r in dead:
            assert torch.isnan(out[rows]).all() and (lse is None or torch.isnan(lse[rows]).all())
        else:
            assert (out[rows, :, 7] == math.inf).all() and (out[rows, :, 8] == -math.inf).all()
        out[rows, :, 7:9] = 0
        # its own pages: entries behind them name other requests' pages
        keep_v[c.table[r][:-(-(ctx[r] + c.cu[r + 1] - c.cu[r]) // page)], :, :, 7:9] = 0
    c.v, c.k = keep_v, keep_k
    rows = [t for r in range(R) if r not in dead for t in range(c.cu[r], c.cu[r + 1])]
    c.check(out, lse if want_lse else c.run()[1], rows=rows)
