"""PagedKVCache where a step does not go as planned: given up, refused in the
middle of a batch, accepted by paths that leave it.  Against the plain
restatements of ``oracle/paged.py`` and dense attention over the rows kept."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged as O
from test_paged_gpu import _dense, _i32, _owners, _rows_of, _small_cache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _case(rng, R, width, page, spare):
    top = width * page
    held = [int(x) for x in rng.integers(0, top + 1, R)]
    ctx = [int(rng.integers(0, h + 1)) if rng.random() < 0.6 else h for h in held]
    counts = [int(x) for x in rng.integers(-2, 3 * page, R)]
    for r in range(R):
        x = rng.random()
        if x < 0.05:
            counts[r] = 2 ** 31 - 1
        elif x < 0.1:
            counts[r] = top - ctx[r]             # the whole table row
        elif x < 0.13:
            ctx[r] = held[r] + 3                 # no state of a cache: refused
    blocks = [-(-n // page) for n in held]
    order = rng.permutation(sum(blocks) + spare).astype(int).tolist()
    table = [[-7] * width for _ in range(R)]
    for r, n in enumerate(blocks):
        table[r][:n], order = order[:n], order[n:]
    return table, held, ctx, counts, order + [-9] * sum(blocks), len(order)


@pytest.mark.parametrize("R,width,page,spare,top", [
    (1, 1, 16, 0, 8), (1, 3, 5, 2, 40), (7, 4, 16, 6, 300), (64, 6, 24, 500, 6000),
    (1025, 3, 8, 700, 20000), (8192, 2, 16, 3000, 9000)])
@pytest.mark.parametrize("seed", [0, 1])
def test_extend_block_tables(cuda_device, R, width, page, spare, top, seed):
    from halo_b200 import ops
    rng = np.random.default_rng(seed * 1000 + R)
    table, held, ctx, counts, free, n_free = _case(rng, R, width, page, spare)
    want = O.extend_block_tables(table, held, ctx, counts, free, n_free, page, top)
    t, h, f, n, rows = _i32(table), _i32(held), _i32(free), _i32([n_free]), _i32([-5] * R)
    slots, pos, cu = ops.extend_block_tables(t, h, _i32(ctx), _i32(counts), rows, f, n,
                                             page_size=page, max_tokens=top)
    got = (t.tolist(), f.tolist(), int(n), slots.tolist(), pos.tolist(), cu.tolist(), rows.tolist(),
           h.tolist())
    for name, a, b in zip(("table", "free", "n_free", "slots", "positions", "cu", "rows", "held"),
                          got, want):
        assert a == b, name


@pytest.mark.parametrize("first,then", [([3, 9], [3, 9]), ([3, 9], [5, 20]), ([12, 20], [1, 2]),
                                        ([4, 0], [0, 4]), ([9, 9], [-1, 40])])
def test_a_step_that_is_given_up(cuda_device, first, then):
    """extend again without accept: the rows begin behind the context again,
    as in a cache that never saw the first step."""
    cache, fresh = _small_cache(12), _small_cache(12)
    cache.extend(_i32(first), 40)
    got, want = cache.extend(_i32(then), 40), fresh.extend(_i32(then), 40)
    assert got.cu.tolist() == want.cu.tolist()
    assert got.positions.tolist() == want.positions.tolist()
    assert _owners(cache) == list(range(12))
    T = 40
    g = torch.Generator().manual_seed(0)
    k = torch.randn(T, 1, 64, generator=g).bfloat16().to(DEV)
    q = torch.randn(T, 4, 64, generator=g).bfloat16().to(DEV)
    mask = torch.ones(T, 40, dtype=torch.bool, device=DEV)
    outs = []
    for c, rows in ((cache, got), (fresh, want)):
        c.write(0, k, k, rows)
        outs.append(c.attend(0, q, rows, mask)[0][:rows.cu[-1]])
        c.accept(None, _i32([2, 3]))
    assert torch.equal(*outs) and cache.lens.tolist() == fresh.lens.tolist()
    for r in range(2):
        assert _rows_of(cache, r) == _rows_of(fresh, r)
    assert _owners(cache) == list(range(12))
    # nothing is kept of a step given up, nor twice of one
    n = cache.lens.tolist()
    cache.accept(None, _i32([5, 5]))
    assert cache.lens.tolist() == n


def test_a_step_refused_after_one_given_up(cuda_device):
    cache = _small_cache(6)
    cache.extend(_i32([6, 2]), 8)
    got = cache.extend(_i32([6, 60]), 70)            # the second wants more than there is
    assert got.cu.tolist() == [0, 6, 6]
    cache.accept(None, _i32([6, 2]))
    assert cache.lens.tolist() == [16, 6] and _owners(cache) == list(range(6))
