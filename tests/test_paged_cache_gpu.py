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
    starts = _i32([-5] * R)
    slots, pos, cu = ops.extend_block_tables(t, h, _i32(ctx), _i32(counts), rows, starts, f, n,
                                             page_size=page, max_tokens=top)
    got = (t.tolist(), f.tolist(), int(n), slots.tolist(), pos.tolist(), cu.tolist(), rows.tolist(),
           starts.tolist(), h.tolist())
    for name, a, b in zip(("table", "free", "n_free", "slots", "positions", "cu", "rows", "starts",
                           "held"), got, want):
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


@pytest.mark.parametrize("refused", ["table", "pool"])
@pytest.mark.parametrize("nodes", [3, 20])
@pytest.mark.parametrize("captured", [False, True])
def test_requests_behind_a_refused_one_keep_their_rows(cuda_device, refused, nodes, captured):
    """K, V and q are packed by the counts; a request in the middle is refused.
    The others' rows are stored, attended and accepted as theirs."""
    from halo_b200 import PagedKVCache
    H, H_kv, D, page, n0 = 8, 2, 64, 16, [20, 35, 3, 50]
    cache = PagedKVCache(1, 12 if refused == "pool" else 60, H_kv, D, max_requests=4,
                         max_len=400 if refused == "pool" else 80, page_size=page,
                         dtype=torch.float16, device=DEV)
    g = torch.Generator().manual_seed(nodes)
    rand = lambda *s: torch.randn(*s, generator=g).half()          # noqa: E731
    k0, v0 = rand(sum(n0), H_kv, D), rand(sum(n0), H_kv, D)
    cache.write(0, k0.to(DEV), v0.to(DEV), cache.extend(_i32(n0), sum(n0)))
    cache.accept(None, _i32(n0))
    # pages held: 2, 3, 1, 4; the last needs no page
    counts = [4, 200 if refused == "pool" else 50, nodes, min(nodes, 14)]
    granted = [True, False, nodes <= 13 or refused == "table", True]
    T = sum(counts) + 2
    k, v, q = rand(T, H_kv, D), rand(T, H_kv, D), rand(T, H, D)
    mask = (torch.rand(T, max(counts), generator=g) < 0.6) | torch.eye(T, max(counts)).bool()
    path, lens = _i32([[1, 2, 3], [0, 1, 2], [0, 2, 0], [2, 0, 0]]), _i32([3, 3, 2, 1])
    kd, vd, qd, md, cd = (x.to(DEV) for x in (k, v, q, mask, torch.tensor(counts, dtype=torch.int32)))
    out = torch.full((T, H, D), 7.0, device=DEV)
    lse = torch.full((T, H), 7.0, device=DEV)

    def step():
        rows = cache.extend(cd, T)
        cache.write(0, kd, vd, rows)
        cache.attend(0, qd, rows, md, out=out, lse=lse)
        cache.accept(path, lens)
        return rows
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            rows = step()
        graph.replay()
    else:
        rows = step()
    assert (rows.cu[1:] - rows.cu[:-1]).tolist() == [c if ok else 0 for c, ok in zip(counts, granted)]
    at, old, kept = 0, 0, []
    for r, (n, c) in enumerate(zip(n0, counts)):
        kk, vv = k0[old:old + n], v0[old:old + n]
        if granted[r]:
            seen = torch.cat([torch.ones(c, n, dtype=torch.bool), mask[at:at + c, :c]], 1)
            want = _dense(q[at:at + c], torch.cat([kk, k[at:at + c]]), torch.cat([vv, v[at:at + c]]),
                          seen)
            assert float((out[at:at + c].cpu() - want).abs().max()) < 1e-3
            pick = path[r, :int(lens[r])].tolist()
            kept.append((torch.cat([kk, k[at:at + c][pick]]), torch.cat([vv, v[at:at + c][pick]])))
        else:
            assert (out[at:at + c] == 7).all() and (lse[at:at + c] == 7).all()
            assert (rows.slots[at:at + c] == -1).all() and (rows.positions[at:at + c] == -1).all()
            kept.append((kk, vv))
        at, old = at + c, old + n
    assert (out[at:] == 7).all() and rows.slots[at:].tolist() == [-1, -1]
    assert cache.lens.tolist() == [x.shape[0] for x, _ in kept] == cache.held.tolist()
    for r, (kk, vv) in enumerate(kept):
        pages = cache.block_tables[r, :-(-kk.shape[0] // page)].tolist()
        assert torch.equal(O.gather_rows(cache.k[0].cpu(), pages, kk.shape[0]), kk.double().transpose(0, 1))
        assert torch.equal(O.gather_rows(cache.v[0].cpu(), pages, kk.shape[0]), vv.double().transpose(0, 1))
    assert _owners(cache) == list(range(cache.k[0].shape[0]))


@pytest.mark.parametrize("node", [3, 7, 10, 13, 53, 2 ** 31 - 1, -1, -2 ** 31])
def test_accept_of_nodes_that_are_not_of_the_step(cuda_device, node):
    """The entries behind a request's rows still name pages it gave back, which
    are another's now: none of their rows comes into its context."""
    cache = _small_cache(8)
    cache.extend(_i32([30, 0]), 30)                        # 5 pages of request 0
    cache.accept(None, _i32([0, 0]))                       # given back, entries stay
    got = cache.extend(_i32([0, 30]), 30)
    x = torch.full((30, 1, 64), 9., dtype=torch.bfloat16, device=DEV)
    cache.write(0, x, x, got)
    cache.accept(None, _i32([0, 30]))
    stale = cache.block_tables[0, 2:5].tolist()
    assert set(stale) & set(cache.block_tables[1, :5].tolist())
    got = cache.extend(_i32([3, 0]), 3)
    y = torch.tensor([4., 5., 6.], device=DEV)[:, None, None].expand(3, 1, 64).bfloat16()
    cache.write(0, y, y, got)
    cache.accept(_i32([[0, node, 2], [0, 0, 0]]), _i32([3, 0]))
    assert _rows_of(cache, 0) == [1.] * 10 + [4., 5., 6.]
    assert _rows_of(cache, 1) == [2.] * 6 + [9.] * 30 and _owners(cache) == list(range(8))
    got = cache.extend(_i32([3, 0]), 3)
    cache.write(0, y, y, got)
    cache.accept(_i32([[2, node, 0], [0, 0, 0]]), _i32([2, 0]))
    assert _rows_of(cache, 0) == [1.] * 10 + [4., 5., 6., 6., 5.]


def test_extend_by_one_count_for_all(cuda_device):
    for one in (torch.tensor(3, dtype=torch.int32, device=DEV), _i32([3])):
        cache = _small_cache(8)
        got = cache.extend(one, 6)
        assert got.cu.tolist() == [0, 3, 6] and got.positions.tolist() == [10, 11, 12, 6, 7, 8]


def test_extend_refuses_other_counts(cuda_device):
    from halo_b200._lib import HaloError
    cache = _small_cache(8)
    for bad in (_i32([1, 2, 3]), torch.tensor([1, 2], device=DEV), torch.tensor([1, 2], dtype=torch.int32)):
        with pytest.raises(HaloError):
            cache.extend(bad, 6)
    with pytest.raises(HaloError):
        cache.extend(_i32([1, 2]), -1)
    assert cache.extend(_i32([1, 0, 2, 0])[::2], 3).cu.tolist() == [0, 1, 3]


@pytest.mark.parametrize("seed", range(4))
def test_any_order_of_calls(cuda_device, seed):
    """Steps begun, given up, refused, accepted by any path and requests ended,
    at random: every row and every page against a list of rows a request."""
    from halo_b200 import PagedKVCache
    rng = np.random.default_rng(seed)
    R, page, n_pages, top = 5, (1, 4, 8, 7)[seed], (60, 20, 9, 12)[seed], 40
    cache = PagedKVCache(1, n_pages, 1, 8, max_requests=R, max_len=top, page_size=page,
                         dtype=torch.float32, device=DEV)
    kept, step, mark = [[] for _ in range(R)], None, 0
    refused = 0
    for _ in range(120):
        what = rng.random()
        if what < 0.5 or step is None:
            counts = [int(x) for x in rng.integers(-1, (3, 12, 45)[int(rng.integers(3))], R)]
            T = sum(max(c, 0) for c in counts) + int(rng.integers(0, 3))
            rows = cache.extend(_i32(counts), T)
            got = (rows.cu[1:] - rows.cu[:-1]).tolist()
            assert all(g in (0, max(c, 0)) for g, c in zip(got, counts))
            assert all(len(k) + g <= -(-top // page) * page for k, g in zip(kept, got))
            refused += sum(g == 0 < c for g, c in zip(got, counts))
            k = torch.arange(mark, mark + T, device=DEV, dtype=torch.float32)[:, None, None]
            cache.write(0, k.expand(T, 1, 8), -k.expand(T, 1, 8), rows)
            step, at = [], 0
            for c, g in zip(counts, got):
                step.append([mark + at + i for i in range(g)])
                at += max(c, 0)
            mark += T
        elif what < 0.85:
            depth = int(rng.integers(1, 14))
            lens = [int(x) for x in rng.integers(-1, depth + 3, R)]
            path = None
            if rng.random() < 0.7:
                path = rng.integers(-2, 20, (R, depth))
                if rng.random() < 0.6:
                    path = np.sort(path, 1)
            for r in range(R):
                n = min(max(lens[r], 0), len(step[r]), 10 ** 9 if path is None else depth)
                p = list(range(n)) if path is None else path[r, :n].tolist()
                kept[r] += [step[r][x if i < x < len(step[r]) else i] for i, x in enumerate(p)]
            cache.accept(None if path is None else _i32(path.tolist()), _i32(lens))
            step = None
        else:
            ended = rng.random(R) < 0.3
            cache.release(torch.from_numpy(ended).to(DEV))
            for r in np.nonzero(ended)[0]:
                kept[r], step[r] = [], []
        assert cache.lens.tolist() == [len(x) for x in kept]
        held = [len(x) + (len(step[r]) if step else 0) for r, x in enumerate(kept)]
        assert all(h >= n for h, n in zip(cache.held.tolist(), held))
        assert _owners(cache) == list(range(n_pages))
        for r in range(R):
            want = kept[r] + (step[r] if step else [])
            pages = cache.block_tables[r, :-(-len(want) // page)].long()
            for x, sign in ((cache.k[0], 1.0), (cache.v[0], -1.0)):
                rows_r = x[pages].transpose(1, 2).reshape(-1, 8)[:len(want)]
                assert (rows_r * sign == torch.tensor(want, device=DEV)[:, None]).all()
    assert refused > 0 and mark > 500
