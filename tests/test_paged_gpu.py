"""Paged-cache operators on the GPU: block tables and slots, row writes, tree
attention and the commit of accepted paths, against the plain restatements of
``oracle/paged.py``, and a decoding loop that uses them together."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import paged as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = torch.int32


def _i32(x):
    return torch.tensor(x, dtype=I32, device=DEV)


# ------------------------------------------------------------ block tables

def _tables_case(rng, R, width, page, spare, top):
    old = [int(x) for x in rng.integers(0, width * page + 1, R)]
    new = [int(x) for x in rng.integers(0, width * page + 1, R)]
    for r in range(R):
        if rng.random() < 0.3:
            new[r] = min(width * page, old[r] + int(rng.integers(0, 2 * page)))
        if rng.random() < 0.05:
            new[r] = (width + 1) * page        # the table cannot hold it
        if rng.random() < 0.05:
            new[r] = -3
    blocks = [-(-n // page) for n in old]
    order = rng.permutation(sum(blocks) + spare).astype(int).tolist()
    table = [[-7] * width for _ in range(R)]
    for r, n in enumerate(blocks):
        table[r][:n], order = order[:n], order[n:]
    free = order + [-9] * sum(blocks)
    return table, old, new, free, len(order), top


@pytest.mark.parametrize("R,width,page,spare,top", [
    (1, 1, 16, 0, 8), (1, 3, 5, 2, 40), (7, 4, 16, 6, 300), (33, 9, 1, 40, 400),
    (64, 6, 24, 500, 6000), (1025, 3, 8, 700, 20000), (3000, 2, 16, 100, 1)])
@pytest.mark.parametrize("seed", [0, 1])
def test_block_tables(cuda_device, R, width, page, spare, top, seed):
    from halo_b200 import ops
    rng = np.random.default_rng(seed * 1000 + R)
    table, old, new, free, n_free, top = _tables_case(rng, R, width, page, spare, top)
    want = O.update_block_tables(table, old, new, free, n_free, page, top)
    # rows of a wider tensor: what lies behind a row stays
    wide = torch.full((R, width + 2), 5, dtype=I32, device=DEV)
    wide[:, :width] = _i32(table)
    t, f, n = wide[:, :width], _i32(free), _i32([n_free])
    n_out = torch.full((1,), -1, dtype=I32, device=DEV) if seed else None
    slots, pos, cu, lens = ops.update_block_tables(t, _i32(old), _i32(new), f, n, page_size=page,
                                                   max_tokens=top, n_free_out=n_out)
    got = (t.tolist(), f.tolist(), int((n_out if seed else n)[0]), slots.tolist(), pos.tolist(),
           cu.tolist(), lens.tolist())
    for name, a, b in zip(("table", "free", "n_free", "slots", "positions", "cu", "lens"), got,
                          want):
        assert a == b, name
    assert (wide[:, width:] == 5).all()
    if seed:
        assert int(n[0]) == n_free          # only n_free_out is written


def test_block_tables_of_no_requests_and_no_tokens(cuda_device):
    from halo_b200 import ops
    n = _i32([3])
    slots, pos, cu, lens = ops.update_block_tables(
        torch.empty(0, 4, dtype=I32, device=DEV), _i32([]), _i32([]), _i32([4, 5, 6]), n,
        page_size=16, max_tokens=2)
    assert slots.tolist() == [-1, -1] and pos.tolist() == [-1, -1]
    assert cu.tolist() == [0] and lens.numel() == 0 and n.tolist() == [3]
    t = _i32([[9, 9]])
    slots, pos, cu, lens = ops.update_block_tables(t, _i32([0]), _i32([17]), _i32([4, 5, 6]), n,
                                                   page_size=16, max_tokens=0)
    assert slots.numel() == 0 and cu.tolist() == [0, 17] and lens.tolist() == [17]
    assert t.tolist() == [[6, 5]] and n.tolist() == [1]


def test_block_tables_captured_and_replayed(cuda_device):
    """n_free is updated in place from replay to replay."""
    from halo_b200 import ops
    t = torch.zeros(2, 8, dtype=I32, device=DEV)
    old, new, free, n = _i32([0, 0]), _i32([0, 0]), _i32(list(range(16))), _i32([16])

    def step():
        return ops.update_block_tables(t, old, new, free, n, page_size=4, max_tokens=16)
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        slots, pos, cu, lens = step()
    table, fr, nf, o = t.tolist(), free.tolist(), 16, [0, 0]
    for to in ([3, 9], [8, 9], [1, 16], [0, 0]):
        new.copy_(_i32(to))
        old.copy_(_i32(o))
        g.replay()
        table, fr, nf, s, p, c, o2 = O.update_block_tables(table, o, to, fr, nf, 4, 16)
        assert (t.tolist(), free.tolist(), n.tolist()[0]) == (table, fr, nf)
        assert (slots.tolist(), pos.tolist(), cu.tolist(), lens.tolist()) == (s, p, c, o2)
        o = o2


# ------------------------------------------------------------ row writes

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,D,page", [(1, 1, 1, 1), (3, 2, 5, 7), (64, 8, 128, 16), (130, 3, 80, 24),
                                        (1000, 4, 12, 64), (17, 1, 64, 256)])
def test_write_kv_pages(cuda_device, dtype, T, H, D, page):
    from halo_b200 import ops
    g = torch.Generator().manual_seed(T)
    n = T // page + 3
    kv = torch.randn(T, 3, H, D, generator=g).to(dtype)
    kp = torch.randn(n, H, page, D, generator=g).to(dtype)
    vp = torch.randn(n, H, page, D, generator=g).to(dtype)
    slots = torch.randperm(n * page, generator=g)[:T].tolist()
    for i in range(0, T, 5):
        slots[i] = (-1, n * page, -2 ** 62, 2 ** 40)[i // 5 % 4]
    # K pages head-major, V pages token-major in memory; k and v views of one tensor
    kd, vd = kp.to(DEV), vp.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    d = kv.to(DEV)
    ops.write_kv_pages(d[:, 0], d[:, 2], kd, vd, torch.tensor(slots, device=DEV))
    O.write_kv_pages(kv[:, 0], kv[:, 2], kp, vp, slots)
    assert torch.equal(kd.cpu(), kp) and torch.equal(vd.cpu(), vp)


def test_write_of_no_rows(cuda_device):
    from halo_b200 import ops
    kp = torch.ones(2, 1, 8, 64, device=DEV)
    e = torch.empty(0, 1, 64, device=DEV)
    ops.write_kv_pages(e, e, kp, kp.clone(), torch.empty(0, dtype=torch.int64, device=DEV))
    assert (kp == 1).all()


# ------------------------------------------------------------ commit

@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64),
                                     (torch.float32, 5), (torch.float16, 7)])
@pytest.mark.parametrize("R,H,page,nodes,depth", [(1, 1, 8, 1, 1), (5, 2, 16, 30, 9),
                                                  (3, 8, 5, 300, 200), (40, 3, 64, 64, 17)])
def test_commit_tree_path(cuda_device, dtype, D, R, H, page, nodes, depth):
    from halo_b200 import ops
    rng = np.random.default_rng(R * depth)
    g = torch.Generator().manual_seed(R)
    ctx = [int(x) for x in rng.integers(0, 50, R)]
    width = -(-(max(ctx) + nodes) // page) + 1
    n = R * width + 1
    order = rng.permutation(n)
    table = order[:R * width].reshape(R, width).astype(int).tolist()
    path = [sorted(rng.choice(nodes, min(depth, nodes), replace=False).tolist()) +
            [0] * max(0, depth - nodes) for _ in range(R)]
    lens = [int(x) for x in rng.integers(0, min(depth, nodes) + 1, R)]
    lens[0] = min(depth, nodes)
    if R > 3:
        lens[1], lens[2] = -1, 0
        table[3][ctx[3] // page] = -1                 # a missing page
        table[4 % R][-1] = n                          # a page beyond the pool
        path[R - 1][-1] = 10 ** 6                     # a node beyond the table
    kp = torch.randn(n, H, page, D, generator=g).to(dtype)
    vp = torch.randn(n, H, page, D, generator=g).to(dtype)
    kd, vd = kp.transpose(1, 2).contiguous().to(DEV).transpose(1, 2), vp.to(DEV)
    ops.commit_tree_path(kd, vd, _i32(table), _i32(ctx), _i32(path), _i32(lens))
    O.commit_tree_path(kp, vp, table, ctx, path, lens)
    assert torch.equal(kd.cpu(), kp) and torch.equal(vd.cpu(), vp)


# ------------------------------------------------------------ tree attention

def random_trees(rng, nodes, N):
    """Visibility rows of random trees: a node sees itself and its ancestors."""
    mask = np.zeros((sum(nodes), N), dtype=bool)
    at = 0
    for n in nodes:
        m = mask[at:at + n]
        for i in range(n):
            if i and rng.random() < 0.9:
                m[i] = m[rng.integers(max(0, i - 4), i)]
            m[i, i] = True
        at += n
    return torch.from_numpy(mask)


class Case:
    """Inputs of one call on the CPU; positions that hold no row are NaN."""

    def __init__(self, seed, ctx, nodes, H, H_kv, D, page, dtype, mask=None, spread=1.0):
        rng = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        self.ctx, self.cu = list(ctx), [0] + np.cumsum(nodes).astype(int).tolist()
        N = max(max(nodes), 1)
        self.mask = random_trees(rng, nodes, N) if mask is None else mask
        need = [-(-(c + n) // page) for c, n in zip(ctx, nodes)]
        width = max(max(need), 1)
        n_pages = sum(need) + 2
        order = rng.permutation(n_pages).astype(int).tolist()
        self.table = []
        for b in need:
            # entries behind the last page: negative, or a page of other rows
            self.table.append(order[:b] + [-1 if rng.random() < 0.5 else 0] * (width - b))
            order = order[b:]
        self.k = torch.randn(n_pages, H_kv, page, D, generator=g).to(dtype)
        self.v = torch.randn(n_pages, H_kv, page, D, generator=g).to(dtype)
        self.k[:, :, :, :2] *= 5
        self.q = (torch.randn(self.cu[-1], H, D, generator=g) * spread).to(dtype)
        for r, (c, n) in enumerate(zip(ctx, nodes)):
            if need[r]:
                last = self.table[r][need[r] - 1]
                self.k[last, :, (c + n - 1) % page + 1:] = math.nan
                self.v[last, :, (c + n - 1) % page + 1:] = math.nan

    def run(self, **kw):
        from halo_b200 import ops
        return ops.tree_attention(self.q.to(DEV), self.k.to(DEV), self.v.to(DEV),
                                  _i32(self.table), _i32(self.ctx), _i32(self.cu),
                                  self.mask.to(DEV), **kw)

    def check(self, out, lse, rows=None, scale=None):
        want, wl, room_o, room_l = O.tree_attention(self.q, self.k, self.v, self.table, self.ctx,
                                                    self.cu, self.mask, scale)
        rows = slice(0, self.cu[-1]) if rows is None else rows
        got, gl = out.cpu()[rows].double(), lse.cpu()[rows].double()
        want, wl, room_o, room_l = want[rows], wl[rows], room_o[rows], room_l[rows]
        half = 0.0 if out.dtype == torch.float32 else torch.finfo(out.dtype).eps / 2
        err = (got - want).abs() - half * want.abs()
        # subnormal halves: half a step of 2^-24
        over = err - room_o * (1 + half) - (2.0 ** -25 if out.dtype == torch.float16 else 0)
        assert not torch.isnan(got).any()
        assert (over <= 0).all(), f"out off by {float(err.max()):.3g}, {int((over > 0).sum())} beyond"
        assert torch.equal(torch.isinf(gl), torch.isinf(wl))
        el = torch.where(torch.isinf(wl), torch.zeros_like(wl), (gl - wl).abs())
        assert (el <= room_l).all(), f"lse off by {float(el.max()):.3g}"
        from halo_b200 import _lib as L
        assert L.device_error() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,H_kv,page", [(4, 4, 8), (8, 2, 16), (6, 2, 48), (14, 2, 24), (16, 1, 128),
                                         (40, 1, 256)])
def test_tree_attention_shapes(cuda_device, dtype, D, H, H_kv, page):
    c = Case(H * page, [0, 1, 63, 300, 129], [1, 5, 2, 9, 3], H, H_kv, D, page, dtype)
    c.check(*c.run())
    c.check(*c.run(out_dtype=torch.float32))


@pytest.mark.parametrize("nodes", [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 100, 129, 257])
def test_tree_attention_tree_sizes(cuda_device, nodes):
    """From one row a K/V head to several row tiles (G = 4)."""
    c = Case(nodes, [130, 3], [nodes, max(1, nodes // 2)], 4, 1, 64, 16, torch.bfloat16)
    c.check(*c.run(out_dtype=torch.float32))


@pytest.mark.parametrize("total", [1, 7, 8, 9, 127, 128, 129, 255, 256, 257, 1023, 1025, 4000])
@pytest.mark.parametrize("nodes", [1, 6])
def test_tree_attention_lengths(cuda_device, total, nodes):
    n = min(nodes, total)
    c = Case(total, [total - n], [n], 8, 2, 128, 16, torch.bfloat16)
    c.check(*c.run(out_dtype=torch.float32))


def test_tree_attention_of_many_ragged_requests(cuda_device):
    """Empty requests among long and short ones, more requests than SMs."""
    rng = np.random.default_rng(4)
    ctx = [int(x) for x in rng.integers(0, 200, 170)]
    nodes = [int(x) for x in rng.integers(0, 4, 170)]
    ctx[3], ctx[90] = 2500, 1700
    ctx[10], nodes[10] = 0, 0
    c = Case(5, ctx, nodes, 4, 2, 64, 16, torch.float16)
    c.check(*c.run(out_dtype=torch.float32))


def test_tree_attention_any_mask_and_rows_that_see_nothing(cuda_device):
    """Masks that are no trees; rows whose mask and context leave nothing."""
    rng = np.random.default_rng(8)
    nodes = [40, 33, 5, 1]
    mask = torch.from_numpy(rng.random((sum(nodes), 40)) < 0.3)
    mask[0] = mask[35] = mask[45] = False
    mask[-1] = False
    c = Case(9, [0, 100, 0, 0], nodes, 8, 2, 128, 16, torch.bfloat16, mask=mask)
    out, lse = c.run()
    c.check(out, lse)
    assert (out[0] == 0).all() and (lse[0] == -math.inf).all()
    assert (out[-1] == 0).all() and (lse[-1] == -math.inf).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("G,D,dtype", [(2, 64, torch.bfloat16), (20, 64, torch.bfloat16),
                                       (1, 128, torch.float16), (2, 128, torch.float16),
                                       (4, 128, torch.bfloat16), (7, 128, torch.float16)])
def test_hidden_rows_reach_no_output(cuda_device, bad, G, D, dtype):
    """A hidden node's K and V may hold anything; a node that sees it gets it."""
    n = 24
    c = Case(3, [130, 0], [n, n], 2 * G, 2, D, 16, dtype)
    c.mask[:, 5] = False
    c.mask[7, 5] = True                      # one row of request 0 sees node 5
    slots = [(c.table[0][(130 + 5) // 16], (130 + 5) % 16), (c.table[1][0], 5)]
    for pg, row in slots:
        c.k[pg, :, row] = bad
        c.v[pg, :, row] = bad
    out, lse = c.run(out_dtype=torch.float32)
    rows = [i for i in range(2 * n) if i != 7]
    k, v = c.k.clone(), c.v.clone()
    for pg, row in slots:                    # the oracle never reads what is hidden
        c.k[pg, :, row] = 0
        c.v[pg, :, row] = 0
    c.check(out, lse, rows=rows)
    c.k, c.v = k, v
    # only V bad: the row that sees it gets it, in every column
    for pg, row in slots:
        c.k[pg, :, row] = 0.25
    out, lse = c.run(out_dtype=torch.float32)
    seen = out[7].cpu()
    assert torch.isnan(seen).all() if math.isnan(bad) else (seen == bad).all()
    assert torch.isfinite(out[rows]).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("page", [8, 16, 24, 40])
@pytest.mark.parametrize("nodes", [3, 7, 14, 30, 70])
def test_small_pages_of_128_columns(cuda_device, page, nodes):
    """12 to 280 rows a K/V head over tiles whose pages are a few rows long,
    with a hidden node whose V is not finite in one column of each half."""
    c = Case(page + nodes, [9003, 0, 261], [nodes, nodes, 1], 4, 1, 128, page,
             torch.bfloat16 if page % 16 else torch.float16)
    c.mask[:2 * nodes, 1] = False
    hidden = [(c.table[r][(x + 1) // page], (x + 1) % page) for r, x in ((0, 9003), (1, 0))]
    for pg, row in hidden:
        c.v[pg, 0, row, 3], c.v[pg, 0, row, 100] = math.nan, -math.inf
    out, lse = c.run(out_dtype=torch.float32)
    for pg, row in hidden:                   # the oracle never reads what is hidden
        c.v[pg, 0, row] = 0
    c.check(out, lse)


def test_tree_attention_large_scores_and_scale(cuda_device):
    """Scores of thousands: the running maximum keeps the weights in range."""
    c = Case(12, [700, 40], [9, 3], 8, 2, 128, 16, torch.bfloat16, spread=60.0)
    c.check(*c.run(out_dtype=torch.float32))
    c.check(*c.run(out_dtype=torch.float32, scale=0.01), scale=0.01)


def test_tree_attention_strides_and_rows_behind_the_last_sequence(cuda_device):
    """Token-major pools, q inside a fused projection, a mask and a table that
    are parts of wider tensors, out with gaps; padded rows stay as they were."""
    from halo_b200 import ops
    c = Case(21, [77, 200, 5], [3, 8, 1], 8, 2, 64, 16, torch.float16)
    T, pad = c.cu[-1], 5
    qkv = torch.full((T + pad, 12, 64), math.nan, dtype=torch.float16)
    qkv[:T, :8] = c.q
    k = c.k.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    kv = torch.stack([c.v, c.v], 2).to(DEV)[:, :, 1]
    mask = torch.ones(T + pad, 61, dtype=torch.bool)
    mask[:T, 3:11] = c.mask
    table = torch.full((3, len(c.table[0]) + 3), -5, dtype=I32)
    table[:, :len(c.table[0])] = torch.tensor(c.table)
    out = torch.full((T + pad, 10, 64), 7.0, dtype=torch.float16, device=DEV)
    lse = torch.full((T + pad, 8), 7.0, device=DEV)
    got = ops.tree_attention(qkv.to(DEV)[:, :8], k, kv, table.to(DEV)[:, :len(c.table[0])],
                             _i32(c.ctx), _i32(c.cu), mask.to(DEV)[:, 3:11], out=out[:, 1:9],
                             lse=lse)
    assert got[1] is lse
    c.check(out[:T, 1:9], lse[:T])
    assert (out[T:] == 7).all() and (lse[T:] == 7).all() and (out[:, 0] == 7).all()
    assert (out[:, 9] == 7).all()
    o2, none = ops.tree_attention(c.q.to(DEV), k, kv, _i32(c.table), _i32(c.ctx), _i32(c.cu),
                                  c.mask.to(DEV), want_lse=False)
    assert none is None and torch.equal(o2, out[:T, 1:9])


def test_entries_that_name_no_page_read_as_zeros(cuda_device):
    c = Case(30, [60], [4], 4, 2, 64, 8, torch.bfloat16)
    c.table[0][2], c.table[0][5] = -1, c.k.shape[0]
    c.check(*c.run(out_dtype=torch.float32))


def test_contexts_longer_than_the_table_end_with_it(cuda_device):
    c = Case(31, [60], [4], 4, 2, 64, 8, torch.bfloat16)      # 64 rows: 8 whole pages
    assert not c.k[c.table[0]].isnan().any()
    c.ctx = [1000]
    out, lse = c.run(out_dtype=torch.float32)
    c.ctx, c.mask = [64], torch.zeros(4, 4, dtype=torch.bool)
    c.check(out, lse)


def test_captured_call_follows_its_lengths_on_another_stream(cuda_device):
    from halo_b200 import ops
    a = Case(40, [500, 20], [6, 6], 8, 2, 64, 16, torch.bfloat16)
    b = Case(41, [90, 430], [2, 6], 8, 2, 64, 16, torch.bfloat16)
    W = max(len(a.table[0]), len(b.table[0]))
    n = max(a.k.shape[0], b.k.shape[0])
    q = torch.zeros(12, 8, 64, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(n, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    t = torch.zeros(2, W, dtype=I32, device=DEV)
    ctx, cu = _i32([0, 0]), _i32([0, 0, 0])
    mask = torch.zeros(12, 6, dtype=torch.bool, device=DEV)

    def call():
        return ops.tree_attention(q, k, v, t, ctx, cu, mask, out_dtype=torch.float32)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        call()
    torch.cuda.synchronize()
    g, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out, lse = call()
    with torch.cuda.graph(g2, stream=s):
        out2, lse2 = call()
    for c in (a, b, a):
        T = c.cu[-1]
        q[:T].copy_(c.q)
        k[:c.k.shape[0]].copy_(c.k)
        v[:c.k.shape[0]].copy_(c.v)
        t[:, :len(c.table[0])].copy_(_i32(c.table))
        ctx.copy_(_i32(c.ctx))
        cu.copy_(_i32(c.cu))
        mask[:T].copy_(c.mask)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
        g2.replay()                      # both at once, on two streams
        torch.cuda.synchronize()
        c.check(out[:T], lse[:T])
        c.check(out2[:T], lse2[:T])


def test_rows_beyond_32_bit_offsets(cuda_device):
    """Pools of more than 2^32 elements: the pages used are their last ones."""
    from halo_b200 import ops
    page, D, H_kv = 64, 128, 8
    n = 2 ** 32 // (page * D * H_kv) + 8
    if torch.cuda.mem_get_info()[0] < 4.2 * n * page * D * H_kv:
        pytest.skip("needs 18 GB")
    c = Case(50, [300], [5], 16, H_kv, D, page, torch.bfloat16)
    m = c.k.shape[0]
    k = torch.empty(n, H_kv, page, D, dtype=torch.bfloat16, device=DEV)
    v = torch.empty_like(k)
    k[n - m:], v[n - m:] = c.k.to(DEV), c.v.to(DEV)
    table = [[p + n - m if p >= 0 else p for p in row] for row in c.table]
    out, lse = ops.tree_attention(c.q.to(DEV), k, v, _i32(table), _i32(c.ctx), _i32(c.cu),
                                  c.mask.to(DEV))
    c.check(out, lse)
    # the same rows written and moved there
    new = torch.randn(3, H_kv, D).bfloat16()
    slots = torch.tensor([(n - 1) * page + 5, (n - 2) * page, -1], device=DEV)
    ops.write_kv_pages(new.to(DEV), new.to(DEV), k, v, slots)
    assert torch.equal(k[n - 1, :, 5].cpu(), new[0]) and torch.equal(v[n - 2, :, 0].cpu(), new[1])
    ops.commit_tree_path(k, v, _i32([[n - 1]]), _i32([2]), _i32([[3]]), _i32([1]))
    assert torch.equal(k[n - 1, :, 2].cpu(), new[0])
    del k, v
    torch.cuda.empty_cache()


def test_long_context_of_one_request(cuda_device):
    """One row over 70000 positions, split over every SM and joined."""
    c = Case(60, [70000], [1], 2, 1, 64, 64, torch.bfloat16)
    c.check(*c.run(out_dtype=torch.float32))


@pytest.mark.parametrize("D,page", [(64, 8), (64, 48), (128, 16), (128, 256)])
@pytest.mark.parametrize("nodes", [1, 3, 7, 20, 40, 70])
def test_long_contexts_at_every_row_count(cuda_device, D, page, nodes):
    """Hundreds of tiles a CTA: every ring, buffer and phase goes round many
    times (G = 4: 4 to 280 rows a K/V head); a second run gives the same bits."""
    dtype = torch.bfloat16 if page % 16 else torch.float16
    c = Case(nodes + D, [18000, 9001], [nodes, max(1, nodes // 3)], 4, 1, D, page, dtype)
    q, k, v, t = c.q.to(DEV), c.k.to(DEV), c.v.to(DEV), _i32(c.table)
    from halo_b200 import ops
    args = (q, k, v, t, _i32(c.ctx), _i32(c.cu), c.mask.to(DEV))
    out, lse = ops.tree_attention(*args, out_dtype=torch.float32)
    c.check(out, lse)
    again, lse2 = ops.tree_attention(*args, out_dtype=torch.float32)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


def test_calls_from_two_threads_and_streams(cuda_device):
    """Each thread's calls have a workspace of their own."""
    import threading
    from halo_b200 import ops
    cases = [Case(80 + i, [3000, 700], [5 + 20 * i, 3], 8, 2, 64, 16, torch.bfloat16)
             for i in range(2)]
    args = [(c.q.to(DEV), c.k.to(DEV), c.v.to(DEV), _i32(c.table), _i32(c.ctx), _i32(c.cu),
             c.mask.to(DEV)) for c in cases]
    want = [ops.tree_attention(*a, out_dtype=torch.float32) for a in args]
    torch.cuda.synchronize()
    wrong = []

    def work(i, stream):
        with torch.cuda.stream(stream):
            for _ in range(50):
                o, l = ops.tree_attention(*args[i], out_dtype=torch.float32)
                if not (torch.equal(o, want[i][0]) and torch.equal(l, want[i][1])):
                    wrong.append(i)
    for streams in ([torch.cuda.Stream(), torch.cuda.Stream()], [torch.cuda.current_stream()] * 2):
        ts = [threading.Thread(target=work, args=(i, s)) for i, s in enumerate(streams)]
        for t in ts:
            t.start()
        for t in ts:
            t.join()
    assert not wrong


# ------------------------------------------------------------ together

def _dense(q, k, v, seen):
    """float64 attention of rows q (n, H, D) over k, v (t, H_kv, D)."""
    n, H, D = q.shape
    G = H // k.shape[1]
    kk, vv = k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    s = torch.einsum("nhd,thd->nht", q.double(), kk) / math.sqrt(D)
    s.masked_fill_(~seen[:, None], -math.inf)
    return torch.einsum("nht,thd->nhd", torch.softmax(s, -1), vv)


def test_tree_decoding_loop(cuda_device):
    """Prompts, drafted trees, accepted paths, an ended request and one that
    takes its pages: every step against dense attention over the kept rows."""
    from halo_b200 import PagedKVCache
    R, H, H_kv, D, page, layers = 3, 8, 2, 64, 16, 2
    rng = np.random.default_rng(2)
    g = torch.Generator().manual_seed(2)
    cache = PagedKVCache(layers, 40, H_kv, D, max_requests=R, max_len=320, page_size=page,
                         dtype=torch.float16, device=DEV)
    kept = [[[] for _ in range(layers)] for _ in range(R)]     # (k, v) rows of each context

    def rows(n):
        return torch.randn(n, H_kv, D, generator=g).half(), torch.randn(n, H_kv, D, generator=g).half()

    def step(counts, path, lens, attend=True):
        T = sum(counts) + 3                                    # a padded batch
        got = cache.extend(_i32(counts), T)
        assert got.cu.tolist() == [0] + np.cumsum(counts).astype(int).tolist()
        mask = torch.zeros(T, max(max(counts), 1), dtype=torch.bool)
        mask[:sum(counts)] = random_trees(rng, counts, mask.shape[1])
        if path == "chains":       # each tree holds its accepted path as a chain
            path = [sorted(rng.choice(n, m, replace=False).tolist()) for n, m in zip(counts, lens)]
        for layer in range(layers):
            k, v = rows(T)
            q = torch.randn(T, H, D, generator=g).half()
            cache.write(layer, k.to(DEV), v.to(DEV), got)
            out = cache.attend(layer, q.to(DEV), got, mask.to(DEV), out_dtype=torch.float32)[0].cpu()
            at = 0
            for r, n in enumerate(counts):
                if n and attend:
                    old = kept[r][layer]
                    kk = torch.cat([x for x, _ in old] + [k[at:at + n]])
                    vv = torch.cat([x for _, x in old] + [v[at:at + n]])
                    seen = torch.ones(n, kk.shape[0], dtype=torch.bool)
                    seen[:, kk.shape[0] - n:] = mask[at:at + n, :n]
                    want = _dense(q[at:at + n], kk, vv, seen)
                    assert float((out[at:at + n] - want).abs().max()) < 1e-3
                pick = path[r][:lens[r]] if path is not None else list(range(lens[r]))
                kept[r][layer].append((k[at:at + n][pick], v[at:at + n][pick]))
                at += n
        wide = None
        if path is not None:
            wide = torch.zeros(R, max(max(lens), 1), dtype=I32)
            for r, p in enumerate(path):
                wide[r, :len(p)] = torch.tensor(p, dtype=I32)
            wide = wide.to(DEV)
        cache.accept(wide, _i32(lens))
        want = [sum(x.shape[0] for x, _ in kept[r][0]) for r in range(R)]
        assert cache.lens.tolist() == want and cache.held.tolist() == want
        used = sum(-(-n // page) for n in want)
        assert int(cache.n_free) == 40 - used
        pages = [p for r, n in enumerate(want) for p in cache.block_tables[r, :-(-n // page)].tolist()]
        pages += cache.free_pages[:40 - used].tolist()
        assert sorted(pages) == list(range(40))                # every page has one owner

    step([50, 3, 100], None, [50, 3, 100])
    for _ in range(4):
        counts = [int(x) for x in rng.integers(1, 20, R)]
        step(counts, "chains", [int(rng.integers(1, n + 1)) for n in counts])
    cache.release(torch.tensor([False, False, True], device=DEV))
    kept[2] = [[] for _ in range(layers)]
    step([1, 4, 90], None, [1, 4, 90])
    step([7, 0, 5], "chains", [3, 0, 5])
    # a request that the pool cannot hold gets no rows; the others do
    got = cache.extend(_i32([1, 300, 1]), 8)
    n = [x for x in cache.lens.tolist()]
    assert got.cu.tolist()[1] == 1 and got.cu.tolist()[2] == 1
    assert cache.held.tolist()[1] == n[1]
    cache.accept(None, _i32([0, 0, 0]))
    assert cache.lens.tolist() == n


def _small_cache(n_pages):
    """Two requests of 10 and 6 rows on pages of 8, each row of K and V its
    request's number."""
    from halo_b200 import PagedKVCache
    cache = PagedKVCache(1, n_pages, 1, 64, max_requests=2, max_len=64, page_size=8, device=DEV)
    got = cache.extend(_i32([10, 6]), 16)
    k = torch.ones(16, 1, 64, dtype=torch.bfloat16, device=DEV)
    k[10:] = 2
    cache.write(0, k, k, got)
    cache.accept(None, _i32([10, 6]))
    return cache


def _rows_of(cache, r):
    """The K rows of a request's context."""
    n, page = int(cache.lens[r]), cache.page_size
    pages = cache.block_tables[r, :-(-n // page)].long()
    return cache.k[0][pages].transpose(1, 2).reshape(-1, *cache.k[0].shape[1::2])[:n, 0, 0].tolist()


def _owners(cache):
    page = cache.page_size
    pages = [p for r, n in enumerate(cache.held.tolist())
             for p in cache.block_tables[r, :-(-n // page)].tolist()]
    return sorted(pages + cache.free_pages[:int(cache.n_free)].tolist())


def test_accept_of_a_request_without_rows(cuda_device):
    """A path given for a request that got no rows, or longer than its rows or
    than the path tensor, keeps what there is and touches no other request."""
    cache = _small_cache(4)
    cache.accept(None, _i32([0, 0]))
    cache.release(torch.tensor([True, False], device=DEV))       # its entries name old pages
    got = cache.extend(_i32([0, 17]), 17)                        # 23 rows: these pages go to the other
    cache.write(0, torch.full((17, 1, 64), 2., dtype=torch.bfloat16, device=DEV),
                torch.full((17, 1, 64), 2., dtype=torch.bfloat16, device=DEV), got)
    cache.accept(None, _i32([0, 17]))
    got = cache.extend(_i32([12, 0]), 12)                        # 2 pages, 1 free
    assert got.cu.tolist() == [0, 0, 0]
    before = cache.k[0].clone()
    before[:] = torch.arange(before.shape[0] * 8, device=DEV).view(-1, 1, 8, 1) % 250
    cache.k[0].copy_(before)
    cache.accept(_i32([[3, 9, 11], [0, 1, 2]]), _i32([3, 0]))
    assert torch.equal(cache.k[0], before)
    assert cache.lens.tolist() == [0, 23]
    got = cache.extend(_i32([3, 0]), 3)
    cache.accept(_i32([[1, 2], [0, 1]]), _i32([5, 0]))           # 3 rows, 2 steps
    assert cache.lens.tolist() == [2, 23] and _owners(cache) == list(range(4))


def test_extend_by_a_negative_count(cuda_device):
    cache = _small_cache(8)
    got = cache.extend(_i32([-9, 2]), 4)
    assert got.cu.tolist() == [0, 0, 2] and cache.held.tolist() == [10, 8]
    assert _owners(cache) == list(range(8)) and _rows_of(cache, 0) == [1.] * 10


def test_release_within_a_step(cuda_device):
    """The other requests' rows of the step under way stay theirs."""
    cache = _small_cache(8)
    got = cache.extend(_i32([1, 5]), 6)
    x = torch.full((6, 1, 64), 3., dtype=torch.bfloat16, device=DEV)
    cache.release(torch.tensor([True, False], device=DEV))
    assert cache.held.tolist() == [0, 11] and cache.lens.tolist() == [0, 6]
    cache.write(0, x, x, got._replace(slots=torch.where(torch.arange(6, device=DEV) < 1, -1, got.slots)))
    cache.accept(None, _i32([0, 5]))
    assert cache.lens.tolist() == [0, 11] and _rows_of(cache, 1) == [2.] * 6 + [3.] * 5
    assert _owners(cache) == list(range(8))


def test_a_whole_step_captured_and_replayed(cuda_device):
    """extend, write, attend and accept in one graph, replayed on new inputs,
    leave the cache as eager steps do, bit for bit."""
    eager, cache = _small_cache(12), _small_cache(12)
    g = torch.Generator().manual_seed(9)
    counts, path, n = _i32([0, 0]), _i32([[0, 0, 0]] * 2), _i32([0, 0])
    k, v = (torch.zeros(12, 1, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q = torch.zeros(12, 4, 64, dtype=torch.bfloat16, device=DEV)
    mask = torch.zeros(12, 6, dtype=torch.bool, device=DEV)
    out, lse = torch.zeros_like(q), torch.zeros(12, 4, device=DEV)

    def step(c, out, lse):
        rows = c.extend(counts, 12)
        c.write(0, k, v, rows)
        c.attend(0, q, rows, mask, out=out, lse=lse)
        c.accept(path, n)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(cache, out, lse)
    want, want_lse = torch.zeros_like(out), torch.zeros_like(lse)
    for c, p, m in (([6, 3], [[0, 2, 5], [0, 1, 2]], [3, 1]), ([1, 6], [[0, 0, 0], [1, 3, 4]], [1, 3]),
                    ([0, 5], [[0, 0, 0], [0, 4, 0]], [0, 2]), ([5, 70], [[2, 3, 0], [9, 9, 9]], [2, 3])):
        for t, x in ((counts, c), (path, p), (n, m)):
            t.copy_(_i32(x))
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g))
        mask.copy_(torch.rand(mask.shape, generator=g) < 0.5)
        graph.replay()
        step(eager, want, want_lse)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        for name in ("lens", "held", "n_free", "block_tables"):
            assert torch.equal(getattr(cache, name), getattr(eager, name)), name
        assert torch.equal(cache.k[0], eager.k[0]) and torch.equal(cache.v[0], eager.v[0])
        assert _owners(cache) == list(range(12))
    assert cache.lens.tolist() == [10 + 3 + 1 + 2, 6 + 1 + 3 + 2]


@pytest.mark.parametrize("n", [3, 40])
def test_tree_attention_in_place(cuda_device, n):
    """out may be q itself: a row is read by the CTA that writes it, or
    written when all have been read."""
    from halo_b200 import ops
    c = Case(91, [5000, 130], [n, n], 8, 2, 128, 16, torch.bfloat16)
    args = (c.k.to(DEV), c.v.to(DEV), _i32(c.table), _i32(c.ctx), _i32(c.cu), c.mask.to(DEV))
    want, lse = ops.tree_attention(c.q.to(DEV), *args)
    q = c.q.to(DEV)
    out, lse2 = ops.tree_attention(q, *args, out=q)
    assert out is q and torch.equal(out, want) and torch.equal(lse, lse2)


# ------------------------------------------------------------ refusals

def test_wrappers_refuse_what_does_not_fit(cuda_device):
    from halo_b200 import ops
    from halo_b200._lib import HaloError
    c = Case(70, [20], [3], 4, 2, 64, 8, torch.bfloat16)
    good = dict(q=c.q.to(DEV), k_pages=c.k.to(DEV), v_pages=c.v.to(DEV),
                block_tables=_i32(c.table), context_lens=_i32(c.ctx), cu_nodes=_i32(c.cu),
                tree_mask=c.mask.to(DEV))
    ops.tree_attention(**good)
    T = c.cu[-1]
    for bad in ({"q": good["q"].half()}, {"q": good["q"][:, :, :32]}, {"q": good["q"][0]},
                {"q": good["q"].cpu()}, {"k_pages": good["k_pages"][:1]},
                {"v_pages": good["v_pages"].half()}, {"k_pages": good["k_pages"].cpu()},
                {"block_tables": good["block_tables"].long()},
                {"block_tables": good["block_tables"][0]},
                {"block_tables": good["block_tables"].cpu()},
                {"context_lens": good["context_lens"].long()}, {"context_lens": _i32([1, 2])},
                {"cu_nodes": good["cu_nodes"][:1]}, {"cu_nodes": good["cu_nodes"].cpu()},
                {"tree_mask": good["tree_mask"].float()}, {"tree_mask": good["tree_mask"][:2]},
                {"tree_mask": good["tree_mask"].T.contiguous().T},
                {"out": torch.empty(T, 4, 32, device=DEV, dtype=torch.bfloat16)},
                {"out": torch.empty(T, 4, 64, device=DEV, dtype=torch.float64)},
                {"out": torch.empty(T, 4, 64, dtype=torch.bfloat16)},
                {"lse": torch.empty(T, 4, device=DEV, dtype=torch.float64)},
                {"lse": torch.empty(4, T, device=DEV).T}, {"scale": 0.0}):
        with pytest.raises(HaloError):
            ops.tree_attention(**{**good, **bad})
    t, o, f, n = _i32([[0, 0]]), _i32([0]), _i32([1, 2, 3]), _i32([3])
    ops.update_block_tables(t, o, o, f, n, page_size=4, max_tokens=2)
    for args, kw in (((t.long(), o, o, f, n), {}), ((t, o.long(), o, f, n), {}),
                     ((t, o, _i32([1, 2]), f, n), {}), ((t, o, o, f.cpu(), n), {}),
                     ((t, o, o, f[::2], n), {}), ((t, o, o, f, f), {}),
                     ((t.T, o, o, f, n), {}), ((t, o, o, f, n), {"page_size": 0}),
                     ((t, o, o, f, n), {"max_tokens": -1}),
                     ((t, o, o, f, n), {"n_free_out": n.cpu()})):
        with pytest.raises(HaloError):
            ops.update_block_tables(*args, **{"page_size": 4, "max_tokens": 2, **kw})
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=DEV)
    s = torch.zeros(2, dtype=torch.int64, device=DEV) - 1
    kp, vp = good["k_pages"], good["v_pages"]
    ops.write_kv_pages(k, k, kp, vp, s)
    for args in ((k.half(), k, kp, vp, s), (k[:1], k, kp, vp, s), (k, k, kp, vp, s.int()),
                 (k, k, kp, vp, s[:1]), (k.cpu(), k, kp, vp, s), (k[:, :1], k[:, :1], kp, vp, s),
                 (k, k, kp.transpose(2, 3), vp.transpose(2, 3), s)):
        with pytest.raises(HaloError):
            ops.write_kv_pages(*args)
    tb, x = good["block_tables"], _i32([[0, 1]])
    ops.commit_tree_path(kp, vp, tb, _i32([20]), x, _i32([2]))
    for args in ((tb, _i32([20]), x.long(), _i32([2])), (tb, _i32([20]), x[0], _i32([2])),
                 (tb, _i32([20, 1]), x, _i32([2])), (tb, _i32([20]), x, _i32([2]).cpu()),
                 (tb.long(), _i32([20]), x, _i32([2])), (tb, _i32([20]), _i32([[1], [2]]), _i32([2]))):
        with pytest.raises(HaloError):
            ops.commit_tree_path(kp, vp, *args)
