"""The paged-cache operators at their limits: 1024 nodes a request, thousands
of requests, 8192 block tables."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged as O
from test_paged_gpu import DEV, I32, Case, _i32, _tables_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nodes", [258, 511, 777, 1023, 1024])
@pytest.mark.parametrize("H,H_kv,D,page,dtype", [(1, 1, 64, 16, torch.float16),
                                                 (3, 1, 128, 24, torch.bfloat16),
                                                 (4, 2, 128, 128, torch.float16)])
def test_many_nodes(cuda_device, nodes, H, H_kv, D, page, dtype):
    """Trees of up to 1024 nodes beside a small one: many row groups a request."""
    c = Case(nodes, [300, 5000, 0], [nodes, 3, nodes // 3], H, H_kv, D, page, dtype)
    c.check(*c.run(out_dtype=torch.float32))


@pytest.mark.parametrize("nodes,ctx", [(1024, 0), (1024, 2048), (1000, 77), (129, 4000)])
def test_a_causal_slice_of_a_prompt(cuda_device, nodes, ctx):
    """A lower triangle of ones: a slice of a prompt behind what is cached."""
    mask = torch.ones(nodes, nodes, dtype=torch.bool).tril()
    c = Case(nodes + ctx, [ctx], [nodes], 4, 2, 64, 64, torch.bfloat16, mask=mask)
    c.check(*c.run(out_dtype=torch.float32))


def test_more_nodes_than_the_mask_is_wide(cuda_device):
    """Nodes beyond the mask's width are not there: neither written nor seen."""
    c = Case(4, [200, 30], [12, 5], 4, 1, 64, 16, torch.bfloat16)
    c.mask = c.mask[:, :5].contiguous()
    out = torch.full((17, 4, 64), 7.0, device=DEV)
    lse = torch.full((17, 4), 7.0, device=DEV)
    c.run(out=out, lse=lse)
    rows = list(range(5)) + list(range(12, 17))
    c.check(out, lse, rows=rows)
    assert (out[5:12] == 7).all() and (lse[5:12] == 7).all()


@pytest.mark.parametrize("R", [1023, 4099])
def test_thousands_of_requests(cuda_device, R):
    """More requests than threads of a CTA; most of them empty or short."""
    rng = np.random.default_rng(R)
    nodes = [int(x) for x in rng.integers(0, 3, R)]
    ctx = [int(x) for x in rng.integers(0, 40, R)]
    ctx[R // 2], nodes[R // 2] = 4000, 2
    c = Case(R, ctx, nodes, 2, 1, 64, 8, torch.float16)
    c.check(*c.run(out_dtype=torch.float32))


def test_block_tables_of_8192_requests(cuda_device):
    from halo_b200 import ops
    from halo_b200._lib import HaloError
    rng = np.random.default_rng(8)
    R, width, page, top = 8192, 3, 16, 70000
    table, old, new, free, n_free, _ = _tables_case(rng, R, width, page, 20000, top)
    want = O.update_block_tables(table, old, new, free, n_free, page, top)
    t, f, n = _i32(table), _i32(free), _i32([n_free])
    slots, pos, cu, lens = ops.update_block_tables(t, _i32(old), _i32(new), f, n, page_size=page,
                                                   max_tokens=top)
    got = (t.tolist(), f.tolist(), int(n), slots.tolist(), pos.tolist(), cu.tolist(), lens.tolist())
    for name, a, b in zip(("table", "free", "n_free", "slots", "positions", "cu", "lens"), got, want):
        assert a == b, name
    z = torch.zeros(8193, dtype=I32, device=DEV)
    with pytest.raises(HaloError):
        ops.update_block_tables(torch.zeros(8193, 3, dtype=I32, device=DEV), z, z, f, n,
                                page_size=page, max_tokens=1)


def test_a_table_row_of_a_million_positions(cuda_device):
    """Positions and slots of long requests on pages of one and of 4096 rows."""
    from halo_b200 import ops
    for page in (1, 3, 4096):
        width = -(-1100000 // page)
        n = 2 * width
        order = np.random.default_rng(page).permutation(n).astype(np.int32)
        t = torch.zeros(2, width, dtype=I32, device=DEV)
        free, n_free = torch.from_numpy(order).to(DEV), _i32([n])
        old = _i32([0, 0])
        for new in ([1048577, 5], [1050000, 1000000]):
            top = sum(new)
            slots, pos, cu, lens = ops.update_block_tables(t, old, _i32(new), free, n_free,
                                                           page_size=page, max_tokens=top)
            assert lens.tolist() == new
            a = [np.arange(o, x) for o, x in zip(old.tolist(), new)]
            want = np.concatenate(a)
            assert (pos[:len(want)].cpu().numpy() == want).all() and (pos[len(want):] == -1).all()
            tab = t.cpu().numpy().astype(np.int64)
            s = np.concatenate([tab[r][x // page] * page + x % page for r, x in enumerate(a)])
            assert (slots[:len(s)].cpu().numpy() == s).all()
            old = lens
        used = [p for r, x in enumerate(old.tolist()) for p in tab[r, :-(-x // page)].tolist()]
        assert sorted(used + free[:int(n_free)].tolist()) == list(range(n))


@pytest.mark.parametrize("nodes", [[3, 0, 5, 1], [40, 2, 0, 33]])
@pytest.mark.parametrize("captured", [False, True])
def test_rows_that_begin_elsewhere(cuda_device, nodes, captured):
    """node_starts: requests' rows in another order and with gaps between them;
    cu_nodes then only counts them."""
    from halo_b200 import ops
    c = Case(sum(nodes), [300, 40, 9, 2000], nodes, 8, 2, 64, 16, torch.bfloat16)
    T, starts = c.cu[-1], [0] * 4
    at = 2
    for r in (2, 0, 3, 1):
        starts[r] = at
        at += nodes[r] + 3
    rows = [starts[r] + i for r in range(4) for i in range(nodes[r])]
    q = torch.full((at, 8, 64), float("nan"), dtype=torch.bfloat16)
    mask = torch.ones(at, c.mask.shape[1], dtype=torch.bool)
    q[rows], mask[rows] = c.q, c.mask
    out = torch.full((at, 8, 64), 7.0, device=DEV)
    lse = torch.full((at, 8), 7.0, device=DEV)
    args = (q.to(DEV), c.k.to(DEV), c.v.to(DEV), _i32(c.table), _i32(c.ctx), _i32(c.cu),
            mask.to(DEV))
    st = _i32(starts)
    if captured:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.tree_attention(*args, out=out, lse=lse, node_starts=st)
            other, none = ops.tree_attention(*args, out_dtype=torch.float32, node_starts=st,
                                             want_lse=False)
        g.replay()
        assert none is None and torch.equal(other[rows], out[rows])
    else:
        ops.tree_attention(*args, out=out, lse=lse, node_starts=st)
    c.check(out[rows], lse[rows])
    rest = [t for t in range(at) if t not in rows]
    assert (out[rest] == 7).all() and (lse[rest] == 7).all()
    assert T == len(rows)


def test_node_starts_that_do_not_fit_are_refused(cuda_device):
    from halo_b200 import ops
    from halo_b200._lib import HaloError
    c = Case(2, [30, 5], [2, 2], 2, 1, 64, 8, torch.float16)
    args = (c.q.to(DEV), c.k.to(DEV), c.v.to(DEV), _i32(c.table), _i32(c.ctx), _i32(c.cu),
            c.mask.to(DEV))
    ops.tree_attention(*args, node_starts=_i32([0, 2]))
    for bad in (_i32([0]), _i32([0, 2, 4]), torch.tensor([0, 2], device=DEV), _i32([0, 2]).cpu(),
                _i32([0, 0, 2, 0])[::2]):
        with pytest.raises(HaloError):
            ops.tree_attention(*args, node_starts=bad)
    # rows that would leave the tensors are not there
    out = torch.full((4, 2, 64), 7.0, dtype=torch.float16, device=DEV)
    lse = torch.full((4, 2), 7.0, device=DEV)
    ops.tree_attention(*args, node_starts=_i32([2, 2 ** 31 - 1]), out=out, lse=lse)
    assert (out[:2] == 7).all() and (lse[:2] == 7).all() and torch.isfinite(out).all()


def test_extend_of_no_requests(cuda_device):
    from halo_b200 import ops
    e, n = _i32([]), _i32([2])
    slots, pos, cu = ops.extend_block_tables(torch.empty(0, 4, dtype=I32, device=DEV), e, e, e,
                                             torch.empty_like(e), torch.empty_like(e), _i32([4, 5]), n,
                                             page_size=16, max_tokens=3)
    assert slots.tolist() == [-1] * 3 and pos.tolist() == [-1] * 3 and cu.tolist() == [0]
    assert n.tolist() == [2]
