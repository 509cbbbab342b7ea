"""Paged-cache operators: refusals of the C ABI and of the tensor wrappers (no
GPU needed), and the oracle against independent small cases."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from oracle import paged as O


def _pool(L, **kw):
    p = L.PagePool(0x10000, 0x20000, 2 * 16 * 128, 16 * 128, 128, 2 * 16 * 128, 16 * 128, 128, 10,
                   2, 16, 128, L.DTYPE_BF16)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _tree(L, **kw):
    p = L.TreeProblem(2, 8, 8, 4, 5, 0.1, 0x30000, 8 * 128, 128, 0x40000, 5, 0x50000, 0x60000,
                      0x70000, 4, 0x80000, 8 * 128, 128, L.DTYPE_BF16, 0x90000)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("pool,prob,code", [
    ({"dtype": 0}, {}, "UNSUPPORTED"), ({"dtype": 9}, {}, "UNSUPPORTED"),
    ({"D": 96}, {}, "UNSUPPORTED"), ({"D": 256}, {}, "UNSUPPORTED"),
    ({"page_size": 12}, {}, "UNSUPPORTED"), ({"page_size": 0}, {}, "INVALID_ARG"),
    ({"n_pages": 0}, {}, "INVALID_ARG"), ({"H_kv": 3}, {}, "INVALID_ARG"),
    ({}, {"R": -1}, "INVALID_ARG"), ({}, {"T": -1}, "INVALID_ARG"),
    ({}, {"max_nodes": 1025}, "UNSUPPORTED"), ({}, {"max_blocks": 2 ** 30}, "UNSUPPORTED"),
    ({}, {"scale": 0.0}, "UNSUPPORTED"), ({}, {"scale": -1.0}, "UNSUPPORTED"),
    ({}, {"scale": math.inf}, "UNSUPPORTED"), ({}, {"scale": math.nan}, "UNSUPPORTED"),
    ({"k": None}, {}, "INVALID_ARG"), ({}, {"q": None}, "INVALID_ARG"),
    ({}, {"out": None}, "INVALID_ARG"), ({}, {"mask": None}, "INVALID_ARG"),
    ({}, {"cu_nodes": None}, "INVALID_ARG"), ({}, {"context_lens": None}, "INVALID_ARG"),
    ({}, {"block_tables": None}, "INVALID_ARG"),
    ({"k": 0x10008}, {}, "MISALIGNED"), ({"v_stride_t": 132}, {}, "MISALIGNED"),
    ({"k_stride_h": 1}, {}, "MISALIGNED"), ({}, {"q": 0x30002}, "MISALIGNED"),
    ({}, {"q_stride_h": 130}, "MISALIGNED"), ({}, {"out_stride_t": 12}, "MISALIGNED"),
    ({}, {"out_dtype": 2}, "UNSUPPORTED")])
def test_tree_attention_refusals(pool, prob, code):
    from halo_b200 import _lib as L
    lib = L.lib()
    po, pr = _pool(L, **pool), _tree(L, **prob)
    rc = lib.halo_tree_attention(ctypes.byref(po), ctypes.byref(pr), 0x100000, 1 << 40, None)
    assert rc == getattr(L, "HALO_ERR_" + code), lib.halo_last_error_string()
    assert lib.halo_last_error_string()


def test_tree_attention_workspace():
    from halo_b200 import _lib as L
    lib = L.lib()
    po, pr = _pool(L), _tree(L)
    need = lib.halo_tree_workspace_bytes(ctypes.byref(po), ctypes.byref(pr))
    assert need > 0
    for ws, n, code in ((None, need, L.HALO_ERR_WORKSPACE), (0x100000, need - 1, L.HALO_ERR_WORKSPACE),
                        (0x100010, need, L.HALO_ERR_MISALIGNED)):
        assert lib.halo_tree_attention(ctypes.byref(po), ctypes.byref(pr), ws, n, None) == code
    # more rows a K/V head, larger parts
    wide = lib.halo_tree_workspace_bytes(ctypes.byref(po), ctypes.byref(_tree(L, max_nodes=1000)))
    assert wide > need


def test_tree_attention_nothing_to_do_and_null_arguments():
    from halo_b200 import _lib as L
    lib = L.lib()
    po = _pool(L)
    for kw in ({"R": 0}, {"T": 0}, {"max_nodes": 0}):
        pr = _tree(L, **kw)
        assert lib.halo_tree_workspace_bytes(ctypes.byref(po), ctypes.byref(pr)) >= 0
        assert lib.halo_tree_attention(ctypes.byref(po), ctypes.byref(pr), None, 0, None) == L.HALO_OK
    assert lib.halo_tree_attention(None, ctypes.byref(_tree(L)), None, 0, None) == L.HALO_ERR_INVALID_ARG
    assert lib.halo_tree_workspace_bytes(ctypes.byref(po), None) == L.HALO_ERR_INVALID_ARG


def test_block_table_refusals():
    from halo_b200 import _lib as L
    lib = L.lib()

    def call(table=0x1000, stride=8, R=4, blocks=8, old=0x2000, cap=10, n=0x4000, page=16, tok=5,
             slots=0x5000, cu=0x7000):
        return lib.halo_update_block_tables(table, stride, R, blocks, old, 0x2800, 0x3000, cap, n,
                                            0x4000, page, tok, slots, 0x6000, cu, 0x8000, None)
    for kw in ({"table": None}, {"old": None}, {"n": None}, {"slots": None}, {"cu": None},
               {"R": -1}, {"blocks": -1}, {"cap": -1}, {"page": 0}, {"tok": -1}, {"stride": 7}):
        assert call(**kw) == L.HALO_ERR_INVALID_ARG, kw
    for kw in ({"R": 8193}, {"blocks": 2 ** 28, "stride": 2 ** 28}):
        assert call(**kw) == L.HALO_ERR_UNSUPPORTED, kw


def test_rows_that_overlap_are_refused():
    from halo_b200 import _lib as L
    lib = L.lib()
    for old, new, lens in ((0x2000, 0x3000, 0x2000), (0x2000, 0x3000, 0x3000),
                           (0x2000, 0x3000, 0x200c), (0x2000, 0x3000, 0x2ff4)):
        assert lib.halo_update_block_tables(0x10000, 8, 4, 8, old, new, 0x12000, 10, 0x14000, 0x14000,
                                            16, 5, 0x15000, 0x16000, 0x17000, lens,
                                            None) == L.HALO_ERR_INVALID_ARG
    po = _pool(L)
    need = lib.halo_tree_workspace_bytes(ctypes.byref(po), ctypes.byref(_tree(L)))
    for kw in ({"out_stride_t": 0}, {"out_stride_h": 0}, {"out_stride_h": po.D // 2}):
        assert lib.halo_tree_attention(ctypes.byref(po), ctypes.byref(_tree(L, **kw)), 0x100000, need,
                                       None) == L.HALO_ERR_INVALID_ARG


def test_write_and_commit_refusals():
    from halo_b200 import _lib as L
    lib = L.lib()

    def write(pool=None, k=0x1000, T=3, slots=0x2000):
        return lib.halo_write_kv_pages(ctypes.byref(pool or _pool(L)), k, 256, 128, 0x3000, 256, 128,
                                       T, slots, None)

    def commit(pool=None, R=2, depth=3, blocks=4, path=0x2000):
        return lib.halo_commit_tree_path(ctypes.byref(pool or _pool(L)), 0x1000, 4, blocks, R,
                                         0x1800, path, 3, depth, 0x2800, None)
    assert write(T=0) == L.HALO_OK and commit(R=0) == L.HALO_OK and commit(depth=0) == L.HALO_OK
    assert write(T=-1) == write(k=None) == write(slots=None) == L.HALO_ERR_INVALID_ARG
    assert commit(R=-1) == commit(depth=-1) == commit(path=None) == L.HALO_ERR_INVALID_ARG
    assert commit(R=65536) == L.HALO_ERR_UNSUPPORTED
    assert write(k=0x1001) == L.HALO_ERR_MISALIGNED
    for call in (write, commit):
        assert call(_pool(L, dtype=5)) == L.HALO_ERR_INVALID_ARG
        assert call(_pool(L, D=0)) == L.HALO_ERR_INVALID_ARG
        assert call(_pool(L, v=None)) == L.HALO_ERR_INVALID_ARG
        assert call(_pool(L, k=0x10001)) == L.HALO_ERR_MISALIGNED


def test_wrappers_refuse_cpu_tensors():
    from halo_b200 import ops
    from halo_b200._lib import HaloError
    i = torch.zeros(2, dtype=torch.int32)
    t = torch.zeros(2, 4, dtype=torch.int32)
    p = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(HaloError, match="CUDA"):
        ops.update_block_tables(t, i, i, i, i[:1], page_size=16, max_tokens=4)
    with pytest.raises(HaloError, match="CUDA"):
        ops.write_kv_pages(p[0], p[0], p, p, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(HaloError, match="CUDA"):
        ops.commit_tree_path(p, p, t, i, t, i)
    with pytest.raises(HaloError, match="CUDA"):
        ops.tree_attention(p[0], p, p, t, i, i, torch.ones(2, 3, dtype=torch.bool))


def test_oracle_block_tables_by_hand():
    # page 4: request 0 shrinks from 9 to 4 rows and gives pages 8, 9 back;
    # request 1 grows from 3 to 10 and takes 9, then 8; request 2 wants more than is left
    t, f, n, s, p, cu, lens = O.update_block_tables(
        [[7, 8, 9], [1, 0, 0], [0, 0, 0]], [9, 3, 0], [4, 10, 9], [5, 6, 0, 0, 0], 2, 4, 9)
    assert t == [[7, 8, 9], [1, 9, 8], [0, 0, 0]] and lens == [4, 10, 0]
    assert n == 2 and f == [5, 6, 0, 0, 0]
    assert p == [3, 4, 5, 6, 7, 8, 9, -1, -1] and cu == [0, 0, 7, 7]
    assert s == [7, 36, 37, 38, 39, 32, 33, -1, -1]


def test_oracle_tree_attention_by_softmax():
    g = torch.Generator().manual_seed(0)
    k, v = torch.randn(4, 1, 8, 16, generator=g), torch.randn(4, 1, 8, 16, generator=g)
    q = torch.randn(3, 2, 16, generator=g)
    mask = torch.tensor([[1, 0, 0], [1, 1, 0], [1, 0, 1]], dtype=torch.bool)
    out, lse, _, _ = O.tree_attention(q, k, v, [[2, 0]], [9], [0, 3], mask)
    kk = torch.cat([k[2, 0], k[0, 0]])[:12].double()
    vv = torch.cat([v[2, 0], v[0, 0]])[:12].double()
    seen = torch.cat([torch.ones(3, 9, dtype=torch.bool), mask], 1)
    s = (q.double() @ kk.T / 4).masked_fill(~seen[:, None], -math.inf)
    assert torch.allclose(out, torch.softmax(s, -1) @ vv)
    assert torch.allclose(lse, torch.logsumexp(s, -1))


def test_oracle_commit_reads_before_it_writes():
    k = torch.arange(8.0).view(1, 1, 8, 1).clone()
    v = -k.clone()
    O.commit_tree_path(k, v, [[0]], [2], [[0, 2, 3]], [3])
    assert k.flatten().tolist() == [0, 1, 2, 4, 5, 5, 6, 7] and torch.equal(v, -k)


def test_packed_descriptions_match_the_structures():
    from halo_b200 import _lib as L
    po, pr = _pool(L), _tree(L)
    fields = lambda x: [getattr(x, n) or 0 for n, _ in x._fields_]      # noqa: E731
    assert L.pack_page_pool(*fields(po)) == bytes(po)
    assert L.pack_tree_problem(*fields(pr)) == bytes(pr)
    assert L.lib().halo_tree_workspace_bytes(L.pack_page_pool(*fields(po)),
                                             L.pack_tree_problem(*fields(pr))) == \
        L.lib().halo_tree_workspace_bytes(ctypes.byref(po), ctypes.byref(pr))


def test_extend_refusals():
    from halo_b200 import _lib as L
    lib = L.lib()

    def call(table=0x1000, stride=8, R=4, blocks=8, held=0x2000, ctx=0x2400, counts=0x2800, cap=10,
             n=0x4000, page=16, tok=5, slots=0x5000, cu=0x7000, rows=0x8000, starts=0x8800):
        return lib.halo_extend_block_tables(table, stride, R, blocks, held, ctx, counts, 0x3000, cap,
                                            n, page, tok, slots, 0x6000, cu, rows, starts, None)
    for kw in ({"table": None}, {"held": None}, {"ctx": None}, {"counts": None}, {"n": None},
               {"slots": None}, {"cu": None}, {"rows": None}, {"R": -1}, {"blocks": -1}, {"cap": -1},
               {"page": 0}, {"tok": -1}, {"stride": 7}, {"rows": 0x2000}, {"rows": 0x2408},
               {"rows": 0x27fc}, {"ctx": 0x2000}, {"counts": 0x200c}, {"starts": None}, {"starts": 0x2000},
               {"starts": 0x2408}, {"starts": 0x27fc}, {"starts": 0x800c}):
        assert call(**kw) == L.HALO_ERR_INVALID_ARG, kw
    for kw in ({"R": 8193}, {"blocks": 2 ** 28, "stride": 2 ** 28}):
        assert call(**kw) == L.HALO_ERR_UNSUPPORTED, kw


def test_oracle_extend_by_hand():
    # page 4: request 0 gave up a step (9 rows held, context 3), asks for 2 rows
    # and gives page 9 back; request 1 takes it and page 6
    t, f, n, s, p, cu, rows, starts, held = O.extend_block_tables(
        [[7, 8, 9], [1, 0, 0]], [9, 3], [3, 3], [2, 9], [5, 6, 0, 0, 0], 2, 4, 12)
    assert starts == [0, 2]
    assert t == [[7, 8, 9], [1, 9, 6]] and held == [5, 12] and rows == [2, 9]
    assert n == 1 and f == [5, 6, 0, 0, 0] and cu == [0, 2, 11]
    assert p == [3, 4, 3, 4, 5, 6, 7, 8, 9, 10, 11, -1]
    assert s == [31, 32, 7, 36, 37, 38, 39, 24, 25, 26, 27, -1]


def test_oracle_extend_keeps_the_places_of_refused_rows():
    t, f, n, s, p, cu, rows, starts, held = O.extend_block_tables(
        [[3, 0], [4, 0], [5, 0]], [2, 2, 2], [2, 2, 2], [1, 50, 2], [6, 7], 2, 4, 60)
    assert starts == [0, 1, 51] and cu == [0, 1, 1, 3] and rows == [1, 0, 2] and held == [3, 2, 4]
    assert s[0] == 14 and s[1:51] == [-1] * 50 and s[51:] == [22, 23] + [-1] * 7
    assert p[0] == 2 and p[51:53] == [2, 3]


def test_out_rows_that_share_elements_are_refused():
    """Any strides of out, against the rows spelled out.  A workspace that is
    too small is refused behind them, so nothing is launched."""
    import random
    from halo_b200 import _lib as L
    lib = L.lib()
    rng = random.Random(5)
    po = _pool(L, D=64, H_kv=1)
    seen = {True: 0, False: 0}
    for _ in range(3000):
        T, H = rng.randint(1, 6), rng.randint(1, 6)
        st, sh = (rng.choice((0, 8, 56, 64, 72, 128, 192, 256, 320, 448)) + 64 * rng.randint(0, 3)
                  for _ in range(2))
        at = sorted(t * st + h * sh for t in range(T) for h in range(H))
        overlap = any(b - a < 64 for a, b in zip(at, at[1:]))
        pr = _tree(L, T=T, H=H, out_stride_t=st, out_stride_h=sh)
        rc = lib.halo_tree_attention(ctypes.byref(po), ctypes.byref(pr), 0x100000, 1, None)
        assert rc == (L.HALO_ERR_INVALID_ARG if overlap else L.HALO_ERR_WORKSPACE), (T, H, st, sh)
        seen[overlap] += 1
    assert min(seen.values()) > 500
    # two dimensions of one stride, and rows of a wide tensor
    for st, sh, rc in ((64, 64, L.HALO_ERR_INVALID_ARG), (2 ** 40, 64, L.HALO_ERR_WORKSPACE),
                       (64, 2 ** 40, L.HALO_ERR_WORKSPACE)):
        pr = _tree(L, T=1000, H=65535, out_stride_t=st, out_stride_h=sh)
        assert lib.halo_tree_attention(ctypes.byref(po), ctypes.byref(pr), 0x100000, 1, None) == rc


@pytest.mark.parametrize("bad,code", [
    ({"max_requests": 8193}, "UNSUPPORTED"), ({"max_len": 2 ** 31}, "UNSUPPORTED"),
    ({"max_len": 2 ** 31 - 64}, "UNSUPPORTED"), ({"n_pages": 2 ** 30 + 1}, "UNSUPPORTED"),
    ({"max_requests": 8192, "max_len": 2 ** 24}, "UNSUPPORTED"), ({"page_size": 0}, "INVALID_ARG"),
    ({"max_requests": 0}, "INVALID_ARG"), ({"dtype": torch.float64}, "UNSUPPORTED")])
def test_caches_that_could_begin_no_step_are_refused(bad, code):
    from halo_b200 import PagedKVCache
    from halo_b200 import _lib as L
    kw = {"n_pages": 2, "max_requests": 2, "max_len": 64, "page_size": 64, **bad}
    with pytest.raises(L.HaloError) as e:
        PagedKVCache(1, kw.pop("n_pages"), 1, 64, device="cpu", **kw)
    assert e.value.code == getattr(L, "HALO_ERR_" + code)


def test_the_largest_tables_are_not_refused():
    from halo_b200 import PagedKVCache
    for kw in ({"max_requests": 8192, "max_len": 64}, {"max_requests": 1, "max_len": 2 ** 31 - 129},
               {"max_requests": 2, "max_len": 64, "dtype": torch.float32, "page_size": 5}):
        PagedKVCache(1, 2, 1, 8, device="cpu", **kw)


def test_workspace_holds_a_log_sum_exp_that_is_not_asked_for():
    from halo_b200 import _lib as L
    lib = L.lib()
    po = _pool(L)
    need = lib.halo_tree_workspace_bytes(ctypes.byref(po), ctypes.byref(_tree(L)))
    more = lib.halo_tree_workspace_bytes(ctypes.byref(po), ctypes.byref(_tree(L, lse=None)))
    assert more == need + 8 * 8 * 4
    assert lib.halo_tree_attention(ctypes.byref(po), ctypes.byref(_tree(L, lse=None)), 0x100000,
                                   more - 1, None) == L.HALO_ERR_WORKSPACE
