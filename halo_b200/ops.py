"""Tensor-level entry points over the C-ABI (``include/halo_b200.h``).

Every function here launches sm_100a kernels from ``libhalo_sm100.so`` on the
current CUDA stream; there is no CPU path.  Tensors follow the reference's
layouts: queries ``(B, H, D)`` / ``(B, H, T_q, D)`` and K/V chunks
``(B, H_kv, T_c, D)`` with a contiguous last dimension.
"""
from __future__ import annotations

import ctypes
import math
import threading
from typing import Optional, Sequence

import torch

from halo_b200 import _lib as L


class _Workspaces:
    """Grow-only device scratch per (device, stream); stream-ordered reuse.
    Allocated zeroed: the decode workspaces start with a control block that
    must be zero before first use (the kernels leave it zero)."""

    def __init__(self):
        self._bufs: dict = {}

    def get(self, device: torch.device, nbytes: int, stream: Optional[int] = None) -> torch.Tensor:
        """``stream``: the raw handle of the stream the buffer is used on
        (default: ``device``'s current stream)."""
        if stream is None:
            stream = L.stream_handle(device)
        key = (device.index, stream)
        buf = self._bufs.get(key)
        if buf is None or buf.numel() < nbytes:
            buf = torch.zeros(max(nbytes, 1 << 16), dtype=torch.uint8, device=device)
            self._bufs[key] = buf
        return buf


WORKSPACES = _Workspaces()
# prefill's staging workspace (fp16 copies of V): kept apart from the decode
# workspaces, whose leading control block must stay zero between calls
PREFILL_WORKSPACES = _Workspaces()


def _require_cuda(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise L.HaloError(f"{name} must be a CUDA tensor (no CPU path)", L.HALO_ERR_INVALID_ARG)


def _last_contig(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 else t.contiguous()


def make_chunk(k: torch.Tensor, v: torch.Tensor, start: int, causal: bool,
               *, batch_stride_zero: bool = False) -> tuple:
    """Describe one ``(B, H_kv, T_c, D)`` chunk for the C-ABI; returns the
    struct plus the tensors it points into (keep them alive)."""
    k = _last_contig(k)
    v = _last_contig(v)
    c = L.KVChunk()
    c.k = k.data_ptr() if k.numel() else None
    c.v = v.data_ptr() if v.numel() else None
    c.k_stride_b = 0 if batch_stride_zero else k.stride(0)
    c.k_stride_h, c.k_stride_t = k.stride(1), k.stride(2)
    c.v_stride_b = 0 if batch_stride_zero else v.stride(0)
    c.v_stride_h, c.v_stride_t = v.stride(1), v.stride(2)
    c.start = int(start)
    c.len = int(k.shape[2]) if k.numel() else 0
    c.causal = int(bool(causal))
    return c, (k, v)


def _problem(q3: torch.Tensor, H_kv: int, D_v: int, q_pos: Optional[torch.Tensor], scale: float,
             max_split_rows: int = 0) -> L.DecodeProblem:
    p = L.DecodeProblem()
    p.B, p.H, p.D = q3.shape
    p.H_kv = H_kv
    p.Dv = D_v
    p.dtype = L.halo_dtype(q3.dtype)
    p.q = q3.data_ptr()
    p.q_stride_b, p.q_stride_h = q3.stride(0), q3.stride(1)
    p.q_pos = q_pos.data_ptr() if q_pos is not None else None
    p.scale = float(scale)
    p.max_split_rows = int(max_split_rows)
    return p


def decode_raw(q3: torch.Tensor, chunk_structs: Sequence[L.KVChunk], H_kv: int, D_v: int, *,
               scale: float, q_pos: Optional[torch.Tensor], merge: L.MergeArgs,
               max_split_rows: int = 0) -> None:
    """Launch split-KV decode + merge for prepared chunk structs."""
    dev = q3.device
    prob = _problem(q3, H_kv, D_v, q_pos, scale, max_split_rows)
    n = len(chunk_structs)
    arr = (L.KVChunk * max(n, 1))(*chunk_structs)
    lib = L.lib()
    need = lib.halo_decode_workspace_bytes(ctypes.byref(prob), arr, n)
    if need < 0:
        L.check(int(need), "halo_decode_workspace_bytes")
    sh = L.stream_handle(dev)
    ws = WORKSPACES.get(dev, int(need), sh)
    with L.on_device(dev):
        rc = lib.halo_chunked_decode(ctypes.byref(prob), arr, n, ws.data_ptr(), ws.numel(),
                                     ctypes.byref(merge), sh)
    L.check(rc, "halo_chunked_decode")


class ChunkTable:
    """A chunk list described once for repeated decode calls.

    Holds the C-ABI chunk array and references to the tensors it points
    into.  Reuse it while the chunks' storage and layout stay unchanged (the
    steady state of a decode loop); the library additionally memoises the
    tensor maps and the split plan for a layout it has seen.
    """

    def __init__(self, chunks: Sequence[tuple], *, batch_stride_zero: bool = False,
                 batch: Optional[slice] = None):
        structs, keep = [], []
        self.H_kv = self.D_v = None
        self.total_rows = 0
        self.any_causal = False
        for (k, v, start, causal) in chunks:
            _require_cuda(k, "k")
            _require_cuda(v, "v")
            if batch is not None:
                k, v = k[batch], v[batch]
            if self.H_kv is None:
                self.H_kv, self.D_v = int(k.shape[1]), int(v.shape[-1])
            st, t = make_chunk(k, v, start, causal, batch_stride_zero=batch_stride_zero)
            structs.append(st)
            keep.append(t)
            self.total_rows += int(k.shape[-2])
            self.any_causal |= bool(causal)
        self.n = len(structs)
        self.arr = (L.KVChunk * max(self.n, 1))(*structs)
        self._keep = keep


def _decode_table(q3: torch.Tensor, table: ChunkTable, *, scale: float,
                  q_pos: Optional[torch.Tensor], merge: L.MergeArgs, max_split_rows: int = 0,
                  events: Optional[tuple] = None):
    dev = q3.device
    H_kv = table.H_kv if table.H_kv is not None else q3.shape[1]
    D_v = table.D_v if table.D_v is not None else q3.shape[2]
    prob = _problem(q3, H_kv, D_v, q_pos, scale, max_split_rows)
    if events is not None:
        prob.event_begin, prob.event_end = events
    lib = L.lib()
    need = lib.halo_decode_workspace_bytes(ctypes.byref(prob), table.arr, table.n)
    if need < 0:
        L.check(int(need), "halo_decode_workspace_bytes")
    sh = L.stream_handle(dev)
    ws = WORKSPACES.get(dev, int(need), sh)
    with L.on_device(dev):
        rc = lib.halo_chunked_decode(ctypes.byref(prob), table.arr, table.n, ws.data_ptr(),
                                     ws.numel(), ctypes.byref(merge), sh)
    L.check(rc, "halo_chunked_decode")


def decode_partials(q3: torch.Tensor, table: ChunkTable, *, scale: float,
                    q_pos: Optional[torch.Tensor] = None, events: Optional[tuple] = None):
    """Split-KV launches only (``halo_chunked_decode_partials``): returns
    ``(workspace, S, (m_off, l_off, o_off))`` -- the per-split fp32 partial
    state left in the workspace, ``m``/``l`` ``[B*H][S]``, ``o``
    ``[B*H][S][D_v]`` at those byte offsets -- for a caller-side merge."""
    dev = q3.device
    H_kv = table.H_kv if table.H_kv is not None else q3.shape[1]
    D_v = table.D_v if table.D_v is not None else q3.shape[2]
    prob = _problem(q3, H_kv, D_v, q_pos, scale)
    if events is not None:
        prob.event_begin, prob.event_end = events
    lib = L.lib()
    need = lib.halo_decode_workspace_bytes(ctypes.byref(prob), table.arr, table.n)
    if need < 0:
        L.check(int(need), "halo_decode_workspace_bytes")
    sh = L.stream_handle(dev)
    ws = WORKSPACES.get(dev, int(need), sh)
    n_parts = ctypes.c_int32(0)
    offs = (ctypes.c_int64 * 3)()
    with L.on_device(dev):
        rc = lib.halo_chunked_decode_partials(ctypes.byref(prob), table.arr, table.n,
                                              ws.data_ptr(), ws.numel(), ctypes.byref(n_parts),
                                              offs, sh)
    L.check(rc, "halo_chunked_decode_partials")
    return ws, int(n_parts.value), (int(offs[0]), int(offs[1]), int(offs[2]))


def sharded_decode(q3: torch.Tensor, table: ChunkTable, exchange, *, scale: float,
                   out: torch.Tensor, lse: Optional[torch.Tensor] = None,
                   q_pos: Optional[torch.Tensor] = None, events: Optional[tuple] = None):
    """One sequence-sharded decode step on this rank (``halo_sharded_decode``):
    attention over this rank's chunks merged with every rank's through the
    NVLink exchange buffers of ``exchange`` (a :class:`halo_b200.sharded.
    P2PExchange`).  Writes ``out (B, H, D_v)`` and ``lse (B, H)``."""
    dev = q3.device
    H_kv = table.H_kv if table.H_kv is not None else q3.shape[1]
    D_v = table.D_v if table.D_v is not None else q3.shape[2]
    prob = _problem(q3, H_kv, D_v, q_pos, scale)
    if events is not None:
        prob.event_begin, prob.event_end = events
    lib = L.lib()
    need = lib.halo_decode_workspace_bytes(ctypes.byref(prob), table.arr, table.n)
    if need < 0:
        L.check(int(need), "halo_decode_workspace_bytes")
    sh = L.stream_handle(dev)
    ws = WORKSPACES.get(dev, int(need), sh)
    with L.on_device(dev):
        rc = lib.halo_sharded_decode(ctypes.byref(prob), table.arr, table.n, ws.data_ptr(),
                                     ws.numel(), exchange.world, exchange.rank, exchange.bufs,
                                     L.halo_dtype(out.dtype), out.data_ptr(), out.stride(0),
                                     out.stride(1), lse.data_ptr() if lse is not None else None,
                                     sh)
    L.check(rc, "halo_sharded_decode")
    return out, lse


def chunked_decode(q: torch.Tensor, chunks, *, scale: Optional[float] = None,
                   q_pos: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                   out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                   prior: Optional[tuple] = None, max_split_rows: int = 0,
                   events: Optional[tuple] = None, want_lse: bool = True):
    """Attention of one decode query over ``chunks`` -- a list of
    ``(k, v, start, causal)`` tuples or a prepared :class:`ChunkTable` --
    merged with log-sum-exp.  Returns ``(out (B, H, D_v), lse (B, H))``;
    with ``want_lse=False`` and no ``lse`` given, the log-sum-exp is not
    written and ``None`` is returned in its place.

    ``prior = (m, l, o)`` folds a running fp32 state in first.  ``q_pos``
    (device int64 ``(B,)``) defaults to ``total_T - 1`` as in
    ``halo/triton_chunked.py:250-253`` (reference path relative to the
    lzbaclz/HALO root).  ``events = (begin, end)`` are raw ``cudaEvent_t``
    handles recorded around the split-KV kernel launches (profiling).
    """
    q3 = q.squeeze(2) if q.dim() == 4 else q
    _require_cuda(q3, "q")
    q3 = q3 if q3.is_contiguous() else q3.contiguous()
    B, H, D = q3.shape
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    table = chunks if isinstance(chunks, ChunkTable) else ChunkTable(chunks)
    D_v = table.D_v if table.D_v is not None else D
    if q_pos is None and table.any_causal:
        q_pos = torch.full((B,), table.total_rows - 1, dtype=torch.int64, device=q3.device)
    elif q_pos is not None and (q_pos.dtype != torch.int64 or q_pos.device != q3.device):
        q_pos = q_pos.to(device=q3.device, dtype=torch.int64).contiguous()
    if out is None:
        out = torch.empty(B, H, D_v, dtype=out_dtype or q3.dtype, device=q3.device)
    if lse is None and want_lse:
        lse = torch.empty(B, H, dtype=torch.float32, device=q3.device)
    mg = L.MergeArgs()
    mg.mode = L.MERGE_FINALIZE
    mg.out_dtype = L.halo_dtype(out.dtype)
    mg.out = out.data_ptr()
    mg.out_stride_b, mg.out_stride_h = out.stride(0), out.stride(1)
    mg.lse = lse.data_ptr() if lse is not None else None
    if prior is not None:
        m, l, o = prior
        mg.m, mg.l, mg.o = m.data_ptr(), l.data_ptr(), o.data_ptr()
    _decode_table(q3, table, scale=scale, q_pos=q_pos, merge=mg, max_split_rows=max_split_rows,
                  events=events)
    return out, lse


def accumulate_decode(q: torch.Tensor, chunks: Sequence[tuple], m: torch.Tensor, l: torch.Tensor,
                      o: torch.Tensor, *, scale: float, q_pos: Optional[torch.Tensor]) -> None:
    """Fold ``chunks`` into running fp32 accumulators ``(m, l, o)`` in place
    (the state ``update_chunk`` of ``halo/triton_chunked.py:151-192`` keeps)."""
    q3 = _last_contig(q.squeeze(2) if q.dim() == 4 else q)
    _require_cuda(q3, "q")
    for t, name in ((m, "m"), (l, "l"), (o, "o")):
        if t.dtype != torch.float32 or not t.is_contiguous():
            raise L.HaloError(f"accumulator {name} must be contiguous fp32", L.HALO_ERR_INVALID_ARG)
    structs, keep = [], []
    H_kv, D_v = q3.shape[1], o.shape[-1]
    for (k, v, start, causal) in chunks:
        H_kv, D_v = int(k.shape[1]), int(v.shape[-1])
        s, t = make_chunk(k, v, start, causal)
        structs.append(s)
        keep.append(t)
    if q_pos is not None:
        q_pos = q_pos.to(device=q3.device, dtype=torch.int64).contiguous()
    mg = L.MergeArgs()
    mg.mode = L.MERGE_ACCUMULATE
    mg.m, mg.l, mg.o = m.data_ptr(), l.data_ptr(), o.data_ptr()
    decode_raw(q3, structs, H_kv, D_v, scale=scale, q_pos=q_pos, merge=mg)


PREFILL_MAX_CHUNKS = 48   # chunk descriptors per halo_prefill_attention call


def prefill_supported(q: torch.Tensor, chunks: Sequence[tuple], scale: Optional[float] = None) -> bool:
    """Whether the tensor-core prefill kernel covers this problem: bf16 or
    fp16, head dim 64 or 128, value head dim equal to it, positive scale."""
    D = q.shape[-1]
    if q.dtype not in (torch.bfloat16, torch.float16) or D not in (64, 128):
        return False
    if scale is not None and not (math.isfinite(scale) and scale > 0):
        return False
    return all(k.dtype == q.dtype and v.dtype == q.dtype and k.shape[-1] == D and
               v.shape[-1] == D for (k, v, _s, _c) in chunks)


def prefill_attention(q: torch.Tensor, chunks: Sequence[tuple], *, query_pos_offset: int,
                      scale: Optional[float] = None, out_dtype: Optional[torch.dtype] = None,
                      out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                      state: Optional[tuple] = None, accumulate: bool = False,
                      events: Optional[tuple] = None):
    """Chunked-prefill attention on the tcgen05 kernel
    (``halo_prefill_attention_ws``): ``q (B, H, T_q, D)`` with query row ``i``
    at global position ``query_pos_offset + i`` over ``(k, v, start, causal)``
    chunks (``halo/kv_cache_chunked.py:873-942``).

    ``state = (m, l, o)``: fp32 running state, ``m, l (B, H, T_q)`` and
    ``o (B, H, T_q, D)`` contiguous.  ``accumulate=True`` folds the chunks
    into it in place and returns ``None``; otherwise the state (if given) is
    folded in and ``(out (B, H, T_q, D), lse (B, H, T_q))`` is returned, and
    the caller's state is left as it was.  Lists longer than one call takes
    (more than ``PREFILL_MAX_CHUNKS`` non-contiguous chunks) run as several
    calls through a running state of their own."""
    _require_cuda(q, "q")
    B, H, T_q, D = q.shape
    if q.stride(-1) != 1:
        q = q.contiguous()
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    H_kv = int(chunks[0][0].shape[1]) if chunks else H
    groups = [chunks[i:i + PREFILL_MAX_CHUNKS] for i in range(0, len(chunks), PREFILL_MAX_CHUNKS)]
    if not groups:
        groups = [[]]
    if accumulate and state is None:
        raise L.HaloError("accumulate needs state=(m, l, o)", L.HALO_ERR_INVALID_ARG)
    if len(groups) > 1 and not accumulate:
        # the groups fold into a state of this call's own (a copy of the
        # caller's, if given): the caller's tensors are only read
        if state is None:
            state = (torch.full((B, H, T_q), float("-inf"), dtype=torch.float32, device=q.device),
                     torch.zeros(B, H, T_q, dtype=torch.float32, device=q.device),
                     torch.zeros(B, H, T_q, D, dtype=torch.float32, device=q.device))
        else:
            state = tuple(t.clone() for t in state)
    lse_view = None
    if not accumulate:
        if out is None:
            out = torch.empty(B, H, T_q, D, dtype=out_dtype or q.dtype, device=q.device)
        if lse is None:
            lse = torch.empty(B, H, T_q, dtype=torch.float32, device=q.device)
        elif not lse.is_contiguous():
            # the kernel writes lse as contiguous (B, H, T_q); a strided
            # view (e.g. one slice of a whole prompt's lse) is filled after
            lse_view, lse = lse, torch.empty(B, H, T_q, dtype=torch.float32, device=q.device)
    lib = L.lib()
    for gi, grp in enumerate(groups):
        last = gi == len(groups) - 1
        prob = L.PrefillProblem()
        prob.B, prob.H, prob.H_kv, prob.T_q, prob.D = B, H, H_kv, T_q, D
        prob.dtype = L.halo_dtype(q.dtype)
        prob.q = q.data_ptr()
        prob.q_stride_b, prob.q_stride_h, prob.q_stride_t = q.stride(0), q.stride(1), q.stride(2)
        prob.q_pos0 = int(query_pos_offset)
        prob.scale = float(scale)
        if events is not None and last:
            prob.event_begin, prob.event_end = events
        structs, keep = [], []
        for (k, v, start, causal) in grp:
            _require_cuda(k, "k")
            st, t = make_chunk(k, v, start, causal)
            structs.append(st)
            keep.append(t)
        arr = (L.KVChunk * max(len(structs), 1))(*structs)
        po = L.PrefillOut()
        if state is not None:
            m, l, o = state
            po.m, po.l, po.o = m.data_ptr(), l.data_ptr(), o.data_ptr()
        if accumulate or not last:
            po.mode = L.MERGE_ACCUMULATE
        else:
            po.mode = L.MERGE_FINALIZE
            po.out_dtype = L.halo_dtype(out.dtype)
            po.out = out.data_ptr()
            po.out_stride_b, po.out_stride_h, po.out_stride_t = out.stride(0), out.stride(1), \
                out.stride(2)
            po.lse = lse.data_ptr()
        with torch.cuda.device(q.device):
            need = lib.halo_prefill_workspace_bytes(ctypes.byref(prob), arr, len(structs))
            if need < 0:
                L.check(int(need), "halo_prefill_workspace_bytes")
            ws = PREFILL_WORKSPACES.get(q.device, int(need)) if need > 0 else None
            rc = lib.halo_prefill_attention_ws(ctypes.byref(prob), arr, len(structs),
                                               ctypes.byref(po),
                                               ws.data_ptr() if ws is not None else None,
                                               ws.numel() if ws is not None else 0,
                                               L.stream_handle(q.device))
        L.check(rc, "halo_prefill_attention_ws")
    if accumulate:
        return None
    if lse_view is not None:
        lse_view.copy_(lse)
        lse = lse_view
    return out, lse


def multi_query_attention(q: torch.Tensor, chunks: Sequence[tuple], *, scale: Optional[float] = None,
                          query_pos_offset: int, out_dtype: Optional[torch.dtype] = None):
    """``T_q > 1`` queries (a chunked-prefill slice) over causal chunks: query
    row ``i`` sits at global position ``query_pos_offset + i``
    (``halo/kv_cache_chunked.py:873-942``).  bf16/fp16 with head dim 64 or
    128 run the tensor-core prefill kernel; other shapes run each query row
    as one decode problem whose K/V batch stride is zero, so every row reuses
    the same chunk memory.  Returns ``(out (B, H, T_q, D_v), lse (B, H, T_q))``."""
    _require_cuda(q, "q")
    B, H, T_q, D = q.shape
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if chunks and prefill_supported(q, chunks, scale):
        return prefill_attention(q, chunks, query_pos_offset=query_pos_offset, scale=scale,
                                 out_dtype=out_dtype)
    D_v = int(chunks[0][1].shape[-1]) if chunks else D
    H_kv = int(chunks[0][0].shape[1]) if chunks else H
    out = torch.empty(B, H, T_q, D_v, dtype=out_dtype or q.dtype, device=q.device)
    lse = torch.empty(B, H, T_q, dtype=torch.float32, device=q.device)
    qp = torch.arange(T_q, dtype=torch.int64, device=q.device) + int(query_pos_offset)
    for b in range(B):
        qb = q[b].transpose(0, 1).contiguous()   # (T_q, H, D)
        structs, keep = [], []
        for (k, v, start, causal) in chunks:
            s, t = make_chunk(k[b:b + 1], v[b:b + 1], start, causal, batch_stride_zero=True)
            structs.append(s)
            keep.append(t)
        ob = out[b].transpose(0, 1)          # (T_q, H, D_v) view
        lb = torch.empty(T_q, H, dtype=torch.float32, device=q.device)
        mg = L.MergeArgs()
        mg.mode = L.MERGE_FINALIZE
        mg.out_dtype = L.halo_dtype(ob.dtype)
        mg.out = ob.data_ptr()
        mg.out_stride_b, mg.out_stride_h = ob.stride(0), ob.stride(1)
        mg.lse = lb.data_ptr()
        decode_raw(qb, structs, H_kv, D_v, scale=scale, q_pos=qp, merge=mg)
        lse[b] = lb.transpose(0, 1)
    return out, lse


def multi_query_accumulate(q: torch.Tensor, chunks: Sequence[tuple], m: torch.Tensor,
                           l: torch.Tensor, o: torch.Tensor, *, scale: float,
                           query_pos_offset: int) -> None:
    """Fold ``chunks`` into running fp32 state for ``T_q > 1`` queries: query
    row ``i`` sits at position ``query_pos_offset + i``; causal chunks hide
    keys after it.  State layout ``m, l (B, T_q, H)``, ``o (B, T_q, H, D_v)``
    (contiguous), i.e. rows ordered (query row, head) per batch."""
    _require_cuda(q, "q")
    B, H, T_q, D = q.shape
    qp = torch.arange(T_q, dtype=torch.int64, device=q.device) + int(query_pos_offset)
    for b in range(B):
        table = ChunkTable(chunks, batch_stride_zero=True, batch=slice(b, b + 1))
        qb = q[b].transpose(0, 1).contiguous()          # (T_q, H, D)
        mg = L.MergeArgs()
        mg.mode = L.MERGE_ACCUMULATE
        mg.m, mg.l, mg.o = m[b].data_ptr(), l[b].data_ptr(), o[b].data_ptr()
        _decode_table(qb, table, scale=scale, q_pos=qp, merge=mg)


def lse_merge(m_parts: torch.Tensor, l_parts: Optional[torch.Tensor], o_parts: torch.Tensor, *,
              out_dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None,
              lse: Optional[torch.Tensor] = None, parts_major: bool = False):
    """Merge ``P`` partial states into ``(out (B, H, D_v), lse (B, H))``; the
    P-way form of ``halo/kv_cache_chunked.py:194-239``.

    Row-major (default): ``m/l (B, H, P)``, ``o (B, H, P, D_v)``.
    ``parts_major``: ``m/l (P, B, H)``, ``o (P, B, H, D_v)`` (e.g. gathered
    from P GPUs).  ``l_parts=None`` means every part is normalised (l = 1,
    ``m`` is its LSE).  All fp32.
    """
    if parts_major:
        P, B, H = m_parts.shape
    else:
        B, H, P = m_parts.shape
    D_v = o_parts.shape[-1]
    R = B * H
    for t in (m_parts, l_parts, o_parts):
        if t is None:
            continue
        _require_cuda(t, "partial")
        if t.dtype != torch.float32 or t.stride(-1) != 1:
            raise L.HaloError("partials must be fp32 with a contiguous last dim",
                              L.HALO_ERR_INVALID_ARG)
    if parts_major:
        ps, rs = m_parts.stride(0), 1
        ops_, ors = o_parts.stride(0), D_v
        if m_parts.stride(2) != 1 or m_parts.stride(1) != H or o_parts.stride(1) != H * D_v:
            raise L.HaloError("parts-major partials need contiguous (B, H) rows", L.HALO_ERR_INVALID_ARG)
    else:
        m_parts = m_parts.contiguous()
        o_parts = o_parts.contiguous()
        l_parts = l_parts.contiguous() if l_parts is not None else None
        ps, rs, ops_, ors = 1, P, D_v, P * D_v
    dev = m_parts.device
    if out is None:
        out = torch.empty(B, H, D_v, dtype=out_dtype, device=dev)
    if lse is None:
        lse = torch.empty(B, H, dtype=torch.float32, device=dev)
    mg = L.MergeArgs()
    mg.mode = L.MERGE_FINALIZE
    mg.out_dtype = L.halo_dtype(out.dtype)
    mg.out = out.data_ptr()
    mg.out_stride_b, mg.out_stride_h = out.stride(0), out.stride(1)
    mg.lse = lse.data_ptr()
    with torch.cuda.device(dev):
        rc = L.lib().halo_lse_merge(B, H, D_v, P, m_parts.data_ptr(),
                                    l_parts.data_ptr() if l_parts is not None else None,
                                    o_parts.data_ptr(), ps, rs, ops_, ors, ctypes.byref(mg),
                                    L.stream_handle(dev))
    L.check(rc, "halo_lse_merge")
    return out, lse


# ------------------------------------------------------------ paged cache
# These calls are a few microseconds of device time, so their host path is
# kept short: one test of everything that has to hold, and the reasons looked
# up only where it fails.

_get_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _call(fn, index: int, *args) -> int:
    """``fn(*args, stream)`` on device ``index`` and its current stream."""
    if _get_device() == index:
        return fn(*args, L.stream_handle_of(index))
    with torch.cuda.device(index):
        return fn(*args, L.stream_handle_of(index))


def _refuse(what: str) -> None:
    raise L.HaloError(what, L.HALO_ERR_INVALID_ARG)


def _int32s(index: int, tensors: dict) -> None:
    """Raise for the first of ``{name: (tensor, entries)}`` that is not
    contiguous int32 of that many entries on device ``index``."""
    for name, (t, n) in tensors.items():
        if not t.is_cuda:
            _refuse(f"{name} must be a CUDA tensor (no CPU path)")
        if t.get_device() != index or t.dtype != torch.int32:
            _refuse(f"{name} must be int32 on device {index}, got {t.dtype} on {t.device}")
        if t.numel() != n or not t.is_contiguous():
            _refuse(f"{name} must hold {n} contiguous entries, got shape {tuple(t.shape)}, "
                    f"strides {t.stride()}")


def _table(t: torch.Tensor, index: int) -> tuple:
    """``(R, max_blocks, row stride)`` of block tables on device ``index``."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or t.dtype is not torch.int32 or t.get_device() != index or \
            (shape[1] > 1 and stride[1] != 1):
        _refuse(f"block_tables must be int32 (R, max_blocks) with contiguous rows on device {index}")
    return shape[0], shape[1], stride[0]


def _page_pool(k: torch.Tensor, v: torch.Tensor, index: int, dtype: torch.dtype):
    """The packed C-ABI description of page pools ``(n_pages, H_kv, page_size,
    D)`` on device ``index``, with ``H_kv`` and ``D``."""
    shape = k.shape
    if len(shape) != 4 or v.shape != shape or k.dtype is not dtype or v.dtype is not dtype or \
            k.get_device() != index or v.get_device() != index:
        _refuse("k_pages and v_pages must be (n_pages, H_kv, page_size, D) of one shape, dtype and "
                "device, those of the rows")
    n, H_kv, page, D = shape
    ks, kh, kt, kd = k.stride()
    vs, vh, vt, vd = v.stride()
    if D > 1 and (kd != 1 or vd != 1):
        _refuse("page rows must be contiguous")
    return L.pack_page_pool(k.data_ptr(), v.data_ptr(), ks, kh, kt, vs, vh, vt, n, H_kv, page, D,
                            L.halo_dtype(dtype)), H_kv, D


def update_block_tables(block_tables: torch.Tensor, old_lens: torch.Tensor, new_lens: torch.Tensor,
                        free_pages: torch.Tensor, n_free: torch.Tensor, *, page_size: int,
                        max_tokens: int, n_free_out: Optional[torch.Tensor] = None):
    """Block tables, slots and positions from request lengths, on the device
    (``halo_update_block_tables``).

    ``block_tables (R, max_blocks)`` and ``free_pages`` (int32) are updated in
    place: requests whose length shrinks from ``old_lens`` to ``new_lens``
    ``(R,)`` give their last pages back to the end of
    ``free_pages[:n_free]``, requests that grow then take pages off its end,
    both in request order.  The length of the list that is left goes to
    ``n_free_out`` (default: ``n_free (1,)`` itself).

    Returns ``(slots, positions, cu_tokens, lens)``: slot and cache position
    (int64, ``max_tokens`` entries, -1 behind the last row) of the new rows of
    all requests packed in request order, their running count ``(R + 1,)``,
    and the lengths the requests now have -- ``old_lens`` for one that the
    free list or its table row cannot hold, which stays as it is."""
    if not block_tables.is_cuda:
        _refuse("block_tables must be a CUDA tensor (no CPU path)")
    i32, dev = torch.int32, block_tables.device
    index = dev.index
    R, max_blocks, tstride = _table(block_tables, index)
    if n_free_out is None:
        n_free_out = n_free
    if not (old_lens.dtype is i32 and new_lens.dtype is i32 and free_pages.dtype is i32 and
            n_free.dtype is i32 and n_free_out.dtype is i32 and
            old_lens.get_device() == index and new_lens.get_device() == index and
            free_pages.get_device() == index and n_free.get_device() == index and
            n_free_out.get_device() == index and
            old_lens.numel() == R and new_lens.numel() == R and n_free.numel() == 1 and
            n_free_out.numel() == 1 and old_lens.is_contiguous() and new_lens.is_contiguous() and
            free_pages.is_contiguous()):
        _int32s(index, {"old_lens": (old_lens, R), "new_lens": (new_lens, R),
                        "free_pages": (free_pages, free_pages.numel()), "n_free": (n_free, 1),
                        "n_free_out": (n_free_out, 1)})
    if max_tokens < 0:
        _refuse("max_tokens must not be negative")
    slots = torch.empty(max_tokens, dtype=torch.int64, device=dev)
    positions = torch.empty(max_tokens, dtype=torch.int64, device=dev)
    cu = torch.empty(R + 1, dtype=i32, device=dev)
    lens = torch.empty(R, dtype=i32, device=dev)
    rc = _call(L.lib().halo_update_block_tables, index, block_tables.data_ptr(),
               tstride, R, max_blocks, old_lens.data_ptr(), new_lens.data_ptr(),
               free_pages.data_ptr(), free_pages.numel(), n_free.data_ptr(), n_free_out.data_ptr(),
               page_size, max_tokens, slots.data_ptr(), positions.data_ptr(), cu.data_ptr(),
               lens.data_ptr())
    if rc:
        L.check(rc, "halo_update_block_tables")
    return slots, positions, cu, lens


def extend_block_tables(block_tables: torch.Tensor, held_lens: torch.Tensor,
                        context_lens: torch.Tensor, counts: torch.Tensor, rows: torch.Tensor,
                        starts: torch.Tensor, free_pages: torch.Tensor, n_free: torch.Tensor,
                        *, page_size: int, max_tokens: int):
    """``update_block_tables`` for a cache's next step
    (``halo_extend_block_tables``): room for ``counts (R,)`` rows (none where
    negative) behind contexts of ``context_lens`` rows, in pages that
    ``held_lens`` rows hold already or off the free list.  ``held_lens`` is
    updated in place and ``rows (R,)`` gets the rows granted to each request,
    0 for one whose rows do not fit.

    Returns ``(slots, positions, cu_tokens)``: places for all rows asked for,
    those of request ``r`` from ``starts[r]`` on (also written, ``(R,)``), -1
    where it is refused, and the running count of rows granted."""
    if not block_tables.is_cuda:
        _refuse("block_tables must be a CUDA tensor (no CPU path)")
    dev = block_tables.device
    index = dev.index
    R, max_blocks, tstride = _table(block_tables, index)
    _int32s(index, {"held_lens": (held_lens, R), "context_lens": (context_lens, R),
                    "counts": (counts, R), "rows": (rows, R), "starts": (starts, R),
                    "free_pages": (free_pages, free_pages.numel()), "n_free": (n_free, 1)})
    if max_tokens < 0:
        _refuse("max_tokens must not be negative")
    slots = torch.empty(max_tokens, dtype=torch.int64, device=dev)
    positions = torch.empty(max_tokens, dtype=torch.int64, device=dev)
    cu = torch.empty(R + 1, dtype=torch.int32, device=dev)
    rc = _call(L.lib().halo_extend_block_tables, index, block_tables.data_ptr(), tstride, R,
               max_blocks, held_lens.data_ptr(), context_lens.data_ptr(), counts.data_ptr(),
               free_pages.data_ptr(), free_pages.numel(), n_free.data_ptr(), page_size, max_tokens,
               slots.data_ptr(), positions.data_ptr(), cu.data_ptr(), rows.data_ptr(),
               starts.data_ptr())
    if rc:
        L.check(rc, "halo_extend_block_tables")
    return slots, positions, cu


def write_kv_pages(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                   slots: torch.Tensor) -> None:
    """Copy K/V rows ``(T, H_kv, D)`` into the slots ``(T,)`` (int64) of page
    pools ``(n_pages, H_kv, page_size, D)`` (``halo_write_kv_pages``).  Rows
    with a slot outside the pools (-1: none) are skipped; slots are distinct."""
    if not k_pages.is_cuda:
        _refuse("k_pages must be a CUDA tensor (no CPU path)")
    index, dtype, shape = k_pages.get_device(), k_pages.dtype, k.shape
    pool, H_kv, D = _page_pool(k_pages, v_pages, index, dtype)
    if len(shape) != 3 or shape[1] != H_kv or shape[2] != D or v.shape != shape or \
            k.dtype is not dtype or v.dtype is not dtype or \
            k.get_device() != index or v.get_device() != index:
        _refuse("k and v must be (T, H_kv, D) of the pools' dtype and device")
    T = shape[0]
    if slots.dtype is not torch.int64 or slots.get_device() != index or slots.numel() != T or \
            not slots.is_contiguous():
        _refuse("slots must be contiguous int64 (T,) on the pools' device")
    kt, kh, kd = k.stride()
    vt, vh, vd = v.stride()
    if D > 1 and (kd != 1 or vd != 1):
        k, v = k.contiguous(), v.contiguous()
        kt, kh, _ = k.stride()
        vt, vh, _ = v.stride()
    rc = _call(L.lib().halo_write_kv_pages, index, pool, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh,
               T, slots.data_ptr())
    if rc:
        L.check(rc, "halo_write_kv_pages")


# workspace bytes of halo_tree_attention by what they depend on, and the
# workspaces of calls outside a capture, which need no initial contents
_TREE_BYTES: dict = {}
_TREE_LOCAL = threading.local()
_TREE_KEPT = 4          # buffers a thread keeps: up to 39 MB each


def _tree_workspace(index: int, stream: int, need: int) -> torch.Tensor:
    """``need`` bytes for a call on ``stream``.  A thread's calls on one stream
    follow one another and share a buffer that grows, kept for the last
    ``_TREE_KEPT`` streams it came to; a captured call gets one of its own from
    the graph's pool, so that no two graphs share one."""
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(need, dtype=torch.uint8, device=f"cuda:{index}")
    bufs = _TREE_LOCAL.__dict__
    ws = bufs.get((index, stream))
    if ws is None or ws.numel() < need:
        ws = torch.empty(need, dtype=torch.uint8, device=f"cuda:{index}")
        if len(bufs) >= _TREE_KEPT and (index, stream) not in bufs:
            # the memory goes back to its own stream, behind the calls that use it
            del bufs[next(iter(bufs))]
        bufs[index, stream] = ws
    return ws


def tree_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                   block_tables: torch.Tensor, context_lens: torch.Tensor, cu_nodes: torch.Tensor,
                   tree_mask: torch.Tensor, *, scale: Optional[float] = None,
                   out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
                   lse: Optional[torch.Tensor] = None, want_lse: bool = True,
                   node_starts: Optional[torch.Tensor] = None):
    """Attention of drafted token trees over a paged K/V cache
    (``halo_tree_attention``).

    ``q (T, H, D)`` holds the nodes of all requests packed: request ``r``'s
    are rows ``cu_nodes[r]`` to ``cu_nodes[r + 1] - 1``, its node ``i`` at
    cache position ``context_lens[r] + i``, where its K/V row was written
    before.  A node sees every position of its context and the nodes ``j``
    with ``tree_mask[row, j]`` (bool ``(T, max_nodes)``); one that sees
    nothing gets zeros and a log-sum-exp of -inf.  With one node a request
    and a mask of ones this is a decode step over the paged cache.  With
    ``node_starts (R,)`` request ``r``'s ``cu_nodes[r + 1] - cu_nodes[r]`` rows
    begin there instead of at ``cu_nodes[r]``.

    Returns ``(out (T, H, D), lse (T, H))``; ``lse`` is ``None`` with
    ``want_lse=False`` and none given.  Rows that are no request's (those
    from ``cu_nodes[R]`` on) are not written.  bf16/fp16, head dim 64 or 128, a page size that is a multiple
    of 8."""
    if not q.is_cuda:
        _refuse("q must be a CUDA tensor (no CPU path)")
    index, dtype, qshape = q.get_device(), q.dtype, q.shape
    pool, H_kv, D = _page_pool(k_pages, v_pages, index, dtype)
    if len(qshape) != 3 or qshape[2] != D:
        _refuse("q must be (T, H, D) of the pools' dtype, device and head dim")
    T, H, _ = qshape
    R, max_blocks, tstride = _table(block_tables, index)
    if not (context_lens.dtype is torch.int32 and cu_nodes.dtype is torch.int32 and
            context_lens.get_device() == index and cu_nodes.get_device() == index and
            context_lens.numel() == R and cu_nodes.numel() == R + 1 and
            context_lens.is_contiguous() and cu_nodes.is_contiguous()):
        _int32s(index, {"context_lens": (context_lens, R), "cu_nodes": (cu_nodes, R + 1)})
    if node_starts is not None:
        _int32s(index, {"node_starts": (node_starts, R)})
    mshape, mstride = tree_mask.shape, tree_mask.stride()
    if len(mshape) != 2 or mshape[0] != T or tree_mask.get_device() != index or \
            tree_mask.dtype not in (torch.bool, torch.uint8) or (mshape[1] > 1 and mstride[1] != 1):
        _refuse("tree_mask must be bool (T, max_nodes) with contiguous rows on q's device")
    qt, qh, qd = q.stride()
    if qd != 1 and D > 1:
        q = q.contiguous()
        qt, qh, _ = q.stride()
    if out is None:
        out = torch.empty_like(q) if (out_dtype is None or out_dtype is dtype) and \
            q.is_contiguous() else torch.empty(T, H, D, dtype=out_dtype or dtype, device=q.device)
        ot, oh = H * D, D
    else:
        if out.shape != qshape or out.get_device() != index or (D > 1 and out.stride(2) != 1):
            _refuse("out must be (T, H, D) with contiguous rows on q's device")
        ot, oh, _ = out.stride()
    if lse is None:
        if want_lse:
            lse = torch.empty(T, H, dtype=torch.float32, device=q.device)
    elif lse.shape != (T, H) or lse.dtype is not torch.float32 or lse.get_device() != index or \
            not lse.is_contiguous():
        _refuse("lse must be contiguous fp32 (T, H) on q's device")
    if _get_device() != index:
        with torch.cuda.device(index):
            return tree_attention(q, k_pages, v_pages, block_tables, context_lens, cu_nodes,
                                  tree_mask, scale=scale, out=out, lse=lse, want_lse=want_lse,
                                  node_starts=node_starts)
    max_nodes = mshape[1]
    prob = L.pack_tree_problem(R, T, H, max_nodes, max_blocks,
                               scale if scale is not None else 1.0 / math.sqrt(D), q.data_ptr(), qt,
                               qh, block_tables.data_ptr(), tstride, context_lens.data_ptr(),
                               cu_nodes.data_ptr(), tree_mask.data_ptr(), mstride[0],
                               out.data_ptr(), ot, oh, L.halo_dtype(out.dtype),
                               lse.data_ptr() if lse is not None else 0,
                               node_starts.data_ptr() if node_starts is not None else 0)
    lib, stream = L.lib(), L.stream_handle_of(index)
    key = (index, D, H_kv, H, max_nodes, R > 0 and T > 0)
    need = _TREE_BYTES.get(key) if lse is not None else None
    if need is None:
        need = int(lib.halo_tree_workspace_bytes(pool, prob))
        if need < 0:
            L.check(need, "halo_tree_workspace_bytes")
        if lse is not None:            # one that is not asked for is kept there, of T rows
            _TREE_BYTES[key] = need
    ws = _tree_workspace(index, stream, need) if need else None
    rc = lib.halo_tree_attention(pool, prob, ws.data_ptr() if need else None, need, stream)
    if rc:
        L.check(rc, "halo_tree_attention")
    return out, lse


def commit_tree_path(k_pages: torch.Tensor, v_pages: torch.Tensor, block_tables: torch.Tensor,
                     context_lens: torch.Tensor, path: torch.Tensor,
                     path_lens: torch.Tensor) -> None:
    """Move the accepted nodes' K/V rows to the end of each request's context
    (``halo_commit_tree_path``): step ``i < path_lens[r]`` moves the row at
    position ``context_lens[r] + path[r, i]`` to ``context_lens[r] + i``.
    ``path (R, max_depth)`` (int32) holds node indices with
    ``path[r, i] >= i``, as paths from a root do when children are numbered
    after their parents; other steps move nothing."""
    if not k_pages.is_cuda:
        _refuse("k_pages must be a CUDA tensor (no CPU path)")
    index = k_pages.get_device()
    pool, _, _ = _page_pool(k_pages, v_pages, index, k_pages.dtype)
    R, max_blocks, tstride = _table(block_tables, index)
    pshape, pstride = path.shape, path.stride()
    if len(pshape) != 2 or pshape[0] != R or path.dtype is not torch.int32 or \
            path.get_device() != index or (pshape[1] > 1 and pstride[1] != 1):
        _refuse("path must be int32 (R, max_depth) with contiguous rows on the pools' device")
    if not (context_lens.dtype is torch.int32 and path_lens.dtype is torch.int32 and
            context_lens.get_device() == index and path_lens.get_device() == index and
            context_lens.numel() == R and path_lens.numel() == R and
            context_lens.is_contiguous() and path_lens.is_contiguous()):
        _int32s(index, {"context_lens": (context_lens, R), "path_lens": (path_lens, R)})
    rc = _call(L.lib().halo_commit_tree_path, index, pool, block_tables.data_ptr(), tstride,
               max_blocks, R, context_lens.data_ptr(), path.data_ptr(),
               pstride[0], pshape[1], path_lens.data_ptr())
    if rc:
        L.check(rc, "halo_commit_tree_path")
