"""Workspaces of tree attention that calls outside a capture keep."""
from __future__ import annotations

import pytest
import torch

from test_paged_gpu import DEV, Case, _i32

pytestmark = pytest.mark.gpu


def test_workspaces_of_many_streams_are_not_kept(cuda_device):
    """A thread that goes through many streams keeps a few buffers, and calls
    whose buffer was given up meanwhile come out right."""
    from halo_b200 import ops
    c = Case(5, [9000, 300], [40, 3], 8, 2, 128, 16, torch.bfloat16)
    args = (c.q.to(DEV), c.k.to(DEV), c.v.to(DEV), _i32(c.table), _i32(c.ctx), _i32(c.cu),
            c.mask.to(DEV))
    want, lse = ops.tree_attention(*args, out_dtype=torch.float32)
    c.check(want, lse)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(20)]
    outs = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ops.tree_attention(*args, out_dtype=torch.float32))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) and torch.equal(l, lse) for o, l in outs)
    assert len(ops._TREE_LOCAL.__dict__) <= ops._TREE_KEPT
    kept = list(ops._TREE_LOCAL.__dict__.values())
    again = ops.tree_attention(*args, out_dtype=torch.float32)      # the first stream again
    assert torch.equal(again[0], want) and len(ops._TREE_LOCAL.__dict__) <= ops._TREE_KEPT
    assert sum(x.numel() for x in kept) <= ops._TREE_KEPT * 40e6
