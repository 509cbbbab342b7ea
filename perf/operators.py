"""What is timed of the paged-cache operators, and their plain forms.

Four operators serve drafted trees of tokens over a paged K/V cache:

* ``update_block_tables`` grows or shrinks every request's block table from
  its lengths and returns the slots of the new tokens;
* ``write_kv_pages`` puts new K/V rows into their slots;
* ``tree_attention`` attends every drafted node to its request's context and
  to the nodes its mask shows;
* ``commit_tree_path`` moves the accepted nodes' rows to the end of the
  context.

``run`` computes them in elementary torch operations where ``own`` is false
and calls ``halo_b200.ops`` where it is true.
"""
import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------- cases
def _tree(name, R, ctx_lo, ctx_hi, nodes_lo, nodes_hi, H, H_kv, D, page, dtype):
    c = {"op": "tree", "R": R, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "nodes_lo": nodes_lo,
         "nodes_hi": nodes_hi, "H": H, "H_kv": H_kv, "D": D, "page": page, "dtype": dtype}
    return {**c, "name": name} if name else c


def _tables(name, R, old_lo, old_hi, new_lo, new_hi, shrink, page, spare):
    c = {"op": "tables", "R": R, "old_lo": old_lo, "old_hi": old_hi, "new_lo": new_lo,
         "new_hi": new_hi, "shrink": shrink, "page": page, "spare": spare}
    return {**c, "name": name} if name else c


def _write(name, T, reqs, pad, H_kv, D, page, dtype):
    c = {"op": "write", "T": T, "reqs": reqs, "pad": pad, "H_kv": H_kv, "D": D, "page": page,
         "dtype": dtype}
    return {**c, "name": name} if name else c


def _commit(name, R, ctx_lo, ctx_hi, nodes, depth, H_kv, D, page, dtype):
    c = {"op": "commit", "R": R, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "nodes": nodes,
         "depth": depth, "H_kv": H_kv, "D": D, "page": page, "dtype": dtype}
    return {**c, "name": name} if name else c


def listed():
    return [
        # one request, one token after a short prompt: latency alone counts
        _tree("tree: one token", 1, 1000, 1000, 1, 1, 32, 8, 128, 16, "bf16"),
        # a few chats with small drafts of different sizes
        _tree("tree: short chats", 8, 200, 3000, 3, 16, 32, 8, 128, 64, "bf16"),
        # eight requests at 32K, the length of the tiered decode workload
        _tree("tree: batch 8 at 32K", 8, 32768, 32768, 16, 16, 32, 8, 128, 64, "bf16"),
        # a ragged batch: small heads, wide groups, a page size that is no power of two
        _tree("tree: ragged batch", 32, 17, 16000, 1, 64, 16, 2, 64, 48, "fp16"),
        # full trees of 64 nodes at 64K, the length of the quantised decode workload
        _tree("tree: 64 nodes at 64K", 4, 65535, 65535, 64, 64, 32, 8, 128, 128, "bf16"),
        # one request of a million tokens, the sharded workload's layer on one GPU
        _tree("tree: 1M tokens", 1, 1048576, 1048576, 4, 4, 64, 8, 128, 256, "bf16"),
        # a decode step of a small batch: every request drafts up to 16 nodes
        _tables("tables: draft step", 8, 100, 30000, 1, 16, 0.0, 16, 64),
        # prompts join a large batch while others end or drop their rejected drafts
        _tables("tables: large batch", 1024, 1, 4000, 1, 128, 0.3, 16, 4096),
        # the drafted rows of one layer
        _write("write: draft rows", 127, 8, 9, 8, 128, 64, "bf16"),
        # the rows of a long prompt slice
        _write("write: prompt slice", 65536, 5, 100, 8, 128, 64, "bf16"),
        # a few accepted rows of a small batch
        _commit("commit: small batch", 8, 100, 3000, 16, 6, 8, 128, 64, "bf16"),
        # a large batch with deep accepted paths
        _commit("commit: large batch", 512, 50, 400, 64, 16, 8, 128, 16, "fp16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = ((32, 8), (64, 8), (16, 16), (28, 4), (16, 2), (12, 1), (24, 8))


def draw(rng):
    kind = rng.choice(("tree", "tree", "tree", "tables", "write", "commit"))
    page = rng.choice((8, 16, 24, 32, 48, 64, 128, 256))
    dtype = rng.choice(("bf16", "fp16"))
    D = rng.choice((64, 128))
    H, H_kv = rng.choice(HEADS)
    if kind == "tree":
        R = _log(rng, 1, 64)
        n_hi = _log(rng, 1, 256)
        n_lo = rng.randint(1, n_hi)
        ctx_hi = _log(rng, 1, 262144)
        # at most the listed cases' cache rows, products and scores
        most = min(4e9 / (R * H_kv * D * 4), 2.5e11 / (4.0 * D * H * n_hi * R),
                   5e8 / (R * H * n_hi))
        ctx_hi = max(1, min(ctx_hi, int(most)))
        ctx_lo = rng.randint(max(1, ctx_hi // 8), ctx_hi)
        return _tree(None, R, ctx_lo, ctx_hi, n_lo, n_hi, H, H_kv, D, page, dtype)
    if kind == "tables":
        R = _log(rng, 1, 1024)
        old_hi = _log(rng, 1, 30000)
        new_hi = _log(rng, 1, max(1, min(65536, 131072 // R)))
        return _tables(None, R, rng.randint(0, old_hi), old_hi, rng.randint(0, new_hi), new_hi,
                       rng.choice((0.0, 0.1, 0.5)), page, _log(rng, 1, 4096))
    if kind == "write":
        T = _log(rng, 1, 65536)
        return _write(None, T, _log(rng, 1, min(T, 256)), rng.randint(0, T // 4), H_kv, D, page,
                      rng.choice(("bf16", "fp16", "fp32")) if T < 30000 else dtype)
    R = _log(rng, 1, 512)
    ctx_hi = _log(rng, 1, 400)
    nodes = _log(rng, 1, 64)
    return _commit(None, R, rng.randint(1, ctx_hi), ctx_hi, nodes, rng.randint(1, min(16, nodes)),
                   H_kv, D, page, dtype)


def _between(case, what, n, lo, hi):
    """n whole numbers in [lo, hi], the same for every seed: the work of a case is fixed."""
    r = random.Random("%s %s %d %d %d" % (case["op"], what, n, lo, hi))
    return [r.randint(lo, hi) for _ in range(n)]


def _blocks(n, page):
    return -(-n // page)


# ----------------------------------------------------------------- prepare
def _rows(g, shape, dtype, outliers=False):
    x = torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32).to(dtype)
    if outliers:   # four channels of every head ten times as large, as keys have them
        at = torch.randint(0, shape[-1], (shape[1], 4), generator=g, device=DEVICE)
        f = torch.ones(shape[1], shape[-1], device=DEVICE, dtype=dtype).scatter_(1, at, 10.0)
        x.mul_(f[None, :, None])
    return x


def _page_table(rng, need, n_pages):
    """Block tables (R, most blocks) over distinct pages in random order; the rest of a row is 0."""
    order = rng.permutation(n_pages)
    t = np.zeros((len(need), max(1, max(need))), dtype=np.int32)
    at = 0
    for r, n in enumerate(need):
        t[r, :n] = order[at:at + n]
        at += n
    return t, order[at:]


def _dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEVICE)


def _prepare_tree(c, g, rng):
    R, D = c["R"], c["D"]
    ctx = _between(c, "ctx", R, c["ctx_lo"], c["ctx_hi"])
    nodes = _between(c, "nodes", R, c["nodes_lo"], c["nodes_hi"])
    N, T = max(nodes), sum(nodes)
    need = [_blocks(a + n, c["page"]) for a, n in zip(ctx, nodes)]
    n_pages = sum(need) + 3
    table, _ = _page_table(rng, need, n_pages)
    mask = np.zeros((T, N), dtype=bool)
    at = 0
    for n in nodes:      # a node sees itself and its ancestors
        m = mask[at:at + n]
        for i in range(n):
            if i:
                m[i] = m[i - 1 if rng.random() < 0.5 else rng.integers(0, i)]
            m[i, i] = True
        at += n
    dt = DTYPES[c["dtype"]]
    return {"q": torch.randn(T, c["H"], D, generator=g, device=DEVICE).to(dt),
            "k": _rows(g, (n_pages, c["H_kv"], c["page"], D), dt, outliers=True),
            "v": _rows(g, (n_pages, c["H_kv"], c["page"], D), dt),
            "table": _dev(table), "ctx": _dev(np.array(ctx, dtype=np.int32)),
            "cu": _dev(np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)),
            "mask": _dev(mask)}


def _tables_lens(c):
    old = _between(c, "old", c["R"], c["old_lo"], c["old_hi"])
    new = _between(c, "new", c["R"], c["new_lo"], c["new_hi"])
    r = random.Random("%d %d" % (c["R"], c["old_hi"]))
    to = []
    for a, n in zip(old, new):
        x = r.random()
        if x < c["shrink"] / 2:
            to.append(0)                     # the request has ended
        elif x < c["shrink"]:
            to.append(max(0, a - n))         # rejected drafts
        elif x > 0.95:
            to.append(a)                     # nothing new
        else:
            to.append(a + n)
    return old, to


def _prepare_tables(c, g, rng):
    old, to = _tables_lens(c)
    ob = [_blocks(a, c["page"]) for a in old]
    nb = [_blocks(a, c["page"]) for a in to]
    most = max(1, max(max(ob), max(nb)) + 1)
    n_pages = sum(ob) + sum(max(0, b - a) for a, b in zip(ob, nb)) + c["spare"]
    table, rest = _page_table(rng, ob, n_pages)
    full = np.zeros((c["R"], most), dtype=np.int32)
    full[:, :table.shape[1]] = table[:, :most]
    free = np.zeros(n_pages, dtype=np.int32)
    free[:len(rest)] = rest
    return {"table": _dev(full), "old": _dev(np.array(old, dtype=np.int32)),
            "new": _dev(np.array(to, dtype=np.int32)), "free": _dev(free),
            "n_free": torch.tensor([len(rest)], dtype=torch.int32, device=DEVICE),
            "n_free_out": torch.zeros(1, dtype=torch.int32, device=DEVICE),
            "tokens": max(1, sum(max(0, b - a) for a, b in zip(old, to)))}


def _prepare_write(c, g, rng):
    T, page = c["T"], c["page"]
    live = T - c["pad"]
    cuts = sorted(rng.integers(0, live + 1, c["reqs"] - 1).tolist())
    lens = np.diff([0] + cuts + [live])
    first = rng.integers(0, page, c["reqs"])
    need = [_blocks(int(a + n), page) if n else 0 for a, n in zip(first, lens)]
    n_pages = max(1, live // page + 2 * c["reqs"] + 2)
    table, _ = _page_table(rng, need, n_pages)
    slots = np.full(T, -1, dtype=np.int64)
    at = 0
    for r, n in enumerate(lens):
        pos = first[r] + np.arange(n)
        slots[at:at + n] = table[r][pos // page].astype(np.int64) * page + pos % page
        at += n
    dt = DTYPES[c["dtype"]]
    kv = torch.randn(T, 2, c["H_kv"], c["D"], generator=g, device=DEVICE).to(dt)
    return {"new_k": kv[:, 0], "new_v": kv[:, 1], "slots": _dev(slots),
            "k": _rows(g, (n_pages, c["H_kv"], page, c["D"]), dt),
            "v": _rows(g, (n_pages, c["H_kv"], page, c["D"]), dt)}


def _prepare_commit(c, g, rng):
    R, page, nodes, depth = c["R"], c["page"], c["nodes"], c["depth"]
    ctx = _between(c, "ctx", R, c["ctx_lo"], c["ctx_hi"])
    lens = _between(c, "path", R, 1, depth)
    need = [_blocks(a + nodes, page) for a in ctx]
    n_pages = sum(need) + 1
    table, _ = _page_table(rng, need, n_pages)
    path = np.zeros((R, depth), dtype=np.int32)
    for r in range(R):
        path[r, :lens[r]] = np.sort(rng.choice(nodes, lens[r], replace=False))
    dt = DTYPES[c["dtype"]]
    return {"k": _rows(g, (n_pages, c["H_kv"], page, c["D"]), dt),
            "v": _rows(g, (n_pages, c["H_kv"], page, c["D"]), dt), "table": _dev(table),
            "ctx": _dev(np.array(ctx, dtype=np.int32)), "path": _dev(path),
            "path_lens": _dev(np.array(lens, dtype=np.int32))}


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    rng = np.random.default_rng(seed)
    make = {"tree": _prepare_tree, "tables": _prepare_tables, "write": _prepare_write,
            "commit": _prepare_commit}[case["op"]]
    return {"op": case["op"], "page": case["page"], **make(case, g, rng)}


# --------------------------------------------------------------------- run
def _plain_tree(s):
    q, kp, vp, ctx, cu, mask = s["q"], s["k"], s["v"], s["ctx"].long(), s["cu"].long(), s["mask"]
    T, H, D = q.shape
    H_kv, page = kp.shape[1], kp.shape[2]
    R, N = ctx.numel(), mask.shape[1]
    dev = q.device
    n = cu[1:] - cu[:-1]
    node = torch.arange(N, device=dev)
    row = (cu[:-1, None] + node).clamp(max=T - 1)                       # (R, N)
    tab = s["table"].long()
    L = tab.shape[1] * page
    k = kp[tab].float().transpose(1, 2).reshape(R, H_kv, L, D)
    qg = q[row].float().view(R, N, H_kv, H // H_kv, D).permute(0, 2, 3, 1, 4)
    sc = torch.matmul(qg.reshape(R, H_kv, -1, D), k.transpose(2, 3))
    del k
    sc = sc.mul_(1.0 / math.sqrt(D)).view(R, H_kv, H // H_kv, N, L)
    at = torch.arange(L, device=dev) - ctx[:, None]                     # node of each position
    seen = mask[row].gather(2, at.clamp(0, N - 1)[:, None].expand(R, N, L))
    seen &= ((at >= 0) & (at < n[:, None]))[:, None]
    seen |= (at < 0)[:, None]
    sc.masked_fill_(~seen[:, None, None], float("-inf"))
    m = sc.amax(-1, keepdim=True)
    m0 = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    p = sc.sub_(m0).exp_()
    l = p.sum(-1, keepdim=True)
    v = vp[tab].float().transpose(1, 2).reshape(R, H_kv, L, D)
    o = torch.matmul(p.view(R, H_kv, -1, L), v).view(R, H_kv, H // H_kv, N, D)
    o = torch.where(l > 0, o / l, torch.zeros_like(o))
    lse = torch.where(l > 0, m0 + l.log(), torch.full_like(l, float("-inf")))
    t = torch.arange(T, device=dev)
    r = torch.searchsorted(cu, t, right=True) - 1
    i = t - cu[r]
    out = o.permute(0, 3, 1, 2, 4).reshape(R, N, H, D)[r, i].to(q.dtype)
    return out, lse.permute(0, 3, 1, 2, 4).reshape(R, N, H)[r, i]


def _plain_tables(s):
    """Pages come off the end of the free list in request order, after the
    pages of the shrunk requests were put there."""
    table, old, new, free, page = (s["table"], s["old"].long(), s["new"].long(), s["free"],
                                   s["page"])
    R, MB = table.shape
    dev = table.device
    n_free = s["n_free"].long()
    ob, nb = (old + page - 1) // page, (new + page - 1) // page
    ok = (old >= 0) & (new >= 0) & (ob <= MB) & (nb <= MB)
    zero = torch.zeros_like(ob)
    give = torch.where(ok, (ob - nb).clamp(min=0), zero)
    need = torch.where(ok, (nb - ob).clamp(min=0), zero)
    give_end, need_end = give.cumsum(0), need.cumsum(0)
    have = n_free + give_end[-1:]
    ok &= (need == 0) | (need_end <= have)
    used = torch.where(ok & (need > 0), need_end, zero).amax(0, keepdim=True)
    lens = torch.where(ok, new, old)
    # the free list with what the shrunk requests give back behind it
    cap = free.numel()
    i = torch.arange(cap, device=dev)
    back = (i - n_free).clamp(min=0)
    r = torch.searchsorted(give_end, back, right=True).clamp(max=R - 1)
    b = (nb[r] + back - (give_end[r] - give[r])).clamp(0, MB - 1)
    stack = torch.where(i < n_free, free.long(), table[r, b].long())
    # the new pages of each request
    blk = torch.arange(MB, device=dev)
    j = blk - ob[:, None]
    gets = (ok & (need > 0))[:, None] & (j >= 0) & (j < need[:, None])
    at = (have - 1 - (need_end - need)[:, None] - j).clamp(0, cap - 1)
    pages = torch.where(gets, stack[at], table.long())
    left = have - used
    free.copy_(torch.where((i >= n_free) & (i < left), stack, free.long()))
    table.copy_(pages)
    # the slots of the new tokens
    count = torch.where(ok, (new - old).clamp(min=0), zero)
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), count.cumsum(0)])
    t = torch.arange(s["tokens"], device=dev)
    r = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=R - 1)
    live = t < cu[-1]
    pos = torch.where(live, old[r] + t - cu[r], torch.full_like(t, -1))
    slot = pages[r, (pos // page).clamp(0, MB - 1)] * page + pos % page
    slot = torch.where(live, slot, torch.full_like(t, -1))
    return {"slots": slot, "positions": pos, "cu": cu.int(), "lens": lens.int(), "table": table,
            "free": free, "n_free": left.int()}


def _plain_write(s):
    kp, vp, slots, page = s["k"], s["v"], s["slots"], s["page"]
    # a row without a slot repeats row 0, which has one
    i = torch.where(slots >= 0, torch.arange(slots.numel(), device=slots.device),
                    torch.zeros_like(slots))
    at = slots[i]
    pg, row = at // page, at % page
    kp[pg, :, row] = s["new_k"][i]
    vp[pg, :, row] = s["new_v"][i]
    return kp, vp


def _plain_commit(s):
    kp, vp, page = s["k"], s["v"], s["page"]
    path, ctx = s["path"].long(), s["ctx"].long()
    i = torch.arange(path.shape[1], device=path.device).expand_as(path)
    i = torch.where(i < s["path_lens"][:, None], i, torch.zeros_like(i))   # others repeat step 0
    src, dst = ctx[:, None] + path.gather(1, i), ctx[:, None] + i
    tab = s["table"].long()
    sp, dp = tab.gather(1, src // page), tab.gather(1, dst // page)
    k, v = kp[sp, :, src % page], vp[sp, :, src % page]
    kp[dp, :, dst % page] = k
    vp[dp, :, dst % page] = v
    return kp, vp


def _own_run(s):
    from halo_b200 import ops
    if s["op"] == "tree":
        return ops.tree_attention(s["q"], s["k"], s["v"], s["table"], s["ctx"], s["cu"], s["mask"])
    if s["op"] == "tables":
        slots, pos, cu, lens = ops.update_block_tables(
            s["table"], s["old"], s["new"], s["free"], s["n_free"], page_size=s["page"],
            max_tokens=s["tokens"], n_free_out=s["n_free_out"])
        return {"slots": slots, "positions": pos, "cu": cu, "lens": lens, "table": s["table"],
                "free": s["free"], "n_free": s["n_free_out"]}
    if s["op"] == "write":
        ops.write_kv_pages(s["new_k"], s["new_v"], s["k"], s["v"], s["slots"])
    else:
        ops.commit_tree_path(s["k"], s["v"], s["table"], s["ctx"], s["path"], s["path_lens"])
    return s["k"], s["v"]


def run(state):
    if own:
        return _own_run(state)
    return {"tree": _plain_tree, "tables": _plain_tables, "write": _plain_write,
            "commit": _plain_commit}[state["op"]](state)


# ------------------------------------------------------------ work and exact
def work(case):
    c, size = case, 4 if case.get("dtype") == "fp32" else 2
    if c["op"] == "tree":
        ctx = _between(c, "ctx", c["R"], c["ctx_lo"], c["ctx_hi"])
        nodes = _between(c, "nodes", c["R"], c["nodes_lo"], c["nodes_hi"])
        T, rows = sum(nodes), sum(a + n for a, n in zip(ctx, nodes))
        return {"bytes": rows * c["H_kv"] * c["D"] * 2 * size + T * c["H"] * (2 * c["D"] * size + 4)
                + T * max(nodes) + 4 * sum(_blocks(a + n, c["page"]) for a, n in zip(ctx, nodes)),
                "flops": 4.0 * c["D"] * c["H"] * sum(a * n for a, n in zip(ctx, nodes))}
    if c["op"] == "tables":
        old, to = _tables_lens(c)
        new = sum(max(0, b - a) for a, b in zip(old, to))
        moved = sum(abs(_blocks(b, c["page"]) - _blocks(a, c["page"])) for a, b in zip(old, to))
        return {"bytes": 16 * c["R"] + 8 * moved + 16 * new, "flops": 0}
    if c["op"] == "write":
        return {"bytes": (c["T"] - c["pad"]) * c["H_kv"] * c["D"] * size * 4 + 8 * c["T"],
                "flops": 0}
    lens = _between(c, "path", c["R"], 1, c["depth"])
    return {"bytes": sum(lens) * c["H_kv"] * c["D"] * size * 4 + 8 * c["R"], "flops": 0}


def _exact_tree(s):
    """Softmax attention of every node over its context and the nodes shown to
    it, one request and one K/V head at a time, in 64 bits."""
    q, mask = s["q"], s["mask"]
    T, H, D = q.shape
    H_kv, page = s["k"].shape[1], s["k"].shape[2]
    G = H // H_kv
    out = torch.zeros(T, H, D, dtype=torch.float64, device=q.device)
    lse = torch.full((T, H), float("-inf"), dtype=torch.float64, device=q.device)
    cu, ctx = s["cu"].tolist(), s["ctx"].tolist()
    for r, a in enumerate(ctx):
        lo, n = cu[r], cu[r + 1] - cu[r]
        pages = s["table"][r, :_blocks(a + n, page)].long()
        hidden = ~mask[lo:lo + n, :n]
        for h in range(H_kv):
            k = s["k"][pages, h].reshape(-1, D)[:a + n].double()
            v = s["v"][pages, h].reshape(-1, D)[:a + n].double()
            for e in range(h * G, h * G + G):
                x = (q[lo:lo + n, e].double() @ k.T) * D ** -0.5
                x[:, a:][hidden] = float("-inf")
                top = x.max(1, keepdim=True).values
                w = torch.exp(x - top)
                z = w.sum(1, keepdim=True)
                out[lo:lo + n, e] = (w @ v) / z
                lse[lo:lo + n, e] = (top + torch.log(z))[:, 0]
    return out, lse


def exact(case, seed):
    s = prepare(case, seed)
    page = s["page"]
    if s["op"] == "tree":
        return _exact_tree(s)
    if s["op"] == "tables":
        return None
    k, v = s["k"].double(), s["v"].double()
    if s["op"] == "write":
        live = torch.nonzero(s["slots"] >= 0)[:, 0]
        slot = s["slots"][live]
        for h in range(k.shape[1]):
            k[slot // page, h, slot % page] = s["new_k"][live, h].double()
            v[slot // page, h, slot % page] = s["new_v"][live, h].double()
        return k, v
    table, path, lens, ctx = (s[x].tolist() for x in ("table", "path", "path_lens", "ctx"))
    src, dst = [], []
    for r, n in enumerate(lens):
        for i in range(n):
            a, b = ctx[r] + path[r][i], ctx[r] + i
            src.append(table[r][a // page] * page + a % page)
            dst.append(table[r][b // page] * page + b % page)
    src, dst = torch.tensor(src, device=k.device), torch.tensor(dst, device=k.device)
    for x in (k, v):
        rows = x[src // page, :, src % page]
        x[dst // page, :, dst % page] = rows
    return k, v
