"""Plain restatement of the paged-cache operators on the CPU: block tables as
lists, row moves one at a time, attention in 64 bits.  Inputs are CPU tensors;
nothing here touches the CUDA library."""
from __future__ import annotations

import math

import torch


def update_block_tables(table, old, new, free, n_free, page, max_tokens):
    """Returns ``(table, free, n_free, slots, positions, cu, lens)`` as lists,
    from lists (``table`` rows of one length, ``free`` with its capacity)."""
    table, free = [list(r) for r in table], list(free)
    width = len(table[0]) if table else 0
    R = len(old)
    blocks = lambda n: -(-n // page)                                    # noqa: E731
    fits = [o >= 0 and n >= 0 and blocks(o) <= width and blocks(n) <= width
            for o, n in zip(old, new)]
    stack = free[:n_free]
    for r in range(R):
        if fits[r] and blocks(new[r]) < blocks(old[r]):
            stack += table[r][blocks(new[r]):blocks(old[r])]
    lens, short = list(old), False
    for r in range(R):
        if not fits[r]:
            continue
        need = max(0, blocks(new[r]) - blocks(old[r]))
        if need and (short or need > len(stack)):
            short = True          # no later request overtakes one that waits for pages
            continue
        for b in range(need):
            table[r][blocks(old[r]) + b] = stack.pop()
        lens[r] = new[r]
    for i in range(n_free, len(stack)):
        free[i] = stack[i]
    slots, pos, cu = [], [], [0]
    for r in range(R):
        for t in range(old[r], lens[r]):
            slots.append(table[r][t // page] * page + t % page)
            pos.append(t)
        cu.append(len(slots))
    slots = (slots + [-1] * max_tokens)[:max_tokens]
    pos = (pos + [-1] * max_tokens)[:max_tokens]
    return table, free, len(stack), slots, pos, cu, lens


def extend_block_tables(table, held, ctx, counts, free, n_free, page, max_tokens):
    """Returns ``(table, free, n_free, slots, positions, cu, rows, starts, held)``."""
    want = [c + max(n, 0) if 0 <= c <= h else -1 for h, c, n in zip(held, ctx, counts)]
    table, free, n_free, _, _, _, lens = update_block_tables(table, held, want, free, n_free, page, 0)
    rows = [max(n, 0) if 0 <= w == got else 0 for n, w, got in zip(counts, want, lens)]
    slots, pos, cu, starts, at = [-1] * max_tokens, [-1] * max_tokens, [0], [], 0
    for r, n in enumerate(rows):
        starts.append(min(at, 2 ** 31 - 1))
        for i in range(min(n, max(0, max_tokens - at))):
            t = ctx[r] + i
            slots[at + i], pos[at + i] = table[r][t // page] * page + t % page, t
        cu.append(cu[-1] + n)
        at += max(counts[r], 0)
    return table, free, n_free, slots, pos, cu, rows, starts, lens


def write_kv_pages(k, v, k_pages, v_pages, slots):
    """In place on CPU pools; rows whose slot is outside the pools stay out."""
    n, _, page, _ = k_pages.shape
    for t, s in enumerate(slots):
        if 0 <= s < n * page:
            k_pages[s // page, :, s % page] = k[t]
            v_pages[s // page, :, s % page] = v[t]


def commit_tree_path(k_pages, v_pages, table, ctx, path, path_lens):
    n, page = k_pages.shape[0], k_pages.shape[2]
    for r, c in enumerate(ctx):
        moves = []
        for i in range(min(max(path_lens[r], 0), len(path[r]))):
            a, b = c + path[r][i], c + i
            if path[r][i] <= i or c < 0 or a // page >= len(table[r]):
                continue
            pa, pb = table[r][a // page], table[r][b // page]
            if 0 <= pa < n and 0 <= pb < n:
                moves.append((pa, a % page, pb, b % page))
        for x in (k_pages, v_pages):
            rows = [x[pa, :, ra].clone() for pa, ra, _, _ in moves]
            for row, (_, _, pb, rb) in zip(rows, moves):
                x[pb, :, rb] = row


def gather_rows(pages, row, n):
    """Rows 0 .. n-1 of a request from its table row, (H_kv, n, D) float64;
    entries that name no page read as zeros."""
    N, H, page, D = pages.shape
    out = torch.zeros(H, n, D, dtype=torch.float64)
    for b in range(-(-n // page)):
        m = min(page, n - b * page)
        if 0 <= row[b] < N:
            out[:, b * page:b * page + m] = pages[row[b], :, :m].double()
    return out


def tree_attention(q, k_pages, v_pages, table, ctx, cu, mask, scale=None):
    """``(out, lse, room)`` in 64 bits for the rows below ``cu[-1]``; ``room``
    is the error that the arithmetic of 32-bit sums allows for each output
    element and each lse (see ``allowed``)."""
    T, H, D = q.shape
    H_kv, page = k_pages.shape[1], k_pages.shape[2]
    G = H // H_kv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(T, H, D, dtype=torch.float64)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    room_o = torch.zeros(T, H, 1, dtype=torch.float64)
    room_l = torch.zeros(T, H, dtype=torch.float64)
    for r, c in enumerate(ctx):
        nodes = min(cu[r + 1] - cu[r], mask.shape[1])
        n = min(c + nodes, len(table[r]) * page)
        k = gather_rows(k_pages, table[r], n)
        v = gather_rows(v_pages, table[r], n)
        for i in range(nodes):
            t = cu[r] + i
            see = torch.ones(n, dtype=torch.bool)
            see[c:] = mask[t, :nodes].bool()[:n - c]
            if not see.any():
                continue
            for h in range(H):
                kk, vv = k[h // G][see], v[h // G][see]
                s = (kk @ q[t, h].double()) * scale
                m = s.max()
                w = torch.exp(s - m)
                z = w.sum()
                out[t, h] = (w @ vv) / z
                lse[t, h] = m + torch.log(z)
                reach = (kk.abs() @ q[t, h].double().abs()).max() * scale
                room_o[t, h], room_l[t, h] = allowed(float(reach), float(vv.abs().max()), D,
                                                     int(see.sum()), float(lse[t, h].abs()))
    return out, lse, room_o, room_l


def allowed(reach, vmax, D, n, lse):
    """Bounds on (|out error|, |lse error|) before out's own rounding.

    ``reach`` = scale * sum |q||k|.  A score is a sum of D exact products in
    32 bits: off by at most D * 2^-23 * reach (2^-23 a step: the tensor pipe
    may truncate).  A weight e^(s - m) is off by that factor twice (its own
    score and the maximum) plus 2^-21 from the exponential.  Weights enter
    P V as two 16-bit parts, the second rounded: off by at most 2^-16 of
    themselves in bf16; in fp16 by 2^-22 of themselves and 2^-32 of the largest
    weight, which for n up to 65536 keys is less than 2^-16 of their sum.  The sums over n keys add (n / 8 + 64) * 2^-23: eight or more
    keys a step of the matrix pipe, and at most 64 partial results joined."""
    e = 2.0 * D * 2.0 ** -23 * reach + 2.0 ** -21
    sums = (n / 8 + 64) * 2.0 ** -23
    return vmax * (2 * e + 2.0 ** -16 + 2 * sums), e + sums + 4 * 2.0 ** -23 * abs(lse)
