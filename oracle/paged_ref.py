"""numpy restatement of the paged cache and the drafted trees, in 64 bits (tests only)."""
from __future__ import annotations

import numpy as np


def page_plan(ctx, new, held, table, free, n_free, page, n_pages, n_tokens):
    """The plan of one call: dict of slot, pos, seq [n_tokens], cu, short, n_held, n_free, table."""
    table, held = table.copy(), list(held)
    slot, pos, seq = (np.full(n_tokens, -1, np.int64) for _ in range(3))
    cu, short, used, asked = [0], [], 0, 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        total = -(-(c + n) // page)
        need = max(0, total - held[b])
        if total > table.shape[1]:
            short.append(need)
            table[b, held[b]:] = -1
        elif need and asked + need > n_free:
            short.append(need)
            asked += need
            table[b, held[b]:total] = -1
        else:
            short.append(0)
            for k in range(need):
                table[b, held[b] + k] = free[n_free - 1 - (asked + k)]
            asked += need
            used += need
            held[b] += need
        for i in range(n):
            r = cu[-1] + i
            if r < n_tokens:
                pos[r], seq[r] = c + i, b
                if short[b] == 0:
                    slot[r] = table[b, (c + i) // page] * page + (c + i) % page
        cu.append(cu[-1] + n)
    return dict(slot=slot, pos=pos, seq=seq, cu=np.array(cu), short=np.array(short), n_held=np.array(held),
                n_free=n_free - used, table=table)


def tree_masks(parent, cu):
    """Ancestor masks (Python ints): bit j of row r = its request's node j is the row's node or above it."""
    out = []
    for b in range(len(cu) - 1):
        line = []
        for j in range(cu[b + 1] - cu[b]):
            up = int(parent[cu[b] + j])
            line.append((1 << j) | (line[up] if up >= 0 else 0))
        out += line
    return out


def tree_attn(q, rows, ctx, cu, masks, table, page, scale, sel=None):
    """(ctx, lse, spread) in float64 for each row r: q [n, H, D], rows [slots, D], sel a list of
    position lists or None. ``spread`` = sum_t p_t |v_t|, the scale of the rounding bounds."""
    n, H, D = q.shape
    dv = 512
    o, lse, a = np.zeros((n, H, dv)), np.full((n, H), -np.inf), np.zeros((n, H, dv))
    for b in range(len(ctx)):
        for r in range(cu[b], cu[b + 1]):
            m = masks[r]
            see = [t for t in range(ctx[b], ctx[b] + cu[b + 1] - cu[b]) if m >> (t - ctx[b]) & 1]
            keys = np.concatenate([np.arange(ctx[b]), np.array(see, np.int64)]).astype(np.int64)
            if sel is not None:
                keys = np.intersect1d(keys, np.asarray(sel[r], np.int64))
            if not len(keys):
                continue
            k = rows[table[b][keys // page].astype(np.int64) * page + keys % page].astype(np.float64)
            z = q[r].astype(np.float64) @ k.T * scale
            top = z.max(1, keepdims=True)
            e = np.exp(z - top)
            lse[r] = top[:, 0] + np.log(e.sum(1))
            p = e / e.sum(1, keepdims=True)
            o[r], a[r] = p @ k[:, :dv], p @ np.abs(k[:, :dv])
    return o, lse, a


def tree_walk(parent, draft, target):
    """Accepted path (node indices) of one request and the next token."""
    if not len(parent):
        return [], -1
    path = [0]
    while True:
        cur = path[-1]
        child = [j for j in range(cur + 1, len(parent)) if parent[j] == cur and draft[j] == target[cur]]
        if not child:
            return path, int(target[cur])
        path.append(child[0])
