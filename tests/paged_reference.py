"""The paged step's operators in plain Python and 64-bit numpy, from their definitions in include/silvann_b200.h."""
import math

import numpy as np

BAD_PAGE, NO_PAGES, BAD_STEP = 0x80000000, 0x20000000, 0x10000000


def tables(lens, counts, table, free, free_at, rows, pool_pages, page):
    """(new_lens, table, row_start, seq, pos, slot, free_at, free, status) of one step."""
    lens, counts = [int(x) for x in lens], [int(x) for x in counts]
    table, free = np.array(table, np.int32), np.array(free, np.int32)
    seqs, most = len(lens), table.shape[1] * page
    held = [-(-n // page) if n > 0 else 0 for n in lens]
    status = 0
    back = sum(held[s] for s in range(seqs) if counts[s] == -1)
    need = sum(max(0, -(-(lens[s] + counts[s]) // page) - held[s]) for s in range(seqs) if counts[s] > 0)
    if any(n < 0 or c < -1 or n + max(c, 0) > most for n, c in zip(lens, counts)) or sum(max(c, 0) for c in counts) > rows or free_at > len(free) or back > free_at:
        status = BAD_STEP
    elif need > len(free) - (free_at - back):
        status = NO_PAGES
    out = {k: np.full(rows, -1, np.int32) for k in ("seq", "pos", "slot")}
    start = np.zeros(seqs + 1, np.int32)
    if status:
        return dict(new_lens=np.array(lens, np.int32), table=table, row_start=start, free_at=free_at, free=free, status=status, **out)
    at = free_at - back
    for s in range(seqs):
        if counts[s] == -1:
            for col in range(held[s]):
                free[at] = table[s, col]
                status |= 0 if 0 <= table[s, col] < pool_pages else BAD_PAGE
                at += 1
    at = free_at - back
    new, r = list(lens), 0
    for s in range(seqs):
        start[s] = r
        if counts[s] == -1:
            new[s] = 0
            continue
        new[s] += counts[s]
        for col in range(held[s], -(-new[s] // page)):
            table[s, col] = free[at]
            status |= 0 if 0 <= free[at] < pool_pages else BAD_PAGE
            at += 1
        for p in range(lens[s], new[s]):
            pg = int(table[s, p // page])
            out["seq"][r], out["pos"][r] = s, p
            if 0 <= pg < pool_pages:
                out["slot"][r] = pg * page + p % page
            else:
                status |= BAD_PAGE
            r += 1
    start[seqs] = r
    return dict(new_lens=np.array(new, np.int32), table=table, row_start=start, free_at=at, free=free, status=status, **out)


def sparse_row(q, k, v, means, row, p, page, block, first, last, top):
    """One row over one kv head: q [group][d], k, v [slots][d], means [blocks][d] in 64 bits; `row` the sequence's page numbers
    (-1: none).  (chosen ids, output [group][d], m [group], l [group], score error scale [group])."""
    n, keep = p // block + 1, first + last + top
    start = lambda b: row[b * block // page] * page + (b * block) % page if row[b * block // page] >= 0 else -1
    ids = list(range(n))
    if n > keep:
        s = []
        for b in range(first, n - last):
            x = float(np.dot(q.sum(0), means[start(b) // block])) if start(b) >= 0 else -math.inf
            s.append(-math.inf if math.isnan(x) else x + 0.0)
        best = sorted(range(len(s)), key=lambda i: (-s[i], i))[:top]
        ids = sorted(list(range(first)) + [first + i for i in best] + list(range(n - last, n)))
    ks, vs = [], []
    for b in ids:
        live = min(block, p + 1 - b * block)
        a = start(b)
        ks.append(k[a:a + live] if a >= 0 else np.zeros((live, k.shape[1])))
        vs.append(v[a:a + live] if a >= 0 else np.zeros((live, k.shape[1])))
    ks, vs = np.concatenate(ks), np.concatenate(vs)
    s = q @ ks.T / math.sqrt(q.shape[1])
    m = s.max(1)
    w = np.exp(s - m[:, None])
    size = (np.abs(q) @ np.abs(ks).T / math.sqrt(q.shape[1])).max(1)
    return ids, (w @ vs) / w.sum(1, keepdims=True), m, w.sum(1), size, np.abs(vs).max()
