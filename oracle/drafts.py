"""Trees of drafted tokens over a K/V cache, in float64 NumPy (no
counterpart in the reference, which decodes one token per sequence): what
the drafts see, their attention, the page pool's bookkeeping and the
accepted path's rows, each written from its definition, one element at a
time."""

from __future__ import annotations

import numpy as np


def tree_visibility(parents, count=None):
    """``sees [N, N]`` (bool) and ``depths [N]`` of one tree: draft i sees
    itself and every ancestor; a parent outside ``[0, i)`` makes a root;
    drafts at or past ``count`` see nothing and have depth -1."""
    n = len(parents)
    count = n if count is None else count
    sees = np.zeros((n, n), dtype=bool)
    depths = np.full(n, -1, dtype=np.int32)
    for i in range(min(n, count)):
        at, steps = i, 0
        sees[i, i] = True
        while 0 <= parents[at] < at:
            at = int(parents[at])
            sees[i, at] = True
            steps += 1
        depths[i] = steps
    return sees, depths


def mask_words(sees):
    """``sees [..., N]`` as 64-bit words ``[..., ceil(N / 64)]`` (int64)."""
    sees = np.asarray(sees, dtype=bool)
    words = (sees.shape[-1] + 63) // 64
    out = np.zeros(sees.shape[:-1] + (words,), dtype=np.uint64)
    for j in range(sees.shape[-1]):
        out[..., j // 64] |= sees[..., j].astype(np.uint64) << np.uint64(j % 64)
    return out.view(np.int64)


def tree_attention(q, k, v, sees, prefix, scale):
    """One sequence: ``q [N, Hq, D]``, its rows ``k [R, Hkv, D]``,
    ``v [R, Hkv, Dv]``, ``sees [N, N]``.  Draft i attends rows below
    ``prefix`` and rows ``prefix + j < R`` with ``sees[i, j]``.  Only those
    rows enter its sums.  Returns ``(out, weight)``: the result and
    ``sum p |v| / sum p``, which bounds what roundings of p do to it."""
    n, hq, _ = q.shape
    rows, hkv, dv = v.shape
    out, weight = np.zeros((n, hq, dv)), np.zeros((n, hq, dv))
    for i in range(n):
        mine = [j for j in range(rows) if j < prefix or sees[i, j - prefix]]
        if not mine:
            continue
        for h in range(hq):
            g = h // (hq // hkv)
            with np.errstate(invalid="ignore", over="ignore"):
                s = (k[mine, g].astype(np.float64) @ q[i, h].astype(np.float64)) * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                x = v[mine, g].astype(np.float64)
                out[i, h] = (p[:, None] * x).sum(0)
                weight[i, h] = (p[:, None] * np.abs(x)).sum(0)
    return out, weight


def resize(table, lengths, free, count, targets, page_size, tokens):
    """The page pool's bookkeeping, sequence after sequence, on lists that
    are changed in place (``free`` is a stack of which ``count`` entries are
    in use).  Returns ``(count, rows, granted)`` with ``rows`` the packed
    ``(slot, position, sequence)`` of every new row."""
    capacity = len(table[0]) * page_size

    def pages(rows):
        return -(-rows // page_size)

    def valid(b):
        return 0 <= targets[b] <= capacity and 0 <= lengths[b] <= capacity

    given = []
    for b in range(len(lengths)):
        if valid(b) and targets[b] < lengths[b]:
            for c in range(pages(targets[b]), pages(lengths[b])):
                given.append(table[b][c])
                table[b][c] = -1
    for page in reversed(given):
        free[count] = page
        count += 1
    have, wanted, new_rows = count, 0, 0
    rows, granted = [], []
    for b in range(len(lengths)):
        if not valid(b):
            granted.append(0)
            continue
        need = max(0, pages(targets[b]) - pages(lengths[b]))
        more = max(0, targets[b] - lengths[b])
        wanted += need
        new_rows += more
        ok = (need == 0 or wanted <= have) and (more == 0 or new_rows <= tokens)
        granted.append(int(ok))
        if not ok:
            continue
        for c in range(need):
            count -= 1
            table[b][pages(lengths[b]) + c] = free[count]
        for p in range(lengths[b], targets[b]):
            rows.append((table[b][p // page_size] * page_size + p % page_size, p, b))
        lengths[b] = targets[b]
    return count, rows, granted


def commit(rows, prefix, path, accepted):
    """``rows [R, ...]`` of one sequence after the accepted path's rows have
    moved up behind the prefix."""
    out = np.array(rows, copy=True)
    last = -1
    for i in range(min(accepted, len(path))):
        if path[i] <= last:
            break
        last = path[i]
        if prefix + path[i] < len(out):
            out[prefix + i] = rows[prefix + path[i]]
    return out
