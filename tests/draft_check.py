"""Plain models for the operators over drafted trees: which rows a node sees, the path that the
targets agree with, what stays of a pool, and a sampled token by its definition."""
import math

import numpy as np
import torch

from paged_check import attend_64


def line_of(parents, node):
    """The node and its ancestors, root last."""
    line = []
    while node >= 0:
        line.append(node)
        node = parents[node]
    return line


def rows_seen(base, parents, node, window, first):
    """Rows of the sequence that a node of its tree sees."""
    line = line_of(parents, node)
    pos = base + len(line) - 1

    def in_sight(p):
        return window == 0 or p > pos - window or p < first
    seen = [r for r in range(base) if in_sight(r)]
    return seen + sorted(base + v for d, v in enumerate(line) if in_sight(pos - d))


def attend_tree_64(q, kv, parents, window, first, sinks):
    """paged_check.attend_64 of one tree's nodes; kv: all rows of the sequence."""
    base, parts = kv.shape[0] - len(parents), []
    for i in range(len(parents)):
        rows = kv[torch.tensor(rows_seen(base, parents, i, window, first), device=q.device)]
        parts.append(attend_64(q[i:i + 1], rows, [rows.shape[0] - 1], 0, 0, sinks))
    cat = lambda xs: torch.cat(list(xs))
    return cat(p[0] for p in parts), (cat(p[1][0] for p in parts), cat(p[1][1] for p in parts)), cat(p[2] for p in parts)


def random_tree(rng, n, shape):
    if shape == "chain":
        return [i - 1 for i in range(n)]
    if shape == "roots":
        return [-1 if rng.random() < 0.3 or i == 0 else rng.randrange(i) for i in range(n)]
    if shape == "star":
        return ([-1] + [0] * (n - 1))[:n]
    return ([-1] + [rng.randrange(max(0, i - 5), i) for i in range(1, n)])[:n]


def walk(parents, tokens, targets):
    """(path, next)"""
    if not parents:
        return [], -1
    path = [0]
    while True:
        t = targets[path[-1]]
        kids = [c for c, p in enumerate(parents) if p == path[-1] and c > path[-1] and tokens[c] == t and t >= 0]
        if not kids:
            return path, t
        path.append(kids[0])


def keep_model(m, seqs, sizes, paths):
    """paged_check.PoolModel m after keep; its status."""
    if len(set(seqs)) < len(seqs) or any(not 0 <= s < len(m.rows) for s in seqs):
        return -22
    for s, n, path in zip(seqs, sizes, paths):
        if n > m.rows[s] or path != sorted(set(path)) or any(not 0 <= v < n for v in path):
            return -22
        if n and any(m.refs[p] != 1 for p in m.table[s][(m.rows[s] - n) // m.page:]):
            return -22
    for s, n, path in zip(seqs, sizes, paths):
        base = m.rows[s] - n
        place = lambda r: m.table[s][r // m.page] * m.page + r % m.page
        for tags in m.tags:
            now = [tags[place(base + v)] for v in path]
            for i, tag in enumerate(now):
                tags[place(base + i)] = tag
    for s, n, path in zip(seqs, sizes, paths):
        assert m.free([s], [m.rows[s] - n + len(path)]) == 0
    return 0


def sample_64(logits, t, k, p, m, u):
    """(token, probability) of one row, from the definition."""
    x = logits.astype(np.float64)
    if np.isnan(x).any() or (x == np.inf).any() or not (x > -np.inf).any():
        return -1, math.nan
    order = np.lexsort((np.arange(x.size), -x))
    if t == 0:
        return int(order[0]), 1.0
    k = k if 0 < k < x.size else x.size
    with np.errstate(under="ignore"):
        w = np.exp((x[order] - x[order[0]]) / np.float64(np.float32(t)))
    first = np.arange(x.size) == 0
    stays = np.arange(x.size) < k
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        stays &= (before < np.float64(np.float32(p)) * w[:k].sum()) | first
    stays &= (w >= np.float64(np.float32(m))) | first
    kept = np.zeros(x.size)
    kept[order[stays]] = w[stays]
    run = np.cumsum(kept)
    over = np.nonzero((run > np.float64(np.float32(u)) * run[-1]) & (kept > 0))[0]
    token = int(over[0]) if over.size else int(np.nonzero(kept)[0][-1])
    return token, kept[token] / run[-1]
