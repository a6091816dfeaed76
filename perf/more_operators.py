"""Operators of a speculative decoding step over a paged FP8 KV cache: attention for
trees of drafted tokens, sampling from logits, and the accepted path's rows kept.

One latent KV head of 512 dims per cache row (448 FP8 E4M3 dims with a power-of-two
scale per 64, 64 RoPE dims in f16), `heads` query heads over it. A pool holds pages of
`page` rows for all layers; a table names each sequence's pages, `refs` says how many
sequences hold a page. A sequence's drafted nodes are its last rows, node 0 the root.

Kinds:

  tree    attention of the nodes of a ragged batch of trees: the cached rows in a window
          with a few first ones kept visible, and each node's ancestors
  sample  tokens from rows of logits and given random numbers: temperature, top-k, top-p,
          min-p, each row with its own
  accept  the path of the tree that the sampled tokens agree with; its rows moved to the
          front of the drafts in all layers, the sequence cut behind them
  step    the operators together: extend, append, attend, sample, accept

`run` computes them in plain torch, or with the framework's calls where `own` is set.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DIM, NOPE, ROT = 512, 448, 64
ROW_BYTES = NOPE + 8 + 2 * ROT
SCALE = 1.0 / math.sqrt(DIM)
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
ITEM = {"bf16": 2, "fp32": 4}
DEV = "cuda"


# ---- the cases ---------------------------------------------------------------------------

def listed():
    return [
        # A small tree of one sequence: launches and latency count.
        {"name": "tree_one", "kind": "tree", "seqs": 1, "cached": 1500, "nodes": 7, "shape": "random", "heads": 64,
         "window": 0, "first": 0, "page": 64, "type": "bf16", "sinks": True},
        # A batch of ragged contexts, every cached row visible: matrix products count.
        {"name": "tree_batch", "kind": "tree", "seqs": 16, "cached": 8192, "nodes": 24, "shape": "random", "heads": 64,
         "window": 0, "first": 0, "page": 256, "type": "bf16", "sinks": True},
        # Many sequences in the model's 128-token window.
        {"name": "tree_window", "kind": "tree", "seqs": 48, "cached": 4096, "nodes": 13, "shape": "wide", "heads": 64,
         "window": 128, "first": 4, "page": 64, "type": "bf16", "sinks": True},
        # A tensor-parallel slice of the heads with fp32 queries, as the Q producer hands them over; chains.
        {"name": "tree_slice_fp32", "kind": "tree", "seqs": 5, "cached": 20000, "nodes": 33, "shape": "chain",
         "heads": 8, "window": 0, "first": 0, "page": 16, "type": "fp32", "sinks": False},
        # One user's next token: latency.
        {"name": "sample_one", "kind": "sample", "rows": 1, "vocab": 129280, "peaked": True, "type": "bf16",
         "filters": "k+p"},
        # Every node of a batch, rows with filters of their own (or none, or the largest logit): the logits' bytes count.
        {"name": "sample_batch", "kind": "sample", "rows": 256, "vocab": 129280, "peaked": True, "type": "bf16",
         "filters": "mixed"},
        # A vocabulary that no vector width divides, fp32 logits, few rows.
        {"name": "sample_odd_fp32", "kind": "sample", "rows": 33, "vocab": 32003, "peaked": True, "type": "fp32",
         "filters": "p+m"},
        # A flat distribution (high temperature) whose nucleus is a good part of the vocabulary.
        {"name": "sample_flat", "kind": "sample", "rows": 24, "vocab": 65536, "peaked": False, "type": "fp32",
         "filters": "p"},
        # Two sequences of one layer: launches and latency count.
        {"name": "accept_small", "kind": "accept", "seqs": 2, "cached": 70, "nodes": 9, "shape": "random", "layers": 1,
         "page": 16},
        # A batch over the model's 43 layers: the rows' copies count.
        {"name": "accept_batch", "kind": "accept", "seqs": 64, "cached": 300, "nodes": 48, "shape": "random",
         "layers": 43, "page": 64},
        # One step of a batch: the operators as they are used together.
        {"name": "step", "kind": "step", "seqs": 8, "cached": 2000, "nodes": 16, "shape": "random", "heads": 64,
         "window": 1000, "first": 16, "page": 64, "type": "bf16", "vocab": 129280, "filters": "k+p", "layers": 1,
         "sinks": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "sample", "sample", "sample", "accept", "accept", "step"])
    page = rng.choice([16, 32, 64, 128, 256])
    shape = rng.choice(["random", "random", "wide", "chain"])
    attn = {"heads": rng.choice([8, 16, 32, 64, 64, 128]), "type": rng.choice(["bf16", "bf16", "fp32"]),
            "sinks": rng.random() < 0.5, "first": rng.choice([0, 1, 4, 37, 128])}
    if kind == "tree":
        seqs, nodes = _log_int(rng, 1, 60), _log_int(rng, 1, 300)
        nodes = max(1, min(nodes, 1200 // seqs))
        most = max(40, min(60000, 2500000 // (seqs * nodes)))
        return {"kind": kind, "seqs": seqs, "cached": _log_int(rng, 1, most), "nodes": nodes, "shape": shape,
                "window": rng.choice([0, 1]) * _log_int(rng, 1, 3000), "page": page, **attn}
    if kind == "sample":
        rows = _log_int(rng, 1, 256)
        return {"kind": kind, "rows": rows, "vocab": _log_int(rng, 8, min(200000, 15000000 // rows)),
                "peaked": rng.random() < 0.7, "type": rng.choice(["bf16", "fp32"]),
                "filters": rng.choice(["none", "k", "p", "m", "k+p", "p+m", "mixed"])}
    if kind == "accept":
        seqs, layers = _log_int(rng, 1, 60), rng.choice([1, 4, 43])
        return {"kind": kind, "seqs": seqs, "cached": rng.choice([0, 1, 63, 64, 200, 301]),
                "nodes": _log_int(rng, 1, 200 if seqs < 12 else 45), "shape": shape, "layers": layers, "page": page}
    return {"kind": kind, "seqs": rng.choice([1, 3, 8]), "cached": _log_int(rng, 1, 3000), "nodes": _log_int(rng, 1, 16),
            "shape": shape, "window": rng.choice([0, 64, 999]), "page": page, "vocab": rng.choice([1000, 32003, 100000]),
            "filters": rng.choice(["none", "k+p", "mixed"]), "layers": 1, **attn}


def _rng(case, what):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")) + what)


def _ragged(case, n, longest, what):
    """n lengths that the case alone fixes, `longest` among them."""
    rng = _rng(case, what)
    some = [_log_int(rng, max(longest // 12, 1), max(longest, 1)) if longest else 0 for _ in range(n)]
    some[rng.randrange(n)] = longest
    return some


def _tree(rng, n, shape):
    """Parents of n nodes, level after level; node 0 is the root. A node has a child or two, or (wide) eight."""
    parents, turn = [-1], {"chain": 1.0, "random": 0.6, "wide": 0.12}[shape]
    for i in range(1, n):
        parents.append(min(i - 1, max(parents[-1], 0) + (i > 1 and rng.random() < turn)))
    return parents


def _path(rng, parents):
    """A path from the root. Passes are repeated on one state and do not write the drafts again, so a moved
    row is none that another one moves to: each pass finds what the first one found."""
    n, best = len(parents), [0]
    for _ in range(40):
        path = [0]
        while rng.random() < 0.85:
            kids = [i for i in range(path[-1] + 1, n) if parents[i] == path[-1]]
            if not kids:
                break
            path.append(rng.choice(kids))
        moved = [v for i, v in enumerate(path) if v != i]
        if all(v >= len(path) for v in moved) and len(path) > len(best):
            best = path
    return best


def _trees(case):
    """Per sequence: cached rows, parents of its nodes, the path that is accepted."""
    cached = _ragged(case, case["seqs"], case["cached"], "cached")
    sizes = _ragged(case, case["seqs"], case["nodes"], "nodes")
    rng = _rng(case, "trees")
    parents = [_tree(rng, n, case["shape"]) for n in sizes]
    return cached, parents, [_path(rng, p) for p in parents]


def _pages(rows, page):
    return -(-rows // page)


def _depths(parents):
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    return depth


def _attention_work(case):
    heads, window, first = case["heads"], case["window"], case["first"]
    pairs, read, nodes = 0, 0, 0
    for base, parents, _ in zip(*_trees(case)):
        nodes += len(parents)
        lo = 0 if window == 0 else max(0, base - window + 1)
        read += base - lo + min(first, lo) + len(parents)
        for d in _depths(parents):
            lo = 0 if window == 0 else max(0, min(base, base + d - window + 1))
            pairs += base - lo + min(first, lo) + (d + 1 if window == 0 else min(d + 1, window))
    return {"bytes": read * ROW_BYTES + 2 * nodes * heads * DIM * ITEM[case["type"]] + 4 * nodes,
            "flops": 4 * DIM * heads * pairs}


def work(case):
    kind = case["kind"]
    if kind == "tree":
        return _attention_work(case)
    if kind == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * ITEM[case["type"]] + 28), "flops": 2 * case["rows"] * case["vocab"]}
    cached, parents, paths = _trees(case)
    nodes = sum(map(len, parents))
    moved = sum(v != i for path in paths for i, v in enumerate(path)) * case["layers"]
    move = 2 * moved * ROW_BYTES + 16 * nodes
    if kind == "accept":
        return {"bytes": move, "flops": 0}
    w = _attention_work(case)
    return {"bytes": w["bytes"] + move + nodes * (2 * case["vocab"] + 4 * DIM + ROW_BYTES), "flops": w["flops"]}


# ---- inputs ------------------------------------------------------------------------------

def _gen(seed, k):
    return torch.Generator(DEV).manual_seed((int(seed) * 1000003 + 7919 * k) % (1 << 62))


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _quantize(x):
    """Rows [n, 512] as the cache's three arrays."""
    blocks = x[:, :NOPE].unflatten(-1, (7, 64))
    e = torch.ceil(torch.log2(blocks.abs().amax(-1).clamp_min(1e-4) / 448.0))
    codes = (blocks * torch.exp2(-e)[..., None]).flatten(1).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, torch.nn.functional.pad(e.to(torch.int8), (0, 1)), x[:, NOPE:].half()


def _rows(gen, n):
    """n cache rows ~N(0,1), one in a hundred eight times as large."""
    parts = []
    for a in range(0, n, 1 << 18):
        m = min(n - a, 1 << 18)
        x = torch.randn((m, DIM), generator=gen, device=DEV)
        parts.append(_quantize(x * torch.where(torch.rand((m, 1), generator=gen, device=DEV) < 0.01, 8.0, 1.0)))
    return [torch.cat(p)[None] for p in zip(*parts)]


def _anything(gen, layers, n):
    """Rows of whatever the layers hold: finite codes, exponents and tails."""
    def ints(width, lo, hi, dtype):
        return torch.randint(lo, hi, (layers, n, width), generator=gen, dtype=dtype, device=DEV)
    return ints(NOPE, 0, 0x7F, torch.uint8), ints(8, -9, 3, torch.int8), ints(ROT, 0, 0x7C00, torch.int16).view(torch.float16)


def _logits(gen, rows, vocab, peaked, dtype):
    """Logits ~1.5 N(0,1), with a few dozen likely tokens where the model is sure of something; else flat."""
    x = torch.randn((rows, vocab), generator=gen, device=DEV)
    if peaked:
        x *= 1.5
        some = min(vocab, 40)
        at = torch.randint(0, vocab, (rows, some), generator=gen, device=DEV)
        up = 8.0 - 2.5 * torch.log(torch.rand((rows, some), generator=gen, device=DEV).clamp_min(1e-4))
        x.scatter_reduce_(1, at, up, "amax")
    return x.to(dtype)


def _filters(case, rows, seed):
    """Temperature, top-k, top-p, min-p and the random number of each row."""
    rng, f = random.Random(seed * 31 + rows), case["filters"]
    flat = case["kind"] == "sample" and not case["peaked"]
    mixes = ["none", "k", "p", "m", "k+p", "p+m", "k+p+m", "greedy"]
    each = [rng.choice(mixes) if f == "mixed" else f for _ in range(rows)]
    t = [0.0 if "greedy" in e else rng.uniform(0.9, 1.3) if flat else rng.uniform(0.5, 1.1) for e in each]
    k = [rng.choice([1, 8, 20, 50, 200]) if "k" in e.split("+") else 0 for e in each]
    p = [rng.uniform(0.5, 0.98) if "p" in e.split("+") else 1.0 for e in each]
    m = [rng.uniform(0.02, 0.2) if "m" in e.split("+") else 0.0 for e in each]
    floats = torch.tensor([t, p, m], dtype=torch.float32, device=DEV)
    return {"temperature": floats[0], "top_k": _i32(k), "top_p": floats[1], "min_p": floats[2],
            "u": torch.rand(rows, generator=_gen(seed, 9), device=DEV)}


def prepare(case, seed):
    kind = case["kind"]
    s = {"case": case}
    if kind == "sample":
        s["logits"] = _logits(_gen(seed, 5), case["rows"], case["vocab"], case["peaked"], TYPES[case["type"]])
        s["filters"] = _filters(case, case["rows"], seed)
        return s
    page = case["page"]
    cached, parents, paths = _trees(case)
    seqs, sizes = len(parents), [len(p) for p in parents]
    rng = random.Random(seed)
    s["sizes"], s["depth"] = sizes, max(map(max, map(_depths, parents))) + 1
    s["q_start"] = _i32([sum(sizes[:i]) for i in range(seqs + 1)])
    s["parents"] = _i32([p for tree in parents for p in tree])
    s["seqs"] = _i32(list(range(seqs)))
    s["n_new"] = _i32(sizes)
    # pages of the cached rows in any order; the drafts take the lowest free ones, as they do when they are appended
    full = [b + n for b, n in zip(cached, sizes)]
    n_pages = sum(_pages(r, page) for r in full) + 3
    free = list(range(n_pages))
    rng.shuffle(free)
    table, refs = [[-1] * _pages(max(full), page) for _ in full], [0] * n_pages
    for i, b in enumerate(cached):
        for c in range(_pages(b, page)):
            table[i][c] = free.pop()
            refs[table[i][c]] = 1
    s["rows_in"] = list(cached)
    if kind != "step":
        free.sort(reverse=True)
        for i, (b, r) in enumerate(zip(cached, full)):
            for c in range(_pages(b, page), _pages(r, page)):
                table[i][c] = free.pop()
                refs[table[i][c]] = 1
        s["rows_in"] = full
    s["table_in"], s["refs_in"], s["rows_in"] = _i32(table), _i32(refs), _i32(s["rows_in"])
    s["table"], s["refs"], s["rows"] = s["table_in"].clone(), s["refs_in"].clone(), s["rows_in"].clone()
    if kind == "accept":
        s["codes"], s["sexp"], s["tail"] = _anything(_gen(seed, 0), case["layers"], n_pages * page)
    else:
        s["codes"], s["sexp"], s["tail"] = _rows(_gen(seed, 0), n_pages * page)
        s["q"] = torch.randn((sum(sizes), case["heads"], DIM), generator=_gen(seed, 1), device=DEV).to(TYPES[case["type"]])
        s["sinks"] = torch.randn((case["heads"],), generator=_gen(seed, 2), device=DEV) if case["sinks"] else None
    if kind == "tree":
        return s
    # drafted tokens, different ones in each tree, and what the model says after each node
    vocab = case.get("vocab", 100000)
    tokens, targets = [], []
    for path, n in zip(paths, sizes):
        mine = rng.sample(range(vocab), n + 1)
        after = [mine[n]] * n
        for a, b in zip(path, path[1:]):
            after[a] = mine[b]
        tokens += mine[:n]
        targets += after
    s["tokens"], s["targets"] = _i32(tokens), _i32(targets)
    if kind == "step":
        s["kv"] = torch.randn((sum(sizes), DIM), generator=_gen(seed, 3), device=DEV)
        s["logits"] = _logits(_gen(seed, 5), sum(sizes), vocab, True, torch.bfloat16)
        s["logits"][torch.arange(sum(sizes), device=DEV), s["targets"].long()] = 40.0
        s["filters"] = _filters(case, sum(sizes), seed)
        s["n_nodes"] = sum(sizes)
    return s


# ---- the operators in plain torch ----------------------------------------------------------

def _values(codes, sexp, tail):
    """Rows as fp32: f16(code * 2^e) and the f16 tail."""
    x = codes.view(torch.float8_e4m3fn).float().unflatten(-1, (7, 64))
    x = (x * torch.exp2(sexp[..., :7].float())[..., None]).half().float()
    return torch.cat([x.flatten(-2), tail.float()], -1)


def _attend(s):
    """Sequence by sequence: the nodes' scores over the rows from the first one that any sees."""
    case, out, a = s["case"], torch.empty_like(s["q"]), 0
    window, first, page = case["window"], case["first"], case["page"]
    cached = _trees(case)[0]
    for i, (n, base) in enumerate(zip(s["sizes"], cached)):
        q, up = s["q"][a:a + n].float(), s["parents"][a:a + n].long()
        # above[v, j]: j is v or one of its ancestors
        each = torch.arange(n, device=DEV)
        above, node, depth = torch.zeros((n, n), dtype=torch.bool, device=DEV), each, torch.zeros_like(each)
        for _ in range(s["depth"]):
            above |= (node[:, None] == each) & (node >= 0)[:, None]
            node = torch.where(node >= 0, up[node.clamp_min(0)], -1)
            depth += node >= 0
        pos = base + depth
        lo = 0 if window == 0 else max(0, base - window + 1)
        old = torch.cat([torch.arange(min(first, lo), device=DEV), torch.arange(lo, base, device=DEV)])
        at = torch.cat([old, pos])   # positions of the rows, and which nodes see them
        sees = torch.cat([torch.ones((n, old.numel()), dtype=torch.bool, device=DEV), above], 1)
        if window:
            sees &= (at[None] > pos[:, None] - window) | (at < first)[None]
        rows = torch.cat([old, base + each])
        rows = s["table"][i, rows // page].long() * page + rows % page
        k = _values(s["codes"][0, rows], s["sexp"][0, rows], s["tail"][0, rows])
        score = torch.where(sees[:, None], (q @ k.T) * SCALE, -math.inf)
        top = score.amax(-1, keepdim=True)
        if s["sinks"] is not None:
            top = torch.maximum(top, s["sinks"][None, :, None])
        p = torch.exp(score - top)
        den = p.sum(-1, keepdim=True)
        if s["sinks"] is not None:
            den = den + torch.exp(s["sinks"][None, :, None] - top)
        out[a:a + n] = ((p @ k) / den).to(out.dtype)
        a += n
    return out


def _sample(logits, temperature, top_k, top_p, min_p, u):
    """In 64 bits: sums over a whole vocabulary are compared with given borders."""
    x, at = torch.sort(logits.float(), dim=-1, descending=True, stable=True)
    greedy = temperature == 0
    t = torch.where(greedy, 1.0, temperature).double()[:, None]
    w = torch.exp((x.double() - x[:, :1].double()) / t)
    rank = torch.arange(x.shape[1], device=x.device)[None]
    keep = (rank < top_k[:, None]) | (top_k <= 0)[:, None]
    w = torch.where(keep, w, 0.0)
    before = torch.cumsum(w, -1) - w
    top_p = top_p.double()[:, None]
    keep &= (before < top_p * w.sum(-1, keepdim=True)) | (top_p >= 1.0) | (rank == 0)
    keep &= (w >= min_p.double()[:, None]) | (rank == 0)
    keep &= ~greedy[:, None] | (rank == 0)
    kept = torch.zeros_like(w).scatter_(1, at, torch.where(keep, w, 0.0))   # in the vocabulary's order
    total = kept.sum(-1, keepdim=True)
    passed = (torch.cumsum(kept, -1) > u.double()[:, None] * total) & (kept > 0)
    token = passed.to(torch.int8).argmax(-1, keepdim=True)
    return token[:, 0].to(torch.int32), (kept.gather(1, token) / total)[:, 0].float()


def _walk(s, targets):
    """The accepted nodes of each tree: packed paths (-1 behind them), their lengths, the next tokens."""
    q_start, dev = s["q_start"].long(), DEV
    n, most = s["parents"].numel(), max(s["sizes"])
    seqs = len(s["sizes"])
    cols = torch.arange(most, device=dev)[None]
    there = cols < (q_start[1:] - q_start[:-1])[:, None]
    at = torch.where(there, q_start[:-1, None] + cols, 0)
    up = torch.where(there, s["parents"][at], -2)
    tokens = s["tokens"][at]
    path = torch.full((n + 1,), -1, dtype=torch.int32, device=dev)
    node = torch.zeros((seqs, 1), dtype=torch.long, device=dev)
    length, going = torch.zeros(seqs, dtype=torch.int32, device=dev), torch.ones(seqs, dtype=torch.bool, device=dev)
    for d in range(s["depth"]):
        path[torch.where(going, q_start[:-1] + d, n)] = node[:, 0].to(torch.int32)
        length += going
        says = targets[q_start[:-1] + node[:, 0]]
        fits = (up == node) & (tokens == says[:, None])
        going = going & fits.any(1)
        node = torch.where(going[:, None], fits.to(torch.int8).argmax(1, keepdim=True), node)
    return path[:n], length, targets[q_start[:-1] + node[:, 0]]


def _keep(s, path, length):
    """Rows of the paths to the front of the drafts; the sequences cut behind them."""
    table, refs, rows, page = s["table"], s["refs"], s["rows"], s["case"]["page"]
    q_start = s["q_start"].long()
    each = torch.arange(path.numel(), device=DEV)
    seq = (each[:, None] >= q_start[None, 1:]).sum(1)
    base = rows.long() - (q_start[1:] - q_start[:-1])
    node = torch.where(path >= 0, path, each - q_start[seq])   # (behind a path: itself)
    src, dst = base[seq] + node, base[seq] + each - q_start[seq]
    src = table[seq, src // page].long() * page + src % page
    dst = table[seq, dst // page].long() * page + dst % page
    for name in ("codes", "sexp", "tail"):
        # a path's row reads what was there before; the rest stays
        s[name][:, dst] = torch.where((path >= 0)[None, :, None], s[name][:, src], s[name][:, dst])
    now = base + length
    cols = torch.arange(table.shape[1], device=DEV)[None] * page
    gone = (cols < rows.long()[:, None]) & (cols >= now[:, None])
    refs.index_add_(0, torch.where(gone, table, 0).flatten().long(), -gone.flatten().int())
    rows.copy_(now)


def _extend(s):
    table, refs, rows, page = s["table"], s["refs"], s["rows"], s["case"]["page"]
    n, q_start = s["parents"].numel(), s["q_start"].long()
    each = torch.arange(n, device=DEV)
    seq = (each[:, None] >= q_start[None, 1:]).sum(1)
    r = rows.long()[seq] + each - q_start[seq]
    opens = r % page == 0
    free = torch.argsort((refs > 0).to(torch.int8), stable=True).to(torch.int32)
    new = free[(torch.cumsum(opens, 0) - 1).clamp_min(0)]
    table[seq[opens], (r // page)[opens]] = new[opens]
    refs[new[opens].long()] = 1
    rows += s["n_new"]
    return table[seq, r // page].long() * page + r % page


# ---- one pass ----------------------------------------------------------------------------

def _handle(s):
    """The pool object that a program keeps next to its buffers."""
    from ds4cuda_amd import pages
    if "pool" not in s:
        s["pool"] = pages.PagePool(s["codes"], s["sexp"], s["tail"], s["refs"], s["table"], s["rows"],
                                   s["case"]["page"])
    return s["pool"]


def _attend_tree(s):
    if not own:
        return _attend(s)
    return _handle(s).attend_tree(s["q"], s["parents"], seqs=s["seqs"], q_start=s["q_start"], window=s["case"]["window"],
                                  n_first=s["case"]["first"], sinks=s["sinks"])


def _sample_tokens(s):
    f = s["filters"]
    if not own:
        return _sample(s["logits"], **f)
    from ds4cuda_amd import ops
    return ops.sample_tokens(s["logits"], f["u"], temperature=f["temperature"], top_k=f["top_k"], top_p=f["top_p"],
                             min_p=f["min_p"])


def _accept(s, targets):
    if own:
        return _handle(s).accept(s["seqs"], s["q_start"], s["parents"], s["tokens"], targets)
    path, length, following = _walk(s, targets)
    _keep(s, path, length)
    return path, length, following


def run(s):
    kind = s["case"]["kind"]
    if kind == "tree":
        return _attend_tree(s)
    if kind == "sample":
        return dict(zip(("tokens", "probs"), _sample_tokens(s)))
    # the step's tables, as the scheduler keeps them
    s["refs"].copy_(s["refs_in"])
    s["rows"].copy_(s["rows_in"])
    out, targets = {}, s["targets"]
    if kind == "step":
        s["table"].copy_(s["table_in"])
        if own:
            dst = _handle(s).extend(s["seqs"], s["n_new"], s["n_nodes"])
            _handle(s).append(s["kv"], dst)
        else:
            dst = _extend(s)
            s["codes"][0, dst], s["sexp"][0, dst], s["tail"][0, dst] = _quantize(s["kv"])
        out["attn"] = _attend_tree(s)
        targets, probs = _sample_tokens(s)
        out.update(tokens=targets, probs=probs)
    path, length, following = _accept(s, targets)
    return {**out, "path": path, "length": length, "next": following, "table": s["table"], "refs": s["refs"],
            "rows": s["rows"], "codes": s["codes"].view(torch.float8_e4m3fn), "sexp": s["sexp"], "tail": s["tail"]}


# ---- the definition in 64 bits --------------------------------------------------------------

def _row_bits(codes, sexp, tail):
    """Cache rows in fp64, decoded from the bits of their format."""
    c = codes.to(torch.int64)
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e == 0, m / 512.0, (1.0 + m / 8.0) * torch.pow(2.0, (e - 7).double()))
    v = torch.where(c >= 128, -v, v) * torch.pow(2.0, sexp[:, :7].double()).repeat_interleave(64, -1)
    return torch.cat([v.half().double(), tail.double()], -1)


def _attend_exact(case, q, sequence, sinks):
    """sequence(i): the rows of sequence i, cached and drafted, in fp64."""
    out, a, window, first = torch.empty_like(q), 0, case["window"], case["first"]
    for i, (base, parents, _) in enumerate(zip(*_trees(case))):
        kv, depth = sequence(i), _depths(parents)
        for v in range(len(parents)):
            line, j = [], v   # the positions and rows of the node and its ancestors
            while j >= 0:
                line.append((base + depth[j], base + j))
                j = parents[j]
            p = base + depth[v]
            lo = 0 if window == 0 else min(base, max(0, p - window + 1))
            rows = list(range(min(first, lo))) + list(range(lo, base))
            rows += [r for at, r in line if window == 0 or at > p - window or at < first]
            k = kv[torch.tensor(rows, device=DEV)]
            w = q[a + v] @ k.T / math.sqrt(DIM)
            if sinks is not None:
                w = torch.cat([w, sinks[:, None]], -1)
            out[a + v] = torch.softmax(w, -1)[:, :len(rows)] @ k
        a += len(parents)
    return out


def _probs_exact(logits, f):
    """The probability of each row's token."""
    probs = []
    for i in range(logits.shape[0]):
        t, k, p, m, u = (f[n][i].item() for n in ("temperature", "top_k", "top_p", "min_p", "u"))
        if t == 0.0:
            probs.append(1.0)
            continue
        x = logits[i].double()
        order = torch.argsort(x, descending=True, stable=True)
        order = order[:k] if k > 0 else order
        w = torch.exp((x[order] - x[order[0]]) / t)
        if p < 1.0:
            before = torch.cumsum(w, 0) - w
            order = order[:max(1, int((before < p * w.sum()).sum()))]
            w = w[:order.numel()]
        order = order[:max(1, int((w >= m).sum()))]
        index = torch.sort(order)[0]
        w = torch.exp((x[index] - x[order[0]]) / t)
        run_sum = torch.cumsum(w, 0)
        at = min(int(torch.searchsorted(run_sum, u * w.sum(), right=True)), w.numel() - 1)
        probs.append(float(w[at] / w.sum()))
    return torch.tensor(probs, dtype=torch.float64, device=DEV)


def exact(case, seed):
    kind = case["kind"]
    if kind == "accept":
        return None
    s = prepare(case, seed)
    if kind == "sample":
        return {"tokens": None, "probs": _probs_exact(s["logits"], s["filters"])}
    page, (cached, parents, _) = case["page"], _trees(case)
    table = s["table_in"].long()

    def held(i, r):
        at = torch.arange(r, device=DEV)
        at = table[i, at // page] * page + at % page
        return _row_bits(s["codes"][0, at], s["sexp"][0, at], s["tail"][0, at])

    def drafted(i):
        x = s["kv"][sum(s["sizes"][:i]):sum(s["sizes"][:i + 1])].double()
        b = x[:, :NOPE].reshape(-1, 7, 64)
        # the smallest power of two that brings the block's largest value to 448 or less
        e = torch.ceil(torch.log2(b.abs().amax(-1).clamp_min(1e-4) / 448.0))
        c = (b * torch.pow(2.0, -e)[..., None]).float().to(torch.float8_e4m3fn).double()
        v = (c * torch.pow(2.0, e)[..., None]).reshape(-1, NOPE).half().double()
        return torch.cat([held(i, cached[i]), torch.cat([v, x[:, NOPE:].half().double()], -1)])

    sinks = s["sinks"].double() if s["sinks"] is not None else None
    if kind == "tree":
        return _attend_exact(case, s["q"].double(), lambda i: held(i, cached[i] + len(parents[i])), sinks)
    return {"attn": _attend_exact(case, s["q"].double(), drafted, sinks), "tokens": None,
            "probs": _probs_exact(s["logits"], s["filters"]), "path": None, "length": None, "next": None, "table": None,
            "refs": None, "rows": None, "codes": None, "sexp": None, "tail": None}
