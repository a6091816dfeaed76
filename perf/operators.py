"""Operators of a paged FP8 KV cache: its pages, and the attention that reads them.

One latent KV head of 512 dims per cache row (448 FP8 E4M3 dims with a power-of-two
scale per 64, 64 RoPE dims in f16), `heads` query heads over it (64 in the model, fewer
on a tensor-parallel slice). A pool holds pages of `page` rows for all layers; a table
names each sequence's pages, `refs` says how many sequences hold a page.

Kinds:

  prompt  attention of prompt tokens over the pages of their sequences, packed over a
          ragged batch: a sliding window and a few first tokens that stay visible
  decode  attention of one new token of each sequence, lengths on the device
  fork    sequences forked (pages shared, a partly filled last page copied, or every
          page copied), extended and freed again: one step of parallel sampling
  compact live pages moved to the front of the pool
  trial   the operators together: fork, extend, append, attend, free

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
DEV = "cuda"


# ---- the cases ---------------------------------------------------------------------------

def listed():
    return [
        # The last odd tokens of one prompt over a short history: launches and latency count.
        {"name": "prompt_tail", "kind": "prompt", "seqs": 1, "cached": 700, "new": 33, "heads": 64, "window": 128,
         "first": 4, "page": 64, "type": "bf16", "sinks": True},
        # A batch of ragged prompts in the model's 128-token window.
        {"name": "prompt_batch", "kind": "prompt", "seqs": 6, "cached": 900, "new": 640, "heads": 64, "window": 128,
         "first": 4, "page": 64, "type": "bf16", "sinks": True},
        # A long prompt's chunk in a wide window: matrix products count.
        {"name": "prompt_long", "kind": "prompt", "seqs": 1, "cached": 4096, "new": 4096, "heads": 64, "window": 1024,
         "first": 64, "page": 256, "type": "bf16", "sinks": True},
        # A tensor-parallel slice of the heads with fp32 queries and outputs, as the Q producer hands them over.
        {"name": "prompt_slice_fp32", "kind": "prompt", "seqs": 3, "cached": 300, "new": 501, "heads": 16,
         "window": 500, "first": 1, "page": 16, "type": "fp32", "sinks": False},
        # One sequence of a few thousand rows, all of them visible: latency.
        {"name": "decode_one", "kind": "decode", "seqs": 1, "cached": 4000, "heads": 64, "window": 0, "first": 0,
         "page": 256, "type": "bf16", "sinks": True},
        # A batch of ragged lengths up to 32K.
        {"name": "decode_batch", "kind": "decode", "seqs": 16, "cached": 32768, "heads": 64, "window": 0, "first": 0,
         "page": 256, "type": "bf16", "sinks": True},
        # Many sequences in a sliding window: little is read of each.
        {"name": "decode_window", "kind": "decode", "seqs": 128, "cached": 4096, "heads": 64, "window": 128,
         "first": 4, "page": 64, "type": "bf16", "sinks": True},
        # A few very long sequences, a slice of the heads, fp32.
        {"name": "decode_long_fp32", "kind": "decode", "seqs": 4, "cached": 131072, "heads": 16, "window": 0,
         "first": 0, "page": 64, "type": "fp32", "sinks": False},
        # Parallel sampling of one layer's cache: little to copy, launches count.
        {"name": "fork_small", "kind": "fork", "parents": 2, "children": 3, "rows": 150, "new": 1, "layers": 1,
         "page": 16, "deep": False},
        # Prompts copied whole for sequences that will go separate ways, over the model's 43 layers.
        {"name": "fork_deep", "kind": "fork", "parents": 4, "children": 1, "rows": 7001, "new": 2, "layers": 43,
         "page": 256, "deep": True},
        # A scattered pool of all 43 layers made dense.
        {"name": "compact_pool", "kind": "compact", "seqs": 40, "rows": 700, "layers": 43, "page": 64},
        # One step of a tree of samples: the operators as they are used together.
        {"name": "trial_tree", "kind": "trial", "parents": 4, "children": 4, "rows": 2500, "new": 3, "heads": 64,
         "window": 1000, "first": 16, "page": 64, "type": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "decode", "decode", "fork", "compact", "trial"])
    page = rng.choice([16, 32, 64, 128, 256])
    attn = {"heads": rng.choice([8, 16, 32, 64, 64, 128]), "page": page, "type": rng.choice(["bf16", "bf16", "fp32"])}
    if kind == "prompt":
        seqs = rng.choice([1, 1, 2, 5, 11])
        new = _log_int(rng, 1, 2000 // seqs)
        # all rows visible only where the plain form's gathered keys stay small
        window = rng.choice([0, 1]) * _log_int(rng, 1, 1500)
        cached = _log_int(rng, 1, 6000) if window else _log_int(rng, 1, 900)
        return {"kind": kind, "seqs": seqs, "cached": cached, "new": new, "window": window,
                "first": rng.choice([0, 1, 4, 37, 128]), "sinks": rng.random() < 0.5, **attn}
    if kind == "decode":
        seqs = _log_int(rng, 1, 200)
        return {"kind": kind, "seqs": seqs, "cached": _log_int(rng, 1, max(64, min(100000, 260000 // seqs))),
                "window": rng.choice([0, 0, 1]) * _log_int(rng, 1, 5000), "first": rng.choice([0, 1, 4, 100]),
                "sinks": rng.random() < 0.5, **attn}
    if kind == "fork":
        deep, layers = rng.random() < 0.4, rng.choice([1, 3, 43])
        parents, children = rng.choice([1, 2, 7]), rng.choice([1, 2, 5])
        rows = _log_int(rng, 1, 150000 // (parents * (children + 1) * (layers if layers > 3 else 3)) + 2)
        return {"kind": kind, "parents": parents, "children": children, "rows": rows, "new": rng.choice([0, 1, 5, 70]),
                "layers": layers, "page": page, "deep": deep}
    if kind == "compact":
        seqs = rng.choice([3, 17, 60])
        return {"kind": kind, "seqs": seqs, "rows": _log_int(rng, 5, 28000 // seqs), "layers": rng.choice([1, 8, 43]),
                "page": page}
    return {"kind": kind, "parents": rng.choice([1, 3, 6]), "children": rng.choice([1, 2, 5]),
            "rows": _log_int(rng, 1, 5000), "new": rng.choice([1, 2, 9]), "window": rng.choice([0, 64, 999]),
            "first": rng.choice([0, 5, 64]), **attn}


def _lengths(case, n, longest, shortest=1):
    """n ragged lengths that the case alone fixes, `longest` among them."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")) + str(longest))
    some = [_log_int(rng, max(shortest, longest // 16, 1), max(shortest, longest, 1)) for _ in range(n)]
    some[rng.randrange(n)] = longest
    return some


def _pages(rows, page):
    return -(-rows // page)


def _visible(pos, window, first):
    """Rows that a query at position pos sees."""
    n = pos + 1
    return n if window == 0 or n <= window else window + min(first, n - window)


def _shape(case):
    """Per sequence: rows in the cache and how many of them are the queries' own."""
    if case["kind"] == "prompt":
        new = _lengths(case, case["seqs"], case["new"])
        cached = [c - 1 for c in _lengths(case, case["seqs"], case["cached"] + 1)]
        return [c + n for c, n in zip(cached, new)], new
    if case["kind"] == "decode":
        return _lengths(case, case["seqs"], case["cached"]), [1] * case["seqs"]
    rows = _lengths(case, case["parents"], case["rows"])
    kids = [rows[i % case["parents"]] for i in range(case["parents"] * case["children"])]
    return [r + case["new"] for r in kids], [case["new"]] * len(kids)


def _attention_work(case, rows, new):
    heads, window, first = case["heads"], case["window"], case["first"]
    item = 4 if case["type"] == "fp32" else 2
    pairs, read = 0, 0
    for r, n in zip(rows, new):
        pairs += sum(_visible(p, window, first) for p in range(r - n, r))
        lo = 0 if window == 0 else max(0, r - n - window + 1)
        read += (r - lo) + min(first, lo)
    return {"bytes": read * ROW_BYTES + 2 * sum(new) * heads * DIM * item, "flops": 4 * DIM * heads * pairs}


def work(case):
    kind = case["kind"]
    if kind in ("prompt", "decode"):
        return _attention_work(case, *_shape(case))
    page = case["page"]
    if kind == "compact":
        lens = _lengths(case, case["seqs"], case["rows"])
        _, live, n_pages = _scattered(case, lens)
        moved = sum(p >= len(live) for p in live)
        return {"bytes": 2 * moved * page * ROW_BYTES * case["layers"] + 8 * n_pages, "flops": 0}
    lens = _lengths(case, case["parents"], case["rows"])
    copied = sum(r if case.get("deep") else r % page for r in lens) * case["children"]
    held = sum(_pages(r + case["new"], page) for r in lens) * case["children"]
    moved = 2 * copied * ROW_BYTES * case.get("layers", 1) + 4 * 4 * held
    if kind == "fork":
        return {"bytes": moved, "flops": 0}
    rows, new = _shape(case)
    w = _attention_work(case, rows, new)
    return {"bytes": w["bytes"] + moved + sum(new) * (4 * DIM + ROW_BYTES), "flops": w["flops"]}


# ---- inputs ------------------------------------------------------------------------------

def _gen(seed, k):
    return torch.Generator(DEV).manual_seed((int(seed) * 1000003 + 7919 * k) % (1 << 62))


def _quantized(gen, n):
    """n cache rows ~N(0,1), one in a hundred eight times as large: the cache's three arrays."""
    codes = torch.empty((n, NOPE), dtype=torch.uint8, device=DEV)
    sexp = torch.zeros((n, 8), dtype=torch.int8, device=DEV)
    tail = torch.empty((n, ROT), dtype=torch.float16, device=DEV)
    for a in range(0, n, 1 << 18):
        b = min(n, a + (1 << 18))
        x = torch.randn((b - a, DIM), generator=gen, device=DEV)
        x *= torch.where(torch.rand((b - a, 1), generator=gen, device=DEV) < 0.01, 8.0, 1.0)
        blocks = x[:, :NOPE].reshape(b - a, 7, 64)
        e = torch.ceil(torch.log2(blocks.abs().amax(-1).clamp_min(1e-4) / 448.0))
        codes[a:b] = (blocks * torch.exp2(-e)[..., None]).reshape(b - a, NOPE).to(torch.float8_e4m3fn).view(torch.uint8)
        sexp[a:b, :7] = e.to(torch.int8)
        tail[a:b] = x[:, NOPE:].half()
    return codes, sexp, tail


def _anything(gen, layers, n):
    """Rows of whatever the layers hold: finite codes, exponents and tails."""
    def ints(shape, lo, hi, dtype):
        return torch.randint(lo, hi, shape, generator=gen, dtype=dtype, device=DEV)
    codes = ints((layers, n, NOPE), 0, 0x7F, torch.uint8)
    sexp = ints((layers, n, 8), -9, 3, torch.int8)
    tail = ints((layers, n, ROT), 0, 0x7C00, torch.int16)
    return codes, sexp, tail.view(torch.float16)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pool(lens, slots, page, extra, stride, order):
    """Tables of `slots` sequences of which the first hold `lens` rows, on pages in `order`."""
    table, refs, used = [[-1] * stride for _ in range(slots)], [0] * (sum(_pages(r, page) for r in lens) + extra), 0
    for s, r in enumerate(lens):
        for i in range(_pages(r, page)):
            table[s][i] = order[used]
            refs[order[used]] = 1
            used += 1
    return _i32(table), _i32(refs), _i32(list(lens) + [0] * (slots - len(lens)))


def _scattered(case, lens):
    """A pool after sequences came and went: every other page or so is free."""
    n = sum(_pages(r, case["page"]) for r in lens)
    rng = random.Random(n * 31 + case["page"])
    live = sorted(rng.sample(range(2 * n), n))
    order = live[:]
    rng.shuffle(order)
    return order, live, 2 * n


def prepare(case, seed):
    kind, page = case["kind"], case["page"]
    s = {"case": case}
    if kind == "compact":
        lens = _lengths(case, case["seqs"], case["rows"])
        order, _, n_pages = _scattered(case, lens)
        table, refs, rows = _pool(lens, len(lens), page, n_pages - len(order), _pages(max(lens), page), order)
        s.update(table=torch.empty_like(table), refs=torch.empty_like(refs), rows=rows, table_in=table, refs_in=refs)
        s["codes"], s["sexp"], s["tail"] = _anything(_gen(seed, 0), case["layers"], n_pages * page)
        return s
    if kind in ("prompt", "decode"):
        lens, new = _shape(case)
        n_pages, slots, extra, layers = sum(_pages(r, page) for r in lens) + 3, len(lens), 3, 1
        stride = _pages(max(lens), page)
    else:
        lens = _lengths(case, case["parents"], case["rows"])
        kids = case["parents"] * case["children"]
        slots, layers = case["parents"] + kids, case.get("layers", 1)
        stride = _pages(max(lens) + case["new"], page)
        extra = kids * (stride if case.get("deep") else _pages(case["new"], page) + 1) + 2
        n_pages = sum(_pages(r, page) for r in lens) + extra
        s["parents"] = _i32([i % case["parents"] for i in range(kids)])
        s["children"] = _i32([case["parents"] + i for i in range(kids)])
        s["n_new"] = _i32([case["new"]] * kids)
        new = [case["new"]] * kids
    rng = random.Random(seed)
    order = list(range(n_pages))
    rng.shuffle(order)
    s["table"], s["refs"], s["rows"] = _pool(lens, slots, page, extra, stride, order)
    if kind == "fork":
        s["codes"], s["sexp"], s["tail"] = _anything(_gen(seed, 0), layers, n_pages * page)
        return s
    s["codes"], s["sexp"], s["tail"] = (t[None] for t in _quantized(_gen(seed, 0), n_pages * page))
    s["q"] = torch.randn((sum(new), case["heads"], DIM), generator=_gen(seed, 1), device=DEV).to(TYPES[case["type"]])
    if case.get("sinks"):
        s["sinks"] = torch.randn((case["heads"],), generator=_gen(seed, 2), device=DEV)
    if kind != "decode":
        s["q_start"] = _i32([sum(new[:i]) for i in range(len(new) + 1)])
    if kind == "trial":
        s["kv"] = torch.randn((sum(new), DIM), generator=_gen(seed, 3), device=DEV)
    return s


# ---- the operators in plain torch ----------------------------------------------------------

def _values(codes, sexp, tail):
    """Rows as fp32: f16(code * 2^e) and the f16 tail."""
    x = codes.view(torch.float8_e4m3fn).float().unflatten(-1, (7, 64))
    x = (x * torch.exp2(sexp[..., :7].float())[..., None]).half().float()
    return torch.cat([x.flatten(-2), tail.float()], -1)


def _attend(s, seq_rows, table):
    """Attention of the packed queries over the rows that their positions see."""
    case, q = s["case"], s["q"].float()
    window, first, page = case["window"], case["first"], case["page"]
    n_q, dev = q.shape[0], q.device
    each = torch.arange(n_q, device=dev)
    if "q_start" in s:
        seq = (each[:, None] >= s["q_start"][None, 1:]).sum(1)
        pos = seq_rows[seq] - s["q_start"][seq + 1] + each
    else:
        seq, pos = each, seq_rows - 1
    longest = max(_shape(case)[0])
    cols = torch.arange(longest if window == 0 else min(longest, window + first), device=dev)[None]
    if window == 0 or longest <= window + first:
        r = cols.expand(n_q, -1)
        sees = (r <= pos[:, None]) & ((r < first) | (r > pos[:, None] - window) if window else (r >= 0))
    else:
        r = torch.where(cols < first, cols, pos[:, None] - window + 1 + cols - first)
        sees = (r >= 0) & (r <= pos[:, None]) & ((cols < first) | (r >= first))
    r = torch.where(sees, r, 0)
    at = table[seq[:, None], r // page].long() * page + r % page
    at = torch.where(sees, at, 0)
    k = _values(s["codes"][0], s["sexp"][0], s["tail"][0])[at]      # [n_q, cols, 512]
    score = (q @ k.transpose(1, 2)) * SCALE
    score = torch.where(sees[:, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    if "sinks" in s:
        sink = s["sinks"][None, :, None]
        top = torch.maximum(top, sink)
    p = torch.exp(score - top)
    den = p.sum(-1, keepdim=True)
    if "sinks" in s:
        den = den + torch.exp(sink - top)
    return ((p @ k) / den).to(s["q"].dtype)


def _lowest_free(refs):
    return torch.argsort((refs > 0).to(torch.int8), stable=True).to(torch.int32)


def _copy_rows(s, src, dst):
    for name in ("codes", "sexp", "tail"):
        s[name][:, dst] = s[name][:, src]


def _fork(s, deep):
    table, refs, rows, page = s["table"], s["refs"], s["rows"], s["case"]["page"]
    parents, children = s["parents"].long(), s["children"].long()
    held = rows[parents].long()
    cols = torch.arange(table.shape[1], device=table.device)[None]
    holds = cols * page < held[:, None]
    fresh = holds if deep else holds & ((cols + 1) * page > held[:, None])
    named = table[parents]
    new = _lowest_free(refs)[(torch.cumsum(fresh.flatten(), 0) - 1).clamp_min(0)].view_as(named)
    table[children] = torch.where(fresh, new, torch.where(holds, named, table[children]))
    refs.index_add_(0, torch.where(holds & ~fresh, named, 0).flatten().long(), (holds & ~fresh).flatten().int())
    refs[new[fresh].long()] = 1
    rows[children] = rows[parents]
    r = torch.arange(page, device=table.device)
    copied = fresh[..., None] & (cols[..., None] * page + r < held[:, None, None])
    _copy_rows(s, (named.long()[..., None] * page + r)[copied], (new.long()[..., None] * page + r)[copied])


def _extend(s):
    table, refs, rows, page = s["table"], s["refs"], s["rows"], s["case"]["page"]
    n_new, seqs = s["case"]["new"], s["children"].long()
    r = (rows[seqs].long()[:, None] + torch.arange(n_new, device=table.device)).flatten()
    seq = seqs.repeat_interleave(n_new)
    opens = r % page == 0
    new = _lowest_free(refs)[(torch.cumsum(opens, 0) - 1).clamp_min(0)]
    table[seq[opens], (r // page)[opens]] = new[opens]
    refs[new[opens].long()] = 1
    rows[seqs] += n_new
    return table[seq, r // page].long() * page + r % page


def _free(s):
    table, refs, rows, page = s["table"], s["refs"], s["rows"], s["case"]["page"]
    seqs = s["children"].long()
    holds = torch.arange(table.shape[1], device=table.device)[None] * page < rows[seqs].long()[:, None]
    refs.index_add_(0, torch.where(holds, table[seqs], 0).flatten().long(), -holds.flatten().int())
    rows[seqs] = 0


def _append(s, dst):
    x = s["kv"]
    blocks = x[:, :NOPE].unflatten(-1, (7, 64))
    e = torch.ceil(torch.log2(blocks.abs().amax(-1).clamp_min(1e-4) / 448.0))
    s["codes"][0, dst] = (blocks * torch.exp2(-e)[..., None]).flatten(1).to(torch.float8_e4m3fn).view(torch.uint8)
    s["sexp"][0, dst] = torch.nn.functional.pad(e.to(torch.int8), (0, 1))
    s["tail"][0, dst] = x[:, NOPE:].half()


def _compact(s):
    table, refs, page = s["table"], s["refs"], s["case"]["page"]
    live, at = refs > 0, torch.arange(refs.numel(), device=refs.device)
    n_live = live.sum().to(torch.int32)
    src, dst = at[live & (at >= n_live)], at[~live & (at < n_live)]
    now = at.to(torch.int32)
    now[src] = dst.to(torch.int32)
    holds = torch.arange(table.shape[1], device=table.device)[None] * page < s["rows"].long()[:, None]
    table.copy_(torch.where(holds, now[table.clamp_min(0).long()], table))
    refs[dst] = refs[src]
    refs[src] = 0
    for name in ("codes", "sexp", "tail"):
        paged = s[name].unflatten(1, (-1, page))
        paged[:, dst] = paged[:, src]
    return n_live


# ---- one pass ----------------------------------------------------------------------------

def _handle(s):
    """The pool object that a program keeps next to its buffers."""
    from ds4cuda_amd import pages
    if "pool" not in s:
        s["pool"] = pages.PagePool(s["codes"], s["sexp"], s["tail"], s["refs"], s["table"], s["rows"],
                                   s["case"]["page"])
    return s["pool"]


def _tables(s):
    return {k: s[k] for k in ("table", "refs", "rows")}


def _rows_out(s):
    """The pool's rows as the values they stand for."""
    return {"codes": s["codes"].view(torch.float8_e4m3fn), "sexp": s["sexp"], "tail": s["tail"]}


def run(s):
    case = s["case"]
    kind = case["kind"]
    if kind in ("prompt", "decode"):
        if own:
            return _handle(s).attend(s["q"], q_start=s.get("q_start"), window=case["window"], n_first=case["first"],
                                     sinks=s.get("sinks"))
        return _attend(s, s["rows"].long(), s["table"])
    if kind == "compact":
        # the step's tables, as the scheduler keeps them
        s["table"].copy_(s["table_in"])
        s["refs"].copy_(s["refs_in"])
        n_live = _handle(s).compact() if own else _compact(s)
        return {"n_live": n_live, **_tables(s), **_rows_out(s)}
    n_dst = case["new"] * s["children"].numel()
    if own:
        pool = _handle(s)
        pool.fork(s["parents"], s["children"], deep=case.get("deep", False))
        dst = pool.extend(s["children"], s["n_new"], n_dst)
    else:
        _fork(s, case.get("deep", False))
        dst = _extend(s)
    out = {"dst": dst}
    if kind == "trial":
        if own:
            pool.append(s["kv"], dst)
            out["attn"] = pool.attend(s["q"], seqs=s["children"], q_start=s["q_start"], window=case["window"],
                                      n_first=case["first"])
        else:
            _append(s, dst)
            kids = s["children"].long()
            out["attn"] = _attend(s, s["rows"][kids].long(), s["table"][kids])
    if own:
        pool.free(s["children"])
    else:
        _free(s)
    return {**out, **_tables(s), **_rows_out(s)}


# ---- the definition in 64 bits --------------------------------------------------------------

def _attend_exact(q, kv_of, rows, new, window, first, sinks):
    """q [n, heads, 512] fp64 packed; kv_of(i): sequence i's rows in fp64, in order."""
    out, a = torch.empty_like(q), 0
    for i, (r, n) in enumerate(zip(rows, new)):
        kv = kv_of(i)
        for b in range(0, n, 256):
            m = min(256, n - b)
            x = q[a + b:a + b + m]
            p = torch.arange(r - n + b, r - n + b + m, device=q.device)[:, None]
            lo = 0 if window == 0 else max(0, r - n + b - window + 1)
            names = torch.cat([torch.arange(min(first, lo), device=q.device), torch.arange(lo, r - n + b + m, device=q.device)])
            k = kv[names]
            seen = names[None] <= p
            if window:
                seen &= (names[None] > p - window) | (names[None] < first)
            w = torch.einsum("qhd,kd->qhk", x, k) / math.sqrt(DIM)
            w = w.masked_fill(~seen[:, None], -math.inf)
            if sinks is not None:
                w = torch.cat([w, sinks.view(1, -1, 1).expand(m, -1, 1)], -1)
            w = torch.softmax(w, -1)[..., :names.numel()]
            out[a + b:a + b + m] = torch.einsum("qhk,kd->qhd", w, k)
        a += n
    return out


def _rows_exact(s, names):
    """Cache rows `names` in fp64, decoded from the bits of their format."""
    c = s["codes"][0, names].to(torch.int64)
    e, m = (c >> 3) & 15, c & 7
    v = torch.where(e == 0, m.double() / 512.0, (1.0 + m.double() / 8.0) * torch.pow(2.0, (e - 7).double()))
    v = torch.where(c >= 128, -v, v)
    v = v * torch.pow(2.0, s["sexp"][0, names, :7].double()).repeat_interleave(64, -1)
    return torch.cat([v.half().double(), s["tail"][0, names].double()], -1)


def exact(case, seed):
    kind = case["kind"]
    if kind in ("fork", "compact"):
        return None
    s = prepare(case, seed)
    page, (rows, new) = case["page"], _shape(case)
    sinks = s["sinks"].double() if "sinks" in s else None
    table = s["table"].long()

    def sequence(slot, r):
        at = torch.arange(r, device=DEV)
        return _rows_exact(s, table[slot, at // page] * page + at % page)

    if kind != "trial":
        return _attend_exact(s["q"].double(), lambda i: sequence(i, rows[i]), rows, new, case["window"], case["first"],
                             sinks)
    n = case["new"]

    def child(i):
        x = s["kv"][i * n:(i + 1) * n].double()
        b = x[:, :NOPE].reshape(n, 7, 64)
        # the smallest power of two that brings the block's largest value to 448 or less
        e = torch.ceil(torch.log2(b.abs().amax(-1).clamp_min(1e-4) / 448.0))
        c = (b * torch.pow(2.0, -e)[..., None]).float().to(torch.float8_e4m3fn).double()
        v = (c * torch.pow(2.0, e)[..., None]).reshape(n, NOPE).half().double()
        return torch.cat([sequence(i % case["parents"], rows[i] - n), torch.cat([v, x[:, NOPE:].half().double()], -1)])

    attn = _attend_exact(s["q"].double(), child, rows, new, case["window"], case["first"], sinks)
    return {"dst": None, "attn": attn, "table": None, "refs": None, "rows": None, "codes": None, "sexp": None, "tail": None}
