"""Attention over pages in a sliding window with first rows kept: against the
definition in 64 bits, where masks, lengths, pages and values can go wrong."""
import random

import pytest
import torch

from paged_check import attend_64, bound_of, quantized_rows, row_values

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


class Batch:
    """Sequences of `rows` rows on shuffled pages; the rows that nothing may read hold
    NaN and infinities."""

    def __init__(self, gpu, rows, page, seed, entries=None, spare=3):
        from ds4cuda_amd import ops
        self.gpu, self.rows, self.page = gpu, rows, page
        need = [-(-r // page) for r in rows]
        self.n_pages = sum(need) + spare
        order = list(range(self.n_pages))
        random.Random(seed).shuffle(order)
        entries = entries or max(need + [1])
        table, used = [], 0
        for n in need:
            table.append(order[used:used + n] + [-1] * (entries - n))
            used += n
        self.table, self.seq_rows = i32(table, gpu), i32(rows, gpu)
        n = self.n_pages * page
        codes, sexp, tail = quantized_rows(n, seed, gpu)
        live = torch.zeros(n, dtype=torch.bool, device=gpu)
        for s in range(len(rows)):
            live[self.at(s)] = True
        codes[~live] = 0x7F
        sexp[~live] = 60
        tail[~live] = float("inf")
        self.cache = ops.Fp8KVCache(codes, sexp, tail)

    def at(self, s):
        r = torch.arange(self.rows[s], device=self.gpu)
        return self.table[s].long()[r // self.page] * self.page + r % self.page

    def values(self, s):
        a = self.at(s)
        return row_values(self.cache.codes[a], self.cache.sexp[a], self.cache.tail[a])


def check(b, q, out, new, window, first, sinks, seqs=None):
    """Every query's output against 64 bits; new[i] queries of entry i."""
    f32, a, off, norm = q.dtype == torch.float32, 0, 0.0, 0.0
    for i, n in enumerate(new):
        s = i if seqs is None else seqs[i]
        if n == 0:
            continue
        pos = [b.rows[s] - n + k for k in range(n)]
        ref, size, err = attend_64(q[a:a + n], b.values(s), pos, window, first, sinks)
        d = (out[a:a + n].double() - ref).abs()
        assert torch.isfinite(out[a:a + n]).all(), (i, s)
        worst = (d - bound_of(ref, size, err, f32)).amax()
        assert worst <= 0, (i, s, float(worst), float(d.amax()))
        off, norm = off + float((d * d).sum()), norm + float((ref * ref).sum())
        a += n
    # taken together: roundings of a result (bf16 2^-8 at most each, half of that and less on
    # average), or for fp32 of scores and parts of 2^-22, with room for ten times as much
    if norm:
        assert (off / norm) ** 0.5 <= (1e-5 if f32 else 4e-3)


def queries(gpu, n, heads, typ, seed):
    g = torch.Generator(gpu).manual_seed(seed)
    return torch.randn((n, heads, 512), generator=g, device=gpu).to(TYPES[typ])


def run(b, q, new, window=0, first=0, sinks=None, seqs=None, **kw):
    from ds4cuda_amd import ops
    start = [sum(new[:i]) for i in range(len(new) + 1)]
    return ops.flash_attn_window_fp8(q, b.cache, b.table, b.seq_rows, page_rows=b.page, window=window, n_first=first,
                                     sinks=sinks, q_start=i32(start, b.gpu),
                                     seq_ids=None if seqs is None else i32(seqs, b.gpu), **kw)


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
@pytest.mark.parametrize("heads", [8, 16, 32, 64, 128])
@pytest.mark.parametrize("rows,page,window,first", [
    ([1], 16, 0, 0), ([0, 1, 2, 31, 32, 33, 64, 65], 16, 0, 0), ([700, 3, 129], 64, 128, 4), ([513], 1, 100, 33),
    ([1500, 40], 256, 1, 0), ([300, 299], 32, 7, 300), ([200], 8, 1000, 1)])
def test_one_token_each(gpu, rows, page, window, first, heads, typ):
    from ds4cuda_amd import ops
    b = Batch(gpu, rows, page, heads + page)
    q = queries(gpu, len(rows), heads, typ, 1)
    sinks = torch.randn(heads, device=gpu) if heads != 16 else None
    out = ops.flash_attn_window_fp8(q, b.cache, b.table, b.seq_rows, page_rows=page, window=window, n_first=first, sinks=sinks)
    for s, r in enumerate(rows):
        if r == 0:
            assert (out[s] == 0).all()
    check(b, q, out, [int(r > 0) for r in rows], window, first, sinks) if 0 not in rows else \
        check(b, q[1:], out[1:], [1] * (len(rows) - 1), window, first, sinks, seqs=list(range(1, len(rows))))


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
@pytest.mark.parametrize("heads", [8, 64, 128])
@pytest.mark.parametrize("rows,new,page,window,first", [
    ([1, 2, 3], [1, 2, 3], 16, 0, 0), ([70], [70], 64, 0, 0), ([301], [37], 32, 0, 5), ([400, 90, 1], [130, 0, 1], 128, 33, 2),
    ([260, 131], [9, 100], 4, 64, 64), ([200], [65], 16, 1, 0), ([150], [150], 64, 40, 200), ([96, 64], [32, 64], 32, 32, 32)])
def test_prompts(gpu, rows, new, page, window, first, heads, typ):
    b = Batch(gpu, rows, page, heads + sum(new))
    q = queries(gpu, sum(new), heads, typ, 2)
    sinks = torch.randn(heads, device=gpu) if window != 33 else None
    check(b, q, run(b, q, new, window, first, sinks), new, window, first, sinks)


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
def test_long_and_short_sequences_together(gpu, typ):
    """Lines of tiles that workgroups share: one long sequence among short ones, heads of
    a slice, and a batch whose sequences are all cut."""
    from ds4cuda_amd import ops
    for rows, heads in (([20000, 5, 900, 33, 1], 64), ([9000, 8000], 16), ([3000] * 7, 128)):
        b = Batch(gpu, rows, 256, len(rows))
        q = queries(gpu, len(rows), heads, typ, 3)
        sinks = torch.randn(heads, device=gpu)
        out = ops.flash_attn_window_fp8(q, b.cache, b.table, b.seq_rows, page_rows=256, sinks=sinks)
        check(b, q, out, [1] * len(rows), 0, 0, sinks)
        again = ops.flash_attn_window_fp8(q, b.cache, b.table, b.seq_rows, page_rows=256, sinks=sinks)
        assert torch.equal(out, again)
    b = Batch(gpu, [6000, 50], 64, 5)
    q = queries(gpu, 310, 64, typ, 4)
    check(b, q, run(b, q, [300, 10], 2000, 64), [300, 10], 2000, 64, None)


def test_many_short_sequences(gpu):
    """Thousands of sequences, most of them empty; the window never cut."""
    rows = [(i * 37) % 90 if i % 3 else 0 for i in range(4096)]
    b = Batch(gpu, rows, 16, 6)
    q = queries(gpu, 4096, 8, "bf16", 5)
    from ds4cuda_amd import ops
    out = ops.flash_attn_window_fp8(q, b.cache, b.table, b.seq_rows, page_rows=16, window=20, n_first=3)
    some = [i for i in range(4096) if rows[i]]
    check(b, q[some[::40]], out[some[::40]], [1] * len(some[::40]), 20, 3, None, seqs=some[::40])
    none = torch.tensor([i for i in range(4096) if rows[i] == 0], device=gpu)
    assert (out[none] == 0).all()


def test_values_of_any_size(gpu):
    """Scores far apart and growing along the sequence (references that move), queries of
    large and small magnitudes, and rows of zeros."""
    from ds4cuda_amd import ops
    b = Batch(gpu, [800, 800], 64, 8)
    for s, step in ((0, 100), (1, 50)):
        a = b.at(s)
        up = (torch.arange(800, device=gpu) // step).to(torch.int8)
        b.cache.sexp[a, :7] += up[:, None] - 4
        b.cache.tail[a] *= torch.exp2(up.float() - 4)[:, None].half()
    b.cache.codes[b.at(1)[:40]] = 0
    b.cache.tail[b.at(1)[:40]] = 0
    for typ in ("bf16", "fp32"):
        for scale in (1.0, 1e-3, 1e-30):
            q = (queries(gpu, 2, 64, typ, 7).float() * scale).to(TYPES[typ])
            q[0, 5] = 0
            q[1, 6] *= 3
            out = ops.flash_attn_window_fp8(q, b.cache, b.table, b.seq_rows, page_rows=64)
            check(b, q, out, [1, 1], 0, 0, None)
    # scores beyond all others: one row takes everything
    q = queries(gpu, 2, 64, "bf16", 9) * 1e20
    out = ops.flash_attn_window_fp8(q, b.cache, b.table, b.seq_rows, page_rows=64)
    for s in range(2):
        kv = b.values(s)
        best = (q[s].double() @ kv.T).argmax(-1)
        assert (out[s].double() - kv[best]).abs().max() <= 2.0 ** -8 * kv.abs().max()


def test_sinks_that_take_much_or_nothing(gpu):
    b = Batch(gpu, [40], 16, 10)
    q = queries(gpu, 1, 64, "fp32", 10)
    sinks = torch.linspace(-200, 200, 64, device=gpu)
    sinks[3] = -float("inf")
    out = run(b, q, [1], sinks=sinks)
    check(b, q, out, [1], 0, 0, sinks)


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
@pytest.mark.parametrize("heads", [8, 64])
@pytest.mark.parametrize("value", ["nan", "inf", "tail"])
def test_rows_that_are_not_finite_reach_only_who_sees_them(gpu, value, heads, typ):
    rows, new, window, first = [150, 90], [40, 3], 16, 2
    b = Batch(gpu, rows, 32, 11)
    hit = {0: [3, 100, 112, 120, 149], 1: [89]}
    clean = [b.values(s) for s in range(2)]
    for s, some in hit.items():
        at = b.at(s)[some]
        if value == "nan":
            b.cache.codes[at, 77] = 0xFF
        elif value == "inf":
            b.cache.sexp[at, 2] = 60
            b.cache.codes[at, 128:192] = 0x40
        else:
            b.cache.tail[at, 9] = -float("inf")
    q = queries(gpu, 43, heads, typ, 12)
    out = run(b, q, new, window, first)
    a = 0
    for s in range(2):
        pos = [rows[s] - new[s] + i for i in range(new[s])]
        kv = clean[s]
        ref, size, err = attend_64(q[a:a + new[s]], kv, pos, window, first, None)
        bound = bound_of(ref, size, err, typ == "fp32")
        for i, p in enumerate(pos):
            sees = any(k <= p and (k > p - window or k < first) for k in hit[s])
            if sees:
                assert not torch.isfinite(out[a + i]).all(-1).any(), (s, p)
            else:
                assert ((out[a + i].double() - ref[i]).abs() <= bound[i]).all(), (s, p)
        a += new[s]
    assert not torch.isfinite(out).all() and torch.isfinite(out[:30]).all(-1).any()


def test_queries_that_are_not_finite_reach_no_others(gpu):
    b = Batch(gpu, [90, 30], 16, 13)
    for heads in (8, 64, 128):
        new = [33, 3]
        q = queries(gpu, 36, heads, "bf16", 14)
        want = run(b, q, new, 20, 1)
        bad = q.clone()
        bad[7] = float("nan")
        bad[20, 3, 100] = float("inf")
        bad[34, 1, 0] = float("nan")
        got = run(b, bad, new, 20, 1)
        assert torch.isnan(got[7]).all() and torch.isnan(got[34, 1]).all() and not torch.isfinite(got[20, 3]).all()
        same = torch.ones((36, heads), dtype=torch.bool, device=gpu)
        same[7] = same[20, 3] = same[34, 1] = False
        assert torch.equal(got[same], want[same])


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
def test_bad_tables_are_nan_and_nothing_else(gpu, typ):
    """Entries outside the pool, rows past the table, slots that are not there: no read,
    NaN for the queries of that sequence alone."""
    rows = [300, 6000, 200, 100]
    for which, change in (("page", -5), ("page", 1 << 29), ("rows", 1 << 30), ("slot", 4), ("slot", -1)):
        b = Batch(gpu, rows, 32, 15)
        q = queries(gpu, 4, 64, typ, 16)
        seqs = i32([0, 1, 2, 3], gpu)
        from ds4cuda_amd import ops
        call = lambda: ops.flash_attn_window_fp8(q, b.cache, b.table, b.seq_rows, page_rows=32, seq_ids=seqs)
        if which == "page":
            b.table[1, 100] = change
            b.table[2, 0] = change
            hit = [1, 2]
        elif which == "rows":
            b.seq_rows[1] = change
            hit = [1]
        else:
            seqs[1] = change
            hit = [1]
        got = call()
        assert torch.isnan(got[hit]).all()
        # (not against another call's: other cuts of the line of tiles round the weights
        # to other references, each as near to 64 bits as the bound says)
        keep = [s for s in range(4) if s not in hit]
        check(b, q[keep], got[keep], [1] * len(keep), 0, 0, None, seqs=keep)
    # rows below zero: a sequence that holds nothing
    b.seq_rows[3] = -7
    seqs[1] = 1
    assert (call()[3] == 0).all()


def test_outputs_that_no_entry_names_stay(gpu):
    b = Batch(gpu, [100, 50, 20], 16, 17)
    q = queries(gpu, 40, 16, "bf16", 18)
    out = torch.full_like(q, 7.0)
    got = run(b, q, [10, 0, 12], 30, 2, seqs=[2, 0, 1], out=out)
    assert got.data_ptr() == out.data_ptr()
    check(b, q, out, [10, 0, 12], 30, 2, None, seqs=[2, 0, 1])
    assert (out[22:] == 7.0).all()
    # more queries than rows: those before the sequence see nothing
    b = Batch(gpu, [3], 16, 19)
    out = run(b, q[:8], [8])
    assert (out[:5] == 0).all()
    check(b, q[5:8], out[5:], [3], 0, 0, None)
    # starts that go back or past the end stay inside the buffers
    from ds4cuda_amd import ops
    out = torch.full_like(q, 7.0)
    b = Batch(gpu, [60, 60, 60], 16, 20)
    for start in ([5, 2, 90, 3], [-4, 60, -1, 40], [1 << 30, 0, 40, 0]):
        ops.flash_attn_window_fp8(q, b.cache, b.table, b.seq_rows, page_rows=16, q_start=i32(start, gpu), out=out)
    torch.cuda.synchronize()


def test_a_captured_call_follows_the_lengths(gpu):
    from ds4cuda_amd import ops
    b = Batch(gpu, [5000, 4000, 300], 64, 21)
    q = queries(gpu, 3, 64, "bf16", 22)
    out = torch.empty_like(q)
    ws = torch.empty(ops.window_workspace_bytes(3, 3, 64), dtype=torch.uint8, device=gpu)

    def call(to):
        return ops.flash_attn_window_fp8(q, b.cache, b.table, b.seq_rows, page_rows=64, window=3000, n_first=4, out=to,
                                         workspace=ws)
    call(out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(out)
    for rows in ([5000, 4000, 300], [1, 3999, 0], [64, 63, 299]):
        b.seq_rows.copy_(i32(rows, gpu))
        out.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, call(torch.empty_like(q)))
        b.rows = rows
        keep = [s for s in range(3) if rows[s]]
        check(b, q[keep], got[keep], [1] * len(keep), 3000, 4, None, seqs=keep)


def test_another_stream_and_a_dirty_workspace(gpu):
    from ds4cuda_amd import ops
    b = Batch(gpu, [3000, 20], 64, 23)
    q = queries(gpu, 2, 64, "fp32", 24)
    want = run(b, q, [1, 1])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    ws = torch.full((ops.window_workspace_bytes(2, 2, 64),), 0xFF, dtype=torch.uint8, device=gpu)
    torch.cuda.synchronize()
    start = i32([0, 1, 2], gpu)
    torch.cuda.synchronize()
    got = ops.flash_attn_window_fp8(q, b.cache, b.table, b.seq_rows, page_rows=64, q_start=start, workspace=ws, stream=s)
    raw = ops.flash_attn_window_fp8(q, b.cache, b.table, b.seq_rows, page_rows=64, q_start=start, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(raw, want)


def test_pages_past_32_bits(gpu):
    """Rows whose codes lie more than 4 GB into the cache."""
    from ds4cuda_amd import ops
    n_pages, page = 37600, 256
    cache = ops.Fp8KVCache(torch.full((n_pages * page, 448), 0x7F, dtype=torch.uint8, device=gpu),
                           torch.zeros((n_pages * page, 8), dtype=torch.int8, device=gpu),
                           torch.zeros((n_pages * page, 64), dtype=torch.float16, device=gpu))
    b = Batch(gpu, [700], page, 25, spare=0)
    small = b.cache
    b.table += n_pages - b.n_pages
    for name in ("codes", "sexp", "tail"):
        getattr(cache, name)[-b.n_pages * page:] = getattr(small, name)
    b.cache = cache
    q = queries(gpu, 3, 64, "bf16", 26)
    check(b, q, run(b, q, [3]), [3], 0, 0, None)
    del b, cache
    torch.cuda.empty_cache()


@pytest.mark.parametrize("typ,heads", [("bf16", 64), ("fp32", 64), ("bf16", 8), ("fp32", 8)])
def test_positions_up_to_2_31(gpu, typ, heads):
    """A page of 2^20 rows named 2048 times: the last rows of the longest sequence are those
    of a short one, to the bit; a longer one is NaN."""
    from ds4cuda_amd import ops
    n, most = 1 << 20, (1 << 31) - 256
    g = torch.Generator(gpu).manual_seed(31)
    codes = torch.randint(0, 0x70, (n, 448), generator=g, device=gpu, dtype=torch.uint8)
    cache = ops.Fp8KVCache(codes, torch.zeros((n, 8), dtype=torch.int8, device=gpu),
                           torch.zeros((n, 64), dtype=torch.float16, device=gpu))
    table = torch.zeros((3, 2048), dtype=torch.int32, device=gpu)
    rows = i32([most, most % n + n, most + 1], gpu)
    q = queries(gpu, 1, heads, typ, 32).expand(3, heads, 512).contiguous()
    out = ops.flash_attn_window_fp8(q, cache, table, rows, page_rows=n, window=100, n_first=3)
    assert torch.isfinite(out[:2]).all() and torch.equal(out[0], out[1]) and bool(out[0].any())
    assert torch.isnan(out[2]).all()


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
def test_many_single_tokens_of_a_slice(gpu, typ):
    """More problems of 16 rows than a workgroup lays out itself, some of them cut."""
    rows = [2500 if i % 50 == 7 else (37 * i) % 90 for i in range(300)]
    b = Batch(gpu, rows, 32, 33)
    q = queries(gpu, len(rows), 16, typ, 34)
    out = run(b, q, [1] * len(rows))
    for i, r in enumerate(rows):
        if r == 0:
            assert not out[i].any()
    live = [i for i, r in enumerate(rows) if r]
    check(b, q[live], out[live], [1] * len(live), 0, 0, None, seqs=live)


@pytest.mark.parametrize("heads", [8, 64, 128])
@pytest.mark.parametrize("rows,new,page,window,first", [
    ([1, 2, 3], [1, 2, 3], 16, 0, 0), ([0, 33, 64], [0, 1, 64], 32, 0, 0), ([700, 90, 1], [130, 0, 1], 128, 640, 2),
    ([1500, 40], [1, 40], 256, 700, 33), ([260, 131], [9, 100], 4, 0, 64), ([2000], [3], 64, 600, 700)])
def test_tables_for_long_sequences(gpu, rows, new, page, window, first, heads):
    """Short sequences too, in tables that have room for long ones."""
    b = Batch(gpu, rows, page, 40, entries=max(-(-r // page) for r in rows) + -(-1024 // page))
    sinks = torch.linspace(-3, 3, heads, device=gpu)
    q = queries(gpu, sum(new), heads, "bf16", 41)
    check(b, q, run(b, q, new, window, first, sinks), new, window, first, sinks)


@pytest.mark.parametrize("value", ["nan", "inf"])
@pytest.mark.parametrize("heads", [8, 64])
def test_rows_that_are_not_finite_in_long_tables(gpu, heads, value):
    b = Batch(gpu, [700], 16, 42, entries=100)
    q = queries(gpu, 60, heads, "bf16", 43)
    want = run(b, q, [60])
    at = int(b.at(0)[660])
    if value == "nan":
        b.cache.codes[at, 5] = 0x7F
    else:
        b.cache.tail[at] = float("inf")
    got = run(b, q, [60])
    assert torch.equal(got[:20], want[:20])   # positions 640 .. 659
    assert not torch.isfinite(got[20:]).all(-1).any()


def test_as_many_sequences_as_a_call_takes(gpu):
    """4096 sequences, more than 8192 problems, a long one among the last."""
    new = [1 + (i % 4 == 0) for i in range(4096)]
    rows = [(7 * i) % 40 + n for i, n in enumerate(new)]
    rows[4050] = 3100
    b = Batch(gpu, rows, 16, 37)
    q = queries(gpu, sum(new), 128, "bf16", 38)
    out = run(b, q, new, window=2500, first=20)
    some = [i for i in range(4096) if i % 37 == 0 or i > 4000]
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    pick = torch.tensor([k for i in some for k in range(start[i], start[i + 1])], device=gpu)
    check(b, q[pick], out[pick], [new[i] for i in some], 2500, 20, None, seqs=some)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
@pytest.mark.parametrize("heads", [16, 64])
def test_one_sequence_over_all_workgroups(gpu, heads, typ):
    """Its rows are joined from more than 64 parts."""
    b = Batch(gpu, [41003], 64, 35)
    sinks = torch.linspace(-2, 2, heads, device=gpu)
    q = queries(gpu, 1, heads, typ, 36)
    check(b, q, run(b, q, [1], sinks=sinks), [1], 0, 0, sinks)


def test_the_pages_and_the_attention_as_they_are_used(gpu):
    """Prompts appended and attended, forked, extended token by token and attended, freed
    and compacted: each step against the rows that the sequences hold."""
    from ds4cuda_amd import ops, pages
    pool = pages.PagePool.empty(64, 16, 8, 400, 2, gpu)
    g = torch.Generator(gpu).manual_seed(27)
    held = {}   # fp32 rows of each sequence

    def append(seqs, new):
        kv = torch.randn((sum(new), 512), generator=g, device=gpu)
        dst = pool.extend(i32(seqs, gpu), i32(new, gpu), sum(new))
        for layer in range(2):
            pool.append(kv, dst, layer=layer)
        a = 0
        for s, n in zip(seqs, new):
            held[s] = torch.cat([held.get(s, kv[:0]), kv[a:a + n]])
            a += n

    def attended(seqs, new, window, first):
        q = torch.randn((sum(new), 32, 512), generator=g, device=gpu)
        start = [sum(new[:i]) for i in range(len(new) + 1)]
        out = pool.attend(q, seqs=i32(seqs, gpu), q_start=i32(start, gpu), window=window, n_first=first, layer=1)
        pool.check()
        a = 0
        for s, n in zip(seqs, new):
            c = ops.Fp8KVCache.empty(held[s].shape[0], gpu)
            c.append(held[s])
            kv = row_values(c.codes, c.sexp, c.tail)
            ref, size, err = attend_64(q[a:a + n], kv, [kv.shape[0] - n + i for i in range(n)], window, first, None)
            assert ((out[a:a + n].double() - ref).abs() <= bound_of(ref, size, err, True)).all()
            a += n

    append([0, 1], [137, 60])
    attended([0, 1], [137, 60], 50, 3)
    pool.fork(i32([0, 0, 1], gpu), i32([2, 3, 4], gpu), i32([-1, 100, -1], gpu))
    held[2], held[3], held[4] = held[0], held[0][:100], held[1]
    for _ in range(20):
        append([2, 3, 4, 0], [1, 1, 1, 1])
    attended([2, 3, 4, 0], [1, 1, 1, 1], 0, 0)
    attended([4, 3], [20, 2], 64, 1)
    pool.free(i32([0, 4], gpu))
    pool.free(i32([2], gpu), i32([150], gpu))
    held[2] = held[2][:150]
    assert int(pool.compact()) == int((pool.refs > 0).sum())
    attended([1, 2, 3], [5, 1, 1], 40, 17)
    pool.fork(i32([2], gpu), i32([0], gpu), deep=True)
    held[0] = held[2]
    append([0, 3], [30, 2])
    attended([0, 2, 3], [30, 1, 2], 0, 0)
