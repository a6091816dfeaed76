"""The page pool against a model of lists: random runs of extend, append, fork, free
and compact, refused calls, large pools, captured calls."""
import random

import pytest
import torch

from paged_check import PoolModel, quantized_rows

pytestmark = pytest.mark.gpu


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def make(gpu, n_pages, page_rows, n_seqs, max_rows, layers=2):
    from ds4cuda_amd import pages
    pool = pages.PagePool.empty(n_pages, page_rows, n_seqs, max_rows, layers, gpu)
    return pool, PoolModel(n_pages, page_rows, n_seqs, -(-max_rows // page_rows), layers)


def same(pool, model, contents=True):
    torch.cuda.synchronize()
    assert pool.refs.tolist() == model.refs
    assert pool.rows.tolist() == model.rows
    table = pool.table.tolist()
    for s, held in enumerate(model.table):
        assert table[s][:len(held)] == held, s
    if contents:
        for layer, tags in enumerate(model.tags):
            held = [p * model.page + i for t, r in zip(model.table, model.rows) for k, p in enumerate(t)
                    for i in range(min(model.page, r - k * model.page))]
            got = tagged(pool, layer)
            assert [got[h] for h in held] == [tags[h] for h in held], layer


def tagged(pool, layer):
    """A row's tag, where all its three arrays carry the same; else -1."""
    c = pool.codes[layer].to(torch.int64)
    t = (c[:, 0] << 8) + c[:, -1]
    whole = (c[:, ::2] == c[:, :1]).all(1) & (c[:, 1::2] == c[:, -1:]).all(1)
    whole &= (pool.sexp[layer].to(torch.int64) & 255 == (t & 255)[:, None]).all(1)
    whole &= (pool.tail[layer].to(torch.int64) == t[:, None]).all(1)
    return torch.where(whole, t, -1).tolist()


def tag(pool, model, dst, first):
    """Writes tags first, first + 1, .. into the rows dst of every layer (another tag
    per layer), as an append would."""
    dst = [d for d in dst if d >= 0]
    for layer in range(pool.n_layers):
        tags = [(first + i * 7 + layer * 1000) % 30000 + 1 for i in range(len(dst))]
        for d, v in zip(dst, tags):
            model.tags[layer][d] = v
        at = torch.tensor(dst, device=pool.device, dtype=torch.int64)
        v = torch.tensor(tags, device=pool.device, dtype=torch.int64)
        hi, lo = (v >> 8).to(torch.uint8), (v & 255).to(torch.uint8)
        pool.codes[layer, at] = torch.stack([hi, lo], -1).repeat(1, 224)
        pool.sexp[layer, at] = lo.view(torch.int8)[:, None].expand(-1, 8)
        pool.tail[layer, at] = v.to(torch.int16)[:, None].expand(-1, 64)


def ok(pool, code):
    from ds4cuda_amd import Ds4HipError
    if code == 0:
        pool.check()
        return
    with pytest.raises(Ds4HipError) as e:
        pool.check()
    assert e.value.code == code
    pool.check()


@pytest.mark.parametrize("page_rows,n_pages,layers", [(1, 40, 1), (16, 60, 2), (64, 30, 1), (128, 24, 3), (2, 300, 2)])
def test_random_runs(gpu, page_rows, n_pages, layers):
    rng = random.Random(page_rows * 1000 + n_pages)
    n_seqs = 12
    pool, model = make(gpu, n_pages, page_rows, n_seqs, 9 * page_rows + 3, layers)
    refused = 0
    for step in range(60):
        what = rng.choice(["extend", "extend", "fork", "deep", "free", "cut", "compact"])
        some = rng.sample(range(n_seqs), rng.randint(1, 4))
        if what == "extend":
            n_new = [rng.randint(0, 3 * page_rows) for _ in some]
            n_dst = sum(n_new) + rng.randint(0, 3)
            code, want = model.extend(some, n_new, n_dst)
            dst = pool.extend(i32(some, gpu), i32(n_new, gpu), n_dst)
            assert dst.tolist() == want
            if code == 0:
                tag(pool, model, want, 100 * step)
        elif what in ("fork", "deep"):
            empty = [s for s in range(n_seqs) if model.rows[s] == 0]
            kids = (empty + some)[:rng.randint(1, 3)]
            parents = [rng.randrange(n_seqs) for _ in kids]
            n_rows = rng.choice([None, [rng.randint(-1, max(model.rows[p], 1)) for p in parents]])
            code = model.fork(parents, kids, n_rows, what == "deep")
            pool.fork(i32(parents, gpu), i32(kids, gpu), None if n_rows is None else i32(n_rows, gpu), what == "deep")
        elif what == "compact":
            code, live = 0, model.compact()
            assert int(pool.compact()) == live
        else:
            keep = None if what == "free" else [rng.randint(0, model.rows[s]) for s in some]
            code = model.free(some, keep)
            pool.free(i32(some, gpu), None if keep is None else i32(keep, gpu))
        refused += code != 0
        ok(pool, code)
        same(pool, model)
    assert refused < 40


def test_refusals_change_nothing(gpu):
    pool, model = make(gpu, 10, 16, 6, 64)
    _, dst = model.extend([0, 1], [40, 16], 56)
    assert pool.extend(i32([0, 1], gpu), i32([40, 16], gpu), 56).tolist() == dst
    tag(pool, model, dst, 5)
    model.fork([0], [2], [32], False)
    pool.fork(i32([0], gpu), i32([2], gpu), i32([32], gpu))
    ok(pool, 0)
    calls = [
        (-22, lambda: pool.extend(i32([0, 0], gpu), i32([1, 1], gpu), 2)),        # a sequence twice
        (-22, lambda: pool.extend(i32([6], gpu), i32([1], gpu), 1)),              # not a sequence
        (-22, lambda: pool.extend(i32([-1], gpu), i32([1], gpu), 1)),
        (-22, lambda: pool.extend(i32([1], gpu), i32([-1], gpu), 1)),             # fewer rows
        (-22, lambda: pool.extend(i32([1], gpu), i32([5], gpu), 4)),              # more than there is room to say
        (-28, lambda: pool.extend(i32([1], gpu), i32([49], gpu), 49)),            # the table row is full
        (-28, lambda: pool.extend(i32([1, 3, 4], gpu), i32([48, 64, 1], gpu), 113)),   # too few pages
        (-22, lambda: pool.fork(i32([0], gpu), i32([1], gpu))),                   # a child that holds rows
        (-22, lambda: pool.fork(i32([0, 1], gpu), i32([3, 3], gpu))),             # a child twice
        (-22, lambda: pool.fork(i32([0], gpu), i32([3], gpu), i32([41], gpu))),   # more rows than there are
        (-22, lambda: pool.fork(i32([9], gpu), i32([3], gpu))),
        (-28, lambda: pool.fork(i32([0, 0, 0], gpu), i32([3, 4, 5], gpu), deep=True)),  # 9 pages of 6
        (-22, lambda: pool.free(i32([1, 1], gpu))),
        (-22, lambda: pool.free(i32([7], gpu))),
        (-22, lambda: pool.free(i32([0], gpu), i32([41], gpu))),
        (-22, lambda: pool.free(i32([0], gpu), i32([20], gpu))),                  # inside a shared page
        (-22, lambda: pool.free(i32([2], gpu), i32([-1], gpu))),
    ]
    for code, call in calls:
        got = call()
        if got is not None:
            assert (got == -1).all()
        ok(pool, code)
        same(pool, model)
    # what is asked for afterwards works
    code, dst = model.extend([3], [64], 64)
    assert pool.extend(i32([3], gpu), i32([64], gpu), 64).tolist() == dst and code == 0
    ok(pool, 0)
    same(pool, model, False)


def test_a_table_that_names_no_page_is_refused(gpu):
    """Entries outside the pool are neither followed nor counted."""
    pool, _ = make(gpu, 8, 16, 4, 64, 1)
    pool.extend(i32([0, 1], gpu), i32([40, 20], gpu), 60)
    pool.check()
    for bad in (-1, 8, 1 << 30, 7):   # 7: a free page
        pool.table[0, 1] = bad
        before = [t.clone() for t in (pool.refs, pool.rows)]
        for call in (lambda: pool.free(i32([1, 0], gpu)), lambda: pool.fork(i32([1, 0], gpu), i32([2, 3], gpu)),
                     lambda: pool.fork(i32([0], gpu), i32([3], gpu), deep=True)):
            call()
            ok(pool, -22)
            assert torch.equal(pool.refs, before[0]) and torch.equal(pool.rows, before[1])
    pool.table[0, 2] = 99
    assert pool.extend(i32([0], gpu), i32([3], gpu), 3).tolist() == [-1] * 3
    ok(pool, -22)
    pool.compact()   # leaves such an entry as it is
    pool.check()
    assert pool.table[0, 2] == 99


def test_append_writes_the_rows_it_is_given(gpu):
    from ds4cuda_amd import ops, pages
    pool = pages.PagePool.empty(5, 16, 2, 64, 3, gpu)
    kv = torch.randn((21, 512), device=gpu)
    dst = pool.extend(i32([1], gpu), i32([20], gpu), 21)   # one place is none
    plain = ops.Fp8KVCache.empty(21, gpu)
    plain.append(kv)
    for layer in (2, 0):
        pool.append(kv, dst, layer=layer)
    pool.check()
    at = dst[:20]
    for layer, some in ((0, True), (1, False), (2, True)):
        c = pool.layer(layer)
        for got, want in ((c.codes, plain.codes), (c.sexp, plain.sexp), (c.tail, plain.tail)):
            assert torch.equal(got[at], want[:20]) if some else not got.any()
            rest = torch.ones(80, dtype=torch.bool, device=gpu)
            rest[at] = False
            assert not got[rest].any()


def test_many_pages_and_jobs(gpu):
    """More pages than a step of the search reads, and the most jobs of a call."""
    n = 1024
    pool, model = make(gpu, 20011, 2, 2 * n, 30, 1)
    seqs = list(range(n))
    n_new = [(i * 7) % 30 for i in range(n)]
    code, dst = model.extend(seqs, n_new, sum(n_new))
    assert pool.extend(i32(seqs, gpu), i32(n_new, gpu), sum(n_new)).tolist() == dst and code == 0
    tag(pool, model, dst, 3)
    model.free(seqs[::3], None)
    pool.free(i32(seqs[::3], gpu))
    kids = [n + i for i in range(n)]
    parents = [(i * 5) % n for i in range(n)]
    assert model.fork(parents, kids, None, False) == 0
    pool.fork(i32(parents, gpu), i32(kids, gpu))
    ok(pool, 0)
    same(pool, model)
    assert int(pool.compact()) == model.compact()
    ok(pool, 0)
    same(pool, model)


def test_rows_past_32_bits(gpu):
    """Pages whose codes lie more than 4 GB into the array move and append like others."""
    from ds4cuda_amd import ops, pages
    n_pages, page = 37600, 256   # 9.6M rows, 4.31 GB of codes
    pool = pages.PagePool.empty(n_pages, page, 4, 1024, 1, gpu)
    pool.refs.fill_(1)
    pool.refs[-4:] = 0
    kv = torch.randn((300, 512), device=gpu)
    dst = pool.extend(i32([0], gpu), i32([300], gpu), 300)
    assert int(dst[0]) == (n_pages - 4) * page
    pool.append(kv, dst)
    plain = ops.Fp8KVCache.empty(300, gpu)
    plain.append(kv)
    pool.fork(i32([0], gpu), i32([1], gpu), deep=True)
    pool.check()
    at = (torch.tensor([n_pages - 2, n_pages - 1], device=gpu)[:, None] * page + torch.arange(page, device=gpu)).flatten()
    assert pool.table[1, :2].tolist() == [n_pages - 2, n_pages - 1]
    for got, want in ((pool.codes[0], plain.codes), (pool.sexp[0], plain.sexp), (pool.tail[0], plain.tail)):
        assert torch.equal(got[at[:300]], want)
    # all but those pages are given back: compaction brings them to the front
    pool.refs[:-4] = 0
    assert int(pool.compact()) == 4
    assert pool.table[1, :2].tolist() == [2, 3]
    assert torch.equal(pool.codes[0, 512:812], plain.codes) and torch.equal(pool.tail[0, 512:812], plain.tail)
    del pool
    torch.cuda.empty_cache()


def test_captured_calls_follow_the_device(gpu):
    """A graph of fork, extend and free: the pages it takes are those that are free
    when it runs."""
    pool, model = make(gpu, 40, 16, 6, 160, 2)
    _, dst = model.extend([0, 1], [37, 50], 87)
    pool.extend(i32([0, 1], gpu), i32([37, 50], gpu), 87)
    tag(pool, model, dst, 9)
    parents, kids, one = i32([0, 1], gpu), i32([2, 3], gpu), i32([1, 2], gpu)
    place = torch.empty(3, dtype=torch.int64, device=gpu)
    n_live = torch.empty((), dtype=torch.int32, device=gpu)
    pool._ws(None)

    def step():
        pool.fork(parents, kids)
        pool.extend(kids, one, 3, dst_rows=place)
        pool.free(parents)
        pool.compact(n_live)

    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for again in range(3):
        a, b = ([0, 1], [2, 3]) if again % 2 == 0 else ([2, 3], [0, 1])
        parents.copy_(i32(a, gpu))
        kids.copy_(i32(b, gpu))
        assert model.fork(a, b, None, False) == 0
        _, want = model.extend(b, [1, 2], 3)
        model.free(a, None)
        live = model.compact()
        g.replay()
        torch.cuda.synchronize()
        assert place.tolist() == want and int(n_live) == live
        ok(pool, 0)
        now = {d: t for d, t in zip(want, range(3))}
        assert len(now) == 3
        # (the compaction may have moved the new rows: their contents are not compared)
        same(pool, model, False)


def test_another_stream(gpu):
    pool, model = make(gpu, 30, 16, 4, 200, 1)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        _, dst = model.extend([0], [100], 100)
        got = pool.extend(i32([0], gpu), i32([100], gpu), 100)
        assert got.tolist() == dst
        tag(pool, model, dst, 4)
        kid = i32([1], gpu)
        zero = i32([0], gpu)
        s.synchronize()
    model.fork([0], [1], None, True)
    pool.fork(zero, kid, deep=True, stream=s)
    s.synchronize()
    same(pool, model)
    pool.free(kid, stream=s.cuda_stream)
    s.synchronize()
    model.free([1], None)
    same(pool, model)


def test_a_check_waits_for_calls_on_other_streams(gpu):
    from ds4cuda_amd import Ds4HipError, pages
    pool = pages.PagePool.empty(4, 16, 2, 64, 1, gpu)
    seqs, n_new = (torch.tensor([v], dtype=torch.int32, device=gpu) for v in (0, 65))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)   # about 10 ms
    pool.extend(seqs, n_new, 65, stream=s)
    with pytest.raises(Ds4HipError) as e:
        pool.check()
    assert e.value.code == -28
    pool.check()
