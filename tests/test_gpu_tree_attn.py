"""Attention of trees of drafted tokens over pages: against the definition in 64 bits, where
trees, windows, pages and lengths can go wrong."""
import random

import pytest
import torch

from draft_check import attend_tree_64, random_tree
from paged_check import bound_of
from test_gpu_window_attn import Batch, i32, queries

pytestmark = pytest.mark.gpu


def run(b, q, trees, window=0, first=0, sinks=None, seqs=None, **kw):
    from ds4cuda_amd import ops
    sizes = [len(t) for t in trees]
    start = i32([sum(sizes[:i]) for i in range(len(sizes) + 1)], b.gpu)
    return ops.flash_attn_tree_fp8(q, i32([p for t in trees for p in t], b.gpu), b.cache, b.table, b.seq_rows, page_rows=b.page,
                                   window=window, n_first=first, sinks=sinks, q_start=start,
                                   seq_ids=None if seqs is None else i32(seqs, b.gpu), **kw)


def check(b, q, out, trees, window, first, sinks, seqs=None):
    f32, a, off, norm = q.dtype == torch.float32, 0, 0.0, 0.0
    for i, tree in enumerate(trees):
        n, s = len(tree), i if seqs is None else seqs[i]
        if n == 0:
            continue
        ref, size, err = attend_tree_64(q[a:a + n], b.values(s), tree, window, first, sinks)
        d = (out[a:a + n].double() - ref).abs()
        assert torch.isfinite(out[a:a + n]).all(), (i, s)
        worst = (d - bound_of(ref, size, err, f32)).amax()
        assert worst <= 0, (i, s, float(worst), float(d.amax()))
        off, norm = off + float((d * d).sum()), norm + float((ref * ref).sum())
        a += n
    # roundings taken together, as for prompts: bf16 2^-8 at most each, fp32 parts of 2^-22 with room for ten times as much
    assert (off / norm) ** 0.5 <= (1e-5 if f32 else 4e-3)


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
@pytest.mark.parametrize("heads", [8, 16, 32, 64, 128])
@pytest.mark.parametrize("shape", ["random", "roots", "star", "chain"])
@pytest.mark.parametrize("rows,new,page,window,first", [
    ([1], [1], 16, 0, 0), ([5, 40], [5, 9], 16, 0, 0), ([97, 64, 33], [1, 32, 33], 32, 0, 0), ([130], [7], 1, 40, 5),
    ([300, 90, 31], [17, 0, 31], 64, 6, 0), ([200, 700], [70, 12], 128, 128, 4), ([60, 61], [40, 20], 8, 1, 50)])
def test_trees(gpu, rows, new, page, window, first, shape, heads, typ):
    b = Batch(gpu, rows, page, heads + sum(new))
    rng = random.Random(heads + page)
    trees = [random_tree(rng, n, shape) for n in new]
    q = queries(gpu, sum(new), heads, typ, 3)
    sinks = torch.randn(heads, device=gpu) if page != 32 else None
    check(b, q, run(b, q, trees, window, first, sinks), trees, window, first, sinks)


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
def test_long_and_short_contexts(gpu, typ):
    """Problems that are cut, whose parts have and have not the tree's rows; more nodes than a tile; sequences in
    any slot."""
    rng = random.Random(4)
    for rows, new, heads, window in (([9000, 60, 700], [12, 3, 40], 64, 0), ([20000], [4], 16, 0), ([5000, 4000], [150, 1], 8, 0),
                                     ([6000, 3000], [33, 65], 64, 2000), ([3000] * 6, [9] * 6, 128, 0)):
        b = Batch(gpu, [17] + rows, 64, len(rows))
        trees = [random_tree(rng, n, "random") for n in new]
        seqs = list(range(len(rows), 0, -1))
        trees = [trees[s - 1] for s in seqs]
        q = queries(gpu, sum(new), heads, typ, 5)
        sinks = torch.randn(heads, device=gpu)
        out = run(b, q, trees, window, 3, sinks, seqs)
        check(b, q, out, trees, window, 3, sinks, seqs)
        assert torch.equal(out, run(b, q, trees, window, 3, sinks, seqs))


def test_the_largest_trees(gpu):
    from ds4cuda_amd import ops
    rng = random.Random(6)
    for heads, shape in ((8, "random"), (64, "chain"), (16, "star")):
        b = Batch(gpu, [1024, 1500], 256, heads)
        trees = [random_tree(rng, 1024, shape), random_tree(rng, 1023, shape)]
        q = queries(gpu, 2047, heads, "bf16", 7)
        out = run(b, q, trees, 100, 5)
        some = [list(range(0, 1024, 37)) + [1023], list(range(1, 1023, 41)) + [1022]]
        from draft_check import rows_seen
        from paged_check import attend_64
        for s, at in enumerate(some):
            kv = b.values(s)
            base = b.rows[s] - len(trees[s])
            for v in at:
                rows = kv[torch.tensor(rows_seen(base, trees[s], v, 100, 5), device=gpu)]
                i = 1024 * s + v
                ref, size, err = attend_64(q[i:i + 1], rows, [rows.shape[0] - 1], 0, 0, None)
                assert ((out[i:i + 1].double() - ref).abs() <= bound_of(ref, size, err, False)).all()
    # one node more: that sequence is NaN, the other is not
    b = Batch(gpu, [1100, 40], 256, 1)
    q = queries(gpu, 1028, 8, "bf16", 8)
    out = run(b, q, [random_tree(rng, 1025, "chain"), [-1, 0, 0]])
    assert out[:1025].isnan().all()
    assert out[1025:].isfinite().all()


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
def test_chains_are_prompts(gpu, typ):
    """Parents i - 1: the windowed attention of the same queries, to the bit where no reference moves."""
    from ds4cuda_amd import ops
    b = Batch(gpu, [500, 77], 16, 9)
    q = queries(gpu, 64, 64, typ, 9)
    trees = [random_tree(None, 50, "chain"), random_tree(None, 14, "chain")]
    for window, first in ((0, 0), (33, 7)):
        a = run(b, q, trees, window, first)
        w = ops.flash_attn_window_fp8(q, b.cache, b.table, b.seq_rows, page_rows=16, window=window, n_first=first,
                                      q_start=i32([0, 50, 64], gpu))
        check(b, q, a, trees, window, first, None)
        assert (a.float() - w.float()).abs().amax() <= (2e-5 if typ == "fp32" else 0.05)


def test_rows_that_are_not_finite(gpu):
    """A row of NaN reaches its node and the ones below it, no other; one before the tree's in the window alone."""
    rng = random.Random(10)
    for heads in (8, 64):
        b = Batch(gpu, [150], 32, 3)
        tree = random_tree(rng, 40, "random")
        q = queries(gpu, 40, heads, "bf16", 11)
        clean = run(b, q, [tree], 30, 2)
        from draft_check import rows_seen
        for row in (110 + 3, 110 + 17, 90, 1, 50):
            a = int(b.at(0)[row])
            keep = b.cache.codes[a].clone()
            b.cache.codes[a] = 0x7F
            out = run(b, q, [tree], 30, 2)
            b.cache.codes[a] = keep
            for v in range(40):
                if row in rows_seen(110, tree, v, 30, 2):
                    assert out[v].isnan().all(), (row, v)
                else:
                    assert torch.isfinite(out[v]).all(), (row, v)
                    assert (out[v].float() - clean[v].float()).abs().amax() <= 0.05


def test_parents_that_are_none(gpu):
    """NaN for the nodes above which one lies (and at most the other queries of their 64 rows); the rest as ever."""
    b = Batch(gpu, [90, 70], 16, 12)
    rng = random.Random(13)
    for heads in (8, 64, 128):
        for bad in (-2, 12, 13, 1 << 30, -(1 << 31)):
            tree = random_tree(rng, 30, "random")
            tree[12] = bad
            other = random_tree(rng, 20, "random")
            q = queries(gpu, 50, heads, "bf16", 14)
            out = run(b, q, [tree, other], 50, 2)
            group = max(1, 64 // heads)
            below = {12}
            for v in range(13, 30):
                if tree[v] in below:
                    below.add(v)
            near = {v for v in range(30) if any(v // group == x // group for x in below)}
            for v in range(30):
                if v in below:
                    assert out[v].isnan().all(), (heads, bad, v)
                elif v not in near:
                    assert out[v].isfinite().all(), (heads, bad, v)
            assert out[30:].isfinite().all()


def test_sequences_that_cannot_be(gpu):
    """More nodes than rows, slots outside the table, page entries outside the pool, counts that go back."""
    from ds4cuda_amd import ops
    b = Batch(gpu, [5, 60, 60], 16, 15)
    q = queries(gpu, 12, 64, "bf16", 16)
    trees = [[-1, 0, 1, 2, 3, 4], [-1, 0, 0], [-1, 0, 1]]
    out = run(b, q, trees)
    assert out[:6].isnan().all() and out[6:].isfinite().all()
    out = run(b, q, trees[:1] + trees[1:], seqs=[1, 7, 2])
    assert out[6:9].isnan().all() and out[:6].isfinite().all() and out[9:].isfinite().all()
    b.table[2, 0] = b.n_pages
    out = run(b, q, trees, seqs=[1, 1, 2])
    assert out[9:].isnan().all() and out[:9].isfinite().all()
    empty = run(b, q[:0], [[], [], []])
    assert empty.shape[0] == 0


def test_q_start_none_is_one_node_each(gpu):
    from ds4cuda_amd import ops
    b = Batch(gpu, [33, 64, 1], 16, 17)
    q = queries(gpu, 3, 64, "bf16", 18)
    out = ops.flash_attn_tree_fp8(q, i32([-1, -1, -1], gpu), b.cache, b.table, b.seq_rows, page_rows=16, window=9, n_first=2)
    check(b, q, out, [[-1], [-1], [-1]], 9, 2, None)


@pytest.mark.parametrize("heads", [8, 64])
def test_many_sequences(gpu, heads):
    """More problems than a workgroup lays out: the plan kernel."""
    rng = random.Random(19)
    rows = [rng.randrange(12, 90) for _ in range(600)]
    new = [rng.randrange(0, 10) for _ in rows]
    b = Batch(gpu, rows, 16, 20)
    trees = [random_tree(rng, n, "random") for n in new]
    q = queries(gpu, sum(new), heads, "bf16", 21)
    out = run(b, q, trees, 30, 4)
    starts = [sum(new[:i]) for i in range(600)]
    some = [i for i in range(0, 600, 23) if new[i]]
    pick = torch.tensor([starts[i] + v for i in some for v in range(new[i])], device=gpu)
    check(b, q[pick], out[pick], [trees[i] for i in some], 30, 4, None, some)


def test_captured_as_the_pool_grows(gpu):
    """One graph over steps in which lengths and trees change; eager calls with a workspace of their own between."""
    from ds4cuda_amd import pages
    rng = random.Random(22)
    pool = pages.PagePool.empty(60, 16, 3, 200, 1, gpu)
    seqs, n = i32([2, 0], gpu), 8
    g = torch.Generator(gpu).manual_seed(23)

    def put(s, k):
        dst = pool.extend(i32([s], gpu), i32([k], gpu), k)
        pool.append(torch.randn((k, 512), generator=g, device=gpu), dst)
    put(2, 40)
    put(0, 90)
    parents, start = i32([-1] * (2 * n), gpu), i32([0, n, 2 * n], gpu)
    q = queries(gpu, 2 * n, 64, "bf16", 24)
    pool.attend_tree(q, parents, seqs=seqs, q_start=start, window=50, n_first=3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pool.attend_tree(q, parents, seqs=seqs, q_start=start, window=50, n_first=3)
    for step in range(4):
        put(2, 5 + step)
        put(0, 3)
        q.copy_(queries(gpu, 2 * n, 64, "bf16", 30 + step))
        trees = [random_tree(rng, n, "random") for _ in range(2)]
        parents.copy_(i32(trees[0] + trees[1], gpu))
        graph.replay()
        eager = pool.attend_tree(q, parents, seqs=seqs, q_start=start, window=50, n_first=3)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
    pool.check()


@pytest.mark.parametrize("heads,typ", [(64, "bf16"), (8, "bf16"), (16, "fp32")])
def test_one_large_tree_among_small_ones_in_a_short_window(gpu, heads, typ):
    """The small ones decide that nothing is cut; the large one's last nodes have many tiles of its own rows before them."""
    rng = random.Random(25)
    rows, new = [1100] + [40] * 30, [1000] + [1] * 29 + [3]
    b = Batch(gpu, rows, 64, 26)
    trees = [random_tree(rng, n, "random") for n in new]
    q = queries(gpu, sum(new), heads, typ, 27)
    out = run(b, q, trees, 64, 3)
    from draft_check import rows_seen
    from paged_check import attend_64
    kv = b.values(0)
    for v in list(range(0, 1000, 53)) + [998, 999]:
        seen = kv[torch.tensor(rows_seen(100, trees[0], v, 64, 3), device=gpu)]
        ref, size, err = attend_64(q[v:v + 1], seen, [seen.shape[0] - 1], 0, 0, None)
        assert ((out[v:v + 1].double() - ref).abs() <= bound_of(ref, size, err, typ == "fp32")).all(), v
    check(b, q[1000:], out[1000:], trees[1:], 64, 3, None, list(range(1, 31)))


@pytest.mark.parametrize("long,short,new,heads,typ", [(3, 14, 24, 64, "bf16"), (3, 22, 24, 64, "bf16"), (5, 30, 13, 64, "fp32"),
                                                      (60, 60, 2, 8, "bf16"), (60, 60, 2, 8, "fp32")])
def test_long_trees_and_many_short_ones(gpu, long, short, new, heads, typ):
    """Workgroups with parts of several trees, cut in any place, from the few problems that each workgroup lays out itself and
    the many that a kernel does."""
    rng = random.Random(long + short)
    rows = [rng.choice([8000, 8031, 7990])] * long + [rng.randint(40, 300) for _ in range(short)]
    rng.shuffle(rows)
    b = Batch(gpu, rows, 64, short)
    trees = [random_tree(rng, new - rng.randint(0, 1), "random") for _ in rows]
    q = queries(gpu, sum(map(len, trees)), heads, typ, 12)
    sinks = torch.randn(heads, device=gpu)
    out = run(b, q, trees, 0, 0, sinks)
    check(b, q, out, trees, 0, 0, sinks)
    assert torch.equal(out, run(b, q, trees, 0, 0, sinks))


def test_more_problems_than_the_plan_holds_in_shared_memory(gpu):
    rng = random.Random(13)
    rows = [270 + rng.randint(0, 140) for _ in range(17)]
    b = Batch(gpu, rows, 32, 14)
    trees = [random_tree(rng, 250 + rng.randint(0, 20), "random") for _ in rows]
    q = queries(gpu, sum(map(len, trees)), 128, "bf16", 15)   # two problems a node, more than 8192
    out = run(b, q, trees)
    assert 2 * q.shape[0] > 8192
    check(b, q, out, trees, 0, 0, None)
