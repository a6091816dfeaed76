"""Drafted trees in the page pool: accepted paths and what stays of their rows, against a model with Python
lists, to the bit; calls that the device refuses; the step's operators together."""
import random

import pytest
import torch

from draft_check import keep_model, random_tree, sample_64, walk
from paged_check import PoolModel

pytestmark = pytest.mark.gpu


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def starts(sizes):
    return [sum(sizes[:i]) for i in range(len(sizes) + 1)]


class Both:
    """A pool and its model; every row's bytes come from its tag."""

    def __init__(self, gpu, n_pages, page, n_seqs, entries, layers):
        from ds4cuda_amd import pages
        self.gpu, self.layers = gpu, layers
        self.pool = pages.PagePool.empty(n_pages, page, n_seqs, entries * page, layers, gpu)
        self.model = PoolModel(n_pages, page, n_seqs, entries, layers)
        self.tag = 0
        self.sync()

    def rows_of(self, tags):
        """codes, sexp, tail of tags [.., rows]"""
        t = tags[..., None]
        mix = lambda n, m: (t * 2654435761 + torch.arange(n, device=self.gpu) * 40503) // 64 % m
        return mix(448, 127).to(torch.uint8), (mix(8, 11) - 5).to(torch.int8), mix(64, 30000).to(torch.int16)

    def sync(self):
        tags = torch.tensor(self.model.tags, device=self.gpu)
        for t, v in zip((self.pool.codes, self.pool.sexp, self.pool.tail), self.rows_of(tags)):
            t.copy_(v)

    def extend(self, seqs, n_new):
        n = sum(n_new)
        dst = self.pool.extend(i32(seqs, self.gpu), i32(n_new, self.gpu), n)
        status, want = self.model.extend(seqs, n_new, n)
        assert status == 0 and dst.tolist() == want
        for tags in self.model.tags:
            for r in want:
                self.tag += 1
                tags[r] = self.tag
        self.sync()

    def check(self):
        self.pool.check()
        assert self.pool.refs.tolist() == self.model.refs and self.pool.rows.tolist() == self.model.rows
        for s, t in enumerate(self.model.table):
            assert self.pool.table[s, :len(t)].tolist() == t
        want = self.rows_of(torch.tensor(self.model.tags, device=self.gpu))
        for s, t in enumerate(self.model.table):   # rows that a sequence holds
            r = torch.arange(self.model.rows[s], device=self.gpu)
            at = torch.tensor(t + [0], device=self.gpu)[r // self.model.page] * self.model.page + r % self.model.page
            for x, w in zip((self.pool.codes, self.pool.sexp, self.pool.tail), want):
                assert torch.equal(x[:, at], w[:, at]), s


def random_path(rng, n):
    return sorted(rng.sample(range(n), rng.randrange(0, n + 1)))


def packed(paths, sizes):
    return [v for p, n in zip(paths, sizes) for v in p + [-7] * (n - len(p))]


@pytest.mark.parametrize("layers", [1, 3])
@pytest.mark.parametrize("page", [1, 4, 16, 64, 256])
def test_keep(gpu, page, layers):
    """Paths whose rows move to places that other rows of them leave, over pages' ends, of none and of all nodes."""
    rng = random.Random(page + layers)
    b = Both(gpu, 4000 // page + 60, page, 9, 700 // page + 2, layers)
    seqs = [7, 0, 3, 5, 8]
    b.extend(seqs, [rng.choice([0, 1, page - 1, page, page + 1, 100]) for _ in seqs])
    for step in range(8):
        some = rng.sample(seqs, rng.randrange(1, 6))
        sizes = [rng.choice([0, 1, 2, 7, 33, 100]) for _ in some]
        if step == 3:
            sizes[0] = 250
        b.extend(some, sizes)
        paths = [random_path(rng, n) for n in sizes]
        if step == 1:
            paths = [list(range(n)) for n in sizes]
        if step == 2:
            paths = [list(range(1, n)) for n in sizes]   # every row moves by one
        b.pool.keep(i32(some, gpu), i32(starts(sizes), gpu), i32(packed(paths, sizes), gpu), i32([len(p) for p in paths], gpu))
        assert keep_model(b.model, some, sizes, paths) == 0
        b.check()
        cut = [s for s in seqs if b.model.rows[s] > 200]
        if cut:
            b.pool.free(i32(cut, gpu))
            b.model.free(cut, None)


@pytest.mark.parametrize("shape", ["random", "chain", "star", "roots"])
def test_accept(gpu, shape):
    rng = random.Random(shape)
    b = Both(gpu, 400, 16, 12, 20, 2)
    seqs = list(range(12))
    for step in range(6):
        some = rng.sample(seqs, rng.randrange(1, 12))
        sizes = [rng.choice([0, 1, 3, 8, 20, 64, 65, 130]) for _ in some]
        b.extend(some, sizes)
        trees = [random_tree(rng, n, shape) for n in sizes]
        few = 3 if step % 2 else 40   # tokens: siblings that are the same, or hardly
        tokens = [[rng.randrange(few) for _ in range(n)] for n in sizes]
        targets = [[rng.randrange(few) if rng.random() < 0.4 else -1 if rng.random() < 0.1 else
                    next((k[c] for c in range(v + 1, n) if t[c] == v), 5) for v in range(n)] for n, t, k in zip(sizes, trees, tokens)]
        flat = lambda xs: i32([v for x in xs for v in x], gpu)
        path, n_path, following = b.pool.accept(i32(some, gpu), i32(starts(sizes), gpu), flat(trees), flat(tokens), flat(targets))
        want = [walk(t, k, y) for t, k, y in zip(trees, tokens, targets)]
        assert path.tolist() == [v for (p, _), n in zip(want, sizes) for v in p + [-1] * (n - len(p))]
        assert n_path.tolist() == [len(p) for p, _ in want] and following.tolist() == [y for _, y in want]
        assert keep_model(b.model, some, sizes, [p for p, _ in want]) == 0
        b.check()
        if step == 3:
            b.pool.free(i32(seqs, gpu))
            b.model.free(seqs, None)


def test_the_largest_tree_and_all_jobs(gpu):
    from ds4cuda_amd import pages
    b = Both(gpu, 1100, 1, 1, 1060, 1)
    b.extend([0], [1029])
    tree, tokens = [i - 1 for i in range(1024)], list(range(1024))
    got = b.pool.accept(i32([0], gpu), i32([0, 1024], gpu), i32(tree, gpu), i32(tokens, gpu), i32(list(range(1, 1025)), gpu))
    assert got[0].tolist() == tokens and got[1].item() == 1024 and got[2].item() == 1024
    b.check()
    n = pages.MAX_JOBS
    b = Both(gpu, 2 * n, 4, n, 3, 1)
    seqs = list(range(n))
    random.Random(1).shuffle(seqs)
    b.extend(seqs, [3] * n)
    paths = [[0, 2] if s % 3 else [1] for s in seqs]
    b.pool.keep(i32(seqs, gpu), i32(starts([3] * n), gpu), i32(packed(paths, [3] * n), gpu), i32([len(p) for p in paths], gpu))
    assert keep_model(b.model, seqs, [3] * n, paths) == 0
    b.check()


@pytest.mark.parametrize("sizes", [[500] * 9, [1024] * 3 + [0, 1, 1023], [4096 // 64] * 64, [63] * 65 + [2]])
def test_many_nodes(gpu, sizes):
    """Around the number of nodes up to which the planning workgroup walks the trees itself (4096)."""
    rng = random.Random(sum(sizes))
    n = len(sizes)
    b = Both(gpu, sum(sizes) // 16 + 3 * n, 16, n, 70, 1)
    seqs = list(range(n))
    rng.shuffle(seqs)
    b.extend(seqs, [rng.randrange(1, 20) for _ in seqs])
    b.extend(seqs, sizes)
    trees = [random_tree(rng, k, rng.choice(["random", "chain", "star"])) for k in sizes]
    tokens = [[rng.randrange(4) for _ in range(k)] for k in sizes]
    targets = [[rng.randrange(4) for _ in range(k)] for k in sizes]
    flat = lambda xs: i32([v for x in xs for v in x], gpu)
    path, n_path, following = b.pool.accept(i32(seqs, gpu), i32(starts(sizes), gpu), flat(trees), flat(tokens), flat(targets))
    want = [walk(t, k, y) for t, k, y in zip(trees, tokens, targets)]
    assert path.tolist() == [v for (p, _), k in zip(want, sizes) for v in p + [-1] * (k - len(p))]
    assert n_path.tolist() == [len(p) for p, _ in want] and following.tolist() == [y for _, y in want]
    assert keep_model(b.model, seqs, sizes, [p for p, _ in want]) == 0
    b.check()


def test_trees_that_lie_over_each_other(gpu):
    """A q_start that goes back names nodes twice: refused, whatever the nodes' links would make of it."""
    from ds4cuda_amd import Ds4HipError
    for nodes in (9, 5000):
        b = Both(gpu, 600, 16, 3, 400, 1)
        b.extend([0, 1, 2], [40, 40, 40])
        for q in ([0, 5, 2, 6], [0, 9, 0, 9], [3, 9, 1, 8], [nodes, 0, 5, 7], [0, nodes, 0, nodes]):
            x = i32([-1] + list(range(nodes - 1)), gpu)
            path, n_path, following = b.pool.accept(i32([0, 1, 2], gpu), i32(q, gpu), x, torch.zeros_like(x), torch.zeros_like(x))
            with pytest.raises(Ds4HipError) as e:
                b.pool.check()
            assert e.value.code == -22
            assert (path == -1).all() and n_path.tolist() == [0] * 3 and following.tolist() == [-1] * 3
            b.check()


def test_refused_calls_change_nothing(gpu):
    from ds4cuda_amd import Ds4HipError
    b = Both(gpu, 60, 8, 6, 8, 2)
    b.extend([0, 1, 2], [13, 16, 20])
    b.pool.fork(i32([1], gpu), i32([4], gpu))   # two full pages that 1 and 4 hold both
    b.model.fork([1], [4], None, False)
    b.extend([0, 1], [5, 4])

    def refused(fn, *args):
        out = fn(*args)
        with pytest.raises(Ds4HipError) as e:
            b.pool.check()
        assert e.value.code == -22
        b.check()
        return out
    keep = lambda s, q, p, n: b.pool.keep(i32(s, gpu), i32(q, gpu), i32(p, gpu), i32(n, gpu))
    good = ([0, 1], [0, 5, 9], [0, 2, 4, 9, 9, 1, 3, 9, 9], [3, 2])
    for s, q, p, n in (([0, 0], *good[1:]), ([0, 6], *good[1:]), ([-1, 1], *good[1:]),
                       ([0, 1], [0, 5, 10], *good[2:]), ([0, 1], [-1, 5, 9], *good[2:]), ([0, 1], [5, 0, 9], *good[2:]),
                       (*good[:2], [0, 0, 4, 9, 9, 1, 3, 9, 9], [3, 2]), (*good[:2], [2, 0, 4, 9, 9, 1, 3, 9, 9], [3, 2]),
                       (*good[:2], [0, 2, 5, 9, 9, 1, 3, 9, 9], [3, 2]), (*good[:2], [0, 2, 4, 9, 9, -1, 3, 9, 9], [3, 2]),
                       (*good[:3], [6, 2]), (*good[:3], [3, -1]), ([0, 3], *good[1:]),
                       ([0, 4], [0, 5, 9], *good[2:])):   # (4 holds its last page with 1)
        refused(keep, s, q, p, n)
    accept = lambda s, q, n: b.pool.accept(i32(s, gpu), i32(q, gpu), i32([-1] * n, gpu), i32([0] * n, gpu), i32([0] * n, gpu))
    for s, q in (([0, 0], [0, 5, 9]), ([0, 4], [0, 5, 9]), ([0, 1], [0, 5, 8192]), ([0, 1], [3, 2, 9]), ([3, 1], [0, 5, 9])):
        path, n_path, following = refused(accept, s, q, 9)
        assert path.tolist() == [-1] * 9 and n_path.tolist() == [0, 0] and following.tolist() == [-1, -1]
    keep(*good)
    assert keep_model(b.model, [0, 1], [5, 4], [[0, 2, 4], [1, 3]]) == 0
    b.check()
    # nodes that no job names
    b.extend([2], [3])
    path, n_path, following = b.pool.accept(i32([2], gpu), i32([2, 5], gpu), i32([9, 9, -1, 0, 0, 9, 9], gpu),
                                            i32([1, 1, 1, 6, 7, 1, 1], gpu), i32([1, 1, 7, 1, 8, 1, 1], gpu))
    assert path.tolist() == [-1, -1, 0, 2, -1, -1, -1] and n_path.tolist() == [2] and following.tolist() == [8]
    assert keep_model(b.model, [2], [3], [[0, 2]]) == 0
    b.check()


def test_refusals_of_the_python_calls(gpu):
    from ds4cuda_amd import Ds4HipError
    b = Both(gpu, 20, 8, 3, 4, 1)
    b.extend([0], [9])
    x = lambda n: torch.zeros(n, dtype=torch.int32, device=gpu)
    for fn in (lambda: b.pool.keep(x(1), x(3), x(4), x(1)), lambda: b.pool.keep(x(1), x(2), x(4), x(2)),
               lambda: b.pool.keep(x(1), x(2), x(4).long(), x(1)), lambda: b.pool.keep(x(1), x(2), x(4).cpu(), x(1)),
               lambda: b.pool.accept(x(1), x(2), x(4), x(3), x(4)), lambda: b.pool.accept(x(1), x(2), x(8)[::2], x(4), x(4)),
               lambda: b.pool.accept(x(1), x(1), x(4), x(4), x(4)), lambda: b.pool.accept(x(1), x(2), x(4), x(4), x(4), path=x(3)),
               lambda: b.pool.accept(x(1025), x(1026), x(4), x(4), x(4))):
        with pytest.raises(Ds4HipError) as e:
            fn()
        assert e.value.code == -22
    b.check()


def test_steps_of_a_loop(gpu):
    """Steps as a serving loop makes them, eager and captured: extend, append, attention of the trees, a token behind
    every node, the path accepted. What stays in the pool is what a sequence without drafts would hold."""
    from ds4cuda_amd import ops, pages
    rng = random.Random(40)
    n, heads, vocab, page, seqs = 7, 64, 500, 16, [1, 0, 2]
    total = n * len(seqs)
    gen = torch.Generator(gpu).manual_seed(41)
    embed = torch.randn((vocab, 512), generator=gen, device=gpu)          # a token's row, at any position
    head = torch.randn((512, vocab), generator=gen, device=gpu)

    def make():
        pool = pages.PagePool.empty(80, page, 3, 320, 1, gpu)
        dst = pool.extend(i32(seqs, gpu), i32([30, 17, 64], gpu), 111)
        pool.append(torch.randn((111, 512), generator=torch.Generator(gpu).manual_seed(42), device=gpu), dst)
        return pool
    pool, other = make(), make()
    ids, n_new, q_start = i32(seqs, gpu), i32([n] * 3, gpu), i32(starts([n] * 3), gpu)
    tokens, parents, u = i32([0] * total, gpu), i32([-1] * total, gpu), torch.zeros(total, device=gpu)

    def step(p):
        rows = embed[tokens.long()]
        dst = p.extend(ids, n_new, total)
        p.append(rows, dst)
        q = rows[:, None].expand(total, heads, 512).to(torch.bfloat16).contiguous()
        x = p.attend_tree(q, parents, seqs=ids, q_start=q_start, window=40, n_first=2)
        logits = x.float().mean(1) @ head
        targets, probs = ops.sample_tokens(logits, u, temperature=0.7, top_k=3)
        return (logits, targets, probs, *p.accept(ids, q_start, parents, tokens, targets))

    def draft(i):
        trees = [random_tree(rng, n, "random") for _ in seqs]
        parents.copy_(i32([v for t in trees for v in t], gpu))
        tokens.copy_(i32([rng.randrange(vocab) for _ in range(total)], gpu))
        u.copy_(torch.rand(total, generator=torch.Generator(gpu).manual_seed(50 + i), device=gpu))
        return trees
    torch.cuda.synchronize()
    trees = draft(0)
    step(pool), step(other)
    pool.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(pool)
    for i in range(1, 6):
        trees = draft(i)
        # what the model says does not depend on the drafted tokens' children: let some children be it
        known = step_targets(other, embed, head, tokens, parents, u, ids, n_new, q_start, total, heads)
        mine = tokens.tolist()
        for s, t in enumerate(trees):
            for v in range(n - 1, 0, -1):
                if rng.random() < 0.5 and t[v] == 0:
                    mine[s * n + v] = known[s * n]
        tokens.copy_(i32(mine, gpu))
        rows_before = pool.rows.tolist()
        graph.replay()
        want = step(other)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
        for name in ("refs", "rows"):
            assert torch.equal(getattr(pool, name), getattr(other, name))
        logits, targets, probs, path, n_path, following = (t.cpu() for t in want)
        for v in range(total):
            token, prob = sample_64(logits[v].numpy(), 0.7, 3, 1.0, 0.0, float(u[v]))
            assert token == int(targets[v]) and abs(prob - float(probs[v])) <= 2.0 ** -23.9 * prob
        for s, t in enumerate(trees):
            line, nxt = walk(t, mine[s * n:s * n + n], targets[s * n:s * n + n].tolist())
            assert path[s * n:s * n + n].tolist() == line + [-1] * (n - len(line)) and int(following[s]) == nxt
            base = rows_before[seqs[s]]
            assert int(pool.rows[seqs[s]]) == base + len(line)
            # the rows that stay are those of the accepted tokens
            r = torch.arange(base, base + len(line), device=gpu)
            at = pool.table[seqs[s]].long()[r // page] * page + r % page
            plain = ops.Fp8KVCache.empty(len(line), gpu)
            plain.append(embed[torch.tensor([mine[s * n + v] for v in line], device=gpu)])
            assert torch.equal(pool.codes[0, at], plain.codes) and torch.equal(pool.sexp[0, at], plain.sexp)
            assert torch.equal(pool.tail[0, at].view(torch.int16), plain.tail)
    pool.check()
    other.check()


def step_targets(pool, embed, head, tokens, parents, u, ids, n_new, q_start, total, heads):
    """The tokens behind every node, with the pool left as it was."""
    from ds4cuda_amd import ops
    before = pool.rows[ids.long()].clone()
    rows = embed[tokens.long()]
    dst = pool.extend(ids, n_new, total)
    pool.append(rows, dst)
    q = rows[:, None].expand(total, heads, 512).to(torch.bfloat16).contiguous()
    x = pool.attend_tree(q, parents, seqs=ids, q_start=q_start, window=40, n_first=2)
    targets, _ = ops.sample_tokens(x.float().mean(1) @ head, u, temperature=0.7, top_k=3)
    pool.free(ids, before)
    return targets.tolist()
