"""Kept rows in pools of many layers and calls of many trees, where a workgroup moves several layers at once: against the
model, to the bit. A job's layers go to 512 / jobs workgroups, which take as many at once as make 64 rows."""
import random

import pytest

from draft_check import keep_model, random_tree, walk
from test_gpu_draft_keep import Both, i32, packed, random_path, starts

pytestmark = pytest.mark.gpu

SIZES = [(64, 43, 16, 20), (64, 43, 4, 7), (300, 3, 4, 9), (40, 43, 64, 150), (100, 11, 16, 70), (1000, 5, 2, 5), (1, 43, 16, 200)]


@pytest.mark.parametrize("jobs,layers,page,most", SIZES)
def test_keep(gpu, jobs, layers, page, most):
    """Paths of 0 to `most` rows, from one row that moves to all of them."""
    rng = random.Random(jobs + layers)
    n_seqs = jobs + 3
    entries = (2 * most + 20) // page + 3
    b = Both(gpu, n_seqs * ((most + 20) // page + 2), page, n_seqs, entries, layers)
    seqs = rng.sample(range(n_seqs), jobs)
    b.extend(seqs, [rng.randrange(1, 12) for _ in seqs])
    sizes = [rng.choice([1, 2, most // 2 + 1, most - 1, most]) for _ in seqs]
    sizes[0] = most
    b.extend(seqs, sizes)
    paths = [random_path(rng, n) for n in sizes]
    paths[0] = list(range(1, most))   # every row moves by one
    if jobs > 1:
        paths[1] = list(range(sizes[1]))   # none does
    b.pool.keep(i32(seqs, gpu), i32(starts(sizes), gpu), i32(packed(paths, sizes), gpu), i32([len(p) for p in paths], gpu))
    assert keep_model(b.model, seqs, sizes, paths) == 0
    b.check()


@pytest.mark.parametrize("jobs,layers,page,most", SIZES)
def test_accept(gpu, jobs, layers, page, most):
    rng = random.Random(7 * jobs + layers)
    entries = (2 * most + 20) // page + 3
    b = Both(gpu, jobs * ((most + 20) // page + 2), page, jobs, entries, layers)
    seqs = list(range(jobs))
    rng.shuffle(seqs)
    b.extend(seqs, [rng.randrange(1, 12) for _ in seqs])
    sizes = [rng.randrange(1, most + 1) for _ in seqs]
    sizes[0] = most
    b.extend(seqs, sizes)
    trees = [random_tree(rng, n, "random") for n in sizes]
    tokens = [[rng.randrange(50) for _ in range(n)] for n in sizes]
    # most targets are a child's token, so that paths are long
    targets = [[next((k[c] for c in range(n - 1, v, -1) if t[c] == v), -1) if rng.random() < 0.95 else 51 for v in range(n)]
               for n, t, k in zip(sizes, trees, tokens)]
    flat = lambda xs: i32([v for x in xs for v in x], gpu)
    path, n_path, following = b.pool.accept(i32(seqs, gpu), i32(starts(sizes), gpu), flat(trees), flat(tokens), flat(targets))
    want = [walk(t, k, y) for t, k, y in zip(trees, tokens, targets)]
    assert path.tolist() == [v for (p, _), n in zip(want, sizes) for v in p + [-1] * (n - len(p))]
    assert n_path.tolist() == [len(p) for p, _ in want] and following.tolist() == [y for _, y in want]
    assert keep_model(b.model, seqs, sizes, [p for p, _ in want]) == 0
    b.check()
