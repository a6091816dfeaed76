"""A page pool whose first fork is captured into a graph."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def test_a_first_fork_inside_a_capture(gpu):
    """The workspace that the pool takes on its first fork may come from a graph's memory: it stays the
    pool's when the graph is gone."""
    import gc
    from ds4cuda_amd import pages
    pool = pages.PagePool.empty(40, 16, 8, 64, 1, gpu)
    a, b, c = i32([0], gpu), i32([1], gpu), i32([2], gpu)
    pool.extend(a, i32([37], gpu), 37)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pool.fork(a, b)
        pool.free(b)
    for _ in range(3):
        g.replay()
        pool.fork(a, c, deep=True)
        pool.check()
        assert pool.rows[:3].tolist() == [37, 0, 37] and pool.table[2, :3].tolist() == [3, 4, 5]
        pool.free(c)
    del g
    gc.collect()
    torch.cuda.empty_cache()
    junk = [torch.full((1 << 20,), 0xFF, dtype=torch.uint8, device=gpu) for _ in range(64)]
    pool.fork(a, c)
    for j in junk:
        j.fill_(1)
    pool.fork(a, b, deep=True)
    pool.check()
    assert pool.rows[:3].tolist() == [37, 37, 37]
    assert int(pool.compact()) == 7
    pool.check()
