"""Page calls of many jobs that a table of a late or an early job makes the device refuse: all waves of
the planning workgroup take the same way, nothing changes, and the pool goes on."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("n", [3, 64, 65, 1024])
def test_one_bad_table_among_many_jobs(gpu, n):
    from ds4cuda_amd import Ds4HipError, pages
    rows = [5 + (3 * i) % 24 for i in range(n)]
    pool = pages.PagePool.empty(8 * n, 4, 2 * n, 40, 1, gpu)
    seqs, kids = i32(range(n), gpu), i32(range(n, 2 * n), gpu)
    pool.extend(seqs, i32(rows, gpu), sum(rows))
    pool.check()
    for bad in sorted({0, 1, n // 2, n - 1}):
        good = int(pool.table[bad, 1])
        for entry in (-1, 8 * n, int((pool.refs == 0).nonzero()[-1])):   # none, outside, a free page
            pool.table[bad, 1] = entry
            before = pool.refs.clone(), pool.rows.clone(), pool.table[:n].clone()
            for call in (lambda: pool.free(seqs), lambda: pool.fork(seqs, kids), lambda: pool.fork(seqs, kids, deep=True),
                         lambda: pool.free(seqs, i32([1] * n, gpu))):
                call()
                with pytest.raises(Ds4HipError) as e:
                    pool.check()
                assert e.value.code == -22
                assert torch.equal(pool.refs, before[0]) and torch.equal(pool.rows, before[1])
                assert torch.equal(pool.table[:n], before[2])
        pool.table[bad, 1] = good
    pool.fork(seqs, kids)
    pool.check()
    assert pool.rows.tolist() == rows + rows
    pool.free(seqs)
    pool.free(kids)
    pool.check()
    assert not pool.refs.any() and not pool.rows.any()


def test_more_jobs_than_a_call_takes(gpu):
    from ds4cuda_amd import Ds4HipError, pages
    n = pages.MAX_JOBS + 1
    pool = pages.PagePool.empty(8, 4, 2 * n, 40, 1, gpu)
    seqs, kids = i32(range(n), gpu), i32(range(n - 1, 2 * n - 1), gpu)
    for call in (lambda: pool.extend(seqs, seqs, 4), lambda: pool.fork(seqs, kids), lambda: pool.free(seqs)):
        with pytest.raises(Ds4HipError, match="1024 sequences at most") as e:
            call()
        assert e.value.code == -22
    pool.check()
    pool.free(seqs[:-1])
    pool.check()
