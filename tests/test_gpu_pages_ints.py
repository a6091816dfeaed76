"""Integer arguments past 32 bits are refused by the Python calls of the paged cache and its attention, not cut
to another value."""
import pytest
import torch

CUT = [(1 << 32) + 5, 1 << 32, 1 << 31, -(1 << 32) + 1]


def refused(fn, *a, **kw):
    from ds4cuda_amd import Ds4HipError
    with pytest.raises(Ds4HipError) as e:
        fn(*a, **kw)
    assert e.value.code == -22


@pytest.mark.parametrize("n", CUT)
def test_workspace_sizes_and_page_rows(n):
    from ds4cuda_amd import ops
    for args in ((n, 5, 64), (2, n, 64), (2, 5, n)):
        refused(ops.window_workspace_bytes, *args)
    table = torch.zeros((2, 4), dtype=torch.int32)
    refused(ops.WindowView, None, table, table[:, 0], n)


@pytest.mark.gpu
@pytest.mark.parametrize("n", CUT)
def test_calls(gpu, n):
    from ds4cuda_amd import pages
    pool = pages.PagePool.empty(4, 16, 2, 32, 1, gpu)
    one = torch.ones(1, dtype=torch.int32, device=gpu)
    kv = torch.ones((1, 512), device=gpu)
    dst = pool.extend(one, one, 1)
    refused(pool.extend, one, one, n)
    refused(pool.extend, one, one, n, dst_rows=dst)
    refused(pool.append, kv, dst, layer=n)
    q = torch.ones((1, 64, 512), dtype=torch.bfloat16, device=gpu)
    refused(pool.attend, q, seqs=one, window=n)
    refused(pool.attend, q, seqs=one, n_first=n)
    torch.cuda.synchronize()
    assert int(pool.rows[1]) == 1 and not pool.codes.any()
    pool.append(kv, dst)
    assert torch.isfinite(pool.attend(q, seqs=one, window=(1 << 31) - 1, n_first=(1 << 31) - 1)).all()
    pool.check()
