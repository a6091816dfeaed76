"""The page calls' workspace: the size that fork and compact have always taken is enough for all of them."""
import ctypes as C

import pytest
import torch

from test_pages_host import pool

GUARD = 4096   # bytes before and after


@pytest.mark.parametrize("n_pages", [1, 4, 63, 4096])
def test_size(n_pages):
    from ds4cuda_amd import lib
    p = pool(n_pages=n_pages, layer_rows=16 * n_pages)
    assert lib().ds4hip_kv_pages_workspace_bytes(C.byref(p)) == 4 * (64 + 4 * n_pages)


@pytest.mark.gpu
@pytest.mark.parametrize("jobs", [3, 1024])
def test_calls_stay_inside(gpu, jobs):
    """A pool of few pages and many sequences, most of which hold nothing: every call between guards."""
    from draft_check import keep_model
    from test_gpu_draft_keep import Both, i32, packed, starts
    b = Both(gpu, 9, 4, 1100, 3, 2)
    need = 4 * (64 + 4 * 9)
    whole = torch.full((need + 2 * GUARD,), 0xA5, dtype=torch.uint8, device=gpu)
    b.pool._workspace, b.pool._ws_args = whole, (whole.data_ptr() + GUARD, need)
    b.extend([5, 700, 2], [6, 3, 1])
    some = [700, 5, 2] + [s for s in range(10, 1040) if s != 700][:jobs - 3]
    for accept in (False, True):
        sizes = [4, 2, 3] + [0] * (jobs - 3)
        b.extend(some[:3], sizes[:3])
        paths = [[0, 2], [0], [0, 2]] + [[]] * (jobs - 3)
        if accept:
            tree, tokens, targets = [-1, 0, 0, 1, -1, 0, -1, 0, 0], [1, 2, 3, 4, 1, 9, 1, 5, 6], [3, 0, 0, 0, 1, 0, 6, 0, 0]
            got = b.pool.accept(i32(some, gpu), i32(starts(sizes), gpu), i32(tree, gpu), i32(tokens, gpu), i32(targets, gpu))
            assert got[0].tolist() == [v for p, n in zip(paths, sizes) for v in p + [-1] * (n - len(p))]
        else:
            b.pool.keep(i32(some, gpu), i32(starts(sizes), gpu), i32(packed(paths, sizes), gpu), i32([len(p) for p in paths], gpu))
        assert keep_model(b.model, some, sizes, paths) == 0
        b.check()
    b.pool.free(i32([5], gpu))
    b.model.free([5], None)
    b.pool.fork(i32([700], gpu), i32([5], gpu))
    b.model.fork([700], [5], None, False)
    b.check()
    b.pool.free(i32([2], gpu))
    b.pool.compact()
    b.pool.check()
    assert (whole[:GUARD] == 0xA5).all() and (whole[-GUARD:] == 0xA5).all()
