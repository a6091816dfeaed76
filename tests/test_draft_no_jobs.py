"""A call for accepted paths that has nodes and no jobs (a padded batch of which no sequence takes part)."""
import ctypes as C

import pytest
import torch

from test_pages_host import BIG, X, pool


def test_needs_the_path_it_writes():
    from ds4cuda_amd import lib
    p = C.byref(pool())
    assert lib().ds4hip_kv_pages_accept(p, X, X, 0, X, X, X, 4, None, X, X, X, BIG, None) == -22


@pytest.mark.gpu
@pytest.mark.parametrize("nodes", [0, 1, 255, 257, 5000])
def test_every_node_is_no_jobs(gpu, nodes):
    from test_gpu_draft_keep import Both, i32
    b = Both(gpu, 20, 8, 3, 4, 1)
    b.extend([0], [9])
    none, x = i32([], gpu), i32([0] * nodes, gpu)
    whole = torch.full((nodes + 600,), 77, dtype=torch.int32, device=gpu)
    path, n_path, following = b.pool.accept(none, i32([0], gpu), x, x, x, path=whole[300:300 + nodes])
    assert (path == -1).all() and (whole[:300] == 77).all() and (whole[300 + nodes:] == 77).all()
    assert n_path.numel() == following.numel() == 0
    path, _, _ = b.pool.accept(none, i32([0], gpu), x, x, x)
    assert path.tolist() == [-1] * nodes
    b.check()
