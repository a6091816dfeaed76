"""Accepted paths with starts of any value: refused, with nothing written outside the outputs."""
import pytest
import torch

from test_gpu_draft_keep import Both, i32

pytestmark = pytest.mark.gpu

LOW, HIGH = -(1 << 31), (1 << 31) - 1
GUARD = 2048   # entries before and after


def guarded(n, gpu):
    whole = torch.full((n + 2 * GUARD,), 77, dtype=torch.int32, device=gpu)
    return whole[GUARD:GUARD + n], whole


@pytest.mark.parametrize("nodes", [9, 4096, 4097, 5000])
def test_starts_near_the_ends_of_32_bits(gpu, nodes):
    from ds4cuda_amd import Ds4HipError
    b = Both(gpu, 600, 16, 3, 400, 1)
    b.extend([0, 1, 2], [40, 40, 40])
    seqs, parents, zeros = i32([0, 1, 2], gpu), i32([-1] + list(range(nodes - 1)), gpu), i32([0] * nodes, gpu)
    for q in ([HIGH, LOW, 3, 9], [HIGH - 3, LOW + 600, LOW + 900, HIGH], [0, 3, 6, HIGH], [0, 3, 6, HIGH - 700],
              [LOW, 3, 6, 9], [LOW + 5, LOW + 9, 0, 9], [0, HIGH, LOW, 9], [HIGH, HIGH, HIGH, HIGH], [LOW, LOW, LOW, LOW],
              [nodes + 1, nodes + 2, nodes + 3, nodes + 4], [0, 3, 6, 1 << 30]):
        outs = [guarded(n, gpu) for n in (nodes, 3, 3)]
        (path, _), (n_path, _), (following, _) = outs
        b.pool.accept(seqs, i32(q, gpu), parents, zeros, zeros, path=path, n_path=n_path, next=following)
        with pytest.raises(Ds4HipError) as e:
            b.pool.check()
        assert e.value.code == -22, q
        assert (path == -1).all() and n_path.tolist() == [0] * 3 and following.tolist() == [-1] * 3, q
        for _, whole in outs:
            assert (whole[:GUARD] == 77).all() and (whole[-GUARD:] == 77).all(), q
        b.check()
