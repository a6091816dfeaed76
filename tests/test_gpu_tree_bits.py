"""Trees' outputs to the bit: chains where nothing is cut, and calls repeated with others in between."""
import random

import pytest
import torch

from draft_check import random_tree
from test_gpu_tree_attn import run
from test_gpu_window_attn import Batch, i32, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
@pytest.mark.parametrize("heads", [8, 64, 128])
@pytest.mark.parametrize("rows,new", [([40], [1]), ([300, 33, 64], [20, 1, 30]), ([128, 97], [32, 33]), ([350, 350], [1, 2])])
def test_uncut_chains_are_prompts(gpu, rows, new, heads, typ):
    """Without a window both have the same tiles in the same order, and short problems that a workgroup each has are
    cut in neither: the same bits."""
    from ds4cuda_amd import ops
    b = Batch(gpu, rows, 16, sum(rows))
    q = queries(gpu, sum(new), heads, typ, heads)
    sinks = torch.randn(heads, device=gpu)
    start = i32([sum(new[:i]) for i in range(len(new) + 1)], gpu)
    trees = run(b, q, [random_tree(None, n, "chain") for n in new], 0, 0, sinks)
    prompts = ops.flash_attn_window_fp8(q, b.cache, b.table, b.seq_rows, page_rows=16, sinks=sinks, q_start=start)
    assert torch.equal(trees, prompts)


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
@pytest.mark.parametrize("heads,window", [(8, 0), (64, 0), (64, 128)])
def test_a_call_repeats_itself(gpu, heads, window, typ):
    rng = random.Random(heads + window)
    calls = []
    for rows, new in (([9000, 60, 700], [12, 3, 40]), ([500, 800], [24, 1]), ([3000] * 6, [9] * 6)):
        b = Batch(gpu, rows, 64, len(rows))
        calls.append((b, queries(gpu, sum(new), heads, typ, 5), [random_tree(rng, n, "random") for n in new]))
    first = [run(*c, window, 3) for c in calls]
    for _ in range(4):
        for i in rng.sample(range(3), 3):
            assert torch.equal(run(*calls[i], window, 3), first[i])
