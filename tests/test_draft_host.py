"""Refusals on the host of the operators over drafted trees and of sampling: no GPU needed."""
import ctypes as C

import pytest
import torch

from test_pages_host import BAD_POOLS, BIG, X, attn, pool


@pytest.mark.parametrize("kw", BAD_POOLS)
def test_pools_that_do_not_fit(kw):
    from ds4cuda_amd import lib
    p = C.byref(pool(**kw))
    assert lib().ds4hip_kv_pages_keep(p, X, X, 1, X, 4, X, X, BIG, None) == -22
    assert lib().ds4hip_kv_pages_accept(p, X, X, 1, X, X, X, 4, X, X, X, X, BIG, None) == -22


def test_keep_and_accept():
    from ds4cuda_amd import lib
    l, p = lib(), C.byref(pool())
    need = l.ds4hip_kv_pages_workspace_bytes(p)
    keep = dict(seqs=X, q_start=X, n_jobs=1, path=X, n_nodes=4, n_path=X, ws=X, size=BIG)
    bad = [dict(seqs=None), dict(q_start=None), dict(n_path=None), dict(path=None), dict(n_jobs=-1), dict(n_jobs=1025),
           dict(n_nodes=-1), dict(n_nodes=(1 << 24) + 1), dict(ws=None), dict(ws=X + 4), dict(size=need - 1)]
    for kw in bad:
        assert l.ds4hip_kv_pages_keep(p, *{**keep, **kw}.values(), None) == -22
    accept = dict(seqs=X, q_start=X, n_jobs=1, parents=X, tokens=X, targets=X, n_nodes=4, path=X, n_path=X, next=X, ws=X,
                  size=BIG)
    for kw in bad + [dict(parents=None), dict(tokens=None), dict(targets=None), dict(next=None)]:
        assert l.ds4hip_kv_pages_accept(p, *{**accept, **kw}.values(), None) == -22
    # nothing to do: no launch
    assert l.ds4hip_kv_pages_keep(p, None, None, 0, None, 0, None, None, 0, None) == 0
    assert l.ds4hip_kv_pages_accept(p, None, None, 0, None, None, None, 0, None, None, None, None, 0, None) == 0


@pytest.mark.parametrize("kw", [dict(q=None), dict(out=None), dict(codes=None), dict(table=None), dict(rows=None), dict(io_f32=2),
                                dict(n_slots=1), dict(page_rows=48), dict(n_seqs=4097), dict(n_q=(1 << 24) + 1),
                                dict(n_head=48), dict(window=-1), dict(n_first=-1), dict(q=X + 8), dict(out=X + 8),
                                dict(q_start=None, n_q=1)])
def test_tree_attention_refuses(kw):
    from ds4cuda_amd import lib
    assert lib().ds4hip_flash_attn_tree_fp8(C.byref(attn(**kw)), X, X, BIG, None) == -22


def test_tree_attention_parents_and_workspace():
    from ds4cuda_amd import lib
    l, a = lib(), C.byref(attn())
    need = l.ds4hip_flash_attn_window_fp8_workspace_bytes(2, 5, 64)
    assert l.ds4hip_flash_attn_tree_fp8(a, None, X, need, None) == -22
    assert l.ds4hip_flash_attn_tree_fp8(a, X, X, need - 1, None) == -22
    assert l.ds4hip_flash_attn_tree_fp8(a, X, None, need, None) == -22
    assert l.ds4hip_flash_attn_tree_fp8(a, X, X + 8, need, None) == -22
    assert l.ds4hip_flash_attn_tree_fp8(None, X, X, need, None) == -22
    assert l.ds4hip_flash_attn_tree_fp8(C.byref(attn(n_q=0)), None, None, 0, None) == 0
    assert l.ds4hip_flash_attn_tree_fp8(C.byref(attn(n_seqs=0)), None, None, 0, None) == 0


def test_sampling():
    from ds4cuda_amd import lib
    from ds4cuda_amd.ops import Sample
    l = lib()
    size = l.ds4hip_sample_workspace_bytes

    def call(ws=X, nbytes=BIG, **kw):
        a = dict(logits=X, logits_f32=0, row_stride=100, n_rows=3, n_vocab=100, u=X, tokens=X, probs=X, all_temperature=1.0,
                 all_top_p=1.0)
        a.update(kw)
        return l.ds4hip_sample_tokens(C.byref(Sample(**a)), ws, nbytes, None)
    for kw in (dict(logits=None), dict(u=None), dict(tokens=None), dict(probs=None), dict(logits_f32=2), dict(row_stride=99),
               dict(n_rows=-1), dict(n_rows=65537), dict(n_vocab=0), dict(n_vocab=-5), dict(n_vocab=262145, row_stride=1 << 20),
               dict(logits=X + 1), dict(logits=X + 2, logits_f32=1), dict(ws=None), dict(ws=X + 4), dict(nbytes=size(3, 100) - 1)):
        assert call(**kw) == -22, kw
    assert l.ds4hip_sample_tokens(None, X, BIG, None) == -22
    assert call(n_rows=0, logits=None, ws=None) == 0
    assert [size(*a) for a in ((0, 5), (65537, 5), (2, 0), (2, 262145))] == [0] * 4
    for rows in (1, 7, 300):
        for vocab in (1, 8192, 8193, 129280):
            assert all(0 < size(r, v) <= size(rows, vocab) for r in (1, rows) for v in (1, (vocab + 1) // 2, vocab))


def test_python_refuses_host_tensors_and_shapes():
    from ds4cuda_amd import Ds4HipError, ops
    f, i = torch.zeros, lambda *s: torch.zeros(s, dtype=torch.int32)
    for x in (f(2, 10), f(10), f(2, 10, dtype=torch.float16)):
        with pytest.raises(Ds4HipError) as e:
            ops.sample_tokens(x, f(2))
        assert e.value.code == -22
    cache = ops.Fp8KVCache(torch.zeros((64, 448), dtype=torch.uint8), torch.zeros((64, 8), dtype=torch.int8),
                           torch.zeros((64, 64), dtype=torch.int16))
    with pytest.raises(Ds4HipError):
        ops.flash_attn_tree_fp8(f(2, 64, 512), i(2), cache, i(2, 4), i(2), page_rows=16)


def test_workspace_sizes_of_any_integers():
    import numpy as np
    from ds4cuda_amd import ops
    n = torch.tensor(4)
    for f, rest in ((ops.window_workspace_bytes, (64, 64)), (ops.sample_workspace_bytes, (4096,))):
        sizes = []
        for k in (4, 4000):
            n.fill_(k)   # (the same tensor with another value)
            sizes.append(f(n, *rest))
            assert sizes[-1] == f(k, *rest) == f(np.array(k), *rest) > 0
        assert sizes[0] < sizes[1]
