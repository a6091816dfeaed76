"""The page pool's and the windowed attention's refusals on the host: no GPU needed."""
import ctypes as C

import pytest
import torch

X, BIG = 4096, 1 << 40   # a stand-in address (never followed) and a workspace that is large enough


def pool(**kw):
    from ds4cuda_amd.pages import KvPages
    a = dict(codes=X, sexp=X, tail=X, layer_rows=64, n_layers=1, n_pages=4, page_rows=16, table_stride=4, n_seqs=2,
             refs=X, table=X, rows=X, status=X)
    a.update(kw)
    return KvPages(**a)


BAD_POOLS = [dict(codes=None), dict(sexp=None), dict(tail=None), dict(refs=None), dict(table=None), dict(rows=None),
             dict(status=None), dict(layer_rows=63), dict(n_layers=0), dict(n_pages=0), dict(n_pages=(1 << 28) + 1),
             dict(page_rows=0), dict(page_rows=24), dict(page_rows=-16), dict(table_stride=0), dict(n_seqs=0),
             dict(n_seqs=65537), dict(codes=X + 8), dict(tail=X + 8), dict(sexp=X + 4)]


@pytest.mark.parametrize("kw", BAD_POOLS)
def test_pools_that_do_not_fit(kw):
    from ds4cuda_amd import lib
    l, p = lib(), C.byref(pool(**kw))
    assert l.ds4hip_kv_pages_init(p, None) == -22
    assert l.ds4hip_kv_pages_extend(p, X, X, 1, X, 1, None) == -22
    assert l.ds4hip_kv_pages_append(p, 0, X, 1, X, None) == -22
    assert l.ds4hip_kv_pages_fork(p, X, X, None, 1, 0, X, BIG, None) == -22
    assert l.ds4hip_kv_pages_free(p, X, None, 1, None) == -22
    assert l.ds4hip_kv_pages_compact(p, X, X, BIG, None) == -22


def test_page_calls():
    from ds4cuda_amd import lib
    l, p = lib(), C.byref(pool())
    need = l.ds4hip_kv_pages_workspace_bytes(p)
    assert need > 0 and l.ds4hip_kv_pages_workspace_bytes(None) == 0
    assert l.ds4hip_kv_pages_init(None, None) == -22
    for seqs, n_new, n, dst, n_dst in ((None, X, 1, X, 1), (X, None, 1, X, 1), (X, X, -1, X, 1), (X, X, 1025, X, 1),
                                       (X, X, 1, None, 1), (X, X, 1, X, -1)):
        assert l.ds4hip_kv_pages_extend(p, seqs, n_new, n, dst, n_dst, None) == -22
    for layer, kv, n, dst in ((1, X, 1, X), (-1, X, 1, X), (0, None, 1, X), (0, X, -1, X), (0, X, 1, None), (0, X + 4, 1, X)):
        assert l.ds4hip_kv_pages_append(p, layer, kv, n, dst, None) == -22
    for a, b, n, deep, ws, size in ((None, X, 1, 0, X, BIG), (X, None, 1, 0, X, BIG), (X, X, 1025, 0, X, BIG), (X, X, -1, 0, X, BIG),
                                    (X, X, 1, 2, X, BIG), (X, X, 1, 0, None, BIG), (X, X, 1, 0, X, need - 1),
                                    (X, X, 1, 0, X + 4, BIG)):
        assert l.ds4hip_kv_pages_fork(p, a, b, None, n, deep, ws, size, None) == -22
    for seqs, n in ((None, 1), (X, -1), (X, 1025)):
        assert l.ds4hip_kv_pages_free(p, seqs, None, n, None) == -22
    for n_live, ws, size in ((None, X, BIG), (X, None, BIG), (X, X, need - 1), (X, X + 4, BIG)):
        assert l.ds4hip_kv_pages_compact(p, n_live, ws, size, None) == -22
    # nothing to do: no launch
    assert l.ds4hip_kv_pages_extend(p, None, None, 0, None, 0, None) == 0
    assert l.ds4hip_kv_pages_append(p, 0, None, 0, None, None) == 0
    assert l.ds4hip_kv_pages_fork(p, None, None, None, 0, 0, None, 0, None) == 0
    assert l.ds4hip_kv_pages_free(p, None, None, 0, None) == 0


def attn(**kw):
    from ds4cuda_amd.ops import WindowAttn
    a = dict(q=X, out=X, io_f32=0, sinks=None, codes=X, sexp=X, tail=X, n_cache_rows=64, table=X, rows=X, n_slots=2,
             table_stride=4, page_rows=16, q_start=X, seq_ids=None, n_seqs=2, n_q=5, n_head=64, window=0, n_first=0)
    a.update(kw)
    return WindowAttn(**a)


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(out=None), dict(codes=None), dict(sexp=None), dict(tail=None), dict(table=None), dict(rows=None),
    dict(io_f32=2), dict(n_cache_rows=15), dict(n_cache_rows=0), dict(n_slots=0), dict(n_slots=1), dict(table_stride=0),
    dict(page_rows=0), dict(page_rows=48), dict(page_rows=-16), dict(n_seqs=-1), dict(n_seqs=4097), dict(n_q=-1),
    dict(n_q=(1 << 24) + 1), dict(n_head=0), dict(n_head=4), dict(n_head=48), dict(n_head=256), dict(window=-1),
    dict(n_first=-1), dict(q=X + 8), dict(out=X + 8, io_f32=1), dict(tail=X + 8), dict(codes=X + 4), dict(sexp=X + 4),
    dict(q_start=None, n_q=1)])
def test_attention_refuses(kw):
    from ds4cuda_amd import lib
    assert lib().ds4hip_flash_attn_window_fp8(C.byref(attn(**kw)), X, BIG, None) == -22


def test_attention_workspace():
    from ds4cuda_amd import lib
    l = lib()
    size = l.ds4hip_flash_attn_window_fp8_workspace_bytes
    need = size(2, 5, 64)
    assert need > 0
    a = C.byref(attn())
    assert l.ds4hip_flash_attn_window_fp8(a, X, need - 1, None) == -22
    assert l.ds4hip_flash_attn_window_fp8(a, None, need, None) == -22
    assert l.ds4hip_flash_attn_window_fp8(a, X + 8, need, None) == -22
    assert l.ds4hip_flash_attn_window_fp8(None, X, need, None) == -22
    assert l.ds4hip_flash_attn_window_fp8(C.byref(attn(n_q=0)), None, 0, None) == 0
    assert l.ds4hip_flash_attn_window_fp8(C.byref(attn(n_seqs=0)), None, 0, None) == 0
    assert [size(*a) for a in ((0, 5, 64), (4097, 5, 64), (2, 0, 64), (2, (1 << 24) + 1, 64), (2, 5, 65))] == [0] * 5


def test_a_workspace_is_enough_for_smaller_calls():
    from ds4cuda_amd import lib
    size = lib().ds4hip_flash_attn_window_fp8_workspace_bytes
    for heads in (8, 16, 64, 128):
        for n_seqs in (1, 2, 16, 200):
            for n_q in (1, 2, 31, 400):
                need = size(n_seqs, n_q, heads)
                assert all(size(s, q, heads) <= need for s in (1, n_seqs) for q in (1, (n_q + 1) // 2, n_q))


def test_attention_outputs_are_aligned():
    from ds4cuda_amd import lib
    assert lib().ds4hip_flash_attn_window_fp8(C.byref(attn(out=X + 8)), X, BIG, None) == -22


def test_python_refuses_host_tensors_and_shapes():
    from ds4cuda_amd import Ds4HipError, ops, pages

    def refused(fn, *a, **kw):
        with pytest.raises(Ds4HipError) as e:
            fn(*a, **kw)
        assert e.value.code == -22

    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    c = (torch.zeros((1, 64, 448), dtype=torch.uint8), torch.zeros((1, 64, 8), dtype=torch.int8),
         torch.zeros((1, 64, 64), dtype=torch.int16))
    refused(pages.PagePool, *c, i32(4), i32(2, 4), i32(2), 16)
    refused(pages.PagePool, c[0][0], c[1], c[2], i32(4), i32(2, 4), i32(2), 16)
    refused(pages.PagePool, *c, i32(4), i32(4), i32(2), 16)
    cache = ops.Fp8KVCache(c[0][0], c[1][0], c[2][0])
    for q in (torch.zeros((2, 64, 512)), torch.zeros((2, 64, 512), dtype=torch.float16), torch.zeros((2, 64, 256)),
              torch.zeros(64, 512)):
        refused(ops.flash_attn_window_fp8, q, cache, i32(2, 4), i32(2), page_rows=16)
