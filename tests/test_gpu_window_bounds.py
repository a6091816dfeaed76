"""Attention over pages with query starts that go back, overlap or lie outside the batch: writes
stay inside the outputs and the workspace, and queries that no entry names keep their values."""
import pytest
import torch

from paged_check import quantized_rows

pytestmark = pytest.mark.gpu

GUARD = 4096   # bytes before and after


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def guarded(n_bytes, fill, gpu):
    """n_bytes of `fill` between two guards, and the whole."""
    whole = torch.full((n_bytes + 2 * GUARD,), 0xA5, dtype=torch.uint8, device=gpu)
    whole[GUARD:-GUARD] = fill
    return whole[GUARD:-GUARD], whole


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
@pytest.mark.parametrize("heads", [8, 64, 128])
@pytest.mark.parametrize("n_q,rows,start", [
    (40, 60, [5, 2, 90, 3]), (40, 60, [-4, 60, -1, 40]), (40, 60, [1 << 30, 0, 40, 0]), (40, 9, [38, 40, 39, 39]),
    (40, 700, [10, 20, 10, 20]), (3, 3000, [-(1 << 31), 1, 1, (1 << 31) - 1]), (1, 5, [0, 1, 0, 1]), (40, 60, [7, 7, 7, 7])])
@pytest.mark.parametrize("window", [0, 50])
def test_starts_outside_the_batch(gpu, n_q, rows, start, window, heads, typ):
    from ds4cuda_amd import ops
    page, n_seqs = 16, len(start) - 1
    per = -(-rows // page)
    codes, sexp, tail = quantized_rows(per * page, 1, gpu)
    cache = ops.Fp8KVCache(codes, sexp, tail)
    table = torch.arange(per, dtype=torch.int32, device=gpu)[None].repeat(n_seqs, 1)   # (the same rows: what overlaps agrees)
    dtype = {"bf16": torch.bfloat16, "fp32": torch.float32}[typ]
    q = torch.randn((n_q, heads, 512), device=gpu).to(dtype)
    need = ops.window_workspace_bytes(n_seqs, n_q, heads)
    ws, ws_all = guarded(need, 0xFF, gpu)
    bits, out_all = guarded(q.numel() * q.element_size(), 0, gpu)
    out = bits.view(dtype).view(q.shape)
    out.fill_(7.0)
    ops.flash_attn_window_fp8(q, cache, table, i32([rows] * n_seqs, gpu), page_rows=page, window=window, n_first=2,
                              q_start=i32(start, gpu), out=out, workspace=ws)
    for whole in (ws_all, out_all):
        assert (whole[:GUARD] == 0xA5).all() and (whole[-GUARD:] == 0xA5).all()
    clamped = [min(max(s, 0), n_q) for s in start]
    named = {i for a, b in zip(clamped, clamped[1:]) for i in range(a, b)}
    rest = [i for i in range(n_q) if i not in named]
    assert (out[rest] == 7.0).all()
    if sum(max(b - a, 0) for a, b in zip(clamped, clamped[1:])) == len(named):   # (no two entries name one query)
        assert torch.isfinite(out).all() and all(bool((out[i] != 7.0).any()) for i in named)


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
@pytest.mark.parametrize("heads", [8, 16, 64, 128])
@pytest.mark.parametrize("n,window,first,bad", [(400, 40, 3, 5), (400, 0, 0, 9), (700, 600, 0, 2), (400, 40, 70, 1), (2000, 100, 0, 40)])
def test_a_bad_entry_reaches_few_neighbours(gpu, n, window, first, bad, heads, typ):
    """NaN where a query sees a row of the 32 that the entry stands for, with up to 64 / heads - 1 queries
    next to it; all others as without it."""
    from ds4cuda_amd import ops
    page = 32
    per = -(-n // page)
    cache = ops.Fp8KVCache(*quantized_rows(per * page, 2, gpu))
    table = torch.arange(per, dtype=torch.int32, device=gpu)[None]
    dtype = {"bf16": torch.bfloat16, "fp32": torch.float32}[typ]
    n_q = n // 2
    q = torch.randn((n_q, heads, 512), device=gpu).to(dtype)
    call = lambda: ops.flash_attn_window_fp8(q, cache, table, i32([n], gpu), page_rows=page, window=window, n_first=first,
                                             q_start=i32([0, n_q], gpu))
    want = call()
    table[0, bad] = per
    got = call()
    lost = torch.isnan(got).flatten(1)
    hit = [any(k <= p and (window == 0 or k > p - window or k < first) for k in range(page * bad, page * bad + page))
           for p in range(n - n_q, n)]
    near = max(64 // heads - 1, 0)
    assert torch.isfinite(want).all() and any(hit)
    for i in range(n_q):
        if hit[i]:
            assert lost[i].all(), i
        elif not any(hit[max(0, i - near):i + near + 1]):
            assert not lost[i].any() and torch.equal(got[i], want[i]), i
