"""Attention over pages where one of the first rows scores far above many others that
together still matter: the others' small weights are not lost, however many they are."""
import math

import pytest
import torch

from paged_check import row_values

pytestmark = pytest.mark.gpu

DIM = 512
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


class Peak:
    """One list of n rows on pages in order: row `at` scores higher than the rest for queries
    along `up`; the rest have values around 1, that row around -1."""

    def __init__(self, gpu, n, page, seed, at=0, noise=0.3):
        from ds4cuda_amd import ops
        g = torch.Generator(gpu).manual_seed(seed)
        x = torch.randn((n, DIM), generator=g, device=gpu) * noise + 1.0
        x[:, :64] *= 0.02
        x[at] -= 2.0
        x[at, :64] = 2.0
        pages = -(-n // page)
        self.cache = ops.Fp8KVCache.empty(pages * page, gpu)
        self.cache.append(torch.cat([x, torch.zeros((pages * page - n, DIM), device=gpu)]))
        self.n, self.page, self.gpu, self.at = n, page, gpu, at
        self.kv = row_values(self.cache.codes[:n], self.cache.sexp[:n], self.cache.tail[:n])
        self.table = torch.arange(pages, dtype=torch.int32, device=gpu)

    def queries(self, n_q, heads, typ, seed, low=11.0, high=14.0):
        """Query i, head h: the row scores low .. high above the mean of the others."""
        g = torch.Generator(self.gpu).manual_seed(seed)
        q = torch.randn((n_q, heads, DIM), generator=g, device=self.gpu) * 0.25
        nats = torch.linspace(low, high, n_q * heads, device=self.gpu)[torch.randperm(n_q * heads, generator=g, device=self.gpu)]
        others = self.kv.float().mean(0)
        gap = (q @ (self.kv[self.at].float() - others)) / math.sqrt(DIM)
        # (the 64 dims that only that row has: 64 * 2 / sqrt(512) a unit)
        q[..., :64] += ((nats.view(n_q, heads) - gap) * math.sqrt(DIM) / 128.0)[..., None]
        return q.to(TYPES[typ])


def check(peak, q, out, positions, f32, window=0, first=0):
    """Queries against 64 bits. A weight is off by its own rounding (one f16 2^-11, hi + lo 2^-22)
    and by its score's error, all those that are subnormal in f16 by 2^-16 (2^-22) of the largest together;
    the sums of rows / 32 tiles, the parts they are joined from (at most 512) and a tile's
    32 products add in fp32, each step truncated at worst: 2^-23. Numerator and denominator
    each. Then the result's rounding. None of it but the sums' steps grows with the rows."""
    k = torch.arange(peak.n, device=peak.gpu)
    lost = 0.0
    for i, p in enumerate(positions):
        seen = k <= p
        if window:
            seen &= (k > p - window) | (k < first)
        rows = peak.kv[seen]
        x = q[i].double()
        s = x @ rows.T / math.sqrt(DIM)
        w = torch.softmax(s, -1)
        ref, size = w @ rows, w @ rows.abs()
        err = 42 * 2.0 ** -23 * (x.abs() @ rows.abs().T / math.sqrt(DIM)).amax(-1) + 2.0 ** -22 * s.abs().amax(-1)
        steps = (rows.shape[0] / 32 + 512 + 32) * 2.0 ** -23
        each = (2.0 ** -22 if f32 else 2.0 ** -11) + err[:, None] + steps
        all_small = (2.0 ** -22 if f32 else 2.0 ** -16) * w.amax(-1, keepdim=True) * rows.abs().amax()
        bound = 2 * each * size + 2 * all_small + (2.0 ** -24 if f32 else 2.0 ** -8) * ref.abs()
        d = (out[i].double() - ref).abs()
        assert (d <= bound).all(), (i, p, float(d.max()), float((d / bound).max()))
        # what the others add to the output: the check means nothing where that is below the bound
        top = s.argmax(-1)
        lost = max(lost, float((ref - rows[top]).abs().amax()))
    return lost


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
@pytest.mark.parametrize("heads", [8, 16, 64, 128])
@pytest.mark.parametrize("n,at", [(32768, 0), (131072, 3)])
def test_one_token_over_many_rows(gpu, n, at, heads, typ):
    """Cut into parts, each with a reference of its own."""
    from ds4cuda_amd import ops
    peak = Peak(gpu, n, 256, 1, at)
    q = peak.queries(2, heads, typ, 2)
    out = ops.flash_attn_window_fp8(q, peak.cache, peak.table[None].repeat(2, 1), i32([n, n - 77], gpu), page_rows=256)
    assert check(peak, q, out, [n - 1, n - 78], typ == "fp32") > 0.1


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
@pytest.mark.parametrize("heads,n_seqs,n", [(64, 256, 8192), (64, 256, 32768), (16, 512, 8192), (16, 512, 32768), (8, 512, 32768)])
def test_uncut_tokens(gpu, heads, n_seqs, n, typ):
    """As many sequences as workgroups: no list is cut."""
    from ds4cuda_amd import ops
    peak = Peak(gpu, n, 256, 3, 1)
    q = peak.queries(n_seqs, heads, typ, 4)
    out = ops.flash_attn_window_fp8(q, peak.cache, peak.table[None].repeat(n_seqs, 1), i32([n] * n_seqs, gpu), page_rows=256)
    some = list(range(0, n_seqs, n_seqs // 8))
    assert check(peak, q[some], out[some], [n - 1] * len(some), typ == "fp32") > (0.3 if n > 8192 else 0.1)


@pytest.mark.parametrize("typ,heads", [("bf16", 64), ("bf16", 8), ("fp32", 64)])
def test_uncut_prompt(gpu, heads, typ):
    """Many queries over all rows before them: problems that are short beside the call."""
    from ds4cuda_amd import ops
    n_q = 4096 if heads == 64 else 20000
    n = 32768 + n_q
    peak = Peak(gpu, n, 256, 5)
    q = peak.queries(n_q, heads, typ, 6)
    out = ops.flash_attn_window_fp8(q, peak.cache, peak.table[None], i32([n], gpu), page_rows=256, q_start=i32([0, n_q], gpu))
    some = list(range(0, n_q, n_q // 8 - 1))
    assert check(peak, q[some], out[some], [n - n_q + i for i in some], typ == "fp32") > 0.3


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
@pytest.mark.parametrize("heads", [8, 64])
@pytest.mark.parametrize("window,first", [(300, 4), (1024, 64), (4000, 1)])
def test_a_kept_row_above_a_window(gpu, window, first, heads, typ):
    from ds4cuda_amd import ops
    n, n_q = 9000, 1500
    peak = Peak(gpu, n, 64, 7)
    q = peak.queries(n_q, heads, typ, 8, 7.0, 12.0)
    out = ops.flash_attn_window_fp8(q, peak.cache, peak.table[None], i32([n], gpu), page_rows=64, window=window,
                                    n_first=first, q_start=i32([0, n_q], gpu))
    some = list(range(0, n_q, 211))
    assert check(peak, q[some], out[some], [n - n_q + i for i in some], typ == "fp32", window, first) > 0.1


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
@pytest.mark.parametrize("heads", [16, 64])
def test_rows_of_one_score(gpu, heads, typ):
    """All others alike, so that their roundings do not cancel; the share of weights that f16
    keeps least of, from far above to far below what counts."""
    from ds4cuda_amd import ops
    n, n_seqs = 32768, 512 if heads == 16 else 256
    peak = Peak(gpu, n, 256, 9, noise=0.0)
    q = peak.queries(n_seqs, heads, typ, 10, 9.0, 19.0)
    out = ops.flash_attn_window_fp8(q, peak.cache, peak.table[None].repeat(n_seqs, 1), i32([n] * n_seqs, gpu), page_rows=256)
    some = list(range(0, n_seqs, n_seqs // 16))
    assert check(peak, q[some], out[some], [n - 1] * len(some), typ == "fp32") > 0.3
