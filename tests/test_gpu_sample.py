"""Tokens sampled from logits: against the definition in 64 bits, where sizes, ties, borders and
values can go wrong."""
import numpy as np
import pytest
import torch

from draft_check import sample_64

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def logits_of(gpu, rows, vocab, typ, seed, spread=2.0, peaks=20):
    g = torch.Generator(gpu).manual_seed(seed)
    x = spread * torch.randn((rows, vocab), generator=g, device=gpu)
    if peaks:
        at = torch.randint(0, vocab, (rows, peaks), generator=g, device=gpu)
        x.scatter_reduce_(1, at, 6.0 + 2.0 * torch.randn((rows, peaks), generator=g, device=gpu), "amax")
    return x.to(TYPES[typ])


def randoms(gpu, rows, seed):
    return torch.rand(rows, generator=torch.Generator(gpu).manual_seed(seed), device=gpu)


def check(logits, u, t, k, p, m, got):
    """got: (tokens, probs). A probability is off by its rounding to fp32, 2^-24, and by the weights' errors of
    2^-50 each."""
    n = logits.shape[0]
    x, u = logits.float().cpu().numpy(), u.cpu().numpy()
    each = [np.broadcast_to(v.cpu().numpy() if isinstance(v, torch.Tensor) else v, n) for v in (t, k, p, m)]
    tokens, probs = got[0].cpu().numpy(), got[1].cpu().numpy()
    for i in range(n):
        token, prob = sample_64(x[i], *(v[i] for v in each), u[i])
        assert tokens[i] == token, (i, [v[i] for v in each], u[i], tokens[i], token)
        if token >= 0:
            assert abs(probs[i] - prob) <= prob * 2.0 ** -23.9, (i, probs[i], prob)
        else:
            assert np.isnan(probs[i])


def sample(logits, u, t=1.0, k=0, p=1.0, m=0.0, **kw):
    from ds4cuda_amd import ops
    return ops.sample_tokens(logits, u, temperature=t, top_k=k, top_p=p, min_p=m, **kw)


FILTERS = [(1.0, 0, 1.0, 0.0), (0.7, 1, 1.0, 0.0), (0.8, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.05),
           (0.6, 40, 0.95, 0.0), (1.0, 200, 0.5, 0.02), (0.9, 0, 0.8, 0.1), (0.0, 5, 0.5, 0.1), (1.0, 700, 0.999, 0.0),
           (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 9, 1.0, 2.0), (1.0, 0, 0.9999, 0.0), (5.0, 3000, 0.9, 0.0)]


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 31, 32, 33, 255, 1000, 8191, 8192, 8193, 32003, 70001, 129280])
def test_sizes_and_filters(gpu, vocab, typ):
    for i, (t, k, p, m) in enumerate(FILTERS):
        x, u = logits_of(gpu, 3, vocab, typ, 100 * i + vocab), randoms(gpu, 3, i + vocab)
        check(x, u, t, k, p, m, sample(x, u, t, k, p, m))


@pytest.mark.parametrize("typ", ["bf16", "fp32"])
@pytest.mark.parametrize("spread", [0.0, 0.3, 1.0])
def test_flat_rows(gpu, spread, typ):
    """Nearly all of the vocabulary stays: more candidates than any list holds, many of them equal."""
    for vocab in (600, 5000, 40000):
        x, u = logits_of(gpu, 4, vocab, typ, vocab, spread, 0), randoms(gpu, 4, vocab)
        for t, k, p, m in ((1.0, 0, 0.5, 0.0), (1.0, 0, 0.97, 0.0), (2.0, vocab // 2, 1.0, 0.0), (0.5, vocab // 3, 0.7, 0.01),
                           (1.0, 0, 1.0, 0.2), (1.0, 0, 1.0, 0.0), (1.0, vocab - 1, 0.25, 0.0)):
            check(x, u, t, k, p, m, sample(x, u, t, k, p, m))


def test_equal_logits_go_by_index(gpu):
    """Shares of equal weights, exact in any order of sums: the first ones stay."""
    for vocab, at in ((8, range(8)), (100, range(3, 90, 2)), (20000, range(0, 20000, 5)), (600, range(600))):
        x = torch.full((1, vocab), -4.0, device=gpu)
        ids = list(at)
        x[0, ids] = 3.0
        n = len(ids)
        for share in (0.25, 0.5, 0.75, 1.0):
            for u in (0.0, 0.5, 0.999):
                from ds4cuda_amd import ops
                k = max(1, int(n * share))
                tokens, probs = sample(x, torch.tensor([u], device=gpu), 1e-3, k, 1.0, 0.0)
                assert int(tokens) == ids[int(np.float64(np.float32(u)) * k)] and float(probs) == np.float32(1.0 / k)
                # before item j lie j of n equal weights: it stays where j < share * n
                tokens, probs = sample(x, torch.tensor([u], device=gpu), 1e-3, 0, share, 0.0)
                kept = int(np.ceil(n * share))
                assert int(tokens) == ids[int(np.float64(np.float32(u)) * kept)], (vocab, share, u)
                assert float(probs) == np.float32(1.0 / kept)
    zeros = torch.tensor([[-1.0, -0.0, 0.0, -0.0]], device=gpu)   # -0 and 0 are equal
    assert int(sample(zeros, torch.zeros(1, device=gpu), 0.0)[0]) == 1
    assert int(sample(zeros, torch.full((1,), 0.99, device=gpu), 1.0, 2)[0]) == 2


def test_each_row_its_own_parameters(gpu):
    n = len(FILTERS) * 4
    x, u = logits_of(gpu, n, 50001, "bf16", 5), randoms(gpu, n, 6)
    t, k, p, m = (torch.tensor([f[i] for f in FILTERS] * 4, dtype=torch.int32 if i == 1 else torch.float32, device=gpu)
                  for i in range(4))
    got = sample(x, u, t, k, p, m)
    check(x, u, t, k, p, m, got)
    for _ in range(3):
        again = sample(x, u, t, k, p, m)
        assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_masked_tokens_and_bad_rows(gpu):
    from ds4cuda_amd import ops
    x = logits_of(gpu, 12, 9000, "fp32", 9)
    x[0, 1:] = -float("inf")
    x[1, ::2] = -float("inf")
    x[2, :] = -float("inf")
    x[3, 8999] = float("nan")
    x[4, 17] = float("inf")
    x[5, :] = torch.finfo(torch.float32).min
    x[6, :] = -3e38
    x[6, 40] = 3e38
    x[7, 100:] = -float("inf")
    x[8, 5] = 1e30
    u = randoms(gpu, 12, 3)
    for t, k, p, m in FILTERS:
        check(x, u, t, k, p, m, sample(x, u, t, k, p, m))
    # parameters outside their ranges: that row alone
    bad = float("nan")
    t = torch.tensor([1.0, -1.0, bad, float("inf")] + [1.0] * 8, device=gpu)
    p = torch.tensor([0.5] * 4 + [bad] + [0.5] * 7, device=gpu)
    m = torch.tensor([0.0] * 5 + [bad] + [0.0] * 6, device=gpu)
    w = torch.cat([u[:6], torch.tensor([1.0, -0.1, bad], device=gpu), u[9:]])
    y = logits_of(gpu, 12, 300, "fp32", 10)
    tokens, probs = ops.sample_tokens(y, w, temperature=t, top_p=p, min_p=m)
    assert [int(v) for v in tokens[1:9]] == [-1] * 8 and probs[1:9].isnan().all()
    ok = torch.tensor([0, 9, 10, 11], device=gpu)
    check(y[ok], w[ok], 1.0, 0, 0.5, 0.0, (tokens[ok], probs[ok]))


def test_rows_with_a_stride_and_any_alignment(gpu):
    for typ in ("bf16", "fp32"):
        buf = logits_of(gpu, 5, 12347, typ, 11)
        x = buf[:, 3:12340]
        assert not x.is_contiguous() and x.data_ptr() % 16
        u = randoms(gpu, 5, 12)
        for t, k, p, m in FILTERS[:8]:
            check(x, u, t, k, p, m, sample(x, u, t, k, p, m))


def test_the_largest_vocabulary_and_many_rows(gpu):
    x, u = logits_of(gpu, 2, 262144, "fp32", 13, 0.2, 0), randoms(gpu, 2, 14)
    for t, k, p, m in ((1.0, 0, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 100000, 0.5, 0.0), (1.0, 64, 1.0, 0.0)):
        check(x, u, t, k, p, m, sample(x, u, t, k, p, m))
    x, u = logits_of(gpu, 20000, 40, "bf16", 15), randoms(gpu, 20000, 16)
    got = sample(x, u, 0.8, 10, 0.9, 0.0)
    some = torch.arange(0, 20000, 61, device=gpu)
    check(x[some], u[some], 0.8, 10, 0.9, 0.0, (got[0][some], got[1][some]))


def test_shares_are_met(gpu):
    """Over the random numbers i / n, each token comes as often as its share says (off by one at most)."""
    n = 4096
    x = logits_of(gpu, 1, 500, "fp32", 17).expand(n, 500)
    u = torch.arange(n, device=gpu) / n
    tokens, probs = sample(x.contiguous(), u, 1.0, 0, 0.95, 0.0)
    count = torch.bincount(tokens.long(), minlength=500)
    for i in range(500):
        if count[i]:
            share = float(probs[tokens == i][0])
            assert abs(int(count[i]) - share * n) <= 1.0 + 1e-3
    assert (tokens[1:] >= tokens[:-1]).all()


def test_captured(gpu):
    """A captured call follows its logits and parameters; eager calls in between do not reach it."""
    x, u = logits_of(gpu, 6, 33000, "bf16", 20), randoms(gpu, 6, 21)
    k = torch.full((6,), 30, dtype=torch.int32, device=gpu)
    sample(x, u, 1.0, k, 0.9, 0.0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = sample(x, u, 1.0, k, 0.9, 0.0)
    for i in range(4):
        x.copy_(logits_of(gpu, 6, 33000, "bf16", 30 + i))
        u.copy_(randoms(gpu, 6, 40 + i))
        k.fill_(5 + 100 * i)
        g.replay()
        want = sample(x, u, 1.0, k, 0.9, 0.0)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        check(x, u, 1.0, 5 + 100 * i, 0.9, 0.0, out)


def test_another_stream(gpu):
    x, u = logits_of(gpu, 9, 60000, "fp32", 50), randoms(gpu, 9, 51)
    want = sample(x, u, 1.0, 0, 0.9, 0.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = sample(x, u, 1.0, 0, 0.9, 0.0, stream=side)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_temperatures_and_logits_of_any_size(gpu):
    for scale, t in ((1e-30, 1e-30), (1e-30, 1.0), (1e30, 1e30), (1e30, 1.0), (1.0, 1e-30), (1.0, 1e-3), (1.0, 1e3),
                     (1.0, 3e38), (1e36, 3e38)):
        for vocab in (500, 12000):
            x, u = scale * logits_of(gpu, 4, vocab, "fp32", 18), randoms(gpu, 4, 19)
            for k, p, m in ((0, 1.0, 0.0), (20, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.1), (700, 0.99, 0.001)):
                check(x, u, t, k, p, m, sample(x, u, t, k, p, m))


def test_rows_past_32_bits(gpu):
    stride, vocab = 1300000007, 9001   # the last row begins 5.2 GB behind the first
    x = torch.empty(2 * stride + vocab, dtype=torch.bfloat16, device=gpu).as_strided((3, vocab), (stride, 1))
    x.copy_(logits_of(gpu, 3, vocab, "bf16", 20))
    u = randoms(gpu, 3, 21)
    for t, k, p, m in FILTERS:
        check(x, u, t, k, p, m, sample(x, u, t, k, p, m))


def test_the_most_rows(gpu):
    x, u = logits_of(gpu, 64, 8256, "bf16", 22).repeat(1024, 1), randoms(gpu, 65536, 23)
    some = torch.arange(0, 65536, 1009, device=gpu)
    for t, k, p, m in ((0.8, 10, 0.9, 0.0), (1.0, 0, 1.0, 0.0), (3.0, 0, 0.95, 0.0)):
        got = sample(x, u, t, k, p, m)
        check(x[some], u[some], t, k, p, m, (got[0][some], got[1][some]))


def test_two_streams_at_once(gpu):
    """Calls that run at the same time, each with its own workspace."""
    inputs = [(logits_of(gpu, 40, 40001, "bf16", 24 + i, 0.5 + i), randoms(gpu, 40, 26 + i)) for i in range(2)]
    want = [sample(x, u, 0.9, 0, 0.9, 0.0) for x, u in inputs]
    streams = [torch.cuda.Stream(gpu) for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (x, u) in enumerate(inputs):
            got[i].append(sample(x, u, 0.9, 0, 0.9, 0.0, stream=streams[i]))
    torch.cuda.synchronize()
    for w, all_got in zip(want, got):
        for g in all_got:
            assert torch.equal(w[0], g[0]) and torch.equal(w[1], g[1])
