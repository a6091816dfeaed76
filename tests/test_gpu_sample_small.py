"""Sampled tokens that are unlikely, and logits whose differences pass fp32's range: token and share as the definition in
64 bits has them."""
import math

import pytest
import torch

from test_gpu_sample import check, sample

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [3, 300, 5000, 9000, 40000])
@pytest.mark.parametrize("many", [False, True])
def test_shares_of_small_weights(gpu, vocab, many):
    """u = 0 takes the first token that stays, here one of weight 2^-e of the largest. Its share is off by its rounding to
    fp32 (2^-24), its weight's error (2^-44) and that of the sum of what stays (256 roundings of 2^-46): 2^-23.9 holds them.
    many: next to hundreds of likelier tokens, more than are compared with each other."""
    t = 0.5
    for e in (1, 8, 18, 20, 22, 24, 30, 37, 41, 44):
        x = torch.full((2, vocab), -math.inf, device=gpu)
        x[:, vocab - 1] = 3.0
        x[:, vocab // 2] = 2.9
        if many and vocab >= 300:
            x[:, vocab // 2 + 1:vocab // 2 + 140] = 2.5
            if vocab >= 5000:
                x[:, vocab // 2 + 1:vocab // 2 + 1200] = 2.5
        x[:, 0] = 3.0 - t * e * math.log(2.0)
        u = torch.zeros(2, device=gpu)
        for k, p, m in ((0, 1.0, 0.0), (vocab, 1.0, 0.0), (vocab - 1, 1.0, 0.0), (0, 1.0, 2.0 ** -46), (vocab - 1, 1.0, 2.0 ** -46),
                        (0, 1.0 - 2.0 ** -24, 0.0)):
            check(x, u, t, k, p, m, sample(x, u, t, k, p, m))


@pytest.mark.parametrize("vocab", [300, 900, 8000, 12000, 70000])
def test_differences_past_fp32(gpu, vocab):
    """Logits from -3.2e38 to 3.2e38 at temperatures of that size: their differences pass fp32's range, while even the
    smallest weight is e^-6.4 of the largest."""
    g = torch.Generator(gpu).manual_seed(vocab)
    for t in (3e38, 1e38):
        x = (2.0 * torch.rand((3, vocab), generator=g, device=gpu) - 1.0) * 3.2e38
        x[1] = torch.where(x[1] > 0, 3.2e38, -3.2e38)
        x[2, ::3] = -math.inf
        u = torch.rand(3, generator=g, device=gpu)
        for k, p, m in ((0, 1.0, 0.0), (vocab - vocab // 10, 1.0, 0.0), (vocab // 2 + vocab // 4, 0.9, 0.0), (0, 0.95, 0.0), (0, 0.8, 0.0),
                        (0, 1.0, 0.2), (50, 1.0, 0.0), (vocab - 1, 0.99, 0.001)):
            check(x, u, t, k, p, m, sample(x, u, t, k, p, m))
