"""Log probabilities are formed in 64 bits and rounded once: where a row's sum is exact, they are off by half a last place."""
import math

import pytest
import torch

from test_verify_sampled import _rejected, _sampled


@pytest.mark.gpu
@pytest.mark.parametrize("walk", [False, True])
def test_rows_whose_sum_is_exact(walk):
    """k tokens of the largest logit (a sum of ones is exact) and a draft of a weight below e^-45 = 2^-64, which fp32 and 64-bit
    sums of ones lose, kept by u = 0. Off by: the rounding to fp32, 2^-24 of the value, and a few roundings to 64 bits."""
    from chain_flow_b200.tree import RejectionVerifier
    V, n, tok = 5000, 400, 4321
    g = torch.Generator().manual_seed(1)
    rows, temps, want = [], [], []
    for i in range(n):
        k, tau = int(torch.randint(1, 900, (1,), generator=g)), (1.0, 0.7, 1.9)[i % 3]
        low = -tau * (46 + 40 * float(torch.rand(1, generator=g)))
        row = torch.full((V,), -math.inf)
        row[torch.randperm(V - 1000, generator=g)[:k]] = 0.75
        row[tok] = low
        rows.append(torch.stack([row, row]))
        temps.append(tau)
        want.append((float(row[tok]) - 0.75) / float(torch.tensor(tau)) - math.log(k))
        assert k * math.exp(want[-1]) < 2.0 ** -64
    logits, temp, want = torch.cat(rows), torch.tensor(temps), torch.tensor(want, dtype=torch.float64)
    flat = torch.arange(1, n + 1).int(), 2 * torch.arange(1, n + 1).int(), torch.full((n,), tok, dtype=torch.int32)
    probs = torch.zeros(n, V)
    probs[:, tok] = 1.0
    ver = RejectionVerifier(2 * n, n, 1024 if walk else 1, V)
    out, count, logp = _rejected(ver, logits, flat, probs, torch.zeros(n), torch.full((n,), 0.3), temp)
    assert bool((count == 1).all()) and bool((out[:, 0] == tok).all())
    off = (logp[:, 0].cpu().double() - want).abs()
    assert bool((off <= 2.0 ** -24 * want.abs() * (1 + 2.0 ** -20)).all()), float((off / want.abs()).max() * 2 ** 24)
