"""Drafts of probabilities at and below fp32's smallest normal number: a draft stays if u q < p, as 64 bits decide it."""
import math

import pytest
import torch

import oracle
from test_verify_sampled import _check, _rejected


@pytest.mark.gpu
@pytest.mark.parametrize("walk", [False, True])
@pytest.mark.parametrize("size", [4, 8])
def test_drafts_of_tiny_probabilities(size, walk):
    """p = 2^-e against u q = 2^-(e + d), d to either side, u q and p normal, denormal and below every fp32 number; random
    numbers that fp32 cannot hold with large q."""
    from chain_flow_b200.tree import RejectionVerifier
    V, tok = 40, 7
    rows, probs, us, sure = [], [], [], []

    def add(e, q, u):
        if size == 4 and not (u == 0 or u >= 2.0 ** -149):
            return
        row = torch.full((V,), -math.inf)
        row[3], row[tok] = 0.0, -e * math.log(2)
        p = math.exp(float(row[tok]))
        for given in {q, -q}:
            rows.append(torch.stack([row, row]))
            probs.append(torch.zeros(V))
            probs[-1][tok] = given
            us.append(u)
            uq = u * float(probs[-1][tok]) if given > 0 else 0.0
            sure.append(uq < p)
            assert uq == 0 or abs(math.log2(uq) - math.log2(p)) > 0.5
    for e in (20, 100, 123, 125, 126, 127, 130, 140, 148, 149, 150, 155, 170, 300):
        for d in (-30, -2, -1, 1, 2, 30):
            for k in (1, 24, 60, 149):
                if 0 <= e + d - k <= 149:
                    add(e, 2.0 ** -(e + d - k), 2.0 ** -k)
            if size == 8:
                add(e, 2.0 ** 100, 2.0 ** -(e + d + 100))
                add(e, 1.0, 2.0 ** -(e + d) if e + d > 0 else 0.0)
                add(e, 2.0 ** -149, 2.0 ** -(e + d - 149) if e + d > 149 else 0.0)
    keep = [i for i, u in enumerate(us) if u < 1]
    rows, probs, us, sure = ([x[i] for i in keep] for x in (rows, probs, us, sure))
    n = len(rows)
    logits, probs = torch.cat(rows), torch.stack(probs)
    u = torch.tensor(us, dtype=torch.float64).to(torch.float32 if size == 4 else torch.float64)
    flat = torch.arange(1, n + 1).int(), 2 * torch.arange(1, n + 1).int(), torch.full((n,), tok, dtype=torch.int32)
    v = torch.full((n,), 0.5, dtype=u.dtype)
    ver = RejectionVerifier(2 * n, n, 1024 if walk else 1, V)
    want = oracle.chain_verify_rejection(logits, *flat, probs, u, v, None, ver.max_spec)
    assert [bool(x) for x in want[1]] == sure and 0 < sum(sure) < n
    _check(_rejected(ver, logits, flat, probs, u, v), want)
