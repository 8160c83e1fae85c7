"""Rows of masks, infinities and NaN, temperatures and numbers at their limits, verified as a walk and as all rows at once. A verifier
for many more drafts than its calls have walks; one as large as its calls takes all rows at once."""
import math

import pytest
import torch

import oracle
from test_verify_sampled import _check, _rejected, _sampled

INF, NAN = math.inf, math.nan
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _odd(V, dtype, g):
    """[(name, row)]"""
    info = torch.finfo(dtype)
    out = []

    def add(name, change):
        row = (torch.randn(V, generator=g) * 2).to(dtype)
        change(row)
        out.append((name, row))

    def at(row, where, x):
        row[torch.tensor(where) % V] = x

    def only(row, where, x, rest):
        row.fill_(rest)
        at(row, where, x)
    far = [3, 1030, V - 1]
    add("plain", lambda r: None)
    for rest in (-INF, info.min):
        add("nothing", lambda r, rest=rest: r.fill_(rest))
        add("one", lambda r, rest=rest: only(r, [V // 2], -7.0, rest))
        add("last", lambda r, rest=rest: only(r, [V - 1], 2.0, rest))
        add("three", lambda r, rest=rest: only(r, far, 0.0, rest))
        add("three, one larger", lambda r, rest=rest: (only(r, far, 0.0, rest), at(r, [1030], 2.0)))
        add("head", lambda r, rest=rest: at(r, range(7, V), rest))
        add("tail", lambda r, rest=rest: at(r, range(V - 5), rest))
        add("inf", lambda r, rest=rest: only(r, [77], INF, rest))
        add("nan", lambda r, rest=rest: only(r, [2], NAN, rest))
    add("infs", lambda r: at(r, [5, V - 2], INF))
    add("more infs", lambda r: at(r, far + [700], INF))
    add("inf and nan", lambda r: (at(r, [12], INF), at(r, [V - 3], NAN)))
    add("nans", lambda r: at(r, far, NAN))
    add("all nan", lambda r: r.fill_(NAN))
    add("largest", lambda r: (r.fill_(info.min), at(r, [V // 3], info.max)))
    add("all largest", lambda r: r.fill_(info.max))
    add("flat", lambda r: r.fill_(0))
    add("steps", lambda r: (r.fill_(0), at(r, range(V // 4, V // 2), 5.0)))
    add("wide", lambda r: r.mul_(100))
    return out


def _alone(n):
    none = torch.zeros(0, dtype=torch.int32)
    return torch.zeros(n, dtype=torch.int32), torch.arange(1, n + 1, dtype=torch.int32), none, none


@pytest.mark.gpu
@pytest.mark.parametrize("walk", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [777, 5003, 40001])
def test_odd_rows_of_trees(V, dtype, walk):
    """Every row with its own temperature and number, and (as it goes on) as the row that an accepted draft leads to."""
    from chain_flow_b200.tree import SampledVerifier
    g = torch.Generator().manual_seed(V)
    rows = [r for _, r in _odd(V, dtype, g)]
    temps = [1.0, 0.0, 0.8, 2.0 ** -20, 50.0, 1e35, INF, NAN, -1.0, 2.0 ** -140, 0.05]
    us = [0.37, 0.0, 1 - 2.0 ** -24, 0.999, 1.0, -3.0, NAN, 2.0 ** -40, 0.61]
    n = 2 * len(rows)
    logits = torch.stack(rows * 2)
    temp, u = (torch.tensor([x[(i * k) % len(x)] for i in range(n)]) for x, k in ((temps, 3), (us, 2)))
    ver = SampledVerifier(n, n, 1024 if walk else 0)
    flat = _alone(n)
    _check(_sampled(ver, logits, flat, u, temp), oracle.tree_verify_sampled(logits, *flat, u, temp, ver.max_spec))
    # chains of two: the first row's draft is taken, its child's row is an odd one
    m = len(rows)
    first = torch.full((V,), -INF, dtype=dtype)
    first[9] = 1.0
    logits = torch.stack([x for r in rows for x in (first, r)])
    flat = (torch.arange(1, m + 1).int(), 2 * torch.arange(1, m + 1).int(), torch.full((m,), 9).int(), torch.full((m,), -1).int())
    u, temp = torch.rand(2 * m, generator=g, dtype=torch.float64), temp[:m]
    temp = torch.where(temp >= 2.0 ** -100, temp, torch.ones(m))          # (greedy rows take the draft too)
    ver = SampledVerifier(2 * m, m, 1024 if walk else 1)
    want = oracle.tree_verify_sampled(logits, *flat, u, temp, ver.max_spec)
    assert bool((want[2] == 1).all())
    _check(_sampled(ver, logits, flat, u, temp), want)


@pytest.mark.gpu
@pytest.mark.parametrize("walk", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V, short", [(777, 0), (5003, 1200)])
def test_odd_rows_of_chains(V, short, dtype, walk):
    """Every row under a draft that is likely, unlikely or no token, with draft probabilities that are ordinary, none, above the
    target's, negative or NaN; the rows after it odd too."""
    from chain_flow_b200.tree import RejectionVerifier
    g = torch.Generator().manual_seed(V + 5)
    named = [r for _, r in _odd(V, dtype, g)]
    ids = torch.randperm(V, generator=g)[:short] if short else None
    cols = short or V
    kinds = [lambda q: q, lambda q: 0 * q, lambda q: 3 * q + 0.01, lambda q: -q, lambda q: q.masked_fill(torch.arange(cols) % 3 == 0, NAN)]
    rows, toks, probs, us, vs, temps = [], [], [], [], [], []
    for i, row in enumerate(named):
        for j in range(6):
            pick = int(row.float().nan_to_num(-INF).argmax()) if j % 2 else int(torch.randint(V, (1,), generator=g))
            toks.append(pick if j < 4 else (ids[0] if short and j == 4 else -1 if j == 4 else V))
            rows += [row, named[(i + j) % len(named)]]
            probs.append(kinds[(i + j) % 5](torch.softmax(torch.randn(cols, generator=g) * 3, 0)))
            us.append([0.3, 0.0, 1.0, NAN, 0.9, 2.0 ** -30][(i + j) % 6])
            vs.append([0.5, 0.0, 0.93, 1.0, NAN, 1 - 2.0 ** -24, 0.25][(i * 2 + j) % 7])
            temps.append([1.0, 0.0, 0.4, 3.0, 2.0 ** -20, 1e35, NAN][(i + 3 * j) % 7])
    n = len(toks)
    flat = torch.arange(1, n + 1).int(), 2 * torch.arange(1, n + 1).int(), torch.tensor([int(t) for t in toks], dtype=torch.int32)
    logits, probs, u, v, temp = torch.stack(rows), torch.stack(probs), torch.tensor(us), torch.tensor(vs), torch.tensor(temps)
    ver = RejectionVerifier(2 * n, n, 1024 if walk else 1, V, draft_ids=ids)
    want = oracle.chain_verify_rejection(logits, *flat, probs, u, v, temp, ver.max_spec, ids)
    assert 0 < int(want[1].sum()) < n
    _check(_rejected(ver, logits, flat, probs, u, v, temp), want)


@pytest.mark.gpu
@pytest.mark.parametrize("sizes, V, dtype", [([5] * 3, 248320, torch.bfloat16), ([4, 0, 8, 1], 32003, torch.float32), ([3] * 9, 70001, torch.float16)])
def test_walks_at_full_vocabularies(sizes, V, dtype):
    from chain_flow_b200.tree import RejectionVerifier, SampledVerifier
    from test_verify_sampled import _case, _chains
    logits, flat, probs, u, v = _chains(sizes, V, dtype, 23)
    ver = RejectionVerifier(len(logits), len(sizes), 1024, V)
    _check(_rejected(ver, logits, flat, probs, u, v), oracle.chain_verify_rejection(logits, *flat, probs, u, v, None, 1024))
    logits, flat, u = _case(sizes, V, dtype, 24)
    ver = SampledVerifier(len(logits), len(sizes), 1024)
    _check(_sampled(ver, logits, flat, u), oracle.tree_verify_sampled(logits, *flat, u, None, 1024))
