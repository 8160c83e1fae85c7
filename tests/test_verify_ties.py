"""Rows whose mass lies in a few equal tokens (a filter's or a grammar's survivors, ties of 16-bit logits), verified with numbers
that fall exactly on a border of two of them: in 64 bits the running sum up to a border equals the threshold, and the token
behind it is drawn. All rows at once and as a walk: a verifier far larger than its call takes the walk."""
import math

import pytest
import torch

import oracle
from test_verify_sampled import _check, _rejected, _sampled

WALK = 1024                                              # max_spec_len of a verifier that walks


def _survivors(V, n, at, g):
    """n tokens of V: neighbours, the ends, or anywhere."""
    if at == "ends":
        return torch.cat([torch.arange(n // 2), torch.arange(V - (n - n // 2), V)])
    return torch.randperm(V, generator=g)[:n].sort().values


def _borders(n, g, few):
    """Numbers k / n (exact, n a power of two), and one step beside them."""
    ks = torch.arange(n) if n <= few else torch.randint(n, (few,), generator=g)
    u = ks.double() / n
    return torch.cat([u, u + 2.0 ** -52, (u - 2.0 ** -52).clamp_min(0)])


def _alone(n):
    """Offsets of n requests of a row each."""
    none = torch.zeros(0, dtype=torch.int32)
    return torch.zeros(n, dtype=torch.int32), torch.arange(1, n + 1, dtype=torch.int32), none, none


def _rows(V, dtype, n, at, g, mask, temp=1.0):
    """A row for every border: n survivors of one logit, the rest masked."""
    u = _borders(n, g, 8)
    rows = []
    for _ in range(len(u)):
        row = torch.full((V,), -math.inf if mask == "inf" else torch.finfo(dtype).min, dtype=dtype)
        row[_survivors(V, n, at, g)] = 0.25 if mask == "inf" else 0.0
        rows.append(row)
    return torch.stack(rows), u, torch.full((len(u),), temp)


def _tied(V, dtype, g):
    """Two tokens share a row's mass: together the others are below 2^-53 of it at temperature 0.1 (V e^-50 = 2^-55.6 at most)."""
    rows, at = [], []
    for _ in range(16):
        row = (torch.randn(V, generator=g) * 1.5).clamp(max=3).to(dtype)
        at.append(_survivors(V, 2, "anywhere", g))
        row[at[-1]] = 8.0
        rows.append(row)
    assert V * math.exp(-50) < 2.0 ** -53
    return torch.stack(rows), torch.full((16,), 0.5, dtype=torch.float64), torch.full((16,), 0.1), torch.stack(at)


@pytest.mark.gpu
@pytest.mark.parametrize("walk", [False, True])
@pytest.mark.parametrize("mask", ["inf", "lowest"])
@pytest.mark.parametrize("dtype, V", [(torch.float32, 8192), (torch.bfloat16, 5003), (torch.float16, 32003), (torch.float32, 32003), (torch.bfloat16, 3)])
def test_borders_of_equal_survivors(dtype, V, mask, walk):
    from chain_flow_b200.tree import SampledVerifier
    g = torch.Generator().manual_seed(V)
    for n in (2, 4, 1024):
        for at in ("ends", "anywhere"):
            if n <= V:
                logits, u, temp = _rows(V, dtype, n, at, g, mask)
                flat = _alone(len(u))
                ver = SampledVerifier(len(u), len(u), WALK if walk else 0)
                _check(_sampled(ver, logits, flat, u, temp), oracle.tree_verify_sampled(logits, *flat, u, temp, ver.max_spec))


@pytest.mark.gpu
@pytest.mark.parametrize("walk", [False, True])
@pytest.mark.parametrize("dtype, V", [(torch.float32, 8192), (torch.bfloat16, 5003), (torch.float16, 32003)])
def test_two_tied_tokens_above_next_to_no_mass(dtype, V, walk):
    from chain_flow_b200.tree import RejectionVerifier, SampledVerifier
    logits, u, temp, at = _tied(V, dtype, torch.Generator().manual_seed(V + 1))
    flat, n = _alone(len(u)), len(u)
    want = oracle.tree_verify_sampled(logits, *flat, u, temp, WALK if walk else 0)
    assert torch.equal(want[0][:, 0], at[:, 1])
    _check(_sampled(SampledVerifier(n, n, WALK if walk else 0), logits, flat, u, temp), want)
    ver = RejectionVerifier(n, n, WALK if walk else 0, V)
    got = _rejected(ver, logits, flat[:3], torch.zeros(0, V), torch.zeros(0), u, temp)
    _check(got, (want[0], want[2], want[3]))


@pytest.mark.gpu
@pytest.mark.parametrize("walk", [False, True])
@pytest.mark.parametrize("mask", ["inf", "lowest"])
@pytest.mark.parametrize("rest", ["bonus", "all", "half", "none"])
def test_borders_of_what_replaces_a_draft(rest, mask, walk):
    """Draws of a chain's bonus row, of all of a row's mass above draft probabilities of 0, of what is left above half of the
    survivors' probability, and (draft probabilities above all of it) of the target's own."""
    from chain_flow_b200.tree import RejectionVerifier
    for dtype, V in ((torch.float32, 8192), (torch.float16, 5003)):
        g = torch.Generator().manual_seed(V)
        for n in (2, 4, 1024):
            logits, v, temp = _rows(V, dtype, n, "anywhere", g, mask)
            m = len(v)
            if rest == "bonus":
                flat, probs = _alone(m)[:3], torch.zeros(0, V)
            else:
                flat = torch.arange(1, m + 1).int(), 2 * torch.arange(1, m + 1).int(), torch.full((m,), -1, dtype=torch.int32)
                probs = torch.full((m, V), dict(all=0.0, half=0.5 / n, none=1.0)[rest])
                logits = logits.repeat_interleave(2, 0)
            u = torch.full((len(probs),), 0.5, dtype=torch.float64)
            ver = RejectionVerifier(len(logits), m, WALK if walk else 1, V)
            want = oracle.chain_verify_rejection(logits, *flat, probs, u, v, temp, ver.max_spec)
            _check(_rejected(ver, logits, flat, probs, u, v, temp), want)


@pytest.mark.gpu
@pytest.mark.parametrize("walk", [False, True])
def test_a_tree_of_tied_rows(walk):
    """A walk that goes on from a token drawn on a border."""
    from chain_flow_b200.tree import SampledVerifier
    V, n = 20000, 6
    g = torch.Generator().manual_seed(2)
    logits = torch.full((n + 1, V), -math.inf)
    tokens = []
    for i in range(n + 1):
        at = _survivors(V, 4, "anywhere", g)
        logits[i, at] = 1.5
        tokens.append(int(at[3]))                        # behind the border at 3 / 4
    flat = (torch.tensor([n]).int(), torch.tensor([n + 1]).int(), torch.tensor(tokens[:n]).int(), torch.arange(-1, n - 1).int())
    u = torch.full((n + 1,), 0.75)
    ver = SampledVerifier(n + 1, 1, WALK if walk else n)
    want = oracle.tree_verify_sampled(logits, *flat, u, None, ver.max_spec)
    assert want[2].tolist() == [n] and want[0][0, :n + 1].tolist() == tokens
    _check(_sampled(ver, logits, flat, u), want)


@pytest.mark.gpu
def test_parts_whose_sums_round_apart():
    """A row of 16 parts of 1024: two of a little less than 2^-53, one of 1, one without mass, three more of 1. Up to the third part
    the running sum is 1 or 1 + 2^-52, by the order of its additions, and the threshold 1: within a rounding either the
    third part's token or the next one's, and nothing else."""
    from chain_flow_b200.tree import SampledVerifier
    V, below = 16 * 1024 - 7, math.nextafter(-53 * math.log(2), -math.inf) - 1e-5
    logits = torch.full((1, V), -math.inf)
    logits[0, [5, 1024 + 5]] = below
    at = [1024 * part + 5 for part in (2, 4, 5, 6)]
    logits[0, at] = 0.0
    assert float(torch.exp(logits[0, 5].double())) < 2.0 ** -53
    got = _sampled(SampledVerifier(1, 1, 0), logits, _alone(1), torch.tensor([0.25]))
    assert int(got[0][0, 0]) in at[:2]


@pytest.mark.gpu
@pytest.mark.parametrize("walk", [False, True])
@pytest.mark.parametrize("n", [3, 7, 100, 999])
def test_borders_that_are_no_dyadic_numbers(n, walk):
    """k / n rounded to 64 bits, and its neighbours: u times the (exact) sum is rounded as the definition rounds it."""
    from chain_flow_b200.tree import SampledVerifier
    V = 20011
    g = torch.Generator().manual_seed(n)
    ks = (torch.arange(n) if n < 20 else torch.randint(n, (20,), generator=g)).tolist()
    u = torch.tensor([x for k in ks for x in (k / n, math.nextafter(k / n, 1), max(math.nextafter(k / n, 0), 0))], dtype=torch.float64)
    for mask, top in ((-math.inf, 3.0), (torch.finfo(torch.float16).min, -2.0)):
        logits = torch.full((len(u), V), mask, dtype=torch.float16)
        for row in logits:
            row[_survivors(V, n, "anywhere", g)] = top
        flat = _alone(len(u))
        ver = SampledVerifier(len(u), len(u), WALK if walk else 0)
        _check(_sampled(ver, logits, flat, u), oracle.tree_verify_sampled(logits, *flat, u, None, ver.max_spec))
