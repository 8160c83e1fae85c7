"""Offsets that fall back over the rows of a request further back: the request reads what its offsets name, and every other
request's output is what it is without it."""
import pytest
import torch

import oracle
from test_verify_sampled import _case, _chains


def _fallen(sizes, at, back):
    """Offsets of requests of `sizes`, but request at + 1 lies over the first rows of request at - back."""
    cu_s = torch.tensor([n + 1 for n in sizes]).cumsum(0).int()
    first = int(cu_s[at - back - 1]) if at - back else 0
    cu_s[at] = first                                     # what it has itself ends where that one's rows begin
    cu_s[at + 1] = first + sizes[at + 1] + 1
    return cu_s, first


def _as_it_reads(sizes, b, first, logits, tokens):
    """A request of request b's drafts over the rows that its offsets name."""
    n, d = sizes[b], sum(sizes[:b])
    rows = slice(first, first + n + 1)
    return (logits[rows], torch.tensor([n]), torch.tensor([n + 1]), tokens[d:d + n]), rows, slice(d, d + n)


@pytest.mark.gpu
@pytest.mark.parametrize("walk", [False, True])
@pytest.mark.parametrize("requests, at, back", [(3, 1, 1), (5, 3, 3), (40, 38, 30), (300, 298, 298)])
def test_offsets_that_fall_over_an_earlier_request(requests, at, back, walk):
    from chain_flow_b200.tree import RejectionVerifier, SampledVerifier
    V, sizes = 700, [2 + b % 2 for b in range(requests)]
    sizes[at + 1] = 1
    cu_s, first = _fallen(sizes, at, back)
    others, spec = [b for b in range(requests) if b not in (at, at + 1)], 1024 if walk else 3
    temp = 0.5 + torch.arange(requests) % 3 * 0.5

    def compare(got, want, own):
        for a, b in zip(got[:-1], want[:-1]):
            assert torch.equal(a[others].cpu().long(), b[others])
        assert int(got[0][at].max()) == -1                # it would begin before the first row, or over the last request's
        for a, b in zip(got[:-1], own[:-1]):
            assert torch.equal(a[at + 1].cpu().long(), b[0])

    logits, flat, u = _case(sizes, V, torch.float32, 3)
    want = oracle.tree_verify_sampled(logits, *flat, u, temp, spec)
    args, rows, drafts = _as_it_reads(sizes, at + 1, first, logits, flat[2])
    own = oracle.tree_verify_sampled(*args, flat[3][drafts], u[rows], temp[at + 1:at + 2], spec)
    dev = [t.cuda() for t in (logits, flat[0], cu_s, *flat[2:], u)]
    ver = SampledVerifier(len(logits), requests, spec)
    for _ in range(3):
        compare(ver(*dev, temperature=temp.cuda()), want, own)
    assert int(ver.err.item()) == 7
    logits, flat, probs, u, v = _chains(sizes, V, torch.float32, 4)
    want = oracle.chain_verify_rejection(logits, *flat, probs, u, v, temp, spec)
    args, rows, drafts = _as_it_reads(sizes, at + 1, first, logits, flat[2])
    own = oracle.chain_verify_rejection(*args, probs[drafts], u[drafts], v[at + 1:at + 2], temp[at + 1:at + 2], spec)
    dev = [t.cuda() for t in (logits, flat[0], cu_s, flat[2], probs, u, v)]
    ver = RejectionVerifier(len(logits), requests, spec, V)
    for _ in range(3):
        compare(ver(*dev, temperature=temp.cuda()), want, own)
    assert int(ver.err.item()) == 7
