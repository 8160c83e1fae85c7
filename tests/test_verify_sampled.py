"""Drafted tokens verified against the target's probabilities from given random numbers (cfb_tree_verify_sampled,
cfb_chain_verify_rejection) against oracle.verify in 64 bits. Tokens, paths and lengths are whole numbers and have to be
equal. Log probabilities: the sum of a row's weights is off by less than 2^-17 (cfb_verify.cu), so its logarithm by
that, and the result is rounded to fp32 once (2^-24 of it); tolerance 2^-16 + 2^-23 |value|."""
import math

import pytest
import torch

import oracle
from chain_flow_b200 import _lib
from chain_flow_b200.gdn import make_tree
from oracle.verify import draw, row_token, row_weights

FAKE = 0x10000


# ---- CPU: the oracle, and the refusals of the entry points ------------------------------------------
def test_a_draw_takes_each_token_as_often_as_it_weighs():
    row = torch.tensor([0.3, -math.inf, 1.7, -2.0, 0.3])
    w, _, greedy = row_weights(row, 0.7)
    p = (w / w.sum()).tolist()
    n = 20000
    seen = [draw(w, (i + 0.5) / n) for i in range(n)]
    assert not greedy and all(abs(seen.count(t) / n - p[t]) <= 1 / n for t in range(5))


def test_a_chain_with_draft_probabilities_gives_the_targets_distribution():
    """Over an even grid of both numbers, and the drafts in proportion to q, the first token is distributed as p."""
    g = torch.Generator().manual_seed(0)
    V, n = 4, 40
    logits = torch.randn(2, V, generator=g)
    q = torch.softmax(torch.randn(1, V, generator=g), 1)
    p = torch.softmax(logits[0].double(), 0)
    cu_d, cu_s = torch.tensor([1]), torch.tensor([2])
    mass = torch.zeros(V, dtype=torch.float64)
    for d in range(V):
        for i in range(n):
            for j in range(n):
                out, count, _ = oracle.chain_verify_rejection(logits, cu_d, cu_s, torch.tensor([d]), q, torch.tensor([(i + 0.5) / n]),
                                                              torch.tensor([(j + 0.5) / n]), None, 1)
                mass[out[0, 0]] += float(q[0, d]) / n ** 2
                assert int(count[0]) == int(out[0, 1] >= 0)
    # a border of the accepting number lies inside a cell of the grid, one of the drawing number too
    assert float((mass - p).abs().max()) <= 2 / n


def test_a_tree_follows_its_rows_draws():
    logits = torch.full((4, 6), -math.inf)
    logits[0, [2, 5]] = 0.0                          # root: token 2 below u = 1/2, then 5
    logits[1, 1] = 0.0
    logits[2, 3] = logits[2, 4] = math.inf           # two share the mass
    args = (torch.tensor([3]), torch.tensor([4]), torch.tensor([2, 5, 3]), torch.tensor([-1, -1, 1]))
    got = oracle.tree_verify_sampled(logits, *args, torch.tensor([0.6, 0.0, 0.2, 0.9]), None, 3)
    assert got[0].tolist() == [[5, 3, -1, -1]] and got[1].tolist() == [[1, 2, -1]] and got[2].tolist() == [2]
    assert torch.allclose(got[3][0, :2], torch.full((2,), math.log(0.5), dtype=torch.float64)) and float(got[3][0, 2]) == 0
    assert row_token(torch.tensor([0.0, math.nan, 9.0]), 1.0, 0.5) == 1 and row_token(torch.tensor([1.0, 3.0, 3.0]), 0.0, 0.9) == 1


def _tree_call(lib, **kw):
    a = dict(logits=FAKE, ld=100, rows=5, V=100, dtype=2, cu_d=FAKE, cu_s=FAKE, tokens=FAKE, parents=FAKE, drafts=3, u=FAKE,
             size=4, temp=None, B=2, spec=3, out=FAKE, path=FAKE, count=FAKE, logp=FAKE, ws=FAKE, bytes=1 << 20, err=None, st=None)
    a.update(kw)
    return lib.cfb_tree_verify_sampled(*a.values())


def _chain_call(lib, **kw):
    a = dict(logits=FAKE, ld=100, rows=5, V=100, dtype=2, cu_d=FAKE, cu_s=FAKE, tokens=FAKE, probs=FAKE, ld_probs=100, drafts=3,
             width=100, index=None, u=FAKE, v=FAKE, size=4, temp=None, B=2, spec=3, out=FAKE, count=FAKE, logp=FAKE, ws=FAKE,
             bytes=1 << 20, err=None, st=None)
    a.update(kw)
    return lib.cfb_chain_verify_rejection(*a.values())


@pytest.mark.parametrize("change, status", [
    (dict(logits=None), 1), (dict(rows=0), 1), (dict(V=0), 1), (dict(B=0), 1), (dict(spec=-1), 1), (dict(ld=99), 1), (dict(cu_d=None), 1),
    (dict(cu_s=None), 1), (dict(tokens=None), 1), (dict(drafts=-1), 1), (dict(u=None), 1), (dict(out=None), 1), (dict(count=None), 1),
    (dict(logp=None), 1), (dict(ws=None), 1), (dict(dtype=3), 2), (dict(size=2), 2), (dict(spec=1025), 2), (dict(V=1 << 22, ld=1 << 22), 2),
    (dict(B=65536), 2), (dict(logits=FAKE + 1), 1), (dict(ws=FAKE + 16), 3), (dict(bytes=5), 3)])
def test_refusals_of_both_entry_points(change, status):
    lib = _lib.load()
    assert _tree_call(lib, **change) == status
    if "V" in change:
        change = dict(change, width=change["V"], ld_probs=max(change["V"], 1))
    assert _chain_call(lib, **change) == status


def test_refusals_of_each():
    lib = _lib.load()
    assert _tree_call(lib, parents=None) == 1 and _tree_call(lib, path=None) == 1
    for change in (dict(probs=None), dict(v=None), dict(width=0), dict(ld_probs=99), dict(width=99), dict(index=FAKE, width=101)):
        assert _chain_call(lib, **change) == 1, change
    assert lib.cfb_verify_workspace(0, 1) == 0 and lib.cfb_verify_workspace(7, 2) >= 7 * 12 + 8


def test_cpu_tensors_are_refused():
    from chain_flow_b200 import tree
    if torch.cuda.is_available():
        pytest.skip("needs a machine without a GPU")
    with pytest.raises((RuntimeError, AssertionError)):
        tree.SampledVerifier(1, 1, 1)


# ---- GPU ----------------------------------------------------------------------------------------------
def _flat(trees):
    cu_d, cu_s, toks, pars = [], [], [], []
    d = s = 0
    for par, tok in trees:
        d += len(par)
        s += len(par) + 1
        cu_d.append(d)
        cu_s.append(s)
        toks += list(tok)
        pars += list(par)
    return (torch.tensor(cu_d, dtype=torch.int32), torch.tensor(cu_s, dtype=torch.int32), torch.tensor(toks, dtype=torch.int32),
            torch.tensor(pars, dtype=torch.int32))


def _case(sizes, V, dtype, seed, spread=2.5):
    """Requests of trees of the given sizes, whose nodes carry tokens that their parents' rows favour."""
    g = torch.Generator().manual_seed(seed)
    rows = sum(n + 1 for n in sizes)
    logits = (torch.randn(rows, V, generator=g) * spread).to(dtype)
    trees, s = [], 0
    for b, n in enumerate(sizes):
        par = [] if n == 0 else [int(p) - 1 for p in make_tree(n + 1, 6, 4, seed=seed + b)[0][1:]]
        tok = []
        for i in range(n):
            row = logits[s + par[i] + 1]
            likely = row.float().topk(min(4, V)).indices
            t = int(likely[i % len(likely)])
            logits[s + par[i] + 1, t] += 3
            tok.append(t)
        trees.append((par, tok))
        s += n + 1
    return logits, _flat(trees), torch.rand(rows, generator=g)


def _check(got, want):
    for a, b in zip(got[:-1], want[:-1]):
        assert torch.equal(a.cpu().long(), b), (a.cpu(), b)
    a, b = got[-1].cpu().double(), want[-1]
    assert torch.equal(torch.isnan(a), torch.isnan(b))
    off = torch.nan_to_num((a - b).abs())
    assert bool((off <= 2.0 ** -16 + 2.0 ** -23 * torch.nan_to_num(b.abs())).all()), float(off.max())


def _sampled(ver, logits, flat, u, temp=None):
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    got = ver(logits.cuda() if not logits.is_cuda else logits, *map(dev, flat), dev(u), temperature=dev(temp))
    torch.cuda.synchronize()
    assert int(ver.err.item()) == 0
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 7, 1000, 1024, 8191, 32003])
def test_sampled_trees(dtype, V):
    from chain_flow_b200.tree import SampledVerifier
    sizes = [12, 0, 1, 5, 30]
    ver = SampledVerifier(60, 6, 30)
    temp = torch.tensor([1.0, 0.3, 0.0, 1.7, 0.9])
    for seed in (1, 2):
        logits, flat, u = _case(sizes, V, dtype, seed)
        _check(_sampled(ver, logits, flat, u, temp), oracle.tree_verify_sampled(logits, *flat, u, temp, 30))
        _check(_sampled(ver, logits, flat, u.double()), oracle.tree_verify_sampled(logits, *flat, u, None, 30))


@pytest.mark.gpu
@pytest.mark.parametrize("requests, n, V, dtype", [(3, 5, 248320, torch.bfloat16), (40, 4, 248320, torch.bfloat16), (200, 2, 70001, torch.float32),
                                                   (310, 1, 65537, torch.float16), (2, 60, 248320, torch.float16)])
def test_sampled_batches(requests, n, V, dtype):
    """From all rows at once to a walk a cluster, with clusters of 8 CTAs down to one."""
    from chain_flow_b200.tree import SampledVerifier
    sizes = [n if b % 5 else max(n - 1, 0) for b in range(requests)]
    logits, flat, u = _case(sizes, V, dtype, 11)
    temp = torch.rand(requests, generator=torch.Generator().manual_seed(3)) * 1.5
    temp[::9] = 0
    ver = SampledVerifier(len(logits), requests, n)
    _check(_sampled(ver, logits, flat, u, temp), oracle.tree_verify_sampled(logits, *flat, u, temp, n))
    assert int(ver.accepted_len.max()) >= 1


@pytest.mark.gpu
@pytest.mark.parametrize("rows_of", ["one", "many"])
def test_rows_that_are_odd(rows_of):
    """Masks, infinities, NaN, temperatures and numbers at their limits; one request a row. "many": so many rows that
    each is a walk of its own."""
    from chain_flow_b200.tree import SampledVerifier
    V = 5003
    g = torch.Generator().manual_seed(5)
    low, inf = torch.finfo(torch.float32).min, math.inf
    base = torch.randn(V, generator=g)
    rows, temps, us = [], [], []

    def add(change, temp=1.0, u=0.5):
        row = base.clone()
        change(row)
        rows.append(row)
        temps.append(temp)
        us.append(u)
    for u in (0.0, 0.37, 1 - 2.0 ** -24, 1.0, -3.0, math.nan, 2.0 ** -40):
        for temp in (0.0, 1.0, 2.0 ** -20, 1e-3, 50.0, 1e35, inf, math.nan, -1.0, 2.0 ** -140):
            add(lambda r: None, temp, u)
    for u in (0.0, 0.4, 0.999):
        for temp in (0.0, 0.8):
            add(lambda r: r.fill_(-inf), temp, u)                                    # nothing left
            add(lambda r: r.fill_(low), temp, u)                                     # masked by the lowest value throughout
            add(lambda r: r[7:].fill_(low), temp, u)
            add(lambda r: r[:-1].fill_(-inf), temp, u)
            add(lambda r: (r.fill_(-inf), r[[3, 1030, 5000]].fill_(0), r.__setitem__(1030, 2.0)), temp, u)
            add(lambda r: r.__setitem__(torch.tensor([5, 4999]), inf), temp, u)      # two share the mass
            add(lambda r: (r.fill_(-inf), r.__setitem__(77, inf)), temp, u)
            add(lambda r: (r.__setitem__(4100, math.nan), r.__setitem__(12, inf)), temp, u)
            add(lambda r: (r.fill_(-inf), r.__setitem__(2, math.nan)), temp, u)
            add(lambda r: (r.fill_(0), r.__setitem__(slice(1000, 2000), 5.0)), temp, u)   # flat: decided in 64 bits
            add(lambda r: (r.fill_(low), r.__setitem__(4, torch.finfo(torch.float32).max)), temp, u)
    if rows_of == "many":
        k = (70 << 20) // (V * 4 * len(rows)) + 1
        rows, temps, us = rows * k, temps * k, us * k
    logits, temp, u = torch.stack(rows), torch.tensor(temps), torch.tensor(us)
    n = len(logits)
    flat = (torch.zeros(n, dtype=torch.int32), torch.arange(1, n + 1, dtype=torch.int32), torch.empty(0, dtype=torch.int32),
            torch.empty(0, dtype=torch.int32))
    ver = SampledVerifier(n, n, 0)
    if rows_of == "one":
        want = oracle.tree_verify_sampled(logits, *flat, u, temp, 0)
    else:
        m = n // k
        want = [t.repeat(k, *[1] * (t.dim() - 1)) for t in oracle.tree_verify_sampled(
            logits[:m], flat[0][:m], flat[1][:m], *flat[2:], u[:m], temp[:m], 0)]
    _check(_sampled(ver, logits, flat, u, temp), want)


@pytest.mark.gpu
@pytest.mark.parametrize("spread", [0.0, 0.5, 3.0])
def test_numbers_next_to_a_border(spread):
    """Numbers 10^-12 to either side of a border between two tokens: nearer than fp32 can tell."""
    from chain_flow_b200.tree import SampledVerifier
    V, n = 20011, 60
    g = torch.Generator().manual_seed(9)
    logits = (torch.randn(n, V, generator=g) * spread).bfloat16()
    u = torch.zeros(n, dtype=torch.float64)
    for r in range(n):
        c = torch.cumsum(torch.softmax(logits[r].double(), 0), 0)
        t = int(torch.randint(V - 1, (1,), generator=g)) if r % 2 else int(logits[r].float().argmax())
        u[r] = c[t] / c[-1] + (1e-12 if r % 4 < 2 else -1e-12)
    flat = (torch.zeros(n, dtype=torch.int32), torch.arange(1, n + 1, dtype=torch.int32), torch.empty(0, dtype=torch.int32),
            torch.empty(0, dtype=torch.int32))
    ver = SampledVerifier(n, n, 0)
    _check(_sampled(ver, logits, flat, u), oracle.tree_verify_sampled(logits, *flat, u, None, 0))


@pytest.mark.gpu
def test_strides_alignment_duplicates_and_limits_of_the_path():
    from chain_flow_b200.tree import SampledVerifier
    V = 3001
    logits, flat, u = _case([6, 6], V, torch.float16, 21)
    wide = torch.full((14, V + 37), 60000.0, dtype=torch.float16)
    wide[:, 3:3 + V] = logits
    view = wide.cuda()[:, 3:3 + V]                       # rows of odd addresses between values that must not be read
    ver = SampledVerifier(14, 2, 6)
    want = oracle.tree_verify_sampled(logits, *flat, u, None, 6)
    _check(_sampled(ver, view, flat, u), want)
    # the same token twice among siblings, tokens outside the vocabulary, indices of 64 bits
    par, tok = [-1, -1, -1, 1], [4, 4, -1, 4]
    logits = torch.full((5, 9), -math.inf)
    logits[:, 4] = 0.0
    flat = _flat([(par, tok)])
    got = _sampled(SampledVerifier(5, 1, 4), logits, tuple(t.long() for t in flat), torch.rand(5))
    assert got[0].tolist() == [[4, 4, -1, -1, -1]] and got[1].tolist() == [[0, -1, -1, -1]]
    # a chain as long as the verifier takes, all accepted; the last row's token follows
    n = 33
    logits = torch.full((n + 1, 50), -math.inf)
    logits[torch.arange(n + 1), torch.arange(n + 1)] = 0.0
    flat = _flat([(list(range(-1, n - 1)), list(range(n)))])
    got = _sampled(SampledVerifier(n + 1, 1, n), logits, flat, torch.rand(n + 1))
    assert got[0].tolist() == [list(range(n + 1))] and got[2].tolist() == [n] and got[1].tolist() == [list(range(n))]


@pytest.mark.gpu
@pytest.mark.parametrize("big", [False, True])
def test_offsets_that_fit_nothing(big):
    from chain_flow_b200.tree import RejectionVerifier, SampledVerifier
    V = 300000 if big else 50                            # more than 64 MiB: a walk a cluster
    rows = 70 if big else 7
    logits = torch.randn(rows, V, device="cuda")
    tok, par = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.full((4,), -1, dtype=torch.int32, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    u = torch.rand(rows, device="cuda")
    for cu_d, cu_s in ((i32(2, 4), i32(3, rows + 3)), (i32(2, 9), i32(3, 6)), (i32(2, 1), i32(3, 6)), (i32(2, 4), i32(3, 1)),
                       (i32(2, -1 << 31), i32(3, 6)), (i32(2, 4), i32(3, 5))):          # (the last: another request's row)
        ver = SampledVerifier(rows, 2, 3)
        out, path, count, logp = ver(logits, cu_d, cu_s, tok, par, u)
        assert int(ver.err.item()) == 7 and out[1].tolist() == [-1] * 4 and path[1].tolist() == [-1] * 3 and int(count[1]) == 0
        assert logp[1].tolist() == [0.0] * 4 and int(out[0, 0]) >= 0
        rej = RejectionVerifier(rows, 2, 3, V)
        out, count, logp = rej(logits, cu_d, cu_s, tok, torch.full((4, V), 1 / V, device="cuda"), u[:4], u[:2])
        assert int(rej.err.item()) == 7 and out[1].tolist() == [-1] * 4 and int(count[1]) == 0 and int(out[0, 0]) >= 0


def _chains(sizes, V, dtype, seed, ids=None, spread=2.5, off=0.7):
    g = torch.Generator().manual_seed(seed)
    rows, drafts = sum(n + 1 for n in sizes), sum(sizes)
    logits = (torch.randn(rows, V, generator=g) * spread).to(dtype)
    cols = V if ids is None else len(ids)
    probs, tok = torch.zeros(drafts, cols), torch.zeros(drafts, dtype=torch.int32)
    d = s = 0
    for n in sizes:
        for i in range(n):
            x = logits[s + i].float() if ids is None else logits[s + i].float()[ids]
            probs[d] = torch.softmax(x + off * torch.randn(cols, generator=g), 0)
            t = int(torch.multinomial(probs[d], 1, generator=g))
            tok[d] = t if ids is None else ids[t]
            d += 1
        s += n + 1
    cu_d = torch.tensor(sizes).cumsum(0).int()
    cu_s = torch.tensor([n + 1 for n in sizes]).cumsum(0).int()
    return logits, (cu_d, cu_s, tok), probs, torch.rand(drafts, generator=g), torch.rand(len(sizes), generator=g)


def _rejected(ver, logits, flat, probs, u, v, temp=None):
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    got = ver(dev(logits), *map(dev, flat), dev(probs), dev(u), dev(v), temperature=dev(temp))
    torch.cuda.synchronize()
    assert int(ver.err.item()) == 0
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V, short", [(1, 0), (2, 1), (9, 4), (1000, 0), (8191, 2000), (32003, 0), (32003, 9001)])
def test_chains_with_draft_probabilities(dtype, V, short):
    from chain_flow_b200.tree import RejectionVerifier
    sizes = [5, 0, 1, 8, 3]
    ids = torch.randperm(V, generator=torch.Generator().manual_seed(1))[:short] if short else None
    ver = RejectionVerifier(30, 6, 8, V, draft_ids=ids)
    temp = torch.tensor([1.0, 0.4, 0.0, 1.3, 0.8])
    for seed in (1, 2):
        logits, flat, probs, u, v = _chains(sizes, V, dtype, seed, ids)
        want = oracle.chain_verify_rejection(logits, *flat, probs, u, v, temp, 8, ids)
        _check(_rejected(ver, logits, flat, probs, u, v, temp), want)
        want = oracle.chain_verify_rejection(logits, *flat, probs, u, v, None, 8, ids)
        _check(_rejected(ver, logits, flat, probs, u.double(), v), want)


@pytest.mark.gpu
@pytest.mark.parametrize("requests, n, V, dtype", [(1, 5, 248320, torch.bfloat16), (30, 4, 248320, torch.bfloat16), (200, 2, 70001, torch.float32),
                                                   (310, 1, 65537, torch.float16)])
def test_batches_of_chains(requests, n, V, dtype):
    from chain_flow_b200.tree import RejectionVerifier
    sizes = [n if b % 5 else n - 1 for b in range(requests)]
    logits, flat, probs, u, v = _chains(sizes, V, dtype, 17)
    ver = RejectionVerifier(len(logits), requests, n, V)
    _check(_rejected(ver, logits, flat, probs, u, v), oracle.chain_verify_rejection(logits, *flat, probs, u, v, None, n))
    assert 0 < int(ver.accepted_len.sum()) < sum(sizes)


@pytest.mark.gpu
def test_draft_probabilities_that_are_odd():
    """Drafts outside the vocabulary, of no probability, in masked places; draft probabilities of the target's own (nothing is
    left above them), above it everywhere, negative, NaN; rows without mass; numbers at their limits."""
    from chain_flow_b200.tree import RejectionVerifier
    V, inf = 2053, math.inf
    g = torch.Generator().manual_seed(6)
    base = torch.randn(V, generator=g) * 2
    p = torch.softmax(base.double(), 0)
    rows, toks, probs, us, vs, temps = [], [], [], [], [], []

    def add(row, tok, q, u, v, temp=1.0):
        rows.append(torch.stack([row, base]))
        toks.append(tok)
        probs.append(q)
        us.append(u)
        vs.append(v)
        temps.append(temp)
    q = torch.softmax(base + 0.5 * torch.randn(V, generator=g), 0)
    top = int(base.argmax())
    masked = base.clone()
    masked[top], masked[100:] = -inf, -inf
    for v in (0.0, 0.5, 1.0, math.nan, 1 - 2.0 ** -24):
        for u in (0.0, 1.0, 0.999):
            for tok in (-1, V, 1 << 30, -1 << 31, top, 7, V - 1):
                add(base, tok, q, u, v)
            for tok in (top, 7, 200):
                add(masked, tok, q, u, v)
                add(torch.full((V,), -inf), tok, q, u, v)
                add(base, tok, p.float(), u, v)                             # the target's own
                add(base, tok, (2 * p).float(), u, v)                       # above it everywhere
                add(base, tok, torch.zeros(V), u, v)
                add(base, tok, -q, u, v)
                add(base, tok, torch.where(torch.arange(V) % 3 == 0, torch.full((V,), math.nan), q), u, v)
                add(base, tok, q, u, v, 0.0)
                add(base, tok, q, u, v, 0.05)
                nan = base.clone()
                nan[1500] = math.nan
                add(nan, tok, q, u, v)
                many = base.clone()
                many[[3, 7, 1900]] = inf
                add(many, tok, q, u, v)
    n = len(rows)
    logits, probs = torch.cat(rows), torch.stack(probs)
    flat = (torch.arange(1, n + 1).int(), (2 * torch.arange(1, n + 1)).int(), torch.tensor(toks, dtype=torch.int32))
    u, v, temp = torch.tensor(us), torch.tensor(vs), torch.tensor(temps)
    ver = RejectionVerifier(2 * n, n, 1, V)
    _check(_rejected(ver, logits, flat, probs, u, v, temp), oracle.chain_verify_rejection(logits, *flat, probs, u, v, temp, 1))


@pytest.mark.gpu
def test_chains_next_to_a_border():
    """Accepting numbers 10^-13 to either side of p / q, and drawing numbers 10^-12 to either side of a border of what is left."""
    from chain_flow_b200.tree import RejectionVerifier
    V, n = 4001, 60
    logits, flat, probs, u, v = _chains([1] * n, V, torch.float32, 33, spread=1.0)
    u, v = u.double(), v.double()
    g = torch.Generator().manual_seed(2)
    for r in range(n):
        p, q, t = torch.softmax(logits[2 * r].double(), 0), probs[r].double(), int(flat[2][r])
        side = 1 if r % 4 < 2 else -1
        if r % 2:
            u[r] = float(p[t] / q[t]) * (1 + side * 1e-13)
        else:
            u[r] = 1.0
            rest = (p - q).clamp_min(0)
            c = torch.cumsum(rest, 0)
            v[r] = c[int(torch.randint(V - 1, (1,), generator=g))] / c[-1] + side * 1e-12
    ver = RejectionVerifier(2 * n, n, 1, V)
    _check(_rejected(ver, logits, flat, probs, u, v), oracle.chain_verify_rejection(logits, *flat, probs, u, v, None, 1))


@pytest.mark.gpu
def test_capture_streams_and_refusals(monkeypatch):
    from chain_flow_b200.tree import RejectionVerifier, SampledVerifier
    logits, flat, u = _case([6, 3, 0], 5000, torch.bfloat16, 41)
    want = oracle.tree_verify_sampled(logits, *flat, u, None, 6)
    dev = [t.cuda() for t in (logits, *flat, u)]
    ver, other = SampledVerifier(12, 3, 6), SampledVerifier(12, 3, 6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = ver(*dev, stream=side)
    again = other(*dev)                                  # two calls at once, a verifier each
    torch.cuda.synchronize()
    _check(got, want)
    _check(again, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ver(*dev)
    for seed in (42, 43):                                # replayed over other inputs
        logits, flat, u = _case([6, 3, 0], 5000, torch.bfloat16, seed)
        for d, t in zip(dev, (logits, *flat, u)):
            d.copy_(t)
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        _check(got, oracle.tree_verify_sampled(logits, *flat, u, None, 6))
    lg, cu_d, cu_s, tok, par, u = dev
    for bad in ((lg.double(), cu_d, cu_s, tok, par, u), (lg.t(), cu_d, cu_s, tok, par, u), (lg[0], cu_d, cu_s, tok, par, u),
                (lg, cu_d.float(), cu_s, tok, par, u), (lg, cu_d, cu_s[:2], tok, par, u), (lg, cu_d, cu_s, tok, par[:3], u),
                (lg, cu_d, cu_s, tok, par, u[:3]), (lg, cu_d, cu_s, tok, par, u.half()), (lg.cpu(), cu_d, cu_s, tok, par, u),
                (lg, cu_d, cu_s, tok, par, u.cpu()), (torch.cat([lg, lg]), cu_d, cu_s, tok, par, torch.cat([u, u])),
                (lg[:1].expand(12, -1), cu_d, cu_s, tok, par, u), (lg[:, :0], cu_d, cu_s, tok, par, u), (lg[:0], cu_d, cu_s, tok, par, u[:0])):
        with pytest.raises(_lib.CfbError):
            ver(*bad)
    for temp in (u[:2], torch.ones(3, dtype=torch.int32, device="cuda"), torch.ones(3)):
        with pytest.raises(_lib.CfbError):
            ver(*dev, temperature=temp)
    assert ver(lg, cu_d[:0], cu_s[:0], tok[:0], par[:0], u)[0].shape == (0, 7)
    rej = RejectionVerifier(12, 3, 6, 5000)
    q = torch.full((9, 5000), 2e-4, device="cuda")
    for bad in ((q[:, :4999], u[:9], u[:3]), (q.half(), u[:9], u[:3]), (q[:8], u[:9], u[:3]), (q, u[:8], u[:3]), (q, u[:9], u[:2]),
                (q[:1].expand(9, -1), u[:9], u[:3]), (q.cpu(), u[:9], u[:3])):
        with pytest.raises(_lib.CfbError):
            rej(lg, cu_d, cu_s, tok, *bad)
    with pytest.raises(_lib.CfbError):
        rej(lg[:, :4000], cu_d, cu_s, tok, q, u[:9], u[:3])
    for ids in ([1, 1], [5000], [-1], []):
        with pytest.raises(_lib.CfbError):
            RejectionVerifier(12, 3, 6, 5000, draft_ids=torch.tensor(ids, dtype=torch.int64))
    for args in ((0, 1, 1), (1, 0, 1), (1, 1, -1), (1, 1, 1025)):
        with pytest.raises(_lib.CfbError):
            SampledVerifier(*args)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    with pytest.raises(_lib.CfbError, match="current device"):
        ver(*dev)
    with pytest.raises(_lib.CfbError, match="current device"):
        rej(lg, cu_d, cu_s, tok, q, u[:9], u[:3])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [777, 4096, 40001])
def test_rows_that_are_odd_in_16_bits(dtype, V):
    from chain_flow_b200.tree import RejectionVerifier, SampledVerifier
    g = torch.Generator().manual_seed(V)
    info, inf = torch.finfo(dtype), math.inf
    rows = []
    for change in (lambda r: None, lambda r: r.fill_(info.min), lambda r: r.fill_(-inf), lambda r: r[5:].fill_(info.min),
                   lambda r: (r.fill_(-inf), r[V - 1:].fill_(-3.0)), lambda r: r[[1, V - 2]].fill_(inf), lambda r: r.__setitem__(torch.tensor([1, V - 2]), inf),
                   lambda r: r.__setitem__(700, math.nan), lambda r: (r.fill_(info.min), r.__setitem__(V // 2, info.max)), lambda r: r.fill_(0),
                   lambda r: r.fill_(info.max), lambda r: r.mul_(100)):
        row = (torch.randn(V, generator=g) * 3).to(dtype)
        change(row)
        rows += [row] * 4
    n = len(rows)
    logits, u = torch.stack(rows), torch.rand(n, generator=g, dtype=torch.float64)
    temp = torch.tensor([1.0, 0.0, 0.2, 3.0] * (n // 4))
    flat = (torch.zeros(n, dtype=torch.int32), torch.arange(1, n + 1, dtype=torch.int32), torch.empty(0, dtype=torch.int32),
            torch.empty(0, dtype=torch.int32))
    _check(_sampled(SampledVerifier(n, n, 0), logits, flat, u, temp), oracle.tree_verify_sampled(logits, *flat, u, temp, 0))
    both = torch.stack([r for row in rows for r in (row, rows[0])])
    tok = torch.randint(V, (n,), generator=g, dtype=torch.int32)
    tok[::3] = both[::2].float().nan_to_num(0).argmax(1).int()[::3]
    q = torch.softmax(torch.randn(n, V, generator=g) * 3, 1)
    flat = (torch.arange(1, n + 1).int(), (2 * torch.arange(1, n + 1)).int(), tok)
    args = (both, *flat, q, u, torch.rand(n, generator=g, dtype=torch.float64), temp)
    ver = RejectionVerifier(2 * n, n, 1, V)
    _check(_rejected(ver, both, flat, *args[4:]), oracle.chain_verify_rejection(*args, 1))


@pytest.mark.gpu
def test_verifiers_far_larger_than_their_calls():
    """A verifier for 1024 drafts and many requests, given few; lists that name columns outside the draft probabilities."""
    from chain_flow_b200.tree import RejectionVerifier, SampledVerifier
    logits, flat, u = _case([3, 0, 7], 2000, torch.float32, 5)
    ver = SampledVerifier(4000, 900, 1024)
    _check(_sampled(ver, logits, flat, u), oracle.tree_verify_sampled(logits, *flat, u, None, 1024))
    V = 600
    logits, flat, probs, u, v = _chains([4, 2], V, torch.float16, 3)
    ver = RejectionVerifier(50, 9, 64, V, draft_ids=torch.arange(V))
    ver.index_of[::2] = 1 << 30                          # as a C caller's list may be wrong: read as probability 0
    probs[:, ::2] = 0
    _check(_rejected(ver, logits, flat, probs, u, v), oracle.chain_verify_rejection(logits, *flat, probs, u, v, None, 64))


@pytest.mark.gpu
def test_calls_of_other_sizes_on_one_verifier():
    """Few requests of many rows, then many of few: nothing of one call is left for the next."""
    from chain_flow_b200.tree import RejectionVerifier, SampledVerifier
    tree, chain = SampledVerifier(300, 150, 8), RejectionVerifier(300, 150, 8, 500)
    for turn, sizes in enumerate([[8] * 12, [1] * 150, [8] * 30, [0, 1] * 70, [2]]):
        logits, flat, u = _case(sizes, 500, torch.bfloat16, turn)
        _check(_sampled(tree, logits, flat, u), oracle.tree_verify_sampled(logits, *flat, u, None, 8))
        logits, flat, probs, u, v = _chains(sizes, 500, torch.bfloat16, turn)
        _check(_rejected(chain, logits, flat, probs, u, v), oracle.chain_verify_rejection(logits, *flat, probs, u, v, None, 8))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [(1 << 20) + 3, (1 << 22) - 8])
def test_the_largest_vocabularies(V):
    from chain_flow_b200.tree import RejectionVerifier, SampledVerifier
    sizes = [1, 2]
    logits, flat, u = _case(sizes, V, torch.float16, 4)
    ver = SampledVerifier(5, 2, 2)
    _check(_sampled(ver, logits, flat, u), oracle.tree_verify_sampled(logits, *flat, u, None, 2))
    logits, flat, probs, u, v = _chains(sizes, V, torch.float16, 4)
    ver = RejectionVerifier(5, 2, 2, V)
    _check(_rejected(ver, logits, flat, probs, u, v), oracle.chain_verify_rejection(logits, *flat, probs, u, v, None, 2))
    # 160 requests, a CTA each: the whole vocabulary's sums in one
    logits = (torch.randn(4, V, generator=torch.Generator().manual_seed(6)) * 2.5).half().cuda().repeat(40, 1)
    flat, u = (torch.zeros(160).int(), torch.arange(1, 161).int(), torch.zeros(0).int(), torch.zeros(0).int()), torch.rand(160)
    got = _sampled(SampledVerifier(160, 160, 0), logits, flat, u)
    want = oracle.tree_verify_sampled(logits[:4].cpu(), flat[0][:4], flat[1][:4], *flat[2:], u[:4], None, 0)
    assert torch.equal(got[0][:4].cpu().long(), want[0]) and bool((got[0] >= 0).all())


def test_random_numbers_at_an_address_that_is_no_elements():
    lib = _lib.load()
    assert _tree_call(lib, u=FAKE + 4, size=8) == 1 and _tree_call(lib, u=FAKE + 2) == 1
    for change in (dict(u=FAKE + 4, size=8), dict(v=FAKE + 4, size=8), dict(v=FAKE + 1)):
        assert _chain_call(lib, **change) == 1, change


@pytest.mark.gpu
@pytest.mark.parametrize("V, n", [(30011, 120), (140001, 190)])
def test_rows_that_rise_and_fall_next_to_a_border(V, n):
    """Rows whose largest element changes all along (every unit's sums change their base), at temperatures that fp32 holds
    badly, with numbers from 10^-12 to 10^-4 beside a border: around and below what an fp32 sum is off by."""
    from chain_flow_b200.tree import RejectionVerifier, SampledVerifier
    g = torch.Generator().manual_seed(7)
    i = torch.arange(V, dtype=torch.float64)
    shapes = [12 * i / V, 12 - 12 * i / V, 6 + 6 * torch.sin(i / 900), (i % 1024) / 90, 10 - 300 * (i / V - 0.5) ** 2, 0 * i]
    temps = [1.0, 0.7, 1.3, 1 / 3, 2.1]
    logits = torch.stack([shapes[r % 6] + 0.3 * torch.randn(V, generator=g) for r in range(n)]).float()
    temp = torch.tensor([temps[r // 6 % 5] for r in range(n)])
    u, off = torch.zeros(n, dtype=torch.float64), [1e-12, 1e-9, 3e-8, 3e-7, 1e-6, 3e-6, 1e-5, 1e-4]
    q, v = torch.zeros(n, V), torch.zeros(n, dtype=torch.float64)
    for r in range(n):
        p = torch.softmax(logits[r].double() / temp[r].double(), 0)
        c = torch.cumsum(p, 0)
        t = int(torch.searchsorted(c, torch.rand(1, generator=g, dtype=torch.float64)).clamp(max=V - 2))
        side = off[int(torch.randint(8, (1,), generator=g))] * (1 if torch.rand(1, generator=g) < 0.5 else -1)
        u[r] = c[t] / c[-1] + side
        q[r] = torch.softmax(logits[r].double() / temp[r].double() + 0.5 * torch.randn(V, generator=g), 0).float()
        c = torch.cumsum((p - q[r].double()).clamp_min(0), 0)
        t = int(torch.searchsorted(c, c[-1] * torch.rand(1, generator=g, dtype=torch.float64)).clamp(max=V - 2))
        v[r] = c[t] / c[-1] + side
    none, ends = torch.zeros(0, dtype=torch.int32), torch.arange(1, n + 1, dtype=torch.int32)
    flat = (torch.zeros(n, dtype=torch.int32), ends, none, none)
    _check(_sampled(SampledVerifier(n, n, 0), logits, flat, u, temp), oracle.tree_verify_sampled(logits, *flat, u, temp, 0))
    m = n // 2                                           # a draft of each, refused: the draw is from what is left
    chain = (ends[:m], 2 * ends[:m], torch.full((m,), -1, dtype=torch.int32))
    rows = logits[:m].repeat_interleave(2, 0)
    args = (rows, *chain, q[:m], torch.zeros(m), v[:m], temp[:m])
    _check(_rejected(RejectionVerifier(2 * m, m, 1, V), rows, chain, *args[4:]), oracle.chain_verify_rejection(*args, 1))
