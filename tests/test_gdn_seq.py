"""The gated delta rule over sequences (cfb_gdn_chunk, cfb_gdn_step).

CPU: the oracle's walk equals the tree verify's oracle on a chain, and the entry points refuse what
they do not take. GPU: against oracle.gdn_sequence (64 bits). Tolerances, as a 2-norm relative to
the request's result per value head:
* state: fp32 throughout. Products whose operands are split keep 22 bits (2^-22 relative a factor,
  three factors a chunk of tokens), and sums of fp32; the errors of successive chunks add at worst
  linearly: 4e-6 covers the lengths here. The token-by-token walk rounds each element three
  times a token, 2^-24 each: the same bound.
* o: rounded once to its type (u = 2^-8 bf16, 2^-11 fp16), from products whose operands keep at
  least 11 bits (2^-11 each, two terms): u + 2 * 2^-11."""
import ctypes as C

import pytest
import torch

import oracle
from chain_flow_b200 import _lib

ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
STATE_RTOL = 4e-6


def _case(lens, H=2, HV=4, V=128, dtype=torch.float16, gate=torch.float32, seed=0, realistic=True, zero_start=True):
    g = torch.Generator().manual_seed(seed)
    T, B, K = sum(lens), len(lens), 128
    wide = torch.randn(T, 2 * H * K + HV * V + 16, generator=g).to(dtype)           # a fused projection's rows
    q = wide[:, :H * K].view(T, H, K)
    k = wide[:, H * K:2 * H * K].view(T, H, K)
    v = wide[:, 2 * H * K:2 * H * K + HV * V].view(T, HV, V)
    if realistic:
        A_log = torch.log(1 + 15 * torch.rand(HV, generator=g))
        step = torch.exp(-6.9 + 4.6 * torch.rand(HV, generator=g))
        dt_bias = step + torch.log(-torch.expm1(-step))
    else:
        A_log, dt_bias = torch.randn(HV, generator=g) * 0.5, torch.randn(HV, generator=g) * 0.5
    slots = B + 2
    order = torch.randperm(slots, generator=g)[:B].int()
    init = order.clone()
    if B > 1 and zero_start:
        init[1] = -1
    return dict(A_log=A_log.to(gate), dt_bias=dt_bias.to(gate), a=torch.randn(T, HV, generator=g).to(gate),
                b=torch.randn(T, HV, generator=g).to(gate), q=q, k=k, v=v,
                state=torch.randn(slots, HV, V, K, generator=g) * 0.1, cu=torch.tensor([0] + list(lens)).cumsum(0).int(),
                init=init, to=order)


def _oracle(c, scale=128 ** -0.5):
    return oracle.gdn_sequence(c["A_log"], c["dt_bias"], c["a"], c["b"], c["q"], c["k"], c["v"], c["state"], c["cu"], c["init"],
                               c["to"], scale)


def _gpu(c):
    d = {n: t.cuda() for n, t in c.items()}
    H, K, HV, V = *c["q"].shape[1:], *c["v"].shape[1:]
    wide = torch.cat([d["q"].flatten(1), d["k"].flatten(1), d["v"].flatten(1), torch.zeros(len(d["q"]), 16, device="cuda", dtype=d["q"].dtype)], 1)
    d["q"], d["k"] = wide[:, :H * K].view(-1, H, K), wide[:, H * K:2 * H * K].view(-1, H, K)
    d["v"] = wide[:, 2 * H * K:2 * H * K + HV * V].view(-1, HV, V)
    d["o"] = torch.full((len(wide), HV, V), 7.0, device="cuda", dtype=wide.dtype)
    return d


def _run(d, step=False, scale=128 ** -0.5, **kw):
    from chain_flow_b200.gdn import ChunkedGdn, gdn_step
    args = (d["A_log"], d["dt_bias"], d["a"], d["b"], d["q"], d["k"], d["v"], d["o"], d["state"])
    if step:
        gdn_step(*args, d["init"], d["to"], scale=scale, **kw)
    else:
        ChunkedGdn(len(d["q"]), len(d["init"]), d["v"].shape[1])(*args, d["cu"], d["init"], d["to"], scale=scale, **kw)
    torch.cuda.synchronize()


def _rel(got, want, dims):
    n = want.norm(dim=dims)
    return ((got.double().cpu() - want).norm(dim=dims) / n.clamp_min(1e-30))[n > 0]


def _check(o, state, c, want):
    wo, ws = want
    u = ROUND[c["q"].dtype]
    for r in range(len(c["init"])):
        t0, t1 = int(c["cu"][r]), int(c["cu"][r + 1])
        if t1 > t0:
            assert float(_rel(o[t0:t1], wo[t0:t1], (0, 2)).max()) <= u + 2 * 2.0 ** -11
    rel = _rel(state, ws, (2, 3))
    assert float(rel.max()) <= STATE_RTOL, float(rel.max())


def test_oracle_sequence_equals_the_verify_walk_of_a_chain():
    c = _case([7], realistic=False)
    T = 7
    chain = torch.tensor([[t - j if j <= t else 0 for j in range(T)] for t in range(T)], dtype=torch.int32)
    depth = torch.arange(T, dtype=torch.int32)
    out = torch.arange(1, T + 1, dtype=torch.int32)
    state = torch.cat([c["state"][c["init"].long()], torch.zeros(T, *c["state"].shape[1:])])
    o, st = oracle.tree_gdn_verify(c["A_log"], c["dt_bias"], c["a"], c["b"], c["q"], c["k"], c["v"], state, chain, depth, out,
                                   torch.zeros(T, dtype=torch.int32), 128 ** -0.5)
    o2, st2 = _oracle(c)
    assert float((o - o2).abs().max()) < 1e-5 and float((st[T] - st2[int(c["to"][0])]).abs().max()) < 1e-5


FAKE = 0x10000


def _args(**kw):
    a = dict(A_log=FAKE, A_log_dtype=0, dt_bias=FAKE, dt_bias_dtype=0, a=FAKE, a_dtype=0, a_stride=4, b=FAKE, b_dtype=0, b_stride=4,
             q=FAKE, q_stride=256, k=FAKE, k_stride=256, v=FAKE, v_stride=512, o=FAKE, o_stride=512, dtype=1, state_in=FAKE,
             state_out=FAKE, slot_stride=4 * 128 * 128, slots=3, init_slot=FAKE, out_slot=FAKE, scale=0.1, H=2, HV=4, K=128, V=128)
    a.update(kw)
    return _lib.GdnArgs(*[a[n] for n, _ in _lib.GdnArgs._fields_])


@pytest.mark.parametrize("change, status", [
    (dict(q=None), 1), (dict(state_out=None), 1), (dict(out_slot=None), 1), (dict(a_dtype=3), 1), (dict(dtype=0), 2), (dict(K=64), 2),
    (dict(V=48), 2), (dict(H=3), 2), (dict(H=0), 1), (dict(slots=0), 1), (dict(q_stride=257), 1), (dict(v=FAKE + 2), 1),
    (dict(state_in=FAKE + 4), 1), (dict(slot_stride=4 * 128 * 128 - 4), 1)])
def test_refusals_of_the_c_entry_points(change, status):
    lib = _lib.load()
    g = _args(**change)
    n = lib.cfb_gdn_chunk_workspace(4, 1, 4)
    assert lib.cfb_gdn_step(C.byref(g), 1, None) == status
    assert lib.cfb_gdn_chunk(C.byref(g), FAKE, 4, 1, FAKE, n, None) == status


def test_refusals_of_the_chunk_call():
    lib = _lib.load()
    g = _args()
    n = lib.cfb_gdn_chunk_workspace(4, 1, 4)
    call = lambda cu=FAKE, T=4, B=1, ws=FAKE, size=n: lib.cfb_gdn_chunk(C.byref(g), cu, T, B, ws, size, None)
    assert call(B=0) == 0 and call(cu=None) == 1 and call(T=-1) == 1 and call(B=-1) == 1 and call(ws=None) == 1
    assert call(ws=FAKE + 8) == 3 and call(size=8) == 3
    assert lib.cfb_gdn_step(None, 1, None) == 1 and lib.cfb_gdn_step(C.byref(g), 0, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, gate", [(torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("lens, H, HV, V", [
    ([1], 2, 4, 128), ([31, 32, 33, 0, 1], 2, 4, 128), ([63, 64, 65, 2], 1, 3, 32), ([200, 5], 2, 2, 64), ([300], 1, 2, 96),
    ([3, 100, 16, 17, 15, 1, 1, 7, 129], 2, 4, 128)])
def test_sequences(dtype, gate, lens, H, HV, V):
    c = _case(lens, H, HV, V, dtype, gate, seed=sum(lens))
    want = _oracle(c)
    d = _gpu(c)
    out = d["state"].clone()
    _run(d, out_state=out)
    assert torch.equal(d["state"].cpu(), c["state"])
    _check(d["o"], out, c, want)
    again, o1 = d["state"].clone(), d["o"].clone()
    _run(d, out_state=again)
    assert torch.equal(again, out) and torch.equal(o1, d["o"])                      # the same bits every time
    _run(d)                                                                          # in place
    assert torch.equal(d["state"], out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, gate", [(torch.float16, torch.float16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("B, H, HV, V", [(1, 16, 32, 128), (5, 2, 4, 64), (70, 1, 2, 32)])
def test_single_tokens(dtype, gate, B, H, HV, V):
    c = _case([1] * B, H, HV, V, dtype, gate, seed=B, realistic=False)
    want = _oracle(c)
    d = _gpu(c)
    _run(d, step=True)
    _check(d["o"], d["state"], c, want)


@pytest.mark.gpu
def test_strong_and_weak_decays():
    """Heads that forget at once, that never forget, and gates at their ends (decay 0 and 1, beta 0 and 1)."""
    c = _case([130], 1, 4, 32, torch.float16, seed=11)
    c["A_log"] = torch.tensor([6.0, -20.0, 0.0, 2.0])
    c["a"][40:60, 2], c["a"][60:80, 2] = 90.0, -90.0
    c["b"][20:50, 3], c["b"][50:70, 3] = 90.0, -90.0
    c["a"][10, 0] = 1e4
    d = _gpu(c)
    _run(d)
    _check(d["o"], d["state"], c, _oracle(c))


@pytest.mark.gpu
def test_repeated_and_zero_keys():
    """The same key at every token (the update's matrix has its largest entries), and rows of zeros."""
    c = _case([100], 1, 2, 64, torch.bfloat16, seed=12)
    c["k"][:] = c["k"][0].clone()
    c["k"][50:60], c["q"][55:65], c["v"][70:75] = 0, 0, 0
    c["b"][:] = 8.0
    d = _gpu(c)
    _run(d)
    _check(d["o"], d["state"], c, _oracle(c))


@pytest.mark.gpu
@pytest.mark.parametrize("step", [False, True])
def test_slots_outside_the_pool_and_untouched_ones(step):
    c = _case([1, 1, 1] if step else [40, 3, 20], seed=13)
    d = _gpu(c)
    c["to"] = torch.tensor([-1, 4, 0], dtype=torch.int32)                          # 5 slots: 0 .. 4
    c["init"] = torch.tensor([3, 1, -1], dtype=torch.int32)
    want = _oracle(c)
    d["init"], d["to"] = c["init"].cuda(), c["to"].cuda()
    out = torch.full_like(d["state"], 5.0)
    _run(d, step=step, out_state=out)
    assert bool((out[1:4] == 5).all())
    assert float(_rel(out[[0, 4]], want[1][[0, 4]], (2, 3)).max()) <= STATE_RTOL
    d["init"][0], d["to"][2] = 5, 99                                               # no such slots
    out.fill_(5.0)
    t0, t1 = int(c["cu"][0]), int(c["cu"][1])
    _run(d, step=step, out_state=out)
    assert bool(torch.isnan(d["o"][t0:t1]).all()) and bool((out[:4] == 5).all()) and bool(torch.isfinite(out[4]).all())


@pytest.mark.gpu
def test_rows_of_no_request_and_bad_offsets():
    c = _case([20, 30], seed=14)
    d = _gpu(c)
    want = _oracle({**c, "cu": torch.tensor([5, 20, 44])})
    d["cu"] = torch.tensor([5, 20, 44], dtype=torch.int32, device="cuda")
    _run(d)
    assert bool((d["o"][:5] == 7).all()) and bool((d["o"][44:] == 7).all())
    assert float(_rel(d["o"][5:44], want[0][5:44], (0, 2)).max()) <= ROUND[torch.float16] + 2 * 2.0 ** -11
    d["cu"] = torch.tensor([-7, 20, 900], dtype=torch.int32, device="cuda")        # clamped into the rows there are
    d["state"].copy_(c["state"])
    _run(d)
    want = _oracle({**c, "cu": torch.tensor([0, 20, 50])})
    _check(d["o"], d["state"], {**c, "cu": torch.tensor([0, 20, 50])}, want)


@pytest.mark.gpu
def test_nan_stays_in_its_request_and_head():
    c = _case([40, 40], 1, 2, 64, torch.float16, seed=15)
    d = _gpu(c)
    d["v"][10, 1, 3] = float("nan")                                                # request 0, value head 1, row 3
    out = d["state"].clone()
    _run(d, out_state=out)
    o = d["o"]
    assert bool(torch.isfinite(o[:, 0]).all()) and bool(torch.isfinite(o[40:]).all()) and bool(torch.isfinite(o[:10]).all())
    assert bool(torch.isnan(o[10:40, 1, 3]).all()) and bool(torch.isnan(out[c["to"][0], 1, 3]).all())
    keep = [i for i in range(64) if i != 3]
    assert bool(torch.isfinite(o[:40, 1, keep]).all())


@pytest.mark.gpu
def test_one_walk_equals_its_pieces_and_the_verify():
    """A prompt in two chunks then single tokens: the states and outputs of one call over all of it; and
    the tree verify's walk of a chain from the chunk's state gives the next tokens' outputs."""
    from chain_flow_b200.gdn import gdn_verify
    c = _case([75], seed=16, zero_start=False)
    d = _gpu(c)
    whole = d["state"].clone()
    _run(d, out_state=whole)
    slot = int(c["to"][0])
    p = {n: (t.clone() if n == "state" else t) for n, t in d.items()}
    o = torch.zeros_like(d["o"])
    for t0, t1 in ((0, 50), (50, 72), (72, 73), (73, 74), (74, 75)):
        x = {**p, **{n: p[n][t0:t1] for n in ("q", "k", "v", "a", "b")}, "o": o[t0:t1]}
        x["cu"] = torch.tensor([0, t1 - t0], dtype=torch.int32, device="cuda")
        if t1 == 72:
            before = None
        _run(x, step=t1 - t0 == 1)
        if t1 == 72:
            before = p["state"].clone()
    assert float(_rel(p["state"][slot], whole[slot].double().cpu(), (1, 2)).max()) <= 2 * STATE_RTOL
    assert float(_rel(o, d["o"].double().cpu(), (0, 2)).max()) <= 2 * (ROUND[torch.float16] + 2 * 2.0 ** -11)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    st = torch.cat([before[slot:slot + 1], torch.zeros(3, *before.shape[1:], device="cuda")])
    vo = torch.zeros(3, *d["v"].shape[1:], device="cuda", dtype=torch.float16)
    gdn_verify(d["A_log"], d["dt_bias"], d["a"][72:].contiguous(), d["b"][72:].contiguous(), d["q"][72:].contiguous(),
               d["k"][72:].contiguous(), d["v"][72:].contiguous(), vo, st, i32([[0, 0, 0], [1, 0, 0], [2, 1, 0]]), i32([0, 1, 2]),
               i32([1, 2, 3]), i32([0, 0, 0]), scale=128 ** -0.5)
    torch.cuda.synchronize()
    assert float(_rel(vo, o[72:].double().cpu(), (0, 2)).max()) <= 2 * (ROUND[torch.float16] + 2 * 2.0 ** -11)
    assert float(_rel(st[3], p["state"][slot].double().cpu(), (1, 2)).max()) <= 2 * STATE_RTOL


@pytest.mark.gpu
@pytest.mark.parametrize("step", [False, True])
def test_another_stream_and_capture(step):
    c = _case([1, 1] if step else [50, 9], seed=17)
    d = _gpu(c)
    want = d["state"].clone()
    _run(d, step=step, out_state=want)
    side = torch.cuda.Stream()
    out = d["state"].clone()
    side.wait_stream(torch.cuda.current_stream())
    _run({**d, "init": d["init"].long(), "to": d["to"].long(), "cu": d["cu"].long()}, step=step, out_state=out, stream=side)
    assert torch.equal(out, want)
    from chain_flow_b200.gdn import ChunkedGdn, gdn_step
    args = (d["A_log"], d["dt_bias"], d["a"], d["b"], d["q"], d["k"], d["v"], d["o"], d["state"])
    chunk = ChunkedGdn(len(d["q"]), 2, 4)
    graph = torch.cuda.CUDAGraph()
    out.zero_()
    with torch.cuda.graph(graph):
        if step:
            gdn_step(*args, d["init"], d["to"], scale=128 ** -0.5, out_state=out)
        else:
            chunk(*args, d["cu"], d["init"], d["to"], scale=128 ** -0.5, out_state=out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[d["to"].long()], want[d["to"].long()])


@pytest.mark.gpu
def test_refusals_in_python():
    from chain_flow_b200.gdn import ChunkedGdn, gdn_step
    d = _gpu(_case([4, 3], seed=18))
    names = ("A_log", "dt_bias", "a", "b", "q", "k", "v", "o", "state")
    for change in (dict(q=d["q"].float()), dict(k=d["k"].bfloat16()), dict(v=d["v"][:5]), dict(a=d["a"].double()), dict(a=d["a"][:, :2]),
                   dict(state=d["state"].half()), dict(state=d["state"].transpose(2, 3)), dict(init=d["init"][:1]), dict(init=d["init"].cpu()),
                   dict(q=d["q"].cpu()), dict(o=d["o"].transpose(1, 2).contiguous().transpose(1, 2))):
        x = {**d, **change}
        with pytest.raises(_lib.CfbError):
            ChunkedGdn(7, 2, 4)(*[x[n] for n in names], x["cu"], x["init"], x["to"], scale=0.1)
    for limits in ((6, 2, 4), (7, 1, 4), (7, 2, 3)):
        with pytest.raises(_lib.CfbError):
            ChunkedGdn(*limits)(*[d[n] for n in names], d["cu"], d["init"], d["to"], scale=0.1)
    with pytest.raises(_lib.CfbError):
        gdn_step(*[d[n] for n in names], d["init"], d["to"], scale=0.1)             # 7 rows, 2 slots
