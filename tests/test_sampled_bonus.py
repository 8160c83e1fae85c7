"""The example's sampled steps leave no token out: each begins with the one that the step before ended with, which joins the
context and the state before the tree that hangs below it. The last decode against whole sequences in 64 bits
(tolerances as in test_target_step.py)."""
import ast
import re
import sys

import pytest
import torch

import oracle
from chain_flow_b200.gdn import make_tree
from test_sampled_step import FP32, U, _example


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [torch.float8_e4m3fn, torch.float16])
def test_committed_tokens_join_before_the_tree(cache):
    ex = _example()
    news, S, N, V, steps = [31, 16], 3, 7, 200, 3
    layers = ex.SampledTarget(S, max(news) + steps * (N + 1) + 1, N, cache_dtype=cache)
    xp = ex.projections(sum(news), seed=1)
    layers.prompt(xp, news + [0])
    layers.fork(torch.tensor([1], device="cuda"), torch.tensor([2], device="cuda"))
    of = [0, 1, 1]
    cpu = lambda x: {n: t.cpu() for n, t in x.items()}  # noqa: E731
    P = cpu(xp)
    starts = [sum(news[:p]) for p in of]
    seqs = [[{n: t[s:s + news[p]] for n, t in P.items()}] for p, s in zip(of, starts)]
    g = torch.Generator().manual_seed(8)
    for step in range(steps):
        x, c = ex.projections(S * N, seed=10 + step), ex.projections(S, seed=40 + step)
        parents = torch.stack([make_tree(N, 4, 3, seed=step * S + b)[0] for b in range(S)])
        logits = 2 * torch.randn(S * (N + 1), V, generator=g)
        best = logits.view(S, N + 1, V).argmax(2)
        tokens = best.gather(1, parents + 1)
        u = torch.rand(S * (N + 1), generator=g)
        temp = torch.tensor([0.0, 0.3, 0.2])
        _, _, out = layers.sampled_step(x, parents.cuda(), tokens.cuda(), logits.cuda(), u.cuda(), temp.cuda(), committed=c)
        b1 = torch.arange(1, S + 1)
        want = oracle.tree_verify_sampled(logits, b1 * N, b1 * (N + 1), tokens.flatten(), parents.flatten(), u, temp, N)
        for a, b in zip(out[:3], want):
            assert torch.equal(a.cpu().long(), b)
        for b in range(S):
            seqs[b].append({n: t[b:b + 1] for n, t in cpu(c).items()})
            seqs[b].append({n: t[[b * N + i for i in want[1][b].tolist() if i >= 0]] for n, t in cpu(x).items()})
    seqs = [{n: torch.cat([p[n] for p in parts]) for n in P} for parts in seqs]
    lens = [len(s["a"]) for s in seqs]
    assert layers.kv_len.tolist() == lens and sum(lens) > sum(news[p] for p in of) + S * steps
    xd = ex.projections(S, seed=30)
    attn, o = layers.decode(xd)
    layers.attention.check()
    layers.chunks.check()
    assert all(bool(t.all()) for t in layers.granted) and int(layers.pool.err.item()) == 0
    table = layers.table.tolist()
    assert layers.pool.refs.tolist() == [sum(row.count(p) for row in table) for p in range(layers.pool.pages)]
    D, A, bias = cpu(xd), layers.A_log.cpu(), layers.dt_bias.cpu()

    def cached(x):
        if cache != torch.float8_e4m3fn:
            return x.double()
        code, scale = oracle.kv_quantise(x)
        return code.double() * scale.double()[..., None]

    for b in range(S):
        seq = {n: torch.cat([t, D[n][b:b + 1]]) for n, t in seqs[b].items()}
        k, v = cached(seq["k"]), cached(seq["v"])
        for h in range(ex.HEADS):
            kh, vh = k[:, h // (ex.HEADS // ex.KV_HEADS)], v[:, h // (ex.HEADS // ex.KV_HEADS)]
            p = torch.softmax(kh @ D["q"][b, h].double() * ex.HEAD_DIM ** -0.5, 0)
            want, w = p @ vh, p @ vh.abs()
            err = (attn[b, h].double().cpu() - want).abs()
            assert bool((err <= U * (want.abs() + w) * 1.01 + FP32 * (w + 1)).all()), (b, h, float((err / w).max()))
        n = len(seq["a"])
        want, _ = oracle.gdn_sequence(A, bias, seq["a"], seq["b"], seq["gq"], seq["gk"], seq["gv"],
                                      torch.zeros(1, ex.VALUE_HEADS, ex.VALUE_DIM, ex.KEY_DIM), [0, n], [-1], [0], ex.KEY_DIM ** -0.5)
        err = (o[b].double().cpu() - want[-1]).abs().amax(-1)
        assert bool((err <= 3 * U * want[-1].abs().amax(-1) + 1e-5).all()), (b, float(err.max()))


@pytest.mark.gpu
def test_the_examples_contexts_hold_every_token(monkeypatch, capsys):
    """A prompt, the token drawn from its last row, and every token of every step: the last one's row is the decode's."""
    ex = _example()
    monkeypatch.setattr(sys, "argv", ["target_step.py", "--prompts", "40,3", "--temperature", "0.6", "--samples", "2", "--cache", "fp16"])
    ex.main()
    out = capsys.readouterr().out
    assert "all granted True" in out
    steps = [ast.literal_eval(m) for m in re.findall(r"tokens (\[\[.*\]\])", out)]
    contexts = ast.literal_eval(re.search(r"contexts (\[[^\]]*\])", out).group(1))
    assert contexts == [n + 1 + sum(len(s[b]) for s in steps) for b, n in enumerate([40, 3, 40, 3])]
