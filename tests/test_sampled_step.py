"""The example's sampled steps as they are used together: prompts into pages of a pool, forked to several samples, trees
verified from given random numbers, accepted rows moved together, refused pages given back, a plain decode. Tokens and
pages against the oracles, the decode's layers against whole sequences in 64 bits (tolerances as in
test_target_step.py)."""
import importlib.util
import pathlib
import sys

import pytest
import torch

import oracle
from chain_flow_b200.gdn import make_tree

U, FP32 = 2.0 ** -11, 4e-6


def _example():
    path = pathlib.Path(__file__).resolve().parents[1] / "examples" / "target_step.py"
    spec = importlib.util.spec_from_file_location("target_step", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [torch.float8_e4m3fn, torch.float16])
def test_prompts_forks_steps_decode(cache):
    ex = _example()
    news, S, N, V = [50, 17], 5, 10, 300
    layers = ex.SampledTarget(S, max(news) + 3 * N + 1, N, cache_dtype=cache)
    xp = ex.projections(sum(news), seed=1)
    layers.prompt(xp, news + [0] * 3)
    parent, child = [0, 1, 0], [2, 3, 4]
    layers.fork(torch.tensor(parent, device="cuda"), torch.tensor(child, device="cuda"))
    of = [0, 1] + parent
    assert layers.kv_len.tolist() == [news[p] for p in of]
    g = torch.Generator().manual_seed(3)
    kept = [[] for _ in range(S)]                                    # per request: (step's projections, accepted rows)
    temp = torch.tensor([1.0, 0.0, 0.7, 1.3, 1.0])
    for step in range(3):
        x = ex.projections(S * N, seed=10 + step)
        parents = torch.stack([make_tree(N, 5, 3, seed=step * S + b)[0] for b in range(S)])
        logits = 2 * torch.randn(S * (N + 1), V, generator=g)
        rows = logits.view(S, N + 1, V).topk(2, dim=2).indices
        tokens = torch.stack([torch.stack([rows[b, parents[b, i] + 1, i % 2] for i in range(N)]) for b in range(S)])
        u = torch.rand(S * (N + 1), generator=g)
        _, _, out = layers.sampled_step(x, parents.cuda(), tokens.cuda(), logits.cuda(), u.cuda(), temp.cuda())
        b1 = torch.arange(1, S + 1)
        want = oracle.tree_verify_sampled(logits, b1 * N, b1 * (N + 1), tokens.flatten(), parents.flatten(), u, temp, N)
        for a, b in zip(out[:3], want):
            assert torch.equal(a.cpu().long(), b)
        assert float((out[3].cpu().double() - want[3]).abs().max()) <= 2.0 ** -16 + 2.0 ** -23 * float(want[3].abs().max())
        for b in range(S):
            kept[b].append((x, [b * N + i for i in want[1][b].tolist() if i >= 0]))
    lens = [news[of[b]] + sum(len(r) for _, r in kept[b]) for b in range(S)]
    assert layers.kv_len.tolist() == lens and sum(lens) > sum(news[p] for p in of)
    xd = ex.projections(S, seed=30)
    attn, o = layers.decode(xd)
    layers.attention.check()
    layers.chunks.check()
    assert all(bool(t.all()) for t in layers.granted) and int(layers.pool.err.item()) == 0 and int(layers.verifier.err.item()) == 0
    # every page has as many holders as rows that name it, and each request's pages cover its context
    table = layers.table.tolist()
    held = [sum(row.count(p) for row in table) for p in range(layers.pool.pages)]
    assert layers.pool.refs.tolist() == held
    assert [sum(p >= 0 for p in row) for row in table] == [-(-(n + 1) // ex.PAGE) for n in lens]
    assert max(held) == 3                                            # a prompt's full page, held by its three samples

    cpu = lambda x: {n: t.cpu() for n, t in x.items()}  # noqa: E731
    P, D = cpu(xp), cpu(xd)
    A, bias = layers.A_log.cpu(), layers.dt_bias.cpu()

    def cached(x):
        if cache != torch.float8_e4m3fn:
            return x.double()
        code, scale = oracle.kv_quantise(x)
        return code.double() * scale.double()[..., None]

    for b in range(S):
        at = sum(news[:of[b]])
        parts = [{n: t[at:at + news[of[b]]] for n, t in P.items()}]
        parts += [{n: t[rows] for n, t in cpu(x).items()} for x, rows in kept[b]]
        parts.append({n: t[b:b + 1] for n, t in D.items()})
        seq = {n: torch.cat([p[n] for p in parts]) for n in P}
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
def test_the_examples_own_run(monkeypatch, capsys):
    ex = _example()
    monkeypatch.setattr(sys, "argv", ["target_step.py", "--prompts", "40,3", "--temperature", "0.8", "--samples", "3", "--cache", "fp16"])
    ex.main()
    assert "all granted True" in capsys.readouterr().out
