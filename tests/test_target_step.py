"""The example that runs the cache, the attention over it and the gated delta rule as a target would
(prompts, a verified tree, a commit, a decode), against the layers computed over whole sequences in 64
bits. A value rounded to fp16 differs by 2^-11 of itself; attention's weights add as much of what they
weigh, the gated-delta outputs 2 x 2^-11 of a head's largest (one rounding of the state's operand each), and
the tree half of a merged row is rounded once more."""
import importlib.util
import pathlib

import pytest
import torch

import oracle

U, FP32 = 2.0 ** -11, 4e-6


def _example():
    path = pathlib.Path(__file__).resolve().parents[1] / "examples" / "target_step.py"
    spec = importlib.util.spec_from_file_location("target_step", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_the_example_imports_without_a_gpu():
    ex = _example()
    assert ex.HEADS % ex.KV_HEADS == 0 and ex.VALUE_HEADS % ex.KEY_HEADS == 0


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [torch.float8_e4m3fn, torch.float16])
def test_prompt_verify_commit_decode(cache):
    ex = _example()
    news, N = [50, 1, 17], 8
    layers = ex.TargetLayers(len(news), max(news) + N + 1, N, cache_dtype=cache)
    A, bias = layers.A_log.cpu(), layers.dt_bias.cpu()
    xp, xt, xd = ex.projections(sum(news), seed=1), ex.projections(len(news) * N, seed=2), ex.projections(len(news), seed=3)
    parents = torch.tensor([[-1, 0, 0, 1, 1, 2, 3, 6], [-1, 0, 1, 2, 3, 4, 5, 6], [-1, -1, 0, 1, 2, 2, 3, 3]])
    paths = [[0, 1, 3, 6, 7], [], [1, 3]]
    got_p = layers.prompt(xp, news)
    got_t = layers.verify(xt, parents.cuda())
    layers.commit(xt, paths)
    got_d = layers.decode(xd)
    layers.attention.check()
    layers.chunks.check()
    P, T, D = ({n: t.cpu() for n, t in x.items()} for x in (xp, xt, xd))

    def cached(x):
        if cache != torch.float8_e4m3fn:
            return x.double()
        code, scale = oracle.kv_quantise(x)
        return code.double() * scale.double()[..., None]

    def attention(got, q, k, v, factor):                         # one row over k, v [n, KV_HEADS, D]
        for h in range(ex.HEADS):
            kh, vh = k[:, h // (ex.HEADS // ex.KV_HEADS)], v[:, h // (ex.HEADS // ex.KV_HEADS)]
            p = torch.softmax(kh @ q[h].double() * ex.HEAD_DIM ** -0.5, 0)
            want, w = p @ vh, p @ vh.abs()
            err = (got[h].double().cpu() - want).abs()
            assert bool((err <= factor * U * (want.abs() + w) * 1.01 + FP32 * (w + 1)).all()), float((err / w).max())

    def delta(got, xs):                                          # the last row of a sequence
        x = {n: torch.cat([y[n] for y in xs]) for n in ("a", "b", "gq", "gk", "gv")}
        n = len(x["a"])
        o, _ = oracle.gdn_sequence(A, bias, x["a"], x["b"], x["gq"], x["gk"], x["gv"],
                                   torch.zeros(1, ex.VALUE_HEADS, ex.VALUE_DIM, ex.KEY_DIM), [0, n], [-1], [0], ex.KEY_DIM ** -0.5)
        err = (got.double().cpu() - o[-1]).abs().amax(-1)
        assert bool((err <= 3 * U * o[-1].abs().amax(-1) + 1e-5).all()), float(err.max())

    at = 0
    for b, n in enumerate(news):
        prompt = {m: t[at:at + n] for m, t in P.items()}
        ck, cv = cached(prompt["k"]), cached(prompt["v"])
        for t in (0, n - 1):
            attention(got_p[0][at + t], prompt["q"][t], ck[:t + 1], cv[:t + 1], 1)
            delta(got_p[1][at + t], [{m: x[:t + 1] for m, x in prompt.items()}])
        at += n
        for m in range(N):
            chain = [m]
            while parents[b, chain[0]] >= 0:
                chain.insert(0, int(parents[b, chain[0]]))
            rows = [b * N + c for c in chain]
            attention(got_t[0][b * N + m], T["q"][b * N + m], torch.cat([ck, T["k"][rows].double()]),
                      torch.cat([cv, T["v"][rows].double()]), 4)
            delta(got_t[1][b * N + m], [prompt, {z: x[rows] for z, x in T.items()}])
        rows = [b * N + c for c in paths[b]]
        one = {z: x[b:b + 1] for z, x in D.items()}
        attention(got_d[0][b], one["q"][0], *(torch.cat([c, cached(T[z][rows]), cached(one[z])]) for z, c in (("k", ck), ("v", cv))), 1)
        delta(got_d[1][b], [prompt, {z: x[rows] for z, x in T.items()}, one])
