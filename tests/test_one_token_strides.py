"""One token's rows as the transpose of a column: the stride of a dim of size 1 is whatever torch left there (here 1), and no
row is anywhere but where it should be."""
import importlib.util
import pathlib

import pytest
import torch

pytestmark = pytest.mark.gpu


def _cases(name):
    spec = importlib.util.spec_from_file_location(name, pathlib.Path(__file__).with_name(name + ".py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _column(t):
    """t [1, heads, dim] with a token stride of 1."""
    return t.as_strided(t.shape, (1, *t.stride()[1:]))


@pytest.mark.parametrize("quant", [False, True])
def test_cache_and_attention(quant):
    from chain_flow_b200.attention import PagedAttention
    from chain_flow_b200.kv_cache import PagedKVCache
    q, c, table, lens, cu = _cases("test_paged_attn")._case([1], [40], 4, 2, 64, 16, torch.float16, quant, seed=6)
    q = q.contiguous()
    attn = PagedAttention(4, 2, 64)
    want = attn(q, c, table, lens, cu)
    out = _column(torch.zeros_like(q))
    got = attn(_column(q), c, table, lens, cu, out=out)
    attn.check()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    x = torch.randn(2, 1, 2, 64, device="cuda").half()
    a, b = (PagedKVCache(2, 16, 2, 64, torch.float8_e4m3fn if quant else torch.float16) for _ in range(2))
    slot = torch.tensor([17], device="cuda")
    a.write(x[0], x[1], slot)
    b.write(_column(x[0]), _column(x[1]), slot)
    for s, t in zip(a.read(slot), b.read(slot)):
        assert torch.equal(s, t) and bool(s.any())


@pytest.mark.parametrize("step", [False, True])
def test_gated_delta_rule(step):
    cases = _cases("test_gdn_seq")
    c = cases._case([1], 2, 4, 64, torch.bfloat16, seed=7)
    d = {n: t.cuda() for n, t in c.items()}
    for n in ("q", "k", "v"):
        d[n] = _column(d[n].contiguous())
    d["o"] = _column(torch.zeros(d["v"].shape, device="cuda", dtype=torch.bfloat16))
    cases._run(d, step=step)
    cases._check(d["o"], d["state"], c, cases._oracle(c))


@pytest.mark.parametrize("step", [False, True])
def test_rows_without_a_heads_dim_are_refused(step):
    from chain_flow_b200 import _lib
    cases = _cases("test_gdn_seq")
    d = cases._gpu(cases._case([1, 1], 2, 4, 64, torch.float16, seed=7))
    for n in ("q", "k", "v", "o"):
        with pytest.raises(_lib.CfbError):
            cases._run({**d, n: d[n].flatten(1)}, step=step)
