"""Attention over a paged cache where requests bring few query rows each (decodes, short steps): the same
bounds as the long steps' (test_paged_attn.py): an output's own rounding and its weights', and 2e-5 for
the fp32 scores. Queries and weights over an e4m3 cache keep 12 bits and more, and a weight below 2^-28 of
the largest is lost: 8000 of them are 2^-15 of it, of which the bounds' fp32 term takes account."""
import importlib.util
import pathlib

import pytest
import torch

_spec = importlib.util.spec_from_file_location("paged_attn_cases", pathlib.Path(__file__).with_name("test_paged_attn.py"))
_cases = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(_cases)
_case, _want, _check, ROUND, FP32 = _cases._case, _cases._want, _cases._check, _cases.ROUND, _cases.FP32

TYPES = [(torch.bfloat16, False), (torch.float16, False), (torch.bfloat16, True), (torch.float16, True)]


def _run(case, H, HKV, D, dtype, causal=True):
    from chain_flow_b200.attention import PagedAttention
    attn = PagedAttention(H, HKV, D)
    got = attn(*case, causal=causal)
    attn.check()
    _check(got, _want(*case, causal), dtype)
    again = attn(*case, causal=causal)
    torch.cuda.synchronize()
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, quant", TYPES)
@pytest.mark.parametrize("H, HKV, D", [(16, 4, 256), (7, 1, 128), (2, 2, 64)])
@pytest.mark.parametrize("page", [16, 17, 64])
@pytest.mark.parametrize("causal", [True, False])
def test_few_rows(dtype, quant, H, HKV, D, page, causal):
    """No tokens, no context, one token, two; lengths round the unit and past several CTAs' shares."""
    case = _case([1, 1, 0, 1, 2, 1, 1], [1, 64, 40, 0, 129, 1000, 65], H, HKV, D, page, dtype, quant, seed=page)
    _run(case, H, HKV, D, dtype, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, quant", TYPES)
def test_a_longer_request_among_decodes(dtype, quant):
    """20 tokens x 4 heads among 30 decodes: several tiles of few rows."""
    case = _case([1] * 30 + [20], [5 + 3 * b for b in range(30)] + [150], 8, 2, 128, 16, dtype, quant, seed=2)
    _run(case, 8, 2, 128, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("requests", [32, 33, 700])
@pytest.mark.parametrize("quant", [False, True])
def test_many_requests(requests, quant):
    news = [(b * 7 + 3) % 5 != 0 for b in range(requests)]
    lens = [(b * 11) % 70 for b in range(requests)]
    case = _case([int(n) for n in news], lens, 2, 1, 64, 16, torch.float16, quant, seed=requests)
    _run(case, 2, 1, 64, torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, quant", TYPES)
@pytest.mark.parametrize("news", [[1], [40]])
def test_one_position_takes_most_of_the_weight(dtype, quant, news):
    """A position whose value is 0 takes nine tenths: the output is what 8000 others add up to."""
    from chain_flow_b200.kv_cache import PagedKVCache
    from chain_flow_b200.attention import PagedAttention
    n, D, L = news[0], 128, 8000
    g = torch.Generator().manual_seed(1)
    q = torch.randn(1, 1, D, generator=g).repeat(n, 1, 1).to(dtype)
    k = 0.02 * torch.randn(L, 1, D, generator=g)
    k[5] = q[0, 0].float() * (11.2 * D ** 0.5 / float((q[0, 0].float() ** 2).sum()))
    v = torch.rand(L, 1, D, generator=g)
    v[5] = 0
    cache = PagedKVCache(L // 16, 16, 1, D, torch.float8_e4m3fn if quant else dtype)
    cache.write(k.to(dtype).cuda(), v.to(dtype).cuda(), torch.arange(L, device="cuda"))
    case = (q.cuda(), cache, torch.arange(L // 16, dtype=torch.int32, device="cuda").view(1, -1),
            torch.tensor([L], dtype=torch.int32, device="cuda"), torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    got = PagedAttention(1, 1, D)(*case, causal=False)
    torch.cuda.synchronize()
    want = _want(*case, False)
    assert 0.02 < float(want[0].mean()) < 0.2                 # the others' part of the weight, halved by their values
    _check(got, want, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_that_are_not_finite(dtype):
    """An infinite value reaches its own column of the rows that see it; a row before it sees nothing of it."""
    from chain_flow_b200.attention import PagedAttention
    H, HKV, D, L = 4, 2, 128, 300
    q, c, table, lens, cu = _case([2, 1], [L, 90], H, HKV, D, 16, dtype, False, seed=8)
    want = _want(q, c, table, lens, cu, True)
    for j, bad in ((100, float("inf")), (L - 1, float("nan"))):
        slot = int(table[0, j // 16]), j % 16
        keep = c.v[slot[0], :, slot[1]].clone()
        c.v[slot[0], :, slot[1], 7] = bad
        got = PagedAttention(H, HKV, D)(q, c, table, lens, cu)
        torch.cuda.synchronize()
        c.v[slot[0], :, slot[1]] = keep
        hit = torch.zeros(3, dtype=torch.bool)
        hit[0 if j < L - 1 else 1:2] = True
        col = got[0][:, :, 7].float().cpu()
        assert bool((col[hit] == bad).all() if bad == bad else torch.isnan(col[hit]).all())
        mask = torch.ones(3, H, D, dtype=torch.bool)
        mask[hit, :, 7] = False
        err, bound = (got[0].double().cpu() - want[0]).abs(), ROUND[dtype] * (want[0].abs() + want[2]) * 1.01 + FP32 * (want[2] + 1)
        assert bool((err[mask] <= bound[mask]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("news", [[2, 1], [40, 1]])
def test_codes_that_are_not_a_number(dtype, news):
    """A NaN code in a later token's key and value: rows before it see nothing of it, rows from it on all of it."""
    from chain_flow_b200.attention import PagedAttention
    H, HKV, D, L = 4, 2, 128, 300
    q, c, table, lens, cu = _case(news, [L, 90], H, HKV, D, 16, dtype, True, seed=9)
    want = _want(q, c, table, lens, cu, True)
    slot = int(table[0, (L - 1) // 16]), (L - 1) % 16
    for pool, columns in ((c.v, [7]), (c.k, range(D))):
        bits = pool.view(torch.uint8)
        keep = bits[slot[0], :, slot[1]].clone()
        bits[slot[0], :, slot[1], 7] = 0x7f
        got = PagedAttention(H, HKV, D)(q, c, table, lens, cu)
        torch.cuda.synchronize()
        bits[slot[0], :, slot[1]] = keep
        last = news[0] - 1
        assert bool(torch.isnan(got[0][last][:, list(columns)]).all())
        mask = torch.ones(sum(news), H, D, dtype=torch.bool)
        mask[last, :, list(columns)] = False
        err, bound = (got[0].double().cpu() - want[0]).abs(), ROUND[dtype] * (want[0].abs() + want[2]) * 1.01 + FP32 * (want[2] + 1)
        assert bool((err[mask] <= bound[mask]).all())


def test_more_units_than_32_bits_are_refused():
    assert _cases._call(T=1 << 23, H=4 * 16, width=1 << 22, st=1 << 22) == 2
    assert _cases._call(T=0, width=1 << 22, st=1 << 22) == 0
