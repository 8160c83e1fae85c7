"""Attention over e4m3 rows whose scale is 0 or next to it: slots that no write has filled (a fresh cache's, a skipped
token's), rows of zeros from a quantiser without a floor. Such a key scores 0, such a value is 0, and the position keeps
its part of the softmax. Bounds as in test_paged_attn.py; a value scale below 2^-60 counts as 2^-60, which moves o by
at most 448 2^-60."""
import importlib.util
import math
import pathlib

import pytest
import torch

_spec = importlib.util.spec_from_file_location("paged_attn_cases", pathlib.Path(__file__).with_name("test_paged_attn.py"))
_cases = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(_cases)
_case, _want, _check, FP8 = _cases._case, _cases._want, _cases._check, _cases.FP8

pytestmark = pytest.mark.gpu
NEWS = [[1, 2, 1, 1], [40, 150, 3, 1]]             # tiles of few rows, of 128


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("news", NEWS)
@pytest.mark.parametrize("causal", [True, False])
def test_slots_that_were_never_written(dtype, news, causal):
    from chain_flow_b200.attention import PagedAttention
    from chain_flow_b200.kv_cache import PagedKVCache
    H, HKV, D, page, lens = 4, 2, 128, 16, [200, 300, 77, 64]
    g = torch.Generator(device="cuda").manual_seed(sum(news))
    width = -(-max(lens) // page)
    cache = PagedKVCache(4 * width, page, HKV, D, FP8)
    table = torch.randperm(4 * width, generator=g, device="cuda").view(4, width).int()
    # request 0: every third position written; 1: all but the last tile's; 2: none; 3: the first only
    kept = [range(0, 200, 3), range(256), (), (0,)]
    slots = torch.tensor([int(table[b, j // page]) * page + j % page for b, js in enumerate(kept) for j in js], device="cuda")
    k, v = (torch.randn(len(slots), HKV, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    cache.write(k, v + 0.5, slots)
    q = torch.randn(sum(news), H, D, device="cuda", generator=g).to(dtype)
    case = (q, cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.tensor([0] + news, device="cuda").cumsum(0).int())
    got = PagedAttention(H, HKV, D)(*case, causal=causal)
    torch.cuda.synchronize()
    _check(got, _want(*case, causal), dtype)
    rows = slice(sum(news[:2]), sum(news[:3]))
    assert bool((got[0][rows] == 0).all())                       # request 2 sees rows of zeros alone
    if not causal:
        assert float((got[1][:, rows] - math.log(77)).abs().max()) <= 1e-5


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("news", NEWS)
@pytest.mark.parametrize("scale", [0.0, 1e-40, 1e-20])
def test_scales_next_to_zero(dtype, news, scale):
    """Codes that are not 0 under such scales, of keys and of values, among ordinary rows."""
    from chain_flow_b200.attention import PagedAttention
    H, HKV, D, page, lens = 4, 2, 64, 17, [200, 300, 77, 64]
    case = _case(news, lens, H, HKV, D, page, dtype, True, seed=sum(news))
    c, table = case[1], case[2]
    for b, j in ((0, 3), (0, 64), (1, 150), (1, 299), (2, 0), (2, 76)):
        c.v_scale[int(table[b, j // page]), :, j % page] = scale
        c.k_scale[int(table[b, j // page]), 0, j % page] = scale
    for j in range(64):
        c.v_scale[int(table[3, j // page]), :, j % page] = scale
    attn = PagedAttention(H, HKV, D)
    got = attn(*case)
    attn.check()
    _check(got, _want(*case, True), dtype)


@pytest.mark.parametrize("news", NEWS)
def test_negative_and_nan_scales_reach_the_rows_that_see_them(news):
    from chain_flow_b200.attention import PagedAttention
    H, HKV, D, page, lens = 4, 2, 64, 16, [200, 300, 77, 64]
    case = _case(news, lens, H, HKV, D, page, torch.float16, True, seed=5)
    c, table = case[1], case[2]
    want = [t.clone() for t in PagedAttention(H, HKV, D)(*case)]
    first, second = news[0], news[0] + news[1]
    for x in (-1.0, float("nan")):
        c.v_scale[int(table[0, 0]), :, 5] = x                    # every row of request 0 sees it
        c.v_scale[int(table[1, 299 // page]), :, 299 % page] = x     # request 1's last row
        o, lse = PagedAttention(H, HKV, D)(*case)
        torch.cuda.synchronize()
        assert bool(torch.isnan(o[:first]).all()) and bool(torch.isnan(lse[:, :first]).all()) and bool(torch.isnan(o[second - 1]).all())
        assert torch.equal(o[first:second - 1], want[0][first:second - 1]) and torch.equal(o[second:], want[0][second:])
