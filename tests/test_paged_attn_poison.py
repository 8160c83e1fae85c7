"""Values that are not finite in a paged cache: they reach the rows that see them, in their own columns, and no other
row, whatever the length, the tile and the way the pages come in. Finite elements are held to the bounds of
test_paged_attn.py; elsewhere an output is what the oracle's is (an infinity of its sign, or NaN)."""
import importlib.util
import math
import pathlib

import pytest
import torch

_spec = importlib.util.spec_from_file_location("paged_attn_cases", pathlib.Path(__file__).with_name("test_paged_attn.py"))
_cases = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(_cases)
_case, _want, ROUND, FP32 = _cases._case, _cases._want, _cases.ROUND, _cases.FP32

pytestmark = pytest.mark.gpu
TYPES = [(torch.bfloat16, False), (torch.float16, False), (torch.bfloat16, True), (torch.float16, True)]


def _compare(o, want, w, dtype):
    o, want, w = o.double().cpu(), want.cpu(), w.cpu()
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(o), finite)
    assert torch.equal(torch.isnan(o), torch.isnan(want)) and bool((o == want)[torch.isinf(want)].all())
    bound = ROUND[dtype] * (want.abs() + w) * 1.01 + FP32 * (w + 1)
    assert bool(((o - want).abs() <= bound)[finite].all()), float(((o - want).abs() / bound)[finite].max())


@pytest.mark.parametrize("dtype, quant", TYPES)
@pytest.mark.parametrize("news, lens, H, HKV, D, page", [
    ([150, 3], [400, 90], 4, 2, 128, 16), ([150, 3], [400, 90], 4, 2, 128, 17), ([70], [90], 8, 2, 256, 16), ([200], [200], 2, 2, 64, 17),
    ([60] * 40, [60] * 40, 2, 2, 64, 16),                        # pieces that are not cut
    ([2, 1, 4], [700, 90, 300], 8, 2, 256, 16), ([2, 1], [130, 90], 2, 2, 64, 17)])     # few rows
def test_rows_that_do_not_see_them_keep_their_values(dtype, quant, news, lens, H, HKV, D, page):
    from chain_flow_b200.attention import PagedAttention
    q, c, table, kv_len, cu = _case(news, lens, H, HKV, D, page, dtype, quant, seed=31)
    n, L = news[0], lens[0]
    v = c.v.view(torch.uint8) if quant else c.v
    inf = 0x7f if quant else float("inf")
    for j, column, x in ((L - n + n // 3, 7, inf), (L - n + n // 3, D - 1, inf), (L - n + 2 * n // 3, 7, 0xff if quant else -inf),
                         (L - n + 2 * n // 3, 40, 0x7f if quant else float("nan")), (L - 1, 9, inf), (L - 1, D - 1, inf), (5, 11, inf)):
        v[int(table[0, j // page]), :, j % page, column] = x
    attn = PagedAttention(H, HKV, D)
    got = attn(q, c, table, kv_len, cu)
    attn.check()
    o, lse, w = _want(q, c, table, kv_len, cu, True)
    _compare(got[0], o, w, dtype)
    finite = torch.isfinite(lse)
    assert torch.equal(finite, torch.isfinite(got[1].cpu()))
    assert bool(((got[1].double().cpu() - lse)[finite].abs() <= FP32 * (1 + lse[finite].abs())).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("news, lens, H, HKV, D", [([150], [400], 4, 2, 128), ([2, 1], [130, 90], 8, 2, 256)])
def test_a_column_that_overflows(dtype, news, lens, H, HKV, D):
    """One column infinite at every token of the context or of the step, its sign changing in another."""
    from chain_flow_b200.attention import PagedAttention
    q, c, table, kv_len, cu = _case(news, lens, H, HKV, D, 16, dtype, False, seed=33)
    for j in range(lens[0]):
        at = c.v[int(table[0, j // 16]), :, j % 16]
        at[:, 3] = float("-inf")
        if j >= lens[0] - news[0]:
            at[:, 5] = float("inf")
            at[:, D - 2] = float("inf") if j % 2 else float("-inf")
    attn = PagedAttention(H, HKV, D)
    got = attn(q, c, table, kv_len, cu)
    attn.check()
    o, _, w = _want(q, c, table, kv_len, cu, True)
    _compare(got[0], o, w, dtype)


@pytest.mark.parametrize("dtype, quant", [(torch.float16, False), (torch.bfloat16, True)])
def test_rows_of_nan_from_a_token_on(dtype, quant):
    """Every new token from the 40th on holds NaN throughout."""
    from chain_flow_b200.attention import PagedAttention
    H, HKV, D, n, L = 4, 4, 128, 100, 300
    q, c, table, kv_len, cu = _case([n], [L], H, HKV, D, 16, dtype, quant, seed=32)
    v = c.v.view(torch.uint8) if quant else c.v
    for j in range(L - n + 40, L):
        v[int(table[0, j // 16]), :, j % 16] = 0x7f if quant else float("nan")
    attn = PagedAttention(H, HKV, D)
    got = attn(q, c, table, kv_len, cu)
    attn.check()
    o, _, w = _want(q, c, table, kv_len, cu, True)
    _compare(got[0], o, w, dtype)


@pytest.mark.parametrize("dtype, quant", [(torch.float16, False), (torch.bfloat16, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("n, requests", [(64, 160), (4, 150)])
def test_long_contexts(dtype, quant, n, requests):
    """131072 positions that all the requests share, the last one's value not finite: every other row is taken again from
    its own positions, which outlasts what a wait between warps may take, and no wait expires."""
    from chain_flow_b200.attention import PagedAttention
    from chain_flow_b200.kv_cache import PagedKVCache
    L, D, page = 131072, 64, 64
    g = torch.Generator(device="cuda").manual_seed(n)
    rows = torch.randn(2, L, 1, D, device="cuda", generator=g).to(dtype)
    cache = PagedKVCache(L // page, page, 1, D, torch.float8_e4m3fn if quant else dtype)
    cache.write(rows[0], rows[1], torch.arange(L, device="cuda"))
    (cache.v.view(torch.uint8) if quant else cache.v)[-1, 0, -1, 7] = 0x7f if quant else float("inf")
    table = torch.arange(L // page, dtype=torch.int32, device="cuda").view(1, -1).expand(requests, -1)
    kv_len = torch.full((requests,), L, dtype=torch.int32, device="cuda")
    q = torch.randn(requests * n, 1, D, device="cuda", generator=g).to(dtype)
    attn = PagedAttention(1, 1, D)
    got = attn(q, cache, table, kv_len, torch.arange(0, requests * n + 1, n, dtype=torch.int32, device="cuda"))
    attn.check()
    o = got[0].view(requests, n, D)
    assert bool(torch.isfinite(o[:, :-1]).all())
    last = o[:, -1, 7].float()
    assert bool(torch.isnan(last).all() if quant else (last == math.inf).all())
    k, v = (p.float().double().view(L, D) for p in (cache.k, cache.v))
    if quant:
        k, v = k * cache.k_scale.view(L, 1).double(), v * cache.v_scale.view(L, 1).double()
    seen = torch.arange(L, device="cuda")[None] <= L - n + torch.arange(n, device="cuda")[:, None]
    v[-1, 7] = 0                                                 # (no other row sees it)
    for b in (0, 1, requests - 1):
        s = (q.view(requests, n, D)[b].double() @ k.T) * D ** -0.5
        p = torch.softmax(s.masked_fill(~seen, -math.inf), 1)
        want, w = p @ v, p @ v.abs()
        keep = torch.ones(n, D, dtype=torch.bool)
        keep[-1, 7] = False
        err = (o[b].double() - want).abs().cpu()
        assert bool((err <= ROUND[dtype] * (want.abs() + w).cpu() * 1.01 + FP32 * (w.cpu() + 1))[keep].all())
