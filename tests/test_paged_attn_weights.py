"""Softmax weights far below the largest: a position whose value is 0 outweighs every other by 2^25 and more, so that the
output is what thousands of such weights add up to. fp16's smallest step is 2^-24: weights at most 1 would vanish in it.
Bounds as in test_paged_attn.py."""
import importlib.util
import pathlib

import pytest
import torch

_spec = importlib.util.spec_from_file_location("paged_attn_cases", pathlib.Path(__file__).with_name("test_paged_attn.py"))
_cases = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(_cases)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, quant", [(torch.bfloat16, False), (torch.float16, False), (torch.bfloat16, True), (torch.float16, True)])
@pytest.mark.parametrize("news, D", [([1], 128), ([40], 128), ([40], 64), ([140], 256)])
@pytest.mark.parametrize("at", [5, 7990])           # the heavy position comes first, last
def test_thousands_of_small_weights(dtype, quant, news, D, at):
    from chain_flow_b200.attention import PagedAttention
    from chain_flow_b200.kv_cache import PagedKVCache
    n, L = news[0], 8000
    g = torch.Generator().manual_seed(D + at)
    q = torch.randn(1, 1, D, generator=g).repeat(n, 1, 1).to(dtype)
    k = 0.02 * torch.randn(L, 1, D, generator=g)
    k[at] = q[0, 0].float() * (25.5 * 0.6931 * D ** 0.5 / float((q[0, 0].float() ** 2).sum()))
    v = torch.rand(L, 1, D, generator=g)
    v[at] = 0
    cache = PagedKVCache(L // 16, 16, 1, D, torch.float8_e4m3fn if quant else dtype)
    cache.write(k.to(dtype).cuda(), v.to(dtype).cuda(), torch.arange(L, device="cuda"))
    # requests enough that one CTA takes all of a request's positions
    requests, table = 160, torch.arange(L // 16, dtype=torch.int32, device="cuda").view(1, -1)
    attn = PagedAttention(1, 1, D)
    o, lse = attn(q.cuda().repeat(requests, 1, 1), cache, table.expand(requests, -1), torch.full((requests,), L, device="cuda"),
                  torch.arange(0, requests * n + 1, n, device="cuda"), causal=False)
    attn.check()
    want = _cases._want(q.cuda(), cache, table, torch.tensor([L]), torch.tensor([0, n]), False)
    assert 5e-5 < float(want[0].mean()) < 2e-4
    for b in (0, 77, requests - 1):
        _cases._check((o[b * n:(b + 1) * n], lse[:, b * n:(b + 1) * n]), want, dtype)
