"""Attention over a paged cache in steps of many short requests, so that every CTA takes several pieces of work one
after another and what a piece hands on between warps meets the next one's: the bounds of the other steps
(test_paged_attn.py), and the same bits every time."""
import importlib.util
import pathlib

import pytest
import torch

_spec = importlib.util.spec_from_file_location("paged_attn_cases", pathlib.Path(__file__).with_name("test_paged_attn.py"))
_cases = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(_cases)

TYPES = [(torch.bfloat16, False), (torch.float16, False), (torch.bfloat16, True), (torch.float16, True)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, quant", TYPES)
@pytest.mark.parametrize("news, H, HKV, D, page", [
    (9, 4, 4, 128, 16),                            # 128-row tiles over e4m3, few rows over 16 bits
    (34, 4, 4, 64, 17),                            # 128-row tiles
    (9, 3, 3, 256, 16), (2, 8, 4, 128, 16)])       # 2: few rows everywhere
def test_many_pieces_a_cta(dtype, quant, news, H, HKV, D, page):
    from chain_flow_b200.attention import PagedAttention
    requests = 120 if news < 30 else 60
    lens = [news + (b * 37) % 150 for b in range(requests)]
    case = _cases._case([news] * requests, lens, H, HKV, D, page, dtype, quant, seed=news)
    attn = PagedAttention(H, HKV, D)
    got = attn(*case)
    attn.check()
    _cases._check(got, _cases._want(*case, True), dtype)
    for _ in range(20):
        again = attn(*case)
        torch.cuda.synchronize()
        assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])
