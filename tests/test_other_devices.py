"""Calls over tensors of one GPU while another is the current one, and objects whose workspace lies on another: refused
before anything is launched. One GPU is enough: the device numbers are what is looked at."""
import importlib.util
import pathlib

import pytest
import torch

from chain_flow_b200 import _lib


def _cases(name):
    spec = importlib.util.spec_from_file_location(name, pathlib.Path(__file__).with_name(name + ".py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_the_stream_is_of_the_tensors_device(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 100 + device, raising=False)
    assert _lib.stream_of(1, "call") == 101
    with pytest.raises(_lib.CfbError, match="cuda:0.*cuda:1"):
        _lib.stream_of(0, "call")


@pytest.mark.gpu
def test_attention_and_cache(monkeypatch):
    from chain_flow_b200.attention import PagedAttention
    q, c, table, lens, cu = _cases("test_paged_attn")._case([3, 1], [40, 7], 4, 2, 64, 16, torch.float16, False)
    attn = PagedAttention(4, 2, 64)
    attn(q, c, table, lens, cu)
    elsewhere = PagedAttention(4, 2, 64)
    elsewhere._dev += 1
    with pytest.raises(_lib.CfbError, match="workspace"):
        elsewhere(q, c, table, lens, cu)
    rows = torch.zeros(1, 2, 64, device="cuda", dtype=torch.float16)
    slot = torch.zeros(1, dtype=torch.int64, device="cuda")
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    for call in (lambda: attn(q, c, table, lens, cu, out=torch.empty_like(q), lse=torch.empty(4, 4, device=q.device)),
                 lambda: c.write(rows, rows, slot), lambda: c.read(slot)):
        with pytest.raises(_lib.CfbError, match="current device"):
            call()


@pytest.mark.gpu
def test_gated_delta_rule(monkeypatch):
    from chain_flow_b200.gdn import ChunkedGdn, gdn_step
    cases = _cases("test_gdn_seq")
    d = cases._gpu(cases._case([1, 1], seed=1))
    args = [d[n] for n in ("A_log", "dt_bias", "a", "b", "q", "k", "v", "o", "state")]
    chunks, elsewhere = ChunkedGdn(2, 2, 4), ChunkedGdn(2, 2, 4)
    elsewhere._dev += 1
    with pytest.raises(_lib.CfbError, match="workspace"):
        elsewhere(*args, d["cu"], d["init"], d["to"], scale=0.1)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    with pytest.raises(_lib.CfbError, match="current device"):
        chunks(*args, d["cu"], d["init"], d["to"], scale=0.1)
    with pytest.raises(_lib.CfbError, match="current device"):
        gdn_step(*args, d["init"], d["to"], scale=0.1)
