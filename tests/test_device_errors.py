"""What check() of the objects with a workspace says before a kernel has written the workspace's error words."""
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


def test_attention_that_has_not_run():
    from chain_flow_b200.attention import PagedAttention
    q, c, table, lens, cu = _cases("test_paged_attn")._case([3, 1], [40, 7], 4, 2, 64, 16, torch.float16, False)
    attn = PagedAttention(4, 2, 64)
    attn.ws.fill_(0x5a)                                          # what the allocator may hand out
    attn.check()
    attn(q[:0], c, table, lens, torch.zeros_like(cu))            # no rows
    attn(q, c, table[:0], lens[:0], cu[:1])                      # no requests
    attn.check()
    attn(q, c, table, lens, cu)
    attn.check()
    attn(q[:0], c, table, lens, torch.zeros_like(cu))
    attn.check()


def test_chunks_that_have_not_run():
    from chain_flow_b200.gdn import ChunkedGdn
    cases = _cases("test_gdn_seq")
    d = cases._gpu(cases._case([5, 2], seed=1))
    chunks = ChunkedGdn(7, 2, 4)
    chunks.ws.fill_(0x5a)
    chunks.check()
    gates, rows = (d["A_log"], d["dt_bias"]), [d[n] for n in ("a", "b", "q", "k", "v", "o")]
    state = (d["state"],)
    chunks(*gates, *(x[:0] for x in rows), *state, torch.zeros_like(d["cu"]), d["init"], d["to"], scale=0.1)       # no tokens
    chunks(*gates, *rows, *state, d["cu"][:1], d["init"][:0], d["to"][:0], scale=0.1)                               # no requests
    chunks.check()
    chunks(*gates, *rows, *state, d["cu"], d["init"], d["to"], scale=0.1)
    chunks.check()
