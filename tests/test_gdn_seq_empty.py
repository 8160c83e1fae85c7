"""Steps of the gated delta rule in which no request has a token: states are copied."""
import ctypes as C
import importlib.util
import pathlib

import pytest
import torch

from chain_flow_b200 import _lib

_spec = importlib.util.spec_from_file_location("gdn_seq_cases", pathlib.Path(__file__).with_name("test_gdn_seq.py"))
_cases = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(_cases)

ROWS = ("a", "b", "q", "k", "v", "o")


def test_rows_are_not_asked_for_where_there_are_no_tokens():
    """The null rows of an empty step get past the checks (the workspace's is the one that refuses here), those of a step
    with tokens do not."""
    lib = _lib.load()
    g = _cases._args(**{n: None for n in ROWS})
    assert lib.cfb_gdn_chunk(C.byref(g), _cases.FAKE, 0, 1, _cases.FAKE, 0, None) == 3
    assert lib.cfb_gdn_chunk(C.byref(g), _cases.FAKE, 4, 1, _cases.FAKE, 1 << 30, None) == 1
    assert lib.cfb_gdn_step(C.byref(g), 1, None) == 1
    for name in ("A_log", "dt_bias", "state_in", "state_out", "init_slot", "out_slot"):
        g = _cases._args(**{n: None for n in ROWS + (name,)})
        assert lib.cfb_gdn_chunk(C.byref(g), _cases.FAKE, 0, 1, _cases.FAKE, 0, None) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_step_without_tokens_copies_its_states(dtype):
    from chain_flow_b200.gdn import ChunkedGdn
    d = _cases._gpu(_cases._case([0, 0, 0], 2, 4, 64, dtype, seed=1))
    assert d["q"].data_ptr() == 0
    d["init"] = torch.tensor([3, -1, 9], dtype=torch.int32, device="cuda")       # 5 slots: a state, zeros, none there is
    d["to"] = torch.tensor([0, 4, 2], dtype=torch.int32, device="cuda")
    out = torch.full_like(d["state"], 5.0)
    args = (d["A_log"], d["dt_bias"], d["a"], d["b"], d["q"], d["k"], d["v"], d["o"], d["state"], d["cu"], d["init"], d["to"])
    chunks = ChunkedGdn(0, 3, 4)
    chunks(*args, scale=0.1, out_state=out)
    chunks.check()
    assert torch.equal(out[0], d["state"][3]) and bool((out[4] == 0).all()) and bool(torch.isnan(out[2]).all())
    assert bool((out[[1, 3]] == 5).all())
