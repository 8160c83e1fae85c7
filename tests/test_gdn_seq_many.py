"""The gated delta rule over sequences where a launch has work for every SM several times over (many requests
and heads): the bounds of the smaller launches (test_gdn_seq.py), whatever the order of the lengths."""
import importlib.util
import pathlib

import pytest
import torch

_spec = importlib.util.spec_from_file_location("gdn_seq_cases", pathlib.Path(__file__).with_name("test_gdn_seq.py"))
_cases = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(_cases)

pytestmark = pytest.mark.gpu
TYPES = [(torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16)]


@pytest.mark.parametrize("dtype, gate", TYPES)
@pytest.mark.parametrize("lens, HV, V", [
    ([5, 70, 0, 33], 32, 128),                     # 4 x 32 x 4 tiles of 32 value rows
    ([1, 31, 32, 96, 2, 64, 65, 40], 32, 64),
    ([33, 1, 40, 2, 7], 32, 96)])                  # value rows in 32s only
def test_many_heads(dtype, gate, lens, HV, V):
    c = _cases._case(lens, 4, HV, V, dtype, gate, seed=V)
    want = _cases._oracle(c)
    d = _cases._gpu(c)
    out = d["state"].clone()
    _cases._run(d, out_state=out)
    _cases._check(d["o"], out, c, want)
    again, o1 = d["state"].clone(), d["o"].clone()
    _cases._run(d, out_state=again)
    assert torch.equal(again, out) and torch.equal(o1, d["o"])


@pytest.mark.parametrize("requests", [300, 600])
def test_many_requests(requests):
    lens = [(b * 7) % 5 for b in range(requests)]
    c = _cases._case(lens, 1, 2, 64, torch.float16, seed=requests)
    want = _cases._oracle(c)
    d = _cases._gpu(c)
    out = d["state"].clone()
    _cases._run(d, out_state=out)
    _cases._check(d["o"], out, c, want)


@pytest.mark.parametrize("dtype, gate", TYPES)
def test_nan_stays_in_its_request_head_and_row(dtype, gate):
    c = _cases._case([40, 70, 40, 3], 4, 32, 128, dtype, gate, seed=15)
    d = _cases._gpu(c)
    d["v"][50, 9, 77] = float("nan")               # request 1, its token 10
    out = d["state"].clone()
    _cases._run(d, out_state=out)
    bad = torch.zeros(d["o"].shape, dtype=torch.bool, device="cuda")
    bad[50:110, 9, 77] = True
    assert torch.equal(torch.isnan(d["o"]), bad)
    lost = torch.zeros(out.shape[:3], dtype=torch.bool, device="cuda")
    lost[int(c["to"][1]), 9, 77] = True
    assert torch.equal(torch.isnan(out).all(-1), lost) and bool(torch.isfinite(out).all(-1)[~lost].all())
