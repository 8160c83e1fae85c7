"""The outputs' products over chunks round their operands (11 bits over bf16, 22 over fp16) to nearest: no share of
every output is lost.

An operand cut off would make each term, and so each output, smaller by its own part: 2^-11 and more of it. Rounding to
nearest errs either way. With o at most 2^-9 of itself off by its own rounding over bf16, the mean of N outputs' errors, taken
along their signs, has a deviation of 2^-9 / sqrt(N) of the mean magnitude: 2^-16.5 for the 32768 here and less over fp16.
The bound, 2^-13, is eleven of them."""
import importlib.util
import pathlib

import pytest
import torch

_spec = importlib.util.spec_from_file_location("gdn_seq_cases", pathlib.Path(__file__).with_name("test_gdn_seq.py"))
_cases = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(_cases)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens, HV", [([64], 4), ([32, 32], 4), ([10, 3, 1, 7, 11] * 2, 4)])
def test_outputs_lean_neither_way(dtype, lens, HV):
    c = _cases._case(lens, 2, HV, 128, dtype, seed=3, zero_start=False)
    want = _cases._oracle(c)[0]
    d = _cases._gpu(c)
    _cases._run(d)
    lean = ((d["o"].double().cpu() - want) * want.sign()).mean() / want.abs().mean()
    assert abs(float(lean)) <= 2.0 ** -13, float(lean) * 2 ** 13


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, HV", [(torch.bfloat16, 4), (torch.float16, 4), (torch.bfloat16, 64)])       # 64: four tiles a CTA
@pytest.mark.parametrize("name", ["q", "k", "v", "a", "b", "state"])
def test_nan_comes_out_where_the_formula_has_it(dtype, HV, name):
    """Rounding a NaN's pattern like a number's would make it one."""
    lens = [40, 70] if HV == 4 else [40, 70, 3, 33]
    c = _cases._case(lens, 2, HV, 128, dtype, seed=4, zero_start=False)
    if name == "state":
        c[name][int(c["init"][0]), 1, 5, 9] = float("nan")
    else:
        x = c[name]
        x[(37, 1) if x.dim() == 2 else (37, 1, 5)] = float("nan")
    want, state = _cases._oracle(c)
    d = _cases._gpu(c)
    _cases._run(d)
    assert torch.equal(torch.isnan(d["o"].cpu()), torch.isnan(want))
    to = c["to"].long()
    assert torch.equal(torch.isnan(d["state"].cpu()[to]).any(-1), torch.isnan(state[to]).any(-1))
