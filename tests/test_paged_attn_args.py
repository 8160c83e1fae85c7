"""What PagedAttention makes of its arguments before the launch: on the CPU with the library's entry point
replaced by one that records what it is given, and on the GPU."""
import ctypes
import importlib.util
import pathlib
from types import SimpleNamespace

import pytest
import torch

from chain_flow_b200 import _lib

_spec = importlib.util.spec_from_file_location("paged_attn_cases", pathlib.Path(__file__).with_name("test_paged_attn.py"))
_cases = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(_cases)

H, HKV, D = 4, 2, 64


def _words(table):
    return table.untyped_storage().nbytes() // 4 - table.storage_offset()


def _read_table(monkeypatch, table, B):
    """The table as the entry point would read it (None: past the buffer's end), and the stride and width it is given."""
    from chain_flow_b200.attention import PagedAttention
    seen = []

    def entry(q, sq_t, sq_h, desc, at, stride, width, *rest):
        words = (B - 1) * stride + width if width else 0
        if at == table.data_ptr() and words > _words(table):
            seen.extend((None, stride, width))
        else:
            x = (ctypes.c_int32 * words).from_address(at) if words else []
            seen.extend(([[x[b * stride + j] for j in range(width)] for b in range(B)], stride, width))
        return 0

    monkeypatch.setattr(_lib, "stream_of", lambda device, what: 0)
    attn = object.__new__(PagedAttention)
    attn.__dict__.update(lib=SimpleNamespace(cfb_paged_attn=entry), device=torch.device("cpu"), heads=H, kv_heads=HKV, head_dim=D,
                         scale=0.125, ws_bytes=0, ws_ptr=0, _dev=-1)
    cache = SimpleNamespace(_dev=-1, device=torch.device("cpu"), k_scale=None, dtype=torch.float16, kv_heads=HKV, head_dim=D, desc=None)
    attn(torch.zeros(3, H, D, dtype=torch.float16), cache, table, torch.zeros(B, dtype=torch.int32), torch.zeros(B + 1, dtype=torch.int32))
    return seen


@pytest.mark.parametrize("table, B", [
    (torch.arange(5, dtype=torch.int32).view(1, 5).expand(3, 5), 3),                 # one prefix of several requests
    (torch.arange(5, dtype=torch.int64).view(1, 5).expand(3, 5), 3),
    (torch.arange(9, dtype=torch.int32).as_strided((3, 5), (2, 1)), 3),              # rows that overlap
    (torch.arange(3, dtype=torch.int32).view(3, 1).expand(3, 4), 3),
    (torch.full((1, 1), 7, dtype=torch.int32).expand(4, 1), 4),
    (torch.arange(40, dtype=torch.int32).view(4, 10)[:, :7], 4),                     # rows of a wider table
    (torch.arange(40, dtype=torch.int32).view(4, 10)[1:2, :7], 1),
    (torch.arange(5, dtype=torch.int32).as_strided((1, 5), (0, 1)), 1),
    (torch.zeros(2, 0, dtype=torch.int32), 2)])
def test_the_entry_point_reads_the_table_that_was_given(monkeypatch, table, B):
    read, stride, width = _read_table(monkeypatch, table, B)
    assert stride >= width == table.shape[1]
    assert read is not None, "the table's rows are read past its end"
    assert read == table.tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
def test_one_prefix_of_several_requests(causal):
    """An expanded table, and overlapping rows, give the bits of their contiguous copies."""
    from chain_flow_b200.attention import PagedAttention
    q, c, table, lens, cu = _cases._case([3, 3, 3], [75, 1, 1], H, HKV, D, 16, torch.float16, False, seed=21, stale=0.25)
    attn = PagedAttention(H, HKV, D)
    lens = torch.full_like(lens, 75)
    flat = table[0, :5].repeat(2)
    for view in (table[:1, :5].expand(3, 5), flat.as_strided((3, 5), (1, 1))):
        want = [t.clone() for t in attn(q, c, view.contiguous(), lens, cu, causal=causal)]
        got = attn(q, c, view, lens, cu, causal=causal)
        attn.check()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        _cases._check(got, _cases._want(q, c, view.contiguous(), lens, cu, causal), torch.float16)
