"""The paged key/value cache (cfb_kv_write / cfb_kv_read): rows written, quantised to e4m3 where the
cache holds it, and read back. Codes and scales are single fp32 operations, so they are compared bit
by bit with oracle.kv_quantise; a read is one product rounded once, so it is too."""
import ctypes as C

import pytest
import torch

import oracle
from chain_flow_b200 import _lib

FP8 = torch.float8_e4m3fn


def test_quantised_rows_stay_within_half_a_step():
    """The oracle's format: the largest element is kept to fp32 accuracy, every other one to half a
    step of e4m3 (2^-4 relative, or 2^-10 of a code below the smallest normal 2^-6)."""
    x = torch.randn(64, 128, generator=torch.Generator().manual_seed(0)) * torch.logspace(-6, 4, 64)[:, None]
    code, scale = oracle.kv_quantise(x)
    err = (code.double() * scale.double()[:, None] - x.double()).abs()
    step = torch.maximum(x.double().abs() * 2.0 ** -4, scale.double()[:, None] * 2.0 ** -10)
    assert bool((err <= step * (1 + 1e-6)).all())
    top = x.abs().argmax(-1, keepdim=True)
    assert bool(((code * scale[:, None]).gather(1, top) - x.gather(1, top)).abs().le(1e-6 * x.abs().amax(-1, keepdim=True)).all())


def test_quantise_edges():
    x = torch.zeros(4, 64)
    x[1, 3], x[2, 5], x[3, :] = float("nan"), float("-inf"), 2.0 ** -30
    code, scale = oracle.kv_quantise(x)
    assert scale[0] > 0 and bool((code[0] == 0).all())
    assert bool(torch.isnan(scale[1:3]).all()) and bool((code[1:3] == 0).all())
    assert float((code[3] * scale[3] - x[3]).abs().max()) <= 2.0 ** -42


FAKE = 0x10000                                       # argument checks only do arithmetic on pointers


def _fake_cache(**kw):
    c = _lib.KvCache(FAKE, FAKE, None, None, 4 * 16 * 64, 16 * 64, 64, 0, 0, 0, 8, 16, 4, 64, 1)
    for n, x in kw.items():
        setattr(c, n, x)
    return c


@pytest.mark.parametrize("change, status", [
    (dict(), 0), (dict(k=None), 1), (dict(pages=0), 1), (dict(page_size=0), 1), (dict(kv_heads=0), 1), (dict(dim=96), 2),
    (dict(dtype=0), 2), (dict(dtype=3), 1), (dict(k_scale=FAKE), 1), (dict(slot_stride=68), 1), (dict(v=FAKE + 8), 1)])
def test_refusals_of_the_c_entry_points(change, status):
    lib = _lib.load()
    c = _fake_cache(**change)
    assert lib.cfb_kv_write(C.byref(c), FAKE, 256, 64, FAKE, 256, 64, 1, FAKE, 0, None) == status
    assert lib.cfb_kv_read(C.byref(c), FAKE, 0, FAKE, 256, 64, FAKE, 256, 64, 1, None) == status


def test_refusals_of_the_rows():
    lib = _lib.load()
    c = _fake_cache()
    w = lambda *a: lib.cfb_kv_write(C.byref(c), *a, None)
    r = lambda *a: lib.cfb_kv_read(C.byref(c), *a, None)
    assert w(FAKE, 256, 64, FAKE, 256, 64, 1, FAKE, -1) == 1
    assert w(None, 256, 64, FAKE, 256, 64, 1, FAKE, 4) == 1
    assert w(FAKE, 256, 64, FAKE, 256, 64, 2, FAKE, 0) == 2          # a 16-bit cache takes its own dtype
    assert w(FAKE, 256, 68, FAKE, 256, 64, 1, FAKE, 0) == 1          # rows not 16-byte aligned
    assert w(FAKE, 256, 64, FAKE, 256, 64, 0, FAKE, 0) == 2          # fp32 rows
    assert r(FAKE, 4, None, 256, 64, FAKE, 256, 64, 1) == 1
    assert r(FAKE, 0, FAKE, 256, 64, FAKE, 256, 64, 3) == 2
    assert lib.cfb_kv_write(None, FAKE, 256, 64, FAKE, 256, 64, 1, FAKE, 0, None) == 1


def test_cpu_tensors_are_refused():
    from chain_flow_b200.kv_cache import PagedKVCache
    k = torch.zeros(2, 1, 16, 64, dtype=torch.float16)
    with pytest.raises(_lib.CfbError):
        PagedKVCache.from_tensors(k, k.clone())


# ---- on the GPU -------------------------------------------------------------------------------------
def _cache(pages, page, heads, dim, dtype, layout="head", seed=1):
    """A cache over random stale rows; layout "token": the buffers are [pages, page, heads, dim]."""
    from chain_flow_b200.kv_cache import PagedKVCache
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (pages, heads, page, dim) if layout == "head" else (pages, page, heads, dim)
    k, v = (torch.randn(shape, device="cuda", generator=g).to(dtype) for _ in range(2))
    ks = vs = None
    if dtype == FP8:
        ks, vs = (torch.rand(shape[:3], device="cuda", generator=g) for _ in range(2))
    if layout == "token":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
        ks, vs = (None if t is None else t.transpose(1, 2) for t in (ks, vs))
    return PagedKVCache.from_tensors(k, v, ks, vs)


def _f32(t):
    return t.float().cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("tokens, page, heads, dim, layout", [
    (1, 16, 4, 256, "head"), (37, 16, 4, 256, "token"), (130, 17, 1, 64, "head"), (65, 48, 3, 128, "token"),
    (513, 32, 8, 64, "head")])
def test_write_and_read(dtype, quant, tokens, page, heads, dim, layout):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    pages = tokens // page + 3
    c = _cache(pages, page, heads, dim, FP8 if quant else dtype, layout)
    before = [None if t is None else _f32(t) for t in (c.k, c.v, c.k_scale, c.v_scale)]
    qkv = (torch.randn(tokens, 3 * heads, dim, device="cuda", generator=g) *
           torch.logspace(-6, 2, tokens, device="cuda")[:, None, None]).to(dtype)
    key, value = qkv[:, heads:2 * heads], qkv[:, 2 * heads:]                       # strided views
    if tokens > 8:
        key[2, 0, 5] = float("nan")
        value[3, heads - 1, dim - 1] = float("inf")
        key[4], value[5] = 0, 2.0 ** -20
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:tokens]
    if tokens > 8:
        slots[0], slots[7] = -1, pages * page                                      # both skipped
    c.write(key, value, slots)
    torch.cuda.synchronize()
    live = ((slots >= 0) & (slots < pages * page)).cpu()
    s = slots.cpu()[live]
    for x, pool, scale, old, old_scale in ((key, c.k, c.k_scale, before[0], before[2]),
                                           (value, c.v, c.v_scale, before[1], before[3])):
        want, want_scale = old.clone(), None if old_scale is None else old_scale.clone()
        rows = _f32(x)[live]
        if quant:
            rows, sc = oracle.kv_quantise(rows)
            want_scale[s // page, :, s % page] = sc
            assert torch.equal(torch.nan_to_num(_f32(scale), nan=-7.0), torch.nan_to_num(want_scale, nan=-7.0))
        want[s // page, :, s % page] = rows
        assert torch.equal(torch.nan_to_num(_f32(pool), nan=-7.0), torch.nan_to_num(want, nan=-7.0))
    for out in (dtype, torch.float32, torch.bfloat16 if dtype == torch.float16 else torch.float16):
        got = c.read(slots, dtype=out)
        for x, pool, scale in ((got[0], c.k, c.k_scale), (got[1], c.v, c.v_scale)):
            want = torch.zeros(tokens, heads, dim)
            rows = _f32(pool)[s // page, :, s % page]
            want[live] = rows if scale is None else rows * _f32(scale)[s // page, :, s % page][..., None]
            assert x.dtype == out
            assert torch.equal(torch.nan_to_num(_f32(x), nan=-7.0), torch.nan_to_num(want.to(out).float(), nan=-7.0))


@pytest.mark.gpu
def test_every_code_reads_as_its_value():
    c = _cache(1, 16, 1, 256, FP8)
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")
    codes[codes & 0x7f == 0x7f] = 0
    c.k.view(torch.uint8)[0, 0, 3], c.k_scale[0, 0, 3] = codes, 0.25
    got, _ = c.read(torch.tensor([3], device="cuda"), dtype=torch.float32)
    assert torch.equal(got[0, 0].cpu(), codes.cpu().view(FP8).float() * 0.25)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A pool whose last rows lie more than 2^32 elements from its first."""
    from chain_flow_b200.kv_cache import PagedKVCache
    page, heads, dim = 16, 8, 256
    pages = (1 << 32) // (page * heads * dim) + 2
    if torch.cuda.mem_get_info()[0] < 3 * pages * page * heads * dim:
        pytest.skip("needs 13 GB of device memory")
    k, v = (torch.empty(pages, heads, page, dim, dtype=torch.uint8, device="cuda").view(FP8) for _ in range(2))
    ks, vs = (torch.zeros(pages, heads, page, device="cuda") for _ in range(2))
    c = PagedKVCache.from_tensors(k, v, ks, vs)
    x = torch.randn(2, heads, dim, device="cuda", dtype=torch.float16)
    slots = torch.tensor([pages * page - 1, 5], device="cuda")
    c.write(x, -x, slots)
    got = c.read(slots, dtype=torch.float32)
    code, scale = oracle.kv_quantise(x.cpu())
    assert torch.equal(got[0].cpu(), code * scale[..., None]) and torch.equal(got[1].cpu(), -code * scale[..., None])


@pytest.mark.gpu
def test_no_tokens_another_stream_and_capture():
    c = _cache(4, 16, 2, 64, FP8)
    old = c.k.clone()
    none = torch.empty(0, 2, 64, device="cuda", dtype=torch.float16)
    c.write(none, none, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert c.read(torch.empty(0, dtype=torch.int64, device="cuda"))[0].shape == (0, 2, 64)
    assert torch.equal(c.k.view(torch.uint8), old.view(torch.uint8))
    x = torch.randn(3, 2, 64, device="cuda", dtype=torch.float16)
    slots = torch.tensor([3, 40, 17], dtype=torch.int32, device="cuda")            # converted on the given stream
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    c.write(x, x, slots, stream=side)
    got = c.read(slots, dtype=torch.float32, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    code, scale = oracle.kv_quantise(x.cpu())
    assert torch.equal(got[0].cpu(), code * scale[..., None])
    s64 = slots.long()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.write(x, x, s64)
    x.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c.read(s64, dtype=torch.float32)[0].cpu(), code * scale[..., None] * 2)


@pytest.mark.gpu
def test_refusals_in_python():
    from chain_flow_b200.kv_cache import PagedKVCache
    c = PagedKVCache(4, 16, 2, 64, dtype=torch.float16)
    x = torch.zeros(3, 2, 64, device="cuda", dtype=torch.float16)
    s = torch.arange(3, device="cuda")
    for key, value, slots in ((x.bfloat16(), x.bfloat16(), s), (x, x.bfloat16(), s), (x[:2], x, s), (x, x, s.float()),
                              (x, x, s.cpu()), (x.cpu(), x, s), (x.transpose(0, 1), x, s),
                              (x, torch.zeros(3, 64, 2, device="cuda", dtype=torch.float16).transpose(1, 2), s)):
        with pytest.raises(_lib.CfbError):
            c.write(key, value, slots)
    with pytest.raises(_lib.CfbError):
        c.read(s, dtype=torch.float64)
    k = torch.zeros(2, 1, 16, 64, device="cuda", dtype=torch.float16)
    k8 = k.to(FP8)
    sc = torch.zeros(2, 1, 16, device="cuda")
    for args in ((k, k.bfloat16()), (k.float(), k.float()), (k, k, sc, sc), (k8, k8), (k8, k8, sc, sc.half()), (k[..., ::2], k[..., ::2]),
                 (torch.zeros(2, 1, 16, 96, device="cuda").half(),) * 2, (k[:0], k[:0])):
        with pytest.raises(_lib.CfbError):
            PagedKVCache.from_tensors(*args)
