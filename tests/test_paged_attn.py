"""Attention of new tokens over a paged key/value cache (cfb_paged_attn).

CPU: the oracle's causal chunks agree with one pass over the whole prompt, and the C entry point
refuses what it does not take. GPU: against oracle.paged_attention (64 bits). With u the output
type's unit roundoff (2^-8 bf16, 2^-11 fp16), an output element may be off by its own rounding, u |o|,
and by the rounding of the softmax weights to the same type, u sum_j p_j |v_j| (the oracle's third
result); the fp32 scores, at most D 2^-24 |q| |k| scale (below 2e-5 here), move o and lse by as much
again. The weights are normalised by an fp32 sum, so nothing else enters."""
import ctypes as C

import pytest
import torch

import oracle
from chain_flow_b200 import _lib

FP8 = torch.float8_e4m3fn
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
FP32 = 2e-5


def test_oracle_chunks_equal_the_whole_prompt():
    g = torch.Generator().manual_seed(0)
    q = torch.randn(20, 4, 64, generator=g)
    k, v = (torch.randn(6, 2, 4, 64, generator=g).double() for _ in range(2))
    table = torch.tensor([[5, 0, 3, 1, 4]])
    whole, lse, _ = oracle.paged_attention(q, k, v, table, [20], [0, 20], 0.125, True)
    for a, b in ((0, 7), (7, 8), (8, 20)):
        part, pl, _ = oracle.paged_attention(q[a:b], k, v, table, [b], [0, b - a], 0.125, True)
        assert torch.allclose(part, whole[a:b]) and torch.allclose(pl, lse[:, a:b])


FAKE = 0x10000


def _call(c=None, **kw):
    lib = _lib.load()
    c = c or _lib.KvCache(FAKE, FAKE, None, None, 4 * 16 * 64, 16 * 64, 64, 0, 0, 0, 8, 16, 4, 64, 1)
    a = dict(q=FAKE, sq_t=512, sq_h=64, table=FAKE, st=8, width=8, kv_len=FAKE, cu_q=FAKE, o=FAKE, so_t=512, so_h=64, lse=FAKE,
             T=4, B=2, H=8, dtype=1, ws=FAKE, ws_bytes=lib.cfb_paged_attn_workspace(8, 4, 64))
    a.update(kw)
    return lib.cfb_paged_attn(a["q"], a["sq_t"], a["sq_h"], C.byref(c), a["table"], a["st"], a["width"], a["kv_len"], a["cu_q"],
                              a["o"], a["so_t"], a["so_h"], a["lse"], 0.125, a["T"], a["B"], a["H"], 1, a["dtype"], a["ws"],
                              a["ws_bytes"], None)


@pytest.mark.parametrize("change, status", [
    (dict(T=0), 0), (dict(B=0), 0), (dict(T=-1), 1), (dict(H=0), 1), (dict(H=6), 2), (dict(H=4 * 129), 2), (dict(st=7), 1),
    (dict(dtype=2), 2), (dict(dtype=0), 2), (dict(q=None), 1), (dict(o=None), 1), (dict(kv_len=None), 1), (dict(cu_q=None), 1),
    (dict(table=None), 1), (dict(ws=None), 1), (dict(sq_h=68), 1), (dict(so_t=516), 1), (dict(q=FAKE + 8), 1),
    (dict(ws=FAKE + 16), 3), (dict(ws_bytes=16), 3)])
def test_refusals_of_the_c_entry_point(change, status):
    assert _call(**change) == status


# ---- on the GPU -------------------------------------------------------------------------------------
def _case(news, lens, H, HKV, D, page, dtype, quant, seed=0, stale=float("nan")):
    """Inputs as a step has them; every slot that no request's positions use holds `stale`."""
    from chain_flow_b200.kv_cache import PagedKVCache
    g = torch.Generator().manual_seed(seed)
    per = [-(-n // page) for n in lens]
    pages = sum(per) + 3
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(lens), max(per + [1])), -5, dtype=torch.int32)         # unused entries: no page
    k, v = (torch.full((pages, HKV, page, D), stale) for _ in range(2))
    at = 0
    for b, n in enumerate(lens):
        table[b, :per[b]] = order[at:at + per[b]].int()
        at += per[b]
        j = torch.arange(n)
        k[table[b, j // page].long(), :, j % page] = torch.randn(n, HKV, D, generator=g)
        v[table[b, j // page].long(), :, j % page] = torch.randn(n, HKV, D, generator=g) + 0.5
    k, v = k.to(dtype), v.to(dtype)
    ks = vs = None
    if quant:
        (k, ks), (v, vs) = oracle.kv_quantise(k), oracle.kv_quantise(v)
        k, v, ks, vs = k.to(FP8), v.to(FP8), ks.cuda(), vs.cuda()
    cu = torch.tensor([0] + news).cumsum(0).int()
    qkv = torch.randn(sum(news), H + 3, D, generator=g).to(dtype).cuda()
    q = qkv[:, 1:H + 1]                                                              # a strided view
    return q, PagedKVCache.from_tensors(k.cuda(), v.cuda(), ks, vs), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), cu.cuda()


def _want(q, c, table, lens, cu, causal, scale=None):
    k, v = (oracle.kv_values(p.float().cpu(), None if s is None else s.cpu()) for p, s in ((c.k, c.k_scale), (c.v, c.v_scale)))
    return oracle.paged_attention(q.cpu(), k, v, table.cpu(), lens.cpu(), cu.cpu(), scale or q.shape[2] ** -0.5, causal)


def _check(got, want, dtype):
    o, lse, w = want
    err = (got[0].double().cpu() - o).abs()
    bound = ROUND[dtype] * (o.abs() + w) * 1.01 + FP32 * (w + 1)
    assert bool((err <= bound).all()), float((err / bound).max())
    finite = torch.isfinite(lse)
    assert torch.equal(finite, torch.isfinite(got[1].cpu()))
    assert bool((got[1].cpu()[~finite] == -torch.inf).all())
    assert bool(((got[1].double().cpu() - lse)[finite].abs() <= FP32 * (1 + lse[finite].abs())).all())


SHAPES = [(16, 4, 256), (6, 1, 256), (8, 2, 128), (5, 5, 128), (8, 8, 64), (7, 1, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("H, HKV, D", SHAPES)
@pytest.mark.parametrize("causal", [True, False])
def test_ragged_step(dtype, quant, H, HKV, D, causal):
    """Requests of no tokens, no context, one token, lengths round the tile and page sizes, and (causal)
    more new tokens than positions, so that rows see nothing. Stale slots hold NaN."""
    from chain_flow_b200.attention import PagedAttention
    news = [1, 0, 3, 64, 1, 33, 5, 1, 17]
    lens = [1, 40, 0, 64, 129, 200, 2, 65, 17]
    case = _case(news, lens, H, HKV, D, 17, dtype, quant, seed=H * D)
    got = PagedAttention(H, HKV, D)(*case, causal=causal)
    torch.cuda.synchronize()
    _check(got, _want(*case, causal), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, quant", [(torch.bfloat16, False), (torch.float16, True), (torch.float16, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("news, lens, H, HKV, D, page", [
    ([1], [5000], 16, 4, 256, 16), ([1] * 7, [1500, 3, 900, 64, 63, 2000, 1], 24, 4, 256, 544), ([41], [1300], 24, 4, 256, 16),
    ([300], [300], 4, 1, 128, 48), ([130, 1], [700, 900], 8, 2, 128, 1), ([150], [500], 2, 2, 64, 33)])
def test_long_contexts(dtype, quant, news, lens, H, HKV, D, page):
    from chain_flow_b200.attention import PagedAttention
    case = _case(news, lens, H, HKV, D, page, dtype, quant, seed=len(news))
    attn = PagedAttention(H, HKV, D)
    got = attn(*case)
    again = attn(*case)
    attn.check()
    _check(got, _want(*case, True), dtype)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.gpu
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_positions_that_are_not_allowed_have_no_influence(quant, poison):
    """A later token of a chunk with a NaN or an infinity in its key and value: earlier tokens do not see it."""
    from chain_flow_b200.attention import PagedAttention
    H, HKV, D, n, L, bad = 4, 2, 128, 40, 150, 130
    q, c, table, lens, cu = _case([n], [L], H, HKV, D, 16, torch.float16, quant, seed=3)
    slot = int(table[0, bad // 16]) * 16 + bad % 16
    row = torch.randn(1, HKV, D, device="cuda").half()
    clean = PagedAttention(H, HKV, D)(q, c, table, lens, cu)
    row[..., 7] = poison
    c.write(row, row, torch.tensor([slot], device="cuda"))
    got = PagedAttention(H, HKV, D)(q, c, table, lens, cu)
    torch.cuda.synchronize()
    first = bad - (L - n)                                   # the first row that sees it
    for x, y in zip(got, clean):
        rows, ref = (x[:first], y[:first]) if x is got[0] else (x[:, :first], y[:, :first])
        assert bool(torch.isfinite(rows).all())
        _close = (rows.double() - ref.double()).abs().max()
        assert float(_close) <= 2 * ROUND[torch.float16] * float(ref.abs().max())
    assert not bool(torch.isfinite(got[0][first:]).all(-1).any())


@pytest.mark.gpu
def test_scores_of_every_size():
    """Scores in the thousands, all alike, and far apart: the running maximum keeps the weights finite."""
    from chain_flow_b200.attention import PagedAttention
    q, c, table, lens, cu = _case([5, 2], [333, 70], 4, 4, 64, 16, torch.bfloat16, False, seed=5)
    for scale in (30.0, 1e-4, 0.125, -20.0):
        got = PagedAttention(4, 4, 64)(q, c, table, lens, cu, scale=scale, causal=False)
        o, lse, w = _want(q, c, table, lens, cu, False, scale)
        # fp32 scores of this size are off by up to D 2^-24 sum|q k| |scale|, and the weights by as much
        off = 64 * 2.0 ** -24 * 64 * 4 * abs(scale)
        assert bool(((got[0].double().cpu() - o).abs() <= ROUND[torch.bfloat16] * (o.abs() + w) * 1.01 + (FP32 + 2 * off) * (w + 1)).all())
        assert bool(((got[1].double().cpu() - lse).abs() <= FP32 * (1 + lse.abs()) + off).all())


@pytest.mark.gpu
@pytest.mark.parametrize("quant", [False, True])
def test_pages_outside_the_pool_and_lengths_past_the_table(quant):
    from chain_flow_b200.attention import PagedAttention
    H, HKV, D = 4, 2, 64
    q, c, table, lens, cu = _case([2, 3, 2, 2], [100, 80, 64, 70], H, HKV, D, 16, torch.float16, quant, seed=9)
    attn = PagedAttention(H, HKV, D)
    want = [t.clone() for t in attn(q, c, table, lens, cu)]
    table[0, 2], table[1, 4] = c.pages, -1                  # request 0: position 32 on; request 1: positions 64 .. 79
    lens[2] = table.shape[1] * 16 + 1                       # past what the table holds
    o, lse = attn(q, c, table, lens, cu)
    torch.cuda.synchronize()
    assert bool(torch.isnan(o[:7]).all()) and bool(torch.isnan(lse[:, :7]).all())
    assert torch.equal(o[7:], want[0][7:]) and torch.equal(lse[:, 7:], want[1][:, 7:])
    lens[2] = -3                                            # a negative length: no positions
    o, lse = attn(q, c, table, lens, cu)
    torch.cuda.synchronize()
    assert bool((o[5:7] == 0).all()) and bool((lse[:, 5:7] == -torch.inf).all())


@pytest.mark.gpu
def test_rows_of_no_request_are_left_alone():
    from chain_flow_b200.attention import PagedAttention
    q, c, table, lens, cu = _case([4, 5], [30, 50], 4, 2, 64, 16, torch.float16, False, seed=2)
    q = torch.cat([q, torch.full_like(q, float("nan"))])
    out, lse = torch.full((18, 4, 64), 7.0, device="cuda").half(), torch.full((4, 18), 7.0, device="cuda")
    PagedAttention(4, 2, 64)(q, c, table, lens, cu + 2, out=out, lse=lse)
    torch.cuda.synchronize()
    assert bool((out[:2] == 7).all()) and bool((out[11:] == 7).all())
    assert bool((lse[:, :2] == 7).all()) and bool((lse[:, 11:] == 7).all())
    assert not bool((out[2:11] == 7).all(-1).any())


@pytest.mark.gpu
def test_prefix_and_tree_join_to_full_attention():
    """The prefix half (causal=False) merged with the tree half equals attention over both."""
    from chain_flow_b200.attention import PagedAttention
    from chain_flow_b200.gdn import make_tree
    from chain_flow_b200.tree import ancestor_mask, tree_attn_merge
    S, N, H, HKV, D, dtype = 2, 12, 8, 2, 128, torch.float16
    q, c, table, lens, cu = _case([N] * S, [90, 33], H, HKV, D, 16, dtype, False, seed=4)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(S * N, HKV, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    parents = torch.stack([make_tree(N, 4, 3, seed=s)[0] for s in range(S)]).cuda()
    mask = ancestor_mask(parents)
    po, pl = PagedAttention(H, HKV, D)(q, c, table, lens, cu, causal=False)
    rows = torch.arange(S * N, device="cuda").view(S, N)
    out = tree_attn_merge(q, k, v, torch.zeros_like(po), po, pl, rows, mask, D ** -0.5)
    torch.cuda.synchronize()
    for s in range(S):
        j = torch.arange(int(lens[s]))
        slot = table[s].cpu().long()[j // 16] * 16 + j % 16
        pk, pv = (x.cpu().transpose(1, 2).reshape(-1, HKV, D)[slot].double() for x in (c.k, c.v))
        for m in range(N):
            anc = [s * N + n for n in range(N) if mask[s, m, n] == 0]
            for h in range(H):
                kh, vh = (torch.cat([p[:, h // 4], t.cpu().double()[anc, h // 4]]) for p, t in ((pk, k), (pv, v)))
                p = torch.softmax(kh @ q[s * N + m, h].cpu().double() * D ** -0.5, 0)
                want, w = p @ vh, p @ vh.abs()
                # prefix and tree half are rounded, weighted and rounded again
                assert bool(((out[s * N + m, h].cpu().double() - want).abs() <= 4 * ROUND[dtype] * (want.abs() + w) + FP32).all())


@pytest.mark.gpu
def test_offsets_past_32_bits():
    from chain_flow_b200.attention import PagedAttention
    from chain_flow_b200.kv_cache import PagedKVCache
    page, HKV, D = 16, 8, 256
    pages = (1 << 32) // (page * HKV * D) + 2
    if torch.cuda.mem_get_info()[0] < 5 * pages * page * HKV * D:
        pytest.skip("needs 22 GB of device memory")
    k, v = (torch.empty(pages, HKV, page, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    lens, cu = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([40], [0, 3]))
    for p in (pages - 1, 0, pages - 2):
        k[p].normal_(), v[p].normal_()
    q = torch.randn(3, 8, D, device="cuda").bfloat16()
    c = PagedKVCache.from_tensors(k, v)
    got = PagedAttention(8, HKV, D)(q, c, table, lens, cu)
    torch.cuda.synchronize()
    small = PagedKVCache.from_tensors(k[[pages - 1, 0, pages - 2]].contiguous(), v[[pages - 1, 0, pages - 2]].contiguous())
    _check(got, _want(q, small, torch.tensor([[0, 1, 2]]), lens, cu, True), torch.bfloat16)


@pytest.mark.gpu
def test_another_layout_stream_and_capture():
    from chain_flow_b200.attention import PagedAttention
    from chain_flow_b200.kv_cache import PagedKVCache
    q, c, table, lens, cu = _case([3, 1], [100, 70], 4, 2, 128, 16, torch.bfloat16, False, seed=8)
    attn = PagedAttention(4, 2, 128)
    want = attn(q, c, table, lens, cu)
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (c.k, c.v)]       # [pages, page, heads, dim]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = attn(q, PagedKVCache.from_tensors(*turned), table.long(), lens.long(), cu.long(), stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    out, lse = torch.empty_like(want[0]), torch.empty_like(want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attn(q, c, table, lens, cu, out=out, lse=lse)
    lens -= 1
    graph.replay()
    want = attn(q, c, table, lens, cu)
    torch.cuda.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


@pytest.mark.gpu
def test_refusals_in_python():
    from chain_flow_b200.attention import PagedAttention
    from chain_flow_b200.kv_cache import PagedKVCache
    for args in ((4, 3, 64), (4, 0, 64), (4, 4, 96), (0, 1, 64), (129, 1, 64)):
        with pytest.raises(_lib.CfbError):
            PagedAttention(*args)
    q, c, table, lens, cu = _case([3, 1], [10, 7], 4, 2, 64, 16, torch.float16, False)
    attn = PagedAttention(4, 2, 64)
    other = PagedKVCache(4, 16, 4, 64)
    good = dict(query=q, cache=c, page_table=table, kv_len=lens, cu_q=cu)
    for change in (dict(query=q.bfloat16()), dict(query=q[:, :2]), dict(query=q.cpu()), dict(cache=other), dict(cu_q=cu[:2]),
                   dict(page_table=table[:1]), dict(kv_len=lens.cpu()), dict(out=torch.empty_like(q).float()),
                   dict(lse=torch.empty(4, 4, device="cuda").half()), dict(lse=torch.empty(4, 5, device="cuda"))):
        with pytest.raises(_lib.CfbError):
            attn(**{**good, **change})
