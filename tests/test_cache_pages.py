"""A cache's pages and rows (cfb_kv_keep, cfb_kv_copy_pages, cfb_pages_reserve / release / fork) against oracle.pages. All
of it is copies and whole numbers: everything has to be equal, what a call leaves alone included."""
import ctypes as C
import random

import pytest
import torch

from chain_flow_b200 import _lib
from oracle import pages as oracle

FP8 = torch.float8_e4m3fn
FAKE = 0x10000


# ---- CPU ------------------------------------------------------------------------------------------------
def test_the_oracle_hands_out_the_lowest_pages_in_order():
    refs, table = [0, 1, 0, 0, 2, 0], [[9, -1, -1], [-1, -1, -1], [-1, -1, -1]]
    assert oracle.reserve(refs, table, [4, 0, 0], [9, 4, 20], 4) == [1, 1, 0]
    assert table == [[9, 0, 2], [3, -1, -1], [-1, -1, -1]] and refs == [1, 1, 1, 1, 2, 0]
    assert oracle.reserve(refs, table, [9, 4, 0], [9, 5, 1], 4) == [1, 1, 0]             # the third finds none left
    length = [9, 5, 0]
    assert oracle.release(refs, table, [9, 5, 0], [4, 0, 0], 4) and refs == [0, 1, 0, 0, 2, 0]
    assert table[0] == [9, -1, -1] and not oracle.release(refs, [[0]], [1], None, 4)
    refs, table = [1, 0, 1], [[2, 0], [-1, -1]]
    assert oracle.fork(refs, table, length[:1] + [0], [0, 0], [1, 7], 5) == ([1, 0], [(0, 1, 4)])
    assert table[1] == [2, 1] and refs == [1, 1, 2]


def _cache(**kw):
    c = _lib.KvCache(FAKE, FAKE, None, None, 4 * 16 * 64, 16 * 64, 64, 0, 0, 0, 8, 16, 4, 64, 1)
    for n, x in kw.items():
        setattr(c, n, x)
    return c


def _array(*caches):
    return (C.c_void_p * len(caches))(*[C.addressof(c) for c in caches])


def test_refusals_of_the_entry_points():
    lib = _lib.load()
    a, b, flat, odd, few = _cache(), _cache(page_stride=2 * 4 * 16 * 64), _cache(dim=96), _cache(page_size=17), _cache(pages=7)
    one, two = _array(a), _array(a, b)
    keep = lambda d, n, *x: lib.cfb_kv_keep(d, n, *x, None)  # noqa: E731
    assert keep(one, 1, FAKE, 4, 4, FAKE, FAKE, 5, FAKE, 5, 0) == 0
    assert keep(two, 2, FAKE, 4, 4, FAKE, FAKE, 5, FAKE, 5, 0) == 1                 # two geometries
    assert keep(None, 1, FAKE, 4, 4, FAKE, FAKE, 5, FAKE, 5, 0) == 1
    assert keep(one, 1, FAKE, 3, 4, FAKE, FAKE, 5, FAKE, 5, 2) == 1                 # rows of the table that share words
    assert keep(one, 1, FAKE, 4, 4, FAKE, FAKE, 4, FAKE, 5, 2) == 1
    assert keep(one, 1, FAKE, 4, 4, FAKE, FAKE, 5, FAKE, 5, -1) == 1
    assert keep(one, 1, None, 4, 4, FAKE, FAKE, 5, FAKE, 5, 2) == 1
    assert keep(one, 1, FAKE, 4, 4, FAKE, FAKE, 2000, FAKE, 2000, 2) == 2
    copy = lambda d, n, *x: lib.cfb_kv_copy_pages(d, n, *x, None)  # noqa: E731
    assert copy(one, 1, None, None, None, 0) == 0 and copy(one, 1, None, FAKE, None, 3) == 1 and copy(one, 1, FAKE, FAKE, None, -1) == 1
    assert copy(two, 2, FAKE, FAKE, None, 3) == 1 and copy(_array(flat), 1, FAKE, FAKE, None, 3) == 2
    reserve = lambda *x: lib.cfb_pages_reserve(*x, None)  # noqa: E731
    assert reserve(FAKE, 10, 16, FAKE, 4, 4, FAKE, FAKE, FAKE, 0) == 0
    for bad in ((None, 10, 16, FAKE, 4, 4, FAKE, FAKE, FAKE, 2), (FAKE, 0, 16, FAKE, 4, 4, FAKE, FAKE, FAKE, 2),
                (FAKE, 10, 0, FAKE, 4, 4, FAKE, FAKE, FAKE, 2), (FAKE, 10, 16, None, 4, 4, FAKE, FAKE, FAKE, 2),
                (FAKE, 10, 16, FAKE, 3, 4, FAKE, FAKE, FAKE, 2), (FAKE, 10, 16, FAKE, 4, 4, None, FAKE, FAKE, 2),
                (FAKE, 10, 16, FAKE, 4, 4, FAKE, None, FAKE, 2), (FAKE, 10, 16, FAKE, 4, 4, FAKE, FAKE, None, 2),
                (FAKE, 10, 16, FAKE, 4, 4, FAKE, FAKE, FAKE, -1)):
        assert reserve(*bad) == 1
    assert reserve(FAKE, (1 << 20) + 1, 16, FAKE, 4, 4, FAKE, FAKE, FAKE, 2) == 2
    release = lambda *x: lib.cfb_pages_release(*x, None, None)  # noqa: E731
    assert release(FAKE, 10, 16, FAKE, 4, 4, FAKE, None, 0) == 0 and release(FAKE, 10, 16, FAKE, 4, 4, None, None, 2) == 1
    fork = lambda *x: lib.cfb_pages_fork(*x, None)  # noqa: E731
    head = (FAKE, 8, 16, FAKE, 4, 4, 6)
    assert fork(*head, FAKE, FAKE, FAKE, FAKE, 0, one, 1) == 0
    for bad in ((None, FAKE, FAKE, FAKE, 2, one, 1), (FAKE, None, FAKE, FAKE, 2, one, 1), (FAKE, FAKE, None, FAKE, 2, one, 1),
                (FAKE, FAKE, FAKE, None, 2, one, 1), (FAKE, FAKE, FAKE, FAKE, -1, one, 1), (FAKE, FAKE, FAKE, FAKE, 2, None, 1),
                (FAKE, FAKE, FAKE, FAKE, 2, _array(odd), 1), (FAKE, FAKE, FAKE, FAKE, 2, _array(few), 1)):
        assert fork(*head, *bad) == 1, bad


# ---- GPU --------------------------------------------------------------------------------------------------
def _caches(layers, pages, page, heads, dim, dtype, layout="head", seed=1):
    from chain_flow_b200.kv_cache import PagedKVCache
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for _ in range(layers):
        shape = (pages, heads, page, dim) if layout == "head" else (pages, page, heads, dim)
        k, v = (torch.randint(0, 127, (*shape, 1 if dtype == FP8 else 2), device="cuda", generator=g, dtype=torch.uint8) for _ in range(2))
        k, v = (t.view(dtype).squeeze(-1) for t in (k, v))
        ks = vs = None
        if dtype == FP8:
            ks, vs = (torch.rand(shape[:3], device="cuda", generator=g) for _ in range(2))
        if layout == "token":
            k, v = k.transpose(1, 2), v.transpose(1, 2)
            ks, vs = (None if t is None else t.transpose(1, 2) for t in (ks, vs))
        out.append(PagedKVCache.from_tensors(k, v, ks, vs))
    return out


def _pools(caches):
    """What the caches hold, as CPU tensors whose equality means equal bytes."""
    bits = lambda t: t.contiguous().view(torch.uint8 if t.dtype == FP8 else torch.int32 if t.dtype == torch.float32 else torch.int16).cpu()  # noqa: E731
    return [bits(t) for c in caches for t in (c.k, c.v, c.k_scale, c.v_scale) if t is not None]


def _same(caches, want):
    torch.cuda.synchronize()
    for a, b in zip(_pools(caches), want):
        assert torch.equal(a, b)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, layout", [(torch.float16, "head"), (torch.bfloat16, "token"), (FP8, "head"), (FP8, "token")])
@pytest.mark.parametrize("layers, B, page, heads, dim, depth", [(1, 1, 16, 4, 256, 5), (8, 3, 17, 1, 64, 1), (35, 2, 16, 2, 128, 9),
                                                                (2, 5, 1, 3, 128, 70), (1, 2, 48, 40, 256, 30), (3, 70, 16, 8, 64, 4)])
def test_kept_rows(dtype, layout, layers, B, page, heads, dim, depth):
    from chain_flow_b200.kv_cache import keep_path
    rng = random.Random(depth + B)
    nodes, width = depth + 9, (30 + depth + 9) // page + 2
    pages = B * width + 2
    caches = _caches(layers, pages, page, heads, dim, dtype, layout)
    order = list(range(pages))
    rng.shuffle(order)
    table = [order[b * width:(b + 1) * width] for b in range(B)]
    base = [rng.randint(0, 30) for _ in range(B)]
    length = [rng.randint(0, depth) if b else depth for b in range(B)]
    path = [sorted(rng.sample(range(nodes), n)) + [rng.choice([-1, 1 << 30])] * (depth - n) for n in length]
    if B > 2:
        path[1], length[1] = list(range(depth)), depth                   # everything stays
        table[2] = [p if j % 2 else rng.choice([-1, pages, 1 << 31 - 1]) for j, p in enumerate(table[2])]
    want = _pools(caches)
    oracle.keep_path(want, table, base, path, length, page)
    keep_path(caches, _i32(table), _i32(base), _i32(path), _i32(length))
    _same(caches, want)


@pytest.mark.gpu
def test_kept_rows_at_the_tables_end():
    """Positions past the table, negative ones, lengths past the path, a verifier's views as they come."""
    from chain_flow_b200.kv_cache import keep_path
    caches = _caches(1, 6, 16, 2, 64, torch.float16)
    want = _pools(caches)
    table, base, path, length = [[0, 1], [2, 3], [4, 5]], [26, -3, 0], [[1, 4, 9], [0, 1, 5], [2, 3, 4]], [3, 3, 7]
    oracle.keep_path(want, table, base, path, length, 16)
    wide = torch.full((3, 9), 7, dtype=torch.int32, device="cuda")
    wide[:, :3] = _i32(path)
    keep_path(caches[0], _i32(table).long(), _i32(base).long(), wide[:, :3], _i32(length))
    _same(caches, want)
    keep_path(caches, _i32(table), _i32(base), _i32(path), _i32([0, -5, 0]))
    keep_path(caches, _i32(table)[:0], _i32(base)[:0], _i32(path)[:0], _i32(length)[:0])
    keep_path(caches, _i32(table), _i32(base), _i32(path)[:, :0], _i32(length))
    _same(caches, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, layout", [(torch.float16, "head"), (torch.bfloat16, "token"), (FP8, "head"), (FP8, "token")])
@pytest.mark.parametrize("layers, pages, page, heads, dim", [(1, 7, 16, 4, 256), (4, 50, 17, 1, 64), (33, 9, 48, 3, 128), (2, 301, 1, 8, 64)])
def test_copied_pages(dtype, layout, layers, pages, page, heads, dim):
    from chain_flow_b200.kv_cache import copy_pages
    rng = random.Random(pages)
    caches = _caches(layers, pages, page, heads, dim, dtype, layout)
    order = list(range(pages))
    rng.shuffle(order)
    n = pages // 2
    src, dst = order[:n], order[n:2 * n]
    src[0], dst[-1] = rng.choice([-1, pages]), rng.choice([-7, pages, 1 << 30])
    slots = [rng.randint(-1, page + 1) for _ in range(n)]
    want = _pools(caches)
    oracle.copy_pages(want, src, dst, None)
    copy_pages(caches, _i32(src), _i32(dst))
    _same(caches, want)
    oracle.copy_pages(want, dst, src, slots)
    copy_pages(caches, _i32(dst).long(), _i32(src), slots=_i32(slots))
    _same(caches, want)
    copy_pages(caches, _i32([]), _i32([]))
    copy_pages([], _i32([]), _i32([]))
    _same(caches, want)


def _check_pool(pool, table, refs, rows):
    torch.cuda.synchronize()
    assert pool.refs.tolist() == refs and table.tolist() == rows


@pytest.mark.gpu
@pytest.mark.parametrize("pages, page, B, width", [(1, 16, 1, 1), (7, 1, 3, 9), (33, 16, 5, 12), (257, 17, 40, 30), (5000, 16, 1500, 11),
                                                   (8193, 16, 300, 700), (70001, 48, 64, 1000), (1 << 20, 16, 9, 2000)])
def test_the_pool(pages, page, B, width):
    """Random steps: taken, given back, forked, until the pool runs out and after."""
    from chain_flow_b200.kv_cache import PagePool
    rng = random.Random(pages + B)
    if pages < 100000:
        refs = [0 if rng.random() < 0.7 else rng.randint(1, 3) for _ in range(pages)]
    else:
        refs = [0 if p > pages - 3000 or p % 5000 == 77 else 1 for p in range(pages)]
    pool = PagePool.from_refs(_i32(refs), page)
    rows = [[-1] * width for _ in range(B)]
    wide = torch.full((B, width + 3), -1, dtype=torch.int32, device="cuda")
    table = wide[:, :width]
    length = [0] * B
    most = min(width * page, max(page, 3 * pages * page // B))
    for step in range(6):
        target = [n if rng.random() < 0.2 else rng.randint(0, most) if rng.random() < 0.8 else n + rng.randint(1, 2 * page) for n in length]
        if step == 3:
            target[rng.randrange(B)] = (width + 1) * page                # longer than a row
            target[rng.randrange(B)] = -5
        got = pool.reserve(table, _i32(length), _i32(target))
        want = oracle.reserve(refs, rows, length, target, page)
        assert got.tolist() == want
        length = [max(n, t) if ok else n for n, t, ok in zip(length, target, want)]
        _check_pool(pool, table, refs, rows)
        free = [b for b in range(B) if length[b] == 0]
        held = [b for b in range(B) if length[b] > 0]
        if free and held:
            n = min(len(free), 5)
            child, parent = free[:n] + [B, held[0]], [rng.choice(held) for _ in range(n)] + [held[0], held[0]]
            at = _i32(length)
            got = pool.fork(table, at, _i32(parent), _i32(child))
            want, _ = oracle.fork(refs, rows, length, parent, child, page)
            assert got.tolist() == want and at.tolist() == length
            _check_pool(pool, table, refs, rows)
        keep = [rng.choice([0, 0, n, max(n - 1, 0), n // 2, n + 5]) for n in length]
        pool.release(table, _i32(length), _i32(keep))
        assert oracle.release(refs, rows, length, keep, page)
        length = [min(n, k) for n, k in zip(length, keep)]
        _check_pool(pool, table, refs, rows)
    pool.release(table, _i32(length))
    assert oracle.release(refs, rows, length, None, page)
    _check_pool(pool, table, refs, rows)
    assert int(pool.err.item()) == 0 and bool((wide[:, width:] == -1).all())


@pytest.mark.gpu
def test_pages_that_nobody_holds_and_entries_outside_the_pool():
    from chain_flow_b200.kv_cache import PagePool
    refs, rows = [1, 0, 2, 1], [[0, 0, -1], [2, 4, 1 << 30], [2, 3, 2]]
    pool, table = PagePool.from_refs(_i32(refs), 4), _i32(rows)
    assert pool.fork(table, _i32([12, 12, 0]), _i32([1]), _i32([2])).tolist() == [1]     # entries outside the pool are shared as they are
    oracle.fork(refs, rows, [12, 12, 0], [1], [2], 4)
    _check_pool(pool, table, refs, rows)
    pool.release(table, _i32([12, 12, 100]))
    assert not oracle.release(refs, rows, [12, 12, 100], None, 4)                           # page 0 twice
    _check_pool(pool, table, refs, rows)
    assert int(pool.err.item()) != 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, FP8])
@pytest.mark.parametrize("layers, page, heads, dim", [(0, 16, 1, 64), (1, 16, 4, 256), (8, 48, 8, 128), (37, 17, 1, 64)])
def test_forks_copy_their_last_page(dtype, layers, page, heads, dim):
    from chain_flow_b200.kv_cache import PagePool
    lens, kids = [5 * page + 3, 2 * page, 1, 0, 3 * page - 1], [3, 2, 1, 2, 1]
    parent = [p for p, n in enumerate(kids) for _ in range(n)]
    child = list(range(len(lens), len(lens) + len(parent)))
    pages, width, total = 40, 6, len(lens) + len(parent)
    caches = _caches(layers, pages, page, heads, dim, dtype)
    pool = PagePool(pages, page)
    table = torch.full((total, width), -1, dtype=torch.int32, device="cuda")
    length = _i32([0] * total)
    target = lens + [0] * len(parent)
    assert pool.reserve(table, length, _i32(target)).tolist() == [1] * total
    length.copy_(_i32(target))
    refs, rows, pools = pool.refs.tolist(), table.tolist(), _pools(caches)
    for _ in range(2):                                   # and again once the children have ended
        got = pool.fork(table, length, _i32(parent), _i32(child), caches)
        granted, copies = oracle.fork(refs, rows, target, parent, child, page)
        for a, b, n in copies:
            oracle.copy_pages(pools, [a], [b], [n])
        assert got.tolist() == granted == [1] * len(parent) and length.tolist() == target
        _check_pool(pool, table, refs, rows)
        _same(caches, pools)
        ended = [n if b >= len(lens) else 0 for b, n in enumerate(target)]
        pool.release(table, _i32(ended))
        oracle.release(refs, rows, ended, None, page)
        _check_pool(pool, table, refs, rows)
    assert refs == [int(p < sum(-(-n // page) for n in lens)) for p in range(pages)]


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows and pages that lie more than 2^32 elements apart."""
    from chain_flow_b200.kv_cache import PagedKVCache, copy_pages, keep_path
    page, heads, dim = 16, 8, 256
    pages = (1 << 32) // (page * heads * dim) + 2
    if torch.cuda.mem_get_info()[0] < 3 * pages * page * heads * dim:
        pytest.skip("needs 13 GB of device memory")
    k, v = (torch.empty(pages, heads, page, dim, dtype=torch.uint8, device="cuda").view(FP8) for _ in range(2))
    ks, vs = (torch.zeros(pages, heads, page, device="cuda") for _ in range(2))
    c = PagedKVCache.from_tensors(k, v, ks, vs)
    x = torch.randn(page, heads, dim, device="cuda", dtype=torch.float16)
    last = pages - 1
    c.write(x, -x, last * page + torch.arange(page, device="cuda"))
    copy_pages(c, _i32([last, 3]), _i32([2, last - 1]))
    keep_path(c, _i32([[last - 1, last]]), _i32([5]), _i32([[11 + 4, 11 + 9]]), _i32([2]))
    at = lambda p: torch.arange(page, device="cuda") + p * page  # noqa: E731
    a, b = c.read(at(2), torch.float32), c.read(at(last), torch.float32)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    got, want = c.read(at(last - 1)[5:7], torch.float32), c.read(at(last)[[4, 9]], torch.float32)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_streams_and_capture():
    from chain_flow_b200.kv_cache import PagePool, copy_pages, keep_path
    caches = _caches(3, 8, 16, 2, 64, torch.float16)
    table, base, path, length = [[0, 1]], [3], [[2, 5]], [2]
    want = _pools(caches)
    args = _i32(table), _i32(base), _i32(path), _i32(length)
    src, dst = _i32([0]), _i32([6])
    pool, tab, zero, ten = PagePool(8, 16), _i32([[-1, -1, -1]]), _i32([0]), _i32([40])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    keep_path(caches, *args, stream=side)
    copy_pages(caches, src, dst, stream=side)
    got = pool.reserve(tab, zero, ten, stream=side)
    pool.release(tab, ten, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    oracle.keep_path(want, table, base, path, length, 16)
    oracle.copy_pages(want, [0], [6], None)
    _same(caches, want)
    assert got.tolist() == [1] and tab.tolist() == [[-1, -1, -1]] and pool.refs.tolist() == [0] * 8
    graph = torch.cuda.CUDAGraph()
    two, lens = torch.full((2, 3), -1, dtype=torch.int32, device="cuda"), _i32([20, 0])
    start, parent, child = _i32([20, 0]), _i32([0]), _i32([1])
    pool.reserve(two, _i32([0, 0]), lens)
    with torch.cuda.graph(graph):
        keep_path(caches, *args)
        copy_pages(caches, src, dst)
        lens.copy_(start)
        pool.fork(two, lens, parent, child, caches)
        pool.release(two[1:], lens[1:])
    for _ in range(2):
        graph.replay()
        oracle.keep_path(want, table, base, path, length, 16)
        oracle.copy_pages(want, [0], [6], None)
        oracle.copy_pages(want, [1], [2], [4])
        _same(caches, want)
        assert two.tolist() == [[0, 1, -1], [-1, -1, -1]] and pool.refs.tolist() == [1, 1] + [0] * 6 and lens.tolist() == [20, 20]


@pytest.mark.gpu
def test_refusals_in_python(monkeypatch):
    from chain_flow_b200.kv_cache import PagePool, copy_pages, keep_path
    caches = _caches(2, 8, 16, 2, 64, torch.float16)
    other = _caches(1, 8, 16, 2, 128, torch.float16) + _caches(1, 8, 16, 2, 64, torch.float16, "token") + _caches(1, 8, 16, 2, 64, torch.bfloat16)
    t, b, p, n = _i32([[0, 1]]), _i32([3]), _i32([[2, 5]]), _i32([2])
    for o in other:
        with pytest.raises(_lib.CfbError, match="differ"):
            keep_path([caches[0], o], t, b, p, n)
        with pytest.raises(_lib.CfbError, match="differ"):
            copy_pages([caches[0], o], b, n)
    for bad in ((t[0], b, p, n), (t, b[:0], p, n), (t, b, p[0], n), (t, b, p, p), (t.float(), b, p, n), (t.cpu(), b, p, n), (t, b.cpu(), p, n),
                (t, b, p.repeat(2, 1), n), (t, b > 0, p, n)):
        with pytest.raises(_lib.CfbError):
            keep_path(caches, *bad)
    for bad in ((b, p), (b, n[:0]), (b.float(), n), (b.cpu(), n), (b, n, p[0])):
        with pytest.raises(_lib.CfbError):
            copy_pages(caches, *bad)
    pool = PagePool(8, 16)
    for bad in ((t.long(), b, n), (t[0], b, n), (t.cpu(), b, n), (t.expand(2, -1), _i32([0, 0]), _i32([1, 1])),
                (_i32([[0, 1], [2, 3]]).t(), _i32([0, 0]), _i32([1, 1])), (t, p[0], n), (t, b, b.float())):
        for call in (pool.reserve, pool.release):
            with pytest.raises(_lib.CfbError):
                call(*bad)
    two, lens = _i32([[0, 1], [2, 3]]), _i32([1, 0])
    for bad in ((two, lens.long(), b, n), (two, lens[:1], b, n), (two, lens, p, n), (two, lens, b, p[0]), (two, lens, b.cpu(), n),
                (two, torch.zeros(2, 2, dtype=torch.int32, device="cuda")[:, 0], b, n)):
        with pytest.raises(_lib.CfbError):
            pool.fork(*bad)
    with pytest.raises(_lib.CfbError, match="other pages"):
        PagePool(9, 16).fork(two, lens, b, n, caches)
    with pytest.raises(_lib.CfbError, match="other pages"):
        PagePool(8, 17).fork(two, lens, b, n, caches[0])
    with pytest.raises(_lib.CfbError, match="differ"):
        pool.fork(two, lens, b, n, [caches[0], other[0]])
    for bad in ((0, 16), (8, 0), ((1 << 20) + 1, 16)):
        with pytest.raises(_lib.CfbError):
            PagePool(*bad)
    for refs in (two, lens.long(), lens.cpu(), two[:, 0]):
        with pytest.raises(_lib.CfbError):
            PagePool.from_refs(refs, 16)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    for call in (lambda: keep_path(caches, t, b, p, n), lambda: copy_pages(caches, b, n), lambda: pool.reserve(t, b, n),
                 lambda: pool.release(t, b), lambda: pool.fork(two, lens, b, n, caches)):
        with pytest.raises(_lib.CfbError, match="current device"):
            call()
