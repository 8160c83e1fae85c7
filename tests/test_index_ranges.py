"""Integers of 64 bits that 32 do not hold are outside every range (of tokens, pages, positions); they do not wrap into it."""
import pytest
import torch

from test_cache_pages import _caches, _i32, _pools, _same

FAR = [1 << 32, -1 << 32, 1 << 40]


def _i64(x):
    return torch.tensor(x, dtype=torch.int64, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("far", FAR)
def test_tokens_and_parents(far):
    from chain_flow_b200.tree import RejectionVerifier, SampledVerifier
    V, tok = 100, 42
    logits = torch.full((2, V), -float("inf"), device="cuda")
    logits[:, tok] = 0.0
    one, u = torch.ones(1, dtype=torch.int64, device="cuda"), torch.full((2,), 0.5, device="cuda")
    ver = SampledVerifier(2, 1, 1)
    for t, p, want in ((tok, -1, 1), (tok + far, -1, 0), (tok, far - 1, 0)):
        assert ver(logits, one, 2 * one, _i64([t]), _i64([p]), u)[2].tolist() == [want]
    q = torch.full((1, V), 0.01, device="cuda")
    rej = RejectionVerifier(2, 1, 1, V)
    for t, want in ((tok, 1), (tok + far, 0)):
        assert rej(logits, one, 2 * one, _i64([t]), q, u[:1], u[:1])[1].tolist() == [want]
    for at in (ver, rej):                                # offsets far outside: nothing is emitted
        args = (_i64([tok]), _i64([-1]), u) if at is ver else (_i64([tok]), q, u[:1], u[:1])
        assert at(logits, one, 2 * one + far, *args)[0].tolist() == [[-1, -1]] and int(at.err.item()) == 7


@pytest.mark.gpu
@pytest.mark.parametrize("far", FAR)
def test_pages_and_positions(far):
    from chain_flow_b200.kv_cache import PagePool, copy_pages, keep_path
    caches = _caches(2, 6, 16, 2, 64, torch.float16)
    want = _pools(caches)
    keep_path(caches, _i64([[far, 1]]), _i64([0]), _i64([[3, 5]]), _i64([2]))
    keep_path(caches, _i64([[0, 1]]), _i64([far]), _i64([[3, 5]]), _i64([2]))
    keep_path(caches, _i64([[0, 1]]), _i64([0]), _i64([[far + 3, far + 5]]), _i64([2]))
    keep_path(caches, _i64([[0, 1]]), _i64([0]), _i64([[3, 5]]), _i64([2 - abs(far)]))
    copy_pages(caches, _i64([far]), _i64([3]))
    copy_pages(caches, _i64([0]), _i64([far + 3]))
    _same(caches, want)
    pool, table = PagePool(6, 16), torch.full((1, 3), -1, dtype=torch.int32, device="cuda")
    if far > 0:
        assert pool.reserve(table, _i64([0]), _i64([far + 5])).tolist() == [0]
        assert pool.reserve(table, _i64([far]), _i64([5])).tolist() == [1]          # it holds more than it asks for
    else:
        assert pool.reserve(table, _i64([0]), _i64([far + 5])).tolist() == [1]      # nothing is asked for
    assert pool.refs.tolist() == [0] * 6 and table.tolist() == [[-1] * 3]
    lens = _i32([0])
    assert pool.fork(table, lens, _i64([far]), _i64([0])).tolist() == [0] and pool.fork(table, lens, _i64([0]), _i64([far])).tolist() == [0]


@pytest.mark.gpu
def test_other_integer_types_are_taken():
    from chain_flow_b200.kv_cache import PagePool
    pool, table = PagePool(6, 16), torch.full((2, 3), -1, dtype=torch.int32, device="cuda")
    for dt in (torch.int8, torch.uint8, torch.int16, torch.int64):
        assert pool.reserve(table, _i32([0, 0]).to(dt), _i32([17, 3]).to(dt)).tolist() == [1, 1]
        assert table.tolist() == [[0, 1, -1], [2, -1, -1]]
        pool.release(table, _i32([17, 3]).to(dt))


def test_a_cache_given_twice():
    """Its rows would be moved twice at once."""
    from chain_flow_b200 import _lib
    from test_cache_pages import FAKE, _array, _cache
    lib = _lib.load()
    a, b, c = _cache(), _cache(k=FAKE + 16 * 4096, v=FAKE + 16 * 4096), _cache(k=FAKE + 32 * 4096)
    call = lambda *x: lib.cfb_kv_keep(_array(*x), len(x), FAKE, 4, 4, FAKE, FAKE, 5, FAKE, 5, 0, None)  # noqa: E731
    assert call(a) == 0 and call(a, b) == 0 and call(a, a) == 1 and call(a, b, a) == 1 and call(a, b, c) == 1      # (c: a's values)


@pytest.mark.gpu
def test_a_cache_given_twice_in_python():
    from chain_flow_b200 import _lib
    from chain_flow_b200.kv_cache import copy_pages, keep_path
    caches = _caches(2, 6, 16, 2, 64, torch.float16)
    want = _pools(caches)
    for twice in (caches + caches[:1], [caches[1]] * 2):
        with pytest.raises(_lib.CfbError, match="twice"):
            keep_path(twice, _i32([[0, 1]]), _i32([0]), _i32([[3, 5]]), _i32([2]))
    _same(caches, want)
    copy_pages(caches + caches[:1], _i32([0]), _i32([4]))                          # the same bytes twice
    for t in want:
        t[4] = t[0]
    _same(caches, want)
