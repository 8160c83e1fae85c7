"""The paged key/value cache of a target's full-attention layer, on the sm_100a kernels of
libcfb.so (cfb_kv.cu, cfb_pages.cu): rows are written to slots of pages, quantised as they are written
where the cache holds e4m3, and read back. ``attention.PagedAttention`` attends over it. Over the caches of
all layers at once, ``keep_path`` moves a step's accepted rows together and ``copy_pages`` copies pages;
``PagePool`` counts who holds a page: it hands pages out, takes them back and forks a request's."""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import _lib

_DT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.float8_e4m3fn: 3}
HEAD_DIMS = (64, 128, 256)


class PagedKVCache:
    """Keys and values of one layer in ``pages`` pages of ``page_size`` slots. A token's flat slot is
    ``page * page_size + offset``. ``dtype``: fp16 or bf16 (rows are kept as they are), or
    ``torch.float8_e4m3fn`` (each row x of a token and kv head as codes and one fp32 scale
    ``max(max|x|, 2**-24) / 448``; a row with a NaN or an infinity reads back as NaN). A slot that was never
    written holds zeros.

    Buffers: ``k``, ``v`` [pages, kv_heads, page_size, head_dim], so that a head's rows of a page
    are contiguous; ``k_scale``, ``v_scale`` fp32 [pages, kv_heads, page_size] (e4m3 only).
    ``from_tensors`` takes a caller's own buffers, in this order of dims with any strides."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.float16, device=None):
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        if dtype not in _DT or dtype == torch.float32:
            raise _lib.CfbError("PagedKVCache: dtype must be fp16, bf16 or float8_e4m3fn")
        shape = (pages, kv_heads, page_size, head_dim)
        k, v = (torch.zeros(shape, dtype=dtype, device=dev) for _ in range(2))
        scales = (None, None)
        if dtype == torch.float8_e4m3fn:
            scales = tuple(torch.zeros(shape[:3], dtype=torch.float32, device=dev) for _ in range(2))
        self._bind(k, v, *scales)

    @classmethod
    def from_tensors(cls, k, v, k_scale=None, v_scale=None) -> "PagedKVCache":
        """A cache over existing buffers [pages, kv_heads, page_size, head_dim] (permuted views of
        another layout are fine; k and v share strides, and so do their scales). Scales are not negative; a row of
        scale 0 stands for zeros."""
        self = cls.__new__(cls)
        self._bind(k, v, k_scale, v_scale)
        return self

    def _bind(self, k, v, k_scale, v_scale) -> None:
        self.lib = _lib.load()
        for t, n in ((k, "k"), (v, "v")):
            _lib.require_cuda(t, n)
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.stride() != v.stride() or k.device != v.device:
            raise _lib.CfbError("PagedKVCache: k and v must be 4-D with one shape, dtype, device and strides")
        if k.dtype not in _DT or k.dtype == torch.float32:
            raise _lib.CfbError("PagedKVCache: dtype must be fp16, bf16 or float8_e4m3fn")
        if k.stride(3) != 1:
            raise _lib.CfbError("PagedKVCache: k and v need a contiguous head dim")
        if k.shape[3] not in HEAD_DIMS:
            raise _lib.CfbError(f"PagedKVCache: head_dim must be one of {HEAD_DIMS}, got {k.shape[3]}")
        if min(k.shape) <= 0:
            raise _lib.CfbError("PagedKVCache: pages, kv_heads and page_size must be positive")
        size = k.element_size()
        if any(t.data_ptr() % 16 for t in (k, v)) or any(st * size % 16 for st in k.stride()[:3]):
            raise _lib.CfbError("PagedKVCache: every row must start on a 16-byte boundary")
        quant = k.dtype == torch.float8_e4m3fn
        if quant != (k_scale is not None) or quant != (v_scale is not None):
            raise _lib.CfbError("PagedKVCache: an e4m3 cache has k_scale and v_scale, a 16-bit one has neither")
        if quant:
            for t, n in ((k_scale, "k_scale"), (v_scale, "v_scale")):
                _lib.require_cuda(t, n)
                if t.dtype != torch.float32 or t.shape != k.shape[:3] or t.stride() != k_scale.stride() or t.device != k.device:
                    raise _lib.CfbError("PagedKVCache: scales must be fp32 [pages, kv_heads, page_size] with one set of strides")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.dtype, self.device, self._dev = k.dtype, k.device, k.get_device()
        ss = k_scale.stride() if quant else (0, 0, 0)
        self._desc = _lib.KvCache(
            k.data_ptr(), v.data_ptr(), k_scale.data_ptr() if quant else None, v_scale.data_ptr() if quant else None,
            k.stride(0), k.stride(1), k.stride(2), *ss, self.pages, self.page_size, self.kv_heads, self.head_dim,
            _DT[k.dtype])
        self.desc = C.byref(self._desc)
        self._at = C.addressof(self._desc)

    def _slots(self, slots):
        if slots.dim() != 1 or slots.is_floating_point() or slots.get_device() != self._dev:
            _lib.require_cuda(slots, "slots")
            raise _lib.CfbError("slots must be a 1-D integer tensor on the cache's device")
        return slots if slots.dtype == torch.int64 and slots.is_contiguous() else slots.to(torch.int64).contiguous()

    def _refuse_rows(self, t, name: str, tokens: int):
        _lib.require_cuda(t, name)
        if t.get_device() != self._dev:
            raise _lib.CfbError(f"{name} is on {t.device}, the cache on {self.device}")
        if tuple(t.shape) != (tokens, self.kv_heads, self.head_dim):
            raise _lib.CfbError(f"{name}: expected [{tokens}, {self.kv_heads}, {self.head_dim}], got {list(t.shape)}")
        raise _lib.CfbError(f"{name} needs a contiguous head dim")

    def write(self, key, value, slots, stream=None) -> None:
        """Rows key, value [T, kv_heads, head_dim] (fp16 or bf16; a 16-bit cache takes its own dtype)
        to the flat slots [T]. A negative slot, or one past the pool, skips its token. The slots
        of a call must be distinct."""
        if stream is not None:
            with torch.cuda.stream(stream):
                return self.write(key, value, slots)
        slots = self._slots(slots)
        T = slots.shape[0]
        shape, sk, sv = (T, self.kv_heads, self.head_dim), key.stride(), value.stride()
        for t, n, st in ((key, "key", sk), (value, "value", sv)):
            if t.shape != shape or st[2] != 1 or t.get_device() != self._dev:
                self._refuse_rows(t, n, T)
        if T == 1:                                       # one token's stride can be any number, as 1 of a transposed column
            sk, sv = (0, sk[1]), (0, sv[1])
        dtype = key.dtype
        dt = _DT.get(dtype)
        if dt not in (1, 2) or value.dtype != dtype or (self.k_scale is None and dtype != self.dtype):
            raise _lib.CfbError("PagedKVCache.write: key and value must share fp16 or bf16, the cache's own unless it is e4m3")
        _lib.check(self.lib.cfb_kv_write(self.desc, key.data_ptr(), sk[0], sk[1], value.data_ptr(), sv[0], sv[1], dt,
                                         slots.data_ptr(), T, _lib.stream_of(self._dev, "PagedKVCache.write")), "cfb_kv_write")

    def read(self, slots, dtype=None, stream=None):
        """(key, value) [T, kv_heads, head_dim] of the flat slots [T] in fp32, fp16 or bf16 (default:
        the cache's own 16-bit dtype, fp16 for e4m3). A slot outside the pool reads as 0."""
        if stream is not None:
            with torch.cuda.stream(stream):
                return self.read(slots, dtype)
        slots = self._slots(slots)
        if dtype is None:
            dtype = self.dtype if self.k_scale is None else torch.float16
        if _DT.get(dtype) not in (0, 1, 2):
            raise _lib.CfbError("PagedKVCache.read: dtype must be fp32, fp16 or bf16")
        T, D = slots.shape[0], self.head_dim
        key, value = torch.empty(2, T, self.kv_heads, D, dtype=dtype, device=self.device).unbind(0)
        _lib.check(self.lib.cfb_kv_read(self.desc, slots.data_ptr(), T, key.data_ptr(), self.kv_heads * D, D, value.data_ptr(),
                                        self.kv_heads * D, D, _DT[dtype], _lib.stream_of(self._dev, "PagedKVCache.read")), "cfb_kv_read")
        return key, value


def _layers(caches, what: str, device=None):
    """(packed descriptor addresses, number, device number) of one cache or a sequence of caches of one geometry."""
    if isinstance(caches, PagedKVCache):
        caches = (caches,)
    n = len(caches)
    dev = caches[0]._dev if n else device
    for c in caches:
        if c._dev != dev:
            raise _lib.CfbError(f"{what}: the caches are on several devices")
    if device is not None and dev != device:
        raise _lib.CfbError(f"{what}: the caches are on cuda:{dev}, the pages on cuda:{device}")
    return struct.pack("%dP" % n, *[c._at for c in caches]), n, dev


def _check_layers(caches, what: str) -> None:
    caches = (caches,) if isinstance(caches, PagedKVCache) else caches
    first = caches[0]
    for c in caches[1:]:
        if (c.k.shape != first.k.shape or c.dtype != first.dtype or c.k.stride() != first.k.stride()
                or (c.k_scale is not None and c.k_scale.stride() != first.k_scale.stride())):
            raise _lib.CfbError(f"{what}: the caches differ in shape, dtype or strides")


def _index(t, name: str, what: str, dev: int, shape):
    """t, an integer tensor of `shape` on device dev, as contiguous int32."""
    if t.dtype is torch.int32 and t.shape == shape and t.get_device() == dev and t.is_contiguous():
        return t
    if t.get_device() != dev or t.is_floating_point() or t.dtype == torch.bool or tuple(t.shape) != tuple(shape):
        _lib.require_cuda(t, name)
        raise _lib.CfbError(f"{what}: {name} must be integers {list(shape)} on cuda:{dev}, got {t.dtype} {list(t.shape)} on {t.device}")
    return _lib.int32_indices(t)


def keep_path(caches, page_table, base, path, length, stream=None) -> None:
    """A step's accepted rows moved together, in the caches of all layers (one PagedKVCache or a sequence of one geometry).
    Request b's tree was written to the positions ``base[b] + node``; its rows ``base[b] + path[b, j]``, j < length[b], go
    to ``base[b] + j``. ``path`` [B, S] and ``length`` [B] are a verifier's accepted_path and accepted_len (increasing
    nodes; S <= 1024), page_table [B, width]: integer tensors on the GPU, nothing is read back. Nodes below 0 and
    positions outside the table or the pool are left out. What lies behind the kept rows is stale: the context ends at
    ``base + length``."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return keep_path(caches, page_table, base, path, length)
    desc, n, dev = _layers(caches, "keep_path")
    if n == 0:
        return
    if page_table.dim() != 2 or path.dim() != 2:
        raise _lib.CfbError("keep_path: page_table [B, width] and path [B, S] must be matrices")
    (B, width), S = page_table.shape, path.shape[1]
    page_table = _index(page_table, "page_table", "keep_path", dev, (B, width))
    base, path = _index(base, "base", "keep_path", dev, (B,)), _index(path, "path", "keep_path", dev, (B, S))
    length = _index(length, "length", "keep_path", dev, (B,))
    status = _lib.load().cfb_kv_keep(desc, n, page_table.data_ptr(), width, width, base.data_ptr(), path.data_ptr(), S,
                                     length.data_ptr(), S, B, _lib.stream_of(dev, "keep_path"))
    if status:
        _check_layers(caches, "keep_path")
        if n > 1 and any(len({t.data_ptr() for t in ts}) < n for ts in ([c.k for c in caches], [c.v for c in caches])):
            raise _lib.CfbError("keep_path: a cache is given twice")
        _lib.check(status, "cfb_kv_keep")


def copy_pages(caches, src, dst, slots=None, stream=None) -> None:
    """Pages src [n] of every cache (one PagedKVCache or a sequence of one geometry) copied to pages dst [n]; with ``slots``
    [n], the first slots[i] slots of them. Pairs with a page outside the pool are left out. The dst of a call are
    distinct, and none of them is a src."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return copy_pages(caches, src, dst, slots)
    desc, n, dev = _layers(caches, "copy_pages")
    if n == 0:
        return
    pairs = src.shape[0] if src.dim() == 1 else -1
    src, dst = _index(src, "src", "copy_pages", dev, (pairs,)), _index(dst, "dst", "copy_pages", dev, (pairs,))
    slots = None if slots is None else _index(slots, "slots", "copy_pages", dev, (pairs,))
    status = _lib.load().cfb_kv_copy_pages(desc, n, src.data_ptr(), dst.data_ptr(), None if slots is None else slots.data_ptr(),
                                           pairs, _lib.stream_of(dev, "copy_pages"))
    if status:
        _check_layers(caches, "copy_pages")
        _lib.check(status, "cfb_kv_copy_pages")


class PagePool:
    """Who holds the pages of a target's caches: ``refs`` int32 [pages] counts the requests that hold a page (0: free).
    Requests' pages are rows of a page table (int32 [rows, width], as PagedAttention takes it; changed in place), in order
    of their positions. Every call is a launch or two on the current stream (or ``stream=``) and reads nothing back;
    calls on a pool are ordered on one stream. Pages handed out are always the lowest free ones, request after request.
    ``err`` int32 [1] becomes non-zero when a page is given back that nobody holds."""

    def __init__(self, pages: int, page_size: int, device=None):
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        if pages <= 0:
            raise _lib.CfbError("PagePool: pages must be positive")
        self._bind(torch.zeros(pages, dtype=torch.int32, device=dev), page_size)

    @classmethod
    def from_refs(cls, refs, page_size: int) -> "PagePool":
        """A pool over existing counts (int32 [pages], contiguous, on the GPU)."""
        self = cls.__new__(cls)
        self._bind(refs, page_size)
        return self

    def _bind(self, refs, page_size: int) -> None:
        _lib.require_cuda(refs, "refs")
        if refs.dim() != 1 or refs.dtype != torch.int32 or not refs.is_contiguous() or not 0 < refs.shape[0] <= 1 << 20:
            raise _lib.CfbError("PagePool: refs must be contiguous int32 [pages], 1 to 2^20 pages")
        if page_size <= 0:
            raise _lib.CfbError("PagePool: page_size must be positive")
        self.lib = _lib.load()
        self.refs, self.page_size, self.pages, self._dev = refs, page_size, refs.shape[0], refs.get_device()
        self.err = torch.zeros(1, dtype=torch.int32, device=refs.device)

    def _table(self, table, what: str):
        """(address, row stride, width, rows) of a table that is changed in place."""
        shape, st = table.shape, table.stride()
        if (len(shape) != 2 or table.dtype is not torch.int32 or table.get_device() != self._dev
                or (shape[1] > 1 and st[1] != 1) or (shape[0] > 1 and st[0] < shape[1])):
            _lib.require_cuda(table, "table")
            raise _lib.CfbError(f"{what}: table must be int32 [rows, width] on the pool's device, its rows contiguous and apart")
        return table.data_ptr(), max(st[0], shape[1]), shape[1], shape[0]

    def reserve(self, table, length, target, stream=None):
        """Pages for the positions [length[b], target[b]) that request b's pages do not cover yet, into its row. Returns
        granted int32 [B]: 0 where the pool ran out (that request and all later ones that ask get nothing) or a row is too
        short."""
        if stream is not None:
            with torch.cuda.stream(stream):
                return self.reserve(table, length, target)
        at, stride, width, B = self._table(table, "PagePool.reserve")
        length = _index(length, "length", "PagePool.reserve", self._dev, (B,))
        target = _index(target, "target", "PagePool.reserve", self._dev, (B,))
        granted = torch.empty(B, dtype=torch.int32, device=self.refs.device)
        _lib.check(self.lib.cfb_pages_reserve(self.refs.data_ptr(), self.pages, self.page_size, at, stride, width,
                                              length.data_ptr(), target.data_ptr(), granted.data_ptr(), B,
                                              _lib.stream_of(self._dev, "PagePool.reserve")), "cfb_pages_reserve")
        return granted

    def release(self, table, length, keep=None, stream=None) -> None:
        """Gives back the pages of request b's positions past keep[b] (all of them without ``keep``) up to length[b]; their
        entries become -1. A page that others hold stays theirs; a kept last page that they hold too stays shared, so a
        request that cuts back into what it shares forks (to a row of its own) before it writes there."""
        if stream is not None:
            with torch.cuda.stream(stream):
                return self.release(table, length, keep)
        at, stride, width, B = self._table(table, "PagePool.release")
        length = _index(length, "length", "PagePool.release", self._dev, (B,))
        keep = None if keep is None else _index(keep, "keep", "PagePool.release", self._dev, (B,))
        _lib.check(self.lib.cfb_pages_release(self.refs.data_ptr(), self.pages, self.page_size, at, stride, width,
                                              length.data_ptr(), None if keep is None else keep.data_ptr(), B,
                                              self.err.data_ptr(), _lib.stream_of(self._dev, "PagePool.release")),
                   "cfb_pages_release")

    def fork(self, table, length, parent, child, caches=(), stream=None):
        """Rows child [n] of the table become copies of rows parent [n]: full pages are shared, the slots of a last page
        that is not full are copied to a page of the child's own in every cache (one PagedKVCache or a sequence of one
        geometry, with this pool's pages). ``length`` int32 [rows], contiguous, is changed in place: length[child] =
        length[parent]. Returns granted int32 [n]: 0 where the pool ran out (that fork and all later ones that need a
        page) or a row is none of the table's. The children are distinct, hold no pages, and none is a parent."""
        if stream is not None:
            with torch.cuda.stream(stream):
                return self.fork(table, length, parent, child, caches)
        at, stride, width, rows = self._table(table, "PagePool.fork")
        if length.shape != (rows,) or length.dtype != torch.int32 or not length.is_contiguous() or length.get_device() != self._dev:
            _lib.require_cuda(length, "length")
            raise _lib.CfbError(f"PagePool.fork: length must be contiguous int32 [{rows}] on the pool's device")
        n = parent.shape[0] if parent.dim() == 1 else -1
        parent = _index(parent, "parent", "PagePool.fork", self._dev, (n,))
        child = _index(child, "child", "PagePool.fork", self._dev, (n,))
        desc, layers, _ = _layers(caches, "PagePool.fork", self._dev)
        granted = torch.empty(n, dtype=torch.int32, device=self.refs.device)
        status = self.lib.cfb_pages_fork(self.refs.data_ptr(), self.pages, self.page_size, at, stride, width, rows,
                                         length.data_ptr(), parent.data_ptr(), child.data_ptr(), granted.data_ptr(), n, desc,
                                         layers, _lib.stream_of(self._dev, "PagePool.fork"))
        if status and layers:
            _check_layers(caches, "PagePool.fork")
            first = caches if isinstance(caches, PagedKVCache) else caches[0]
            if first.page_size != self.page_size or first.pages < self.pages:
                raise _lib.CfbError("PagePool.fork: the caches have other pages than the pool")
        _lib.check(status, "cfb_pages_fork")
        return granted
