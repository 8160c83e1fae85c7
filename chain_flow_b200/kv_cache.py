"""The paged key/value cache of a target's full-attention layer, on the sm_100a kernels of
libcfb.so (cfb_kv.cu): rows are written to slots of pages, quantised as they are written where the
cache holds e4m3, and read back. ``attention.PagedAttention`` attends over it."""
from __future__ import annotations

import ctypes as C

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
