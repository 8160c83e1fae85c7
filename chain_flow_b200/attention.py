"""Attention of a step's new tokens over a paged key/value cache, with its log-sum-exp, on
cfb_paged_attn (cfb_attn.cu): prompt chunks and single tokens (causal), and the prefix half of a
tree step, whose outputs ``tree.tree_attn_merge`` joins with the tree's own part."""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .kv_cache import HEAD_DIMS, PagedKVCache

_DT = {torch.float16: 1, torch.bfloat16: 2}


class PagedAttention:
    """Owns the workspace of calls with ``heads`` query heads over ``kv_heads`` kv heads of
    ``head_dim``; a call allocates only outputs it is not given. Calls share the workspace: order
    them on one stream."""

    def __init__(self, heads: int, kv_heads: int, head_dim: int, device=None):
        self.lib = _lib.load()
        if heads <= 0 or kv_heads <= 0 or heads % kv_heads or heads // kv_heads > 128 or head_dim not in HEAD_DIMS:
            raise _lib.CfbError(f"PagedAttention: heads must be a multiple (up to 128) of kv_heads and head_dim one of "
                                f"{HEAD_DIMS}, got {heads} / {kv_heads} / {head_dim}")
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.heads, self.kv_heads, self.head_dim, self.scale = heads, kv_heads, head_dim, head_dim ** -0.5
        self.ws_bytes = int(self.lib.cfb_paged_attn_workspace(heads, kv_heads, head_dim))
        self.ws = torch.empty(self.ws_bytes + 256, dtype=torch.uint8, device=self.device)
        self.ws_ptr = (self.ws.data_ptr() + 255) // 256 * 256
        self._dev, self._ran = self.ws.get_device(), False

    def _refuse(self, query, cache, page_table, kv_len, cu_q):
        for t, n in ((query, "query"), (page_table, "page_table"), (kv_len, "kv_len"), (cu_q, "cu_q")):
            _lib.require_cuda(t, n)
            if t.device != cache.device:
                raise _lib.CfbError(f"{n} is on {t.device}, the cache on {cache.device}")
        if query.dim() != 3 or query.shape[1] != self.heads or query.shape[2] != self.head_dim or query.stride(2) != 1:
            raise _lib.CfbError(f"query: expected [T, {self.heads}, {self.head_dim}] with a contiguous head dim, got {list(query.shape)}")
        if cache._dev != self._dev:
            raise _lib.CfbError(f"PagedAttention: the cache is on {cache.device}, this object's workspace on {self.device}")
        if cache.kv_heads != self.kv_heads or cache.head_dim != self.head_dim:
            raise _lib.CfbError("PagedAttention: the cache has other kv heads or another head dim")
        if query.dtype not in _DT or (cache.k_scale is None and query.dtype != cache.dtype):
            raise _lib.CfbError("PagedAttention: query must be fp16 or bf16, the cache's own dtype unless it is e4m3")
        raise _lib.CfbError("PagedAttention: page_table [B, width], kv_len [B] and cu_q [B + 1] disagree")

    def check(self) -> None:
        """Raises if a device-side wait of the last call with rows and requests expired (its outputs are then invalid;
        without such a call there is nothing to raise). Waits for the GPU."""
        err = C.c_int(0)
        torch.cuda.synchronize(self.device)
        if not self._ran:                                # the error words are the kernel's to write
            return
        _lib.check(self.lib.cfb_paged_attn_error(self.ws_ptr, C.byref(err)), "cfb_paged_attn_error")
        if err.value:
            raise _lib.CfbError(f"PagedAttention: device error {err.value} (a bounded wait expired); outputs are invalid")

    def __call__(self, query, cache: PagedKVCache, page_table, kv_len, cu_q, *, scale: float | None = None,
                 causal: bool = True, out=None, lse=None, stream=None):
        """(out [T, heads, head_dim], lse fp32 [heads, T], natural log). Request b owns the query rows
        [cu_q[b], cu_q[b + 1]) and the first kv_len[b] positions of the pages page_table[b]; with
        ``causal`` its new tokens are the last of those positions and see up to themselves, without
        it they see all of them. Rows that see nothing get 0 and -inf. query fp16 or bf16 (the
        cache's dtype, or either over an e4m3 cache), page_table int32 [B, width], kv_len int32 [B],
        cu_q int32 [B + 1], all on the GPU: nothing is read back. scale defaults to
        head_dim ** -0.5. Rows outside every request are left as they are (given buffers) or
        undefined (new ones)."""
        if stream is not None:
            with torch.cuda.stream(stream):
                return self(query, cache, page_table, kv_len, cu_q, scale=scale, causal=causal, out=out, lse=lse)
        B, shape, dev, dtype = kv_len.shape[0] if kv_len.dim() else -1, query.shape, cache._dev, query.dtype
        dt, sq = _DT.get(dtype), query.stride()
        if (len(shape) != 3 or shape[1] != self.heads or shape[2] != self.head_dim or sq[2] != 1 or dt is None
                or (cache.k_scale is None and dtype != cache.dtype)
                or cache.kv_heads != self.kv_heads or cache.head_dim != self.head_dim or dev != self._dev
                or page_table.dim() != 2 or page_table.shape[0] != B or kv_len.dim() != 1 or cu_q.shape != (B + 1,)
                or any(t.get_device() != dev for t in (query, page_table, kv_len, cu_q))):
            self._refuse(query, cache, page_table, kv_len, cu_q)
        st, width = page_table.stride(), page_table.shape[1]
        # (rows that share words, as one prefix expanded over several requests, are copied out)
        if page_table.dtype != torch.int32 or st[1] != 1 or (B > 1 and st[0] < width):
            page_table = page_table.to(torch.int32).contiguous()
            st = page_table.stride()
        kv_len, cu_q = _lib.int32(kv_len), _lib.int32(cu_q)
        T = shape[0]
        if out is None:
            out = torch.empty(shape, dtype=dtype, device=cache.device)
        elif out.shape != shape or out.dtype != dtype or out.get_device() != dev or out.stride(2) != 1:
            raise _lib.CfbError("out must have the query's shape, dtype and device, and a contiguous head dim")
        if lse is None:
            lse = torch.empty((self.heads, T), dtype=torch.float32, device=cache.device)
        elif lse.shape != (self.heads, T) or lse.dtype != torch.float32 or lse.get_device() != dev or not lse.is_contiguous():
            raise _lib.CfbError(f"lse must be contiguous fp32 [{self.heads}, {T}] on the query's device")
        so = out.stride()
        if T == 1:                                       # one token's stride can be any number, as 1 of a transposed column
            sq, so = (0, sq[1]), (0, so[1])
        _lib.check(self.lib.cfb_paged_attn(
            query.data_ptr(), sq[0], sq[1], cache.desc, page_table.data_ptr(), max(st[0], width),
            width, kv_len.data_ptr(), cu_q.data_ptr(), out.data_ptr(), so[0], so[1], lse.data_ptr(),
            self.scale if scale is None else scale, T, B, self.heads, causal, dt, self.ws_ptr, self.ws_bytes,
            _lib.stream_of(dev, "PagedAttention")), "cfb_paged_attn")
        if T and B:
            self._ran = True
        return out, lse
