"""Tree verification around the draft: the target model's side of a tree step, on the sm_100a
kernels of libcfb.so (cfb_tree.cu).

* ``tree_attn_merge``: the tree-attention fix-up of one full-attention layer (the reference fork's
  ``suffix_merge``, src/chain_flow/patches/vllm-0.25.1-chain-flow-tree.patch:5516-5537; eager form
  ``_tree_suffix_eager`` :529-575 + vLLM's ``merge_attn_states``).
* ``TreeVerifier``: greedy verification of draft trees.
* ``SampledVerifier``, ``RejectionVerifier`` (cfb_verify.cu): drafts verified against the target's
  probabilities at a temperature, from given random numbers; trees (and chains) without draft
  probabilities, chains with them. The reference's fork leaves requests above temperature 0 to the
  engine's own sampler (src/chain_flow/vllm_plugin/tree_sampling.py).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

_DT = {torch.float16: 1, torch.bfloat16: 2}


def tree_attn_merge(query, key, value, output, prefix_out, prefix_lse, idx, not_anc, scale: float,
                    stream=None) -> torch.Tensor:
    """Each tree node attends to its ancestors (``not_anc[s, m, n] == 0``) and the result is merged by
    log-sum-exp with the paged-prefix attention (``prefix_out [S*N, H, D]``, ``prefix_lse [H, S*N]``);
    the merged rows are written into ``output`` at the nodes' query rows ``idx [S, N]``.
    query/output ``[T, H, D]``, key/value ``[T, HKV, D]``, fp16 or bf16. Returns ``output``."""
    lib = _lib.load()
    for t, n in ((query, "query"), (key, "key"), (value, "value"), (output, "output"), (prefix_out, "prefix_out"),
                 (prefix_lse, "prefix_lse"), (idx, "idx"), (not_anc, "not_anc")):
        _lib.require_cuda(t, n)
    dt = _DT.get(query.dtype)
    if dt is None or any(t.dtype != query.dtype for t in (key, value, output, prefix_out)):
        raise _lib.CfbError("tree_attn_merge: query/key/value/output/prefix_out must share fp16 or bf16")
    for t, n in ((query, "query"), (key, "key"), (value, "value"), (output, "output"), (prefix_out, "prefix_out")):
        if t.stride(2) != 1:
            raise _lib.CfbError(f"tree_attn_merge: {n} needs a contiguous head dim")
    S, N = idx.shape
    H, D = query.shape[1], query.shape[2]
    idx = idx.to(torch.int64).contiguous()
    not_anc = not_anc.to(torch.uint8).contiguous()
    prefix_lse = prefix_lse.to(torch.float32).contiguous()
    _lib.check(lib.cfb_tree_attn_merge(
        query.data_ptr(), query.stride(0), query.stride(1), key.data_ptr(), key.stride(0), key.stride(1),
        value.data_ptr(), value.stride(0), value.stride(1), output.data_ptr(), output.stride(0), output.stride(1),
        prefix_out.data_ptr(), prefix_out.stride(0), prefix_out.stride(1), prefix_lse.data_ptr(), idx.data_ptr(),
        not_anc.data_ptr(), float(scale), S, N, H, key.shape[1], D, dt, C.c_void_p(_lib.stream_ptr(stream))),
        "cfb_tree_attn_merge")
    return output


def ancestor_mask(parents: torch.Tensor) -> torch.Tensor:
    """[S, N] parents (-1 = the committed token, parent < child) -> [S, N, N] uint8 not-ancestor mask
    (0 where column n is node m itself or one of its ancestors), on the parents' device."""
    S, N = parents.shape
    anc = torch.eye(N, dtype=torch.bool, device=parents.device).unsqueeze(0).repeat(S, 1, 1)
    p = parents.long()
    for m in range(N):                       # BFS order: a parent's row is complete before its child's
        pm = p[:, m]
        has = pm >= 0
        rows = anc[torch.arange(S, device=parents.device), pm.clamp(min=0)]
        anc[:, m] |= rows & has.unsqueeze(1)
    return (~anc).to(torch.uint8)


class TreeVerifier:
    """Greedy tree verification (the reference fork's tree_rejection_sample,
    vllm-0.25.1-chain-flow-tree.patch:640-723) on cfb_tree_verify_greedy: one launch computes the
    argmax of every logits row and walks each request's draft tree. The workspace and outputs are
    allocated once for up to ``max_rows`` logits rows and ``max_batch`` requests and reused, so a
    call allocates nothing (CUDA-graph capturable)."""

    def __init__(self, max_rows: int, max_batch: int, max_spec_len: int, device=None):
        self.lib = _lib.load()
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.max_rows, self.max_batch, self.max_spec = max_rows, max_batch, max_spec_len
        nbytes = int(self.lib.cfb_tree_verify_workspace(max_rows, max_batch))
        self.ws = torch.zeros(nbytes + 256, dtype=torch.uint8, device=dev)
        self.ws_ptr = (self.ws.data_ptr() + 255) // 256 * 256
        self.ws_bytes = nbytes
        self.out_tokens = torch.empty(max_batch, max_spec_len + 1, dtype=torch.int32, device=dev)
        self.accepted_path = torch.empty(max_batch, max_spec_len, dtype=torch.int32, device=dev)
        self.accepted_len = torch.empty(max_batch, dtype=torch.int32, device=dev)
        self.row_argmax = torch.empty(max_rows, dtype=torch.int32, device=dev)
        self.err = torch.zeros(1, dtype=torch.int32, device=dev)

    def __call__(self, logits, cu_num_draft, cu_num_sampled, draft_tokens, parents, stream=None):
        """(output_tokens [B, max_spec + 1], accepted_path [B, max_spec], accepted_len [B]) int32
        views of this verifier's buffers, for B = len(cu_num_draft) requests."""
        for t, n in ((logits, "logits"), (cu_num_draft, "cu_num_draft"), (cu_num_sampled, "cu_num_sampled"),
                     (draft_tokens, "draft_tokens"), (parents, "parents")):
            _lib.require_cuda(t, n)
        dt = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}.get(logits.dtype)
        if dt is None or logits.stride(1) != 1:
            raise _lib.CfbError("logits: fp32 / fp16 / bf16 rows with a contiguous vocabulary dim")
        rows, V = logits.shape
        B = cu_num_draft.numel()
        if rows > self.max_rows or B > self.max_batch:
            raise _lib.CfbError(f"{rows} rows / {B} requests exceed this verifier ({self.max_rows} / {self.max_batch})")
        i32 = lambda t: t.to(torch.int32).contiguous()
        cu_d, cu_s, dtok, par = i32(cu_num_draft), i32(cu_num_sampled), i32(draft_tokens), i32(parents)
        _lib.check(self.lib.cfb_tree_verify_greedy(
            logits.data_ptr(), logits.stride(0), rows, V, dt, cu_d.data_ptr(), cu_s.data_ptr(), dtok.data_ptr(),
            par.data_ptr(), B, self.max_spec, self.out_tokens.data_ptr(), self.accepted_path.data_ptr(),
            self.accepted_len.data_ptr(), self.row_argmax.data_ptr(), C.c_void_p(self.ws_ptr), self.ws_bytes,
            self.err.data_ptr(), C.c_void_p(_lib.stream_ptr(stream))), "cfb_tree_verify_greedy")
        return self.out_tokens[:B], self.accepted_path[:B], self.accepted_len[:B]


class _ProbabilityVerifier:
    """What SampledVerifier and RejectionVerifier share: their buffers, allocated once for up to ``max_rows`` logits rows
    and ``max_batch`` requests and reused, so a call allocates nothing (CUDA-graph capturable) and calls of one verifier
    are ordered on one stream. ``err`` int32 [1] becomes non-zero when a request's offsets do not fit its rows."""

    def __init__(self, max_rows: int, max_batch: int, max_spec_len: int, device=None):
        self.lib = _lib.load()
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        if max_rows <= 0 or max_batch <= 0 or not 0 <= max_spec_len <= 1024:
            raise _lib.CfbError(f"{type(self).__name__}: max_rows and max_batch must be positive, max_spec_len 0 to 1024")
        self.max_rows, self.max_batch, self.max_spec = max_rows, max_batch, max_spec_len
        self.ws_bytes = int(self.lib.cfb_verify_workspace(max_rows, max_batch))
        self.ws = torch.zeros(self.ws_bytes + 256, dtype=torch.uint8, device=dev)
        self.ws_ptr = (self.ws.data_ptr() + 255) // 256 * 256
        self._dev = self.ws.get_device()
        self.out_tokens = torch.empty(max_batch, max_spec_len + 1, dtype=torch.int32, device=dev)
        self.accepted_len = torch.empty(max_batch, dtype=torch.int32, device=dev)
        self.logprobs = torch.empty(max_batch, max_spec_len + 1, dtype=torch.float32, device=dev)
        self.err = torch.zeros(1, dtype=torch.int32, device=dev)
        self._views = {}                                 # of the buffers, by the number of requests: a slice takes a microsecond

    def _outputs(self, B):
        views = self._views.get(B)
        if views is None:
            views = self._views[B] = tuple(t[:B] for t in self._buffers())
        return views

    def _refuse(self, what, wrong):
        raise _lib.CfbError(f"{type(self).__name__}: {what} {wrong}")

    def _ints(self, t, name, shape):
        if t.dtype is torch.int32 and t.shape == shape and t.get_device() == self._dev and t.is_contiguous():
            return t
        if t.get_device() != self._dev or t.is_floating_point() or t.dtype == torch.bool or tuple(t.shape) != shape:
            _lib.require_cuda(t, name)
            self._refuse(name, f"must be integers {list(shape)} on cuda:{self._dev}, got {t.dtype} {list(t.shape)} on {t.device}")
        return _lib.int32_indices(t)

    def _numbers(self, t, name, n):
        if t.get_device() != self._dev or t.dtype not in (torch.float32, torch.float64) or t.shape != (n,):
            _lib.require_cuda(t, name)
            self._refuse(name, f"must be fp32 or fp64 [{n}] on cuda:{self._dev}, got {t.dtype} {list(t.shape)} on {t.device}")
        return t.contiguous()

    def _common(self, logits, cu_num_draft, cu_num_sampled, draft_tokens, temperature):
        """The checked arguments that both verifiers take: (logits' dtype code, row stride, B, ...)."""
        dt, shape, st = _LOGITS.get(logits.dtype), logits.shape, logits.stride()
        if logits.get_device() != self._dev or dt is None or len(shape) != 2 or shape[1] == 0 or (st[1] != 1 and shape[1] > 1):
            _lib.require_cuda(logits, "logits")
            self._refuse("logits", f"must be fp32, fp16 or bf16 rows with a contiguous vocabulary dim on cuda:{self._dev}")
        rows, V = shape
        B = cu_num_draft.shape[0] if cu_num_draft.dim() == 1 else -1
        if rows > self.max_rows or B > self.max_batch:
            self._refuse(f"{rows} rows / {B} requests", f"exceed this verifier ({self.max_rows} / {self.max_batch})")
        ld = st[0] if rows > 1 else V
        if ld < V:
            self._refuse("logits", "has rows that share words")
        cu_d, cu_s = self._ints(cu_num_draft, "cu_num_draft", (B,)), self._ints(cu_num_sampled, "cu_num_sampled", (B,))
        tokens = self._ints(draft_tokens, "draft_tokens", (draft_tokens.numel(),))
        if temperature is not None:
            if temperature.get_device() != self._dev or not temperature.is_floating_point() or temperature.shape != (B,):
                _lib.require_cuda(temperature, "temperature")
                self._refuse("temperature", f"must be floating-point [{B}] on cuda:{self._dev}")
            if temperature.dtype is not torch.float32 or not temperature.is_contiguous():
                temperature = temperature.to(torch.float32).contiguous()
        return dt, ld, rows, V, B, cu_d, cu_s, tokens, temperature


_LOGITS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class SampledVerifier(_ProbabilityVerifier):
    """Verification of draft trees (a chain is a tree) at a temperature, on cfb_tree_verify_sampled. Every row draws a
    token from the target's softmax(logits / temperature) with its given number; from the root, a request's walk moves to
    the first child that carries the row's token and ends where none does, with that token as the bonus. The output is
    distributed as the target's own. Requests of temperature 0 take the argmax, as TreeVerifier."""

    def __init__(self, max_rows: int, max_batch: int, max_spec_len: int, device=None):
        super().__init__(max_rows, max_batch, max_spec_len, device)
        self.accepted_path = torch.empty(max_batch, max_spec_len, dtype=torch.int32, device=self.ws.device)
        self._ptrs = tuple(t.data_ptr() for t in self._buffers()) + (self.ws_ptr, self.ws_bytes, self.err.data_ptr())

    def _buffers(self):
        return self.out_tokens, self.accepted_path, self.accepted_len, self.logprobs

    def __call__(self, logits, cu_num_draft, cu_num_sampled, draft_tokens, parents, uniforms, temperature=None, stream=None):
        """(output_tokens [B, max_spec + 1], accepted_path [B, max_spec], accepted_len [B]) int32 and logprobs fp32
        [B, max_spec + 1], views of this verifier's buffers, -1 (logprobs 0) after a request's tokens. logits, offsets,
        draft_tokens and parents as TreeVerifier takes them; uniforms fp32 or fp64 [rows] in [0, 1), one number a logits
        row; temperature [B] (None: 1 for all; 0: greedy). logprobs are the output tokens' log probabilities under
        softmax(logits / temperature) (greedy requests: softmax(logits)), off by less than 2^-17 and a rounding to fp32. A
        token of logit -inf is never drawn; a row of nothing else ends its walk with token -1."""
        if stream is not None:
            with torch.cuda.stream(stream):
                return self(logits, cu_num_draft, cu_num_sampled, draft_tokens, parents, uniforms, temperature)
        dt, ld, rows, V, B, cu_d, cu_s, tokens, temp = self._common(logits, cu_num_draft, cu_num_sampled, draft_tokens, temperature)
        par, u = self._ints(parents, "parents", tuple(tokens.shape)), self._numbers(uniforms, "uniforms", rows)
        if B and rows:
            _lib.check(self.lib.cfb_tree_verify_sampled(
                logits.data_ptr(), ld, rows, V, dt, cu_d.data_ptr(), cu_s.data_ptr(), tokens.data_ptr(), par.data_ptr(),
                tokens.shape[0], u.data_ptr(), u.element_size(), None if temp is None else temp.data_ptr(), B, self.max_spec,
                *self._ptrs, _lib.stream_of(self._dev, "SampledVerifier")), "cfb_tree_verify_sampled")
        elif B:
            self._refuse("logits", "has no rows")
        return self._outputs(B)


class RejectionVerifier(_ProbabilityVerifier):
    """Verification of drafted chains whose draft model gave probabilities, on cfb_chain_verify_rejection. A draft stays if
    u q < p (its draft and target probability); the first that does not is replaced by a draw from max(p - q, 0), and a
    chain that stays whole is followed by a draw from its last row. The output is distributed as the target's own.

    ``draft_ids`` [R] (distinct, as a shortlist file's ids): the tokens that the columns of draft_probs stand for; all
    other tokens have draft probability 0. None: the columns are the vocabulary."""

    def __init__(self, max_rows: int, max_batch: int, max_spec_len: int, vocab_size: int, draft_ids=None, device=None):
        super().__init__(max_rows, max_batch, max_spec_len, device)
        self.vocab, self.width, self.index_of = vocab_size, vocab_size, None
        if draft_ids is not None:
            ids = draft_ids.to(device=self.ws.device, dtype=torch.int64)
            if ids.dim() != 1 or ids.numel() == 0 or int(ids.min()) < 0 or int(ids.max()) >= vocab_size or ids.unique().numel() != ids.numel():
                self._refuse("draft_ids", f"must be distinct token ids [R] below {vocab_size}")
            self.width = ids.numel()
            self.index_of = torch.full((vocab_size,), -1, dtype=torch.int32, device=self.ws.device)
            self.index_of[ids] = torch.arange(self.width, dtype=torch.int32, device=self.ws.device)
        self._ptrs = tuple(t.data_ptr() for t in self._buffers()) + (self.ws_ptr, self.ws_bytes, self.err.data_ptr())

    def _buffers(self):
        return self.out_tokens, self.accepted_len, self.logprobs

    def __call__(self, logits, cu_num_draft, cu_num_sampled, draft_tokens, draft_probs, uniforms, resample, temperature=None,
                 stream=None):
        """(output_tokens [B, max_spec + 1], accepted_len [B]) int32 and logprobs fp32 [B, max_spec + 1], as
        SampledVerifier's. Request b's drafts are the flat rows [cu_num_draft[b - 1], cu_num_draft[b]) of draft_tokens and
        of draft_probs fp32 [drafts, R] (contiguous rows; what is not a positive number counts as 0); uniforms [drafts]
        accept them, resample [B] draws, each fp32 or fp64 in [0, 1). A greedy request (temperature 0) keeps the drafts
        that are its rows' argmax."""
        if stream is not None:
            with torch.cuda.stream(stream):
                return self(logits, cu_num_draft, cu_num_sampled, draft_tokens, draft_probs, uniforms, resample, temperature)
        dt, ld, rows, V, B, cu_d, cu_s, tokens, temp = self._common(logits, cu_num_draft, cu_num_sampled, draft_tokens, temperature)
        n = tokens.shape[0]
        if V != self.vocab:
            self._refuse("logits", f"has {V} columns, this verifier's vocabulary {self.vocab}")
        if (draft_probs.get_device() != self._dev or draft_probs.dtype != torch.float32 or draft_probs.shape != (n, self.width)
                or (draft_probs.stride(1) != 1 and self.width > 1) or (n > 1 and draft_probs.stride(0) < self.width)):
            _lib.require_cuda(draft_probs, "draft_probs")
            self._refuse("draft_probs", f"must be fp32 [{n}, {self.width}] with contiguous rows on cuda:{self._dev}")
        u, v = self._numbers(uniforms, "uniforms", n), self._numbers(resample, "resample", B)
        if u.dtype != v.dtype:
            u, v = u.double(), v.double()
        if B and rows:
            _lib.check(self.lib.cfb_chain_verify_rejection(
                logits.data_ptr(), ld, rows, V, dt, cu_d.data_ptr(), cu_s.data_ptr(), tokens.data_ptr(), draft_probs.data_ptr(),
                draft_probs.stride(0) if n > 1 else self.width, n, self.width,
                None if self.index_of is None else self.index_of.data_ptr(), u.data_ptr(), v.data_ptr(), v.element_size(),
                None if temp is None else temp.data_ptr(), B, self.max_spec, *self._ptrs,
                _lib.stream_of(self._dev, "RejectionVerifier")), "cfb_chain_verify_rejection")
        elif B:
            self._refuse("logits", "has no rows")
        return self._outputs(B)
