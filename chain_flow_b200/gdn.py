"""Tree-aware Gated-DeltaNet verification on the sm_100a kernel (cfb_tree_gdn).

``tree_gated_delta_scan`` keeps the reference's signature and semantics
(src/chain_flow/kernels/tree_scan.py:43-78) for a single tree, and ``tree_gdn_batched`` runs B
independent trees in one launch. ``make_tree`` builds the seeded BFS parent arrays the
benchmarks use (parent < child, bounded depth and branching). ``gdn_verify`` is the in-engine
variant of the reference's vLLM patch (gate from the model's raw parameters, slot-addressed
states, a path-parallel walk of each row's ancestor chain; cfb_tree_gdn_verify). ``ChunkedGdn`` and
``gdn_step`` run the same recurrence without a tree, over prompts and single tokens (cfb_gdn_chunk,
cfb_gdn_step).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib


def make_tree(n_nodes: int, max_depth: int, max_branch: int, seed: int):
    """(parent [N] int64, depth [N] int64) of a random BFS-ordered tree: node 0 is the root,
    every parent index is smaller than its child's, depth < max_depth, children <= max_branch."""
    g = torch.Generator().manual_seed(seed)
    parent, depth, nchild = [], [], []
    while len(parent) < n_nodes:
        i = len(parent)
        if i == 0:
            parent.append(-1); depth.append(0); nchild.append(0)
            continue
        cands = [j for j in range(i) if depth[j] < max_depth - 1 and nchild[j] < max_branch]
        if not cands:
            raise ValueError("tree shape cannot hold that many nodes")
        dmin = min(depth[j] for j in cands)
        cands = [j for j in cands if depth[j] == dmin]
        p = cands[int(torch.randint(len(cands), (1,), generator=g))]
        parent.append(p); depth.append(depth[p] + 1); nchild[p] += 1; nchild.append(0)
    return torch.tensor(parent), torch.tensor(depth)


def tree_gdn_batched(q, k, v, g, beta, parent, init, *, use_qk_l2norm: bool = True,
                     states: torch.Tensor | None = None):
    """q,k [B,N,H,128] fp16; v [B,N,H,Dv] fp16; g,beta [B,N,H] fp32; parent [B,N] (parent < child,
    -1 = reads init); init [B,H,128,Dv] fp32 -> (o [B,N,H,Dv] fp32, states [B,N,H,128,Dv] fp32)."""
    for t, n in ((q, "q"), (k, "k"), (v, "v"), (g, "g"), (beta, "beta"), (init, "init")):
        _lib.require_cuda(t, n)
    B, N, H, Dk = q.shape
    Dv = v.shape[-1]
    q = q.to(torch.float16).contiguous(); k = k.to(torch.float16).contiguous()
    v = v.to(torch.float16).contiguous()
    g = g.to(torch.float32).contiguous(); beta = beta.to(torch.float32).contiguous()
    par = parent.to(device=q.device, dtype=torch.int32).contiguous()
    init = init.to(torch.float32).contiguous()
    o = torch.empty(B, N, H, Dv, device=q.device, dtype=torch.float32)
    if states is None:
        states = torch.empty(B, N, H, Dk, Dv, device=q.device, dtype=torch.float32)
    lib = _lib.load()
    _lib.check(lib.cfb_tree_gdn(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(),
                                par.data_ptr(), init.data_ptr(), o.data_ptr(), states.data_ptr(),
                                B, N, H, Dk, Dv, int(use_qk_l2norm), C.c_void_p(_lib.stream_ptr())),
               "cfb_tree_gdn")
    return o, states


def tree_gated_delta_scan(query, key, value, g, beta, parent, depth, initial_state, *,
                          use_qk_l2norm: bool = True):
    """Reference-signature single tree: query,key [N,H,Dk]; value [N,H,Dv]; g,beta [N,H];
    parent [N] (-1 = root); depth [N] (accepted for signature parity: nodes must be in BFS order,
    parent < child, which the kernel relies on instead); initial_state [H,Dk,Dv]. No host sync: a
    node whose parent is neither -1 nor an earlier node gets NaN output and state (so do its
    descendants), and the bad index is never dereferenced."""
    par = parent.view(1, -1)
    o, st = tree_gdn_batched(query[None], key[None], value[None], g[None], beta[None], par,
                             initial_state[None], use_qk_l2norm=use_qk_l2norm)
    return o[0], st[0]


_DTYPE_CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_HALVES = (torch.float16, torch.bfloat16)


def ancestor_chains(parent: torch.Tensor, max_depth: int):
    """(chain [N, max_depth + 1] int32, depth [N] int32) from a parent array (parent < child,
    -1 = root) on the parent's device: chain[t, kk] is the ancestor kk levels above node t
    (chain[t, 0] = t; entries past depth[t] repeat the top ancestor), the layout the in-engine
    verify walks from chain[t, depth[t]] (the root) down to t. Pointer jumping with device ops
    only: no host sync, so it can be captured in a CUDA graph."""
    p = parent.to(torch.int64).view(-1)
    N = p.numel()
    cur = torch.arange(N, device=p.device)
    cols, depth = [cur], torch.zeros(N, dtype=torch.int64, device=p.device)
    for _ in range(max_depth):
        up = p[cur] if N else cur
        has = up >= 0
        depth = depth + has.to(torch.int64)
        cur = torch.where(has, up, cur)
        cols.append(cur)
    return torch.stack(cols, dim=1).to(torch.int32), depth.to(torch.int32)


def gdn_verify(A_log, dt_bias, a, b, q, k, v, o, state, chain, depth, out_slot, init_slot, rows=None, *,
               scale: float, write_out: bool = True, write_state: bool = True) -> None:
    """The in-engine tree GDN verify (reference vLLM patch ``gdn_verify``,
    src/chain_flow/patches/vllm-0.25.1-chain-flow-tree.patch:4606) on cfb_tree_gdn_verify: for
    each query row (``rows``, default all), walk its ancestor chain from ``state[init_slot]``,
    write o and ``state[out_slot]`` in place. q, k [T, H, 128] and v, o [T, HV, V] fp16 or
    bf16; a, b [T, HV] and A_log, dt_bias [HV] fp32 / fp16 / bf16; state fp32
    [slots, HV, V, 128]; chain, depth, slots, rows int32, all on one CUDA device."""
    lib = _lib.load()
    for t_, n in ((q, "q"), (k, "k"), (v, "v"), (state, "state"), (chain, "chain")):
        _lib.require_cuda(t_, n)
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise _lib.CfbError("gdn_verify: q, k, v must share one dtype, fp16 or bf16")
    if state.dtype != torch.float32 or state.stride(-1) != 1 or not state[0].is_contiguous():
        raise _lib.CfbError("gdn_verify: state must be fp32 [slots, HV, V, K] with contiguous slots")
    for t_ in (q, k, v, a, b, A_log, dt_bias):
        if not t_.is_contiguous():
            raise _lib.CfbError("gdn_verify: q, k, v, a, b, A_log, dt_bias must be contiguous")
    ints = [t_.to(torch.int32).contiguous() for t_ in (chain, depth, out_slot, init_slot)]
    rows_i = rows.to(torch.int32).contiguous() if rows is not None else None
    T_rows = rows_i.numel() if rows_i is not None else q.shape[0]
    H, K = q.shape[1], q.shape[2]
    HV, V = v.shape[1], v.shape[2]
    _lib.check(lib.cfb_tree_gdn_verify(
        A_log.data_ptr(), _DTYPE_CODE[A_log.dtype], dt_bias.data_ptr(), _DTYPE_CODE[dt_bias.dtype],
        a.data_ptr(), _DTYPE_CODE[a.dtype], b.data_ptr(), _DTYPE_CODE[b.dtype],
        q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr() if o is not None else None,
        _DTYPE_CODE[q.dtype], state.data_ptr(), state.stride(0), ints[0].data_ptr(), ints[0].stride(0),
        ints[1].data_ptr(), ints[2].data_ptr(), ints[3].data_ptr(),
        rows_i.data_ptr() if rows_i is not None else None, float(scale), T_rows, H, HV, K, V,
        int(write_out), int(write_state), _lib.stream_ptr()), "cfb_tree_gdn_verify")


def gdn_factor(A_log, dt_bias, a, b, q, k, v, o, state, chain, depth, init_slot, row_start, row_count, *,
               scale: float, n_max: int) -> None:
    """The shared-root factorisation of the in-engine verify (reference fork ``gdn_factor``,
    src/chain_flow/patches/vllm-0.25.1-chain-flow-tree.patch:4664-5094) on cfb_tree_gdn_factor:
    the outputs ``o`` of ``gdn_verify`` for requests whose rows [row_start[s], + row_count[s]) all
    start from the state slot ``init_slot[row_start[s]]``, reading that state once per (request,
    head) and writing no state. ``chain`` rows hold global row ids. Same dtypes as ``gdn_verify``;
    n_max >= every row_count (<= 64)."""
    lib = _lib.load()
    for t_, n in ((q, "q"), (k, "k"), (v, "v"), (o, "o"), (state, "state"), (chain, "chain")):
        _lib.require_cuda(t_, n)
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype or o.dtype != q.dtype:
        raise _lib.CfbError("gdn_factor: q, k, v, o must share one dtype, fp16 or bf16")
    if state.dtype != torch.float32 or state.stride(-1) != 1 or not state[0].is_contiguous():
        raise _lib.CfbError("gdn_factor: state must be fp32 [slots, HV, V, K] with contiguous slots")
    for t_ in (q, k, v, o, a, b, A_log, dt_bias):
        if not t_.is_contiguous():
            raise _lib.CfbError("gdn_factor: q, k, v, o, a, b, A_log, dt_bias must be contiguous")
    ch, dp, isl, rs, rc = (t_.to(torch.int32).contiguous() for t_ in (chain, depth, init_slot, row_start, row_count))
    H, K = q.shape[1], q.shape[2]
    HV, V = v.shape[1], v.shape[2]
    _lib.check(lib.cfb_tree_gdn_factor(
        A_log.data_ptr(), _DTYPE_CODE[A_log.dtype], dt_bias.data_ptr(), _DTYPE_CODE[dt_bias.dtype],
        a.data_ptr(), _DTYPE_CODE[a.dtype], b.data_ptr(), _DTYPE_CODE[b.dtype], q.data_ptr(), k.data_ptr(),
        v.data_ptr(), o.data_ptr(), _DTYPE_CODE[q.dtype], state.data_ptr(), state.stride(0), ch.data_ptr(),
        ch.stride(0), dp.data_ptr(), isl.data_ptr(), rs.data_ptr(), rc.data_ptr(), rs.numel(), int(n_max),
        float(scale), H, HV, K, V, _lib.stream_ptr()), "cfb_tree_gdn_factor")


def _refuse_sequence(what, A_log, dt_bias, a, b, q, k, v, o, state, init_slot, out_slot, out_state, B):
    """Raises with what is wrong with the arguments that _sequence_args does not take."""
    if q.dim() != 3 or v.dim() != 3 or state.dim() != 4:
        raise _lib.CfbError(f"{what}: q must be [T, H, K], v [T, HV, V] and state [slots, HV, V, K]")
    T, H, K = q.shape
    HV, V = v.shape[1], v.shape[2]
    for t, n, shape in ((q, "q", (T, H, K)), (k, "k", (T, H, K)), (v, "v", (T, HV, V)), (o, "o", (T, HV, V)),
                        (a, "a", (T, HV)), (b, "b", (T, HV)), (A_log, "A_log", (HV,)), (dt_bias, "dt_bias", (HV,)),
                        (state, "state", (state.shape[0], HV, V, K)), (out_state, "out_state", tuple(state.shape)),
                        (init_slot, "init_slot", (B,)), (out_slot, "out_slot", (B,))):
        _lib.require_cuda(t, n)
        if t.device != q.device:
            raise _lib.CfbError(f"{what}: {n} is on {t.device}, q on {q.device}")
        if tuple(t.shape) != shape:
            raise _lib.CfbError(f"{what}: {n} must be {list(shape)}, got {list(t.shape)}")
    if q.dtype not in (torch.float16, torch.bfloat16) or any(t.dtype != q.dtype for t in (k, v, o)):
        raise _lib.CfbError(f"{what}: q, k, v, o must share one dtype, fp16 or bf16")
    if any(t.dtype not in _DTYPE_CODE for t in (A_log, dt_bias, a, b)):
        raise _lib.CfbError(f"{what}: a, b, A_log and dt_bias must be fp32, fp16 or bf16")
    raise _lib.CfbError(f"{what}: q, k, v, o need contiguous heads (any token stride), a, b, A_log, dt_bias too, and state "
                        "and out_state must be fp32 with contiguous slots and one slot stride")


def _token_stride(st, T, heads, dim):
    """The token stride of a [T, heads, dim] tensor of strides ``st`` with contiguous heads, else None. (One token's
    can be any number, as 1 of a transposed column: what the heads take stands for it.)"""
    if st[2] != 1 or (st[1] != dim and heads != 1):
        return None
    return st[0] if T > 1 else heads * dim


def _sequence_args(what, A_log, dt_bias, a, b, q, k, v, o, state, init_slot, out_slot, scale, out_state, B):
    """(the packed cfb_gdn_args, the converted index tensors, which the caller keeps until the launch)."""
    out_state = state if out_state is None else out_state
    qs, vs, ss, dev, dt = q.shape, v.shape, state.shape, q.get_device(), q.dtype
    good = len(qs) == 3 and len(vs) == 3 and len(ss) == 4 and dev >= 0 and dt in _HALVES and k.dim() == 3 and o.dim() == 3
    if good:
        T, H, K = qs
        HV, V = vs[1], vs[2]
        gates = (T, HV)
        sq, sk = _token_stride(q.stride(), T, H, K), _token_stride(k.stride(), T, H, K)
        sv, so = _token_stride(v.stride(), T, HV, V), _token_stride(o.stride(), T, HV, V)
        sa, sb, s_in, s_out = a.stride(), b.stride(), state.stride(), out_state.stride()
        c_A, c_d, c_a, c_b = (_DTYPE_CODE.get(t.dtype) for t in (A_log, dt_bias, a, b))
        good = (k.shape == qs and vs[0] == T and o.shape == vs and a.shape == gates and b.shape == gates
                and A_log.shape == (HV,) and dt_bias.shape == (HV,) and ss[1:] == (HV, V, K) and out_state.shape == ss
                and init_slot.shape == (B,) and out_slot.shape == (B,)
                and k.dtype == dt and v.dtype == dt and o.dtype == dt
                and state.dtype == torch.float32 and out_state.dtype == torch.float32
                and None not in (sq, sk, sv, so, c_A, c_d, c_a, c_b)
                and (HV == 1 or (sa[1] == 1 and sb[1] == 1 and A_log.stride(0) == 1 and dt_bias.stride(0) == 1))
                and s_in[3] == 1 and s_in[2] == K and (HV == 1 or s_in[1] == V * K) and s_out[2:] == s_in[2:]
                and (HV == 1 or s_out[1] == s_in[1]) and s_out[0] == s_in[0]
                and all(t.get_device() == dev for t in (k, v, o, a, b, A_log, dt_bias, state, out_state, init_slot, out_slot)))
    if not good:
        _refuse_sequence(what, A_log, dt_bias, a, b, q, k, v, o, state, init_slot, out_slot, out_state, B)
    init, to = _lib.int32(init_slot), _lib.int32(out_slot)
    return _lib.PACK_GDN_ARGS(
        A_log.data_ptr(), c_A, dt_bias.data_ptr(), c_d, a.data_ptr(), c_a, sa[0], b.data_ptr(), c_b, sb[0], q.data_ptr(), sq,
        k.data_ptr(), sk, v.data_ptr(), sv, o.data_ptr(), so, _DTYPE_CODE[dt], state.data_ptr(), out_state.data_ptr(), s_in[0],
        ss[0], init.data_ptr(), to.data_ptr(), scale, H, HV, K, V), (init, to)


def gdn_step(A_log, dt_bias, a, b, q, k, v, o, state, init_slot, out_slot, *, scale: float, out_state=None,
             stream=None) -> None:
    """One token of the gated delta rule for each of B requests (cfb_gdn_step): row b walks from
    ``state[init_slot[b]]`` (negative: zeros), writes ``o[b]`` and ``out_state[out_slot[b]]``
    (default: ``state`` itself; negative: not kept). q, k [B, H, 128], v, o [B, HV, V] fp16 or bf16
    with contiguous heads; a, b [B, HV] and A_log, dt_bias [HV] fp32 / fp16 / bf16; state fp32
    [slots, HV, V, 128]."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return gdn_step(A_log, dt_bias, a, b, q, k, v, o, state, init_slot, out_slot, scale=scale, out_state=out_state)
    lib = _lib.load()
    B = q.shape[0]
    args, keep = _sequence_args("gdn_step", A_log, dt_bias, a, b, q, k, v, o, state, init_slot, out_slot, scale, out_state, B)
    _lib.check(lib.cfb_gdn_step(args, B, _lib.stream_of(q.get_device(), "gdn_step")), "cfb_gdn_step")


class ChunkedGdn:
    """The gated delta rule over whole sequences (cfb_gdn_chunk) for calls of up to ``max_tokens``
    tokens of up to ``max_requests`` requests and ``value_heads`` value heads. Owns the workspace,
    so a call allocates nothing; calls share it, so order them on one stream."""

    def __init__(self, max_tokens: int, max_requests: int, value_heads: int, device=None):
        self.lib = _lib.load()
        if max_tokens < 0 or max_requests <= 0 or value_heads <= 0:
            raise _lib.CfbError("ChunkedGdn: max_requests and value_heads must be positive, max_tokens not negative")
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.max_tokens, self.max_requests, self.value_heads = max_tokens, max_requests, value_heads
        self.ws_bytes = int(self.lib.cfb_gdn_chunk_workspace(max_tokens, max_requests, value_heads))
        self.ws = torch.empty(self.ws_bytes + 256, dtype=torch.uint8, device=self.device)
        self.ws_ptr = (self.ws.data_ptr() + 255) // 256 * 256
        self._dev, self._ran = self.ws.get_device(), False

    def check(self) -> None:
        """Raises if a device-side wait of the last call with tokens expired (its outputs are then invalid, its
        states NaN; without such a call there is nothing to raise). Waits for the GPU."""
        err = C.c_int(0)
        torch.cuda.synchronize(self.device)
        if not self._ran:                                # the error word is the kernels' to write
            return
        _lib.check(self.lib.cfb_gdn_chunk_error(self.ws_ptr, C.byref(err)), "cfb_gdn_chunk_error")
        if err.value:
            raise _lib.CfbError(f"ChunkedGdn: device error {err.value} (a bounded wait expired); outputs are invalid")

    def __call__(self, A_log, dt_bias, a, b, q, k, v, o, state, cu_seqlens, init_slot, out_slot, *, scale: float,
                 out_state=None, stream=None) -> None:
        """Request b's tokens are the rows [cu_seqlens[b], cu_seqlens[b + 1]) (int32 [B + 1], on the
        GPU), walked from ``state[init_slot[b]]``; arguments otherwise as ``gdn_step``. Rows of no
        request are not written."""
        if stream is not None:
            with torch.cuda.stream(stream):
                return self(A_log, dt_bias, a, b, q, k, v, o, state, cu_seqlens, init_slot, out_slot, scale=scale,
                            out_state=out_state)
        _lib.require_cuda(cu_seqlens, "cu_seqlens")
        B = cu_seqlens.numel() - 1
        if cu_seqlens.dim() != 1 or B < 0 or cu_seqlens.get_device() != q.get_device() or q.dim() != 3 or v.dim() != 3:
            raise _lib.CfbError("ChunkedGdn: cu_seqlens must be 1-D [requests + 1] on q's device, q [T, H, K], v [T, HV, V]")
        if q.get_device() != self._dev:
            raise _lib.CfbError(f"ChunkedGdn: q is on {q.device}, this object's workspace on {self.device}")
        T, HV = q.shape[0], v.shape[1]
        if T > self.max_tokens or B > self.max_requests or HV > self.value_heads:
            raise _lib.CfbError(f"ChunkedGdn: {T} tokens / {B} requests / {HV} value heads exceed this object's "
                                f"{self.max_tokens} / {self.max_requests} / {self.value_heads}")
        args, keep = _sequence_args("ChunkedGdn", A_log, dt_bias, a, b, q, k, v, o, state, init_slot, out_slot, scale,
                                    out_state, B)
        cu = _lib.int32(cu_seqlens)
        _lib.check(self.lib.cfb_gdn_chunk(args, cu.data_ptr(), T, B, self.ws_ptr, self.ws_bytes,
                                          _lib.stream_of(self._dev, "ChunkedGdn")), "cfb_gdn_chunk")
        if T and B:
            self._ran = True
