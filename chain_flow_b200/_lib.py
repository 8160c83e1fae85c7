"""ctypes binding of libcfb.so (include/cfb.h).

The product path is CUDA only: importing the binding never falls back to anything. If the
shared library is missing it is built in-tree with nvcc (chain_flow_b200/build.py); if that is
impossible, or no CUDA device is visible when a kernel is requested, the call raises.
"""
from __future__ import annotations

import ctypes as C
import struct
import threading
from pathlib import Path

_PKG = Path(__file__).resolve().parent
LIB_PATH = _PKG / "libcfb.so"

CFB_OK = 0
STATUS_NAMES = {
    0: "CFB_OK", 1: "CFB_ERR_INVALID_ARG", 2: "CFB_ERR_UNSUPPORTED", 3: "CFB_ERR_WORKSPACE",
    4: "CFB_ERR_CUDA", 5: "CFB_ERR_COOP_LAUNCH", 6: "CFB_ERR_DEVICE_TIMEOUT",
}
MODE_FLOW, MODE_CHAIN, MODE_TREE, MODE_BEAM_CHAIN, MODE_BEAM_TREE = range(5)
INIT_GIVEN, INIT_REPEAT_LAST, INIT_DELTA = range(3)
INIT_MODES = {"noise": INIT_GIVEN, "repeat_last": INIT_REPEAT_LAST, "delta": INIT_DELTA}

# every extern "C" symbol declared in include/cfb.h
EXPORTED = [
    "cfb_abi_version", "cfb_last_cuda_error", "cfb_packed_bytes", "cfb_pack_linear",
    "cfb_fold_bias", "cfb_time_embed", "cfb_plan_workspace", "cfb_plan_build", "cfb_plan_run",
    "cfb_plan_error", "cfb_plan_info", "cfb_plan_buffer", "cfb_tree_gdn", "cfb_tree_gdn_noalloc",
    "cfb_plan_segments", "cfb_plan_run_segment", "cfb_wide_gemm", "cfb_wide_packed_bytes", "cfb_wide_pack", "cfb_wide_workspace",
    "cfb_wide_create", "cfb_wide_run", "cfb_wide_error", "cfb_wide_info", "cfb_wide_destroy",
    "cfb_ring_write", "cfb_ring_gather", "cfb_tree_gdn_verify", "cfb_vae_workspace", "cfb_vae_create",
    "cfb_vae_plan_workspace", "cfb_vae_plan_build", "cfb_tree_attn_merge", "cfb_tree_verify_workspace",
    "cfb_tree_verify_greedy", "cfb_tree_gdn_factor", "cfb_kv_write", "cfb_kv_read", "cfb_paged_attn_workspace",
    "cfb_paged_attn", "cfb_paged_attn_error", "cfb_gdn_step", "cfb_gdn_chunk_workspace", "cfb_gdn_chunk", "cfb_gdn_chunk_error",
    "cfb_verify_workspace", "cfb_tree_verify_sampled", "cfb_chain_verify_rejection", "cfb_kv_keep", "cfb_kv_copy_pages",
    "cfb_pages_reserve", "cfb_pages_release", "cfb_pages_fork",
]
ABI_VERSION = 5
XROWS, XFLOATS = 64, 18          # CFB_XROWS, CFB_XFLOATS: the merged-list exchange rows
BUF_PATH_H16, BUF_PATH_MID, BUF_HEAD_IN, BUF_LASTP, BUF_CUM, BUF_QKV0, BUF_X32_0, BUF_KVC0, BUF_PROF, BUF_PHASES, \
    BUF_TP_CAND, BUF_TP_CHEAD = range(12)
PK_PREP, PK_GEMM, PK_ATTN, PK_BEAM, PK_RMERGE, PK_GATHER, PK_TPXA, PK_TPSEL, PK_TPGATH = range(9)  # CFB_BUF_PHASES [0]
PO_NONE, PO_BEAM_CHAIN, PO_BEAM_TREE, PO_PUBLISH = range(4)        # CFB_BUF_PHASES [6]
RUN_PROFILE = 1
# device error word codes (cfb_plan_error / cfb_wide_error)
DEV_ERRORS = {1: "grid barrier wait expired", 2: "loaded-stage wait expired", 3: "free-stage wait expired",
              4: "slot or descriptor wait expired", 5: "bad phase", 6: "split-tile wait expired",
              7: "token or row id outside its table"}
EPI_F32, EPI_F16, EPI_GELU16, EPI_PART = 0, 1, 2, 3      # cfb_wide_gemm epilogues


class CfbError(RuntimeError):
    pass


class Linear(C.Structure):
    _fields_ = [("w", C.c_void_p), ("bias", C.c_void_p), ("colsum", C.c_void_p),
                ("nout", C.c_int), ("k", C.c_int)]


class Block(C.Structure):
    _fields_ = [("qkv", Linear), ("self_out", Linear), ("cross_q", Linear), ("cross_kv", Linear),
                ("cross_out", Linear), ("ffn_up", Linear), ("ffn_down", Linear)]


class Expert(C.Structure):
    _fields_ = [("pos_emb", C.c_void_p), ("temb", C.c_void_p), ("out_proj", Linear),
                ("blocks", C.POINTER(Block))]


class Drafter(C.Structure):
    _fields_ = [("hidden", C.c_int), ("heads", C.c_int), ("layers", C.c_int), ("steps", C.c_int),
                ("draft_len", C.c_int), ("chunk", C.c_int), ("ctx_rows", C.c_int),
                ("n_experts", C.c_int), ("experts", C.POINTER(Expert)),
                ("path_order", C.c_int), ("markov_rank", C.c_int), ("vocab", C.c_int),
                ("shortlist_rows", C.c_int), ("embed", C.c_void_p), ("path_offsets", Linear),
                ("path_offset_bias", C.c_void_p), ("path_up", Linear), ("path_down", Linear),
                ("markov_w1", C.c_void_p), ("head", Linear), ("shortlist", C.c_void_p),
                ("head_row0", C.c_int)]


class Run(C.Structure):
    _fields_ = [("mode", C.c_int), ("init_mode", C.c_int), ("batch", C.c_int), ("width", C.c_int), ("depth", C.c_int),
                ("tree_keep", C.c_int), ("tree_topb", C.c_int), ("grid", C.c_int), ("flags", C.c_int),
                ("ctx", C.c_void_p), ("z0", C.c_void_p), ("known0", C.c_void_p),
                ("pred", C.c_void_p), ("tokens", C.c_void_p),
                ("ranks", C.c_int), ("rank", C.c_int), ("xloc", C.c_void_p), ("xall", C.c_void_p),
                ("twopass_m", C.c_int), ("wait_budget_ns", C.c_uint64)]


class VaeLayer(C.Structure):
    _fields_ = [("qkv", Linear), ("attn_out", Linear), ("ffn_up", Linear), ("ffn_down", Linear)]


class VaeSide(C.Structure):
    _fields_ = [("in_dim", C.c_int), ("width", C.c_int), ("out_dim", C.c_int), ("layers", C.c_int),
                ("heads", C.c_int), ("max_len", C.c_int), ("in_proj", Linear), ("pos", C.c_void_p),
                ("layer", C.POINTER(VaeLayer)), ("out_proj", Linear)]


class KvCache(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("page_stride", C.c_int64), ("head_stride", C.c_int64), ("slot_stride", C.c_int64),
                ("scale_page_stride", C.c_int64), ("scale_head_stride", C.c_int64), ("scale_slot_stride", C.c_int64),
                ("pages", C.c_int), ("page_size", C.c_int), ("kv_heads", C.c_int), ("dim", C.c_int), ("dtype", C.c_int)]


class GdnArgs(C.Structure):
    _fields_ = [("A_log", C.c_void_p), ("A_log_dtype", C.c_int), ("dt_bias", C.c_void_p), ("dt_bias_dtype", C.c_int),
                ("a", C.c_void_p), ("a_dtype", C.c_int), ("a_stride", C.c_int64),
                ("b", C.c_void_p), ("b_dtype", C.c_int), ("b_stride", C.c_int64),
                ("q", C.c_void_p), ("q_stride", C.c_int64), ("k", C.c_void_p), ("k_stride", C.c_int64),
                ("v", C.c_void_p), ("v_stride", C.c_int64), ("o", C.c_void_p), ("o_stride", C.c_int64),
                ("dtype", C.c_int), ("state_in", C.c_void_p), ("state_out", C.c_void_p), ("slot_stride", C.c_int64),
                ("slots", C.c_int), ("init_slot", C.c_void_p), ("out_slot", C.c_void_p), ("scale", C.c_float),
                ("H", C.c_int), ("HV", C.c_int), ("K", C.c_int), ("V", C.c_int)]


# a cfb_gdn_args from its fields in order: packing takes a third of the time of filling a ctypes structure
PACK_GDN_ARGS = struct.Struct("@" + "".join(
    {C.c_void_p: "P", C.c_int: "i", C.c_int64: "q", C.c_float: "f"}[t] for _, t in GdnArgs._fields_) + "0P").pack

_lock = threading.Lock()
_lib = None


def _declare(lib):
    vp, i32, i64, sz = C.c_void_p, C.c_int, C.c_int64, C.c_size_t
    lib.cfb_abi_version.restype = i32
    lib.cfb_last_cuda_error.restype = C.c_char_p
    lib.cfb_packed_bytes.argtypes = [i32, i32]
    lib.cfb_packed_bytes.restype = sz
    lib.cfb_pack_linear.argtypes = [vp, i64, vp, i32, i32, vp, vp, i32, i32, vp]
    lib.cfb_fold_bias.argtypes = [vp, i64, i32, i32, vp, vp, vp, vp, vp, vp]
    lib.cfb_time_embed.argtypes = [vp, vp, vp, vp, i32, i32, vp, vp]
    lib.cfb_plan_workspace.argtypes = [C.POINTER(Drafter), C.POINTER(Run), C.POINTER(sz)]
    lib.cfb_plan_build.argtypes = [C.POINTER(Drafter), C.POINTER(Run), vp, sz]
    lib.cfb_plan_run.argtypes = [vp, vp]
    lib.cfb_plan_segments.argtypes = [vp, C.POINTER(i32)]
    lib.cfb_plan_run_segment.argtypes = [vp, i32, vp]
    lib.cfb_plan_error.argtypes = [vp, C.POINTER(i32)]
    lib.cfb_plan_info.argtypes = [vp, C.POINTER(i32), C.POINTER(i32), C.POINTER(i32), C.POINTER(i32)]
    lib.cfb_plan_buffer.argtypes = [vp, i32, C.POINTER(vp), C.POINTER(sz)]
    lib.cfb_tree_gdn.argtypes = [vp, vp, vp, vp, vp, vp, vp, vp, vp, i32, i32, i32, i32, i32, i32, vp]
    lib.cfb_tree_gdn_noalloc.argtypes = [vp, vp, vp, vp, vp, vp, vp, vp, i32, i32, i32, i32, i32, i32, vp]
    lib.cfb_wide_gemm.argtypes = [vp, i64, vp, i64, vp, vp, i64, i32, i32, i32, i32, i32, vp, vp]
    lib.cfb_wide_packed_bytes.argtypes = [i32, i32]
    lib.cfb_wide_packed_bytes.restype = sz
    lib.cfb_wide_pack.argtypes = [vp, i64, i32, i32, vp, vp]
    lib.cfb_wide_workspace.argtypes = [C.POINTER(Drafter), C.POINTER(Run), C.POINTER(sz)]
    lib.cfb_wide_create.argtypes = [C.POINTER(Drafter), C.POINTER(Run), vp, sz, C.POINTER(vp)]
    lib.cfb_wide_run.argtypes = [vp, vp]
    lib.cfb_wide_error.argtypes = [vp, C.POINTER(i32)]
    lib.cfb_wide_info.argtypes = [vp, C.POINTER(i32)]
    lib.cfb_wide_destroy.argtypes = [vp]
    lib.cfb_wide_destroy.restype = None
    lib.cfb_ring_write.argtypes = [vp, vp, vp, i32, i32, i32, vp, i64, vp, vp, vp, vp, vp, i64, i32, i32, vp]
    lib.cfb_ring_gather.argtypes = [vp, vp, vp, i32, i32, i32, vp, i32, vp, vp]
    lib.cfb_tree_gdn_verify.argtypes = [vp, i32, vp, i32, vp, i32, vp, i32, vp, vp, vp, vp, i32, vp, i64, vp, i32,
                                        vp, vp, vp, vp, C.c_float, i32, i32, i32, i32, i32, i32, i32, vp]
    lib.cfb_vae_workspace.argtypes = [C.POINTER(VaeSide), i32, i32, i32, C.POINTER(sz)]
    lib.cfb_vae_create.argtypes = [C.POINTER(VaeSide), i32, i32, i32, vp, vp, vp, sz, C.POINTER(vp)]
    lib.cfb_vae_plan_workspace.argtypes = [C.POINTER(VaeSide), i32, i32, i32, C.POINTER(sz)]
    lib.cfb_vae_plan_build.argtypes = [C.POINTER(VaeSide), i32, i32, i32, vp, vp, vp, sz]
    lib.cfb_tree_attn_merge.argtypes = [vp, i64, i64, vp, i64, i64, vp, i64, i64, vp, i64, i64, vp, i64, i64,
                                        vp, vp, vp, C.c_float, i32, i32, i32, i32, i32, i32, vp]
    lib.cfb_tree_gdn_factor.argtypes = [vp, i32, vp, i32, vp, i32, vp, i32, vp, vp, vp, vp, i32, vp, i64, vp, i32,
                                        vp, vp, vp, vp, i32, i32, C.c_float, i32, i32, i32, i32, vp]
    lib.cfb_tree_verify_workspace.argtypes = [i32, i32]
    lib.cfb_tree_verify_workspace.restype = sz
    lib.cfb_tree_verify_greedy.argtypes = [vp, i64, i32, i32, i32, vp, vp, vp, vp, i32, i32, vp, vp, vp, vp, vp,
                                           sz, vp, vp]
    lib.cfb_verify_workspace.argtypes = [i32, i32]
    lib.cfb_verify_workspace.restype = sz
    lib.cfb_tree_verify_sampled.argtypes = [vp, i64, i32, i32, i32, vp, vp, vp, vp, i32, vp, i32, vp, i32, i32, vp, vp, vp, vp,
                                            vp, sz, vp, vp]
    lib.cfb_chain_verify_rejection.argtypes = [vp, i64, i32, i32, i32, vp, vp, vp, vp, i64, i32, i32, vp, vp, vp, i32, vp, i32,
                                               i32, vp, vp, vp, vp, sz, vp, vp]
    lib.cfb_kv_keep.argtypes = [vp, i32, vp, i64, i32, vp, vp, i64, vp, i32, i32, vp]
    lib.cfb_kv_copy_pages.argtypes = [vp, i32, vp, vp, vp, i32, vp]
    lib.cfb_pages_reserve.argtypes = [vp, i32, i32, vp, i64, i32, vp, vp, vp, i32, vp]
    lib.cfb_pages_release.argtypes = [vp, i32, i32, vp, i64, i32, vp, vp, i32, vp, vp]
    lib.cfb_pages_fork.argtypes = [vp, i32, i32, vp, i64, i32, i32, vp, vp, vp, vp, i32, vp, i32, vp]
    lib.cfb_kv_write.argtypes = [C.POINTER(KvCache), vp, i64, i64, vp, i64, i64, i32, vp, i32, vp]
    lib.cfb_kv_read.argtypes = [C.POINTER(KvCache), vp, i32, vp, i64, i64, vp, i64, i64, i32, vp]
    lib.cfb_paged_attn_workspace.argtypes = [i32, i32, i32]
    lib.cfb_paged_attn_workspace.restype = sz
    lib.cfb_paged_attn.argtypes = [vp, i64, i64, C.POINTER(KvCache), vp, i64, i32, vp, vp, vp, i64, i64, vp, C.c_float,
                                   i32, i32, i32, i32, i32, vp, sz, vp]
    lib.cfb_paged_attn_error.argtypes = [vp, C.POINTER(i32)]
    # cfb_gdn_args as a GdnArgs by reference or as its packed bytes (PACK_GDN_ARGS)
    lib.cfb_gdn_step.argtypes = [vp, i32, vp]
    lib.cfb_gdn_chunk_workspace.argtypes = [i32, i32, i32]
    lib.cfb_gdn_chunk_workspace.restype = sz
    lib.cfb_gdn_chunk.argtypes = [vp, vp, i32, i32, vp, sz, vp]
    lib.cfb_gdn_chunk_error.argtypes = [vp, C.POINTER(i32)]
    return lib


def load(build_if_missing: bool = True):
    """The loaded libcfb.so (built in-tree with nvcc on first use if it is missing)."""
    global _lib
    with _lock:
        if _lib is None:
            if build_if_missing and not LIB_PATH.exists():
                from . import build as _build
                _build.build()
            if not LIB_PATH.exists():
                raise CfbError(f"{LIB_PATH} is missing; build it with `python -m chain_flow_b200.build`")
            _lib = _declare(C.CDLL(str(LIB_PATH)))
            if _lib.cfb_abi_version() != ABI_VERSION:
                raise CfbError("libcfb.so ABI version mismatch; rebuild it")
    return _lib


def check(status: int, what: str) -> None:
    if status != CFB_OK:
        lib = load(False)
        detail = lib.cfb_last_cuda_error().decode(errors="replace") if status == 4 else ""
        raise CfbError(f"{what}: {STATUS_NAMES.get(status, status)} {detail}".strip())


def stream_ptr(stream=None) -> int:
    import torch
    if stream is not None:
        return stream.cuda_stream
    # the raw handle: building a torch.cuda.Stream takes as long as a small launch
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def stream_of(device: int, what: str) -> int:
    """The current stream, for a launch over tensors of cuda device ``device``. That has to be the current
    device: a kernel launched on another would meet addresses that are not its own."""
    import torch
    current = torch._C._cuda_getDevice()
    if device != current:
        raise CfbError(f"{what}: the tensors are on cuda:{device}, the current device (or the given stream's) is cuda:{current}")
    return torch._C._cuda_getCurrentRawStream(current)


def require_cuda(t, name: str) -> None:
    if not t.is_cuda:
        raise CfbError(f"{name} must be a CUDA tensor: the chain_flow_b200 engine has no CPU path")


def int32(t):
    """t as a contiguous int32 tensor (itself if it is one)."""
    import torch
    return t if t.dtype == torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def int32_indices(t):
    """t as a contiguous int32 tensor; what 32 bits do not hold becomes their largest or smallest number, which is outside every
    range of tokens, pages and positions (to(int32) keeps the low bits, which may name one)."""
    import torch
    return int32(t.clamp(-1 << 31, (1 << 31) - 1) if t.dtype == torch.int64 else t)
