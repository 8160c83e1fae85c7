// cfb_types.cuh -- what the target-side kernels share: their element types and conversions, tensor-map
// copies, argument checks.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <atomic>
#include <cstdint>

#include "../../include/cfb.h"
#include "cfb_common.cuh"

namespace cfb {

enum DType : int { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2, DT_E4M3 = 3 };

CFB_DEV float to_float(float x) { return x; }
CFB_DEV float to_float(__half x) { return __half2float(x); }
CFB_DEV float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> CFB_DEV T from_float(float x);
template <> CFB_DEV float from_float<float>(float x) { return x; }
template <> CFB_DEV __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> CFB_DEV __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// two 16-bit elements <-> one 32-bit word
template <typename T> CFB_DEV float2 unpack16(uint32_t w);
template <> CFB_DEV float2 unpack16<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <> CFB_DEV float2 unpack16<__nv_bfloat16>(uint32_t w) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
template <typename T> CFB_DEV uint32_t pack16(float a, float b);
template <> CFB_DEV uint32_t pack16<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> CFB_DEV uint32_t pack16<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// element i of an array of dtype code `code` (DT_F32, DT_F16 or DT_BF16)
CFB_DEV float load_coded(const void* p, int code, long long i) {
  if (code == DT_F32) return static_cast<const float*>(p)[i];
  if (code == DT_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// ---- tensor-map copies into this CTA's shared memory (no multicast) -------------------------------
CFB_DEV void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
CFB_DEV void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
CFB_DEV void tma_load_5d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, int u, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
      :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(u), "r"(smem_u32(bar))
      : "memory");
}
CFB_DEV void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" :: "l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
// host: the driver's tensor-map encoder, or null
inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      f = nullptr;
    }
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }();
  return fn;
}

// host: the current device's SMs (0 where there is none: no launch will follow), and a kernel's dynamic
// shared memory allowed on it, both asked of the runtime once a device
inline int device_sms() {
  static std::atomic<int> sms[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  if (dev < 64 && (n = sms[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  if (dev < 64) sms[dev].store(n, std::memory_order_relaxed);
  return n;
}
template <auto Kernel>
inline cudaError_t allow_smem(int bytes) {
  static std::atomic<bool> done[64];
  int dev = 0;
  if (const cudaError_t e = cudaGetDevice(&dev)) return e;
  if (dev < 64 && done[dev].load(std::memory_order_relaxed)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done[dev].store(true, std::memory_order_relaxed);
  return e;
}
// host: base and row strides (in elements of `size` bytes) keep every row 16-byte aligned
inline bool rows_aligned(const void* p, int size, int64_t s0, int64_t s1) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (s0 * size) % 16 == 0 && (s1 * size) % 16 == 0;
}
// host: what every call over a cfb_kv_cache checks of it
inline cfb_status check_cache(const cfb_kv_cache* c) {
  if (!c || !c->k || !c->v || c->pages <= 0 || c->page_size <= 0 || c->kv_heads <= 0) return CFB_ERR_INVALID_ARG;
  if (c->dtype != DT_F16 && c->dtype != DT_BF16 && c->dtype != DT_E4M3) return CFB_ERR_UNSUPPORTED;
  if (c->dim != 64 && c->dim != 128 && c->dim != 256) return CFB_ERR_UNSUPPORTED;
  if ((c->dtype == DT_E4M3) != (c->k_scale != nullptr) || (c->dtype == DT_E4M3) != (c->v_scale != nullptr))
    return CFB_ERR_INVALID_ARG;
  const int size = c->dtype == DT_E4M3 ? 1 : 2;
  if (!rows_aligned(c->k, size, c->page_stride, c->head_stride) || !rows_aligned(c->v, size, c->slot_stride, 0))
    return CFB_ERR_INVALID_ARG;
  return CFB_OK;
}

}  // namespace cfb
