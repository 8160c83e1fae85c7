// cfb_kv.cu -- the paged key/value cache of a full-attention layer (sm_100a): rows written, with
// quantisation to e4m3 where the cache is e4m3, and read back.
//
// A row x of D = 64, 128 or 256 elements is quantised with one fp32 scale:
//   m = max(max_i |x_i|, 2^-24),   scale = m / 448,   code_i = e4m3(x_i * (448 / m)),
// so the largest element lands on e4m3's largest value (448); the floor 2^-24 keeps 448 / m finite
// for rows of zeros, where it costs nothing (every code is 0) and for rows below it an absolute
// error of at most 2^-42. The maximum, the scale and the product are fp32; the codes and a read
// row's elements are each rounded once, to nearest even.
//
// Bound: HBM (a step's rows) or launch latency (a decode step's). A row is independent of every
// other, so a group of D / 8 lanes holds a row in registers, 8 elements a lane: one pass over the data,
// one shuffle reduction for the maximum, one store. A group takes kRows rows, neighbours in the order
// [token][k or v][head], and has all their loads in flight before the first is used; a row's data is
// loaded beside its slot, not after it.
#include <cuda_runtime.h>
#include <cuda_fp8.h>
#include <type_traits>

#include "cfb_types.cuh"

using namespace cfb;

namespace {

constexpr int kThreads = 128;
constexpr int kRows = 4;
constexpr float kFloor = 5.9604644775390625e-8f;      // 2^-24
constexpr float kMaxCode = 448.f;

struct Rows {                             // rows [T, kv_heads, D] on the caller's side
  void* k; long long sk_t, sk_h;
  void* v; long long sv_t, sv_h;
};

// where the row of (slot, kv head) lies; false if the slot is not in the pool
__device__ __forceinline__ bool locate(const cfb_kv_cache& c, long long slot, int h, long long* row, long long* sc) {
  if (slot < 0 || slot >= (long long)c.pages * c.page_size) return false;
  long long page, off;
  if (slot <= 0x7fffffffll) {             // 32-bit division where the slot allows it
    page = (unsigned)slot / (unsigned)c.page_size;
    off = (unsigned)slot % (unsigned)c.page_size;
  } else {
    page = slot / c.page_size;
    off = slot % c.page_size;
  }
  *row = page * c.page_stride + h * c.head_stride + off * c.slot_stride;
  *sc = page * c.scale_page_stride + h * c.scale_head_stride + off * c.scale_slot_stride;
  return true;
}

// row r over [T][k or v][kv_heads]
__device__ __forceinline__ void row_of(const cfb_kv_cache& c, unsigned r, long long* t, int* which, int* h) {
  const unsigned per = 2u * (unsigned)c.kv_heads, q = r / per, x = r - q * per;
  *t = q;
  *which = x >= (unsigned)c.kv_heads;
  *h = (int)x - *which * c.kv_heads;
}

template <typename T, int D, bool QUANT>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const cfb_kv_cache c, const Rows in, const int64_t* slots,
                                                            unsigned rows) {
  constexpr int kLanes = D / 8;                        // lanes a row
  const unsigned r0 = (blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes) * kRows;
  const int lane = threadIdx.x % kLanes;
  uint4 w[kRows];
  long long slot[kRows];
  int which[kRows], h[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    w[i] = make_uint4(0, 0, 0, 0);
    slot[i] = -1;
    which[i] = h[i] = 0;
    if (r0 + i < rows) {
      long long t;
      row_of(c, r0 + i, &t, &which[i], &h[i]);
      slot[i] = __ldg(slots + t);
      const T* src = which[i] ? static_cast<const T*>(in.v) + t * in.sv_t + h[i] * in.sv_h
                              : static_cast<const T*>(in.k) + t * in.sk_t + h[i] * in.sk_h;
      w[i] = __ldg(reinterpret_cast<const uint4*>(src) + lane);
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    long long row = 0, sc = 0;
    const bool put = locate(c, slot[i], h[i], &row, &sc);
    if constexpr (!QUANT) {
      if (put) reinterpret_cast<uint4*>(static_cast<T*>(which[i] ? c.v : c.k) + row)[lane] = w[i];
    } else {
      float x[8];
      const uint32_t ws[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
      float m = 0.f;
      bool bad = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack16<T>(ws[e]);
        x[2 * e] = f.x;
        x[2 * e + 1] = f.y;
        m = fmaxf(m, fmaxf(fabsf(f.x), fabsf(f.y)));
        bad |= !isfinite(f.x) || !isfinite(f.y);
      }
      if (bad) m = INFINITY;                           // fmaxf drops NaN: an infinity carries it
#pragma unroll
      for (int off = kLanes / 2; off; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off, kLanes));
      bad = isinf(m);
      m = fmaxf(m, kFloor);
      const float inv = kMaxCode / m;
      uint2 q = make_uint2(0, 0);
      if (!bad) {
        uint32_t p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          p[e] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * e] * inv, x[2 * e + 1] * inv), __NV_SATFINITE, __NV_E4M3);
        q = make_uint2(p[0] | p[1] << 16, p[2] | p[3] << 16);
      }
      if (put) {
        reinterpret_cast<uint2*>(static_cast<uint8_t*>(which[i] ? c.v : c.k) + row)[lane] = q;
        if (lane == 0) (which[i] ? c.v_scale : c.k_scale)[sc] = bad ? __int_as_float(0x7fc00000) : m / kMaxCode;
      }
    }
  }
}

// C: stored type (uint8_t = e4m3), T: type read
template <typename C, typename T, int D>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const cfb_kv_cache c, const int64_t* slots, const Rows out,
                                                           unsigned rows) {
  constexpr int kLanes = D / 8;
  using Word = typename std::conditional<sizeof(C) == 1, uint2, uint4>::type;
  const unsigned r0 = (blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes) * kRows;
  const int lane = threadIdx.x % kLanes;
  Word w[kRows];
  float scale[kRows];
  T* dst[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    w[i] = Word{};
    scale[i] = 0.f;
    dst[i] = nullptr;
    if (r0 + i >= rows) continue;
    long long t, row, sc;
    int which, h;
    row_of(c, r0 + i, &t, &which, &h);
    dst[i] = which ? static_cast<T*>(out.v) + t * out.sv_t + h * out.sv_h : static_cast<T*>(out.k) + t * out.sk_t + h * out.sk_h;
    if (locate(c, __ldg(slots + t), h, &row, &sc)) {
      w[i] = __ldg(reinterpret_cast<const Word*>(static_cast<const C*>(which ? c.v : c.k) + row) + lane);
      if constexpr (sizeof(C) == 1) scale[i] = __ldg((which ? c.v_scale : c.k_scale) + sc);
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    if (!dst[i]) continue;
    float x[8];
    if constexpr (sizeof(C) == 1) {
      const uint32_t ws[2] = {w[i].x, w[i].y};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const __half2 f = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(ws[e / 2] >> (16 * (e & 1))), __NV_E4M3));
        x[2 * e] = __low2float(f) * scale[i];
        x[2 * e + 1] = __high2float(f) * scale[i];
      }
    } else {
      const uint32_t ws[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack16<C>(ws[e]);
        x[2 * e] = f.x;
        x[2 * e + 1] = f.y;
      }
    }
    if constexpr (sizeof(T) == 4) {
      float4* d = reinterpret_cast<float4*>(dst[i]) + 2 * lane;
      d[0] = make_float4(x[0], x[1], x[2], x[3]);
      d[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      reinterpret_cast<uint4*>(dst[i])[lane] =
          make_uint4(pack16<T>(x[0], x[1]), pack16<T>(x[2], x[3]), pack16<T>(x[4], x[5]), pack16<T>(x[6], x[7]));
    }
  }
}

template <typename T, bool QUANT>
void launch_write(const cfb_kv_cache& c, const Rows& in, const int64_t* slots, long long rows, cudaStream_t st) {
  const auto go = [&](auto kernel, int lanes) {
    const long long per = kThreads / lanes * kRows;
    kernel<<<(unsigned)((rows + per - 1) / per), kThreads, 0, st>>>(c, in, slots, (unsigned)rows);
  };
  if (c.dim == 64) go(kv_write_kernel<T, 64, QUANT>, 8);
  else if (c.dim == 128) go(kv_write_kernel<T, 128, QUANT>, 16);
  else go(kv_write_kernel<T, 256, QUANT>, 32);
}

template <typename C, typename T>
void launch_read(const cfb_kv_cache& c, const int64_t* slots, const Rows& out, long long rows, cudaStream_t st) {
  const auto go = [&](auto kernel, int lanes) {
    const long long per = kThreads / lanes * kRows;
    kernel<<<(unsigned)((rows + per - 1) / per), kThreads, 0, st>>>(c, slots, out, (unsigned)rows);
  };
  if (c.dim == 64) go(kv_read_kernel<C, T, 64>, 8);
  else if (c.dim == 128) go(kv_read_kernel<C, T, 128>, 16);
  else go(kv_read_kernel<C, T, 256>, 32);
}

template <typename C>
void launch_read_as(const cfb_kv_cache& c, const int64_t* slots, const Rows& out, long long rows, int dtype, cudaStream_t st) {
  if (dtype == DT_F32) launch_read<C, float>(c, slots, out, rows, st);
  else if (dtype == DT_F16) launch_read<C, __half>(c, slots, out, rows, st);
  else launch_read<C, __nv_bfloat16>(c, slots, out, rows, st);
}

}  // namespace

extern "C" cfb_status cfb_kv_write(const cfb_kv_cache* c, const void* key, int64_t sk_t, int64_t sk_h, const void* value,
                                   int64_t sv_t, int64_t sv_h, int dtype, const int64_t* slots, int T, void* stream) {
  if (const cfb_status s = check_cache(c)) return s;
  if (T < 0 || (T > 0 && (!key || !value || !slots))) return CFB_ERR_INVALID_ARG;
  if ((dtype != DT_F16 && dtype != DT_BF16) || (c->dtype != DT_E4M3 && c->dtype != dtype)) return CFB_ERR_UNSUPPORTED;
  if (!rows_aligned(key, 2, sk_t, sk_h) || !rows_aligned(value, 2, sv_t, sv_h)) return CFB_ERR_INVALID_ARG;
  if (T == 0) return CFB_OK;
  const Rows in{const_cast<void*>(key), sk_t, sk_h, const_cast<void*>(value), sv_t, sv_h};
  const long long rows = 2ll * T * c->kv_heads;
  if (rows >= 1ll << 31) return CFB_ERR_UNSUPPORTED;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool quant = c->dtype == DT_E4M3;
  if (dtype == DT_F16 && quant) launch_write<__half, true>(*c, in, slots, rows, st);
  else if (dtype == DT_F16) launch_write<__half, false>(*c, in, slots, rows, st);
  else if (quant) launch_write<__nv_bfloat16, true>(*c, in, slots, rows, st);
  else launch_write<__nv_bfloat16, false>(*c, in, slots, rows, st);
  return cfb_launch_status("kv_write_kernel");
}

extern "C" cfb_status cfb_kv_read(const cfb_kv_cache* c, const int64_t* slots, int T, void* key, int64_t sk_t,
                                  int64_t sk_h, void* value, int64_t sv_t, int64_t sv_h, int dtype, void* stream) {
  if (const cfb_status s = check_cache(c)) return s;
  if (T < 0 || (T > 0 && (!key || !value || !slots))) return CFB_ERR_INVALID_ARG;
  if (dtype < DT_F32 || dtype > DT_BF16) return CFB_ERR_UNSUPPORTED;
  const int size = dtype == DT_F32 ? 4 : 2;
  if (!rows_aligned(key, size, sk_t, sk_h) || !rows_aligned(value, size, sv_t, sv_h)) return CFB_ERR_INVALID_ARG;
  if (T == 0) return CFB_OK;
  const Rows out{key, sk_t, sk_h, value, sv_t, sv_h};
  const long long rows = 2ll * T * c->kv_heads;
  if (rows >= 1ll << 31) return CFB_ERR_UNSUPPORTED;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (c->dtype == DT_E4M3) launch_read_as<uint8_t>(*c, slots, out, rows, dtype, st);
  else if (c->dtype == DT_F16) launch_read_as<__half>(*c, slots, out, rows, dtype, st);
  else launch_read_as<__nv_bfloat16>(*c, slots, out, rows, dtype, st);
  return cfb_launch_status("kv_read_kernel");
}
