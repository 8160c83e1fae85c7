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
// one shuffle reduction for the maximum, one store. A group takes kRows rows of one token, neighbours in
// the order [k or v][head]: the token's slot is taken apart once, and all the rows' loads are in flight
// before the first is used. What is left is instructions: a first form, a row a group and tests element
// by element, spent 230 a row and ran at 59 % of the issue rate. So the maximum is taken of the bit
// patterns, two a register (magnitudes order like integers, and what is not finite is largest).
// Measured: 8192 tokens of 4 heads of 256, fp16 to e4m3, 16.4 us (51 MB: 3.1 TB/s, 0.47 of a copy's rate; a row
// a group 22.6); 20001 tokens of 8 heads of 128, e4m3 to bf16, 26.7 us (124 MB: 4.65 TB/s, 0.71; 43).
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

// where a slot lies: element offsets of its rows and scales, head 0; false if it is not in the pool
__device__ __forceinline__ bool locate(const cfb_kv_cache& c, long long slot, long long* row, long long* sc) {
  if (slot < 0 || slot >= (long long)c.pages * c.page_size) return false;
  long long page, off;
  if (slot <= 0x7fffffffll) {             // 32-bit division where the slot allows it
    const unsigned p = (unsigned)slot / (unsigned)c.page_size;
    page = p;
    off = (unsigned)slot - p * (unsigned)c.page_size;
  } else {
    page = slot / c.page_size;
    off = slot % c.page_size;
  }
  *row = page * c.page_stride + off * c.slot_stride;
  *sc = page * c.scale_page_stride + off * c.scale_slot_stride;
  return true;
}

// a group's token and its first row of the token's 2 kv_heads
struct Share { unsigned t; int x; bool live; };
template <int D>
__device__ __forceinline__ Share share_of(const cfb_kv_cache& c, unsigned shares) {
  const unsigned u = blockIdx.x * (kThreads / (D / 8)) + threadIdx.x / (D / 8);
  const unsigned per = (2u * (unsigned)c.kv_heads + kRows - 1) / kRows, t = u / per;
  return {t, (int)(u - t * per) * kRows, u < shares};
}

template <typename T, int D, bool QUANT>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const cfb_kv_cache c, const Rows in, const int64_t* slots,
                                                            unsigned shares) {
  constexpr int kLanes = D / 8;                        // lanes a row
  constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  const int lane = threadIdx.x % kLanes;
  const Share u = share_of<D>(c, shares);
  uint4 w[kRows];
  const long long slot = u.live ? __ldg(slots + u.t) : -1;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    w[i] = make_uint4(0, 0, 0, 0);
    const int x = u.x + i, h = x < c.kv_heads ? x : x - c.kv_heads;
    if (u.live && x < 2 * c.kv_heads) {
      const T* src = x < c.kv_heads ? static_cast<const T*>(in.k) + u.t * in.sk_t + h * in.sk_h
                                    : static_cast<const T*>(in.v) + u.t * in.sv_t + h * in.sv_h;
      w[i] = __ldg(reinterpret_cast<const uint4*>(src) + lane);
    }
  }
  long long row = 0, sc = 0;
  const bool in_pool = locate(c, slot, &row, &sc);
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int x = u.x + i, h = x < c.kv_heads ? x : x - c.kv_heads;
    const bool put = in_pool && x < 2 * c.kv_heads, key = x < c.kv_heads;
    const long long at = row + h * c.head_stride;
    if constexpr (!QUANT) {
      if (put) reinterpret_cast<uint4*>(static_cast<T*>(key ? c.k : c.v) + at)[lane] = w[i];
    } else {
      constexpr uint32_t kMag = 0x7fff7fffu;
      uint32_t top = __vmaxu2(__vmaxu2(w[i].x & kMag, w[i].y & kMag), __vmaxu2(w[i].z & kMag, w[i].w & kMag));
#pragma unroll
      for (int off = kLanes / 2; off; off >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, off, kLanes));
      top = max(top & 0xffffu, top >> 16);
      const bool bad = top >= kInf;
      const float m = fmaxf(unpack16<T>(top).x, kFloor), inv = kMaxCode / m;
      const auto four = [&](uint32_t a, uint32_t b) {
        const float2 f = unpack16<T>(a), g = unpack16<T>(b);
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f.x * inv, f.y * inv), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(g.x * inv, g.y * inv), __NV_SATFINITE, __NV_E4M3);
        return bad ? 0u : lo | hi << 16;
      };
      if (put) {
        reinterpret_cast<uint2*>(static_cast<uint8_t*>(key ? c.k : c.v) + at)[lane] =
            make_uint2(four(w[i].x, w[i].y), four(w[i].z, w[i].w));
        if (lane == 0) (key ? c.k_scale : c.v_scale)[sc + h * c.scale_head_stride] = bad ? __int_as_float(0x7fc00000) : m / kMaxCode;
      }
    }
  }
}

// C: stored type (uint8_t = e4m3), T: type read
template <typename C, typename T, int D>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const cfb_kv_cache c, const int64_t* slots, const Rows out,
                                                           unsigned shares) {
  constexpr int kLanes = D / 8;
  using Word = typename std::conditional<sizeof(C) == 1, uint2, uint4>::type;
  const int lane = threadIdx.x % kLanes;
  const Share u = share_of<D>(c, shares);
  if (!u.live) return;
  long long row = 0, sc = 0;
  const bool in_pool = locate(c, __ldg(slots + u.t), &row, &sc);
  Word w[kRows];
  float scale[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    w[i] = Word{};
    scale[i] = 0.f;
    const int x = u.x + i, h = x < c.kv_heads ? x : x - c.kv_heads;
    if (in_pool && x < 2 * c.kv_heads) {
      const bool key = x < c.kv_heads;
      w[i] = __ldg(reinterpret_cast<const Word*>(static_cast<const C*>(key ? c.k : c.v) + row + h * c.head_stride) + lane);
      if constexpr (sizeof(C) == 1) scale[i] = __ldg((key ? c.k_scale : c.v_scale) + sc + h * c.scale_head_stride);
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = u.x + i, h = r < c.kv_heads ? r : r - c.kv_heads;
    if (r >= 2 * c.kv_heads) return;
    T* const dst = r < c.kv_heads ? static_cast<T*>(out.k) + u.t * out.sk_t + h * out.sk_h
                                  : static_cast<T*>(out.v) + u.t * out.sv_t + h * out.sv_h;
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
      float4* d = reinterpret_cast<float4*>(dst) + 2 * lane;
      d[0] = make_float4(x[0], x[1], x[2], x[3]);
      d[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      reinterpret_cast<uint4*>(dst)[lane] =
          make_uint4(pack16<T>(x[0], x[1]), pack16<T>(x[2], x[3]), pack16<T>(x[4], x[5]), pack16<T>(x[6], x[7]));
    }
  }
}

// groups of a launch over T tokens
long long shares_of(const cfb_kv_cache& c, int T) { return (long long)T * ((2ll * c.kv_heads + kRows - 1) / kRows); }

template <typename T, bool QUANT>
void launch_write(const cfb_kv_cache& c, const Rows& in, const int64_t* slots, long long shares, cudaStream_t st) {
  const auto go = [&](auto kernel, int lanes) {
    const long long per = kThreads / lanes;
    kernel<<<(unsigned)((shares + per - 1) / per), kThreads, 0, st>>>(c, in, slots, (unsigned)shares);
  };
  if (c.dim == 64) go(kv_write_kernel<T, 64, QUANT>, 8);
  else if (c.dim == 128) go(kv_write_kernel<T, 128, QUANT>, 16);
  else go(kv_write_kernel<T, 256, QUANT>, 32);
}

template <typename C, typename T>
void launch_read(const cfb_kv_cache& c, const int64_t* slots, const Rows& out, long long shares, cudaStream_t st) {
  const auto go = [&](auto kernel, int lanes) {
    const long long per = kThreads / lanes;
    kernel<<<(unsigned)((shares + per - 1) / per), kThreads, 0, st>>>(c, slots, out, (unsigned)shares);
  };
  if (c.dim == 64) go(kv_read_kernel<C, T, 64>, 8);
  else if (c.dim == 128) go(kv_read_kernel<C, T, 128>, 16);
  else go(kv_read_kernel<C, T, 256>, 32);
}

template <typename C>
void launch_read_as(const cfb_kv_cache& c, const int64_t* slots, const Rows& out, long long shares, int dtype, cudaStream_t st) {
  if (dtype == DT_F32) launch_read<C, float>(c, slots, out, shares, st);
  else if (dtype == DT_F16) launch_read<C, __half>(c, slots, out, shares, st);
  else launch_read<C, __nv_bfloat16>(c, slots, out, shares, st);
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
  const long long shares = shares_of(*c, T);
  if (shares >= 1ll << 31) return CFB_ERR_UNSUPPORTED;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool quant = c->dtype == DT_E4M3;
  if (dtype == DT_F16 && quant) launch_write<__half, true>(*c, in, slots, shares, st);
  else if (dtype == DT_F16) launch_write<__half, false>(*c, in, slots, shares, st);
  else if (quant) launch_write<__nv_bfloat16, true>(*c, in, slots, shares, st);
  else launch_write<__nv_bfloat16, false>(*c, in, slots, shares, st);
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
  const long long shares = shares_of(*c, T);
  if (shares >= 1ll << 31) return CFB_ERR_UNSUPPORTED;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (c->dtype == DT_E4M3) launch_read_as<uint8_t>(*c, slots, out, shares, dtype, st);
  else if (c->dtype == DT_F16) launch_read_as<__half>(*c, slots, out, shares, dtype, st);
  else launch_read_as<__nv_bfloat16>(*c, slots, out, shares, dtype, st);
  return cfb_launch_status("kv_read_kernel");
}
