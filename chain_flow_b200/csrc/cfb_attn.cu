// cfb_attn.cu -- attention of new tokens over a paged key/value cache (sm_100a), with its
// log-sum-exp: prompt chunks and single tokens (causal), and the prefix half of a tree step.
//
// For query row i of a request with n new tokens and L cached positions, over the allowed positions
// j (j < L, or j <= L - n + i):
//   s_j = scale q_i . k_j,  m = max s_j,  l = sum exp(s_j - m),  o_i = sum exp(s_j - m) v_j / l,
//   lse_i = m + log l.
// One warp per (query row, head), lanes over the head dim, positions one by one with the running
// maximum and sum; positions that are not allowed are never read.
#include <cuda_runtime.h>
#include <cuda_fp8.h>

#include "cfb_types.cuh"

using namespace cfb;

namespace {

constexpr int kWarps = 8;

struct AttnArgs {
  const void* q; long long sq_t, sq_h;
  cfb_kv_cache c;
  const int32_t* table; long long st; int width;
  const int32_t* kv_len;
  const int32_t* cu_q;
  void* o; long long so_t, so_h;
  float* lse;
  float scale;
  int T, B, H, causal;
};

template <typename C, int E>
CFB_DEV void load_elems(const C* p, float (&x)[E]) {
#pragma unroll
  for (int i = 0; i < E; ++i) {
    if constexpr (sizeof(C) == 1) x[i] = __half2float(__half(__nv_cvt_fp8_to_halfraw(p[i], __NV_E4M3)));
    else x[i] = to_float(p[i]);
  }
}

template <typename T, typename C, int D>
__global__ void __launch_bounds__(kWarps * 32) attn_rows_kernel(const AttnArgs A) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const long long task = (long long)blockIdx.x * kWarps + threadIdx.x / 32;
  if (task >= (long long)A.T * A.H) return;
  const int t = (int)(task / A.H), h = (int)(task - (long long)t * A.H);
  // the request that owns row t: the last b with cu_q[b] <= t
  int lo = 0, hi = A.B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (A.cu_q[mid] <= t) lo = mid; else hi = mid;
  }
  const int first = A.cu_q[lo], end = A.cu_q[lo + 1];
  if (t < first || t >= end) return;
  const long long cap = (long long)A.width * A.c.page_size;
  long long L = max(A.kv_len[lo], 0);
  const bool over = L > cap;
  L = over ? cap : L;
  const long long stop = A.causal ? min(L, L - (end - first) + (t - first) + 1) : L;
  const int kh = h / (A.H / A.c.kv_heads);
  float q[E], acc[E];
  load_elems(static_cast<const T*>(A.q) + t * A.sq_t + h * A.sq_h + lane * E, q);
#pragma unroll
  for (int i = 0; i < E; ++i) acc[i] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (long long j = 0; j < stop; ++j) {
    const int page = A.table[lo * A.st + j / A.c.page_size];
    const int off = (int)(j % A.c.page_size);
    float s = __int_as_float(0x7fc00000), vs = 1.f;
    float v[E];
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = 0.f;
    if (page >= 0 && page < A.c.pages) {
      const long long row = page * A.c.page_stride + kh * A.c.head_stride + off * A.c.slot_stride + lane * E;
      float k[E];
      load_elems(static_cast<const C*>(A.c.k) + row, k);
      load_elems(static_cast<const C*>(A.c.v) + row, v);
      s = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) s = fmaf(q[i], k[i], s);
#pragma unroll
      for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      s *= A.scale;
      if constexpr (sizeof(C) == 1) {
        const long long sc = page * A.c.scale_page_stride + kh * A.c.scale_head_stride + off * A.c.scale_slot_stride;
        s *= A.c.k_scale[sc];
        vs = A.c.v_scale[sc];
      }
    }
    const float top = fmaxf(m, s);
    const float keep = m == -INFINITY ? 0.f : expf(m - top), p = s == -INFINITY ? 0.f : expf(s - top);
    l = l * keep + p;
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = acc[i] * keep + p * vs * v[i];
    m = top;
  }
  if (over) l = __int_as_float(0x7fc00000);
  T* o = static_cast<T*>(A.o) + t * A.so_t + h * A.so_h + lane * E;
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = from_float<T>(l == 0.f ? 0.f : acc[i] / l);
  if (A.lse && lane == 0) A.lse[(long long)h * A.T + t] = l == 0.f ? -INFINITY : m + logf(l);
}

template <typename T, typename C>
void launch(const AttnArgs& A, cudaStream_t st) {
  const unsigned grid = (unsigned)(((long long)A.T * A.H + kWarps - 1) / kWarps);
  if (A.c.dim == 64) attn_rows_kernel<T, C, 64><<<grid, kWarps * 32, 0, st>>>(A);
  else if (A.c.dim == 128) attn_rows_kernel<T, C, 128><<<grid, kWarps * 32, 0, st>>>(A);
  else attn_rows_kernel<T, C, 256><<<grid, kWarps * 32, 0, st>>>(A);
}

}  // namespace

extern "C" size_t cfb_paged_attn_workspace(int H, int kv_heads, int dim) {
  (void)H; (void)kv_heads; (void)dim;
  return 256;
}

extern "C" cfb_status cfb_paged_attn(const void* q, int64_t sq_t, int64_t sq_h, const cfb_kv_cache* c,
                                     const int32_t* page_table, int64_t table_stride, int table_width,
                                     const int32_t* kv_len, const int32_t* cu_q, void* o, int64_t so_t, int64_t so_h,
                                     float* lse, float scale, int T, int B, int H, int causal, int dtype, void* ws,
                                     size_t ws_bytes, void* stream) {
  if (const cfb_status s = check_cache(c)) return s;
  if (T < 0 || B < 0 || H <= 0 || table_width < 0 || table_stride < table_width) return CFB_ERR_INVALID_ARG;
  if ((dtype != DT_F16 && dtype != DT_BF16) || (c->dtype != DT_E4M3 && c->dtype != dtype)) return CFB_ERR_UNSUPPORTED;
  if (H % c->kv_heads || H / c->kv_heads > 128) return CFB_ERR_UNSUPPORTED;
  if (T == 0 || B == 0) return CFB_OK;
  if (!q || !o || !kv_len || !cu_q || (table_width && !page_table) || !ws) return CFB_ERR_INVALID_ARG;
  if (!rows_aligned(q, 2, sq_t, sq_h) || !rows_aligned(o, 2, so_t, so_h)) return CFB_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(ws) & 255) || ws_bytes < cfb_paged_attn_workspace(H, c->kv_heads, c->dim))
    return CFB_ERR_WORKSPACE;
  const AttnArgs A{q, sq_t, sq_h, *c, page_table, table_stride, table_width, kv_len, cu_q, o, so_t, so_h, lse, scale,
                   T, B, H, causal};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == DT_F16) c->dtype == DT_E4M3 ? launch<__half, uint8_t>(A, st) : launch<__half, __half>(A, st);
  else c->dtype == DT_E4M3 ? launch<__nv_bfloat16, uint8_t>(A, st) : launch<__nv_bfloat16, __nv_bfloat16>(A, st);
  return cfb_launch_status("attn_rows_kernel");
}
