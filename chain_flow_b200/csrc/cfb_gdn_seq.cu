// cfb_gdn_seq.cu -- the gated delta rule over sequences (sm_100a): a target's prompts and its
// single-token decode steps, from and to the state slots the tree verify (cfb_gdn.cu) works on.
//
// Per value head hv (key head h = hv / (HV / H)), S the [V, K] fp32 state, K = 128:
//   g_t = -exp(A_log) softplus(a_t + dt_bias),  beta_t = sigmoid(b_t),
//   kn = k rsqrt(|k|^2 + 1e-6),  qn = q rsqrt(|q|^2 + 1e-6) scale,
//   S <- e^g S,  S <- S + beta (v - S kn) kn^T,  o = S qn.
#include <cuda_runtime.h>

#include "cfb_types.cuh"

using namespace cfb;

namespace {

constexpr int kK = 128;
constexpr float kSoftplusLinear = 20.f;   // softplus(x) = x above this
constexpr float kNormEps = 1e-6f;

CFB_DEV float softplus(float x) { return x <= kSoftplusLinear ? log1pf(expf(x)) : x; }
CFB_DEV float sigmoid(float x) { return 1.f / (1.f + expf(-x)); }

// ---- token by token ------------------------------------------------------------------------------
// One CTA per (request, value head, 32 value rows), no shared memory, no barrier. A value row's 128
// keys lie on 8 lanes, 16 a lane in four 16-byte pieces 32 columns apart, so that a warp's access
// covers 4 rows x 128 contiguous bytes of the state; a warp holds 8 rows, two per lane. A row's two
// sums close over its 8 lanes with 3 shuffles each. q, k, v and the gates of the next token are
// fetched while this one is worked on.
constexpr int kStepThreads = 128;
constexpr int kStepRows = 32;             // value rows a CTA

template <typename T>
struct TokenRegs {                        // one token's inputs as a lane holds them
  uint2 q[4], k[4];
  float v[2], a, b;
};

template <typename T>
CFB_DEV void fetch(const cfb_gdn_args& g, long long t, int h, int hv, int col, int row, TokenRegs<T>& r) {
  const T* k = static_cast<const T*>(g.k) + t * g.k_stride + (long long)h * kK + col;
  const T* q = static_cast<const T*>(g.q) + t * g.q_stride + (long long)h * kK + col;
  const T* v = static_cast<const T*>(g.v) + t * g.v_stride + (long long)hv * g.V + row;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    r.k[j] = __ldg(reinterpret_cast<const uint2*>(k + 32 * j));
    r.q[j] = __ldg(reinterpret_cast<const uint2*>(q + 32 * j));
  }
  r.v[0] = to_float(v[0]);
  r.v[1] = to_float(v[4]);
  r.a = load_coded(g.a, g.a_dtype, t * g.a_stride + hv);
  r.b = load_coded(g.b, g.b_dtype, t * g.b_stride + hv);
}
template <typename T>
CFB_DEV void widen(const uint2 (&w)[4], float (&x)[16]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 lo = unpack16<T>(w[j].x), hi = unpack16<T>(w[j].y);
    x[4 * j] = lo.x; x[4 * j + 1] = lo.y; x[4 * j + 2] = hi.x; x[4 * j + 3] = hi.y;
  }
}
CFB_DEV float sum8(float x) {             // over the 8 lanes of a row
#pragma unroll
  for (int off = 4; off; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

template <typename T>
__global__ void __launch_bounds__(kStepThreads) gdn_walk_kernel(const cfb_gdn_args g, const int32_t* cu, int total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int hv = blockIdx.y, b = blockIdx.z, h = hv / (g.HV / g.H);
  const int col = (lane & 7) * 4;
  const int row = blockIdx.x * kStepRows + warp * 8 + (lane >> 3);        // and row + 4
  int t0 = b, t1 = b + 1;
  if (cu) {
    t0 = min(max(cu[b], 0), total);
    t1 = min(max(cu[b + 1], t0), total);
  }
  const int from = g.init_slot[b], to = g.out_slot[b];
  const long long in_slot = ((long long)hv * g.V + row) * kK + col;
  float S[2][16];
  TokenRegs<T> r;
  if (t0 < t1) fetch<T>(g, t0, h, hv, col, row, r);
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const float fill = from < 0 ? 0.f : __int_as_float(0x7fc00000);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float4 x = make_float4(fill, fill, fill, fill);
      if (from >= 0 && from < g.slots)
        x = *reinterpret_cast<const float4*>(g.state_in + from * g.slot_stride + in_slot + p * 4 * kK + 32 * j);
      S[p][4 * j] = x.x; S[p][4 * j + 1] = x.y; S[p][4 * j + 2] = x.z; S[p][4 * j + 3] = x.w;
    }
  }
  const float rate = -expf(load_coded(g.A_log, g.A_log_dtype, hv));
  const float bias = load_coded(g.dt_bias, g.dt_bias_dtype, hv);
  for (int t = t0; t < t1; ++t) {
    float q[16], k[16];
    widen<T>(r.q, q);
    widen<T>(r.k, k);
    const float decay = expf(rate * softplus(r.a + bias)), beta = sigmoid(r.b);
    const float v[2] = {r.v[0], r.v[1]};
    if (t + 1 < t1) fetch<T>(g, t + 1, h, hv, col, row, r);
    float kk = 0.f, qq = 0.f, ks[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      kk = fmaf(k[i], k[i], kk);
      qq = fmaf(q[i], q[i], qq);
      ks[0] = fmaf(S[0][i], k[i], ks[0]);
      ks[1] = fmaf(S[1][i], k[i], ks[1]);
    }
    const float rk = rsqrtf(sum8(kk) + kNormEps), rq = rsqrtf(sum8(qq) + kNormEps) * g.scale;
    float o[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const float u = beta * (v[p] - decay * rk * sum8(ks[p])) * rk;
      o[p] = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        S[p][i] = fmaf(u, k[i], decay * S[p][i]);
        o[p] = fmaf(S[p][i], q[i], o[p]);
      }
      o[p] = sum8(o[p]) * rq;
    }
    if ((lane & 7) == 0) {
      T* out = static_cast<T*>(g.o) + t * g.o_stride + (long long)hv * g.V + row;
      out[0] = from_float<T>(o[0]);
      out[4] = from_float<T>(o[1]);
    }
  }
  if (to >= 0 && to < g.slots)
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<float4*>(g.state_out + to * g.slot_stride + in_slot + p * 4 * kK + 32 * j) =
            make_float4(S[p][4 * j], S[p][4 * j + 1], S[p][4 * j + 2], S[p][4 * j + 3]);
}

cfb_status check_gdn(const cfb_gdn_args* g, int B) {
  if (!g || B < 0) return CFB_ERR_INVALID_ARG;
  if (!g->A_log || !g->dt_bias || !g->a || !g->b || !g->q || !g->k || !g->v || !g->o || !g->state_in || !g->state_out ||
      !g->init_slot || !g->out_slot || g->H <= 0 || g->HV <= 0 || g->slots <= 0)
    return CFB_ERR_INVALID_ARG;
  for (int c : {g->A_log_dtype, g->dt_bias_dtype, g->a_dtype, g->b_dtype})
    if (c < DT_F32 || c > DT_BF16) return CFB_ERR_INVALID_ARG;
  if ((g->dtype != DT_F16 && g->dtype != DT_BF16) || g->K != kK || g->V <= 0 || g->V % 32 || g->HV % g->H ||
      g->HV > 65535 || B > 65535)
    return CFB_ERR_UNSUPPORTED;
  if (!rows_aligned(g->q, 2, g->q_stride, 0) || !rows_aligned(g->k, 2, g->k_stride, 0) ||
      !rows_aligned(g->v, 2, g->v_stride, 0) || !rows_aligned(g->o, 2, g->o_stride, 0) ||
      !rows_aligned(g->state_in, 4, g->slot_stride, 0) || !rows_aligned(g->state_out, 4, g->slot_stride, 0))
    return CFB_ERR_INVALID_ARG;
  if (g->slot_stride < (int64_t)g->HV * g->V * g->K) return CFB_ERR_INVALID_ARG;
  return CFB_OK;
}

void launch_walk(const cfb_gdn_args& g, const int32_t* cu, int total, int B, cudaStream_t st) {
  const dim3 grid((unsigned)(g.V / kStepRows), (unsigned)g.HV, (unsigned)B);
  if (g.dtype == DT_F16) gdn_walk_kernel<__half><<<grid, kStepThreads, 0, st>>>(g, cu, total);
  else gdn_walk_kernel<__nv_bfloat16><<<grid, kStepThreads, 0, st>>>(g, cu, total);
}

}  // namespace

extern "C" cfb_status cfb_gdn_step(const cfb_gdn_args* g, int B, void* stream) {
  if (B == 0 && g) return CFB_OK;
  if (const cfb_status s = check_gdn(g, B)) return s;
  launch_walk(*g, nullptr, B, B, static_cast<cudaStream_t>(stream));
  return cfb_launch_status("gdn_walk_kernel");
}

extern "C" size_t cfb_gdn_chunk_workspace(int T, int B, int HV) {
  (void)T; (void)B; (void)HV;
  return 256;
}

extern "C" cfb_status cfb_gdn_chunk(const cfb_gdn_args* g, const int32_t* cu, int T, int B, void* ws, size_t ws_bytes,
                                    void* stream) {
  if (B == 0 && g) return CFB_OK;
  if (const cfb_status s = check_gdn(g, B)) return s;
  if (T < 0 || !cu || !ws) return CFB_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(ws) & 255) || ws_bytes < cfb_gdn_chunk_workspace(T, B, g->HV)) return CFB_ERR_WORKSPACE;
  launch_walk(*g, cu, T, B, static_cast<cudaStream_t>(stream));
  return cfb_launch_status("gdn_walk_kernel");
}
