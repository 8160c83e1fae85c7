// cfb_gdn_seq.cu -- the gated delta rule over sequences (sm_100a): a target's prompts and its
// single-token decode steps, from and to the state slots the tree verify (cfb_gdn.cu) works on.
//
// Per value head hv (key head h = hv / (HV / H)), S the [V, K] fp32 state, K = 128:
//   g_t = -exp(A_log) softplus(a_t + dt_bias),  beta_t = sigmoid(b_t),
//   kn = k rsqrt(|k|^2 + 1e-6),  qn = q rsqrt(|q|^2 + 1e-6) scale,
//   S <- e^g S,  S <- S + beta (v - S kn) kn^T,  o = S qn.
#include <cuda_runtime.h>
#include <type_traits>

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

// ---- chunk by chunk ------------------------------------------------------------------------------
// A chunk of kC tokens in matrix form, S0 the state before it, G_i = sum_{j<=i} g_j, r_i and rq_i the
// reciprocal norms of k_i and q_i:
//   (I + A) U = beta (v - e^G r (S0 k)),   A_ij = beta_i e^{G_i-G_j} r_i r_j (k_i . k_j)  (j < i),
//   o_i = e^{G_i} scale rq_i (S0 q_i) + sum_{j<=i} P_ij u_j,   P_ij = scale rq_i e^{G_i-G_j} r_j (k_j . q_i),
//   S  = e^{G_C} S0 + sum_j (e^{G_C-G_j} r_j u_j) k_j^T.
// gdn_prep_kernel forms T = (I + A)^-1 and P of every chunk at once; gdn_scan_kernel then walks a
// request's chunks with three products a chunk that depend on one another.
//
// Precision. The state is fp32 and has to stay so over thousands of chunks, so no product rounds an
// operand to fewer than 22 bits: k and q are exact in tf32 as they are (their norms are applied
// afterwards, in fp32), and S, U and T are split into two tf32 terms, x = hi + lo, lo * lo dropped
// (relative error about 2^-22). Exponents of differences G_i - G_j are of sums kept in 64 bits: in 32,
// a strong decay's G of a few hundred would cost 1e-5. S is updated by one fp32 fma an element from a
// product that starts at zero, because sums carried through the tensor cores lose a little towards zero
// with every step. o is rounded to 16 bits, so its own products take hi terms only over bf16 (11 bits
// against its 8), and both terms over fp16.
//
// Why mma.sync and not tcgen05: the scan is a chain over a head's chunks, and what bounds it is the
// latency of one link, not throughput. With 16 value rows a warp, the state lives in the warp's
// registers in the accumulator layout, which, with the summed index permuted (2t, 2t + 1 for t, t + 4;
// the other operand is read as pairs of neighbours anyway), is the first operand's layout too: S feeds
// S k, that feeds T, U feeds the update, without a trip through shared or tensor memory and without
// a barrier between warps.
constexpr int kC = 32, kBlocks = kC / 8;                       // tokens a chunk; blocks of 8
constexpr int kPairs = kBlocks * (kBlocks + 1) / 2;            // lower-triangular 8 x 8 blocks
// What the scan reads of a chunk and value head: T and P as the second operand of its products, a
// float4 (two neighbours' hi, their lo) a lane for each lower-triangular block, then per token beta,
// beta e^G r, e^{G_C-G} r, e^G scale rq, then e^{G_C}.
constexpr int kFragFloats = kPairs * 32 * 4;
constexpr int kPrepFloats = 2 * kFragFloats + 4 * kC + 4;
constexpr int kRowHalves = kK + 8;                             // padded row of a staged K or Q tile

CFB_DEV float tf32(float x) {
  uint32_t y;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(y) : "f"(x));
  return __uint_as_float(y);
}
CFB_DEV void split(float x, float& hi, float& lo) {
  hi = tf32(x);
  lo = tf32(x - hi);
}
CFB_DEV void mma_tf32(float (&d)[4], const float (&a)[4], float b0, float b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])), "r"(__float_as_uint(a[3])),
        "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}
// 16-bit operands, fp32 sums (products of two 16-bit numbers are exact)
template <typename T> CFB_DEV void mma_16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> CFB_DEV void mma_16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> CFB_DEV void mma_16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
CFB_DEV void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
CFB_DEV void ldmatrix4_t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
CFB_DEV uint32_t transpose8(uint32_t x) {                      // an 8 x 8 matrix of 16-bit elements
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
CFB_DEV void cp_async16z(uint32_t dst, const void* src, bool in) {       // 16 bytes, or zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}

// Chunk x of the launch: request b's chunks are numbered from cu[b] / kC + b (requests cannot run
// into one another so: ceil(n / kC) <= (cu + n) / kC - cu / kC + 1). False if x is no chunk.
CFB_DEV bool chunk_of(const int32_t* cu, int total, int B, int x, int* b, int* t0, int* n) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (min(max(cu[mid], 0), total) / kC + mid <= x) lo = mid; else hi = mid;
  }
  const int first = min(max(cu[lo], 0), total), end = min(max(cu[lo + 1], first), total);
  *b = lo;
  *t0 = first + (x - (first / kC + lo)) * kC;
  *n = min(kC, end - *t0);
  return *t0 >= first && *n > 0;
}

// One CTA of two warps per (chunk, value head): warp 0 forms K K^T and T, warp 1 Q K^T and P. Rows of
// tokens that the chunk does not have are zeros with beta = 0 and no decay.
template <typename T>
__global__ void __launch_bounds__(64) gdn_prep_kernel(const cfb_gdn_args g, const int32_t* cu, int total, int B, float* ws) {
  __shared__ __align__(16) T sk[kC][kRowHalves];
  __shared__ __align__(16) T sq[kC][kRowHalves];
  __shared__ __align__(16) float sa[kC][kC + 4];               // A, then T
  __shared__ float sp[kC][kC + 1];                             // q . k
  __shared__ double sG[kC];
  __shared__ float sr[kC], srq[kC];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hv = blockIdx.y, h = hv / (g.HV / g.H);
  int b, t0, n;
  if (!chunk_of(cu, total, B, blockIdx.x, &b, &t0, &n)) return;
  for (int x = threadIdx.x; x < kC * 16 * 2; x += 64) {
    const int row = (x >> 4) % kC, c = x & 15;
    const bool is_q = x >= kC * 16;
    const T* src = is_q ? static_cast<const T*>(g.q) + (long long)(t0 + row) * g.q_stride : static_cast<const T*>(g.k) + (long long)(t0 + row) * g.k_stride;
    uint4 y = make_uint4(0, 0, 0, 0);
    if (row < n) y = __ldg(reinterpret_cast<const uint4*>(src + (long long)h * kK) + c);
    *reinterpret_cast<uint4*>(is_q ? &sq[row][c * 8] : &sk[row][c * 8]) = y;
  }
  float beta = 0.f, decay = 0.f;
  if (lane < n) {
    const float rate = -expf(load_coded(g.A_log, g.A_log_dtype, hv));
    const float bias = load_coded(g.dt_bias, g.dt_bias_dtype, hv);
    decay = rate * softplus(load_coded(g.a, g.a_dtype, (long long)(t0 + lane) * g.a_stride + hv) + bias);
    beta = sigmoid(load_coded(g.b, g.b_dtype, (long long)(t0 + lane) * g.b_stride + hv));
  }
  // G by token (a decay of e^-1e6 is 0 all the same; sums and differences stay numbers)
  double G = decay < -1e6f ? -1e6 : (double)decay;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, G, off);
    if (lane >= off) G += y;
  }
  const double G_end = __shfl_sync(0xffffffffu, G, 31);
  __syncthreads();
  // norms: warp 0 of k, warp 1 of q, a lane a row
  {
    const T* row = warp ? sq[lane] : sk[lane];
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      const uint4 y = *reinterpret_cast<const uint4*>(row + 8 * c);
      const uint32_t ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack16<T>(ys[e]);
        sum = fmaf(f.x, f.x, sum);
        sum = fmaf(f.y, f.y, sum);
      }
    }
    (warp ? srq : sr)[lane] = rsqrtf(sum + kNormEps);
    if (warp == 0) sG[lane] = G;
  }
  // X K^T, X = K (warp 0) or Q (warp 1)
  const int gid = lane >> 2, t = lane & 3;
#pragma unroll
  for (int mt = 0; mt < 2; ++mt) {
    float acc[kBlocks][4] = {};
    const uint32_t a_at = smem_u32(&(warp ? sq : sk)[mt * 16 + (lane & 15)][(lane >> 4) * 8]);
    const uint32_t b_at = smem_u32(&sk[lane][0]);
#pragma unroll
    for (int k = 0; k < kK / 16; ++k) {
      uint32_t a[4], b0[4], b1[4];
      ldmatrix4(a, a_at + k * 32);
      ldmatrix4(b0, b_at + k * 32);
      ldmatrix4(b1, b_at + k * 32 + 16);
#pragma unroll
      for (int nt = 0; nt < kBlocks; ++nt) mma_16<T>(acc[nt], a, b0[nt], b1[nt]);
    }
#pragma unroll
    for (int nt = 0; nt < kBlocks; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = mt * 16 + gid + (e >> 1) * 8, j = nt * 8 + 2 * t + (e & 1);
        if (warp) sp[i][j] = acc[nt][e];
        else sa[i][j] = acc[nt][e];
      }
  }
  __syncthreads();
  float* const out = ws + ((long long)blockIdx.x * g.HV + hv) * kPrepFloats;
  const auto put = [&](float4* dst, auto value) {              // the lower-triangular blocks, as the scan reads them
#pragma unroll
    for (int nt = 0; nt < kBlocks; ++nt)
#pragma unroll
      for (int jb = 0; jb <= nt; ++jb) {
        const int i = nt * 8 + gid, j = jb * 8 + 2 * t;
        float4 f;
        split(j <= i ? value(i, j) : 0.f, f.x, f.z);
        split(j + 1 <= i ? value(i, j + 1) : 0.f, f.y, f.w);
        dst[(nt * (nt + 1) / 2 + jb) * 32 + lane] = f;
      }
  };
  if (warp == 0) {
    // A, a lane a column; then T column by column: x_i = [i = j] - sum_{m<i} A_im x_m
    const double Gj = sG[lane];
    const float rj = sr[lane];
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      const float bi = __shfl_sync(0xffffffffu, beta, i);
      sa[i][lane] = lane < i ? bi * sr[i] * rj * expf((float)(sG[i] - Gj)) * sa[i][lane] : 0.f;
    }
    __syncwarp();
    float x[kC];
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      float sum[4] = {i == lane ? 1.f : 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int m = 0; m < i; m += 4) {
        const float4 y = *reinterpret_cast<const float4*>(&sa[i][m]);
        sum[0] = fmaf(-y.x, x[m], sum[0]);
        if (m + 1 < i) sum[1] = fmaf(-y.y, x[m + 1], sum[1]);
        if (m + 2 < i) sum[2] = fmaf(-y.z, x[m + 2], sum[2]);
        if (m + 3 < i) sum[3] = fmaf(-y.w, x[m + 3], sum[3]);
      }
      x[i] = i < lane ? 0.f : (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kC; ++i) sa[i][lane] = x[i];
    __syncwarp();
    put(reinterpret_cast<float4*>(out), [&](int i, int j) { return sa[i][j]; });
  } else {
    put(reinterpret_cast<float4*>(out + kFragFloats),
        [&](int i, int j) { return g.scale * srq[i] * sr[j] * expf((float)(sG[i] - sG[j])) * sp[i][j]; });
    float* const v = out + 2 * kFragFloats;
    const float eG = expf((float)G);
    v[lane] = beta;
    v[kC + lane] = beta * eG * sr[lane];
    v[2 * kC + lane] = expf((float)(G_end - G)) * sr[lane];
    v[3 * kC + lane] = eG * g.scale * srq[lane];
    if (lane == 0) v[4 * kC] = expf((float)G_end);
  }
}

// One CTA per (32 value rows, value head, request): 2 * KS warps, a warp 16 value rows and 128 / KS of
// the state's columns. KS = 2 halves the longest chain of a chunk at the price of an exchange of the
// partial sums of S k and S q; it is taken where KS = 1 would leave SM quarters without a warp.
constexpr int kScanRows = 32, kScanStages = 3;
struct ScanStage {
  static constexpr int kKV = kC * kRowHalves * 2, kVPitch = kScanRows * 2 + 16;
  static constexpr int off_q = kKV, off_v = 2 * kKV, off_prep = off_v + kC * kVPitch, bytes = off_prep + kPrepFloats * 4;
};
static_assert(ScanStage::off_prep % 16 == 0 && ScanStage::bytes % 16 == 0 && kPrepFloats % 4 == 0, "16-byte copies");

template <typename T, int KS>
__global__ void __launch_bounds__(64 * KS) gdn_scan_kernel(const cfb_gdn_args g, const int32_t* cu, int total, const float* ws) {
  constexpr int NJ = 16 / KS;                                  // 8-column blocks of the state a warp holds
  constexpr bool kFine = std::is_same<T, __half>::value;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float2 sx[KS == 2 ? 2 : 1][2][kBlocks][2][32];    // partial sums that the two halves exchange
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, t = lane & 3;
  const int vt = warp / KS, ks = warp % KS;                    // value tile, column half
  const int hv = blockIdx.y, b = blockIdx.z, h = hv / (g.HV / g.H), v0 = blockIdx.x * kScanRows;
  const int first = min(max(cu[b], 0), total), end = min(max(cu[b + 1], first), total);
  const int chunks = (end - first + kC - 1) / kC;
  const float* const prep = ws + ((long long)(first / kC + b) * g.HV + hv) * kPrepFloats;
  const uint32_t sm = smem_u32(smem);

  const auto load = [&](int c) {
    const uint32_t at = sm + (c % kScanStages) * ScanStage::bytes;
    const int t0 = first + c * kC, n = min(kC, end - t0);
    const T* k = static_cast<const T*>(g.k) + (long long)t0 * g.k_stride + (long long)h * kK;
    const T* q = static_cast<const T*>(g.q) + (long long)t0 * g.q_stride + (long long)h * kK;
    const T* v = static_cast<const T*>(g.v) + (long long)t0 * g.v_stride + (long long)hv * g.V + v0;
    for (int x = threadIdx.x; x < kC * 16; x += 64 * KS) {
      const int row = x >> 4, p = x & 15;
      const bool in = row < n;
      cp_async16z(at + row * (kRowHalves * 2) + p * 16, k + (in ? (long long)row * g.k_stride : 0) + p * 8, in);
      cp_async16z(at + ScanStage::off_q + row * (kRowHalves * 2) + p * 16, q + (in ? (long long)row * g.q_stride : 0) + p * 8, in);
    }
    for (int x = threadIdx.x; x < kC * kScanRows / 8; x += 64 * KS) {
      const int row = x / (kScanRows / 8), p = x % (kScanRows / 8);
      const bool in = row < n;
      cp_async16z(at + ScanStage::off_v + row * ScanStage::kVPitch + p * 16, v + (in ? (long long)row * g.v_stride : 0) + p * 8, in);
    }
    const float* src = prep + (long long)c * g.HV * kPrepFloats;
    for (int x = threadIdx.x; x < kPrepFloats / 4; x += 64 * KS) cp_async16z(at + ScanStage::off_prep + x * 16, src + x * 4, true);
  };

#pragma unroll
  for (int c = 0; c < kScanStages - 1; ++c) {
    if (c < chunks) load(c);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // the state: lane (gid, t) holds rows gid and gid + 8, columns 2t and 2t + 1 of every 8-column block
  float S[NJ][4];
  {
    const int from = g.init_slot[b];
    const float fill = from < 0 ? 0.f : __int_as_float(0x7fc00000);
    const bool read = from >= 0 && from < g.slots;
    const float* src = g.state_in + (read ? from * g.slot_stride : 0) + ((long long)hv * g.V + v0 + vt * 16 + gid) * kK + ks * NJ * 8 + 2 * t;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      float2 x = make_float2(fill, fill), y = x;
      if (read) {
        x = *reinterpret_cast<const float2*>(src + 8 * j);
        y = *reinterpret_cast<const float2*>(src + 8 * kK + 8 * j);
      }
      S[j][0] = x.x; S[j][1] = x.y; S[j][2] = y.x; S[j][3] = y.y;
    }
  }
  // an accumulator as the first operand of the next product (see above)
  const auto operand = [](const float (&s)[4], float (&hi)[4], float (&lo)[4]) {
    split(s[0], hi[0], lo[0]);
    split(s[2], hi[1], lo[1]);
    split(s[1], hi[2], lo[2]);
    split(s[3], hi[3], lo[3]);
  };

  for (int c = 0; c < chunks; ++c) {
    asm volatile("cp.async.wait_group %0;" :: "n"(kScanStages - 2) : "memory");
    __syncthreads();
    if (c + kScanStages - 1 < chunks) load(c + kScanStages - 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    const uint32_t at = sm + (c % kScanStages) * ScanStage::bytes;
    const uint8_t* const st = smem + (c % kScanStages) * ScanStage::bytes;
    const float4* const tf = reinterpret_cast<const float4*>(st + ScanStage::off_prep) + lane;
    const float4* const pf = tf + kFragFloats / 4;
    const float* const vec = reinterpret_cast<const float*>(st + ScanStage::off_prep) + 2 * kFragFloats;

    // S k and S q of the chunk's tokens
    float R[kBlocks][4] = {}, Rl[kBlocks][4] = {}, O[kBlocks][4] = {};
    const uint32_t row_at = at + lane * (kRowHalves * 2) + ks * NJ * 16;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      float hi[4], lo[4];
      operand(S[j], hi, lo);
      uint32_t kw[4], qw[4];
      ldmatrix4(kw, row_at + j * 16);
      ldmatrix4(qw, row_at + ScanStage::off_q + j * 16);
#pragma unroll
      for (int nt = 0; nt < kBlocks; ++nt) {
        const float2 k2 = unpack16<T>(kw[nt]), q2 = unpack16<T>(qw[nt]);
        mma_tf32(R[nt], hi, k2.x, k2.y);
        mma_tf32(Rl[nt], lo, k2.x, k2.y);
        mma_tf32(O[nt], hi, q2.x, q2.y);
        if (kFine) mma_tf32(O[nt], lo, q2.x, q2.y);
      }
    }
#pragma unroll
    for (int nt = 0; nt < kBlocks; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) R[nt][e] += Rl[nt][e];
    // With two column halves: both need all of S k; of S q each takes two blocks of tokens to finish.
    constexpr int kOut = kBlocks / KS;                         // token blocks whose outputs this warp writes
    const int o0 = ks * kOut;
    if constexpr (KS == 2) {
#pragma unroll
      for (int nt = 0; nt < kBlocks; ++nt) {
        sx[vt][ks][nt][0][lane] = make_float2(R[nt][0], R[nt][1]);
        sx[vt][ks][nt][1][lane] = make_float2(R[nt][2], R[nt][3]);
      }
      __syncthreads();
#pragma unroll
      for (int nt = 0; nt < kBlocks; ++nt) {
        const float2 x = sx[vt][ks ^ 1][nt][0][lane], y = sx[vt][ks ^ 1][nt][1][lane];
        // in one order, so that both halves go on with the same bits
        const float mine[4] = {R[nt][0], R[nt][1], R[nt][2], R[nt][3]}, other[4] = {x.x, x.y, y.x, y.y};
#pragma unroll
        for (int e = 0; e < 4; ++e) R[nt][e] = ks ? other[e] + mine[e] : mine[e] + other[e];
      }
      __syncthreads();
#pragma unroll
      for (int x = 0; x < kOut; ++x) {
        const int nt = (ks ^ 1) * kOut + x;
        float give[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) give[e] = ks ? O[x][e] : O[kOut + x][e];
        sx[vt][ks][nt][0][lane] = make_float2(give[0], give[1]);
        sx[vt][ks][nt][1][lane] = make_float2(give[2], give[3]);
      }
      __syncthreads();
#pragma unroll
      for (int x = 0; x < kOut; ++x) {
        const float2 u = sx[vt][ks ^ 1][o0 + x][0][lane], y = sx[vt][ks ^ 1][o0 + x][1][lane];
        const float add[4] = {u.x, u.y, y.x, y.y};
#pragma unroll
        for (int e = 0; e < 4; ++e) O[x][e] = (ks ? O[kOut + x][e] : O[x][e]) + add[e];
      }
    }

    // beta (v - e^G r (S k)), value rows by tokens like the accumulators
    float hi[kBlocks][4], lo[kBlocks][4];
    float odd = 0.f;                                           // turns NaN where something is not finite
#pragma unroll
    for (int nt = 0; nt < kBlocks; nt += 2) {
      uint32_t vw[4];
      ldmatrix4_t(vw, at + ScanStage::off_v + (nt * 8 + (lane & 7) + (lane & 16 ? 8 : 0)) * ScanStage::kVPitch + vt * 32 + (lane & 8 ? 16 : 0));
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const float2 bt = *reinterpret_cast<const float2*>(vec + (nt + z) * 8 + 2 * t);
        const float2 be = *reinterpret_cast<const float2*>(vec + kC + (nt + z) * 8 + 2 * t);
        const float2 va = unpack16<T>(vw[2 * z]), vb = unpack16<T>(vw[2 * z + 1]);
        float (&r)[4] = R[nt + z];
        r[0] = fmaf(-be.x, r[0], bt.x * va.x);
        r[1] = fmaf(-be.y, r[1], bt.y * va.y);
        r[2] = fmaf(-be.x, r[2], bt.x * vb.x);
        r[3] = fmaf(-be.y, r[3], bt.y * vb.y);
#pragma unroll
        for (int e = 0; e < 4; ++e) odd = fmaf(r[e], 0.f, odd);
      }
    }
    // A value that is not finite reaches its own row from its token on, and nothing else: the products
    // below would carry it, through their zeros, to tokens before it. It is taken out of them, and
    // what it reaches is set to NaN afterwards.
    int lost[2] = {kC, kC};                                    // rows gid, gid + 8: the first such token
    const bool any_lost = __any_sync(0xffffffffu, odd != 0.f);
    if (any_lost) {
#pragma unroll
      for (int nt = kBlocks - 1; nt >= 0; --nt)
#pragma unroll
        for (int e = 3; e >= 0; --e)
          if (!isfinite(R[nt][e])) {
            R[nt][e] = 0.f;
            lost[e >> 1] = min(lost[e >> 1], nt * 8 + 2 * t + (e & 1));
          }
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        lost[z] = min(lost[z], __shfl_xor_sync(0xffffffffu, lost[z], 1));
        lost[z] = min(lost[z], __shfl_xor_sync(0xffffffffu, lost[z], 2));
      }
    }
#pragma unroll
    for (int nt = 0; nt < kBlocks; ++nt) operand(R[nt], hi[nt], lo[nt]);

    // U = T (...)
    float U[kBlocks][4] = {};
#pragma unroll
    for (int jb = 0; jb < kBlocks; ++jb)
#pragma unroll
      for (int nt = jb; nt < kBlocks; ++nt) {
        const float4 f = tf[(nt * (nt + 1) / 2 + jb) * 32];
        mma_tf32(U[nt], hi[jb], f.z, f.w);
        mma_tf32(U[nt], lo[jb], f.x, f.y);
        mma_tf32(U[nt], hi[jb], f.x, f.y);
      }
    if (any_lost) {
#pragma unroll
      for (int nt = 0; nt < kBlocks; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!isfinite(U[nt][e])) {                           // (T's own entries, or an overflow)
            U[nt][e] = 0.f;
            lost[e >> 1] = min(lost[e >> 1], nt * 8 + 2 * t + (e & 1));
          }
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        lost[z] = min(lost[z], __shfl_xor_sync(0xffffffffu, lost[z], 1));
        lost[z] = min(lost[z], __shfl_xor_sync(0xffffffffu, lost[z], 2));
      }
    }

    // o = e^G scale rq (S q) + P U
#pragma unroll
    for (int jb = 0; jb < kBlocks; ++jb) operand(U[jb], hi[jb], lo[jb]);
#pragma unroll
    for (int x = 0; x < kOut; ++x) {
      const int nt = o0 + x;
      const float2 f = *reinterpret_cast<const float2*>(vec + 3 * kC + nt * 8 + 2 * t);
      O[x][0] *= f.x; O[x][1] *= f.y; O[x][2] *= f.x; O[x][3] *= f.y;
#pragma unroll
      for (int jb = 0; jb < kBlocks; ++jb) {
        if (jb > nt) break;
        const float4 p = pf[(nt * (nt + 1) / 2 + jb) * 32];
        if (kFine) {
          mma_tf32(O[x], hi[jb], p.z, p.w);
          mma_tf32(O[x], lo[jb], p.x, p.y);
        }
        mma_tf32(O[x], hi[jb], p.x, p.y);
      }
      if (any_lost) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (nt * 8 + 2 * t + (e & 1) >= lost[e >> 1]) O[x][e] = __int_as_float(0x7fc00000);
      }
      // rows to tokens: lane (gid, t) then holds token gid, value rows 2t and 2t + 1
      const int tok = first + c * kC + nt * 8 + gid;
      const uint32_t a = transpose8(pack16<T>(O[x][0], O[x][1])), bb = transpose8(pack16<T>(O[x][2], O[x][3]));
      if (tok < end) {
        T* out = static_cast<T*>(g.o) + (long long)tok * g.o_stride + (long long)hv * g.V + v0 + vt * 16 + 2 * t;
        *reinterpret_cast<uint32_t*>(out) = a;
        *reinterpret_cast<uint32_t*>(out + 8) = bb;
      }
    }

    // S = e^{G_C} S + (e^{G_C-G} r U) K
#pragma unroll
    for (int nt = 0; nt < kBlocks; ++nt) {
      const float2 f = *reinterpret_cast<const float2*>(vec + 2 * kC + nt * 8 + 2 * t);
      U[nt][0] *= f.x; U[nt][1] *= f.y; U[nt][2] *= f.x; U[nt][3] *= f.y;
      operand(U[nt], hi[nt], lo[nt]);
    }
    const float dec = vec[4 * kC];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      uint32_t kw[4];
      ldmatrix4_t(kw, row_at + j * 16);
      float acc[4] = {}, accl[4] = {};
#pragma unroll
      for (int nt = 0; nt < kBlocks; ++nt) {
        const float2 k2 = unpack16<T>(kw[nt]);
        mma_tf32(acc, hi[nt], k2.x, k2.y);
        mma_tf32(accl, lo[nt], k2.x, k2.y);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) S[j][e] = fmaf(S[j][e], dec, acc[e] + accl[e]);
    }
    if (any_lost) {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (lost[e >> 1] < kC) S[j][e] = __int_as_float(0x7fc00000);
    }
  }

  const int to = g.out_slot[b];
  if (to >= 0 && to < g.slots) {
    float* dst = g.state_out + to * g.slot_stride + ((long long)hv * g.V + v0 + vt * 16 + gid) * kK + ks * NJ * 8 + 2 * t;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      *reinterpret_cast<float2*>(dst + 8 * j) = make_float2(S[j][0], S[j][1]);
      *reinterpret_cast<float2*>(dst + 8 * kK + 8 * j) = make_float2(S[j][2], S[j][3]);
    }
  }
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

int chunk_slots(int T, int B) { return T / kC + B; }

template <typename T, int KS>
cfb_status launch_scan(const cfb_gdn_args& g, const int32_t* cu, int total, int B, const float* ws, cudaStream_t st) {
  constexpr int bytes = kScanStages * ScanStage::bytes;
  if (cudaFuncSetAttribute(gdn_scan_kernel<T, KS>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return cfb_launch_status("gdn_scan_kernel attribute");
  const dim3 grid((unsigned)(g.V / kScanRows), (unsigned)g.HV, (unsigned)B);
  gdn_scan_kernel<T, KS><<<grid, 64 * KS, bytes, st>>>(g, cu, total, ws);
  return cfb_launch_status("gdn_scan_kernel");
}
template <typename T>
cfb_status launch_chunks(const cfb_gdn_args& g, const int32_t* cu, int total, int B, float* ws, cudaStream_t st) {
  gdn_prep_kernel<T><<<dim3((unsigned)chunk_slots(total, B), (unsigned)g.HV), 64, 0, st>>>(g, cu, total, B, ws);
  if (const cfb_status s = cfb_launch_status("gdn_prep_kernel")) return s;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return cfb_launch_status("cudaDeviceGetAttribute");
  // KS = 1 has two warps a CTA for an SM's four quarters
  const bool wide = (long long)(g.V / kScanRows) * g.HV * B * 2 <= 4ll * sms;
  return wide ? launch_scan<T, 2>(g, cu, total, B, ws, st) : launch_scan<T, 1>(g, cu, total, B, ws, st);
}

}  // namespace

extern "C" cfb_status cfb_gdn_step(const cfb_gdn_args* g, int B, void* stream) {
  if (B == 0 && g) return CFB_OK;
  if (const cfb_status s = check_gdn(g, B)) return s;
  launch_walk(*g, nullptr, B, B, static_cast<cudaStream_t>(stream));
  return cfb_launch_status("gdn_walk_kernel");
}

extern "C" size_t cfb_gdn_chunk_workspace(int T, int B, int HV) {
  if (T < 0 || B <= 0 || HV <= 0) return 0;
  return (size_t)chunk_slots(T, B) * HV * kPrepFloats * sizeof(float);
}

extern "C" cfb_status cfb_gdn_chunk(const cfb_gdn_args* g, const int32_t* cu, int T, int B, void* ws, size_t ws_bytes,
                                    void* stream) {
  if (B == 0 && g) return CFB_OK;
  if (const cfb_status s = check_gdn(g, B)) return s;
  if (T < 0 || !cu || !ws) return CFB_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(ws) & 255) || ws_bytes < cfb_gdn_chunk_workspace(T, B, g->HV)) return CFB_ERR_WORKSPACE;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  float* const prep = static_cast<float*>(ws);
  if (g->dtype == DT_F16) return launch_chunks<__half>(*g, cu, T, B, prep, st);
  return launch_chunks<__nv_bfloat16>(*g, cu, T, B, prep, st);
}
