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
// fetched while this one is worked on. Bound: HBM, the states read and written once a step (96 requests of 32
// value heads of 128 x 128: 403 MB in 84 us, 4.8 TB/s, 0.73 of a copy's rate), or launch latency (one: 4.2 us).
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
// Precision. The state is fp32 and has to stay so over thousands of chunks, so no product on its way rounds an
// operand to fewer than 22 bits. k and q are exact as they are (their norms are applied afterwards, in
// fp32). Over bf16, S and U meet k as three bf16 pieces, exactly, 16 columns a product (a chunk of one head
// at 8191 tokens: 1.9 us; the tf32 terms, 8 columns a product, 2.0). Else, S, U and T are split into two
// tf32 terms, x = hi + lo, lo * lo dropped (relative error about 2^-22): fp16 pieces would need a scale a row
// and chunk. Exponents of differences G_i - G_j are of sums kept in 64 bits: in 32, a strong decay's G of a
// few hundred would cost 1e-5. S is updated by one fp32 fma an element from a product that starts at zero,
// because sums carried through the tensor cores lose a little towards zero with every step. o is rounded to
// 16 bits and nothing depends on it, so its own products' S, U and P are the exception: over fp16 both terms, over bf16
// one, rounded to nearest (11 bits against o's 8; cut off, every output came out 2^-10.7 short).
//
// Why mma.sync and not tcgen05: the scan is a chain over a head's chunks, and what bounds it is the
// latency of one link, not throughput. With 16 value rows a warp, the state lives in the warp's
// registers in the accumulator layout, which, with the summed index permuted (2t, 2t + 1 for t, t + 4;
// the other operand is read as pairs of neighbours anyway), is the first operand's layout too: S feeds
// S k, that feeds T, U feeds the update, without a trip through shared or tensor memory and with one
// exchange between the two warps of a tile. Measured, 32 value heads of 128: 8191 tokens of one request 515 us
// (scan 457, prep 58), nine prompts of up to 1500 tokens 480; a chunk 1.8 us, in which each quarter of the SM
// issues 1660 instructions and 165 products of 8.4 cycles in 3300 cycles: no pipe is full, the chain of dependent
// steps of one state warp a quarter is the time. (Four warps a tile, a quarter of the columns each, repeat
// U's product twice as often: 700 us. Two CTAs an SM leave 96 registers a thread: 1070.)
constexpr int kC = 32, kBlocks = kC / 8;                       // tokens a chunk; blocks of 8
constexpr int kPairs = kBlocks * (kBlocks + 1) / 2;            // lower-triangular 8 x 8 blocks
// What the scan reads of a chunk and value head: T and P as the second operand of its products, a
// float4 (two neighbours' hi, their lo) a lane for each lower-triangular block, then per token beta,
// beta e^G r, e^{G_C-G} r, e^G scale rq, then e^{G_C}.
constexpr int kFragFloats = kPairs * 32 * 4;
constexpr int kPrepFloats = 2 * kFragFloats + 4 * kC + 4;      // (over bf16 P's lo terms are left out)
template <typename T>
struct Prep {
  static constexpr int kP = std::is_same<T, __half>::value ? 4 : 2;          // floats of P a lane and block
  static constexpr int kVec = kFragFloats + kPairs * 32 * kP, kFloats = kVec + 4 * kC + 4;
};
constexpr int kRowHalves = kK + 8;                             // padded row of a staged K or Q tile

// x = hi + lo, both of 11 bits (tf32): hi is x cut off, lo the remainder rounded. Integer operations: a
// conversion instruction takes eight cycles a warp, and a chunk splits 128 values a lane.
CFB_DEV void split(float x, float& hi, float& lo) {
  hi = __uint_as_float(__float_as_uint(x) & 0xffffe000u);
  lo = __uint_as_float((__float_as_uint(x - hi) + 0x1000u) & 0xffffe000u);
}
// x = b1 + b2 + b3, bf16 each and exactly so: a piece is the top 16 bits of what is left, 8 of the 24 bits of
// x's mantissa. Two neighbours' pieces as one register of an m16n8k16 operand.
CFB_DEV void split3(float x, float y, uint32_t (&p)[3]) {
  p[0] = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
#pragma unroll
  for (int i = 1; i < 3; ++i) {
    x -= __uint_as_float(__float_as_uint(x) & 0xffff0000u);
    y -= __uint_as_float(__float_as_uint(y) & 0xffff0000u);
    p[i] = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
  }
}
// x rounded to 11 bits (tf32); a NaN may come out as anything
CFB_DEV float nearest11(float x) { return __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xffffe000u); }
CFB_DEV float nearest11_nan(float x) { return x == x ? nearest11(x) : x; }
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

// One CTA of two warps per (chunk, value head): warp 0 forms K K^T, A and T, warp 1 Q K^T and P, both in
// their accumulators (P's are already in the order that the scan reads). The norms are diagonals of
// K K^T and Q Q^T. Rows of tokens that the chunk does not have are zeros with beta = 0 and no decay.
template <typename T>
__global__ void __launch_bounds__(64) gdn_prep_kernel(const cfb_gdn_args g, const int32_t* cu, int total, int B, float* ws, int* err) {
  __shared__ __align__(16) T sk[kC][kRowHalves];
  __shared__ __align__(16) T sq[kC][kRowHalves];
  __shared__ __align__(16) float sa[kC][kC + 4];               // A, then T
  __shared__ float2 sG[kC];                                    // G log2(e) as a sum of two floats
  __shared__ float sd[2][kC];                                  // reciprocal norms of k, of q
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hv = blockIdx.y, h = hv / (g.HV / g.H);
  int b, t0, n;
  if (blockIdx.x == 0 && hv == 0 && threadIdx.x == 0) *err = 0;
  if (!chunk_of(cu, total, B, blockIdx.x, &b, &t0, &n)) return;
  {
    const T* k = static_cast<const T*>(g.k) + (long long)t0 * g.k_stride + (long long)h * kK;
    const T* q = static_cast<const T*>(g.q) + (long long)t0 * g.q_stride + (long long)h * kK;
#pragma unroll
    for (int x = 0; x < kC * 16 / 64; ++x) {
      const int row = x * 4 + (threadIdx.x >> 4), c = threadIdx.x & 15;
      const bool in = row < n;
      cp_async16z(smem_u32(&sk[row][c * 8]), k + (in ? (long long)row * g.k_stride : 0) + c * 8, in);
      cp_async16z(smem_u32(&sq[row][c * 8]), q + (in ? (long long)row * g.q_stride : 0) + c * 8, in);
    }
  }
  float beta = 0.f, decay = 0.f;
  if (lane < n) {
    const float rate = -expf(load_coded(g.A_log, g.A_log_dtype, hv));
    const float bias = load_coded(g.dt_bias, g.dt_bias_dtype, hv);
    decay = rate * softplus(load_coded(g.a, g.a_dtype, (long long)(t0 + lane) * g.a_stride + hv) + bias);
    beta = sigmoid(load_coded(g.b, g.b_dtype, (long long)(t0 + lane) * g.b_stride + hv));
  }
  // G by token (a decay of e^-1e6 is 0 all the same; sums and differences stay numbers)
  double G = (decay < -1e6f ? -1e6 : (double)decay) * 1.4426950408889634;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, G, off);
    if (lane >= off) G += y;
  }
  // differences of G from two floats each: the sum of 32 decays in 48 bits
  const float2 G2 = make_float2((float)G, (float)(G - (double)(float)G));
  const float2 G_end = make_float2(__shfl_sync(0xffffffffu, G2.x, 31), __shfl_sync(0xffffffffu, G2.y, 31));
  const auto decay_between = [](float2 to, float2 from) { return exp2f((to.x - from.x) + (to.y - from.y)); };
  if (warp == 0) sG[lane] = G2;
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  // X K^T, X = K (warp 0) or Q (warp 1): blocks on and below the diagonal
  const int gid = lane >> 2, t = lane & 3;
  float acc[2][kBlocks][4] = {};
  {
    const uint32_t a_at = smem_u32(&(warp ? sq : sk)[lane & 15][(lane >> 4) * 8]), b_at = smem_u32(&sk[lane][0]);
    float dq[2][2][4] = {};                                    // Q Q^T's diagonal blocks (warp 1)
#pragma unroll
    for (int k = 0; k < kK / 16; ++k) {
      uint32_t a[2][4], b0[4], b1[4];
      ldmatrix4(a[0], a_at + k * 32);
      ldmatrix4(a[1], a_at + 16 * kRowHalves * 2 + k * 32);
      ldmatrix4(b0, b_at + k * 32);
      ldmatrix4(b1, b_at + k * 32 + 16);
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int nt = 0; nt < 2 * mt + 2; ++nt) mma_16<T>(acc[mt][nt], a[mt], b0[nt], b1[nt]);
      if (warp) {
        // a's fragments hold Q's own rows as the second operand too: rows 0-7 in a[0], a[2], 8-15 in a[1], a[3]
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          mma_16<T>(dq[mt][0], a[mt], a[mt][0], a[mt][2]);
          mma_16<T>(dq[mt][1], a[mt], a[mt][1], a[mt][3]);
        }
      }
    }
    // the diagonals: row gid of a block is column 2t (+ 1) in lane t = gid / 2
    if (t == gid >> 1) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const float even = warp ? dq[mt][z][2 * z] : acc[mt][2 * mt + z][2 * z];
          const float odd = warp ? dq[mt][z][2 * z + 1] : acc[mt][2 * mt + z][2 * z + 1];
          sd[warp][mt * 16 + z * 8 + gid] = rsqrtf((gid & 1 ? odd : even) + kNormEps);
        }
    }
  }
  __syncthreads();
  const float* const rk = sd[0];
  float* const out = ws + ((long long)blockIdx.x * g.HV + hv) * kPrepFloats;
  if (warp == 0) {
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const int i = mt * 16 + z * 8 + gid;
        const float f = __shfl_sync(0xffffffffu, beta, i) * rk[i];
        const float2 Gi = sG[i];
#pragma unroll
        for (int nt = 0; nt <= 2 * mt + z; ++nt) {
          const int j = nt * 8 + 2 * t;
          const float2 x = make_float2(j < i ? f * rk[j] * decay_between(Gi, sG[j]) * acc[mt][nt][2 * z] : 0.f,
                                       j + 1 < i ? f * rk[j + 1] * decay_between(Gi, sG[j + 1]) * acc[mt][nt][2 * z + 1] : 0.f);
          *reinterpret_cast<float2*>(&sa[i][j]) = x;
        }
      }
    __syncwarp();
    // T column by column, a lane a column: x_i = [i = j] - sum_{m<i} A_im x_m
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
    float4* const tf = reinterpret_cast<float4*>(out) + lane;
#pragma unroll
    for (int nt = 0; nt < kBlocks; ++nt)
#pragma unroll
      for (int jb = 0; jb <= nt; ++jb) {
        const float2 y = *reinterpret_cast<const float2*>(&sa[nt * 8 + gid][jb * 8 + 2 * t]);
        float4 f;
        split(y.x, f.x, f.z);
        split(y.y, f.y, f.w);
        tf[(nt * (nt + 1) / 2 + jb) * 32] = f;
      }
  } else {
    const float* const rq = sd[1];
    float* const pf = out + kFragFloats + lane * Prep<T>::kP;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const int nt = 2 * mt + z, i = nt * 8 + gid;
        const float f = g.scale * rq[i];
        const float2 Gi = sG[i];
#pragma unroll
        for (int jb = 0; jb <= nt; ++jb) {
          const int j = jb * 8 + 2 * t;
          const float x = j <= i ? f * rk[j] * decay_between(Gi, sG[j]) * acc[mt][jb][2 * z] : 0.f;
          const float y = j + 1 <= i ? f * rk[j + 1] * decay_between(Gi, sG[j + 1]) * acc[mt][jb][2 * z + 1] : 0.f;
          float* const dst = pf + (nt * (nt + 1) / 2 + jb) * 32 * Prep<T>::kP;
          float4 w;
          split(x, w.x, w.z);
          split(y, w.y, w.w);
          if constexpr (Prep<T>::kP == 4) *reinterpret_cast<float4*>(dst) = w;
          else *reinterpret_cast<float2*>(dst) = make_float2(nearest11_nan(x), nearest11_nan(y));
        }
      }
    float* const v = out + Prep<T>::kVec;
    const float eG = exp2f(G2.x + G2.y);
    v[lane] = beta;
    v[kC + lane] = beta * eG * rk[lane];
    v[2 * kC + lane] = decay_between(G_end, G2) * rk[lane];
    v[3 * kC + lane] = eG * g.scale * rq[lane];
    if (lane < 4) v[4 * kC + lane] = exp2f(G_end.x + G_end.y);
  }
}

// One CTA per (16 TILES value rows, value head, request), TILES value tiles of 16 rows, four warps a tile and one that
// copies, so that every quarter of the SM has warps of the first two kinds:
//   the state, two warps a tile: each holds the tile's rows and half of the columns. A chunk is S k (the two halves
//        exchange partial sums), U and the update, nothing else;
//   the outputs, two warps a tile, a chunk behind, half of the tokens each: S, as it was before the chunk, and U
//        reach them through shared memory (two buffers), so that S q and P U are off the chain that bounds the
//        kernel;
//   the copies: one lane issues those of the chunks to come: K and Q as [64 columns][32 tokens] 128-byte-swizzled
//        boxes, V as plain boxes of 32 columns, T, P and the vectors in one piece. (The same copies by 16-byte
//        cp.async kept a warp busy for longer than a chunk takes.)
constexpr int kHandThreads = 4 * 32;                           // a tile's two state and two output warps
template <typename T, int TILES>
struct Scan {
  static constexpr int kStages = TILES == 2 ? 4 : 3, kWarps = 2 * TILES, kRows = 16 * TILES, kThreads = (2 * kWarps + (TILES == 2 ? 1 : 4)) * 32;
  static constexpr int kKV = kC * kK * 2, kV = kC * kRows * 2, kPrep = Prep<T>::kFloats * 4;
  static constexpr int off_q = kKV, off_v = 2 * kKV, off_prep = off_v + kV;
  static constexpr int stage = (off_prep + kPrep + 1023) / 1024 * 1024, off_swap = kStages * stage;
  static constexpr int kSwap = kBlocks * 2 * 32 * 8;           // one warp's partial sums of S k
  // what a tile's output warp reads: S ([16 blocks][lane] of four), U ([4 blocks][lane]), the first tokens lost
  static constexpr int off_hand = off_swap + 2 * kWarps * kSwap, off_u = 16 * 512, off_lost = off_u + kBlocks * 512;
  static constexpr int kHand = off_lost + 256;
  static constexpr int bytes = off_hand + 2 * TILES * kHand + 1024;
  static constexpr int tx = 2 * kKV + kV + kPrep;
};
CFB_DEV void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" :: "r"(id), "r"(threads) : "memory"); }
CFB_DEV void bar_arrive(int id, int threads) { asm volatile("bar.arrive %0, %1;" :: "r"(id), "r"(threads) : "memory"); }

// An accumulator as the first operand of the next product: the summed index is permuted, 2t and 2t + 1 for
// t and t + 4, and the second operand is read so.
CFB_DEV void operand(const float (&s)[4], float (&hi)[4], float (&lo)[4]) {
  split(s[0], hi[0], lo[0]);
  split(s[2], hi[1], lo[1]);
  split(s[1], hi[2], lo[2]);
  split(s[3], hi[3], lo[3]);
}
// the same in one term, rounded to nearest
template <bool NAN_KEPT>
CFB_DEV void operand11(const float (&s)[4], float (&hi)[4]) {
  const auto near = [](float x) { return NAN_KEPT ? nearest11_nan(x) : nearest11(x); };
  hi[0] = near(s[0]);
  hi[1] = near(s[2]);
  hi[2] = near(s[1]);
  hi[3] = near(s[3]);
}

template <typename T, int TILES>
__global__ void __launch_bounds__((4 * TILES + (TILES == 2 ? 1 : 4)) * 32, 1)
gdn_scan_kernel(const cfb_gdn_args g, const int32_t* cu, int total, int B, const float* ws, int* err,
                const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                const __grid_constant__ CUtensorMap v_map) {
  using Lay = Scan<T, TILES>;
  constexpr int kScanStages = Lay::kStages, kStateWarps = Lay::kWarps, kOutWarps = Lay::kWarps;
  constexpr int NJ = 8;                                        // 8-column blocks of the state a warp holds
  constexpr bool kFine = std::is_same<T, __half>::value;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kScanStages], empty[kScanStages], freed[TILES][2];
  __shared__ int dead;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, t = lane & 3;
  const int hv = blockIdx.y, h = hv / (g.HV / g.H), v0 = blockIdx.x * Lay::kRows;
  // The longest requests first, as many as threads can rank (a long one begun last is the launch's tail: nine
  // prompts of up to 1500 tokens 487 us in the order they came, 480 so).
  __shared__ int sh_len[Lay::kThreads], sh_b;
  if (B <= Lay::kThreads) {
    const int x = threadIdx.x;
    int n = 0, before = 0;
    if (x < B) sh_len[x] = n = min(max(cu[x + 1], 0), total) - min(max(cu[x], 0), total);
    __syncthreads();
    if (x < B) {
#pragma unroll 8
      for (int i = 0; i < B; ++i) before += sh_len[i] > n || (sh_len[i] == n && i < x);
      if (before == (int)blockIdx.z) sh_b = x;
    }
    __syncthreads();
  }
  const int b = B <= Lay::kThreads ? sh_b : blockIdx.z;
  const int first = min(max(cu[b], 0), total), end = min(max(cu[b + 1], first), total);
  const int chunks = (end - first + kC - 1) / kC;
  const uint32_t sm = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (sm - smem_u32(smem_raw));
  if (threadIdx.x == 0) {
    for (int i = 0; i < kScanStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kStateWarps + kOutWarps);
    }
    for (int i = 0; i < 2 * TILES; ++i) mbar_init(&freed[i >> 1][i & 1], 2);
    fence_mbar_init();
    dead = 0;
  }
  __syncthreads();
  // A wait that outlasts its limit marks the CTA dead: from then on nothing waits for copies, the chunks run through
  // to the end on whatever is there, and the state is set to NaN. What a tile's warps wait for from one another they
  // wait for all the same: the state warps, a hand-over buffer ahead, would else arrive at a barrier twice where
  // the output warps have not been once, and those would then stay there for good. (Such a wait is for warps that get
  // on: they wait for copies, 1 s at most and once, and for these warps. Its own limit is well above that.)
  volatile int* const is_dead = &dead;
  const auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (mbar_test_wait(bar, parity)) return;
    if (*is_dead == 0 && !mbar_wait(bar, parity)) *is_dead = 1;
  };
  const auto wait_freed = [&](uint64_t* bar, uint32_t parity) {
    if (!mbar_test_wait(bar, parity) && !mbar_wait(bar, parity, nullptr, 8 * kWaitBudgetNs)) *is_dead = 1;
  };
  // barriers of a tile: the state warps' exchange; S and U handed over (freed: a hand-over buffer free again)
  const int tile = (warp % kStateWarps) / 2;
  const int swap_bar = 1 + tile * 3, hand_bar = swap_bar + 1;        // (+ chunk & 1)
  const auto hand_at = [&](int c) { return smem + Lay::off_hand + ((c & 1) * TILES + tile) * Lay::kHand; };
  // token `lane`'s row of a K or Q tile, 8-column block x: 128-byte rows of half the columns, 16-byte pieces
  // XORed with token & 7
  const auto block = [&](uint32_t at, int x) { return at + lane * 128 + (x >> 3) * (kC * 128) + (((x & 7) ^ (lane & 7)) << 4); };

  // (four tiles: 20 warps of 96 registers at launch, 61440; then 8 of 152, 8 of 72 and 4 of 24, 60416)
  if (warp >= kStateWarps + kOutWarps) {
    if (TILES > 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 24;");
    if (warp > kStateWarps + kOutWarps) return;
    // ------------------------------------------------------------ copies
    if (lane == 0) {
      prefetch_map(&q_map);
      prefetch_map(&k_map);
      prefetch_map(&v_map);
      const float* const prep = ws + ((long long)(first / kC + b) * g.HV + hv) * kPrepFloats;
      int c = 0;
      for (; c < chunks; ++c) {
        const int st = c % kScanStages;
        if (c >= kScanStages) wait(&empty[st], (c / kScanStages - 1) & 1);
        if (*is_dead) break;
        const uint32_t at = sm + st * Lay::stage;
        mbar_arrive_expect_tx(&full[st], Lay::tx);
        tma_load_4d(at, &k_map, 0, first + c * kC, 0, h, &full[st]);
#pragma unroll
        for (int x = 0; x < TILES / 2; ++x)
          tma_load_3d(at + Lay::off_v + x * kC * 64, &v_map, v0 + x * 32, first + c * kC, hv, &full[st]);
        bulk_g2s(smem + st * Lay::stage + Lay::off_prep, prep + (long long)c * g.HV * kPrepFloats, Lay::kPrep, &full[st]);
        tma_load_4d(at + Lay::off_q, &q_map, 0, first + c * kC, 0, h, &full[st]);
      }
      // a CTA that gave up must not end before these copies have landed
      for (int x = max(c - kScanStages, 0); x < c; ++x) mbar_wait(&full[x % kScanStages], (x / kScanStages) & 1);
    }
    return;
  }

  if (warp >= kStateWarps) {
    if (TILES > 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    // ------------------------------------------------------------ outputs: o = e^G scale rq (S q) + P U
    for (int c = 0; c < chunks; ++c) {
      wait(&full[c % kScanStages], (c / kScanStages) & 1);
      const uint8_t* const st = smem + (c % kScanStages) * Lay::stage;
      const uint32_t q_at = sm + (c % kScanStages) * Lay::stage + Lay::off_q;
      const float* const pf = reinterpret_cast<const float*>(st + Lay::off_prep) + kFragFloats + lane * Prep<T>::kP;
      const float* const vec = reinterpret_cast<const float*>(st + Lay::off_prep) + Prep<T>::kVec;
      const uint8_t* const hand = hand_at(c);
      bar_sync(hand_bar + (c & 1), kHandThreads);
      float O[2][4] = {}, hi[kBlocks][4], lo[kBlocks][4];
      const int n0 = 2 * (warp & 1);                           // this warp's token blocks: n0, n0 + 1
#pragma unroll 4
      for (int j = 0; j < 16; ++j) {
        const float4 s4 = reinterpret_cast<const float4*>(hand)[j * 32 + lane];
        const float sj[4] = {s4.x, s4.y, s4.z, s4.w};
        uint32_t qw[4];
        ldmatrix4(qw, block(q_at, j));
        if constexpr (kFine) operand(sj, hi[0], lo[0]);
        else operand11<false>(sj, hi[0]);                      // (a row of S with a NaN in it has lost its first token)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float2 q2 = unpack16<T>(n0 ? qw[2 + x] : qw[x]);
          mma_tf32(O[x], hi[0], q2.x, q2.y);
          if (kFine) mma_tf32(O[x], lo[0], q2.x, q2.y);
        }
      }
      const int2 lost = reinterpret_cast<const int2*>(hand + Lay::off_lost)[lane];
#pragma unroll
      for (int jb = 0; jb < kBlocks; ++jb) {
        const float4 u4 = reinterpret_cast<const float4*>(hand + Lay::off_u)[jb * 32 + lane];
        const float u[4] = {u4.x, u4.y, u4.z, u4.w};
        if constexpr (kFine) operand(u, hi[jb], lo[jb]);
        else operand11<true>(u, hi[jb]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&freed[tile][c & 1]);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int nt = n0 + x;
        const float2 f = *reinterpret_cast<const float2*>(vec + 3 * kC + nt * 8 + 2 * t);
        O[x][0] *= f.x; O[x][1] *= f.y; O[x][2] *= f.x; O[x][3] *= f.y;
#pragma unroll
        for (int jb = 0; jb < kBlocks; ++jb) {
          if (jb > nt) break;
          const float* const p = pf + (nt * (nt + 1) / 2 + jb) * 32 * Prep<T>::kP;
          if constexpr (kFine) {
            const float4 w = *reinterpret_cast<const float4*>(p);
            mma_tf32(O[x], hi[jb], w.z, w.w);
            mma_tf32(O[x], lo[jb], w.x, w.y);
            mma_tf32(O[x], hi[jb], w.x, w.y);
          } else {
            const float2 w = *reinterpret_cast<const float2*>(p);
            mma_tf32(O[x], hi[jb], w.x, w.y);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (nt * 8 + 2 * t + (e & 1) >= (e < 2 ? lost.x : lost.y)) O[x][e] = __int_as_float(0x7fc00000);
        // rows to tokens: lane (gid, t) then holds token gid, value rows 2t and 2t + 1
        const int tok = first + c * kC + nt * 8 + gid;
        const uint32_t a = transpose8(pack16<T>(O[x][0], O[x][1])), bb = transpose8(pack16<T>(O[x][2], O[x][3]));
        if (tok < end) {
          T* out = static_cast<T*>(g.o) + (long long)tok * g.o_stride + (long long)hv * g.V + v0 + tile * 16 + 2 * t;
          *reinterpret_cast<uint32_t*>(out) = a;
          *reinterpret_cast<uint32_t*>(out + 8) = bb;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[c % kScanStages]);
    }
    return;
  }

  // -------------------------------------------------------------- state: lane (gid, t) holds rows gid and
  // gid + 8, columns 2t and 2t + 1 of every 8-column block
  if (TILES > 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
  const int ks = warp & 1;
  float S[NJ][4];
  const long long state_at = ((long long)hv * g.V + v0 + tile * 16 + gid) * kK + ks * NJ * 8 + 2 * t;
  {
    const int from = g.init_slot[b];
    const float fill = from < 0 ? 0.f : __int_as_float(0x7fc00000);
    const bool read = from >= 0 && from < g.slots;
    const float* src = g.state_in + (read ? from * g.slot_stride : 0) + state_at;
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
  for (int c = 0; c < chunks; ++c) {
    uint8_t* const hand = hand_at(c);
    if (c >= 2) wait_freed(&freed[tile][c & 1], ((c >> 1) - 1) & 1);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      reinterpret_cast<float4*>(hand)[(ks * NJ + j) * 32 + lane] = make_float4(S[j][0], S[j][1], S[j][2], S[j][3]);
    wait(&full[c % kScanStages], (c / kScanStages) & 1);
    const uint32_t at = sm + (c % kScanStages) * Lay::stage;
    uint8_t* const st = smem + (c % kScanStages) * Lay::stage;
    const float4* const tf = reinterpret_cast<const float4*>(st + Lay::off_prep) + lane;
    const float* const vec = reinterpret_cast<const float*>(st + Lay::off_prep) + Prep<T>::kVec;
    const int live = end - first - c * kC;                     // tokens of the chunk, if fewer than kC
    if (live < kC) {
      // the boxes hold the next request's rows there: keys whose zero weights must not meet a NaN (every
      // warp zeroes all of them for itself)
      for (int x = live * 8 + lane; x < kC * 8; x += 32) {
        *reinterpret_cast<uint4*>(st + x * 16) = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(st + kC * 128 + x * 16) = make_uint4(0, 0, 0, 0);
      }
      __syncwarp();
    }

    // what the next steps read, ahead of them
    uint32_t vw[kBlocks / 2][4];
#pragma unroll
    for (int nt = 0; nt < kBlocks; nt += 2)
      ldmatrix4_t(vw[nt / 2], at + Lay::off_v + (tile >> 1) * (kC * 64) + (nt * 8 + (lane & 7) + (lane & 16 ? 8 : 0)) * 64 + (tile & 1) * 32 + (lane & 8 ? 16 : 0));
    float2 bt[kBlocks], be[kBlocks], eg[kBlocks];
    float4 tw[kPairs];
#pragma unroll
    for (int nt = 0; nt < kBlocks; ++nt) {
      bt[nt] = *reinterpret_cast<const float2*>(vec + nt * 8 + 2 * t);
      be[nt] = *reinterpret_cast<const float2*>(vec + kC + nt * 8 + 2 * t);
      eg[nt] = *reinterpret_cast<const float2*>(vec + 2 * kC + nt * 8 + 2 * t);
    }
#pragma unroll
    for (int x = 0; x < kPairs; ++x) tw[x] = tf[x * 32];
    const float dec = vec[4 * kC];

    // S k of the chunk's tokens
    float R[kBlocks][4] = {}, Rl[kBlocks][4] = {};
    uint32_t kw[2][4];                                         // a block ahead
    ldmatrix4(kw[0], block(at, ks * NJ));
    if constexpr (!kFine) {
      // two blocks of 8 columns a product, the accumulators as its first operand as they lie
#pragma unroll
      for (int j = 0; j < NJ; j += 2) {
        uint32_t p[4][3], now[2][4];
        split3(S[j][0], S[j][1], p[0]);
        split3(S[j][2], S[j][3], p[1]);
        split3(S[j + 1][0], S[j + 1][1], p[2]);
        split3(S[j + 1][2], S[j + 1][3], p[3]);
        if (j == 0) ldmatrix4(kw[1], block(at, ks * NJ + 1));
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
          for (int e = 0; e < 4; ++e) now[z][e] = kw[z][e];
        if (j + 2 < NJ) {
          ldmatrix4(kw[0], block(at, ks * NJ + j + 2));
          ldmatrix4(kw[1], block(at, ks * NJ + j + 3));
        }
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          const uint32_t a[4] = {p[0][i], p[1][i], p[2][i], p[3][i]};
#pragma unroll
          for (int nt = 0; nt < kBlocks; ++nt) mma_16<T>(i ? Rl[nt] : R[nt], a, now[0][nt], now[1][nt]);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        float hi[4], lo[4];
        operand(S[j], hi, lo);
        if (j + 1 < NJ) ldmatrix4(kw[(j + 1) & 1], block(at, ks * NJ + j + 1));
#pragma unroll
        for (int nt = 0; nt < kBlocks; ++nt) {
          const float2 k2 = unpack16<T>(kw[j & 1][nt]);
          mma_tf32(R[nt], hi, k2.x, k2.y);
          mma_tf32(Rl[nt], lo, k2.x, k2.y);
        }
      }
    }
    // both halves need all of S k (two buffers in turn: the next chunk's barrier comes between a value's
    // reading and its overwriting)
    {
      using Sums = float2[kBlocks][2][32];
      uint8_t* const swap = smem + Lay::off_swap + ((c & 1) * TILES + tile) * 2 * Lay::kSwap;
      Sums& mine = *reinterpret_cast<Sums*>(swap + ks * Lay::kSwap);
      Sums& theirs = *reinterpret_cast<Sums*>(swap + (ks ^ 1) * Lay::kSwap);
#pragma unroll
      for (int nt = 0; nt < kBlocks; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) R[nt][e] += Rl[nt][e];
        mine[nt][0][lane] = make_float2(R[nt][0], R[nt][1]);
        mine[nt][1][lane] = make_float2(R[nt][2], R[nt][3]);
      }
      bar_sync(swap_bar, 64);
#pragma unroll
      for (int nt = 0; nt < kBlocks; ++nt) {                   // (a + b is b + a: both halves go on with the same bits)
        const float2 x = theirs[nt][0][lane], y = theirs[nt][1][lane];
        R[nt][0] += x.x; R[nt][1] += x.y; R[nt][2] += y.x; R[nt][3] += y.y;
      }
    }

    // beta (v - e^G r (S k)), value rows by tokens like the accumulators
    float hi[kBlocks][4], lo[kBlocks][4];
    float odd[kBlocks];                                        // turns NaN where something is not finite
#pragma unroll
    for (int nt = 0; nt < kBlocks; ++nt) {
      const float2 va = unpack16<T>(vw[nt / 2][2 * (nt & 1)]), vb = unpack16<T>(vw[nt / 2][2 * (nt & 1) + 1]);
      float (&r)[4] = R[nt];
      r[0] = fmaf(-be[nt].x, r[0], bt[nt].x * va.x);
      r[1] = fmaf(-be[nt].y, r[1], bt[nt].y * va.y);
      r[2] = fmaf(-be[nt].x, r[2], bt[nt].x * vb.x);
      r[3] = fmaf(-be[nt].y, r[3], bt[nt].y * vb.y);
      if (live < kC) {                                         // rows of no token (v there is the next request's)
        const int tok = nt * 8 + 2 * t;
        if (tok >= live) r[0] = r[2] = 0.f;
        if (tok + 1 >= live) r[1] = r[3] = 0.f;
      }
      odd[nt] = fmaf(r[0], 0.f, r[1] * 0.f) + fmaf(r[2], 0.f, r[3] * 0.f);
    }
    // A value that is not finite reaches its own row from its token on, and nothing else: the products
    // below would carry it, through their zeros, to tokens before it. It is taken out of them, and
    // what it reaches is set to NaN afterwards.
    int lost[2] = {kC, kC};                                    // rows gid, gid + 8: the first such token
    const bool any_lost = __any_sync(0xffffffffu, (odd[0] + odd[1]) + (odd[2] + odd[3]) != 0.f);
    const auto take_out = [&](float (&x)[kBlocks][4]) {
#pragma unroll
      for (int nt = 0; nt < kBlocks; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!isfinite(x[nt][e])) {
            x[nt][e] = 0.f;
            lost[e >> 1] = min(lost[e >> 1], nt * 8 + 2 * t + (e & 1));
          }
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        lost[z] = min(lost[z], __shfl_xor_sync(0xffffffffu, lost[z], 1));
        lost[z] = min(lost[z], __shfl_xor_sync(0xffffffffu, lost[z], 2));
      }
    };
    if (any_lost) take_out(R);
#pragma unroll
    for (int nt = 0; nt < kBlocks; ++nt) operand(R[nt], hi[nt], lo[nt]);

    // U = T (...)
    float U[kBlocks][4] = {}, Ul[kBlocks][4] = {}, Um[kBlocks][4] = {};
#pragma unroll
    for (int jb = 0; jb < kBlocks; ++jb)
#pragma unroll
      for (int nt = jb; nt < kBlocks; ++nt) {
        const float4 f = tw[nt * (nt + 1) / 2 + jb];
        mma_tf32(U[nt], hi[jb], f.x, f.y);
        mma_tf32(Ul[nt], lo[jb], f.x, f.y);
        mma_tf32(Um[nt], hi[jb], f.z, f.w);
      }
    uint32_t kt[2][4];
    ldmatrix4_t(kt[0], block(at, ks * NJ));
    ldmatrix4_t(kt[1], block(at, ks * NJ + 1));
#pragma unroll
    for (int nt = 0; nt < kBlocks; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) U[nt][e] += Ul[nt][e] + Um[nt][e];
    if (any_lost) take_out(U);                                 // (T's own entries, or an overflow)
    if (ks == 0) {
#pragma unroll
      for (int nt = 0; nt < kBlocks; ++nt)
        reinterpret_cast<float4*>(hand + Lay::off_u)[nt * 32 + lane] = make_float4(U[nt][0], U[nt][1], U[nt][2], U[nt][3]);
      reinterpret_cast<int2*>(hand + Lay::off_lost)[lane] = make_int2(lost[0], lost[1]);
    }
    bar_arrive(hand_bar + (c & 1), kHandThreads);

    // S = e^{G_C} S + (e^{G_C-G} r U) K
#pragma unroll
    for (int nt = 0; nt < kBlocks; ++nt) {
      U[nt][0] *= eg[nt].x; U[nt][1] *= eg[nt].y; U[nt][2] *= eg[nt].x; U[nt][3] *= eg[nt].y;
      if constexpr (kFine) operand(U[nt], hi[nt], lo[nt]);
    }
    uint32_t up[3][kBlocks / 2][4];                            // U's pieces, 16 tokens an operand
    if constexpr (!kFine) {
#pragma unroll
      for (int nt = 0; nt < kBlocks; ++nt)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          uint32_t p[3];
          split3(U[nt][2 * z], U[nt][2 * z + 1], p);
#pragma unroll
          for (int i = 0; i < 3; ++i) up[i][nt / 2][2 * (nt & 1) + z] = p[i];
        }
    }
#pragma unroll
    for (int j = 0; j < NJ; j += 2) {                          // four sums side by side cover a product's latency
      float acc[2][4] = {}, accl[2][4] = {};
      uint32_t now[2][4];
#pragma unroll
      for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int e = 0; e < 4; ++e) now[z][e] = kt[z][e];
      if (j + 2 < NJ) {
        ldmatrix4_t(kt[0], block(at, ks * NJ + j + 2));
        ldmatrix4_t(kt[1], block(at, ks * NJ + j + 3));
      }
      if constexpr (!kFine) {
#pragma unroll
        for (int nt = 0; nt < kBlocks; nt += 2)
#pragma unroll
          for (int i = 0; i < 3; ++i)
#pragma unroll
            for (int z = 0; z < 2; ++z) mma_16<T>(i ? accl[z] : acc[z], up[i][nt / 2], now[z][nt], now[z][nt + 1]);
      } else {
#pragma unroll
        for (int nt = 0; nt < kBlocks; ++nt)
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const float2 k2 = unpack16<T>(now[z][nt]);
            mma_tf32(acc[z], hi[nt], k2.x, k2.y);
            mma_tf32(accl[z], lo[nt], k2.x, k2.y);
          }
      }
#pragma unroll
      for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int e = 0; e < 4; ++e) S[j + z][e] = fmaf(S[j + z][e], dec, acc[z][e] + accl[z][e]);
    }
    if (any_lost) {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (lost[e >> 1] < kC) S[j][e] = __int_as_float(0x7fc00000);
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[c % kScanStages]);
  }
  if (*is_dead) {
    if (lane == 0) *err = DEV_TIMEOUT_FULL;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[j][e] = __int_as_float(0x7fc00000);
  }
  const int to = g.out_slot[b];
  if (to >= 0 && to < g.slots) {
    float* dst = g.state_out + to * g.slot_stride + state_at;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      *reinterpret_cast<float2*>(dst + 8 * j) = make_float2(S[j][0], S[j][1]);
      *reinterpret_cast<float2*>(dst + 8 * kK + 8 * j) = make_float2(S[j][2], S[j][3]);
    }
  }
}

cfb_status check_gdn(const cfb_gdn_args* g, int T, int B) {
  if (!g || T < 0 || B < 0) return CFB_ERR_INVALID_ARG;
  if (!g->A_log || !g->dt_bias || !g->state_in || !g->state_out || !g->init_slot || !g->out_slot || g->H <= 0 || g->HV <= 0 ||
      g->slots <= 0)
    return CFB_ERR_INVALID_ARG;
  // (rows of no tokens are read nowhere, and an empty array's address may be null)
  if (T > 0 && (!g->a || !g->b || !g->q || !g->k || !g->v || !g->o)) return CFB_ERR_INVALID_ARG;
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

constexpr size_t kErrBytes = 256;                              // the device error word, at the workspace's start
int chunk_slots(int T, int B) { return T / kC + B; }

// q or k [T, H, 128] as [head][half][token][64 columns], v [T, HV, V] as [head][token][columns]
bool key_map(CUtensorMap* map, const void* base, int64_t stride, int total, int heads) {
  const cuuint64_t dims[4] = {64, (cuuint64_t)total, 2, (cuuint64_t)heads}, strides[3] = {(cuuint64_t)stride * 2, 128, 256};
  const cuuint32_t box[4] = {64, kC, 2, 1}, step[4] = {1, 1, 1, 1};
  return tensor_map_encoder()(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void*>(base), dims, strides, box, step,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool value_map(CUtensorMap* map, const void* base, int64_t stride, int total, int heads, int V) {
  const cuuint64_t dims[3] = {(cuuint64_t)V, (cuuint64_t)total, (cuuint64_t)heads}, strides[2] = {(cuuint64_t)stride * 2, (cuuint64_t)V * 2};
  const cuuint32_t box[3] = {32, kC, 1}, step[3] = {1, 1, 1};
  return tensor_map_encoder()(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(base), dims, strides, box, step,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int TILES>
cfb_status launch_tiles(const cfb_gdn_args& g, const int32_t* cu, int total, int B, const float* ws, int* err, const CUtensorMap& q,
                        const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st) {
  using Lay = Scan<T, TILES>;
  if (allow_smem<gdn_scan_kernel<T, TILES>>(Lay::bytes) != cudaSuccess) return cfb_launch_status("gdn_scan_kernel attribute");
  if constexpr (TILES > 2) {                                   // the registers that setmaxnreg shares out are those of the launch
    static const bool enough = [] {
      cudaFuncAttributes a;
      return cudaFuncGetAttributes(&a, gdn_scan_kernel<T, TILES>) == cudaSuccess && a.numRegs >= 96;
    }();
    if (!enough) return CFB_ERR_UNSUPPORTED;
  }
  const dim3 grid((unsigned)(g.V / Lay::kRows), (unsigned)g.HV, (unsigned)B);
  gdn_scan_kernel<T, TILES><<<grid, Lay::kThreads, Lay::bytes, st>>>(g, cu, total, B, ws, err, q, k, v);
  return cfb_launch_status("gdn_scan_kernel");
}
template <typename T>
cfb_status launch_chunks(const cfb_gdn_args& g, const int32_t* cu, int total, int B, float* ws, int* err, cudaStream_t st) {
  if (total == 0) {                                            // states only
    launch_walk(g, cu, total, B, st);
    return cfb_launch_status("gdn_walk_kernel");
  }
  CUtensorMap q, k, v;
  if (!tensor_map_encoder()) return CFB_ERR_CUDA;
  if (!key_map(&q, g.q, g.q_stride, total, g.H) || !key_map(&k, g.k, g.k_stride, total, g.H) ||
      !value_map(&v, g.v, g.v_stride, total, g.HV, g.V))
    return CFB_ERR_INVALID_ARG;
  gdn_prep_kernel<T><<<dim3((unsigned)chunk_slots(total, B), (unsigned)g.HV), 64, 0, st>>>(g, cu, total, B, ws, err);
  if (const cfb_status s = cfb_launch_status("gdn_prep_kernel")) return s;
  // Four tiles a CTA where even so each SM has one and a half and more: more chains side by side, fewer CTAs (32 value
  // heads of 128: nine requests 480 us against 518; one request, 64 CTAs on 148 SMs, would leave half of them idle).
  const bool four = g.V % 64 == 0 && (long long)g.V / 32 * g.HV * B >= 3ll * device_sms();
  return four ? launch_tiles<T, 4>(g, cu, total, B, ws, err, q, k, v, st) : launch_tiles<T, 2>(g, cu, total, B, ws, err, q, k, v, st);
}

}  // namespace

extern "C" cfb_status cfb_gdn_step(const cfb_gdn_args* g, int B, void* stream) {
  if (B == 0 && g) return CFB_OK;
  if (const cfb_status s = check_gdn(g, B, B)) return s;
  launch_walk(*g, nullptr, B, B, static_cast<cudaStream_t>(stream));
  return cfb_launch_status("gdn_walk_kernel");
}

extern "C" size_t cfb_gdn_chunk_workspace(int T, int B, int HV) {
  if (T < 0 || B <= 0 || HV <= 0) return 0;
  return kErrBytes + (size_t)chunk_slots(T, B) * HV * kPrepFloats * sizeof(float);
}

extern "C" cfb_status cfb_gdn_chunk(const cfb_gdn_args* g, const int32_t* cu, int T, int B, void* ws, size_t ws_bytes,
                                    void* stream) {
  if (B == 0 && g) return CFB_OK;
  if (const cfb_status s = check_gdn(g, T, B)) return s;
  if (!cu || !ws) return CFB_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(ws) & 255) || ws_bytes < cfb_gdn_chunk_workspace(T, B, g->HV)) return CFB_ERR_WORKSPACE;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  int* const err = static_cast<int*>(ws);
  float* const prep = reinterpret_cast<float*>(static_cast<char*>(ws) + kErrBytes);
  if (g->dtype == DT_F16) return launch_chunks<__half>(*g, cu, T, B, prep, err, st);
  return launch_chunks<__nv_bfloat16>(*g, cu, T, B, prep, err, st);
}

extern "C" cfb_status cfb_gdn_chunk_error(const void* ws, int* device_error) {
  if (!ws || !device_error) return CFB_ERR_INVALID_ARG;
  if (cudaMemcpy(device_error, ws, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess) return cfb_launch_status("cfb_gdn_chunk_error");
  return CFB_OK;
}
