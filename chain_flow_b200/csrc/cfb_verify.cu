// cfb_verify.cu -- drafted tokens verified against the target's probabilities, from given random
// numbers (sm_100a): a tree or chain without draft probabilities (cfb_tree_verify_sampled) and a chain
// with them (cfb_chain_verify_rejection).
//
// A logits row l at temperature tau has the weights w_i = 2^((l_i - max l) c), c = log2(e) / tau, and a
// number u in [0, 1) draws the first token i with w_0 + .. + w_i > u sum w. A refused draft draws from
// r_i = max(w_i / sum w - q_i, 0) instead. Which token that is, is a whole number, so it has to be the
// one that exact arithmetic gives, although the pass over the row is fp32: the pass carries a bound of
// its error (kBand), and where a sum comes nearer to its threshold than that, the row is taken again in
// 64 bits. A language model's row at temperature 1 has a token of some hundredths where the draw falls,
// so that happens to one row in thousands; rows that are flat over a whole vocabulary pay it always.
//
// One pass over the row: a warp takes 1024 elements in registers, their largest, their weights relative
// to it and the weights' sum, which stay in shared memory (no running rescale: the sums of all such
// units are brought to one base at the end, in 64 bits). The draw then lies in one unit, which is read again
// (from L2) and scanned by one warp. A row is shared by a cluster of CTAs, which exchange their
// totals through distributed shared memory.
//
// Error of the pass, with u = 2^-24 and x = (l - max l) c: an element's exponent is off by 3 u |x| (difference, c,
// product; its unit's base likewise), each of its two exponentials by 4 u, and sums of V weights by 15 u (chains of 8,
// pairs, the warp) and 5 u where the draw's unit is scanned. Under the weights the mean of |x| is their entropy less
// log2 of their sum Z relative to the largest: at most log2(V / Z). What decides is C - t = C - u Z: an error that is
// the same share of every weight cancels in it but for a half. So C - t is off by less than
//   Z u (3 ln 2 log2(V / Z) + (8 + 15) / 2 + 5).
// Rows of 248320 normal logits of deviation 2.5 fall into that band once in ten draws, a language model's less.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <cmath>

#include "cfb_types.cuh"

using namespace cfb;
namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kPerLane = 32;                 // elements of a unit in a lane's registers
constexpr int kUnit = 32 * kPerLane;
constexpr int kMaxCluster = 8;
constexpr int kMaxVocab = 1 << 22;
constexpr int kMaxNodes = 1024;              // draft nodes per request (max_spec_len)
constexpr double kRound = 1.0 / 16777216;    // 2^-24
constexpr float kLowTemp = 1.17549435e-38f;  // 2^-126: below it (or NaN) a request is greedy
constexpr float kHighTemp = 1.26765060e30f;  // 2^100

// a row's token, whether it is the draft that stays, and what its log probability is made of: ln 2 scaled - log(mass)
struct alignas(8) RowResult { int token, accept; double scaled, mass; };

struct VerifyArgs {
  const void* logits; long long ld; int V, num_rows;
  const int32_t* cu_draft; const int32_t* cu_sampled;      // [batch]
  const int32_t* draft_tokens; const int32_t* parents;     // parents: trees only
  const float* probs; long long ld_probs;                  // draft probabilities [drafts, probs_width]
  const int32_t* index_of;                                 // [V] column of a token, or -1; NULL: the token itself
  const void* uniforms; const void* resample; int uniform_size;   // 4 or 8 bytes
  const float* temperature;
  int batch, max_spec, num_drafts;
  int32_t* out_tokens; int32_t* out_path; int32_t* out_len; float* out_logp;
  RowResult* rows;                                         // [num_rows]
  unsigned* counter;                                       // [batch]
  int* err;
};

enum Kind : int { ROW_MASS = 0, ROW_EMPTY = 1, ROW_NAN = 2 };

struct Pub { float top; int nan; double sum; };            // a CTA's part of a row
struct Found { int token, unsure; float logit; int pad; };

struct Shared {
  Pub pub[2];
  Found found[2];
  double z, r;               // of the whole row: sum of weights, of what is left above q
  double before, end;        // the running sum before this CTA's part and behind it
  float top;                 // of the whole row
  int kind;
};

CFB_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
CFB_DEV float warp_max(float v) {                          // NaN counts as nothing
  float m;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
template <typename F> CFB_DEV F warp_sum(F v) {
#pragma unroll
  for (int off = 16; off; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
template <typename F> CFB_DEV F warp_scan(F v, int lane) {  // inclusive
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const F o = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += o;
  }
  return v;
}
// two fp32 operations an instruction
struct Pair { unsigned long long v; };
CFB_DEV Pair pair(float a, float b) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(a), "f"(b));
  return p;
}
CFB_DEV float2 both(Pair p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p.v));
  return f;
}
CFB_DEV Pair add2(Pair a, Pair b) {
  Pair p;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(a.v), "l"(b.v));
  return p;
}
CFB_DEV Pair mul2(Pair a, Pair b) {
  Pair p;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(a.v), "l"(b.v));
  return p;
}

// A logits row: element i lies at p[i]. Vectors of 16 bytes start at element -shift, so that they are aligned.
template <typename T> struct Row {
  const T* p;
  int V, shift;
  float c;                    // log2(e) / tau
  double c64;
  const float* q;             // draft probabilities of the row, or null
  const int32_t* index_of;
};
template <typename T> constexpr int kE = 16 / (int)sizeof(T);          // elements a vector
template <typename T> constexpr int kVectors = kPerLane / kE<T>;       // vectors of a unit a lane

// the first element of a lane's vector j of a unit; elements are in order of (j, lane)
template <typename T> CFB_DEV int first_of(const Row<T>& w, int unit, int j, int lane) {
  return unit * kUnit + (j * 32 + lane) * kE<T> - w.shift;
}
template <typename T> CFB_DEV T lowest();
template <> CFB_DEV float lowest<float>() { return -INFINITY; }
template <> CFB_DEV __half lowest<__half>() { return __ushort_as_half(0xfc00); }
template <> CFB_DEV __nv_bfloat16 lowest<__nv_bfloat16>() { return __ushort_as_bfloat16(0xff80); }
// elements [i, i + kE) as they lie in memory, -inf outside the row
template <typename T> CFB_DEV uint4 load_vector(const Row<T>& w, int i) {
  if (i >= 0 && i + kE<T> <= w.V) return __ldg(reinterpret_cast<const uint4*>(w.p + i));
  union { uint4 v; T e[kE<T>]; } u;
#pragma unroll
  for (int e = 0; e < kE<T>; ++e) u.e[e] = i + e >= 0 && i + e < w.V ? w.p[i + e] : lowest<T>();
  return u.v;
}
template <typename T> CFB_DEV void load_unit(const Row<T>& w, int unit, int lane, uint4 (&u)[kVectors<T>]) {
#pragma unroll
  for (int j = 0; j < kVectors<T>; ++j) u[j] = load_vector(w, first_of(w, unit, j, lane));
}
// element pair k (of kE / 2) of a vector
template <typename T> CFB_DEV float2 pair_of(const uint4& v, int k) {
  const uint32_t s[4] = {v.x, v.y, v.z, v.w};
  if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1]));
  else return unpack16<T>(s[k]);
}
// the largest element of a vector (NaN counts as nothing)
template <typename T> CFB_DEV float vector_max(const uint4& v) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2* h = reinterpret_cast<const T2*>(&v);
    const T2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    const float2 f = unpack16<T>(*reinterpret_cast<const uint32_t*>(&m));
    return fmaxf(f.x, f.y);
  }
}

// weights relative to a base: of a largest +inf the tokens that have it share the mass
CFB_DEV float weight(float l, float base, float c) {
  return l == base ? 1.f : isinf(base) ? 0.f : ex2((l - base) * c);
}
// 2^y for y <= 0 to 10^-14, denormals kept: the series of 2^r, |r| <= 1/2, cut after r^11 (the first term left out is
// 6 10^-15), and the power of two in two factors, since one alone does not reach the denormals. Inlined and without a branch,
// so that several run side by side: the library's function took this pass 4 times as long.
CFB_DEV double exp2_neg(double y) {
  y = fmax(y, -1100.);
  const double magic = 6755399441055744.;                  // 1.5 2^52: adding it rounds to a whole number
  const double shifted = y + magic, r = y - (shifted - magic);
  const int n = __double2loint(shifted), h = n >> 1;
  double p = 0x1.e8cac7351bb25p-32;                       // ln2^k / k!
  p = fma(p, r, 0x1.e4cf5158b8ecap-28);
  p = fma(p, r, 0x1.b5253d395e7c4p-24);
  p = fma(p, r, 0x1.62c0223a5c824p-20);
  p = fma(p, r, 0x1.ffcbfc588b0c7p-17);
  p = fma(p, r, 0x1.430912f86c787p-13);
  p = fma(p, r, 0x1.5d87fe78a6731p-10);
  p = fma(p, r, 0x1.3b2ab6fba4e77p-7);
  p = fma(p, r, 0x1.c6b08d704a0c0p-5);
  p = fma(p, r, 0x1.ebfbdff82c58fp-3);
  p = fma(p, r, 0x1.62e42fefa39efp-1);
  p = fma(p, r, 1.);
  return p * __hiloint2double((1023 + h) << 20, 0) * __hiloint2double((1023 + n - h) << 20, 0);
}
// the fp32 number as a double, by its bits (conversions are slow): what is 0 becomes 2^-127 and -inf -2^128, which
// differ from them by nothing that a weight shows
CFB_DEV double widen(float f) {
  const uint32_t b = __float_as_uint(f);
  return __hiloint2double((int)((b & 0x80000000u) | (((b >> 3) & 0x0fffffffu) + 0x38000000u)), (int)(b << 29));
}
CFB_DEV double weight64(float l, float base, double c64) {
  return l == base ? 1. : isinf(base) ? 0. : exp2_neg(((double)l - (double)base) * c64);
}
// the draft probability of token i (0 outside the row and for what is not a positive number)
template <typename T> CFB_DEV float draft_prob(const Row<T>& w, int i) {
  if (i < 0 || i >= w.V) return 0.f;
  const int at = w.index_of ? __ldg(w.index_of + i) : i;
  return at >= 0 ? fmaxf(__ldg(w.q + at), 0.f) : 0.f;
}

enum Mode : int { W32 = 0, W64 = 1, R32 = 2, R64 = 3 };    // weights, or what is left of them above q
template <int MODE> constexpr bool kNarrow = MODE == W32 || MODE == R32;

// iz: 1 / the row's sum of weights (R32, R64)
template <int MODE, typename T> CFB_DEV auto value_of(const Row<T>& w, float l, int i, float base, double iz) {
  if constexpr (MODE == W32) return weight(l, base, w.c);
  else if constexpr (MODE == W64) return weight64(l, base, w.c64);
  else if constexpr (MODE == R32) return fmaxf(weight(l, base, w.c) * (float)iz - draft_prob(w, i), 0.f);
  else return fmax(weight64(l, base, w.c64) * iz - (double)draft_prob(w, i), 0.);
}

// The part of a row that a CTA has: units [u0, u1) of it
struct Span { int u0, u1; };
template <typename T> CFB_DEV Span span_of(const Row<T>& w, int rank, int ranks) {
  const int units = (w.V + w.shift + kUnit - 1) / kUnit;
  return {(int)((long long)units * rank / ranks), (int)((long long)units * (rank + 1) / ranks)};
}

// every unit's largest and its sum of weights relative to that; a unit's loads are under way while the one before is summed
template <typename T> CFB_DEV void stats_units(const Row<T>& w, Span s, float* tops, double* sums) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint4 next[kVectors<T>];
  if (s.u0 + warp < s.u1) load_unit(w, s.u0 + warp, lane, next);
  for (int u = s.u0 + warp; u < s.u1; u += kWarps) {
    uint4 v[kVectors<T>];
#pragma unroll
    for (int j = 0; j < kVectors<T>; ++j) v[j] = next[j];
    if (u + kWarps < s.u1) load_unit(w, u + kWarps, lane, next);
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kVectors<T>; ++j) m = fmaxf(m, vector_max<T>(v[j]));
    const float top = warp_max(m);
    float sum = 0.f;
    if (fabsf(top) < INFINITY) {
      const Pair base = pair(-top, -top), c = pair(w.c, w.c);
      Pair a[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
      for (int j = 0; j < kVectors<T>; ++j)
#pragma unroll
        for (int k = 0; k < kE<T> / 2; ++k) {
          const float2 l = pair_of<T>(v[j], k);
          const float2 x = both(mul2(add2(pair(l.x, l.y), base), c));
          a[k & 1] = add2(a[k & 1], pair(ex2(x.x), ex2(x.y)));
        }
      const float2 t = both(add2(a[0], a[1]));
      sum = t.x + t.y;
    } else {                                               // +inf, or nothing but -inf; NaN makes the sum NaN
#pragma unroll
      for (int j = 0; j < kVectors<T>; ++j)
#pragma unroll
        for (int k = 0; k < kE<T> / 2; ++k) {
          const float2 l = pair_of<T>(v[j], k);
          sum += l.x != l.x ? l.x : l.x == INFINITY ? 1.f : 0.f;
          sum += l.y != l.y ? l.y : l.y == INFINITY ? 1.f : 0.f;
        }
    }
    sum = warp_sum(sum);
    if (lane == 0) {
      tops[u - s.u0] = top;
      sums[u - s.u0] = sum;
    }
  }
}

// eight or four entries of a table from entry i on, in 16-byte loads where they are aligned; entries outside are not read
template <typename F> CFB_DEV void table_entries(const F* t, int i, int n, int V, F (&x)[8], F none) {
  if (i >= 0 && i + n <= V && (reinterpret_cast<uintptr_t>(t + i) & 15) == 0) {
    for (int e = 0; e < n; e += 4) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(t + i + e));
      x[e] = *reinterpret_cast<const F*>(&v.x); x[e + 1] = *reinterpret_cast<const F*>(&v.y);
      x[e + 2] = *reinterpret_cast<const F*>(&v.z); x[e + 3] = *reinterpret_cast<const F*>(&v.w);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) x[e] = i + e >= 0 && i + e < V ? __ldg(t + i + e) : none;
  }
}

// every unit's sum of what is left above q
template <typename T> CFB_DEV void rest_units(const Row<T>& w, Span s, float base, float iz, double* sums) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int u = s.u0 + warp; u < s.u1; u += kWarps) {
    uint4 v[kVectors<T>];
    load_unit(w, u, lane, v);
    float a[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kVectors<T>; ++j) {
      const int i = first_of(w, u, j, lane);
      float q[8];
      if (w.index_of) {
        int at[8];
        table_entries(w.index_of, i, kE<T>, w.V, at, -1);
#pragma unroll
        for (int e = 0; e < kE<T>; ++e) q[e] = at[e] >= 0 ? __ldg(w.q + at[e]) : 0.f;
      } else {
        table_entries(w.q, i, kE<T>, w.V, q, 0.f);
      }
#pragma unroll
      for (int k = 0; k < kE<T> / 2; ++k) {
        const float2 l = pair_of<T>(v[j], k);
        a[0] += fmaxf(weight(l.x, base, w.c) * iz - fmaxf(q[2 * k], 0.f), 0.f);
        a[1] += fmaxf(weight(l.y, base, w.c) * iz - fmaxf(q[2 * k + 1], 0.f), 0.f);
      }
    }
    const float sum = warp_sum(a[0] + a[1]);
    if (lane == 0) sums[u - s.u0] = sum;
  }
}
// every unit's sum in 64 bits
template <int MODE, typename T> CFB_DEV void exact_units(const Row<T>& w, Span s, float base, double iz, double* sums) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const double top = base;
  for (int u = s.u0 + warp; u < s.u1; u += kWarps) {
    double a[2] = {0., 0.};
    if (isinf(base) || MODE == R64) {
#pragma unroll 1
      for (int k = 0; k < kPerLane; ++k) {
        const int i = u * kUnit + k * 32 + lane - w.shift;
        if (i >= 0 && i < w.V) a[0] += value_of<MODE>(w, to_float(w.p[i]), i, base, iz);
      }
    } else {
#pragma unroll 1
      for (int j = 0; j < kVectors<T>; ++j) {
        const uint4 v = load_vector(w, first_of(w, u, j, lane));
#pragma unroll
        for (int k = 0; k < kE<T> / 2; ++k) {
          const float2 l = pair_of<T>(v, k);
          a[0] += exp2_neg((widen(l.x) - top) * w.c64);
          a[1] += exp2_neg((widen(l.y) - top) * w.c64);
        }
      }
    }
    const double sum = warp_sum(a[0] + a[1]);
    if (lane == 0) sums[u - s.u0] = sum;
  }
}

// Warp 0: the units' sums become running ones
CFB_DEV double run_up(double* sums, int n, int lane) {
  double before = 0.;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const double v = warp_scan(i0 + lane < n ? sums[i0 + lane] : 0., lane);
    if (i0 + lane < n) sums[i0 + lane] = before + v;
    before += __shfl_sync(0xffffffffu, v, 31);
  }
  __syncwarp();
  return before;
}

// Warp 0: the first token of this CTA's part whose running sum passes t (relative to the part's start). A lane takes 32
// neighbours of the unit that holds it. The fp32 modes sum in fp32 inside the unit: 37 additions in a row at most,
// another 2^-18 of the unit's mass.
template <int MODE, typename T>
CFB_DEV Found find(const Row<T>& w, Span s, const double* sums, double t, float base, double iz, double band) {
  using F = typename std::conditional<kNarrow<MODE>, float, double>::type;
  constexpr int kRoll = kNarrow<MODE> ? kPerLane : 1;
  const int lane = threadIdx.x & 31, n = s.u1 - s.u0;
  int u = -1;
  for (int i0 = 0; i0 < n && u < 0; i0 += 32) {
    const unsigned hit = __ballot_sync(0xffffffffu, i0 + lane < n && sums[i0 + lane] > t);
    if (hit) u = i0 + __ffs(hit) - 1;
  }
  bool unsure = false;
  if (u < 0) {                                             // rounding put the threshold past the end: the last unit with mass
    unsure = true;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + lane;
      const unsigned hit = __ballot_sync(0xffffffffu, i < n && sums[i] > (i ? sums[i - 1] : 0.));
      if (hit) u = i0 + 31 - __clz(hit);
    }
    if (u < 0) return {-1, 1, 0.f, 0};
  }
  t -= u ? sums[u - 1] : 0.;
  const int i0 = (s.u0 + u) * kUnit + lane * kPerLane - w.shift;
  uint4 v[kVectors<T>];
  if constexpr (kNarrow<MODE>)
#pragma unroll
    for (int j = 0; j < kVectors<T>; ++j) v[j] = load_vector(w, i0 + j * kE<T>);
  const auto logit = [&](int e) {
    if constexpr (kNarrow<MODE>) {
      const float2 l = pair_of<T>(v[e / kE<T>], e % kE<T> / 2);
      return e & 1 ? l.y : l.x;
    } else {
      return i0 + e >= 0 && i0 + e < w.V ? to_float(w.p[i0 + e]) : -INFINITY;
    }
  };
  F x[kNarrow<MODE> ? kPerLane : 1], a = 0;
  int last = -1;                                           // this lane's last token with mass
#pragma unroll kRoll
  for (int e = 0; e < kPerLane; ++e) {
    const F y = value_of<MODE>(w, logit(e), i0 + e, base, iz);
    if constexpr (kNarrow<MODE>) x[e] = y;
    a += y;
    if (y > 0) last = e;
  }
  const F scan = warp_scan(a, lane), up = __shfl_up_sync(0xffffffffu, scan, 1);
  const unsigned some = __ballot_sync(0xffffffffu, a > 0);
  unsigned hit = __ballot_sync(0xffffffffu, a > 0 && (double)scan > t);
  if (!hit) {                                              // as above, inside the unit
    if (!some) return {-1, 1, 0.f, 0};
    unsure = true;
    hit = 1u << (31 - __clz(some));
  }
  const int who = __ffs(hit) - 1;
  int token = -1;
  float l = 0.f;
  F run = lane ? up : (F)0, lo = 0, hi = 0;
  if (lane == who) {
#pragma unroll kRoll
    for (int e = 0; e < kPerLane; ++e) {
      F y;
      if constexpr (kNarrow<MODE>) y = x[e];
      else y = value_of<MODE>(w, logit(e), i0 + e, base, iz);
      if (token < 0 && y > 0 && ((double)(run + y) > t || e == last)) {
        token = i0 + e;
        l = logit(e);
        lo = run;
        hi = run + y;
      }
      run += y;
    }
  }
  unsure |= !(t - (double)lo >= band && (double)hi - t >= band);
  return {__shfl_sync(0xffffffffu, token, who), (int)__shfl_sync(0xffffffffu, (int)unsure, who), __shfl_sync(0xffffffffu, l, who), 0};
}

// Warp 0: the first element that equals the row's largest (or the first NaN)
template <typename T>
CFB_DEV int find_top(const Row<T>& w, Span s, const float* tops, const double* sums, float top, bool nan) {
  const int lane = threadIdx.x & 31, n = s.u1 - s.u0;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int k = i0 + lane;
    const unsigned hit = __ballot_sync(0xffffffffu, k < n && (nan ? sums[k] != sums[k] : tops[k] == top));
    if (!hit) continue;
    const int u = s.u0 + i0 + __ffs(hit) - 1;
    uint4 v[kVectors<T>];
    load_unit(w, u, lane, v);
    int best = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < kVectors<T>; ++j)
#pragma unroll
      for (int e = 0; e < kE<T>; ++e) {
        const float2 l = pair_of<T>(v[j], e / 2);
        const float x = e & 1 ? l.y : l.x;
        const int i = first_of(w, u, j, lane) + e;
        if (i >= 0 && i < w.V && (nan ? x != x : x == top)) best = min(best, i);
      }
    return __reduce_min_sync(0xffffffffu, best);
  }
  return -1;
}

// What a cluster finds of a row. `ph` alternates the exchanged buffers.
template <typename T> struct Team {
  Shared* sh;
  float* tops;
  double* sums;
  int rank, ranks, ph;

  // this CTA's part, handed to the others by the next cluster barrier
  CFB_DEV void publish(float top, int nan, double sum) {
    sh->pub[ph] = {top, nan, sum};
    sh->found[ph] = {-1, 1, 0.f, 0};                       // kept where no part has the threshold
  }

  // totals of all CTAs -> the row's, and what lies before this one's part. `scaled`: each relative to its own largest
  CFB_DEV void exchange(float c, bool scaled, double* whole) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (threadIdx.x < 32) {
      const int lane = threadIdx.x;
      Pub p{-INFINITY, 0, 0.};
      if (lane < ranks) p = *cluster.map_shared_rank(&sh->pub[ph], lane);
      if (scaled) {
        const float top = warp_max(p.top);
        const bool nan = __any_sync(0xffffffffu, p.nan);
        if (lane == 0) {
          sh->top = top;
          sh->kind = nan ? ROW_NAN : top == -INFINITY ? ROW_EMPTY : ROW_MASS;
        }
        p.sum *= p.top == -INFINITY ? 0. : (double)weight(p.top, top, c);
      }
      double scan = p.sum;
#pragma unroll
      for (int off = 1; off < kMaxCluster; off <<= 1) {
        const double o = __shfl_up_sync(0xffffffffu, scan, off);
        if (lane >= off) scan += o;
      }
      // (the sum before, not the one behind less this part's, which would lose small ones)
      const double before = __shfl_up_sync(0xffffffffu, scan, 1);
      if (lane == rank) {
        sh->before = rank ? before : 0.;
        sh->end = scan;
      }
      if (lane == kMaxCluster - 1) *whole = scan;
    }
    __syncthreads();
  }

  // the pass over the row
  CFB_DEV void stats(const Row<T>& w) {
    const Span s = span_of(w, rank, ranks);
    stats_units(w, s, tops, sums);
    __syncthreads();
    ph ^= 1;
    if (threadIdx.x < 32) {
      const int lane = threadIdx.x, n = s.u1 - s.u0;
      float top = -INFINITY;
      bool nan = false;
      for (int i = lane; i < n; i += 32) {
        top = fmaxf(top, tops[i]);
        nan |= sums[i] != sums[i];
      }
      top = warp_max(top);
      nan = __any_sync(0xffffffffu, nan);
      double sum = 0.;
      if (!nan) {
        for (int i = lane; i < n; i += 32) sums[i] *= tops[i] == -INFINITY ? 0. : (double)weight(tops[i], top, w.c);
        __syncwarp();
        sum = run_up(sums, n, lane);
      }
      if (lane == 0) publish(top, nan, sum);
    }
    exchange(w.c, true, &sh->z);
  }

  // a pass that knows the row's largest
  template <int MODE> CFB_DEV void pass(const Row<T>& w, double* whole) {
    const Span s = span_of(w, rank, ranks);
    if constexpr (MODE == R32) rest_units(w, s, sh->top, (float)(1. / sh->z), sums);
    else exact_units<MODE>(w, s, sh->top, 1. / sh->z, sums);
    __syncthreads();
    ph ^= 1;
    if (threadIdx.x < 32) {
      const double sum = run_up(sums, s.u1 - s.u0, threadIdx.x);
      if (threadIdx.x == 0) publish(sh->top, 0, sum);
    }
    exchange(w.c, false, whole);
  }

  // Warp 0 of the CTA that found it hands it to all
  CFB_DEV Found share(bool mine, Found f) {
    cg::cluster_group cluster = cg::this_cluster();
    if (mine && threadIdx.x < ranks) *cluster.map_shared_rank(&sh->found[ph], (int)threadIdx.x) = f;
    cluster.sync();
    return sh->found[ph];
  }

  // the draw of threshold u among the running sums of the last pass, whose whole is `whole`
  template <int MODE> CFB_DEV Found draw(const Row<T>& w, double u, double whole) {
    bool mine = false;
    Found f{-1, 1, 0.f, 0};
    if (threadIdx.x < 32) {
      const Pub own = sh->pub[ph];
      const double t = fmin(u * whole, whole * (1. - 2.220446049250313e-16));
      // relative to the base of this CTA's sums
      const double scale = MODE == W32 ? (own.top == -INFINITY ? 0. : (double)weight(own.top, sh->top, w.c)) : 1.;
      mine = own.sum * scale > 0. && sh->before <= t && (t < sh->end || last_with_mass(w.c, MODE == W32));
      // (of what is left above q, the error is that of the probabilities, whose whole is 1)
      if (mine)
        f = find<MODE>(w, span_of(w, rank, ranks), sums, (t - sh->before) / scale, MODE == W32 ? own.top : sh->top, 1. / sh->z,
                       MODE == W32 ? band(w) * whole / scale : MODE == R32 ? band(w) + 24 * kRound : 0.);
    }
    return share(mine, f);
  }
  // how far a sum may be from its threshold's side, as a share of the row's mass (from what is left above q: and the
  // probabilities' own rounding)
  CFB_DEV double band(const Row<T>& w) const { return kRound * (2.08 * (double)__log2f((float)w.V / (float)sh->z) + 17.); }
  // no later part has any
  CFB_DEV bool last_with_mass(float c, bool scaled) {
    for (int r = rank + 1; r < ranks; ++r) {
      const Pub p = *cg::this_cluster().map_shared_rank(&sh->pub[ph], r);
      if (p.sum > 0. && (!scaled || weight(p.top, sh->top, c) > 0.f)) return false;
    }
    return true;
  }

  // the first of the row's largest
  CFB_DEV int top_token(const Row<T>& w, bool nan) {
    bool mine = false;
    Found f{-1, 0, 0.f, 0};
    if (threadIdx.x < 32) {
      mine = nan ? sh->pub[ph].nan : sh->pub[ph].top == sh->top;
      for (int r = 0; r < rank && mine; ++r) {
        const Pub p = *cg::this_cluster().map_shared_rank(&sh->pub[ph], r);
        mine = !(nan ? p.nan != 0 : p.top == sh->top);
      }
      if (mine) f.token = find_top(w, span_of(w, rank, ranks), tops, sums, sh->top, nan);
    }
    return share(mine, f).token;
  }
};

// the draw in 64 bits, and the alternation of the exchanged buffers after it. rest: from what is left above q
struct Exact { Found f; int ph; };
template <typename T>
__device__ __noinline__ Exact exact_draw(Team<T> team, Row<T> w, bool rest, double v) {
  Shared& sh = *team.sh;
  team.template pass<W64>(w, &sh.z);
  if (rest) {
    team.template pass<R64>(w, &sh.r);
    if (sh.r > 0.) {
      const Found f = team.template draw<R64>(w, v, sh.r);
      return {f, team.ph};
    }
    team.template pass<W64>(w, &sh.z);                     // nothing above q: the target's own
  }
  const Found f = team.template draw<W64>(w, v, sh.z);
  return {f, team.ph};
}
// the sum of the row's weights in 64 bits
template <typename T> __device__ __noinline__ int exact_sum(Team<T> team, Row<T> w) {
  team.template pass<W64>(w, &team.sh->z);
  return team.ph;
}

// One row, by a whole cluster; every thread gets the result. drafted: the row has a draft with probabilities, `draft`,
// which u accepts; v draws.
template <bool CHAIN, typename T>
CFB_DEV RowResult resolve(Team<T>& team, const Row<T>& w, bool greedy, bool drafted, int draft, double u, double v) {
  Shared& sh = *team.sh;
  const bool in = CHAIN && drafted && draft >= 0 && draft < w.V;       // a draft that is no token is refused
  const float of_draft = in ? to_float(w.p[draft]) : -INFINITY;
  const double uq = in ? u * (double)draft_prob(w, draft) : 0.;
  team.stats(w);
  const auto scaled = [&](float l) { return l == sh.top ? 0. : ((double)l - (double)sh.top) * w.c64; };     // log2
  if (sh.kind == ROW_EMPTY) return {-1, 0, 0., 1.};
  if (greedy || sh.kind == ROW_NAN) {
    const int t = team.top_token(w, sh.kind == ROW_NAN);
    return {t, drafted && t == draft, sh.kind == ROW_NAN ? (double)NAN : 0., sh.z};
  }
  Found f{-1, 1, 0.f, 0};
  if constexpr (CHAIN) {
    if (drafted) {
      if (in) {
        double p = (double)weight(of_draft, sh.top, w.c) / sh.z;
        // (every CTA computes the same)
        if (fabs(uq - p) <= p * (2. * team.band(w) + kRound * (2.08 * fabs(scaled(of_draft)) + 8.))) {
          team.ph = exact_sum(team, w);
          p = weight64(of_draft, sh.top, w.c64) / sh.z;
        }
        if (uq < p) return {draft, 1, scaled(of_draft), sh.z};
      }
      team.template pass<R32>(w, &sh.r);
      if (sh.r > 2. * team.band(w) + 48 * kRound) f = team.template draw<R32>(w, v, sh.r);
    } else {
      f = team.template draw<W32>(w, v, sh.z);
    }
  } else {
    f = team.template draw<W32>(w, v, sh.z);
  }
  if (f.unsure) {
    const Exact e = exact_draw(team, w, drafted, v);
    f = e.f;
    team.ph = e.ph;
  }
  return {f.token, 0, scaled(f.logit), sh.z};
}

CFB_DEV double number_at(const void* p, int size, long long i) {
  const double u = size == 4 ? (double)static_cast<const float*>(p)[i] : static_cast<const double*>(p)[i];
  return fmin(fmax(u, 0.), 1. - 0x1p-32);                  // (an upper end that sums of 64 bits still resolve)
}

template <typename T> CFB_DEV Row<T> row_of(const VerifyArgs& A, int row, float temp, bool greedy) {
  Row<T> w;
  w.p = static_cast<const T*>(A.logits) + (long long)row * A.ld;
  w.V = A.V;
  w.shift = (int)((reinterpret_cast<uintptr_t>(w.p) & 15) / sizeof(T));
  const float tau = greedy ? 1.f : fminf(temp, kHighTemp);
  w.c64 = 1.4426950408889634 / (double)tau;
  w.c = (float)fmin(w.c64, 3.4e38);
  w.q = nullptr;
  w.index_of = A.index_of;
  return w;
}

// FLAT: a cluster a row (grid.y: rows of a request, grid.z: requests), every row at once; the request's last
// cluster walks. Otherwise a cluster a request (grid.y), which takes the rows of its walk in turn.
// CHAIN: draft probabilities; a node's only child is the next one.
template <typename T, bool CHAIN, bool FLAT>
__global__ void __launch_bounds__(kThreads, 2) verify_kernel(const VerifyArgs A, int most) {
  extern __shared__ double s_dyn[];
  __shared__ Shared sh;
  __shared__ int s_last;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  // what a walk keeps: the results of its rows (in turn, or FLAT: of all rows), the rows it took, the tree
  RowResult* const s_row = reinterpret_cast<RowResult*>(s_dyn + most);
  int* const s_node = reinterpret_cast<int*>(s_row + A.max_spec + 1);
  int* const s_parent = s_node + A.max_spec + 1;
  int* const s_token = s_parent + A.max_spec;
  Team<T> team{&sh, reinterpret_cast<float*>(s_token + A.max_spec), s_dyn, rank, ranks, 0};
  const int b = FLAT ? blockIdx.z : blockIdx.y;
  const int d0 = b ? A.cu_draft[b - 1] : 0;
  const long long drafts = (long long)A.cu_draft[b] - d0, start = A.cu_sampled[b] - (drafts + 1);
  const float temp = A.temperature ? A.temperature[b] : 1.f;
  // offsets that do not describe rows of this logits matrix (or drafts) are never dereferenced
  const bool sane = drafts >= 0 && drafts <= A.max_spec && start >= 0 && start + drafts < A.num_rows && d0 >= 0 &&
                    d0 + drafts <= A.num_drafts;
  const int n = (int)drafts, s0 = (int)start;
  const bool greedy = !(temp >= kLowTemp);
  const auto take = [&](int j) {                           // row j of the request
    Row<T> w = row_of<T>(A, s0 + j, temp, greedy);
    if constexpr (CHAIN) {
      const bool drafted = j < n;
      if (drafted) w.q = A.probs + (long long)(d0 + j) * A.ld_probs;
      return resolve<true>(team, w, greedy, drafted, drafted ? A.draft_tokens[d0 + j] : -1,
                           drafted ? number_at(A.uniforms, A.uniform_size, d0 + j) : 0., number_at(A.resample, A.uniform_size, b));
    } else {
      return resolve<false>(team, w, greedy, false, -1, 0., number_at(A.uniforms, A.uniform_size, s0 + j));
    }
  };
  if constexpr (FLAT) {
    const int j = blockIdx.y;
    if (sane && j <= n) {
      const RowResult r = take(j);
      if (rank == 0 && threadIdx.x == 0) A.rows[s0 + j] = r;
      cluster.sync();                                      // no CTA ends while another reads its shared memory
    }
    if (rank != 0) return;
    if (threadIdx.x == 0) {
      __threadfence();
      const unsigned prev = atomicAdd(A.counter + b, 1u);
      s_last = prev + 1 == gridDim.y;
      if (s_last) { __threadfence(); A.counter[b] = 0u; }
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    if (sane)
      for (int i = threadIdx.x; i <= n; i += kThreads) {
        const RowResult* const r = A.rows + s0 + i;
        const int2 t = __ldcg(reinterpret_cast<const int2*>(r));
        s_row[i] = {t.x, t.y, __ldcg(&r->scaled), __ldcg(&r->mass)};
      }
  }
  int pos = -1;                                            // the last token's place: accepted drafts
  if (sane) {
    for (int i = threadIdx.x; !CHAIN && i < n; i += kThreads) {
      s_parent[i] = A.parents[d0 + i];
      s_token[i] = A.draft_tokens[d0 + i];
    }
    __syncthreads();
    int cur = -1;
    for (;;) {                                             // (every thread of every CTA takes the same steps)
      RowResult r;
      if constexpr (FLAT) r = s_row[cur + 1];
      else r = take(cur + 1);
      ++pos;
      if (threadIdx.x == 0) {
        s_node[pos] = cur;
        if constexpr (!FLAT) s_row[pos] = r;
      }
      int nxt = -1;
      if (pos < A.max_spec && r.token >= 0) {
        if constexpr (CHAIN) {
          nxt = r.accept && cur + 1 < n ? cur + 1 : -1;
        } else {                                           // the first child of cur that carries the token
          for (int i0 = 0; i0 < n && nxt < 0; i0 += 32) {
            const int i = i0 + (int)(threadIdx.x & 31);
            const unsigned hit = __ballot_sync(0xffffffffu, i < n && s_parent[i] == cur && s_token[i] == r.token);
            if (hit) nxt = i0 + __ffs(hit) - 1;
          }
        }
      }
      if (nxt < 0) break;
      cur = nxt;
    }
    if constexpr (!FLAT) cluster.sync();
    __syncthreads();
  }
  if (rank != 0) return;
  for (int p = threadIdx.x; p <= A.max_spec; p += kThreads) {
    int token = -1;
    float logp = 0.f;
    if (p <= pos) {
      const RowResult r = s_row[FLAT ? s_node[p] + 1 : p];
      token = r.token;
      if (token >= 0) logp = (float)(r.scaled * 0.6931471805599453 - log(r.mass));
    }
    A.out_tokens[(long long)b * (A.max_spec + 1) + p] = token;
    A.out_logp[(long long)b * (A.max_spec + 1) + p] = logp;
    if constexpr (!CHAIN)
      if (p < A.max_spec) A.out_path[(long long)b * A.max_spec + p] = p < pos ? s_node[p + 1] : -1;
  }
  if (threadIdx.x == 0) {
    A.out_len[b] = max(pos, 0);
    if (!sane && A.err) atomicCAS(A.err, 0, DEV_BAD_INDEX);      // inconsistent offsets: emit nothing, flag it
  }
}

template <typename T, bool CHAIN, bool FLAT>
cfb_status launch(const VerifyArgs& a, int cluster, cudaStream_t st) {
  const auto bytes = [](long long units, long long spec) { return (int)(units * 12 + (spec + 1) * 28 + spec * 8); };
  const long long units = (a.V + 7 + kUnit - 1) / kUnit, most = (units + cluster - 1) / cluster + 1;
  if (allow_smem<verify_kernel<T, CHAIN, FLAT>>(bytes(kMaxVocab / kUnit + 2, kMaxNodes)) != cudaSuccess)
    return cfb_launch_status("verify_kernel");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = FLAT ? dim3(cluster, a.max_spec + 1, a.batch) : dim3(cluster, a.batch, 1);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes(most, a.max_spec);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, verify_kernel<T, CHAIN, FLAT>, a, (int)most);
  return cfb_launch_status("verify_kernel");
}

template <bool CHAIN> cfb_status launch_as(const VerifyArgs& a, int dtype, cudaStream_t st) {
  const int sms = device_sms() > 0 ? device_sms() : 148;
  const long long row = (long long)a.V * (dtype == DT_F32 ? 4 : 2);
  const bool flat = row * a.num_rows <= (64ll << 20);
  // clusters of as many CTAs as the rows at hand leave SMs for
  const long long teams = flat ? a.num_rows : a.batch;
  int cluster = kMaxCluster;
  while (cluster > 1 && teams * cluster > 2 * sms) cluster >>= 1;
  const auto go = [&](auto t) {
    using T = decltype(t);
    return flat ? launch<T, CHAIN, true>(a, cluster, st) : launch<T, CHAIN, false>(a, cluster, st);
  };
  if (dtype == DT_F32) return go(float{});
  if (dtype == DT_F16) return go(__half{});
  return go(__nv_bfloat16{});
}

// what both entry points check, and their common arguments
cfb_status common_args(VerifyArgs& a, const void* logits, int64_t ld, int num_rows, int V, int dtype, const int32_t* cu_draft,
                       const int32_t* cu_sampled, const int32_t* draft_tokens, const void* uniforms, int uniform_size,
                       const float* temperature, int num_drafts, int batch, int max_spec, int32_t* out_tokens, int32_t* out_len,
                       float* out_logp, void* ws, size_t ws_bytes, int* err) {
  if (num_rows <= 0 || V <= 0 || batch <= 0 || max_spec < 0 || ld < V) return CFB_ERR_INVALID_ARG;
  if (!logits || !cu_draft || !cu_sampled || !out_tokens || !out_len || !out_logp || !ws) return CFB_ERR_INVALID_ARG;
  if (num_drafts < 0 || (num_drafts > 0 && !draft_tokens)) return CFB_ERR_INVALID_ARG;
  if (dtype < DT_F32 || dtype > DT_BF16 || (uniform_size != 4 && uniform_size != 8)) return CFB_ERR_UNSUPPORTED;
  if (max_spec > kMaxNodes || V > kMaxVocab - 8 || batch > 65535) return CFB_ERR_UNSUPPORTED;
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == DT_F32 ? 4 : 2)) return CFB_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(ws) & 255) || ws_bytes < cfb_verify_workspace(num_rows, batch)) return CFB_ERR_WORKSPACE;
  a.logits = logits; a.ld = ld; a.V = V; a.num_rows = num_rows;
  a.cu_draft = cu_draft; a.cu_sampled = cu_sampled; a.draft_tokens = draft_tokens;
  a.uniforms = uniforms; a.uniform_size = uniform_size; a.temperature = temperature;
  a.num_drafts = num_drafts; a.batch = batch; a.max_spec = max_spec;
  a.out_tokens = out_tokens; a.out_len = out_len; a.out_logp = out_logp;
  a.counter = static_cast<unsigned*>(ws);
  a.rows = reinterpret_cast<RowResult*>(static_cast<char*>(ws) + ((size_t)batch * 4 + 255) / 256 * 256);
  a.err = err;
  return CFB_OK;
}

}  // namespace

extern "C" size_t cfb_verify_workspace(int num_rows, int batch) {
  if (num_rows <= 0 || batch <= 0) return 0;
  return ((size_t)batch * 4 + 255) / 256 * 256 + (size_t)num_rows * sizeof(RowResult);
}

extern "C" cfb_status cfb_tree_verify_sampled(const void* logits, int64_t ld, int num_rows, int V, int dtype,
                                              const int32_t* cu_num_draft, const int32_t* cu_num_sampled,
                                              const int32_t* draft_tokens, const int32_t* parents, int num_drafts,
                                              const void* uniforms, int uniform_size, const float* temperature, int batch,
                                              int max_spec_len,
                                              int32_t* output_tokens, int32_t* accepted_path, int32_t* accepted_len,
                                              float* logprobs, void* ws, size_t ws_bytes, int* err, void* stream) {
  VerifyArgs a{};
  if (const cfb_status s = common_args(a, logits, ld, num_rows, V, dtype, cu_num_draft, cu_num_sampled, draft_tokens, uniforms,
                                       uniform_size, temperature, num_drafts, batch, max_spec_len, output_tokens, accepted_len,
                                       logprobs, ws, ws_bytes, err))
    return s;
  if (!uniforms || (num_drafts > 0 && !parents) || (max_spec_len > 0 && !accepted_path)) return CFB_ERR_INVALID_ARG;
  a.parents = parents;
  a.out_path = accepted_path;
  return launch_as<false>(a, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" cfb_status cfb_chain_verify_rejection(const void* logits, int64_t ld, int num_rows, int V, int dtype,
                                                 const int32_t* cu_num_draft, const int32_t* cu_num_sampled,
                                                 const int32_t* draft_tokens, const float* draft_probs, int64_t ld_probs,
                                                 int num_drafts, int probs_width, const int32_t* index_of,
                                                 const void* uniforms, const void* resample, int uniform_size,
                                                 const float* temperature, int batch, int max_spec_len,
                                                 int32_t* output_tokens, int32_t* accepted_len, float* logprobs, void* ws,
                                                 size_t ws_bytes, int* err, void* stream) {
  VerifyArgs a{};
  if (const cfb_status s = common_args(a, logits, ld, num_rows, V, dtype, cu_num_draft, cu_num_sampled, draft_tokens, uniforms,
                                       uniform_size, temperature, num_drafts, batch, max_spec_len, output_tokens, accepted_len,
                                       logprobs, ws, ws_bytes, err))
    return s;
  if (probs_width <= 0 || ld_probs < probs_width || !resample || (num_drafts > 0 && (!draft_probs || !uniforms))) return CFB_ERR_INVALID_ARG;
  if (!index_of && probs_width != V) return CFB_ERR_INVALID_ARG;
  a.probs = draft_probs;
  a.ld_probs = ld_probs;
  a.index_of = index_of;
  a.resample = resample;
  return launch_as<true>(a, dtype, static_cast<cudaStream_t>(stream));
}
