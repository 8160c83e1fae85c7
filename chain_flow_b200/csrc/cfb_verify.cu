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
// Error of the pass, relative to sum w: an element's exponent x is off by 3 2^-24 |x| (difference,
// c, product), a unit's base the same, each exponential by 2^-22, a unit's sum by 15 2^-24 (chains of 8,
// then pairs). The mean of |x| under w is at most log2 V <= 22, so a sum is off by at most
// (3 ln 2 22 + 8 + 15) 2^-24 < 2^-17, and the difference of a sum and its threshold by twice that.
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
constexpr double kBand = 1.0 / 65536;        // 2^-16
constexpr float kLowTemp = 1.17549435e-38f;  // 2^-126: below it (or NaN) a request is greedy
constexpr float kHighTemp = 1.26765060e30f;  // 2^100

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
  int32_t* row_token; float* row_logp; int32_t* row_accept;       // [num_rows]
  unsigned* counter;                                              // [batch]
  int* err;
};

enum Kind : int { ROW_MASS = 0, ROW_EMPTY = 1, ROW_NAN = 2 };

struct Pub { float top; int nan; double sum; };            // a CTA's part of a row
struct Found { int token; int unsure; };

struct Shared {
  Pub pub[2];
  Found found[2];
  double z, r;               // of the whole row: sum of weights, of what is left above q
  double before, end;        // the running sum before this CTA's part and behind it
  float top;                 // of the whole row
  int kind, owner;
};

CFB_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
CFB_DEV float warp_max(float v) {
#pragma unroll
  for (int off = 16; off; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}
template <typename F> CFB_DEV F warp_sum(F v) {
#pragma unroll
  for (int off = 16; off; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
CFB_DEV double warp_scan(double v, int lane) {             // inclusive
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const double o = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += o;
  }
  return v;
}

// A logits row: element i lies at p[i]. Vectors of 16 bytes start at element -shift, so that they are aligned.
template <typename T> struct Row {
  const T* p;
  int V, shift;
  float c;                    // log2(e) / tau
  double inv_tau;
  const float* q;             // draft probabilities of the row, or null
  const int32_t* index_of;
};

// elements of a lane in a unit, in order of (j, lane, e); outside the row -inf
template <typename T> CFB_DEV int first_of(const Row<T>& w, int unit, int j, int lane) {
  constexpr int E = 16 / (int)sizeof(T);
  return unit * kUnit + (j * 32 + lane) * E - w.shift;
}
template <typename T> CFB_DEV void unpack(const uint4& u, float* x) {
  const uint32_t s[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = unpack16<T>(s[e]);
    x[2 * e] = f.x;
    x[2 * e + 1] = f.y;
  }
}
template <> CFB_DEV void unpack<float>(const uint4& u, float* x) {
  x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y); x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
}
template <typename T> CFB_DEV void load_unit(const Row<T>& w, int unit, int lane, float (&x)[kPerLane]) {
  constexpr int E = 16 / (int)sizeof(T), NV = kPerLane / E;
  uint4 u[NV];
  bool whole[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int i = first_of(w, unit, j, lane);
    whole[j] = i >= 0 && i + E <= w.V;
    if (whole[j]) u[j] = __ldg(reinterpret_cast<const uint4*>(w.p + i));
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (whole[j]) {
      unpack<T>(u[j], x + j * E);
    } else {
      const int i = first_of(w, unit, j, lane);
#pragma unroll
      for (int e = 0; e < E; ++e) x[j * E + e] = i + e >= 0 && i + e < w.V ? to_float(w.p[i + e]) : -INFINITY;
    }
  }
}
// the draft probability of token i (0 outside the row and for what is not a positive number)
template <typename T> CFB_DEV float draft_prob(const Row<T>& w, int i) {
  if (i < 0 || i >= w.V) return 0.f;
  const int at = w.index_of ? __ldg(w.index_of + i) : i;
  return at >= 0 ? fmaxf(__ldg(w.q + at), 0.f) : 0.f;
}

// weights relative to a base: of a largest +inf the tokens that have it share the mass
CFB_DEV float weight(float l, float base, float c) {
  return l == base ? 1.f : isinf(base) ? 0.f : ex2((l - base) * c);
}
CFB_DEV double weight64(float l, float base, double inv_tau) {
  return l == base ? 1. : isinf(base) ? 0. : exp(((double)l - (double)base) * inv_tau);
}

enum Mode : int { W32 = 0, W64 = 1, R32 = 2, R64 = 3 };    // weights, or what is left of them above q

template <int MODE> constexpr bool kNarrow = MODE == W32 || MODE == R32;

// iz: 1 / the row's sum of weights (R32, R64)
template <int MODE, typename T> CFB_DEV auto value_of(const Row<T>& w, float l, int i, float base, double iz) {
  if constexpr (MODE == W32) return weight(l, base, w.c);
  else if constexpr (MODE == W64) return weight64(l, base, w.inv_tau);
  else if constexpr (MODE == R32) return fmaxf(weight(l, base, w.c) * (float)iz - draft_prob(w, i), 0.f);
  else return fmax(weight64(l, base, w.inv_tau) * iz - (double)draft_prob(w, i), 0.);
}

// The part of a row that a CTA has: units [u0, u1) of it
struct Span { int u0, u1; };
template <typename T> CFB_DEV Span span_of(const Row<T>& w, int rank, int ranks) {
  const int units = (w.V + w.shift + kUnit - 1) / kUnit;
  return {(int)((long long)units * rank / ranks), (int)((long long)units * (rank + 1) / ranks)};
}

// every unit's largest and its sum of weights relative to that
template <typename T> CFB_DEV void stats_units(const Row<T>& w, Span s, float* tops, double* sums) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int u = s.u0 + warp; u < s.u1; u += kWarps) {
    float x[kPerLane];
    load_unit(w, u, lane, x);
    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) m[i & 3] = fmaxf(m[i & 3], x[i]);
    const float top = warp_max(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
    float a[4] = {0.f, 0.f, 0.f, 0.f};
    if (fabsf(top) < INFINITY) {
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) a[i & 3] += ex2((x[i] - top) * w.c);
    } else {                                               // +inf, or nothing but -inf; NaN makes the sum NaN
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) a[i & 3] += x[i] != x[i] ? x[i] : x[i] == INFINITY ? 1.f : 0.f;
    }
    const float sum = warp_sum((a[0] + a[1]) + (a[2] + a[3]));
    if (lane == 0) {
      tops[u - s.u0] = top;
      sums[u - s.u0] = sum;
    }
  }
}
// every unit's sum of values relative to the row's largest. (In 64 bits, which few rows need, an element at a time:
// small code instead of 32 exponentials in a row.)
template <int MODE, typename T>
__device__ __noinline__ void value_units(const Row<T>& w, Span s, float base, double iz, double* sums) {
  constexpr int E = 16 / (int)sizeof(T), NV = kPerLane / E;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int u = s.u0 + warp; u < s.u1; u += kWarps) {
    double sum = 0.;
    if constexpr (kNarrow<MODE>) {
      float x[kPerLane], a[4] = {0.f, 0.f, 0.f, 0.f};
      load_unit(w, u, lane, x);
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) a[e & 3] += value_of<MODE>(w, x[j * E + e], first_of(w, u, j, lane) + e, base, iz);
      sum = warp_sum((a[0] + a[1]) + (a[2] + a[3]));
    } else {
#pragma unroll 1
      for (int k = 0; k < kPerLane; ++k) {
        const int i = first_of(w, u, k / E, lane) + k % E;
        if (i >= 0 && i < w.V) sum += value_of<MODE>(w, to_float(w.p[i]), i, base, iz);
      }
      sum = warp_sum(sum);
    }
    if (lane == 0) sums[u - s.u0] = sum;
  }
}

// Warp 0: the units' sums become running ones (of the stats pass: brought to the CTA's largest first)
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

// Warp 0: the first token of this CTA's part whose running sum passes t (relative to the part's start)
template <int MODE, typename T>
__device__ __noinline__ Found find(const Row<T>& w, Span s, const double* sums, double t, float base, double iz, double band) {
  constexpr int E = 16 / (int)sizeof(T), NV = kPerLane / E, kJ = kNarrow<MODE> ? NV : 1, kE = kNarrow<MODE> ? E : 1;
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
    if (u < 0) return {-1, 1};
  }
  double before = u ? sums[u - 1] : 0.;
  float x[kPerLane];
  if constexpr (kNarrow<MODE>) load_unit(w, s.u0 + u, lane, x);
  const auto value = [&](int j, int e) -> double {
    const int i = first_of(w, s.u0 + u, j, lane) + e;
    if constexpr (kNarrow<MODE>) return value_of<MODE>(w, x[j * E + e], i, base, iz);
    else return i >= 0 && i < w.V ? value_of<MODE>(w, to_float(w.p[i]), i, base, iz) : 0.;
  };
  int token = -1, last = -1;
  double lo = 0., hi = 0.;
#pragma unroll kJ
  for (int j = 0; j < NV; ++j) {
    double a = 0.;
    int top = -1;                                          // this lane's last token with mass
#pragma unroll kE
    for (int e = 0; e < E; ++e) {
      const double v = value(j, e);
      a += v;
      if (v > 0.) top = e;
    }
    const double scan = warp_scan(a, lane);
    const double up = __shfl_up_sync(0xffffffffu, scan, 1);
    const unsigned hit = __ballot_sync(0xffffffffu, token < 0 && before + scan > t && a > 0.);
    if (hit) {
      const int who = __ffs(hit) - 1;
      if (lane == who) {
        double run = lane ? before + up : before;
#pragma unroll kE
        for (int e = 0; e < E; ++e) {
          const double v = value(j, e);
          if (token < 0 && v > 0. && (run + v > t || e == top)) {
            token = e;
            lo = run;
            hi = run + v;
          }
          run += v;
        }
        token += first_of(w, s.u0 + u, j, lane);
      }
      token = __shfl_sync(0xffffffffu, token, who);
      lo = __shfl_sync(0xffffffffu, lo, who);
      hi = __shfl_sync(0xffffffffu, hi, who);
    }
    before += __shfl_sync(0xffffffffu, scan, 31);
    const unsigned some = __ballot_sync(0xffffffffu, top >= 0);
    if (some) last = __shfl_sync(0xffffffffu, top + first_of(w, s.u0 + u, j, lane), 31 - __clz(some));
  }
  if (token < 0) return {last, 1};
  return {token, unsure || !(t - lo >= band && hi - t >= band)};
}

// Warp 0: the first element that equals the row's largest (or the first NaN)
template <typename T>
__device__ __noinline__ int find_top(const Row<T>& w, Span s, const float* tops, const double* sums, float top, bool nan) {
  constexpr int E = 16 / (int)sizeof(T), NV = kPerLane / E;
  const int lane = threadIdx.x & 31, n = s.u1 - s.u0;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int k = i0 + lane;
    const unsigned hit = __ballot_sync(0xffffffffu, k < n && (nan ? sums[k] != sums[k] : tops[k] == top));
    if (!hit) continue;
    const int u = s.u0 + i0 + __ffs(hit) - 1;
    float x[kPerLane];
    load_unit(w, u, lane, x);
    int best = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float l = x[j * E + e];
        const int i = first_of(w, u, j, lane) + e;
        if (i >= 0 && i < w.V && (nan ? l != l : l == top)) best = min(best, i);
      }
    return __reduce_min_sync(0xffffffffu, best);
  }
  return -1;
}

// What a cluster finds of a row. `ph` alternates the exchanged buffers.
template <typename T> struct Team {
  cg::cluster_group cluster;
  Shared& sh;
  float* tops;
  double* sums;
  int rank, ranks, ph;

  // totals of all CTAs -> the row's, and what lies before this one's part. `scaled`: each relative to its own largest
  __device__ void exchange(const Row<T>& w, bool scaled, double* whole) {
    cluster.sync();
    if (threadIdx.x < 32) {
      const int lane = threadIdx.x;
      Pub p{-INFINITY, 0, 0.};
      if (lane < ranks) p = *cluster.map_shared_rank(&sh.pub[ph], lane);
      float top = sh.top;
      if (scaled) {
        top = warp_max(p.top);
        const bool nan = __any_sync(0xffffffffu, p.nan);
        if (lane == 0) {
          sh.top = top;
          sh.kind = nan ? ROW_NAN : top == -INFINITY ? ROW_EMPTY : ROW_MASS;
        }
        p.sum *= p.top == -INFINITY ? 0. : (double)weight(p.top, top, w.c);
      }
      const double scan = warp_scan(p.sum, lane), total = __shfl_sync(0xffffffffu, scan, 31);
      const double end = __shfl_sync(0xffffffffu, scan, rank);
      const double before = __shfl_sync(0xffffffffu, scan, max(rank - 1, 0));      // (not end - sum, which would lose small ones)
      if (lane == 0) {
        *whole = total;
        sh.before = rank ? before : 0.;
        sh.end = end;
      }
    }
    __syncthreads();
  }

  // the pass over the row
  __device__ void stats(const Row<T>& w) {
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
      if (lane == 0) sh.pub[ph] = {top, nan, sum};
    }
    exchange(w, true, &sh.z);
  }

  // a pass that knows the row's largest
  template <int MODE> __device__ void pass(const Row<T>& w, double* whole) {
    const Span s = span_of(w, rank, ranks);
    value_units<MODE>(w, s, sh.top, 1. / sh.z, sums);
    __syncthreads();
    ph ^= 1;
    if (threadIdx.x < 32) {
      const double sum = run_up(sums, s.u1 - s.u0, threadIdx.x);
      if (threadIdx.x == 0) sh.pub[ph] = {sh.top, 0, sum};
    }
    exchange(w, false, whole);
  }

  // Warp 0 of the CTA that found it hands it to all
  __device__ Found share(bool mine, Found f) {
    if (mine && threadIdx.x < ranks) *cluster.map_shared_rank(&sh.found[ph], (int)threadIdx.x) = f;
    cluster.sync();
    return sh.found[ph];
  }

  // the draw of threshold u among the running sums of the last pass, whose whole is `whole`
  template <int MODE> __device__ Found draw(const Row<T>& w, double u, double whole) {
    if (threadIdx.x == 0) sh.found[ph] = {-1, 1};          // kept where no part has the threshold
    cluster.sync();
    bool mine = false;
    Found f{-1, 1};
    if (threadIdx.x < 32) {
      const Pub own = sh.pub[ph];
      const double t = fmin(u * whole, whole * (1. - 2.220446049250313e-16));
      // relative to the base of this CTA's sums
      const double scale = MODE == W32 ? (own.top == -INFINITY ? 0. : (double)weight(own.top, sh.top, w.c)) : 1.;
      mine = own.sum * scale > 0. && sh.before <= t && (t < sh.end || last_with_mass(w, MODE == W32));
      // (of what is left above q, the error is that of the probabilities, whose whole is 1)
      const double band = MODE == W32 ? kBand * whole / scale : MODE == R32 ? kBand : 0.;
      if (mine)
        f = find<MODE>(w, span_of(w, rank, ranks), sums, (t - sh.before) / scale, MODE == W32 ? own.top : sh.top, 1. / sh.z, band);
    }
    return share(mine, f);
  }
  // no later part has any
  __device__ bool last_with_mass(const Row<T>& w, bool scaled) {
    for (int r = rank + 1; r < ranks; ++r) {
      const Pub p = *cluster.map_shared_rank(&sh.pub[ph], r);
      if (p.sum > 0. && (!scaled || weight(p.top, sh.top, w.c) > 0.f)) return false;
    }
    return true;
  }

  // the first of the row's largest
  __device__ int top_token(const Row<T>& w, bool nan) {
    bool mine = false;
    Found f{-1, 0};
    if (threadIdx.x < 32) {
      mine = nan ? sh.pub[ph].nan : sh.pub[ph].top == sh.top;
      for (int r = 0; r < rank && mine; ++r) {
        const Pub p = *cluster.map_shared_rank(&sh.pub[ph], r);
        mine = !(nan ? p.nan != 0 : p.top == sh.top);
      }
      if (mine) f = {find_top(w, span_of(w, rank, ranks), tops, sums, sh.top, nan), 0};
    }
    return share(mine, f).token;
  }
};

struct RowResult { int token, accept; float logp; };

template <typename T> CFB_DEV float log_prob(const Row<T>& w, int token, float top, double z) {
  if (token < 0) return 0.f;
  const float l = to_float(w.p[token]);
  return (float)((l == top ? 0. : ((double)l - (double)top) * w.inv_tau) - log(z));
}

// (an upper end that sums of 64 bits still resolve)
CFB_DEV double number_at(const void* p, int size, long long i) {
  const double u = size == 4 ? (double)static_cast<const float*>(p)[i] : static_cast<const double*>(p)[i];
  return fmin(fmax(u, 0.), 1. - 0x1p-32);
}

// One row, by a whole cluster; every thread gets the result. drafted: the row has a draft with probabilities, `draft`,
// which u accepts; v draws.
template <typename T>
__device__ RowResult resolve(Team<T>& team, const Row<T>& w, bool greedy, bool drafted, int draft, double u, double v) {
  Shared& sh = team.sh;
  team.stats(w);
  if (sh.kind == ROW_EMPTY) return {-1, 0, 0.f};
  if (greedy || sh.kind == ROW_NAN) {
    const int t = team.top_token(w, sh.kind == ROW_NAN);
    return {t, drafted && t == draft, sh.kind == ROW_NAN ? NAN : log_prob(w, t, sh.top, sh.z)};
  }
  Found f{-1, 1};
  if (drafted) {
    const bool in = draft >= 0 && draft < w.V;             // a draft that is no token is refused
    bool exact = false;
    if (in) {
      const float l = to_float(w.p[draft]);
      const double uq = u * (double)draft_prob(w, draft);
      double p = (double)weight(l, sh.top, w.c) / sh.z;
      if (fabs(uq - p) <= 2. * kBand * p) {                // (every CTA computes the same)
        team.template pass<W64>(w, &sh.z);
        exact = true;
        p = weight64(l, sh.top, w.inv_tau) / sh.z;
      }
      if (uq < p) return {draft, 1, log_prob(w, draft, sh.top, sh.z)};
    }
    if (!exact) {
      team.template pass<R32>(w, &sh.r);
      if (sh.r > 2. * kBand) f = team.template draw<R32>(w, v, sh.r);
    }
    if (f.unsure) {
      if (!exact) team.template pass<W64>(w, &sh.z);
      team.template pass<R64>(w, &sh.r);
      if (sh.r > 0.) {
        f = team.template draw<R64>(w, v, sh.r);
      } else {                                             // nothing above q: the target's own
        team.template pass<W64>(w, &sh.z);
        f = team.template draw<W64>(w, v, sh.z);
      }
    }
  } else {
    f = team.template draw<W32>(w, v, sh.z);
    if (f.unsure) {
      team.template pass<W64>(w, &sh.z);
      f = team.template draw<W64>(w, v, sh.z);
    }
  }
  return {f.token, 0, log_prob(w, f.token, sh.top, sh.z)};
}

template <typename T> CFB_DEV Row<T> row_of(const VerifyArgs& A, int row, float temp, bool greedy) {
  Row<T> w;
  w.p = static_cast<const T*>(A.logits) + (long long)row * A.ld;
  w.V = A.V;
  w.shift = (int)((reinterpret_cast<uintptr_t>(w.p) & 15) / sizeof(T));
  const float tau = greedy ? 1.f : fminf(temp, kHighTemp);
  w.inv_tau = 1. / (double)tau;
  w.c = (float)fmin(1.4426950408889634 / (double)tau, 3.4e38);
  w.q = nullptr;
  w.index_of = A.index_of;
  return w;
}

// FLAT: a cluster a row (grid.y: rows of a request, grid.z: requests), every row at once; the request's last
// cluster walks. Otherwise a cluster a request (grid.y), which takes the rows of its walk in turn.
// CHAIN: draft probabilities; a node's only child is the next one.
template <typename T, bool CHAIN, bool FLAT>
__global__ void __launch_bounds__(kThreads) verify_kernel(const VerifyArgs A) {
  extern __shared__ double s_dyn[];
  __shared__ Shared sh;
  __shared__ int s_last;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int most = (int)(((long long)(A.V + 7 + kUnit - 1) / kUnit + ranks - 1) / ranks + 1);
  Team<T> team{cluster, sh, reinterpret_cast<float*>(s_dyn + most), s_dyn, rank, ranks, 0};
  const int b = FLAT ? blockIdx.z : blockIdx.y;
  const int d0 = b ? A.cu_draft[b - 1] : 0;
  const long long drafts = (long long)A.cu_draft[b] - d0, start = A.cu_sampled[b] - (drafts + 1);
  // offsets that do not describe rows of this logits matrix (or drafts) are never dereferenced
  const bool sane = drafts >= 0 && drafts <= A.max_spec && start >= 0 && start + drafts < A.num_rows && d0 >= 0 &&
                    d0 + drafts <= A.num_drafts;
  const int n = (int)drafts, s0 = (int)start;
  const float temp = A.temperature ? A.temperature[b] : 1.f;
  const bool greedy = !(temp >= kLowTemp);
  int32_t* const ot = A.out_tokens + (long long)b * (A.max_spec + 1);
  float* const ol = A.out_logp + (long long)b * (A.max_spec + 1);
  int32_t* const op = CHAIN ? nullptr : A.out_path + (long long)b * A.max_spec;
  const auto take = [&](int j) {                           // row j of the request
    Row<T> w = row_of<T>(A, s0 + j, temp, greedy);
    if constexpr (CHAIN) {
      const bool drafted = j < n;
      if (drafted) w.q = A.probs + (long long)(d0 + j) * A.ld_probs;
      return resolve(team, w, greedy, drafted, drafted ? A.draft_tokens[d0 + j] : -1,
                     drafted ? number_at(A.uniforms, A.uniform_size, d0 + j) : 0., number_at(A.resample, A.uniform_size, b));
    } else {
      return resolve(team, w, greedy, false, -1, 0., number_at(A.uniforms, A.uniform_size, s0 + j));
    }
  };
  const auto child = [&](int cur, int tok) {               // the first child of cur that carries tok, by a warp
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + (int)(threadIdx.x & 31);
      const unsigned hit = __ballot_sync(0xffffffffu, i < n && A.parents[d0 + i] == cur && A.draft_tokens[d0 + i] == tok);
      if (hit) return i0 + __ffs(hit) - 1;
    }
    return -1;
  };
  const auto clear = [&](int from) {                       // what follows the tokens
    for (int p = from + (int)threadIdx.x; p <= A.max_spec; p += kThreads) { ot[p] = -1; ol[p] = 0.f; }
    if constexpr (!CHAIN) for (int p = from - 1 + (int)threadIdx.x; p < A.max_spec; p += kThreads) if (p >= 0) op[p] = -1;
  };
  if constexpr (FLAT) {
    const int j = blockIdx.y;
    if (sane && j <= n) {
      const RowResult r = take(j);
      if (rank == 0 && threadIdx.x == 0) {
        A.row_token[s0 + j] = r.token;
        A.row_logp[s0 + j] = r.logp;
        if constexpr (CHAIN) A.row_accept[s0 + j] = r.accept;
      }
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
  }
  if (!sane) {                                             // inconsistent offsets: emit nothing, flag it
    if (rank == 0) {
      clear(0);
      if (threadIdx.x == 0) {
        A.out_len[b] = 0;
        if (A.err) atomicCAS(A.err, 0, DEV_BAD_INDEX);
      }
    }
    return;
  }
  int cur = -1, pos = 0;
  for (;;) {                                               // (every thread of every CTA takes the same steps)
    RowResult r;
    if constexpr (FLAT) {
      r = {__ldcg(A.row_token + s0 + cur + 1), CHAIN ? __ldcg(A.row_accept + s0 + cur + 1) : 0, __ldcg(A.row_logp + s0 + cur + 1)};
    } else {
      r = take(cur + 1);
    }
    int nxt = -1;
    if (pos < A.max_spec && r.token >= 0) {
      if constexpr (CHAIN) nxt = r.accept && cur + 1 < n ? cur + 1 : -1;
      else nxt = child(cur, r.token);
    }
    if (rank == 0 && threadIdx.x == 0) {
      ot[pos] = r.token;
      ol[pos] = r.logp;
      if constexpr (!CHAIN) if (nxt >= 0) op[pos] = nxt;
    }
    if (nxt < 0) break;
    cur = nxt;
    ++pos;
  }
  if constexpr (!FLAT) cluster.sync();
  if (rank == 0) {
    clear(pos + 1);
    if (threadIdx.x == 0) A.out_len[b] = pos;
  }
}

template <typename T, bool CHAIN, bool FLAT>
cfb_status launch(const VerifyArgs& a, int cluster, cudaStream_t st) {
  const long long units = (a.V + 7 + kUnit - 1) / kUnit, most = (units + cluster - 1) / cluster + 1;
  const int smem = (int)(most * 12);
  if (allow_smem<verify_kernel<T, CHAIN, FLAT>>((kMaxVocab / kUnit + 2) * 12) != cudaSuccess) return cfb_launch_status("verify_kernel");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = FLAT ? dim3(cluster, a.max_spec + 1, a.batch) : dim3(cluster, a.batch, 1);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, verify_kernel<T, CHAIN, FLAT>, a);
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
  a.row_token = reinterpret_cast<int32_t*>(static_cast<char*>(ws) + ((size_t)batch * 4 + 255) / 256 * 256);
  a.row_accept = a.row_token + num_rows;
  a.row_logp = reinterpret_cast<float*>(a.row_accept + num_rows);
  a.err = err;
  return CFB_OK;
}

}  // namespace

extern "C" size_t cfb_verify_workspace(int num_rows, int batch) {
  if (num_rows <= 0 || batch <= 0) return 0;
  return ((size_t)batch * 4 + 255) / 256 * 256 + (size_t)num_rows * 12;
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
