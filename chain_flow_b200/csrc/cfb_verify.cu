// cfb_verify.cu -- drafted tokens verified against the target's probabilities, from given random
// numbers (sm_100a): a tree or chain without draft probabilities (cfb_tree_verify_sampled) and a chain
// with them (cfb_chain_verify_rejection).
//
// A logits row l at temperature tau has the weights w_i = 2^((l_i - max l) c), c = log2(e) / tau, and a
// number u in [0, 1) draws the first token i with w_0 + .. + w_i > u sum w. A refused draft draws from
// r_i = max(w_i / sum w - q_i, 0) instead. Which token that is, is a whole number, so it has to be the
// one that exact arithmetic gives, although the pass over the row is fp32: the pass carries a bound of
// its error, and where a sum comes nearer to its threshold than that, the row is taken again in
// 64 bits. That happens the more, the more of a row's mass lies in tokens as small as the bound: to one in eight rows of
// 248320 normal logits of deviation 2.5 (one in three draws from what is left above q there), seldom where a few tokens
// hold most, always where a row is flat over a vocabulary.
//
// One pass over the row: a warp takes 1024 elements in registers, their largest, their weights relative
// to it and the weights' sum, which stay in shared memory (no running rescale of elements: such units' sums are brought
// to one base). A row is shared by a cluster of CTAs, a CTA's part by its warps, each with neighbouring units; CTAs
// exchange their totals through distributed shared memory. The draw then descends: CTA, warp, unit, a lane's neighbours,
// element; only its unit is read again (from L2).
//
// Error of the pass, with u = 2^-24 and x = (l - max l) c, in relative terms: an element's exponent is off by
// (2 + d) u |x| (difference, product, and d u of c itself), on its way to the row's largest that counts once; the exponential and
// the three changes of base (unit, warp, CTA, row) by 4 u each, their products by u; a unit's sum by 11 u (chains of 4,
// pairs, the warp), a warp's sum of q units by (5 + q / 32) u; the sums over warps and CTAs are 64 bits. Under the weights the mean of
// |x| is their entropy less log2 of their sum Z relative to the largest: at most log2(V / Z). What decides is
// C - t = C - v Z: of an error that every weight has in both, at most half remains, since 2 v (1 - v) <= 1 / 2. Where C comes from other
// sums than Z does, their errors count in full: the sum over the CTA's warps (6 u of its part), over the warp's units (their
// changes of base and two sums, (35 + q / 16) u of the warp's mass), inside the unit (18 u of its mass). So C - t is off by less than
//   u Z (ln 2 (2 + d) log2(V / Z) + (16 + 3 + 11 + 5 + q / 32) / 2 + 2) + u (6 part + (35 + q / 16) warp + 18 unit).
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <cmath>

#include "cfb_types.cuh"

using namespace cfb;
namespace cg = cooperative_groups;

namespace {

// Small CTAs, several an SM, in large clusters: their serial steps cover one another (a batch of 64 trees took 80 us with 2
// CTAs of 512 threads an SM, 71 with 4 of 256). Chains, whose steps hold more, take 80 registers a thread and 3 CTAs an SM
// (48 chains 100 us; with 4 CTAs 105), trees 64 and 4 (64 trees 69; with 3 CTAs 78).
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kPerLane = 32;                 // elements of a unit in a lane's registers
constexpr int kUnit = 32 * kPerLane;
constexpr int kMaxCluster = 16;
constexpr int kMaxVocab = 1 << 22;
constexpr int kMaxNodes = 1024;              // draft nodes per request (max_spec_len)
constexpr int kMaxBatch = 65535;
// the workspace: a counter for every request that a call may have, so that no call's rows lie where another's counters do
constexpr size_t kCounters = (kMaxBatch + 1) * sizeof(unsigned);
constexpr double kRound = 1.0 / 16777216;    // 2^-24
constexpr float kLowTemp = 1.17549435e-38f;  // 2^-126: below it (or NaN) a request is greedy
constexpr float kHighTemp = 1.26765060e30f;  // 2^100

// a row's token, whether it is the draft that stays, and what its log probability is made of: ln 2 scaled - log(mass)
struct alignas(8) RowResult { int token, accept; double scaled, mass; };

struct VerifyArgs {
  const void* logits; long long ld; int V, num_rows;
  const int32_t* cu_draft; const int32_t* cu_sampled;      // [batch]
  const int32_t* draft_tokens; const int32_t* parents;     // parents: trees only
  const float* probs; long long ld_probs; int probs_width; // draft probabilities [drafts, probs_width]
  const int32_t* index_of;                                 // [V] column of a token, or -1; NULL: the token itself
  const void* uniforms; const void* resample; int uniform_size;   // 4 or 8 bytes
  const float* temperature;
  int batch, max_spec, num_drafts;
  int32_t* out_tokens; int32_t* out_path; int32_t* out_len; float* out_logp;
  RowResult* rows;                                         // [batch, max_spec + 1], where all rows are taken at once
  unsigned* counter;                                       // [batch]
  int* err;
};

enum Kind : int { ROW_MASS = 0, ROW_EMPTY = 1, ROW_NAN = 2 };
// RowResult::accept, left for the walk (scaled: the row's largest, mass: the sum of its weights): fp32 did not decide; a draft
// that is refused, so that something else is to be drawn
constexpr int kUndecided = 2, kRefused = 3;

struct Pub { float top; int nan; double sum; };      // a CTA's part of a row
struct Found { int token, unsure; float logit; int pad; };

struct Shared {
  Pub pub[2];
  Found found[2];
  double z, whole;           // sum of the row's weights; of what the last pass summed
  double before, end;        // the running sums of the last pass before this CTA's part and behind it
  float warp_top[kWarps], warp_sum[kWarps];                // of a warp's units (the sum relative to its largest)
  double warp_sum64[kWarps];
  float top;                 // of the row
  int kind;
  int owner;                 // the CTA whose part has the threshold, or (greedy rows) the first of the largest
  int last;
};

CFB_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
CFB_DEV float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
CFB_DEV float reciprocal(float x) {                        // (a division takes 280 cycles)
  float y;
  asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
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

// A logits row: element i lies at p[i]. Vectors of 16 bytes start at element -shift, so that they are aligned. Units of kUnit
// elements from there on; this CTA has [u0, u1) of them, and each of its warps `each` neighbours.
template <typename T> struct Row {
  int u0, u1, each;
  const T* p;
  int V, shift;
  float c;                    // log2(e) / tau
  double c64;
  const float* probs;         // draft probabilities of the row, or null
  const int32_t* index_of;
  int width;                  // columns that index_of may name
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
template <typename T> __device__ __noinline__ uint4 load_edge(const T* p, int V, int i) {
  union { uint4 v; T e[kE<T>]; } u;
#pragma unroll
  for (int e = 0; e < kE<T>; ++e) u.e[e] = i + e >= 0 && i + e < V ? p[i + e] : lowest<T>();
  return u.v;
}
// N vectors, `step` elements apart from element i on, of a unit of `span` elements that starts at `first`
template <int N, typename T> CFB_DEV void load_vectors(const Row<T>& w, int first, int span, int i, int step, uint4 (&u)[N]) {
  if (first >= 0 && first + span <= w.V) {
#pragma unroll
    for (int j = 0; j < N; ++j) u[j] = __ldg(reinterpret_cast<const uint4*>(w.p + i + j * step));
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) u[j] = load_edge(w.p, w.V, i + j * step);
  }
}
template <typename T> CFB_DEV void load_unit(const Row<T>& w, int unit, int lane, uint4 (&u)[kVectors<T>]) {
  load_vectors(w, unit * kUnit - w.shift, kUnit, first_of(w, unit, 0, lane), 32 * kE<T>, u);
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

// the weight relative to a finite base
CFB_DEV float weight(float l, float base, float c) { return ex2((l - base) * c); }
// a sum's scale where a larger base takes over (of a largest +inf only what has it counts)
CFB_DEV float rescale(float top, float base, float c) { return top == base ? 1.f : top == -INFINITY || base == INFINITY ? 0.f : weight(top, base, c); }

// The weight 2^((l - base) c) in 64 bits, relative to a finite base, by a whole warp: with 32 (l - base) c = k + r, |r| <= 1/2,
// the series of 2^(r / 32) cut after r^5 (the first term left out is 2 10^-15), times 2^(k mod 32 / 32) from the lane that
// holds it. Nothing is below 2^-1000 (CUT: is 0). Eleven 64-bit operations, N elements side by side; the library's
// function branches, which kept several from running side by side: a pass took 4 times as long.
CFB_DEV float lowest_logit(float base, float c) { return base - 1000.f * reciprocal(c); }
CFB_DEV double exp2_table(int lane) { return exp2((double)lane * 0.03125); }
template <bool CUT, int N> CFB_DEV void fast_weights64(const float* l, float base, float c, double c32, double table, double* out) {
  const double magic = 6755399441055744.;                  // 1.5 2^52: adding it rounds to a whole number
  const float low = lowest_logit(base, c);
  double r[N], p[N];
  int k[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const double d = (double)fmaxf(l[i], low) - (double)base, shifted = fma(d, c32, magic);
    k[i] = __double2loint(shifted);
    r[i] = fma(d, c32, magic - shifted);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {                            // (ln2 / 32)^k / k!
    p[i] = fma(0x1.5d87fe78a6731p-35, r[i], 0x1.3b2ab6fba4e77p-27);
    p[i] = fma(p[i], r[i], 0x1.c6b08d704a0c0p-20);
    p[i] = fma(p[i], r[i], 0x1.ebfbdff82c58fp-13);
    p[i] = fma(p[i], r[i], 0x1.62e42fefa39efp-6) * r[i];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const double t = __shfl_sync(0xffffffffu, table, k[i]);
    p[i] = fma(p[i], t, t);
    p[i] = __hiloint2double(__double2hiint(p[i]) + ((k[i] << 15) & 0xfff00000), __double2loint(p[i]));
    out[i] = CUT && l[i] <= low ? 0. : p[i];
  }
}
// by one thread, of any base, to the smallest denormal
CFB_DEV double weight64(float l, float base, double c) {
  return l == base ? 1. : isinf(base) ? 0. : exp2(((double)l - (double)base) * c);
}
// (by the sign: the library's maximum looks for NaN, which there is none of)
CFB_DEV double positive(double r) { return __double2hiint(r) < 0 ? 0. : r; }
// the draft probability of token i (0 outside the row and for what is not a positive number)
template <typename T> CFB_DEV float draft_prob(const Row<T>& w, int i) {
  if (i < 0 || i >= w.V) return 0.f;
  const int at = w.index_of ? __ldg(w.index_of + i) : i;
  return (unsigned)at < (unsigned)w.width ? fmaxf(__ldg(w.probs + at), 0.f) : 0.f;
}

enum Mode : int { W32 = 0, W64 = 1, R32 = 2, R64 = 3 };    // weights, or what is left of them above q
template <int MODE> constexpr bool kNarrow = MODE == W32 || MODE == R32;
// elements of a summed unit, and a lane's of them: in 64 bits, where an element costs much more, smaller ones to scan
template <int MODE> constexpr int kSpan = kNarrow<MODE> ? kUnit : 256;
// Sums up to this are no mass: masked tokens count as 2^-1000 each in the fast sums of weights (without the cut a batch of
// trees takes 1 us less), and the search, which cuts them, would find nothing among them.
template <int MODE, bool SLOW> constexpr double kNothing = MODE == W64 && !SLOW ? 0x1p-960 : 0.;

// an element's value, by a whole warp. iz: 1 / the row's sum of weights (R32, R64). SLOW (64 bits): any base, denormals kept
template <int MODE, bool SLOW, typename T>
CFB_DEV auto value_of(const Row<T>& w, float l, int i, float base, double iz, double table) {
  if constexpr (MODE == W32) {
    return weight(l, base, w.c);
  } else if constexpr (MODE == R32) {
    return fmaxf(weight(l, base, w.c) * (float)iz - draft_prob(w, i), 0.f);
  } else {
    double v;
    if constexpr (SLOW) v = weight64(l, base, w.c64);
    else fast_weights64<true, 1>(&l, base, w.c, 32. * w.c64, table, &v);
    if constexpr (MODE == W64) return v;
    else return positive(v * iz - (double)draft_prob(w, i));
  }
}

// every unit's largest and its sum of weights relative to that. (Other warps cover a unit's loads: the next unit's under way in
// registers cost a batch of chains 145 us against 129.)
template <typename T> CFB_DEV void stats_units(const Row<T>& w, Shared* sh, float* tops, float* sums) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = w.u0 + warp * w.each, end = min(first + w.each, w.u1);
  float most = -INFINITY;
  for (int u = first; u < end; ++u) {
    uint4 v[kVectors<T>];
    load_unit(w, u, lane, v);
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kVectors<T>; ++j) m = fmaxf(m, vector_max<T>(v[j]));
    const float top = warp_max(m);
    float sum = 0.f;
    if (fabsf(top) < INFINITY) {
      const Pair base = pair(-top, -top), c = pair(w.c, w.c);
      Pair a[4] = {pair(0.f, 0.f), pair(0.f, 0.f), pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
      for (int j = 0; j < kVectors<T>; ++j)
#pragma unroll
        for (int k = 0; k < kE<T> / 2; ++k) {
          const float2 l = pair_of<T>(v[j], k);
          const float2 x = both(mul2(add2(pair(l.x, l.y), base), c));
          const int i = (j * (kE<T> / 2) + k) & 3;
          a[i] = add2(a[i], pair(ex2(x.x), ex2(x.y)));
        }
      const float2 t = both(add2(add2(a[0], a[1]), add2(a[2], a[3])));
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
    most = fmaxf(most, top);
    if (lane == 0) {
      tops[u - w.u0] = top;
      sums[u - w.u0] = sum;
    }
  }
  __syncwarp();
  float total = 0.f;
  for (int u = first + lane; u < end; u += 32) total += sums[u - w.u0] * rescale(tops[u - w.u0], most, w.c);
  total = warp_sum(total);
  if (lane == 0) {
    sh->warp_top[warp] = most;
    sh->warp_sum[warp] = total;
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

// the draft probabilities of n tokens from i on
template <typename T> CFB_DEV void draft_probs(const Row<T>& w, int i, int n, float (&q)[8]) {
  if (w.index_of) {
    int at[8];
    table_entries(w.index_of, i, n, w.V, at, -1);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) q[e] = (unsigned)at[e] < (unsigned)w.width ? __ldg(w.probs + at[e]) : 0.f;
  } else {
    table_entries(w.probs, i, n, w.V, q, 0.f);
  }
}

// every unit's sum of what is left above q
template <typename T> CFB_DEV void rest_units(const Row<T>& w, Shared* sh, float base, float iz, float* sums) {
  constexpr int N = 16 / kE<T>;                            // vectors whose loads are in flight together
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int begin = w.u0 + warp * w.each, end = min(begin + w.each, w.u1);
  float total = 0.f;
  for (int u = begin; u < end; ++u) {
    float a[2] = {0.f, 0.f};
#pragma unroll 1
    for (int j0 = 0; j0 < kVectors<T>; j0 += N) {
      const int i = first_of(w, u, j0, lane);
      uint4 v[N];
      float q[N][8];
      load_vectors(w, u * kUnit - w.shift, kUnit, i, 32 * kE<T>, v);
#pragma unroll
      for (int j = 0; j < N; ++j) draft_probs(w, i + j * 32 * kE<T>, kE<T>, q[j]);
#pragma unroll
      for (int j = 0; j < N; ++j)
#pragma unroll
        for (int k = 0; k < kE<T> / 2; ++k) {
          const float2 l = pair_of<T>(v[j], k);
          a[0] += fmaxf(weight(l.x, base, w.c) * iz - fmaxf(q[j][2 * k], 0.f), 0.f);
          a[1] += fmaxf(weight(l.y, base, w.c) * iz - fmaxf(q[j][2 * k + 1], 0.f), 0.f);
        }
    }
    const float sum = warp_sum(a[0] + a[1]);
    total += sum;
    if (lane == 0) sums[u - w.u0] = sum;
  }
  if (lane == 0) sh->warp_sum[warp] = total;
}

// every unit's sum in 64 bits, by quarters: a lane has 8 neighbours of 256. (A unit's loads together and its four sums
// reduced side by side: chains of a batch 104 -> 100 us.)
template <int MODE, bool SLOW, typename T>
CFB_DEV void exact_units(const Row<T>& w, Shared* sh, float base, double iz, double* sums) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const double table = exp2_table(lane);
  constexpr int kPer = kUnit / kSpan<MODE>, N = 8 / kE<T>;
  static_assert(kPer == 4);
  const int begin = (w.u0 + warp * w.each) * kPer, end = min(begin + w.each * kPer, w.u1 * kPer);
  double total = 0.;
  for (int u = begin; u < end; u += kPer) {
    const int first = u * kSpan<MODE> - w.shift, i = first + lane * 8;
    uint4 v[kPer * N];
    if (first >= 0 && first + kUnit <= w.V) {
#pragma unroll
      for (int k = 0; k < kPer * N; ++k) v[k] = __ldg(reinterpret_cast<const uint4*>(w.p + i + k / N * kSpan<MODE> + k % N * kE<T>));
    } else {
#pragma unroll
      for (int k = 0; k < kPer * N; ++k) v[k] = load_edge(w.p, w.V, i + k / N * kSpan<MODE> + k % N * kE<T>);
    }
    float qnext[8];
    if constexpr (MODE == R64) draft_probs(w, i, 8, qnext);
    double part[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      float q[8], l[8];
      if constexpr (MODE == R64) {
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = qnext[e];
        if (k + 1 < kPer) draft_probs(w, i + (k + 1) * kSpan<MODE>, 8, qnext);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 x = pair_of<T>(v[k * N + e / (kE<T> / 2)], e % (kE<T> / 2));
        l[2 * e] = x.x;
        l[2 * e + 1] = x.y;
      }
      double a = 0.;
      if constexpr (SLOW) {
#pragma unroll 1
        for (int e = 0; e < 8; ++e) {
          const double x = weight64(l[e], base, w.c64);
          a += MODE == R64 ? positive(x * iz - (double)fmaxf(q[e], 0.f)) : x;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          double x[4];
          fast_weights64<MODE == R64, 4>(l + e, base, w.c, 32. * w.c64, table, x);
#pragma unroll
          for (int n = 0; n < 4; ++n) a += MODE == R64 ? positive(x[n] * iz - (double)fmaxf(q[e + n], 0.f)) : x[n];
        }
      }
      part[k] = a;
    }
    // the four sums over the warp: of sum i + 2 j the lanes of the low bits i, j
    const bool odd = lane & 1, high = lane & 2;
    const double x = (odd ? part[1] : part[0]) + __shfl_xor_sync(0xffffffffu, odd ? part[0] : part[1], 1);
    const double y = (odd ? part[3] : part[2]) + __shfl_xor_sync(0xffffffffu, odd ? part[2] : part[3], 1);
    double sum = (high ? y : x) + __shfl_xor_sync(0xffffffffu, high ? x : y, 2);
#pragma unroll
    for (int off = 4; off < 32; off *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    total += sum;
    if (lane < kPer) sums[u - w.u0 * kPer + lane] = sum;
  }
  total += __shfl_xor_sync(0xffffffffu, total, 1);
  total += __shfl_xor_sync(0xffffffffu, total, 2);
  if (lane == 0) sh->warp_sum64[warp] = total;
}

// Of n values, by a warp: the first above `floor` whose running sum, from *head on, passes t; where none does, for rounding, the
// last above it (unsure), or -1. *head becomes the running sum in front of it
template <typename F, typename G> CFB_DEV int pick(int n, G value, F* head, F t, F floor, bool* unsure) {
  const int lane = threadIdx.x & 31;
  F before = *head, before_last = before;
  int last = -1;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const F v = i0 + lane < n ? value(i0 + lane) : (F)0, scan = before + warp_scan(v, lane);
    const F up = __shfl_up_sync(0xffffffffu, scan, 1), front = lane ? up : before;
    const unsigned hit = __ballot_sync(0xffffffffu, v > floor && scan > t), some = __ballot_sync(0xffffffffu, v > floor);
    if (hit) {
      const int e = __ffs(hit) - 1;
      *head = __shfl_sync(0xffffffffu, front, e);
      return i0 + e;
    }
    if (some) {
      const int e = 31 - __clz(some);
      last = i0 + e;
      before_last = __shfl_sync(0xffffffffu, front, e);
    }
    before = __shfl_sync(0xffffffffu, scan, 31);
  }
  *unsure = true;
  *head = before_last;
  return last;
}

// Warp 0: the first token of this CTA's part whose running sum passes the threshold t. In 64 bits that is the sum over the whole row,
// `head` in front of the part, carried down as it is: where it comes to exactly t at a border, what has next to no mass
// behind the border leaves it at t, as in one sum over the row, while against a rest of 0 it would pass. In fp32 (which is not
// decided near a border) t is relative to the part's start, then to each step's. W32: warps' sums are relative to
// part_top. band: for all but what the warp and the unit add.
template <int MODE, bool SLOW, typename T, typename F>
CFB_DEV Found find(const Row<T>& w, const Shared* sh, const float* tops, const F* sums, F head, F t, double iz, float part_top, float band) {
  constexpr int kPer = kUnit / kSpan<MODE>, kLane = kSpan<MODE> / 32;   // summed units a unit; a lane's elements
  constexpr int N = kLane / kE<T>;
  const int lane = threadIdx.x & 31;
  const double table = kNarrow<MODE> ? 0. : exp2_table(lane);
  const float base = sh->top;
  bool unsure = false;
  const auto warp_mass = [&](int i) -> F {
    if constexpr (MODE == W32) return sh->warp_sum[i] * rescale(part_top, base, w.c);
    else if constexpr (MODE == R32) return sh->warp_sum[i];
    else return sh->warp_sum64[i];
  };
  const auto step = [&](int n, auto value) {
    const int i = pick<F>(n, value, &head, t, (F)kNothing<MODE, SLOW>, &unsure);
    if constexpr (kNarrow<MODE>) {
      t -= head;
      head = 0;
    }
    return i;
  };
  const int part = step(kWarps, warp_mass);
  if (part < 0) return {-1, 1, 0.f, 0};
  const int begin = part * w.each, n = (min(begin + w.each, w.u1 - w.u0) - begin) * kPer;
  const auto unit_sum = [&](int i) -> F {
    if constexpr (MODE == W32) return sums[begin + i] * rescale(tops[begin + i], base, w.c);
    else return sums[begin * kPer + i];
  };
  const int u = step(n, unit_sum);
  if (u < 0) return {-1, 1, 0.f, 0};
  const F mass = unit_sum(u);
  const int first = (w.u0 + begin) * kUnit + u * kSpan<MODE> - w.shift, i0 = first + lane * kLane;
  uint4 x[N];
  load_vectors(w, first, kSpan<MODE>, i0, kE<T>, x);
  F a = 0;
#pragma unroll SLOW ? 1 : N
  for (int j = 0; j < N; ++j) {
    F v[4] = {0, 0, 0, 0};
#pragma unroll SLOW ? 1 : kE<T> / 2
    for (int k = 0; k < kE<T> / 2; ++k) {
      const float2 l = pair_of<T>(x[j], k);
      v[k] = value_of<MODE, SLOW>(w, l.x, i0 + j * kE<T> + 2 * k, base, iz, table);
      v[k] += value_of<MODE, SLOW>(w, l.y, i0 + j * kE<T> + 2 * k + 1, base, iz, table);
    }
    a += (v[0] + v[1]) + (v[2] + v[3]);
  }
  const int who = step(32, [&](int) { return a; });
  if (who < 0) return {-1, 1, 0.f, 0};
  const int i = first + who * kLane + lane;
  const float l = lane < kLane && i >= 0 && i < w.V ? to_float(w.p[i]) : -INFINITY;
  const F y = value_of<MODE, SLOW>(w, l, lane < kLane ? i : -1, base, iz, table);
  const int e = step(32, [&](int) { return y; });
  if (e < 0) return {-1, 1, 0.f, 0};
  if constexpr (kNarrow<MODE>) {
    float off = band + 18.f * (float)kRound * mass;
    if constexpr (MODE == W32) off += (float)kRound * (36.f + 0.07f * (float)w.each) * warp_mass(part);
    unsure |= !(t >= off && __shfl_sync(0xffffffffu, y, e) - t >= off);
  }
  return {first + who * kLane + e, unsure, __shfl_sync(0xffffffffu, l, e), 0};
}

// Warp 0: the first element that equals the row's largest (or the first NaN)
template <typename T>
__device__ __noinline__ int find_top(Row<T> w, const float* tops, const float* sums, float top, bool nan) {
  const int lane = threadIdx.x & 31, n = w.u1 - w.u0;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int k = i0 + lane;
    const unsigned hit = __ballot_sync(0xffffffffu, k < n && (nan ? sums[k] != sums[k] : tops[k] == top));
    if (!hit) continue;
    const int u = w.u0 + i0 + __ffs(hit) - 1;
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

// (the numbers as they lie in memory: what uses them comes after the pass, and so does the wait for them)
CFB_DEV double number(uint2 raw, int size) {
  const double u = size == 4 ? (double)__uint_as_float(raw.x) : __hiloint2double((int)raw.y, (int)raw.x);
  return fmin(fmax(u, 0.), 1. - 0x1p-32);                  // (an upper end that sums of 64 bits still resolve)
}

// What a cluster finds of a row. `ph` alternates the exchanged buffers.
template <typename T> struct Team {
  Shared* sh;
  float* tops;
  void* room;                // the units' sums
  int rank, ranks, ph;

  // The mean error of the exponents, and how far an fp32 sum over the row may be from its side of a threshold, as a share
  // of the row's mass z, in u
  CFB_DEV float mean_off(const Row<T>& w, float z) const {
    const float d = fabsf((float)(w.c64 - (double)w.c)) * reciprocal(w.c) * 16777216.f;
    return 0.6932f * (2.001f + d) * (lg2((float)w.V) - lg2(z));
  }
  CFB_DEV float band(const Row<T>& w, float z) const { return mean_off(w, z) + 20.f + (float)w.each * 0.02f; }

  // The CTAs' totals, handed over by the cluster's barrier -> the row's; who has the threshold u of it. SCALED: each
  // total is relative to its CTA's largest; greedy: the owner is the first that has the row's largest. floor: as in pick.
  template <bool SCALED> CFB_DEV void exchange(const Row<T>& w, double u, bool greedy, double floor) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (threadIdx.x < 32) {
      const int lane = threadIdx.x;
      Pub p{-INFINITY, 0, 0.};
      if (lane < ranks) p = *cluster.map_shared_rank(&sh->pub[ph], lane);
      double m = p.sum;
      bool nan = false;
      float top = 0.f;
      if constexpr (SCALED) {
        top = warp_max(p.top);
        nan = __any_sync(0xffffffffu, p.nan);
        m *= (double)rescale(p.top, top, w.c);
      }
      double scan = m;
#pragma unroll
      for (int off = 1; off < kMaxCluster; off <<= 1) {
        const double o = __shfl_up_sync(0xffffffffu, scan, off);
        if (lane >= off) scan += o;
      }
      const double whole = __shfl_sync(0xffffffffu, scan, kMaxCluster - 1);
      // (the sum before, not the one behind less this part's, which would lose small ones)
      const double up = __shfl_up_sync(0xffffffffu, scan, 1), before = lane ? up : 0.;
      const double t = threshold(u, whole);
      // (not by `before`: the sums of two lanes may round apart, and t fall between one's end and the next one's start)
      unsigned hit = __ballot_sync(0xffffffffu, m > floor && t < scan);
      if (!hit) hit = 1u << (31 - __clz(__ballot_sync(0xffffffffu, m > floor) | 1u));
      if (SCALED && (greedy || nan)) hit = __ballot_sync(0xffffffffu, nan ? p.nan != 0 : p.top == top);
      if (lane == rank) {
        sh->before = before;
        sh->end = scan;
      }
      if (lane == 0) {
        sh->owner = __ffs(hit) - 1;
        sh->whole = whole;
        if (SCALED) {
          sh->z = whole;
          sh->top = top;
          sh->kind = nan ? ROW_NAN : top == -INFINITY ? ROW_EMPTY : ROW_MASS;
        }
      }
    }
    __syncthreads();
  }
  static CFB_DEV double threshold(double u, double whole) { return fmin(u * whole, whole * (1. - 0x1p-52)); }

  // Warp 0: the warps' sums handed over
  static CFB_DEV double warps_sum(double v) {
#pragma unroll
    for (int off = kWarps / 2; off; off >>= 1) v += __shfl_down_sync(0xffffffffu, v, off);
    return v;
  }
  template <typename F> CFB_DEV void hand_over() {
    const int lane = threadIdx.x;
    double v = 0.;
    if (lane < kWarps) {
      if constexpr (sizeof(F) == 8) v = sh->warp_sum64[lane];
      else v = (double)sh->warp_sum[lane];
    }
    v = warps_sum(v);
    if (lane == 0) sh->pub[ph].sum = v;
  }

  // the pass over the row
  CFB_DEV void stats(const Row<T>& w, uint2 raw, int size, bool greedy) {
    stats_units(w, sh, tops, static_cast<float*>(room));
    __syncthreads();
    ph ^= 1;
    if (threadIdx.x < 32) {
      const int lane = threadIdx.x;
      const float mine = lane < kWarps ? sh->warp_top[lane] : -INFINITY, sum = lane < kWarps ? sh->warp_sum[lane] : 0.f;
      const float top = warp_max(mine), scaled = sum * rescale(mine, top, w.c);
      const bool nan = __any_sync(0xffffffffu, sum != sum);
      const double total = warps_sum((double)scaled);
      if (lane < kWarps) sh->warp_sum[lane] = scaled;      // (relative to the CTA's largest from here on)
      if (lane == 0) sh->pub[ph] = {top, nan, nan ? 0. : total};
    }
    exchange<true>(w, number(raw, size), greedy, 0.);
  }

  // a pass that knows the row's largest, and its sum where it needs it
  CFB_DEV void rest_pass(const Row<T>& w, double u) {
    rest_units(w, sh, sh->top, reciprocal((float)sh->z), static_cast<float*>(room));
    __syncthreads();
    ph ^= 1;
    if (threadIdx.x < 32) hand_over<float>();
    exchange<false>(w, u, false, 0.);
  }
  template <int MODE, bool SLOW> CFB_DEV void exact_pass(const Row<T>& w, double u) {
    exact_units<MODE, SLOW>(w, sh, sh->top, MODE == R64 ? 1. / sh->z : 0., static_cast<double*>(room));
    __syncthreads();
    ph ^= 1;
    if (threadIdx.x < 32) hand_over<double>();
    exchange<false>(w, u, false, kNothing<MODE, SLOW>);
  }

  // Warp 0 of the owner: the token of the last pass's threshold
  CFB_DEV Found found(const Row<T>& w, double u) const {
    if (isinf(sh->top)) return {-1, 1, 0.f, 0};            // several of +inf: in 64 bits
    const float whole = (float)sh->whole;
    return find<W32, false>(w, sh, tops, static_cast<const float*>(room), 0.f, (float)(threshold(u, sh->whole) - sh->before), 0.,
                            sh->pub[ph].top, (float)kRound * (band(w, whole) * whole + 6.f * (float)(sh->end - sh->before)));
  }
  // (from what is left above q, R: every p is off by its exponent's error and 6 u, and all of them by 1 / Z's, of which
  // C - v R keeps the share that q has where p is larger, at most 1 - R; a unit's sum is off by 23 u (chains of 16, pairs, the
  // warp), a warp's by q u, of which half remains, the sum over warps by 4 u, the one over units by (5 + q / 6) u, and by q u, since it is another)
  CFB_DEV Found found_rest(const Row<T>& w, double u) const {
    const float whole = (float)sh->whole, z = (float)sh->z, mean = mean_off(w, z), other = fmaxf(1.f - whole, 0.f), q = (float)w.each;
    const float off = (float)kRound * (mean * (1.f + other) + 6.f + (39.f + 0.04f * q) * other + (22.f + 2.f * q) * whole);
    if (!(whole > 2.f * off)) return {-1, 1, 0.f, 0};
    return find<R32, false>(w, sh, tops, static_cast<const float*>(room), 0.f, (float)(threshold(u, sh->whole) - sh->before),
                            (double)reciprocal(z), 0.f, off);
  }
  template <int MODE, bool SLOW> CFB_DEV Found found64(const Row<T>& w, double u) const {
    return find<MODE, SLOW>(w, sh, tops, static_cast<const double*>(room), sh->before, threshold(u, sh->whole),
                            MODE == R64 ? 1. / sh->z : 0., 0.f, 0.f);
  }

  // Warp 0 of the owner hands what it found to all
  CFB_DEV Found share(const Found& f) {
    cg::cluster_group cluster = cg::this_cluster();
    if (rank == sh->owner && threadIdx.x < ranks) *cluster.map_shared_rank(&sh->found[ph], (int)threadIdx.x) = f;
    cluster.sync();
    return sh->found[ph];
  }
};

// What a row is asked: drafted: it has a draft with probabilities, `draft`, which u accepts; v draws
struct Asked { bool greedy, drafted; int draft, size; uint2 raw_u, raw_v; };
// The row decided in 64 bits, its largest in sh.top. Every thread of the cluster gets the result (in bit 8 of accept,
// whether the exchanged buffers have been alternated).
template <bool CHAIN, bool SLOW, typename T>
CFB_DEV RowResult exact_steps(Team<T> team, const Row<T>& w, const Asked& a, double u, double v) {
  Shared& sh = *team.sh;
  const int ph = team.ph;
  const auto result = [&](int token, int accept, float l) {
    const double scaled = l == sh.top ? 0. : ((double)l - (double)sh.top) * w.c64;
    return RowResult{token, accept | (team.ph ^ ph) << 8, scaled, sh.z};
  };
  Found f{-1, 1, 0.f, 0};
  bool rest = false;
  for (;;) {
    team.template exact_pass<W64, SLOW>(w, v);
    if (threadIdx.x == 0) sh.z = sh.whole;
    __syncthreads();
    if constexpr (CHAIN) {
      if (a.drafted && !rest) {
        if (a.draft >= 0 && a.draft < w.V) {
          const float l = to_float(w.p[a.draft]);
          if (u * (double)draft_prob(w, a.draft) < weight64(l, sh.top, w.c64) / sh.z) return result(a.draft, 1, l);
        }
        team.template exact_pass<R64, SLOW>(w, v);
        if (sh.whole > 0.) {
          if (team.rank == sh.owner && threadIdx.x < 32) f = team.template found64<R64, SLOW>(w, v);
          break;
        }
        rest = true;                                       // nothing above q: the target's own
        continue;
      }
    }
    if (team.rank == sh.owner && threadIdx.x < 32) f = team.template found64<W64, SLOW>(w, v);
    break;
  }
  f = team.share(f);
  return result(f.token, 0, f.logit);
}
template <bool CHAIN, typename T> __device__ __noinline__ RowResult exact_row(Team<T> team, Row<T> w, Asked a) {
  // (weights below 2^-1000, which the fast ones cut, count where the threshold is that small, and only there: all of a row's
  // together are below 2^-78 of a threshold of 2^-900)
  const double u = number(a.raw_u, a.size), v = number(a.raw_v, a.size);
  const float top = team.sh->top, depth = (top - lowest_logit(top, w.c)) * w.c;       // (fp32 may not hold such a logit)
  return isinf(top) || !(depth > 990.f && depth < 1010.f) || v < 0x1p-900 ? exact_steps<CHAIN, true>(team, w, a, u, v)
                                                                          : exact_steps<CHAIN, false>(team, w, a, u, v);
}

// What replaces a refused draft, the row's largest and the sum of its weights in sh. Every thread of the cluster gets it.
template <typename T> __device__ __noinline__ RowResult other_token(Team<T> team, Row<T> w, Asked a) {
  Shared& sh = *team.sh;
  const int ph = team.ph;
  const double v = number(a.raw_v, a.size);
  team.rest_pass(w, v);
  Found f{-1, 1, 0.f, 0};
  if (team.rank == sh.owner && threadIdx.x < 32) f = team.found_rest(w, v);
  f = team.share(f);
  if (f.unsure) {
    RowResult r = exact_row<true>(team, w, a);
    r.accept ^= (team.ph ^ ph) << 8;
    return r;
  }
  const double scaled = f.logit == sh.top ? 0. : ((double)f.logit - (double)sh.top) * w.c64;
  return {f.token, (team.ph ^ ph) << 8, scaled, sh.z};
}

// One row, by a whole cluster. LAZY: what fp32 does not decide, and what replaces a refused draft, is left for the walk, and
// the result is valid in warp 0 of the CTA *holder; otherwise every thread gets it.
template <bool CHAIN, bool LAZY, typename T>
CFB_DEV RowResult resolve(Team<T>& team, const Row<T>& w, const Asked& a, int* holder) {
  Shared& sh = *team.sh;
  const bool in = CHAIN && a.drafted && a.draft >= 0 && a.draft < w.V;       // a draft that is no token is refused
  const float of_draft = in ? to_float(w.p[a.draft]) : -INFINITY, q = in ? draft_prob(w, a.draft) : 0.f;
  team.stats(w, a.raw_v, a.size, a.greedy);
  const auto scaled = [&](float l) { return l == sh.top ? 0. : ((double)l - (double)sh.top) * w.c64; };     // log2
  const auto later = [&](int what) { return RowResult{-1, what, (double)sh.top, sh.z}; };
  const auto taken = [&](RowResult r) {
    team.ph ^= r.accept >> 8;
    r.accept &= 1;
    return r;
  };
  *holder = 0;
  if (sh.kind == ROW_EMPTY) return {-1, 0, 0., 1.};
  const bool plain = a.greedy || sh.kind == ROW_NAN;
  if (CHAIN && a.drafted && !plain) {
    if (in) {
      const float z = (float)sh.z, x = (of_draft - sh.top) * w.c, p = weight(of_draft, sh.top, w.c) * reciprocal(z);
      const float uq = (float)(number(a.raw_u, a.size) * (double)q);         // (u alone may be below fp32's range)
      // (every CTA computes the same) Weights below 2^-126 are flushed to 0, and uq and p rounded to 2^-149 there: 2^-124 for it
      const float off = p * (float)kRound * (2.f * team.band(w, z) + 2.08f * fabsf(x) + 16.f) + 0x1p-124f;
      if (!(fabsf(uq - p) > off)) {
        if constexpr (LAZY) return later(kUndecided);
        else return taken(exact_row<CHAIN>(team, w, a));
      }
      if (uq < p) return {a.draft, 1, scaled(of_draft), sh.z};
    }
    if constexpr (LAZY) return later(kRefused);
    else return taken(other_token(team, w, a));
  }
  *holder = sh.owner;
  Found f{-1, 1, 0.f, 0};
  if (team.rank == sh.owner && threadIdx.x < 32) {
    if (plain) f = {find_top(w, team.tops, static_cast<const float*>(team.room), sh.top, sh.kind == ROW_NAN), 0, sh.top, 0};
    else f = team.found(w, number(a.raw_v, a.size));
  }
  if constexpr (!LAZY) f = team.share(f);
  if (f.unsure) {
    if constexpr (LAZY) return later(kUndecided);
    else return taken(exact_row<CHAIN>(team, w, a));
  }
  return {f.token, CHAIN && plain && a.drafted && f.token == a.draft, sh.kind == ROW_NAN ? (double)NAN : scaled(f.logit), sh.z};
}

CFB_DEV uint2 number_at(const void* p, int size, long long i) {
  return size == 4 ? make_uint2(__ldg(static_cast<const uint32_t*>(p) + i), 0) : __ldg(static_cast<const uint2*>(p) + i);
}

// row j of request b, and what it is asked
template <typename T, bool CHAIN>
CFB_DEV void row_of(const VerifyArgs& A, int rank, int per, int b, int d0, int n, int s0, int j, float temp, Row<T>& w, Asked& a) {
  w.p = static_cast<const T*>(A.logits) + (long long)(s0 + j) * A.ld;
  w.V = A.V;
  w.shift = (int)((reinterpret_cast<uintptr_t>(w.p) & 15) / sizeof(T));
  const int units = (w.V + w.shift + kUnit - 1) / kUnit;
  w.u0 = min(rank * per, units);
  w.u1 = min(w.u0 + per, units);
  w.each = (per + kWarps - 1) / kWarps;
  a.greedy = !(temp >= kLowTemp);
  const float tau = a.greedy ? 1.f : fminf(temp, kHighTemp);
  w.c64 = tau == 1.f ? 1.4426950408889634 : 1.4426950408889634 / (double)tau;
  w.c = fminf((float)w.c64, 3.4e38f);
  w.probs = nullptr;
  w.index_of = A.index_of;
  w.width = A.index_of ? A.probs_width : A.V;
  a.drafted = CHAIN && j < n;
  a.draft = a.drafted ? A.draft_tokens[d0 + j] : -1;
  a.size = A.uniform_size;
  a.raw_u = a.drafted ? number_at(A.uniforms, A.uniform_size, d0 + j) : make_uint2(0, 0);
  a.raw_v = CHAIN ? number_at(A.resample, A.uniform_size, b) : number_at(A.uniforms, A.uniform_size, s0 + j);
  if (a.drafted) w.probs = A.probs + (long long)(d0 + j) * A.ld_probs;
}

// Bound by latency, not by a pipe (64 trees of 41 bf16 rows over 248320 tokens: SM 25 %, DRAM 19 %; a warp waits longest at
// barriers, for another CTA's totals or warp 0's descent): the rows of a walk come one after another. Cycles of a row, in a
// walk alone on the GPU / among 64 trees: units 3500 / 8900, reduction 600 / 1300, exchange 1900 / 3000, descent 3400 / 3700,
// handing over 900 / 1000; together 10400 / 17900, five of which are the deepest walk. A row that goes through 64 bits
// takes 17000 / 31500 more (with draft probabilities up to 80000). Measured at V = 248320: one chain of 5 drafts 13
// us, one tree of 40 22, 64 trees 68 (the visited rows' bytes: 14), one chain with draft probabilities 33, 48 of them 98 (17);
// without the rows in 64 bits 12, 17, 54, 27 and 63.
// FLAT: a cluster a row (grid.y: rows of a request, grid.z: requests), every row at once; the request's last
// cluster walks, and takes again what was left for the walk where it comes by. Otherwise a cluster a request (grid.y), which
// takes the rows of its walk in turn. CHAIN: draft probabilities; a node's only child is the next one.
template <typename T, bool CHAIN, bool FLAT>
__global__ void __launch_bounds__(kThreads, CHAIN ? 3 : 4) verify_kernel(const __grid_constant__ VerifyArgs A, int per) {
  extern __shared__ double s_dyn[];
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  // what a walk keeps: the results of its rows (in turn, or FLAT: of all rows), the rows it took, the tree
  constexpr int kPer = kUnit / kSpan<W64>;
  RowResult* const s_row = reinterpret_cast<RowResult*>(s_dyn + kPer * per);
  int* const s_node = reinterpret_cast<int*>(s_row + A.max_spec + 1);
  int* const s_next = s_node + A.max_spec + 1;             // FLAT: the child that a row's token leads to
  int* const s_parent = s_next + A.max_spec + 1;
  int* const s_token = s_parent + A.max_spec;
  Team<T> team{&sh, reinterpret_cast<float*>(s_token + A.max_spec), s_dyn, rank, ranks, 0};
  const int b = FLAT ? blockIdx.z : blockIdx.y;
  const int d0 = b ? A.cu_draft[b - 1] : 0;
  const long long drafts = (long long)A.cu_draft[b] - d0, start = A.cu_sampled[b] - (drafts + 1);
  const int before = b ? A.cu_sampled[b - 1] : 0;
  const float temp = A.temperature ? A.temperature[b] : 1.f;
  // Offsets that do not describe rows of this logits matrix (or drafts), or rows before the end of the last request's, are never
  // dereferenced. (Whether they fall on those of a request further back would take a look at all of them: such a request
  // reads what is another's, and writes to places of its own.)
  const bool sane = drafts >= 0 && drafts <= A.max_spec && start >= max(before, 0) && start + drafts < A.num_rows && d0 >= 0 &&
                    d0 + drafts <= A.num_drafts;
  const int n = (int)drafts, s0 = (int)start;
  RowResult* const rows = A.rows + (long long)b * (A.max_spec + 1);
  // a thread's node of the tree, on its way while the rows are taken
  const bool node = !CHAIN && sane && (int)threadIdx.x < n;
  const int my_parent = node ? A.parents[d0 + threadIdx.x] : 0, my_token = node ? A.draft_tokens[d0 + threadIdx.x] : 0;
  Row<T> w;
  Asked a;
  if constexpr (FLAT) {
    const int j = blockIdx.y;
    const bool live = sane && j <= n;
    int holder = 0;
    RowResult r{};
    if (live) {
      row_of<T, CHAIN>(A, rank, per, b, d0, n, s0, j, temp, w, a);
      r = resolve<CHAIN, true>(team, w, a, &holder);
    }
    if (rank == holder && threadIdx.x < 32) {              // count the row in, and tell the cluster if it was the last
      int last = 0;
      if (threadIdx.x == 0) {
        if (live) rows[j] = r;
        last = atom_add_acqrel(A.counter + b, 1u) + 1 == gridDim.y;
        if (last) A.counter[b] = 0u;
      }
      last = __shfl_sync(0xffffffffu, last, 0);
      if (threadIdx.x < ranks) *cluster.map_shared_rank(&sh.last, (int)threadIdx.x) = last;
    }
    cluster.sync();
    if (!sh.last) return;
  }
  if (sane) {
    for (int i = threadIdx.x; i <= n; i += kThreads) {
      if constexpr (FLAT) {
        const RowResult* const r = rows + i;
        const int2 t = __ldcg(reinterpret_cast<const int2*>(r));
        s_row[i] = {t.x, t.y, __ldcg(&r->scaled), __ldcg(&r->mass)};
        s_next[i] = n;
      }
      if (!CHAIN && i < n) {
        s_parent[i] = i < kThreads ? my_parent : A.parents[d0 + i];
        s_token[i] = i < kThreads ? my_token : A.draft_tokens[d0 + i];
      }
    }
    __syncthreads();
    if constexpr (FLAT && !CHAIN) {
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const int up = s_parent[i] + 1;                    // the row that leads to node i
        if (up >= 0 && up <= n && s_row[up].accept < kUndecided && s_row[up].token >= 0 && s_row[up].token == s_token[i])
          atomicMin(s_next + up, i);
      }
      __syncthreads();
    }
  }
  int pos = -1;                                            // the last token's place: accepted drafts
  bool remote = !FLAT;                                     // others may be reading this CTA's shared memory
  if (sane) {
    int cur = -1;
    for (;;) {                                             // (every thread of every CTA takes the same steps)
      RowResult r;
      bool known = FLAT;
      if constexpr (FLAT) {
        r = s_row[cur + 1];
        if (r.accept >= kUndecided) {
          row_of<T, CHAIN>(A, rank, per, b, d0, n, s0, cur + 1, temp, w, a);
          __syncthreads();                                   // (warps may still be deciding the row before from them)
          if (threadIdx.x == 0) {
            sh.top = (float)r.scaled;
            sh.z = r.mass;
          }
          __syncthreads();
          if constexpr (CHAIN) r = r.accept == kRefused ? other_token(team, w, a) : exact_row<true>(team, w, a);
          else r = exact_row<false>(team, w, a);
          team.ph ^= r.accept >> 8;
          r.accept &= 1;
          if (threadIdx.x == 0) s_row[cur + 1] = r;
          known = false;
          remote = true;
        }
      } else {
        int holder;
        row_of<T, CHAIN>(A, rank, per, b, d0, n, s0, cur + 1, temp, w, a);
        r = resolve<CHAIN, false>(team, w, a, &holder);
      }
      ++pos;
      if (threadIdx.x == 0) {
        s_node[pos] = cur;
        if constexpr (!FLAT) s_row[pos] = r;
      }
      int nxt = -1;
      if (pos < A.max_spec && r.token >= 0) {
        if constexpr (CHAIN) {
          nxt = r.accept && cur + 1 < n ? cur + 1 : -1;
        } else if (known) {
          nxt = s_next[cur + 1] < n ? s_next[cur + 1] : -1;
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
    if (remote) cluster.sync();                            // no CTA ends while another reads its shared memory
    __syncthreads();
  }
  if (rank != 0) return;
  for (int p = threadIdx.x; p <= A.max_spec; p += kThreads) {
    int token = -1;
    float logp = 0.f;
    if (p <= pos) {
      const RowResult r = s_row[FLAT ? s_node[p] + 1 : p];
      token = r.token;
      // formed in 64 bits and rounded once; the mass is the first pass's sum where the row was not taken again
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

// clusters of more than 8 CTAs allowed, once a device
template <typename T, bool CHAIN, bool FLAT> cudaError_t allow_clusters() {
  static std::atomic<bool> done[64];
  int dev = 0;
  if (const cudaError_t e = cudaGetDevice(&dev)) return e;
  if (dev < 64 && done[dev].load(std::memory_order_relaxed)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(verify_kernel<T, CHAIN, FLAT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess && dev < 64) done[dev].store(true, std::memory_order_relaxed);
  return e;
}
// clusters of a size that the current device holds at a time, asked of the runtime once a device
template <typename T, bool CHAIN, bool FLAT> int resident(int cluster) {
  static std::atomic<int> known[64][kMaxCluster + 1];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  if (dev < 64 && (n = known[dev][cluster].load(std::memory_order_relaxed)) > 0) return n;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(cluster);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = 16384;                            // (a large vocabulary's or tree's share of an SM)
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, verify_kernel<T, CHAIN, FLAT>, &cfg) != cudaSuccess) {
    cudaGetLastError();
    n = 0;
  }
  if (n > 0 && dev < 64) known[dev][cluster].store(n, std::memory_order_relaxed);
  return n;
}

template <typename T, bool CHAIN, bool FLAT>
cfb_status launch(const VerifyArgs& a, cudaStream_t st) {
  const auto bytes = [](long long units, long long spec) { return (int)(units * (kUnit / kSpan<W64> * 8 + 4) + (spec + 1) * 32 + spec * 8); };
  if (allow_smem<verify_kernel<T, CHAIN, FLAT>>(bytes(kMaxVocab / kUnit + 2, kMaxNodes)) != cudaSuccess ||
      allow_clusters<T, CHAIN, FLAT>() != cudaSuccess)
    return cfb_launch_status("verify_kernel");
  const long long units = (a.V + 7 + kUnit - 1) / kUnit;
  // as large clusters as are resident together (a cluster that waits for another's end doubles the time)
  const long long teams = FLAT ? a.num_rows : a.batch;
  int cluster = kMaxCluster;
  while (cluster > 1 && (cluster > units || teams > resident<T, CHAIN, FLAT>(cluster))) --cluster;
  const long long per = (units + cluster - 1) / cluster;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = FLAT ? dim3(cluster, a.max_spec + 1, a.batch) : dim3(cluster, a.batch, 1);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes(per, a.max_spec);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, verify_kernel<T, CHAIN, FLAT>, a, (int)per);
  return cfb_launch_status("verify_kernel");
}

// rows' results that the workspace of a call over num_rows rows holds
long long most_results(int num_rows) { return 4ll * num_rows + 256; }

template <bool CHAIN> cfb_status launch_as(const VerifyArgs& a, int dtype, cudaStream_t st) {
  // All rows at once take the GPU's whole width, but read what no walk reaches, the more so the more rows a request has, and
  // with more rows there are fewer CTAs for what the walk takes again. Measured, all rows at once / walk, us. Without draft probabilities,
  // 6 rows a request, V = 248320: 1 request 14 / 18, 8 33 / 46, 16 49 / 55, 64 160 / 80; V = 32003: 64 40 / 60. 41 rows a request,
  // V = 248320: 1 request 22 / 23 (eight draws of it), 2 35 / 24; V = 32003: 1 17 / 18, 4 25 / 30, 16 47 / 38; V = 5000: 16 20 / 29. With draft probabilities,
  // 6 rows, V = 248320: 1 request 17 / 24, 2 34 / 34, 4 53 / 51, 8 68 / 54; V = 32003: 16 41 / 46, 48 78 / 61.
  // (and a cluster goes to every row that a request may have: many that have none would cost more than they save)
  const long long most = (CHAIN ? 5ll : a.num_rows <= 16ll * a.batch ? 24ll : 12ll) << 20;      // elements
  const bool flat = (long long)a.V * a.num_rows <= most && (a.max_spec + 1ll) * a.batch <= most_results(a.num_rows);
  const auto go = [&](auto t) {
    using T = decltype(t);
    return flat ? launch<T, CHAIN, true>(a, st) : launch<T, CHAIN, false>(a, st);
  };
  if (dtype == DT_F32) return go(float{});
  if (dtype == DT_F16) return go(__half{});
  return go(__nv_bfloat16{});
}

// what both entry points check, and their common arguments
cfb_status common_args(VerifyArgs& a, const void* logits, int64_t ld, int num_rows, int V, int dtype, const int32_t* cu_draft,
                       const int32_t* cu_sampled, const int32_t* draft_tokens, const void* uniforms, const void* resample,
                       int uniform_size, const float* temperature, int num_drafts, int batch, int max_spec, int32_t* out_tokens, int32_t* out_len,
                       float* out_logp, void* ws, size_t ws_bytes, int* err) {
  if (num_rows <= 0 || V <= 0 || batch <= 0 || max_spec < 0 || ld < V) return CFB_ERR_INVALID_ARG;
  if (!logits || !cu_draft || !cu_sampled || !out_tokens || !out_len || !out_logp || !ws) return CFB_ERR_INVALID_ARG;
  if (num_drafts < 0 || (num_drafts > 0 && !draft_tokens)) return CFB_ERR_INVALID_ARG;
  if (dtype < DT_F32 || dtype > DT_BF16 || (uniform_size != 4 && uniform_size != 8)) return CFB_ERR_UNSUPPORTED;
  if (max_spec > kMaxNodes || V > kMaxVocab - 8 || batch > kMaxBatch) return CFB_ERR_UNSUPPORTED;
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == DT_F32 ? 4 : 2)) return CFB_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(uniforms) | reinterpret_cast<uintptr_t>(resample)) % uniform_size) return CFB_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(ws) & 255) || ws_bytes < cfb_verify_workspace(num_rows, batch)) return CFB_ERR_WORKSPACE;
  a.logits = logits; a.ld = ld; a.V = V; a.num_rows = num_rows;
  a.cu_draft = cu_draft; a.cu_sampled = cu_sampled; a.draft_tokens = draft_tokens;
  a.uniforms = uniforms; a.resample = resample; a.uniform_size = uniform_size; a.temperature = temperature;
  a.num_drafts = num_drafts; a.batch = batch; a.max_spec = max_spec;
  a.out_tokens = out_tokens; a.out_len = out_len; a.out_logp = out_logp;
  a.counter = static_cast<unsigned*>(ws);
  a.rows = reinterpret_cast<RowResult*>(static_cast<char*>(ws) + kCounters);
  a.err = err;
  return CFB_OK;
}

}  // namespace

extern "C" size_t cfb_verify_workspace(int num_rows, int batch) {
  if (num_rows <= 0 || batch <= 0) return 0;
  return kCounters + (size_t)most_results(num_rows) * sizeof(RowResult);
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
                                       nullptr, uniform_size, temperature, num_drafts, batch, max_spec_len, output_tokens, accepted_len,
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
                                       resample, uniform_size, temperature, num_drafts, batch, max_spec_len, output_tokens, accepted_len,
                                       logprobs, ws, ws_bytes, err))
    return s;
  if (probs_width <= 0 || ld_probs < probs_width || !resample || (num_drafts > 0 && (!draft_probs || !uniforms))) return CFB_ERR_INVALID_ARG;
  if (!index_of && probs_width != V) return CFB_ERR_INVALID_ARG;
  a.probs = draft_probs;
  a.ld_probs = ld_probs;
  a.probs_width = probs_width;
  a.index_of = index_of;
  return launch_as<true>(a, dtype, static_cast<cudaStream_t>(stream));
}
