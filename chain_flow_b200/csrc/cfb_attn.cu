// cfb_attn.cu -- attention of new tokens over a paged key/value cache (sm_100a), with its
// log-sum-exp: prompt chunks and single tokens (causal), and the prefix half of a tree step.
//
// For query row i of a request with n new tokens and L cached positions, over the allowed positions
// j (j < L, or j <= L - n + i):
//   s_j = scale q_i . k_j,  m = max s_j,  l = sum exp(s_j - m),  o_i = sum exp(s_j - m) v_j / l,
//   lse_i = m + log l.
// Over an e4m3 cache k_j = ks_j kc_j and v_j = vs_j vc_j (codes and scales), and
//   s_j = (scale ks_j) (q_i . kc_j),  w_j = s_j + log vs_j,  m = max w_j,
//   o_i = sum exp(w_j - m) vc_j / l,  l = sum exp(w_j - m) / vs_j,
// so the weights stay at most a fixed power of two, whatever the scales. Scores are formed on the 8-bit
// tensor path: keys as the codes they are, the query in e4m3 pieces of 4 bits, q = q1 + q2 (+ q3), two over
// bf16 (8 bits) and three over fp16 (11); a query row is first brought to a largest element of 128 to 256 by a
// power of two, so that what e4m3's smallest step (2^-9) loses of a small element is 2^-17 of the largest.
//
// Tiles of rows (a row: a query head of a token). 128, a row a lane of tensor memory. Where a request has at
// most few_rows on average (T rep <= few_rows B), tiles of that many, repeated in all four quarters of the
// lanes, each of which weighs a quarter of a unit's positions, so that a decode's softmax runs on eight warps:
//   16-bit: 32 rows (one decode of 9001 positions, 16 heads on 4 of 256: 21 us; with 128-row tiles 26);
//   e4m3: 8 rows, and in each quarter 8 lanes for each of four pieces of the query (piece_of), so that one product
//   forms all their scores; the weights are cut into pieces in the same lanes and meet the values' codes as they
//   are. (48 decodes
//   of up to 8192 positions, the same heads: 126 us. Over 128-row tiles, with V widened: 250; with the weights
//   in pieces: 170.)
// Over 128-row tiles the value codes are widened to 16 bits (exactly) on their way and meet 16-bit weights:
// there pieces of the weights would keep the conversion unit (a warp instruction in 16 cycles) busy (five
// prompts of up to 1500 tokens, 32 heads on 8 of 128: 440 us against 248, 253 since), and keys widened too would
// spend shared memory's bandwidth.
//
// What bounds it: over long prompts the tensor work (a prompt's chunk of 2048 tokens on 16384, 16 heads on 4 of
// 256: 429 us in a short run, 1200 TFLOP/s, 495 to 500 us and 1040 under the power cap; a 64-position product is
// issue-bound, 45 cycles for 32 of work, and D = 256 leaves tensor memory no room for wider ones); over short pieces
// and decodes what a piece costs besides its units (about 8 units' time) and a unit's chain of dependent steps.
#include <cuda_runtime.h>
#include <cuda_fp8.h>
#include <algorithm>
#include <cstdlib>
#include <numeric>
#include <type_traits>

#include "cfb_types.cuh"

using namespace cfb;

namespace {

// ---- the split ------------------------------------------------------------------------------------
// The query rows of one kv head of a request (its n tokens x rep heads, token-major) are cut into
// tiles of kM = 128 rows, the allowed positions of a tile into units of kKeys = 64. A piece of work
// is (request, kv head, row tile); the pieces, laid end to end, each its units and a fixed cost long, are dealt
// to the CTAs in equal contiguous shares, so one long context and a thousand short ones both keep every SM
// busy (without the cost, a CTA of 7 short pieces took 274000 cycles where one of a single piece took 176000:
// 48 decodes 150 us against 118). A piece cut by a share's end leaves partial results (unnormalised o, m, l,
// fp32) in the workspace, which attn_join_kernel adds up in unit order; a share holds at most two such pieces
// (its first and its last), so the workspace does not depend on the lengths. Shares depend only on the
// lengths: the same call gives the same bits.
constexpr int kM = 128, kKeys = 64;
__host__ __device__ constexpr int few_rows(bool e4m3) { return e4m3 ? 8 : 32; }
constexpr int kSoftWarps = 8, kMmaWarp = kSoftWarps, kLoadWarps = 4;
constexpr int kScaleStages = 4;
// A softmax thread holds a row; memory wants a warp's access to run along rows. 64 bytes of 32 rows at a time
// are turned in a buffer of the warp's own (row by row, a warp's access touched 32 lines: a piece's Q and O
// took 12000 and 5000 cycles so at 128 columns).
constexpr int kTurnPitch = 80;
constexpr uint32_t kScaleBytes = kKeys * 12;   // a unit's scales: [64] (k's with the softmax's, log2 v's), [64] 1 / v's
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// How the cache's rows come in: 16-bit or e4m3, by TMA where boxes of 8 rows or more tile both the pages
// and the units (gcd(page size, 64) >= 8), else row by row.
enum Source : int { TMA16 = 0, ROWS16 = 1, TMA8 = 2, ROWS8 = 3 };
__host__ __device__ constexpr bool is_e4m3(int src) { return src >= TMA8; }
__host__ __device__ constexpr bool is_tma(int src) { return (src & 1) == 0; }
// warps 0-7 softmax, 8 products, then two that issue the TMA copies of K and of V (over e4m3 one: registers, and
// over tiles of few rows a second one took 160 us where one took 151) or four that copy rows, and over e4m3 four
// that widen V and bring the scales, or two that bring the scales
__host__ __device__ constexpr int load_warps(int src) { return !is_tma(src) ? 4 : src == TMA8 ? 1 : 2; }
__host__ __device__ constexpr int code_warps(int src, int m) { return !is_e4m3(src) ? 0 : m == kM ? 4 : kKeys / 32; }
__host__ __device__ constexpr int threads_of(int src, int m) { return (9 + load_warps(src) + code_warps(src, m)) * 32; }

// division of 0 <= n < 2^31 by a fixed d: with 2^k >= 2^31 d, mul = ceil(2^k / d) < 2^32 is above 2^k / d by
// less than 1, so (n mul) >> k is floor(n / d)
struct Divisor {
  uint32_t mul; int k;
  CFB_DEV int of(int n) const { return (int)(((unsigned long long)(unsigned)n * mul) >> k); }
};

struct AttnArgs {
  const void* q; long long sq_t, sq_h;
  cfb_kv_cache c;
  const int32_t* table; long long st; int width;
  const int32_t* kv_len;
  const int32_t* cu_q;
  void* o; long long so_t, so_h;
  float* lse;
  float scale;
  int T, B, H, causal, rep;
  int m;                                  // rows of a row tile
  Divisor by_rep, by_page;
  int box;                                // rows of a TMA box
  uint32_t slab, group;                   // bytes between a tile's 64-column slabs and its 8-row groups
  struct Desc* desc;                      // [grid]
  float* part;                            // part_row
};

// What a piece costs besides its units (queries, results, a pipeline that fills and drains), in units.
constexpr int kPieceCost = 8;

struct Desc {                             // a piece that begins in this CTA's share and runs past its end
  int last;                               // the last CTA that holds a part of it; -1: no such piece
  int kh, t0, rows, row0;                 // kv head, first token row of the request, valid rows, first row of the tile
  int err;
  long long each;                         // the deal: units a CTA, and how many CTAs have one more
  int extra;
};

// where CTA `cta`'s share begins
CFB_DEV long long share(long long each, int extra, int cta) { return each * cta + min(cta, extra); }

struct Request { int t0, n, L; bool over; };
CFB_DEV Request request(const AttnArgs& A, int b) {
  Request r;
  r.t0 = min(max(A.cu_q[b], 0), A.T);
  r.n = min(max(A.cu_q[b + 1], r.t0), A.T) - r.t0;
  const long long cap = (long long)A.width * A.c.page_size;
  const int len = max(A.kv_len[b], 0);
  r.over = len > cap;
  r.L = r.over ? (int)cap : len;
  return r;
}
CFB_DEV int row_limit(const AttnArgs& A, const Request& r, int tok) {      // positions that token `tok` may see
  return A.causal ? max(min(r.L - r.n + tok + 1, r.L), 0) : r.L;
}
CFB_DEV int tiles_of(const AttnArgs& A, const Request& r) { return (r.n * A.rep + A.m - 1) / A.m; }
CFB_DEV int units_of(const AttnArgs& A, const Request& r, int tile) {
  const int last = A.by_rep.of(min((tile + 1) * A.m, r.n * A.rep) - 1);
  return max(1, (row_limit(A, r, last) + kKeys - 1) / kKeys);
}
// A kv head's units of request b, and its pieces' cost (0 past the last request), for the warp's 32 requests at
// once: a lane a request where it has one tile, else a request at a time with a lane a tile (a prompt of 1500
// tokens and 4 heads a kv head has 47; a lane adding those up took 26000 cycles).
__device__ __noinline__ int head_units(const AttnArgs& A, int b) {
  const int lane = threadIdx.x & 31;
  Request r = {0, 0, 0, false};
  if (b < A.B) r = request(A, b);
  const int tiles = tiles_of(A, r);
  unsigned longer = __ballot_sync(0xffffffffu, tiles > 1);
  int u = tiles == 1 ? units_of(A, r, 0) + kPieceCost : 0;
#pragma unroll 1
  for (; longer; longer &= longer - 1) {
    const int x = __ffs(longer) - 1;
    const Request y = {0, __shfl_sync(0xffffffffu, r.n, x), __shfl_sync(0xffffffffu, r.L, x), false};
    const int n = tiles_of(A, y);
    int sum = 0;
#pragma unroll 1
    for (int t = lane; t < n; t += 32) sum += units_of(A, y, t) + kPieceCost;
    sum = __reduce_add_sync(0xffffffffu, sum);
    if (lane == x) u = sum;
  }
  return u;
}

// A share, piece by piece; every warp of the CTA walks it alike. What runs once a piece or less is kept out of
// line, here and below: the kernel's roles run side by side, and their code has to share the instruction
// cache (inlined everywhere, a quarter of all warp cycles went by without an instruction to issue).
struct Walk {
  long long at, end;                      // where the piece begins and the share ends, with the pieces' costs
  int b, kh, tile, tiles, units, first;   // units of the piece; first unit of it in this share
  Request r;
  __device__ __noinline__ void start(const AttnArgs& A, long long from, long long to, int req, long long rest, int per_head) {
    end = to; b = req;
    r = request(A, b);
    tiles = tiles_of(A, r);
    kh = (int)(rest <= 0x7fffffff ? (unsigned)rest / (unsigned)per_head : rest / per_head);
    first = (int)(rest - (long long)kh * per_head);
    // the tile that holds it: 32 at a time, a lane a tile
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (tile = 0;; tile += 32) {
      const int mine = tile + lane < tiles ? units_of(A, r, tile + lane) + kPieceCost : 0;
      int run = mine;
#pragma unroll 1
      for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, run, off);
        if (lane >= off) run += y;
      }
      const unsigned here = __ballot_sync(0xffffffffu, first < run);
      if (here) {
        const int x = __ffs(here) - 1;
        tile += x;
        units = __shfl_sync(0xffffffffu, mine, x) - kPieceCost;
        first -= __shfl_sync(0xffffffffu, run - mine, x);
        at = from - first;
        first = max(first - kPieceCost, 0);
        break;
      }
      first -= __shfl_sync(0xffffffffu, run, 31);
    }
  }
  CFB_DEV bool done() const { return at + kPieceCost >= end; }
  CFB_DEV int stop() const { return (int)min((long long)units, end - at - kPieceCost); }     // first unit past this share's part
  __device__ __noinline__ void next(const AttnArgs& A) {
    at += kPieceCost + units;
    if (done()) return;
    first = 0;
    if (++tile == tiles) {
      tile = 0;
      if (++kh == A.c.kv_heads) {
        kh = 0;
        do {
          r = request(A, ++b);
          tiles = tiles_of(A, r);
        } while (tiles == 0);
      }
    }
    units = units_of(A, r, tile);
  }
};

// ---- shared and tensor memory ------------------------------------------------------------------------
// K and V tiles are 128-byte-swizzled: groups of 8 rows of 64 columns (128 B), a row's 16-byte pieces
// XORed with row & 7, as [slab of 64 columns][group] or, where the pages are no multiple of a unit,
// [group][slab], so that one TMA box of 8 rows brings all their columns. K is read K-major (the head dim is
// summed over), V MN-major (the positions are), from the same image. Q lies in tensor memory: as the first operand of S = Q K^T it would be read from
// shared memory again with every unit, and a 128 x 64 product of 16 reads 4 KB of it in its 32 cycles,
// the whole shared-memory bandwidth. Tensor memory columns: two units' S (fp32), each overwritten by
// its P (16-bit), then Q, then O.
// The partial results: rows of kPart floats (o, m, l), eight rows of a CTA side by side and then the CTAs,
// so that the few rows of a decode step lie together however many CTAs share them.
template <int D> constexpr int kPart = D + 4;
template <int D>
CFB_DEV float* part_row(float* part, int grid, int cta, int which, int row) {
  return part + ((((long long)(row >> 3) * 2 + which) * grid + cta) * 8 + (row & 7)) * kPart<D>;
}
template <int D, int SRC, int M>
struct Layout {
  static constexpr bool kWiden = is_e4m3(SRC) && M == kM;                   // V's codes to 16 bits
  static constexpr int kElem = is_e4m3(SRC) ? 1 : 2;                       // stored bytes an element
  static constexpr int kRowB = D * kElem < 128 ? 64 : 128, kSlabs = D * kElem / kRowB;   // a slab's row
  static constexpr int kStages = SRC == ROWS16 ? 2 : D == 256 && (kWiden || !is_e4m3(SRC)) ? 3 : 4;
  static constexpr uint32_t kTile = kKeys * D * kElem;
  // over e4m3: two stages of V widened, [64-column slab][row]; a third piece of Q that tensor memory has no
  // room for (D = 256)
  static constexpr uint32_t kWide = kKeys * D * 2;
  static constexpr uint32_t off_k = 0, off_v = kStages * kTile, off_w = 2 * kStages * kTile, off_q3 = off_w + (kWiden ? 2 * kWide : 0);
  static constexpr uint32_t off_turn = off_q3 + (kWiden && D == 256 ? kM * D : 0);
  static constexpr uint32_t off_scale = off_turn + kSoftWarps * 32 * kTurnPitch;
  static constexpr uint32_t bytes = off_scale + (is_e4m3(SRC) ? kScaleStages * kScaleBytes : 0) + 1024;
  static constexpr uint32_t s_col = 0, q_col = 2 * kKeys, o_col = D == 64 ? 192 : 256;
  static constexpr uint32_t cols = D == 64 ? 256 : 512;
};

// full / empty: a stage's tile has landed / its product has read it (sc: a unit's scales; w: V widened, the
// codes' stage then free). q_ready: Q is in
// tensor memory. s_done / o_done: the product S(i) / O += P(i) V(i) has completed. p_full: P(i) is written
// (and S(i) read). m_set: the rows' maximum after unit i is in shared memory. o_free: the piece's O has
// been read.
struct Bars {
  uint64_t q_ready, k_full[4], k_empty[4], v_full[4], v_empty[4], w_full[2], w_empty[2], s_done[2], p_full[2], o_done[2], o_free, meet,
      sc_full[kScaleStages], sc_empty[kScaleStages], m_set[2][4], swap[4], drain;
};

CFB_DEV void st_shared16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
CFB_DEV void tmem_ld32(uint32_t taddr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
CFB_DEV void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
CFB_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
CFB_DEV void tmem_st4(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
CFB_DEV void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
CFB_DEV void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
         "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// D[tmem] (+)= A[tmem] . B[smem] over N steps of 32 bytes of the summed dim in one statement, by one elected
// lane (one election and one statement for four take less issue time than four), B's descriptor advancing
// by `step`. F8: e4m3, else 16-bit operands.
template <int N, bool F8>
CFB_DEV void mma_ts_warp(uint32_t tmem_d, uint32_t tmem_a, uint64_t b, uint32_t step, uint32_t idesc, uint32_t accumulate) {
#define CFB_TS4(KIND)                                                                                                        \
  asm volatile("{\n\t.reg .pred p, q;\n\telect.sync _|p, 0xffffffff;\n\tsetp.ne.b32 q, %4, 0;\n\t"                           \
               "@p tcgen05.mma.cta_group::1.kind::" KIND " [%0], [%1], %2, %3, q;\n\t"                                       \
               "@p tcgen05.mma.cta_group::1.kind::" KIND " [%0], [%5], %8, %3, 1;\n\t"                                       \
               "@p tcgen05.mma.cta_group::1.kind::" KIND " [%0], [%6], %9, %3, 1;\n\t"                                       \
               "@p tcgen05.mma.cta_group::1.kind::" KIND " [%0], [%7], %10, %3, 1;\n\t}"                                     \
               :: "r"(tmem_d), "r"(tmem_a), "l"(b), "r"(idesc), "r"(accumulate), "r"(tmem_a + 8),                           \
                  "r"(tmem_a + 16), "r"(tmem_a + 24), "l"(b + step), "l"(b + 2 * step), "l"(b + 3 * step) : "memory")
#define CFB_TS2(KIND)                                                                                                        \
  asm volatile("{\n\t.reg .pred p, q;\n\telect.sync _|p, 0xffffffff;\n\tsetp.ne.b32 q, %4, 0;\n\t"                           \
               "@p tcgen05.mma.cta_group::1.kind::" KIND " [%0], [%1], %2, %3, q;\n\t"                                       \
               "@p tcgen05.mma.cta_group::1.kind::" KIND " [%0], [%5], %6, %3, 1;\n\t}"                                      \
               :: "r"(tmem_d), "r"(tmem_a), "l"(b), "r"(idesc), "r"(accumulate), "r"(tmem_a + 8), "l"(b + step) : "memory")
  static_assert(N == 4 || (N == 2 && F8), "steps");
  if constexpr (!F8) CFB_TS4("f16");
  else if constexpr (N == 4) CFB_TS4("f8f6f4");
  else CFB_TS2("f8f6f4");
#undef CFB_TS4
#undef CFB_TS2
}
// D[tmem] += A[smem] . B[smem], e4m3, over four steps of 32 columns (128-byte rows of both)
CFB_DEV void mma_ss4_f8_warp(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, 1;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %4, %7, %3, 1;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %5, %8, %3, 1;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %6, %9, %3, 1;\n\t}"
      :: "r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "l"(a + 2), "l"(a + 4), "l"(a + 6), "l"(b + 2), "l"(b + 4), "l"(b + 6) : "memory");
}
// swizzled operands of rows of 128 bytes, or of 64: K-major, 8-row groups `group` bytes apart; MN-major, slabs
// of a row's elements `slab` and 8-row groups `group` bytes apart
template <int ROWB> CFB_DEV constexpr uint64_t swizzle_bits() { return (1ull << 46) | (ROWB == 128 ? 2ull << 61 : 4ull << 61); }
template <int ROWB> CFB_DEV uint64_t k_major(uint32_t saddr, uint32_t group) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (1ull << 16) | ((uint64_t)(group >> 4) << 32) | swizzle_bits<ROWB>();
}
template <int ROWB> CFB_DEV uint64_t mn_major(uint32_t saddr, uint32_t slab, uint32_t group) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(slab >> 4) << 16) | ((uint64_t)(group >> 4) << 32) | swizzle_bits<ROWB>();
}
template <typename T>
CFB_DEV constexpr uint32_t type_bits() {          // operand formats of the instruction descriptor
  return sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
}
CFB_DEV void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {     // 16 bytes, zeros past `bytes`
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(bytes) : "memory");
}
// one arrival on `bar` when every earlier cp.async of this thread has landed
CFB_DEV void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" :: "r"(smem_u32(bar)) : "memory");
}
CFB_DEV void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// two fp32 operations in one instruction
CFB_DEV float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)));
  return d;
}
CFB_DEV float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)));
  return d;
}
CFB_DEV float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)),
        "l"(reinterpret_cast<const unsigned long long&>(c)));
  return d;
}
CFB_DEV float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
CFB_DEV float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A value's scale as the weights take it, with its logarithm and its inverse: at least 2^-60, so that a row whose scale
// is 0 (a slot never written, a row of zeros) keeps its part of the sum, and stays out of o but for 448 2^-60. The sum loses
// a position only where its weight is less than 2^-66 of another's of scale 1. (Patterns order like integers: what is NaN
// or negative is larger, and its logarithm is NaN.)
CFB_DEV float value_scale(float x) {
  return __uint_as_float(max(__float_as_uint(x + 0.f), __float_as_uint(0x1p-60f)));
}

// What the key rows of a page outside the pool read: NaN in both 16-bit types.
__device__ const uint4 kNanRow[1] = {{0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu}};

// Where the row of position j lies; -1 if its page is none of the pool's.
CFB_DEV long long row_offset(const AttnArgs& A, int b, int kh, int j, long long* scale_off) {
  const int p = A.by_page.of(j), off = j - p * A.c.page_size;
  const int page = __ldg(A.table + (long long)b * A.st + p);
  if (page < 0 || page >= A.c.pages) return -1;
  if (scale_off)
    *scale_off = (long long)page * A.c.scale_page_stride + kh * A.c.scale_head_stride + off * A.c.scale_slot_stride;
  return (long long)page * A.c.page_stride + kh * A.c.head_stride + off * A.c.slot_stride;
}

// eight e4m3 codes -> eight elements of T, exactly: exponent and mantissa bits moved to T's places are the value
// times 2^(7 - T's bias) (subnormals come out as subnormals), and a product by the inverse undoes that
template <typename T>
CFB_DEV uint4 widen8(uint32_t lo, uint32_t hi) {
  const auto two = [](uint32_t w, uint32_t pick) {
    const uint32_t t = __byte_perm(w, 0, pick);                // each half: code << 8
    if constexpr (std::is_same<T, __half>::value) {
      const uint32_t x = (t & 0x80008000u) | (t >> 1 & 0x3f803f80u);
      const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&x), __float2half2_rn(256.f));
      return *reinterpret_cast<const uint32_t*>(&y);
    } else {
      const uint32_t x = (t & 0x80008000u) | (t >> 4 & 0x07f007f0u);
      const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&x),
                                       __halves2bfloat162(__ushort_as_bfloat16(0x7b80), __ushort_as_bfloat16(0x7b80)));   // 2^120
      return *reinterpret_cast<const uint32_t*>(&y);
    }
  };
  return make_uint4(two(lo, 0x1404), two(lo, 0x3424), two(hi, 0x1404), two(hi, 0x3424));
}

// the same where a code may be a NaN (0x7f, 0xff; any_nan: a word of four has one), which widen8 would read as 480
CFB_DEV uint32_t any_nan(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
template <typename T>
__device__ __noinline__ uint4 widen8_nan(uint32_t lo, uint32_t hi) {
  const auto two = [](uint32_t w) {
    __nv_fp8_e4m3 a, b;
    a.__x = w & 0xff;
    b.__x = w >> 8 & 0xff;
    return pack16<T>((float)a, (float)b);
  };
  return make_uint4(two(lo), two(lo >> 16), two(hi), two(hi >> 16));
}

// Four values as e4m3: the leading piece, and what it leaves. The piece is the value rounded to 4 bits by an
// integer addition, which the conversion then takes as it is (it rounds only below e4m3's normal range,
// by at most half its smallest step).
CFB_DEV uint32_t e4m3_of(const float (&x)[4]) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}
CFB_DEV uint32_t take_piece(float (&x)[4]) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[i] = __uint_as_float((__float_as_uint(x[i]) + 0x00080000u) & 0xfff00000u);
    x[i] -= y[i];
  }
  return e4m3_of(y);
}
template <typename T> constexpr int kPieces = std::is_same<T, __half>::value ? 3 : 2;

// eight elements of a query row, times `up`, in pieces
template <typename T> struct QPieces { uint32_t w[kPieces<T>][2]; };
template <typename T>
__device__ __noinline__ QPieces<T> query_pieces(uint4 q, float up) {
  QPieces<T> p;
  const uint32_t y[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int z = 0; z < 2; ++z) {
    const float2 f = unpack16<T>(y[2 * z]), h = unpack16<T>(y[2 * z + 1]);
    float v[4] = {f.x * up, f.y * up, h.x * up, h.y * up};
#pragma unroll
    for (int n = 0; n < kPieces<T> - 1; ++n) p.w[n][z] = take_piece(v);
    p.w[kPieces<T> - 1][z] = e4m3_of(v);
  }
  return p;
}

// Piece n of four values, |v| < 2^8.6, where every piece has lanes, and so a scale, of its own: v = p0 + p1 / 16 +
// p2 / 256 + p3 / 4096. With c_n the value rounded to 4 (n + 1) bits, but to no less than 2^(-9 - 4 n), p_n =
// 16^n (c_n - c_(n-1)) is at most 8 steps of c_n's, 4 bits, in e4m3's range: the conversion takes it as it is.
// (Rounding: adding and taking off 1.5 times the power of two whose last place is the step.) So a value keeps 16
// bits, and nothing above 2^-22 is lost: of a row's weights, one of 2^-29 of the largest. (Pieces of one scale
// lose what is below 2^-10: under a position that takes most of a row's weight, 8000 others can be a tenth of it
// together and vanish so. They took 118 us where these take 128, at the 48 decodes above.)
CFB_DEV uint32_t piece_of(float (&v)[4], int n) {
  const float up = __uint_as_float((127u + 4u * n) << 23), prev = n ? -up : 0.f;               // 16^n
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    float2 m, before;
    const auto step = [&](float x) {
      return ((__float_as_uint(fmaxf(fabsf(x), 0x1p-6f)) & 0x7f800000u) | 0x00400000u) + ((20u - 4u * n) << 23);
    };
    const uint32_t a = step(v[i]), b = step(v[i + 1]);
    m = make_float2(__uint_as_float(a), __uint_as_float(b));
    before = make_float2(__uint_as_float(a + (4u << 23)), __uint_as_float(b + (4u << 23)));
    const float2 x = make_float2(v[i], v[i + 1]);
    const float2 c = add2(add2(x, m), make_float2(-m.x, -m.y)), c1 = add2(add2(x, before), make_float2(-before.x, -before.y));
    const float2 p = fma2(c1, make_float2(prev, prev), mul2(c, make_float2(up, up)));
    v[i] = p.x;
    v[i + 1] = p.y;
  }
  return e4m3_of(v);
}
template <typename T>
__device__ __noinline__ uint2 query_piece(uint4 q, float up, int n) {
  const float2 a = unpack16<T>(q.x), b = unpack16<T>(q.y), c = unpack16<T>(q.z), d = unpack16<T>(q.w);
  float v[4] = {a.x * up, a.y * up, b.x * up, b.y * up}, w[4] = {c.x * up, c.y * up, d.x * up, d.y * up};
  return make_uint2(piece_of(v, n), piece_of(w, n));
}

// What the CTA's waits watch besides their barriers: dead, a wait has expired; alive, when mend_rows last got on.
struct Watch { int dead; unsigned long long alive; };

// The rest of a wait that was not over at once; false if it never was, or another one of the CTA was not. The limit
// starts anew while rows are mended (loops over a row's positions, which end, but take what they take).
__device__ __noinline__ bool wait_on(uint64_t* b, uint32_t parity, volatile Watch* watch) {
  bool ok = true;
  const unsigned long long t0 = globaltimer();
#pragma unroll 1
  for (unsigned it = 1; !mbar_try_wait(b, parity); ++it)
    if (it % kPollsPerCheck == 0) {
      if (wait_expired(max(t0, watch->alive), kWaitBudgetNs)) watch->dead = 1;
      if (watch->dead != 0) {
        ok = false;
        break;
      }
    }
  return __all_sync(0xffffffffu, ok) != 0;
}

// N stored elements (e4m3 codes or T) as fp32; their words as one access
template <int BYTES> struct WordsOf;
template <> struct WordsOf<1> { using type = uint8_t; };
template <> struct WordsOf<2> { using type = uint16_t; };
template <> struct WordsOf<4> { using type = uint32_t; };
template <> struct WordsOf<8> { using type = uint2; };
template <> struct WordsOf<16> { using type = uint4; };
template <typename Stored, int N>
CFB_DEV void widen_all(const typename WordsOf<N * sizeof(Stored)>::type& words, float (&x)[N]) {
  const Stored* const y = reinterpret_cast<const Stored*>(&words);
#pragma unroll
  for (int e = 0; e < N; ++e) {
    if constexpr (sizeof(Stored) == 1) x[e] = (float)y[e];
    else x[e] = to_float(y[e]);
  }
}
template <typename T, bool QUANT> using StoredOf = std::conditional_t<QUANT, __nv_fp8_e4m3, T>;

// Rows whose product met a value that is not finite, among them rows that do not see its position and met it with a
// weight of 0. A column in which a row sees such values is what they add up to (an infinity, or NaN); the columns
// [half * D / 2, ...) are put so in the CTA's partial result `which`, or (-1) the output. Returned: the rows that have a column
// in which they see none but whose product met one, to be taken again. `again`: the warp's rows, a lane each (the
// tile's row row0 + lane), with `seen`, where a row's positions end, in the lane. The tile's positions: [from, to),
// of which every row sees those before `hidden`; nothing is wrong where none of the others holds such a value.
template <typename T, int D, bool QUANT>
__device__ __noinline__ unsigned put_spoilt(const AttnArgs& A, const Walk& w, int row0, unsigned again, int from, int hidden, int to, int seen,
                                            int half, int which, volatile Watch* watch) {
  constexpr int E = D / 64, kAhead = 4;
  using Stored = StoredOf<T, QUANT>;
  using Words = typename WordsOf<E * sizeof(Stored)>::type;
  const int lane = threadIdx.x & 31;
  int nan[E], up[E], down[E];                                  // of this lane's columns: the first NaN, infinity, negative infinity
#pragma unroll
  for (int e = 0; e < E; ++e) nan[e] = up[e] = down[e] = to;
  const auto look = [&](int a, int z) {
#pragma unroll 1
    for (int j0 = a; j0 < z; j0 += 32) {
      // (no such page: zeros in the product)
      const long long off = j0 + lane < z ? row_offset(A, w.b, w.kh, j0 + lane, nullptr) : -1;
#pragma unroll 1
      for (int c = 0; c < 32 && j0 + c < z; c += kAhead) {
        Words vw[kAhead];
#pragma unroll
        for (int x = 0; x < kAhead; ++x) {
          const long long o = __shfl_sync(0xffffffffu, off, c + x);
          vw[x] = Words{};
          if (o >= 0) vw[x] = __ldg(reinterpret_cast<const Words*>(static_cast<const Stored*>(A.c.v) + o + half * (D / 2)) + lane);
        }
#pragma unroll
        for (int x = 0; x < kAhead; ++x) {
          float v[E];
          widen_all<Stored, E>(vw[x], v);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            if (v[e] != v[e]) nan[e] = min(nan[e], j0 + c + x);
            if (v[e] == INFINITY) up[e] = min(up[e], j0 + c + x);
            if (v[e] == -INFINITY) down[e] = min(down[e], j0 + c + x);
          }
        }
      }
      if (lane == 0) watch->alive = globaltimer();
    }
  };
  const auto first = [&](int e) { return min(nan[e], min(up[e], down[e])); };
  look(hidden, to);
  bool any = false;
#pragma unroll
  for (int e = 0; e < E; ++e) any |= first(e) < to;
  if (!__any_sync(0xffffffffu, any)) return 0;
  look(from, hidden);
  unsigned rest = 0;
#pragma unroll 1
  for (; again; again &= again - 1) {
    const int src = __ffs(again) - 1, stop = __shfl_sync(0xffffffffu, seen, src);
    const int R = w.tile * A.m + row0 + src, tok = A.by_rep.of(R), head = w.kh * A.rep + R - tok * A.rep;
    const int at = half * (D / 2) + lane * E;
    T* const out = static_cast<T*>(A.o) + (long long)(w.r.t0 + tok) * A.so_t + head * A.so_h + at;
    float* const part = part_row<D>(A.part, gridDim.x, blockIdx.x, max(which, 0), row0 + src) + at;
    bool met = false;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool n = nan[e] < stop || (up[e] < stop && down[e] < stop), p = up[e] < stop;
      if (n || p || down[e] < stop) {
        const float y = n ? __int_as_float(0x7fc00000) : p ? INFINITY : -INFINITY;
        if (which < 0) out[e] = from_float<T>(y);
        else part[e] = y;
      } else {
        met |= first(e) < to;
      }
    }
    if (__any_sync(0xffffffffu, met)) rest |= 1u << src;
  }
  return rest;
}

// Rows taken again: o over positions [from, seen) of each row's own, from its m, the columns [half * D / 2, ...) of it,
// into the CTA's partial result `which` or (-1) divided by its sum into the output; rows as above. Two rows at a time share
// the keys and values, in few registers (four rows of two positions ahead took 0.28 to 0.8 s where two take 0.46 to 0.8
// below, but the kernel spilled round the call: 48 decodes 131 us against 125).
// (148 tiles of 64 to 128 rows over 131072 positions: each spoilt by its last token's value alone, so that all other rows are
// taken again, 0.46 s, 0.8 at 256 columns; by every value of a column, so that put_spoilt does, 20 to 29 ms; clean, 1.5 to 4.)
template <typename T, int D, bool QUANT>
__device__ __noinline__ void rows_again(const AttnArgs& A, const Walk& w, int row0, unsigned again, int from, int seen, float m, float inv,
                                        int half, int which, volatile Watch* watch) {
  constexpr int E = D / 32, EV = D / 64, kRows = 2, kAhead = 2;
  using Stored = StoredOf<T, QUANT>;
  using KeyWords = typename WordsOf<E * sizeof(Stored)>::type;
  using ValueWords = typename WordsOf<EV * sizeof(Stored)>::type;
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  while (again) {
    int src[kRows], to[kRows], stop = 0, n = 0;
    float x[kRows][E], acc[kRows][EV], top[kRows], over[kRows];
    T* out[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      src[i] = again ? __ffs(again) - 1 : src[0];              // (rows short of four repeat the first, unwritten)
      if (again) ++n;
      again &= again - 1;
      to[i] = __shfl_sync(0xffffffffu, seen, src[i]);
      top[i] = __shfl_sync(0xffffffffu, m, src[i]);
      over[i] = __shfl_sync(0xffffffffu, inv, src[i]);
      stop = max(stop, to[i]);
      const int R = w.tile * A.m + row0 + src[i], tok = A.by_rep.of(R), head = w.kh * A.rep + R - tok * A.rep;
      const T* const q = static_cast<const T*>(A.q) + (long long)(w.r.t0 + tok) * A.sq_t + head * A.sq_h;
      out[i] = static_cast<T*>(A.o) + (long long)(w.r.t0 + tok) * A.so_t + head * A.so_h;
#pragma unroll
      for (int e = 0; e < E; ++e) x[i][e] = to_float(q[lane * E + e]);
#pragma unroll
      for (int e = 0; e < EV; ++e) acc[i][e] = 0.f;
    }
#pragma unroll 1
    for (int j0 = from; j0 < stop; j0 += 32) {
      long long so = 0;                                        // this lane's position; -1: no such page
      const long long off = j0 + lane < stop ? row_offset(A, w.b, w.kh, j0 + lane, QUANT ? &so : nullptr) : -1;
      float ks = A.scale * kLog2e, vs = 0.f;
      if (QUANT && off >= 0) {
        ks *= __ldg(A.c.k_scale + so);
        vs = log2f(value_scale(__ldg(A.c.v_scale + so)));
      }
#pragma unroll 1
      for (int c = 0; c < 32 && j0 + c < stop; c += kAhead) {
        KeyWords kw[kAhead];
        ValueWords vw[kAhead];
        bool there[kAhead];
#pragma unroll
        for (int z = 0; z < kAhead; ++z) {
          const long long o = __shfl_sync(0xffffffffu, off, c + z);
          there[z] = o >= 0;
          kw[z] = KeyWords{};
          vw[z] = ValueWords{};
          if (o >= 0) {
            kw[z] = __ldg(reinterpret_cast<const KeyWords*>(static_cast<const Stored*>(A.c.k) + o) + lane);
            vw[z] = __ldg(reinterpret_cast<const ValueWords*>(static_cast<const Stored*>(A.c.v) + o + half * (D / 2)) + lane);
          }
        }
        float s[kAhead][kRows];
#pragma unroll
        for (int z = 0; z < kAhead; ++z) {
          float k[E];
          widen_all<Stored, E>(kw[z], k);
#pragma unroll
          for (int i = 0; i < kRows; ++i) {
            s[z][i] = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) s[z][i] = fmaf(x[i][e], k[e], s[z][i]);
          }
        }
#pragma unroll
        for (int y = 16; y; y >>= 1)
#pragma unroll
          for (int z = 0; z < kAhead; ++z)
#pragma unroll
            for (int i = 0; i < kRows; ++i) s[z][i] += __shfl_xor_sync(0xffffffffu, s[z][i], y);
#pragma unroll
        for (int z = 0; z < kAhead; ++z) {
          const float f = __shfl_sync(0xffffffffu, ks, c + z), add = __shfl_sync(0xffffffffu, vs, c + z);
          float v[EV];
          widen_all<Stored, EV>(vw[z], v);
#pragma unroll
          for (int i = 0; i < kRows; ++i) {
            if (!there[z] || j0 + c + z >= to[i]) continue;    // (no such page: the score is NaN, so is l, and the row is not here)
            const float p = exp2_approx(fmaf(s[z][i], f, add) - top[i]);
#pragma unroll
            for (int e = 0; e < EV; ++e) acc[i][e] = fmaf(p, v[e], acc[i][e]);
          }
        }
      }
      if (lane == 0) watch->alive = globaltimer();
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (i >= n) continue;
      const int at = half * (D / 2) + lane * EV;
      if (which < 0) {
#pragma unroll
        for (int e = 0; e < EV; ++e) out[i][at + e] = from_float<T>(acc[i][e] * over[i]);
      } else {
        float* const p = part_row<D>(A.part, gridDim.x, blockIdx.x, which, row0 + src[i]);
#pragma unroll
        for (int e = 0; e < EV; ++e) p[at + e] = acc[i][e];
      }
    }
  }
}

// The rows `again` (a lane each) of a softmax warp whose product met a value that is not finite; m and inv in the lanes.
template <typename T, int D, bool QUANT>
__device__ __noinline__ void mend_rows(const AttnArgs& A, const Walk& w, unsigned again, float m, float inv, volatile Watch* watch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = warp >> 2, row0 = A.m == kM ? (warp & 3) * 32 : 0;
  const int from = w.first * kKeys, stop = w.stop() * kKeys, to = min(row_limit(A, w.r, w.r.n - 1), stop);
  const int which = w.first == 0 && stop == w.units * kKeys ? -1 : w.first == 0;
  const int seen = min(row_limit(A, w.r, A.by_rep.of(w.tile * A.m + row0 + lane)), stop);
  // (tiles of few rows: every value has met weights of 0)
  const int low = A.m == kM ? __reduce_min_sync(0xffffffffu, again >> lane & 1 ? seen : 0x7fffffff) : 0;
  again = put_spoilt<T, D, QUANT>(A, w, row0, again, from, max(low, from), to, seen, half, which, watch);
  if (again) rows_again<T, D, QUANT>(A, w, row0, again, from, seen, m, inv, half, which, watch);
}

// ---- the kernel -----------------------------------------------------------------------------------
// One CTA per SM. The loading warps (Source) fill, per unit, a K and a V tile: pages are found through the page
// table a unit early, positions past the end are zeros where it matters (V). Warp 8 issues the tensor work:
// S(i) = Q K(i)^T into one of two fp32 tiles in tensor memory, then O += P(i-1) V(i-1) with P read from tensor
// memory, so the softmax of a unit runs beside the next unit's product. Warps 0-7 are the softmax, a thread a
// lane, units alternating between two groups: the lane's scores come from tensor memory, and the weights go
// back there in the operands' type (the one rounding of the weights: unit roundoff 2^-8 bf16, 2^-11 fp16, 2^-17
// in pieces; their sum is of the unrounded fp32 values). O is rescaled only when the row's maximum has grown by
// more than 2^kSlack since the last time: weights are then at most 2^8 (fp16: 2^15, and the largest at least 2^7; in
// pieces 2^8.5 and 2^6.5), inside the types, and most units touch O not at all.
template <typename T, int D, int SRC, int M>
__global__ void __launch_bounds__(threads_of(SRC, M), 1)
attn_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  using Lay = Layout<D, SRC, M>;
  constexpr bool QUANT = is_e4m3(SRC);
  constexpr bool SPREAD = M < kM;
  constexpr bool PIECES = QUANT && SPREAD, WIDEN = QUANT && !SPREAD;
  constexpr int kCols = SPREAD ? kKeys / 4 : kKeys;            // a unit's columns of a softmax thread
  // the weights are at most 2^(kLift + kSlack), and o is rescaled only when the maximum has grown by 2^kSlack. (fp16: at
  // most 2^15, so that its smallest step, 2^-24, is 2^-31 of the largest or less: at 2^-24, thousands of small weights
  // under a large one vanished together.)
  constexpr float kLift = PIECES ? 6.5f : std::is_same<T, __half>::value ? 7.f : 0.f, kSlack = PIECES ? 2.f : 8.f;
  constexpr int kSt = Lay::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Bars bar;
  __shared__ uint32_t tmem_slot;
  __shared__ Watch watch;
  __shared__ long long sh_total[32];
  __shared__ float sh_m[2][kM];
  __shared__ float2 sh_swap[2][2 * kM];                        // [buffer][group][lane of tensor memory]: its maximum and sum
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const sm = smem_raw + (base - smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int grid = gridDim.x, cta = blockIdx.x;

  if (threadIdx.x == 0) {
    mbar_init(&bar.q_ready, kSoftWarps);
#pragma unroll 1
    for (int i = 0; i < kSt; ++i) {
      mbar_init(&bar.k_full[i], is_tma(SRC) ? 1 : kLoadWarps * 32); mbar_init(&bar.k_empty[i], 1);
      mbar_init(&bar.v_full[i], is_tma(SRC) ? 1 : kLoadWarps * 32); mbar_init(&bar.v_empty[i], WIDEN ? 4 : 1);
    }
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.w_full[i], 4 * 32); mbar_init(&bar.w_empty[i], 1);
      mbar_init(&bar.s_done[i], 1); mbar_init(&bar.p_full[i], kSoftWarps / 2); mbar_init(&bar.o_done[i], 1);
#pragma unroll 1
      for (int j = 0; j < 4; ++j) mbar_init(&bar.m_set[i][j], 1);
    }
    mbar_init(&bar.o_free, kSoftWarps);
#pragma unroll 1
    for (int i = 0; i < kScaleStages; ++i) { mbar_init(&bar.sc_full[i], kKeys / 32); mbar_init(&bar.sc_empty[i], kSoftWarps / 2); }
#pragma unroll 1
    for (int i = 0; i < 4; ++i) mbar_init(&bar.swap[i], 2);
    mbar_init(&bar.drain, 1);
    mbar_init(&bar.meet, kSoftWarps);
    fence_mbar_init();
    watch.dead = 0;
    watch.alive = 0;
    A.desc[cta].last = -1;
    A.desc[cta].err = 0;
  }
  if (warp == kMmaWarp) tmem_alloc(&tmem_slot, Lay::cols);
  if (is_tma(SRC) && threadIdx.x == blockDim.x - 1) {
    prefetch_map(&k_map);
    prefetch_map(&v_map);
  }

  // Where this CTA's share begins: the running sum of the requests' units, a lane a request. Up to 32 requests
  // every warp looks at for itself; of more, each warp adds up a stretch, and all then search the one that matters.
  const int warps = threads_of(SRC, M) / 32, span = (A.B + 32 * warps - 1) / (32 * warps);     // a stretch: span * 32 requests
  const auto scan = [&](long long x) {                         // inclusive, over the lanes
#pragma unroll 1
    for (int off = 1; off < 32; off <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, off);
      if (lane >= off) x += y;
    }
    return x;
  };
  int per = 0;
  long long run;                                               // units up to and with this lane's request (or stretch)
  if (A.B <= 32) {
    per = head_units(A, lane);
    run = (long long)per * A.c.kv_heads;
  } else {
    long long sum = 0;
#pragma unroll 1
    for (int c = 0; c < span; ++c) sum += (long long)head_units(A, (warp * span + c) * 32 + lane) * A.c.kv_heads;
    sum = scan(sum);
    if (lane == 31) sh_total[warp] = sum;
    __syncthreads();
    run = lane < warps ? sh_total[lane] : 0;
  }
  run = scan(run);
  const long long total = __shfl_sync(0xffffffffu, run, 31);
  const long long each = total <= 0x7fffffff ? (long long)((unsigned)total / (unsigned)grid) : total / grid;
  const int extra = (int)(total - each * grid);
  const long long from = share(each, extra, cta), to = share(each, extra, cta + 1);
  Walk w;
  w.at = w.end = 0;
  if (from < to) {
    int b0 = 0;
    long long before = 0;
    const auto shift = [&](int x) { return x ? __shfl_sync(0xffffffffu, run, x - 1) : 0; };    // what lies before lane x
    if (A.B > 32) {
      const int x = __ffs(__ballot_sync(0xffffffffu, from < run)) - 1;
      before = shift(x);
      for (b0 = x * span * 32;; b0 += 32) {
        per = head_units(A, b0 + lane);
        run = before + scan((long long)per * A.c.kv_heads);
        const long long last = __shfl_sync(0xffffffffu, run, 31);
        if (from < last) break;
        before = last;
      }
    }
    const int x = __ffs(__ballot_sync(0xffffffffu, from < run)) - 1;               // the first whose units reach past `from`
    w.start(A, from, to, b0 + x, from - (x ? shift(x) : before), __shfl_sync(0xffffffffu, per, x));
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  // A wait that outlasts its limit marks the CTA dead; every role then leaves its loop at its next wait
  // that is not over at once.
  const auto wait = [&](uint64_t* b, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_test_wait(b, parity)) || wait_on(b, parity, &watch);
  };

  if (warp < kSoftWarps) {
    // ---------------------------------------------------------------- softmax: a thread a row
    // Two groups of four warps take the units in turn, so that two units' softmax run side by side. The
    // row's maximum passes from unit to unit through shared memory; each group keeps its own sum.
    const int half = warp >> 2, pair = warp & 3;               // warps w and w + 4 share 32 rows
    const uint32_t tw = tmem + ((uint32_t)(pair * 32) << 16);
    const int r = pair * 32 + lane, tr = PIECES ? lane & 7 : SPREAD ? lane : r;    // lane of tensor memory, row of the tile
    const int col0 = SPREAD ? pair * kCols : 0;
    const float piece_scale = __uint_as_float((127u - 4u * (lane >> 3)) << 23);                  // PIECES: what this lane's pieces are multiplied by
    const float c2 = A.scale * kLog2e;
    uint32_t g0 = 0, swaps = 0, meets = 0;                     // units before this piece; exchanges of the two groups, of all eight warps
    uint8_t* const turn = sm + Lay::off_turn + warp * (32 * kTurnPitch);
    uint8_t* const turn_row = turn + lane * kTurnPitch;                              // this lane's row
    uint8_t* const turn_at = turn + (lane >> 2) * kTurnPitch + (lane & 3) * 16;      // its piece of row lane / 4, then every 8th
    // With the row's thread of the other group. Two buffers in turn: a warp that goes on to the next exchange (the
    // next piece's queries after this one's sums, with no barrier between) must not overwrite what the other has
    // yet to read of this one, and cannot get to the one after that before the other has arrived in the next.
    const auto exchange = [&](float2 mine, float2* other) {
      float2* const at = sh_swap[swaps & 1];
      at[half * kM + r] = mine;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.swap[pair]);
      if (!wait(&bar.swap[pair], swaps++ & 1)) return false;
      *other = at[(half ^ 1) * kM + r];
      return true;
    };
    const auto meet = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.meet);
      return wait(&bar.meet, meets++ & 1);
    };
#pragma unroll 1
    for (; !w.done(); g0 += w.stop() - w.first, w.next(A)) {
      const int stop = w.stop(), first = w.first;
      const int rows = min(M, w.r.n * A.rep - w.tile * M);
      const bool valid = tr < rows;
      const int R = w.tile * M + tr, tok = A.by_rep.of(R), head = w.kh * A.rep + R - tok * A.rep;
      const int lim = valid ? row_limit(A, w.r, tok) : 0;
      const bool warp_live = SPREAD || pair * 32 < rows;
      bool ok = true;
      // Q to tensor memory, a half of the head dim a group
      float rowf = c2;                                         // the softmax's scale, with the row's own over e4m3
      if (warp_live) {
        const long long q_off = valid ? (long long)(w.r.t0 + tok) * A.sq_t + head * A.sq_h + half * (D / 2) : -1;
        constexpr int kChunks = D / 64;                        // 32 elements of this group's half each
        // the warp's rows, all loads in flight, then turned 64 bytes a row at a time: y[c] of this lane's row
        uint4 y[kChunks][4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const long long o = __shfl_sync(0xffffffffu, q_off, x * 8 + (lane >> 2));
          const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(A.q) + (o < 0 ? 0 : o)) + (lane & 3);
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            y[c][x] = make_uint4(0, 0, 0, 0);
            if (o >= 0) y[c][x] = __ldg(src + c * 4);
          }
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
#pragma unroll
          for (int x = 0; x < 4; ++x) *reinterpret_cast<uint4*>(turn_at + x * 8 * kTurnPitch) = y[c][x];
          __syncwarp();
#pragma unroll
          for (int x = 0; x < 4; ++x) y[c][x] = *reinterpret_cast<const uint4*>(turn_row + x * 16);
          __syncwarp();
        }
        if constexpr (!QUANT) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            uint32_t u[16];
#pragma unroll
            for (int x = 0; x < 4; ++x) { u[4 * x] = y[c][x].x; u[4 * x + 1] = y[c][x].y; u[4 * x + 2] = y[c][x].z; u[4 * x + 3] = y[c][x].w; }
            tmem_st16(tw + Lay::q_col + half * (D / 4) + c * 16, u);
          }
        } else {
          // the row's largest magnitude (patterns order like integers; what is not finite is largest)
          constexpr uint32_t kMag = 0x7fff7fffu, kInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
          uint32_t top = 0;
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int x = 0; x < 4; ++x)
              top = __vmaxu2(top, __vmaxu2(__vmaxu2(y[c][x].x & kMag, y[c][x].y & kMag), __vmaxu2(y[c][x].z & kMag, y[c][x].w & kMag)));
          top = max(top & 0xffffu, top >> 16);
          float2 other;
          if (!exchange(make_float2(__uint_as_float(top), 0.f), &other)) break;
          top = max(top, __float_as_uint(other.x));
          // 2^(7 - exponent): the largest element lands in [128, 256)
          const int e2 = min(max((int)(__float_as_uint(unpack16<T>(top).x) >> 23) - 127, -100), 127);
          const float up = __uint_as_float((uint32_t)(127 + 7 - e2) << 23);
          rowf = top >= kInf ? __int_as_float(0x7fc00000) : c2 * __uint_as_float((uint32_t)(127 + e2 - 7) << 23);
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            if constexpr (PIECES) {                            // this lane's piece alone
              uint32_t piece[8];
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const uint2 z = query_piece<T>(y[c][x], up, lane >> 3);
                piece[2 * x] = z.x;
                piece[2 * x + 1] = z.y;
              }
              tmem_st8(tw + Lay::q_col + half * (D / 8) + c * 8, piece);
            } else {
              uint32_t piece[kPieces<T>][8];
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const QPieces<T> z = query_pieces<T>(y[c][x], up);
#pragma unroll
                for (int n = 0; n < kPieces<T>; ++n) {
                  piece[n][2 * x] = z.w[n][0];
                  piece[n][2 * x + 1] = z.w[n][1];
                }
              }
#pragma unroll
              for (int n = 0; n < kPieces<T>; ++n) {
                if (D < 256 || n < 2) tmem_st8(tw + Lay::q_col + n * (D / 4) + half * (D / 8) + c * 8, piece[n]);
                else {
                  // the third piece of D = 256: 128-byte-swizzled rows in shared memory, one slab a group
                  const uint32_t at = base + Lay::off_q3 + half * (kM * 128) + r * 128;
#pragma unroll
                  for (int z = 0; z < 2; ++z)
                    st_shared16(at + (((c * 2 + z) ^ (r & 7)) << 4), piece[n][4 * z], piece[n][4 * z + 1], piece[n][4 * z + 2], piece[n][4 * z + 3]);
                }
              }
            }
          }
          if (WIDEN && D == 256 && kPieces<T> == 3) fence_async_shared();
        }
        tmem_wait_st();
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.q_ready);

      // the next tile's Q (of the same heads and request, the common case), into L2 by the time it is wanted
      if (w.tile + 1 < w.tiles && valid && w.at + w.units + 2 * kPieceCost < w.end) {
        const int next = R + M, nt = A.by_rep.of(next);
        if (nt < w.r.n) {
          const T* p = static_cast<const T*>(A.q) + (long long)(w.r.t0 + nt) * A.sq_t + (w.kh * A.rep + next - nt * A.rep) * A.sq_h + half * (D / 2);
#pragma unroll
          for (int z = 0; z < (D >= 128 ? D / 128 : 1); ++z) asm volatile("prefetch.global.L2 [%0];" :: "l"(p + z * 64));
        }
      }
      float m = -INFINITY, l = 0.f;                            // this group's: l in units of 2^m
#pragma unroll 1
      for (int i = first; i < stop; ++i) {
        const uint32_t g = g0 + (i - first);
        const int s = g & 1;
        if (s != half) continue;
        if (!(ok = wait(&bar.s_done[s], (g >> 1) & 1))) break;
        if (warp_live) {
          tc_fence_after();
          const float4* const sc = reinterpret_cast<const float4*>(sm + Lay::off_scale + (g % kScaleStages) * kScaleBytes);
          const int j0 = i * kKeys;
          const bool masked = __any_sync(0xffffffffu, lim < j0 + col0 + kCols);
          if (QUANT && !(ok = wait(&bar.sc_full[g % kScaleStages], (g / kScaleStages) & 1))) break;
          // the scaled scores of this thread's columns
          float x[kCols];
#pragma unroll
          for (int c = 0; c < kCols; c += 32) {
            if constexpr (SPREAD) tmem_ld16(tw + Lay::s_col + s * kKeys + col0, x);
            else tmem_ld32(tw + Lay::s_col + s * kKeys + c, x + c);
            tmem_wait_ld();
            if constexpr (PIECES) {                            // the products of the query's pieces, added up alike in every lane
#pragma unroll
              for (int e = 0; e < kCols; ++e) x[e] *= piece_scale;
#pragma unroll
              for (int e = 0; e < kCols; ++e) x[e] += __shfl_xor_sync(0xffffffffu, x[e], 8);
#pragma unroll
              for (int e = 0; e < kCols; ++e) x[e] += __shfl_xor_sync(0xffffffffu, x[e], 16);
            }
#pragma unroll
            for (int e = c; e < c + 32 && e < kCols; e += 2) {
              float2 y = mul2(make_float2(x[e], x[e + 1]), make_float2(rowf, rowf));
              if constexpr (QUANT) {
                const float4 f = sc[(col0 + e) / 2];
                y = fma2(y, make_float2(f.x, f.y), make_float2(f.z, f.w));
              }
              x[e] = y.x;
              x[e + 1] = y.y;
            }
          }
          if (masked) {
#pragma unroll
            for (int e = 0; e < kCols; ++e)
              if (j0 + col0 + e >= lim) x[e] = -INFINITY;
          }
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < kCols; e += 2) top[e / 2 & 3] = max3(top[e / 2 & 3], x[e], x[e + 1]);
          const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
          float now = -INFINITY;                               // the maximum the weights so far are relative to
          if (i > first) {
            if (!(ok = wait(&bar.m_set[s ^ 1][pair], ((g - 1) >> 1) & 1))) break;
            now = sh_m[s ^ 1][r];
          }
          const float before = now;
          if (now == -INFINITY || high > now + (kLift + kSlack)) now = high - kLift;
          sh_m[s][r] = now;
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar.m_set[s][pair]);
          // (o is zero, or not begun, while nothing has been seen)
          const float keep = before == -INFINITY ? 1.f : exp2_approx(before - now);
          if (__any_sync(0xffffffffu, keep != 1.f)) {
            if (!(ok = wait(&bar.o_done[s ^ 1], ((g - 1) >> 1) & 1))) break;
            tc_fence_after();
#pragma unroll 1
            for (int d = 0; d < D; d += 16) {
              float o[16];
              uint32_t u[16];
              tmem_ld16(tw + Lay::o_col + d, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(o[e] * keep);
              tmem_st16(tw + Lay::o_col + d, u);
            }
          }
          l *= m == -INFINITY ? 1.f : exp2_approx(m - now);
          m = now;
          const float mm = m == -INFINITY ? 0.f : m;
          const float2 less = make_float2(-mm, -mm);
          float2 sum[2] = {};
#pragma unroll
          for (int c = 0; c < kCols; c += 32) {
            uint32_t p[16];
#pragma unroll
            for (int e = 0; e < 32 && e < kCols; e += 4) {
              float y[4];
#pragma unroll
              for (int z = 0; z < 4; z += 2) {
                const float2 d = add2(make_float2(x[c + e + z], x[c + e + z + 1]), less);
                y[z] = exp2_approx(d.x);
                y[z + 1] = exp2_approx(d.y);
              }
              if constexpr (QUANT) {
                const float4 f = sc[kKeys / 2 + (col0 + c + e) / 4];
                sum[0] = fma2(make_float2(y[0], y[1]), make_float2(f.x, f.y), sum[0]);
                sum[1] = fma2(make_float2(y[2], y[3]), make_float2(f.z, f.w), sum[1]);
              } else {
                sum[0] = add2(make_float2(y[0], y[1]), sum[0]);
                sum[1] = add2(make_float2(y[2], y[3]), sum[1]);
              }
              if constexpr (PIECES) {
                p[e / 4] = piece_of(y, lane >> 3);
              } else {
                p[e / 2] = pack16<T>(y[0], y[1]);
                p[e / 2 + 1] = pack16<T>(y[2], y[3]);
              }
            }
            if constexpr (PIECES) {                            // (as below, a code a column)
              const uint32_t none[4] = {};
              const uint32_t at = tw + Lay::s_col + s * kKeys;
              tmem_st4(at + 4 * pair, p);
              tmem_st4(at + 4 * (pair ^ 1), none);
              tmem_st4(at + 4 * (pair ^ 2), none);
              tmem_st4(at + 4 * (pair ^ 3), none);
            } else if constexpr (SPREAD) {                            // the other lanes' columns have no weight here
              const uint32_t none[8] = {};
              const uint32_t at = tw + Lay::s_col + s * kKeys;
              tmem_st8(at + 8 * pair, p);
              tmem_st8(at + 8 * (pair ^ 1), none);
              tmem_st8(at + 8 * (pair ^ 2), none);
              tmem_st8(at + 8 * (pair ^ 3), none);
            } else {
              tmem_st16(tw + Lay::s_col + s * kKeys + c / 2, p);
            }
          }
          l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
          tmem_wait_st();
          tc_fence_before();
        } else {
          if (lane == 0) mbar_arrive(&bar.m_set[s][pair]);
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bar.p_full[s]);
          if (QUANT) mbar_arrive(&bar.sc_empty[g % kScaleStages]);
        }
      }
      if (!ok) break;
      // the last product of the piece
      const uint32_t gl = g0 + (stop - first) - 1;
      if (!wait(&bar.o_done[gl & 1], (gl >> 1) & 1)) break;
      tc_fence_after();
      if (warp_live) {
        const bool whole = first == 0 && stop == w.units;
        // the groups' sums (SPREAD: of all the row's lanes) relative to the latest maximum, which this lane's
        // O then meets by `mine`
        float mine = 1.f;
        if constexpr (SPREAD) {
          sh_swap[0][half * kM + r] = make_float2(m, l);
          if (!meet()) break;
          float lane_m = -INFINITY, top = -INFINITY;
#pragma unroll
          for (int z = 0; z < kSoftWarps; ++z) top = fmaxf(top, sh_swap[0][z * 32 + lane].x);
          lane_m = fmaxf(m, sh_swap[0][(half ^ 1) * kM + r].x);
          l = 0.f;
#pragma unroll
          for (int z = 0; z < kSoftWarps; ++z) {
            const float2 y = sh_swap[0][z * 32 + lane];
            l += y.x == -INFINITY ? y.y : y.y * exp2_approx(y.x - top);
          }
          mine = lane_m == -INFINITY ? 1.f : exp2_approx(lane_m - top);
          if (PIECES) mine *= piece_scale;
          m = top;
        } else {
          float2 other;
          if (!exchange(make_float2(m, l), &other)) break;
          const float top = fmaxf(m, other.x);
          const auto to_top = [&](float mm, float ll) { return mm == top || mm == -INFINITY ? ll : ll * exp2_approx(mm - top); };
          l = to_top(m, l) + to_top(other.x, other.y);
          m = top;
        }
        if (w.r.over) l = __int_as_float(0x7fc00000);
        const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
        float* const part = part_row<D>(A.part, grid, cta, first == 0, tr);
        const long long o_off = (long long)(w.r.t0 + tok) * A.so_t + head * A.so_h;
        float bad[4] = {0.f, 0.f, 0.f, 0.f};                   // turn NaN where an element is not finite
        const auto put = [&](float4 y, float row_inv, float row_l, long long off, int row, int d) {      // four columns of a row
          if (whole)
            *reinterpret_cast<uint2*>(static_cast<T*>(A.o) + off + d) =
                row_l == 0.f ? make_uint2(0, 0) : make_uint2(pack16<T>(y.x * row_inv, y.y * row_inv), pack16<T>(y.z * row_inv, y.w * row_inv));
          else
            *reinterpret_cast<float4*>(part_row<D>(A.part, grid, cta, first == 0, row) + d) = y;
        };
        if constexpr (SPREAD) {
          // The row's four lanes are added up through the warps' buffers, 64 columns at a time (16 where there are
          // more than 8 rows): warp `pair` then takes a quarter of the rows, four columns a lane.
          const int per_row = rows <= 8 ? 16 : 4, pitch = per_row * 16 + 16;                // 16-byte pieces; bytes
          const int row = (pair * 32 + lane) / per_row, piece = lane % per_row;
          const long long off = __shfl_sync(0xffffffffu, o_off, row);
          const float row_inv = __shfl_sync(0xffffffffu, inv, row), row_l = __shfl_sync(0xffffffffu, l, row);
          uint8_t* const mine4 = turn + lane * pitch;
          const uint8_t* const from4 = turn - pair * (32 * kTurnPitch) + row * pitch + piece * 16;
#pragma unroll 1
          for (int d = half * (D / 2); d < (half + 1) * (D / 2); d += 4 * per_row) {
#pragma unroll 1
            for (int x = 0; x < 4 * per_row && d + x < (half + 1) * (D / 2); x += 16) {
              float o[16];
              tmem_ld16(tw + Lay::o_col + d + x, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] *= mine;
              if constexpr (PIECES) {                          // the products of the weights' pieces
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] += __shfl_xor_sync(0xffffffffu, o[e], 8);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] += __shfl_xor_sync(0xffffffffu, o[e], 16);
              }
              if (lane < rows) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  *reinterpret_cast<float4*>(mine4 + x * 4 + e * 16) = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
              }
            }
            if (!(ok = meet())) break;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row < rows && d + piece * 4 < (half + 1) * (D / 2)) {
#pragma unroll
              for (int z = 0; z < 4; ++z) {
                const float4 v = *reinterpret_cast<const float4*>(from4 + z * (32 * kTurnPitch));
                y.x += v.x; y.y += v.y; y.z += v.z; y.w += v.w;
              }
              bad[0] = fmaf(y.x, 0.f, fmaf(y.y, 0.f, fmaf(y.z, 0.f, fmaf(y.w, 0.f, bad[0]))));
              put(y, row_inv, row_l, off, row, d + piece * 4);
            }
            if (!(ok = meet())) break;
          }
          if (!ok) break;
        } else {
#pragma unroll 1
          for (int d = half * (D / 2); d < (half + 1) * (D / 2); d += 16) {
            float o[16];
            tmem_ld16(tw + Lay::o_col + d, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              bad[e] = fmaf(o[4 * e], 0.f, fmaf(o[4 * e + 1], 0.f, fmaf(o[4 * e + 2], 0.f, fmaf(o[4 * e + 3], 0.f, bad[e]))));
              *reinterpret_cast<float4*>(turn_row + e * 16) = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            }
            __syncwarp();
#pragma unroll 1
            for (int x = 0; x < 4; ++x) {
              const int row = x * 8 + (lane >> 2);
              const long long off = __shfl_sync(0xffffffffu, o_off, row);
              const float row_inv = __shfl_sync(0xffffffffu, inv, row), row_l = __shfl_sync(0xffffffffu, l, row);
              if (pair * 32 + row < rows)
                put(*reinterpret_cast<const float4*>(turn_at + x * 8 * kTurnPitch), row_inv, row_l, off, pair * 32 + row, d + (lane & 3) * 4);
            }
            __syncwarp();
          }
        }
        if (valid && half == 0 && (!SPREAD || r < M)) {
          if (!whole) {
            part[D] = m;
            part[D + 1] = l;
          } else if (A.lse) {
            A.lse[(long long)head * A.T + w.r.t0 + tok] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
          }
        }
        // A value that is not finite at a position that this row may not see has met a weight of 0 in
        // the product. Only a causal row's last units can hold one: where they do, such a row is taken again from
        // its own positions alone, with m and l as they are.
        // (SPREAD: a position's weight is 0 in three of a row's lanes, so any such value does this.)
        const float worst = (bad[0] + bad[1]) + (bad[2] + bad[3]);
        unsigned again = __ballot_sync(0xffffffffu, worst != 0.f);
        const unsigned take = __ballot_sync(0xffffffffu, valid && l == l && (SPREAD || (A.causal && lim < stop * kKeys)));
        if constexpr (SPREAD) {                              // from the lanes that added a row up to the row's own
          const int per_row = rows <= 8 ? 16 : 4, base_row = pair * 32 / per_row;
          again = __ballot_sync(0xffffffffu, lane >= base_row && lane < base_row + 32 / per_row &&
                                                 (again >> ((lane - base_row) * per_row & 31) & ((1u << per_row) - 1)) != 0);
        }
        if (again & take) mend_rows<T, D, QUANT>(A, w, again & take, m, inv, &watch);
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.o_free);
      if (threadIdx.x == 0 && first == 0 && stop < w.units) {  // begins here, ends elsewhere
        const long long end = w.at + kPieceCost + w.units;
        Desc d;
        d.last = cta + 1;
#pragma unroll 1
        while (share(each, extra, d.last + 1) < end) ++d.last;
        d.kh = w.kh; d.t0 = w.r.t0; d.rows = rows; d.row0 = w.tile * M; d.err = 0; d.each = each; d.extra = extra;
        A.desc[cta] = d;
      }
    }
  } else if (warp == kMmaWarp) {
    // ---------------------------------------------------------------- tensor work
    // operand formats: 16-bit types, or e4m3 (0) for the scores; the second product's B is MN-major
    constexpr uint32_t idesc_s = tc_idesc(kM, kKeys) | (QUANT ? 0u : type_bits<T>()), idesc_o = tc_idesc(kM, D) | (PIECES ? 0u : type_bits<T>()) | (1u << 16);
    constexpr int kRowB = Lay::kRowB;
    uint32_t g = 0, pieces = 0;
    bool ok = true;
    const auto pv = [&](uint32_t u, int i, bool fresh) {       // O (+)= P(u) V(u), u the piece's unit i
      const int s = u & 1, st = WIDEN ? s : u % kSt;
      uint64_t* const full = WIDEN ? &bar.w_full[s] : &bar.v_full[st];
      if (!wait(full, (WIDEN ? u >> 1 : u / kSt) & 1)) return false;
      const uint32_t v = WIDEN ? base + Lay::off_w + s * Lay::kWide : base + Lay::off_v + st * Lay::kTile;
      if constexpr (is_tma(SRC) && !WIDEN) {
        // rows past the end hold what the pages or the last tile left there: 0 x NaN must not happen
        const int rows = row_limit(A, w.r, w.r.n - 1) - i * kKeys;
        if (rows < kKeys) {
          constexpr int kRowP = kRowB / 16;                    // 16-byte pieces of a slab's row
#pragma unroll 1
          for (int x = max(rows, 0) * kRowP + lane; x < kKeys * kRowP; x += 32)
#pragma unroll
            for (int c = 0; c < Lay::kSlabs; ++c) st_shared16(v + c * A.slab + x / (8 * kRowP) * A.group + x % (8 * kRowP) * 16, 0, 0, 0, 0);
          fence_async_shared();
          __syncwarp();
        }
      }
      if (!wait(&bar.p_full[s], (u >> 1) & 1)) return false;
      if constexpr (!is_tma(SRC) && !WIDEN) fence_async_shared();                          // the tile was stored by threads
      tc_fence_after();
      if constexpr (PIECES) {                                  // two steps of 32 positions
        mma_ts_warp<2, true>(tmem + Lay::o_col, tmem + Lay::s_col + s * kKeys, mn_major<kRowB>(v, A.slab, A.group), A.group >> 2, idesc_o, !fresh);
      } else {                                                 // four steps of 16
        const uint32_t slab = WIDEN ? kKeys * 128u : A.slab, group = WIDEN ? 1024u : A.group;
        mma_ts_warp<4, false>(tmem + Lay::o_col, tmem + Lay::s_col + s * kKeys, mn_major<128>(v, slab, group), group >> 3, idesc_o, !fresh);
      }
      tc_commit_warp(WIDEN ? &bar.w_empty[s] : &bar.v_empty[st]);
      tc_commit_warp(&bar.o_done[s]);
      return true;
    };
#pragma unroll 1
    for (; ok && !w.done(); w.next(A), ++pieces) {
      const int count = w.stop() - w.first;
#pragma unroll 1
      for (int i = 0; i <= count; ++i) {                       // S(i), then O(i - 1)
        if (i < count) {
          const uint32_t u = g + i;
          const int s = u & 1, st = u % kSt;
          if (i == 0 && !(ok = wait(&bar.q_ready, pieces & 1))) break;
          if (!(ok = wait(&bar.k_full[st], (u / kSt) & 1))) break;
          if constexpr (!is_tma(SRC)) fence_async_shared();
          tc_fence_after();
          const uint32_t k_at = base + Lay::off_k + st * Lay::kTile;
#pragma unroll (QUANT ? 1 : 4)
          for (int n = 0; n < (WIDEN ? kPieces<T> : 1); ++n)
#pragma unroll (QUANT ? 1 : 4)
            for (int k = 0; k < Lay::kSlabs; ++k) {
              const uint64_t desc = k_major<kRowB>(k_at + k * A.slab, A.group);
              if (WIDEN && D == 256 && n == 2)
                mma_ss4_f8_warp(tmem + Lay::s_col + s * kKeys, k_major<128>(base + Lay::off_q3 + k * (kM * 128), 1024), desc, idesc_s);
              else
                mma_ts_warp<kRowB / 32, QUANT>(tmem + Lay::s_col + s * kKeys, tmem + Lay::q_col + n * (D / 4) + k * 32, desc, 2, idesc_s, n + k > 0);
            }
          tc_commit_warp(&bar.s_done[s]);
          tc_commit_warp(&bar.k_empty[st]);
        }
        if (i > 0) {
          // the piece's first product overwrites O: the last piece's must have been read
          if (i == 1 && pieces > 0 && !(ok = wait(&bar.o_free, (pieces - 1) & 1))) break;
          if (!(ok = pv(g + i - 1, w.first + i - 1, i == 1))) break;
        }
      }
      g += count;
    }
    tc_commit_warp(&bar.drain);                                // everything issued has completed
    mbar_wait(&bar.drain, 0);
  } else {
    // ---------------------------------------------------------------- loads
    const int lw = warp - kMmaWarp - 1;
    uint32_t g = 0;                                            // units so far
    bool ok = true;
    const auto k_free = [&] { return g < kSt || wait(&bar.k_empty[g % kSt], (g / kSt - 1) & 1); };
    const auto v_free = [&](uint32_t u) { return u < kSt || wait(&bar.v_empty[u % kSt], (u / kSt - 1) & 1); };
    if (QUANT && lw >= load_warps(SRC)) {
      // -------- V's codes to 16 bits, and (the first two warps, a lane a position) the scales, looked up a unit
      // early
      const int cw = lw - load_warps(SRC), ct = cw * 32 + lane;
      float2 sc = make_float2(0.f, 1.f);
      const auto look = [&](const Walk& w, int i) {
        sc = make_float2(0.f, 1.f);
        const int j = i * kKeys + ct;
        if (ct < kKeys && j < row_limit(A, w.r, w.r.n - 1)) {
          long long so = 0;
          if (row_offset(A, w.b, w.kh, j, &so) >= 0) sc = make_float2(__ldg(A.c.k_scale + so), __ldg(A.c.v_scale + so));
          else sc.x = __int_as_float(0x7fc00000);              // no such page: its scores are NaN
        }
      };
      constexpr int kRowP = D / 16, kPasses = kKeys * kRowP / 128, kBatch = kPasses < 4 ? kPasses : 4;    // 16-code pieces of a row; of a lane; in flight
      if (!w.done()) look(w, w.first);
#pragma unroll 1
      while (ok && !w.done()) {
        const int stop = w.stop(), lim = row_limit(A, w.r, w.r.n - 1);
#pragma unroll 1
        for (int i = w.first; i < stop; ++i, ++g) {
          const uint32_t ss = g % kScaleStages, st = g % kSt, ws = g & 1;
          if (cw < kKeys / 32) {
            if (g >= kScaleStages && !(ok = wait(&bar.sc_empty[ss], (g / kScaleStages - 1) & 1))) break;
            // a scale of NaN reaches the row through its score; where the row may not see the position, its
            // weight of 0 meets a finite factor
            uint8_t* const at = sm + Lay::off_scale + ss * kScaleBytes;
            float* const two = reinterpret_cast<float*>(at) + (ct >> 1) * 4 + (ct & 1);            // k's of two positions, then log2 v's
            two[0] = sc.x;
            const float vs = value_scale(sc.y);
            two[2] = log2f(vs);
            reinterpret_cast<float*>(at + kKeys * 8)[ct] = vs > 0.f ? 1.f / vs : 1.f;
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.sc_full[ss]);
            if (i + 1 < stop) look(w, i + 1);
          }
          if constexpr (WIDEN) {
            if (!(ok = wait(&bar.v_full[st], (g / kSt) & 1))) break;
            const uint8_t* const raw = sm + Lay::off_v + st * Lay::kTile;
#pragma unroll 1
            for (int x0 = 0; x0 < kPasses; x0 += kBatch) {
              uint4 y[kBatch];
              uint32_t nan = 0;
#pragma unroll
              for (int x = 0; x < kBatch; ++x) {
                const int z = (x0 + x) * 128 + ct, r = z / kRowP, p = z % kRowP;
                constexpr int kSlabP = Lay::kRowB / 16;
                const int swz = Lay::kRowB == 128 ? (p % kSlabP) ^ (r & 7) : (p % kSlabP) ^ (r >> 1 & 3);
                y[x] = *reinterpret_cast<const uint4*>(raw + p / kSlabP * A.slab + (r >> 3) * A.group + (r & 7) * Lay::kRowB + swz * 16);
                if (i * kKeys + r >= lim) y[x] = make_uint4(0, 0, 0, 0);     // past the end: whatever the page holds
                nan |= any_nan(y[x].x) | any_nan(y[x].y) | any_nan(y[x].z) | any_nan(y[x].w);
              }
              if (x0 + kBatch >= kPasses) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar.v_empty[st]);
              }
              if (x0 == 0 && g >= 2 && !(ok = wait(&bar.w_empty[ws], ((g >> 1) + 1) & 1))) break;
#pragma unroll
              for (int x = 0; x < kBatch; ++x) {
                const int z = (x0 + x) * 128 + ct, r = z / kRowP, p = z % kRowP;
                uint4 a, b;
                if (nan == 0) {
                  a = widen8<T>(y[x].x, y[x].y);
                  b = widen8<T>(y[x].z, y[x].w);
                } else {
                  a = widen8_nan<T>(y[x].x, y[x].y);
                  b = widen8_nan<T>(y[x].z, y[x].w);
                }
                const uint32_t row = base + Lay::off_w + ws * Lay::kWide + (p >> 2) * (kKeys * 128) + r * 128;
                const int c0 = (p & 3) * 2, odd = p >> 2 & 1;    // (lanes of odd slabs store their halves in the other order: no two on a bank)
                const uint4 u = odd ? b : a, v = odd ? a : b;
                st_shared16(row + (((c0 + odd) ^ (r & 7)) << 4), u.x, u.y, u.z, u.w);
                st_shared16(row + (((c0 + 1 - odd) ^ (r & 7)) << 4), v.x, v.y, v.z, v.w);
              }
            }
            if (!ok) break;
            fence_async_shared();
            mbar_arrive(&bar.w_full[ws]);
          }
        }
        if (!ok) break;
        w.next(A);
        if (!w.done()) look(w, w.first);
      }
    } else if constexpr (is_tma(SRC)) {
      // -------- the warps that issue TMA copies: a lane a box, whose page it looks up
      const int box = A.box;
      const uint32_t bytes = box * D * Lay::kElem;
      int page = -1, off = 0;
      bool need = false;
      uint32_t sent_k = 0, sent_v = 0;                         // units whose copies this warp has issued
      const auto look = [&](const Walk& w, int i) {
        const int j = i * kKeys + lane * box;
        need = lane * box < kKeys && j < row_limit(A, w.r, w.r.n - 1);
        page = -1;
        if (need) {
          const int p = A.by_page.of(j);
          off = j - p * A.c.page_size;
          page = __ldg(A.table + (long long)w.b * A.st + p);
          if (page >= A.c.pages) page = -1;
        }
      };
      if (!w.done()) look(w, w.first);
#pragma unroll 1
      while (ok && !w.done()) {
        const int stop = w.stop();
#pragma unroll 1
        for (int i = w.first; i < stop; ++i, ++g) {
          const unsigned all = __ballot_sync(0xffffffffu, need && page >= 0);
#pragma unroll
          for (int z = 0; z < 2 / load_warps(SRC); ++z) {
            const int kv = load_warps(SRC) == 2 ? lw : z;
            if (!(ok = kv ? v_free(g) : k_free())) break;
            const uint32_t dst = base + (kv ? Lay::off_v : Lay::off_k) + (g % kSt) * Lay::kTile + lane * bytes;
            uint64_t* const full = kv ? &bar.v_full[g % kSt] : &bar.k_full[g % kSt];
            if (need && page < 0) {                            // no such page: its scores are NaN (over e4m3 by its scales)
              const uint32_t fill = !QUANT && kv == 0 ? 0x7fff7fffu : 0u;
#pragma unroll 1
              for (uint32_t x = 0; x < bytes; x += 16) st_shared16(dst + x, fill, fill, fill, fill);
              fence_async_shared();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive_expect_tx(full, __popc(all) * bytes);
            __syncwarp();
            if (need && page >= 0) tma_load_5d(dst, kv ? &v_map : &k_map, 0, off, 0, w.kh, page, full);
            (kv ? sent_v : sent_k) = g + 1;
          }
          if (!ok) break;
          if (i + 1 < stop) look(w, i + 1);
        }
        if (!ok) break;
        w.next(A);
        if (!w.done()) look(w, w.first);
      }
      // A CTA whose products gave up does not wait for these copies: it must not end before they have landed.
      const auto landed = [&](uint64_t* full, uint32_t sent) {
#pragma unroll 1
        for (uint32_t u = sent < kSt ? 0 : sent - kSt; u < sent; ++u) mbar_wait(&full[u % kSt], (u / kSt) & 1);
      };
      landed(bar.k_full, sent_k);
      landed(bar.v_full, sent_v);
    } else {
      // -------- the warps that copy rows. A thread's copies arrive on the stage's barrier by themselves when
      // they land. Stages come free in the order K(g + 1), V(g) (the products are issued S(g - 1),
      // O(g - 2)): they are filled so.
      constexpr int kLanesRow = D * Lay::kElem / 16;           // lanes a row of 16-byte pieces
      constexpr int kRowsPass = 32 / kLanesRow;                // rows a warp's access covers
      constexpr int kPasses = kKeys / (kLoadWarps * kRowsPass);
      constexpr int kOwn = kPasses * kRowsPass;                // positions a warp handles of a unit
      constexpr int kRowP = Lay::kRowB / 16;                   // pieces of a slab's row
      static_assert(kPasses >= 1 && kOwn <= 32, "a lane a position, a pass for every warp");
      const int sub = lane / kLanesRow, piece = lane % kLanesRow;
      const auto position = [&](int x) { return (x / kRowsPass) * (kLoadWarps * kRowsPass) + lw * kRowsPass + x % kRowsPass; };
      const auto find = [&](const Walk& w, int i) {            // the row of this lane's position; -1 no such page, -2 past the end
        const int j = i * kKeys + position(lane % kOwn);
        return j < row_limit(A, w.r, w.r.n - 1) ? row_offset(A, w.b, w.kh, j, nullptr) : -2ll;
      };
      const auto fill = [&](const void* pool, uint32_t tile, long long off, uint64_t* full, bool key) {
        const uint32_t dst = base + tile + piece / kRowP * A.slab;
        const uint8_t* src = static_cast<const uint8_t*>(pool);
#pragma unroll
        for (int x = 0; x < kPasses; ++x) {
          const int r = position(x * kRowsPass + sub);
          const long long o = __shfl_sync(0xffffffffu, off, x * kRowsPass + sub);
          const bool nan_row = !QUANT && key && o == -1;
          const int swz = Lay::kRowB == 128 ? (piece % kRowP) ^ (r & 7) : (piece % kRowP) ^ (r >> 1 & 3);
          cp_async16(dst + (r >> 3) * A.group + (r & 7) * Lay::kRowB + (swz << 4),
                     o >= 0 ? static_cast<const void*>(src + o * Lay::kElem + piece * 16) : static_cast<const void*>(kNanRow),
                     o >= 0 || nan_row ? 16 : 0);
        }
        cp_async_arrive(full);
      };
      long long off = w.done() ? -2 : find(w, w.first), v_off = -2;
      const auto fill_v = [&](uint32_t u) {
        if (!v_free(u)) return false;
        fill(A.c.v, Lay::off_v + (u % kSt) * Lay::kTile, v_off, &bar.v_full[u % kSt], false);
        return true;
      };
#pragma unroll 1
      while (ok && !w.done()) {
        const int stop = w.stop();
#pragma unroll 1
        for (int i = w.first; i < stop; ++i, ++g) {
          if (!(ok = k_free())) break;
          fill(A.c.k, Lay::off_k + (g % kSt) * Lay::kTile, off, &bar.k_full[g % kSt], true);
          if (g > 0 && !(ok = fill_v(g - 1))) break;
          v_off = off;
          if (i + 1 < stop) off = find(w, i + 1);
        }
        if (!ok) break;
        w.next(A);
        if (!w.done()) off = find(w, w.first);
      }
      if (ok && g > 0) fill_v(g - 1);
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && watch.dead) A.desc[cta].err = DEV_TIMEOUT_FULL;
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, Lay::cols);
  }
}

// ---- the pieces that were cut --------------------------------------------------------------------
// o = sum_i 2^(m_i - m) o_i / l,  l = sum_i 2^(m_i - m) l_i,  m = max m_i over the parts in unit order.
// CTA x takes the piece that begins in share x, WARPS warps a row: 8 where a piece has many parts (few
// pieces, as in a step of a few decodes), else 1. A warp takes every WARPS-th part, kBatch of them at a
// time with all their loads in flight together: the kernel is a chain of memory latencies, so it is
// made short.
constexpr int kJoinWarps = 8;

template <typename T, int D, int WARPS>
__global__ void __launch_bounds__(kJoinWarps * 32) attn_join_kernel(const AttnArgs A) {
  asm volatile("griddepcontrol.wait;" ::: "memory");           // launched before the parts are complete
  const int grid = gridDim.x, cta = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Desc d = A.desc[cta];
  const int r = blockIdx.y * (kJoinWarps / WARPS) + warp / WARPS;
  if (d.last < 0 || r >= d.rows) return;                       // (WARPS == 8: the whole CTA alike)
  // the parts: this CTA's second one, then the first one of every later CTA that has a share
  const int last = d.each > 0 ? d.last : min(d.last, d.extra - 1);
  constexpr int E = D / 32, V = E < 4 ? E : 4;                 // elements a lane; of one access
  constexpr int kBatch = WARPS > 1 ? 8 : 2;                    // parts in flight (rarely more than two or three where a warp has a row)
  float acc[E], l = 0.f, m = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  const int first = cta + (WARPS > 1 ? warp : 0);
#pragma unroll 1
  for (int c0 = first; c0 <= last; c0 += kBatch * WARPS) {
    float x[kBatch][E], pm[kBatch], pl[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int c = c0 + i * WARPS;
      pm[i] = -INFINITY;
      pl[i] = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) x[i][e] = 0.f;
      if (c <= last) {
        const float* p = part_row<D>(A.part, grid, c, c == cta, r);
        pm[i] = p[D];
        pl[i] = p[D + 1];
#pragma unroll
        for (int e = 0; e < E; e += V) {
          if constexpr (V == 4) {
            const float4 y = *reinterpret_cast<const float4*>(p + lane * V + e * 32);
            x[i][e] = y.x; x[i][e + 1] = y.y; x[i][e + 2] = y.z; x[i][e + 3] = y.w;
          } else {
            const float2 y = *reinterpret_cast<const float2*>(p + lane * V + e * 32);
            x[i][e] = y.x; x[i][e + 1] = y.y;
          }
        }
      }
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) top = fmaxf(top, pm[i]);
    const float mm = top == -INFINITY ? 0.f : top, keep = exp2_approx(m - mm);
    l *= keep;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= keep;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float w = exp2_approx(pm[i] - mm);
      // a part with nothing in it has m = -inf, and l = 0 or (scores of NaN only) NaN
      l += pm[i] == -INFINITY ? pl[i] : w * pl[i];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(w, x[i][e], acc[e]);
    }
    m = top;
  }
  if constexpr (WARPS > 1) {
    __shared__ float sh_acc[WARPS][D], sh_m[WARPS], sh_l[WARPS];
#pragma unroll
    for (int e = 0; e < E; e += V)
#pragma unroll
      for (int z = 0; z < V; ++z) sh_acc[warp][lane * V + e * 32 + z] = acc[e + z];
    if (lane == 0) { sh_m[warp] = m; sh_l[warp] = l; }
    __syncthreads();
    if (warp > 0) return;
    float top = sh_m[0];
#pragma unroll
    for (int i = 1; i < WARPS; ++i) top = fmaxf(top, sh_m[i]);
    const float mm = top == -INFINITY ? 0.f : top;
    l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      const float w = exp2_approx(sh_m[i] - mm);
      l += sh_m[i] == -INFINITY ? sh_l[i] : w * sh_l[i];
#pragma unroll
      for (int e = 0; e < E; e += V)
#pragma unroll
        for (int z = 0; z < V; ++z) acc[e + z] = fmaf(w, sh_acc[i][lane * V + e * 32 + z], acc[e + z]);
    }
    m = top;
  }
  const int R = d.row0 + r, tok = A.by_rep.of(R), head = d.kh * A.rep + R - tok * A.rep;
  T* out = static_cast<T*>(A.o) + (long long)(d.t0 + tok) * A.so_t + head * A.so_h;
  const float inv = 1.f / l;
#pragma unroll
  for (int e = 0; e < E; e += V)
#pragma unroll
    for (int z = 0; z < V; z += 2)
      *reinterpret_cast<uint32_t*>(out + e * 32 + lane * V + z) = l == 0.f ? 0u : pack16<T>(acc[e + z] * inv, acc[e + z + 1] * inv);
  if (A.lse && lane == 0) A.lse[(long long)head * A.T + d.t0 + tok] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

Divisor divisor(int d) {
  int k = 31;
  while ((1ll << (k - 31)) < d) ++k;
  return {(uint32_t)(((1ull << k) + d - 1) / d), k};
}

// CTAs of a launch (without a device, as in a size computed on the host alone: a B200's)
int sm_count() {
  const int n = device_sms();
  return n > 0 ? n : 148;
}
size_t desc_bytes(int grid) { return ((size_t)grid * sizeof(Desc) + 255) / 256 * 256; }

// The pool as [page][kv head][slot][dim], read in boxes of `rows` slots and all their columns, as slabs of 128
// bytes (64 where a row has no more). False where a tensor map cannot describe it (rows are then copied
// one by one).
bool pool_map(CUtensorMap* map, const cfb_kv_cache& c, void* base, int rows) {
  const bool codes = c.dtype == DT_E4M3;
  const cuuint64_t size = codes ? 1 : 2, row = c.dim * size < 128 ? 64 : 128, slabs = c.dim * size / row;
  const cuuint64_t dims[5] = {row / size, (cuuint64_t)c.page_size, slabs, (cuuint64_t)c.kv_heads, (cuuint64_t)c.pages};
  const cuuint64_t strides[4] = {(cuuint64_t)c.slot_stride * size, row, (cuuint64_t)c.head_stride * size, (cuuint64_t)c.page_stride * size};
  const cuuint32_t box[5] = {(cuuint32_t)(row / size), (cuuint32_t)rows, (cuuint32_t)slabs, 1, 1}, step[5] = {1, 1, 1, 1, 1};
  const auto encode = tensor_map_encoder();
  return encode && encode(map, codes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 5, base, dims, strides, box,
                          step, CU_TENSOR_MAP_INTERLEAVE_NONE, row == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, int SRC, int M>
cfb_status launch(const AttnArgs& A, const CUtensorMap* maps, int grid, cudaStream_t st) {
  if (allow_smem<attn_kernel<T, D, SRC, M>>((int)Layout<D, SRC, M>::bytes) != cudaSuccess)
    return cfb_launch_status("attn_kernel attribute");
  attn_kernel<T, D, SRC, M><<<grid, threads_of(SRC, M), Layout<D, SRC, M>::bytes, st>>>(A, maps[0], maps[1]);
  if (const cfb_status s = cfb_launch_status("attn_kernel")) return s;
  const long long rows = std::min((long long)M, (long long)A.T * A.rep);
  // pieces: at least a row tile a kv head and request that has tokens; parts of one: the CTAs over those
  const long long pieces = (long long)A.c.kv_heads * std::max((long long)std::min(A.B, A.T), ((long long)A.T * A.rep + M - 1) / M);
  const bool many = grid > 8 * pieces;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, (unsigned)(many ? rows : (rows + kJoinWarps - 1) / kJoinWarps));
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, many ? attn_join_kernel<T, D, kJoinWarps> : attn_join_kernel<T, D, 1>, A);
  return cfb_launch_status("attn_join_kernel");
}
template <typename T, int D, int SRC>
cfb_status launch_rows(const AttnArgs& A, const CUtensorMap* maps, int grid, cudaStream_t st) {
  return A.m == kM ? launch<T, D, SRC, kM>(A, maps, grid, st) : launch<T, D, SRC, few_rows(is_e4m3(SRC))>(A, maps, grid, st);
}
template <typename T, int D>
cfb_status launch_source(const AttnArgs& A, int src, const CUtensorMap* maps, int grid, cudaStream_t st) {
  switch (src) {
    case TMA16: return launch_rows<T, D, TMA16>(A, maps, grid, st);
    case ROWS16: return launch_rows<T, D, ROWS16>(A, maps, grid, st);
    case TMA8: return launch_rows<T, D, TMA8>(A, maps, grid, st);
    default: return launch_rows<T, D, ROWS8>(A, maps, grid, st);
  }
}
template <typename T>
cfb_status launch_dim(const AttnArgs& A, int src, const CUtensorMap* maps, int grid, cudaStream_t st) {
  if (A.c.dim == 64) return launch_source<T, 64>(A, src, maps, grid, st);
  if (A.c.dim == 128) return launch_source<T, 128>(A, src, maps, grid, st);
  return launch_source<T, 256>(A, src, maps, grid, st);
}

}  // namespace

extern "C" size_t cfb_paged_attn_workspace(int H, int kv_heads, int dim) {
  if (H <= 0 || kv_heads <= 0 || dim <= 0) return 0;
  const int grid = sm_count();
  return desc_bytes(grid) + (size_t)grid * 2 * kM * (dim + 4) * sizeof(float);
}

extern "C" cfb_status cfb_paged_attn_error(const void* ws, int* device_error) {
  if (!ws || !device_error) return CFB_ERR_INVALID_ARG;
  *device_error = 0;
  const int grid = sm_count();
  Desc* d = static_cast<Desc*>(malloc(grid * sizeof(Desc)));
  if (!d) return CFB_ERR_CUDA;
  const cudaError_t e = cudaMemcpy(d, ws, grid * sizeof(Desc), cudaMemcpyDeviceToHost);
  for (int i = 0; e == cudaSuccess && i < grid; ++i)
    if (d[i].err) *device_error = d[i].err;
  free(d);
  return e == cudaSuccess ? CFB_OK : cfb_launch_status("cfb_paged_attn_error");
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
  if ((long long)T * (H / c->kv_heads) > 0x7fffffffll - kM || (long long)table_width * c->page_size > 0x7fffffffll - kKeys)
    return CFB_ERR_UNSUPPORTED;
  // (a request's units are counted in 32 bits)
  const int rep = H / c->kv_heads, few = few_rows(c->dtype == DT_E4M3), m = (long long)T * rep <= (long long)few * B ? few : kM;
  if (((long long)T * rep / m + 1) * ((long long)table_width * c->page_size / kKeys + 1 + kPieceCost) > 0x7fffffffll)
    return CFB_ERR_UNSUPPORTED;
  if (T == 0 || B == 0) return CFB_OK;
  if (!q || !o || !kv_len || !cu_q || (table_width && !page_table) || !ws) return CFB_ERR_INVALID_ARG;
  if (!rows_aligned(q, 2, sq_t, sq_h) || !rows_aligned(o, 2, so_t, so_h)) return CFB_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(ws) & 255) || ws_bytes < cfb_paged_attn_workspace(H, c->kv_heads, c->dim))
    return CFB_ERR_WORKSPACE;
  const int grid = sm_count();
  // Boxes: a whole unit where pages hold whole units, else of 8 rows (the tile is then [group][slab]).
  const int fit = std::gcd(c->page_size, kKeys), box = fit < kKeys ? std::min(fit, 8) : fit;
  const uint32_t row = c->dim * (c->dtype == DT_E4M3 ? 1 : 2) < 128 ? 64 : 128, slabs = c->dim * (c->dtype == DT_E4M3 ? 1 : 2) / row;
  const bool grouped = box == 8;
  const AttnArgs A{q, sq_t, sq_h, *c, page_table, table_stride, table_width, kv_len, cu_q, o, so_t, so_h, lse, scale,
                   T, B, H, causal, rep, m, divisor(rep), divisor(c->page_size), box, grouped ? 8 * row : kKeys * row, grouped ? slabs * 8 * row : 8 * row,
                   static_cast<Desc*>(ws), reinterpret_cast<float*>(static_cast<char*>(ws) + desc_bytes(grid))};
  CUtensorMap maps[2] = {};
  const bool tma = box >= 8 && pool_map(&maps[0], *c, c->k, box) && pool_map(&maps[1], *c, c->v, box);
  const int src = c->dtype == DT_E4M3 ? (tma ? TMA8 : ROWS8) : (tma ? TMA16 : ROWS16);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == DT_F16) return launch_dim<__half>(A, src, maps, grid, st);
  return launch_dim<__nv_bfloat16>(A, src, maps, grid, st);
}
