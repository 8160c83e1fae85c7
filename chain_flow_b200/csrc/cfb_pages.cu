// cfb_pages.cu -- the pages of a paged key/value cache (sm_100a): a step's accepted rows moved together
// (cfb_kv_keep), pages copied (cfb_kv_copy_pages), and pages taken, given back and forked by their reference
// counts (cfb_pages_reserve, cfb_pages_release, cfb_pages_fork).
//
// No arithmetic: whole rows move, and page numbers are counted. Moves are bound by HBM where there are many
// rows and by launch latency where there are few, so all layers of a target go in one launch.
//
// The free pages of a pool are those whose count is 0, and a call takes the lowest of them, request after
// request, so that its result does not depend on any order of execution. One CTA finds them: it turns the
// counts into a bit a page in shared memory (32 loads in flight a thread), counts the bits, and then gives
// every page that is asked for a thread, which looks up its request and its free page by bisection. Of a large pool a
// cluster of 8 CTAs does that, an eighth of the counts and of the pages each.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include "cfb_types.cuh"

using namespace cfb;
namespace cg = cooperative_groups;

namespace {

constexpr int kLayers = 32;                  // caches a launch
constexpr int kThreads = 256;
constexpr int kHeld = 8;                     // 16-byte pieces a thread holds
constexpr int kCopied = 4;                   // and of a copied page: 5 CTAs an SM instead of 3
constexpr int kMaxPath = 1024;

struct Layers {                              // caches of one geometry
  cfb_kv_cache c;                            // of the first: strides, sizes
  struct { char *k, *v; float *ks, *vs; } at[kLayers];
  int size, pieces;                          // bytes an element, log2 of a row's 16-byte pieces
};

// The pool's kernels follow one another in a stream (given back, taken, forked): each is launched while the one before
// still runs and waits for its end before it reads anything, which hides part of a launch (a scheduler's step of two kernels 13.8 -> 12.3 us).
__device__ __forceinline__ void after_the_kernel_before() {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
template <typename... P, typename... A>
cfb_status launch_after(const char* name, void (*kernel)(P...), dim3 grid, int threads, int smem, int cluster, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  return cfb_launch_status(name);
}

// ---- accepted rows ----------------------------------------------------------------------------------
struct KeepArgs {
  const int32_t* table; long long table_stride; int width;
  const int32_t* base; const int32_t* path; long long path_stride; const int32_t* count;
  int max_len, heads;                        // heads a CTA
};

// A CTA: a request (x), a layer (y), a group of heads (z). The rows of a batch are all read before the first is written; a
// later batch reads rows behind every one that was written, since a path's j-th node is not before j.
// Bound by latency: three loads that wait for each other (path, page table, rows), then the stores. Keys and values by one
// CTA, so that 64 requests of 8 layers are in flight at once. Measured, 8 layers of 4 heads of 256, up to 5 rows a request: one
// request, bf16, 5 us; 64, e4m3, 7 (bytes: 0.8).
__global__ void __launch_bounds__(kThreads, 3) kv_keep_kernel(const __grid_constant__ Layers L, const KeepArgs A) {
  extern __shared__ longlong4 s_move[];      // of a position: byte offsets of its row, from and to (or -1), and its scales'
  const int b = blockIdx.x, S = L.c.page_size;
  const int count = A.count[b];
  const long long base = A.base[b];
  for (int j = threadIdx.x; j < A.max_len; j += kThreads) {
    const int node = A.path[b * A.path_stride + j];
    const long long from = base + node, to = base + j, end = (long long)A.width * S;
    longlong4 m = make_longlong4(-1, 0, 0, 0);
    if (j < count && node >= 0 && node != j && from >= 0 && to >= 0 && from < end && to < end) {
      const long long fp = from / S, tp = to / S, fo = from - fp * S, to_ = to - tp * S;
      const int fpage = A.table[b * A.table_stride + fp], tpage = A.table[b * A.table_stride + tp];
      if (fpage >= 0 && fpage < L.c.pages && tpage >= 0 && tpage < L.c.pages) {
        m.x = (fpage * L.c.page_stride + fo * L.c.slot_stride) * L.size;
        m.y = (tpage * L.c.page_stride + to_ * L.c.slot_stride) * L.size;
        m.z = fpage * L.c.scale_page_stride + fo * L.c.scale_slot_stride;
        m.w = tpage * L.c.scale_page_stride + to_ * L.c.scale_slot_stride;
      }
    }
    s_move[j] = m;
  }
  __syncthreads();
  const int n = min(count, A.max_len);
  const auto& at = L.at[blockIdx.y];
  const int h0 = blockIdx.z * A.heads, hn = min(A.heads, L.c.kv_heads - h0);
  const int wide = hn << L.pieces, batch = kThreads * kHeld / 2 / wide;    // pieces a position, positions a batch
  const long long head = L.c.head_stride * L.size;
  for (int j0 = 0; j0 < n; j0 += batch) {
    const int m = min(batch, n - j0), half = m * wide;
    uint4 w[kHeld];
    char* to[kHeld];
    float sc[4];
    float* scale_to[4];
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int i = k * kThreads + threadIdx.x, x = i < half ? i : i - half;
      to[k] = nullptr;
      if (i < 2 * half) {
        const int j = x / wide, y = x - j * wide;
        const longlong4 v = s_move[j0 + j];
        if (v.x >= 0) {
          char* const rows = (i < half ? at.k : at.v) + (h0 + (y >> L.pieces)) * head + ((y & ((1 << L.pieces) - 1)) << 4);
          w[k] = *reinterpret_cast<const uint4*>(rows + v.x);
          to[k] = rows + v.y;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = k * kThreads + threadIdx.x, x = i < m * hn ? i : i - m * hn;
      scale_to[k] = nullptr;
      if (at.ks && i < 2 * m * hn) {
        const longlong4 v = s_move[j0 + x / hn];
        if (v.x >= 0) {
          float* const scales = (i < m * hn ? at.ks : at.vs) + (h0 + x % hn) * L.c.scale_head_stride;
          sc[k] = scales[v.z];
          scale_to[k] = scales + v.w;
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
      if (to[k]) *reinterpret_cast<uint4*>(to[k]) = w[k];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (scale_to[k]) *scale_to[k] = sc[k];
  }
}

// ---- whole pages --------------------------------------------------------------------------------------
// the leading `slots` slots of page src to page dst, of one layer's keys or values
__device__ __forceinline__ void copy_page(const Layers& L, int layer, bool value, int src, int dst, int slots) {
  const int pages = L.c.pages, n = min(slots, L.c.page_size);
  if (src < 0 || src >= pages || dst < 0 || dst >= pages || src == dst || n <= 0) return;
  const auto& at = L.at[layer];
  const char* const from = (value ? at.v : at.k) + src * L.c.page_stride * L.size;
  char* const to = (value ? at.v : at.k) + dst * L.c.page_stride * L.size;
  const int total = (L.c.kv_heads * n) << L.pieces;
  for (int i0 = threadIdx.x; i0 < total; i0 += kCopied * kThreads) {
    uint4 w[kCopied];
    long long o[kCopied];
#pragma unroll
    for (int k = 0; k < kCopied; ++k) {
      const int i = i0 + k * kThreads;
      if (i < total) {
        const unsigned r = (unsigned)i >> L.pieces, h = r / (unsigned)n, slot = r - h * n;
        o[k] = ((long long)h * L.c.head_stride + slot * L.c.slot_stride) * L.size + ((i & ((1 << L.pieces) - 1)) << 4);
        w[k] = __ldg(reinterpret_cast<const uint4*>(from + o[k]));
      }
    }
#pragma unroll
    for (int k = 0; k < kCopied; ++k)
      if (i0 + k * kThreads < total) *reinterpret_cast<uint4*>(to + o[k]) = w[k];
  }
  if (const float* const s = value ? at.vs : at.ks) {
    float* const d = value ? at.vs : at.ks;
    for (int i = threadIdx.x; i < L.c.kv_heads * n; i += kThreads) {
      const int h = i / n;
      const long long o_ = h * L.c.scale_head_stride + (i - h * n) * L.c.scale_slot_stride;
      d[dst * L.c.scale_page_stride + o_] = s[src * L.c.scale_page_stride + o_];
    }
  }
}

// A CTA: a pair of pages (x), a layer's keys or values (y). Bound by HBM: 1.07 GB read and written in 165 us, 6.5 TB/s, as
// a plain copy's rate.
__global__ void __launch_bounds__(kThreads, 5) kv_copy_pages_kernel(const __grid_constant__ Layers L, const int32_t* src,
                                                                 const int32_t* dst, const int32_t* slots) {
  copy_page(L, blockIdx.y >> 1, blockIdx.y & 1, src[blockIdx.x], dst[blockIdx.x], slots ? slots[blockIdx.x] : L.c.page_size);
}

// ---- the pool -------------------------------------------------------------------------------------------
struct Pool {
  int32_t* refs; int pages, page_size;
  int32_t* table; long long stride; int width, rows;
};
__device__ __forceinline__ int pages_for(int positions, int page_size) {
  return (int)(((long long)max(positions, 0) + page_size - 1) / page_size);
}

constexpr int kTake = 1024;                  // threads of the CTA that takes pages, and requests it takes at a time
constexpr int kGroup = 8;                    // 32-page words a counted group
constexpr int kMaxPages = 1 << 20;
constexpr int kLarge = 8192;                 // pages from which on 8 CTAs look for free ones

struct TakeArgs {
  Pool P;
  const int32_t* length; const int32_t* target;            // reserve: positions held and wanted; fork: length by row
  const int32_t* parent; const int32_t* child;             // fork
  int32_t* granted;
  int n;
};

// inclusive running sum over the CTA; every thread has to come
template <typename F> __device__ __forceinline__ F cta_scan(F v, F* s_warp, F* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const F o = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += o;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  // (every warp sums the warps' totals for itself: no third barrier)
  F x = s_warp[lane];
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const F o = __shfl_up_sync(0xffffffffu, x, off);
    if (lane >= off) x += o;
  }
  *total = __shfl_sync(0xffffffffu, x, 31);
  const F before = __shfl_sync(0xffffffffu, x, max(warp - 1, 0));
  return v + (warp ? before : (F)0);
}
// the position of the n-th set bit (n < number of bits)
__device__ __forceinline__ int nth_bit(uint32_t bits, int n) {
  int at = 0;
#pragma unroll
  for (int half = 16; half; half >>= 1) {
    const int c = __popc(bits & ((1u << half) - 1));
    if (n >= c) {
      n -= c;
      at += half;
      bits >>= half;
    }
  }
  return at;
}

// FORK: request i is the fork of row parent[i] into row child[i], which needs a page for what its last one holds.
// Bound by latency: the counts' loads, a barrier or two a running sum, a bisection a page that is asked for. Measured: 256
// requests of a pool of 65536 pages, the release before it included, 12.4 us (bytes: 0.07); one CTA for all of it took 34 with it.
template <bool FORK>
__global__ void __launch_bounds__(kTake) pages_take_kernel(const TakeArgs A) {
  after_the_kernel_before();
  extern __shared__ uint32_t s_free[];       // a bit a page; then the free pages up to each group of words
  __shared__ long long s_warp[32];
  __shared__ int s_sum[32];
  __shared__ int s_start[kTake];                           // pages asked for up to a request, in order (up to 2^30)
  __shared__ int s_first[kTake];                           // where a request's pages go in its row, or -1
  const cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
  const Pool& P = A.P;
  const int words = (P.pages + 31) / 32, groups = (words + kGroup - 1) / kGroup;
  int* const s_count = reinterpret_cast<int*>(s_free + groups * kGroup);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // the first requests' needs are on their way while the counts are read
  const auto need_of = [&](int b, int* first) {            // -1: it cannot be granted
    *first = 0;
    if (b >= A.n) return 0;
    if constexpr (FORK) {
      const int from = A.parent[b], to = A.child[b];
      if (from < 0 || from >= P.rows || to < 0 || to >= P.rows || from == to) return -1;
      const int len = max(A.length[from], 0), need = len % P.page_size ? 1 : 0;
      *first = len / P.page_size;
      return *first + need <= P.width ? need : -1;
    } else {
      *first = pages_for(A.length[b], P.page_size);
      const int upto = pages_for(A.target[b], P.page_size), need = max(upto - *first, 0);
      return need == 0 || upto <= P.width ? need : -1;
    }
  };
  int first, need = need_of(threadIdx.x, &first);
  // a CTA's share of the words, in whole 32s
  const int share = ((groups * kGroup + ranks - 1) / ranks + 31) / 32 * 32;
  const int share0 = rank * share, share1 = min(share0 + share, groups * kGroup);
  for (int w0 = share0 + warp * 32; w0 < share1; w0 += kTake) {
    int r[32];
    uint32_t mine = 0;
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      const int p = (w0 + k) * 32 + lane;
      r[k] = p < P.pages ? P.refs[p] : 1;
    }
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      const uint32_t bits = __ballot_sync(0xffffffffu, r[k] == 0);
      if (lane == k) mine = bits;
    }
    if (w0 + lane < share1) s_free[w0 + lane] = mine;
  }
  if (ranks > 1) {                           // every CTA needs all of them; none writes a count before all are read
    cluster.sync();
    for (int w = threadIdx.x; w < groups * kGroup; w += kTake)
      if (w / share != rank) s_free[w] = cluster.map_shared_rank(s_free, w / share)[w];
    cluster.sync();
  }
  __syncthreads();
  int free = 0;
  for (int g0 = 0; g0 < groups; g0 += kTake) {
    int c = 0;
    const int g = g0 + threadIdx.x;
    if (g < groups)
#pragma unroll
      for (int k = 0; k < kGroup; ++k) c += __popc(s_free[g * kGroup + k]);
    int total;
    const int up = cta_scan(c, s_sum, &total);
    if (g < groups) s_count[g] = free + up;
    free += total;
  }
  long long asked = 0;                       // by the requests before
  for (int b0 = 0; b0 < A.n; b0 += kTake) {
    const int b = b0 + threadIdx.x;
    if (b0) need = need_of(b, &first);
    long long total;
    const long long up = asked + cta_scan((long long)max(need, 0), s_warp, &total);
    const bool ok = need >= 0 && (need == 0 || up <= free);
    if (b < A.n && rank == 0) A.granted[b] = ok;
    s_start[threadIdx.x] = (int)min(up, 1ll << 30);
    s_first[threadIdx.x] = ok ? first : -1;
    __syncthreads();
    const int end = (int)min(asked + total, (long long)free);
    for (long long at = asked + rank * kTake + threadIdx.x; at < end; at += ranks * kTake) {
      const int r = (int)at;
      int lo = 0, hi = kTake - 1;            // the first request with s_start > r
#pragma unroll
      for (int step = 0; step < 10; ++step) {
        const int mid = (lo + hi) >> 1;
        if (s_start[mid] > r) hi = mid; else lo = mid + 1;
      }
      if (s_first[lo] < 0) continue;
      const int before = lo ? s_start[lo - 1] : (int)asked;
      int g = 0, gh = groups - 1;            // the group that holds free page r
      while (g < gh) {
        const int mid = (g + gh) >> 1;
        if (s_count[mid] > r) gh = mid; else g = mid + 1;
      }
      int left = r - (g ? s_count[g - 1] : 0), w = g * kGroup;
      for (int c; left >= (c = __popc(s_free[w])); ++w) left -= c;
      const int page = w * 32 + nth_bit(s_free[w], left);
      const int row = FORK ? A.child[b0 + lo] : b0 + lo;
      P.table[row * P.stride + s_first[lo] + (r - before)] = page;
      P.refs[page] = 1;
    }
    asked += total;
    __syncthreads();
  }
}

// A CTA: a request. Counts fall; a page that nobody holds is left alone and flagged.
__global__ void __launch_bounds__(kThreads) pages_release_kernel(const Pool P, const int32_t* length, const int32_t* keep, int* err) {
  const int b = blockIdx.x;
  after_the_kernel_before();
  const int from = keep ? pages_for(keep[b], P.page_size) : 0, to = min(pages_for(length[b], P.page_size), P.width);
  int32_t* const row = P.table + b * P.stride;
  for (int j = from + threadIdx.x; j < to; j += kThreads) {
    const int page = row[j];
    if (page >= 0 && page < P.pages) {
      if (atomicSub(P.refs + page, 1) <= 0) {
        atomicAdd(P.refs + page, 1);
        if (err) atomicCAS(err, 0, DEV_BAD_INDEX);
      }
    }
    row[j] = -1;
  }
}

// After pages_take_kernel<true>. A CTA: a fork (x); its row and counts (the first `lead` y, 0 or 1), or its last page in
// a layer's keys or values. Measured, both kernels: 8 forks of 9001 positions, a page in 8 layers each, 13.4 us (bytes: 0.7); 64
// of 1500, pages of 48 slots in e4m3, 22.6 (7.9).
__global__ void __launch_bounds__(kThreads, 5) pages_fork_kernel(const __grid_constant__ Layers L, const Pool P, int32_t* length,
                                                              const int32_t* parent, const int32_t* child,
                                                              const int32_t* granted, int lead) {
  const int i = blockIdx.x, y = (int)blockIdx.y - lead;
  after_the_kernel_before();
  if (!granted[i]) return;
  const int from = parent[i], to = child[i], len = max(length[from], 0), full = len / P.page_size;
  const int32_t* const src = P.table + from * P.stride;
  int32_t* const dst = P.table + to * P.stride;
  if (y >= 0) {
    if (len % P.page_size) copy_page(L, y >> 1, y & 1, src[full], dst[full], len % P.page_size);
    return;
  }
  for (int j = threadIdx.x; j < full; j += kThreads) {
    const int page = src[j];
    dst[j] = page;
    if (page >= 0 && page < P.pages) atomicAdd(P.refs + page, 1);
  }
  if (threadIdx.x == 0) length[to] = len;
}

// ---- host -------------------------------------------------------------------------------------------------
bool same_geometry(const cfb_kv_cache& a, const cfb_kv_cache& b) {
  return a.page_stride == b.page_stride && a.head_stride == b.head_stride && a.slot_stride == b.slot_stride &&
         a.scale_page_stride == b.scale_page_stride && a.scale_head_stride == b.scale_head_stride &&
         a.scale_slot_stride == b.scale_slot_stride && a.pages == b.pages && a.page_size == b.page_size &&
         a.kv_heads == b.kv_heads && a.dim == b.dim && a.dtype == b.dtype;
}
cfb_status check_layers(const cfb_kv_cache* const* caches, int n) {
  if (n < 0 || (n > 0 && !caches)) return CFB_ERR_INVALID_ARG;
  for (int i = 0; i < n; ++i) {
    if (const cfb_status s = check_cache(caches[i])) return s;
    if (!same_geometry(*caches[0], *caches[i])) return CFB_ERR_INVALID_ARG;
  }
  return CFB_OK;
}
Layers layers_of(const cfb_kv_cache* const* caches, int n) {
  Layers L{};
  L.c = *caches[0];
  L.size = L.c.dtype == DT_E4M3 ? 1 : 2;
  for (int p = L.c.dim * L.size / 16; p > 1; p >>= 1) ++L.pieces;
  for (int i = 0; i < n; ++i)
    L.at[i] = {static_cast<char*>(caches[i]->k), static_cast<char*>(caches[i]->v), caches[i]->k_scale, caches[i]->v_scale};
  return L;
}
cfb_status check_pool(const int32_t* refs, int pages, int page_size, const int32_t* table, int64_t stride, int width, int rows) {
  if (!refs || pages <= 0 || page_size <= 0 || width < 0 || rows < 0 || stride < width || (rows > 0 && width > 0 && !table))
    return CFB_ERR_INVALID_ARG;
  return pages > kMaxPages ? CFB_ERR_UNSUPPORTED : CFB_OK;
}
template <bool FORK> cfb_status launch_take(const TakeArgs& a, cudaStream_t st) {
  const auto bytes = [](int pages) { return ((pages + 31) / 32 + kGroup - 1) / kGroup * (kGroup + 1) * 4; };
  if (allow_smem<pages_take_kernel<FORK>>(bytes(kMaxPages)) != cudaSuccess) return cfb_launch_status("pages_take_kernel");
  const int ctas = a.P.pages >= kLarge ? 8 : 1;
  return launch_after("pages_take_kernel", pages_take_kernel<FORK>, dim3(ctas), kTake, bytes(a.P.pages), ctas, st, a);
}

}  // namespace

extern "C" cfb_status cfb_kv_keep(const cfb_kv_cache* const* caches, int n_caches, const int32_t* page_table, int64_t table_stride,
                                  int table_width, const int32_t* base, const int32_t* path, int64_t path_stride,
                                  const int32_t* count, int max_len, int B, void* stream) {
  if (const cfb_status s = check_layers(caches, n_caches)) return s;
  if (B < 0 || max_len < 0 || table_width < 0 || table_stride < table_width || path_stride < max_len) return CFB_ERR_INVALID_ARG;
  for (int i = 0; i < n_caches; ++i)                       // (moved twice at once, rows would be read behind the first move's writes)
    for (int j = 0; j < i; ++j)
      if (caches[i]->k == caches[j]->k || caches[i]->v == caches[j]->v) return CFB_ERR_INVALID_ARG;
  if (B == 0 || n_caches == 0 || max_len == 0 || table_width == 0) return CFB_OK;
  if (!page_table || !base || !path || !count) return CFB_ERR_INVALID_ARG;
  if (max_len > kMaxPath) return CFB_ERR_UNSUPPORTED;
  KeepArgs a{page_table, table_stride, table_width, base, path, path_stride, count, max_len, 0};
  for (int i = 0; i < n_caches; i += kLayers) {
    const int n = n_caches - i < kLayers ? n_caches - i : kLayers;
    const Layers L = layers_of(caches + i, n);
    a.heads = kThreads >> L.pieces;                        // up to kThreads pieces a position
    if (a.heads > L.c.kv_heads) a.heads = L.c.kv_heads;
    const dim3 grid(B, n, (L.c.kv_heads + a.heads - 1) / a.heads);
    if (grid.z > 65535) return CFB_ERR_UNSUPPORTED;
    kv_keep_kernel<<<grid, kThreads, max_len * sizeof(longlong4), static_cast<cudaStream_t>(stream)>>>(L, a);
    if (const cfb_status s = cfb_launch_status("kv_keep_kernel")) return s;
  }
  return CFB_OK;
}

extern "C" cfb_status cfb_kv_copy_pages(const cfb_kv_cache* const* caches, int n_caches, const int32_t* src, const int32_t* dst,
                                        const int32_t* slots, int pairs, void* stream) {
  if (const cfb_status s = check_layers(caches, n_caches)) return s;
  if (pairs < 0) return CFB_ERR_INVALID_ARG;
  if (pairs == 0 || n_caches == 0) return CFB_OK;
  if (!src || !dst) return CFB_ERR_INVALID_ARG;
  for (int i = 0; i < n_caches; i += kLayers) {
    const int n = n_caches - i < kLayers ? n_caches - i : kLayers;
    const Layers L = layers_of(caches + i, n);
    if ((long long)L.c.kv_heads * L.c.page_size << L.pieces >= 1ll << 30) return CFB_ERR_UNSUPPORTED;
    kv_copy_pages_kernel<<<dim3(pairs, 2 * n), kThreads, 0, static_cast<cudaStream_t>(stream)>>>(L, src, dst, slots);
    if (const cfb_status s = cfb_launch_status("kv_copy_pages_kernel")) return s;
  }
  return CFB_OK;
}

extern "C" cfb_status cfb_pages_reserve(int32_t* refs, int pages, int page_size, int32_t* table, int64_t table_stride, int table_width,
                                        const int32_t* length, const int32_t* target, int32_t* granted, int B, void* stream) {
  if (const cfb_status s = check_pool(refs, pages, page_size, table, table_stride, table_width, B)) return s;
  if (B == 0) return CFB_OK;
  if (!length || !target || !granted) return CFB_ERR_INVALID_ARG;
  TakeArgs a{};
  a.P = {refs, pages, page_size, table, table_stride, table_width, B};
  a.length = length; a.target = target; a.granted = granted; a.n = B;
  return launch_take<false>(a, static_cast<cudaStream_t>(stream));
}

extern "C" cfb_status cfb_pages_release(int32_t* refs, int pages, int page_size, int32_t* table, int64_t table_stride, int table_width,
                                        const int32_t* length, const int32_t* keep, int B, int* err, void* stream) {
  if (const cfb_status s = check_pool(refs, pages, page_size, table, table_stride, table_width, B)) return s;
  if (B == 0 || table_width == 0) return CFB_OK;
  if (!length) return CFB_ERR_INVALID_ARG;
  const Pool P{refs, pages, page_size, table, table_stride, table_width, B};
  return launch_after("pages_release_kernel", pages_release_kernel, dim3(B), kThreads, 0, 1, static_cast<cudaStream_t>(stream), P, length,
                      keep, err);
}

extern "C" cfb_status cfb_pages_fork(int32_t* refs, int pages, int page_size, int32_t* table, int64_t table_stride, int table_width,
                                     int rows, int32_t* length, const int32_t* parent, const int32_t* child, int32_t* granted, int n,
                                     const cfb_kv_cache* const* caches, int n_caches, void* stream) {
  if (const cfb_status s = check_pool(refs, pages, page_size, table, table_stride, table_width, rows)) return s;
  if (const cfb_status s = check_layers(caches, n_caches)) return s;
  if (n < 0) return CFB_ERR_INVALID_ARG;
  if (n_caches > 0 && (caches[0]->page_size != page_size || caches[0]->pages < pages)) return CFB_ERR_INVALID_ARG;
  if (n == 0) return CFB_OK;
  if (!length || !parent || !child || !granted) return CFB_ERR_INVALID_ARG;
  if (n_caches > 0 && (long long)caches[0]->kv_heads * page_size * caches[0]->dim >= 1ll << 30) return CFB_ERR_UNSUPPORTED;
  TakeArgs a{};
  a.P = {refs, pages, page_size, table, table_stride, table_width, rows};
  a.length = length; a.parent = parent; a.child = child; a.granted = granted; a.n = n;
  if (const cfb_status s = launch_take<true>(a, static_cast<cudaStream_t>(stream))) return s;
  for (int i = 0; i == 0 || i < n_caches; i += kLayers) {
    const int m = n_caches - i < kLayers ? n_caches - i : kLayers, lead = i == 0;
    const Layers L = m > 0 ? layers_of(caches + i, m) : Layers{};
    if (const cfb_status s = launch_after("pages_fork_kernel", pages_fork_kernel, dim3(n, lead + 2 * m), kThreads, 0, 1,
                                          static_cast<cudaStream_t>(stream), L, a.P, length, parent, child, granted, lead))
      return s;
  }
  return CFB_OK;
}
