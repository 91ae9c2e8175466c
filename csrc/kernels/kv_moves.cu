// Pages of the KV pool copied inside it (forks, branches) and live pages moved to its front (compaction).
//
// Pool layout [layers, pages, kv_heads, page_size, head_dim] bf16, K and V pools alike; one page of one layer is
// contiguous. Both operations are bound by memory: every byte moved is read once and written once. Measured with 32 layers
// of 8 KV heads of 128: 200 pages copied (839 MB read and written) 129.8 us, the rate of a plain copy; 9 tokens of 3 pages
// 4.5 us, the host's share of a launch; 210 pages compacted (881 MB) 157.7 us, 0.87 of a copy (the plan comes first, in one CTA). A
// small pool (22 layers of 4 heads of 64, 29 MB moved) compacts in 10.9 us: the two launches and the plan's one CTA.
#include "../include/launch.h"
#include "../include/sharing.h"
#include "../include/sm100.cuh"

namespace mesh {

// n 16-byte vectors, at(v) = their place in both pages. Eight loads per thread are in flight before the first store
// (source and destination lie in one pool, so the compiler would keep each load behind the store before it), and
// both stream past the caches: nothing is read twice.
template <typename At>
__device__ __forceinline__ void copy_vectors(uint4* dp, const uint4* sp, int n, At at) {
  constexpr int U = 8;
  for (int v0 = threadIdx.x; v0 < n; v0 += U * blockDim.x) {
    uint4 r[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v0 + u * blockDim.x < n) r[u] = __ldcs(sp + at(v0 + u * blockDim.x));
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v0 + u * blockDim.x < n) __stcs(dp + at(v0 + u * blockDim.x), r[u]);
  }
}

// Copies inside one pool (a fork's last page, a branch that will rewrite a page): the first tokens[i]
// tokens of page src[i] go to page dst[i] in every layer of K and V. A page of one layer is
// [kv_heads, page_size, D], so the first t tokens are kv_heads runs of t * D elements.
// grid (pairs, layers, 2): one CTA copies one pair in one layer of K or V. Ids outside the pool are recorded as an
// error and skipped; a negative id leaves the pair out (padding of a fixed-size list).
__global__ void __launch_bounds__(256) kv_pages_move_kernel(const KvMoveArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  const int i = blockIdx.x, layer = blockIdx.y;
  const int s = a.src[i], d = a.dst[i];
  if (layer == 0 && blockIdx.z == 0 && s >= 0 && d >= 0) {
    // a destination that is also a source or another pair's destination has no defined result
    for (int j = threadIdx.x; j < a.n; j += blockDim.x) {
      const int sj = a.src[j], dj = a.dst[j];
      if (sj >= 0 && dj >= 0 && ((dj == d && j != i) || sj == d)) record_error(a.err, ERR_BAD_ARGUMENT);
    }
  }
  if (s < 0 || d < 0) return;
  if (s >= a.pool_pages || d >= a.pool_pages) {
    if (threadIdx.x == 0) record_error(a.err, ERR_BAD_ARGUMENT);
    return;
  }
  const int t = a.tokens ? max(0, min(a.tokens[i], a.page_size)) : a.page_size;
  uint4* pool = static_cast<uint4*>(blockIdx.z == 0 ? a.k : a.v);
  const int head_vec = a.page_size * a.row_vec, page_vec = a.heads * head_vec, run = t * a.row_vec;
  const uint4* sp = pool + ((long)layer * a.pool_pages + s) * page_vec;
  uint4* dp = pool + ((long)layer * a.pool_pages + d) * page_vec;
  if (t == a.page_size)
    copy_vectors(dp, sp, page_vec, [](int v) { return v; });
  else
    copy_vectors(dp, sp, a.heads * run, [=](int v) {
      const int h = v / run;
      return h * head_vec + (v - h * run);
    });
}

// Compaction, step 1 (one CTA): which pages are live (reserved, or named by a used block-table entry), how
// many (`live`), and where each goes: a live page below `live` stays, the k-th live page from `live` up
// goes to the k-th hole below it, so the fewest pages move. Order is by page id, so the result does not
// depend on the order of the marks.
// Shared memory: one bit per page, and the live pages before each 32-page word.
__global__ void __launch_bounds__(1024) kv_compact_plan_kernel(const int* __restrict__ tables,
                                                               const int* __restrict__ counts, int rows, int width,
                                                               int pages, int reserved, int* __restrict__ remap,
                                                               int* __restrict__ live_out, int* __restrict__ src,
                                                               int* __restrict__ dst, int* __restrict__ n_moves,
                                                               int* err) {
  extern __shared__ uint32_t sm[];
  __shared__ int warp_sum[32];
  const int words = (pages + 31) / 32;
  uint32_t* bits = sm;
  int* before = reinterpret_cast<int*>(sm + words);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  griddep_wait();
  griddep_launch_dependents();
  for (int w = tid; w < words; w += blockDim.x) {
    const int lo = w * 32;
    bits[w] = reserved >= lo + 32 ? 0xffffffffu : reserved > lo ? (1u << (reserved - lo)) - 1u : 0u;
  }
  __syncthreads();
  for (int r = warp; r < rows; r += 32) {
    const int c1 = min(counts[r], width);
    const int* row = tables + (long)r * width;
    for (int c = lane; c < c1; c += 32) {
      const int p = row[c];
      if (p < 0 || p >= pages)
        record_error(err, ERR_BAD_ARGUMENT);
      else
        atomicOr(&bits[p >> 5], 1u << (p & 31));
    }
  }
  __syncthreads();
  // exclusive prefix of the words' live counts: a contiguous run of words per thread
  const int per = (words + blockDim.x - 1) / blockDim.x;
  const int w0 = min(words, tid * per), w1 = min(words, w0 + per);
  int mine = 0;
  for (int w = w0; w < w1; ++w) mine += __popc(bits[w]);
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int base = 0, live = 0;
  for (int w = 0; w < 32; ++w) {
    if (w < warp) base += warp_sum[w];
    live += warp_sum[w];
  }
  int run = base + incl - mine;
  for (int w = w0; w < w1; ++w) {
    before[w] = run;
    run += __popc(bits[w]);
  }
  __syncthreads();
  auto live_before = [&](int p) -> int {  // live pages with an id below p (p < pages)
    return before[p >> 5] + __popc(bits[p >> 5] & ((1u << (p & 31)) - 1u));
  };
  const int below = live < pages ? live_before(live) : live;  // live pages that stay
  for (int p = tid; p < pages; p += blockDim.x) {
    const bool used = (bits[p >> 5] >> (p & 31)) & 1u;
    const int rank = live_before(p);
    if (used && p >= live)
      src[rank - below] = p;
    else if (!used && p < live)
      dst[p - rank] = p;
  }
  __syncthreads();
  for (int p = tid; p < pages; p += blockDim.x) {
    const bool used = (bits[p >> 5] >> (p & 31)) & 1u;
    remap[p] = !used ? -1 : p < live ? p : dst[live_before(p) - below];
  }
  if (tid == 0) {
    *live_out = live;
    *n_moves = live - below;
  }
}

// Compaction, step 2: rewrite the used table entries and copy the moved pages in every layer of K and V.
// The number of moves is known on the device only, so a fixed grid walks the (move, layer, K or V) blocks.
// Sources lie at or above the live count and destinations below it, so no block is read after it is written.
__global__ void __launch_bounds__(256) kv_compact_move_kernel(const KvCompactArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  const int pages = (int)a.pool_pages;
  const int *remap = a.ws, *src = a.ws + pages + 2, *dst = src + pages;
  const int moves = a.ws[pages + 1];
  const int warp = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  for (int r = warp; r < a.rows; r += (gridDim.x * blockDim.x) >> 5) {
    const int used = a.counts[r];
    for (int c = lane; c < a.width; c += 32) {
      const int p = a.tables[(long)r * a.width + c];
      a.out_tables[(long)r * a.width + c] = (c < used && p >= 0 && p < pages) ? remap[p] : p;
    }
  }
  const long blocks = (long)moves * a.layers * 2;
  for (long b = blockIdx.x; b < blocks; b += gridDim.x) {
    const int i = (int)(b / (2 * a.layers)), x = (int)(b - (long)i * (2 * a.layers));  // x: layer, K or V
    uint4* pool = static_cast<uint4*>((x & 1) == 0 ? a.k : a.v) + (long)(x >> 1) * a.pool_pages * a.page_vec;
    copy_vectors(pool + dst[i] * a.page_vec, pool + src[i] * a.page_vec, (int)a.page_vec, [](int v) { return v; });
  }
}

cudaError_t launch_kv_move(const KvMoveArgs& a, cudaStream_t st) {
  return launch_k(kv_pages_move_kernel, dim3((unsigned)a.n, (unsigned)a.layers, 2), dim3(256), 0, st, a);
}

cudaError_t launch_kv_compact(const KvCompactArgs& a, cudaStream_t st) {
  const size_t smem = kv_compact_smem(a.pool_pages);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kv_compact_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  const int pages = (int)a.pool_pages;
  int *remap = a.ws, *live = a.ws + pages, *moves = a.ws + pages + 1, *src = a.ws + pages + 2, *dst = a.ws + 2 * pages + 2;
  const cudaError_t e = launch_k(kv_compact_plan_kernel, dim3(1), dim3(1024), smem, st, a.tables, a.counts, a.rows, a.width,
                                 pages, a.reserved, remap, live, src, dst, moves, a.err);
  if (e != cudaSuccess) return e;
  return launch_k(kv_compact_move_kernel, dim3((unsigned)(8 * a.num_sms)), dim3(256), 0, st, a);
}

}  // namespace mesh
