// Pages of the KV pool copied inside it (forks, branches) and live pages moved to its front (compaction).
//
// Pool layout [layers, pages, kv_heads, page_size, head_dim] bf16, K and V pools alike; one page of one layer is
// contiguous. Both operations are bound by memory: every byte moved is read once and written once.
#include "../include/launch.h"
#include "../include/sharing.h"
#include "../include/sm100.cuh"

namespace mesh {

// Copies inside one pool (a fork's last page, a branch that will rewrite a page): the first tokens[i]
// tokens of page src[i] go to page dst[i] in every layer of K and V. A page of one layer is
// [kv_heads, page_size, D], so the first t tokens are kv_heads runs of t * D elements.
// grid (pairs, layers, 2): one CTA copies one pair in one layer of K or V, 16 bytes per thread step.
// Bound by memory: every byte is read once and written once. Ids outside the pool are recorded as an
// error and skipped; a negative id leaves the pair out (padding of a fixed-size list).
__global__ void __launch_bounds__(256) kv_pages_move_kernel(uint4* __restrict__ k_pool, uint4* __restrict__ v_pool,
                                                            const int* __restrict__ src, const int* __restrict__ dst,
                                                            const int* __restrict__ tokens, int n, long pool_pages,
                                                            int heads, int page_size, int row_vec, int* err) {
  const int i = blockIdx.x, layer = blockIdx.y;
  const int s = src[i], d = dst[i];
  if (layer == 0 && blockIdx.z == 0) {
    // a destination that is also a source or another pair's destination has no defined result
    for (int j = threadIdx.x; j < n; j += blockDim.x)
      if (d >= 0 && s >= 0 && ((dst[j] == d && j != i && src[j] >= 0) || (src[j] == d && dst[j] >= 0)))
        record_error(err, ERR_BAD_ARGUMENT);
  }
  if (s < 0 || d < 0) return;
  if (s >= pool_pages || d >= pool_pages) {
    if (threadIdx.x == 0) record_error(err, ERR_BAD_ARGUMENT);
    return;
  }
  const int t = tokens ? max(0, min(tokens[i], page_size)) : page_size;
  uint4* pool = blockIdx.z == 0 ? k_pool : v_pool;
  const long page_vec = (long)heads * page_size * row_vec;
  const uint4* sp = pool + ((long)layer * pool_pages + s) * page_vec;
  uint4* dp = pool + ((long)layer * pool_pages + d) * page_vec;
  const int run = t * row_vec, head_vec = page_size * row_vec;
  if (t == page_size) {
    for (long v = threadIdx.x; v < page_vec; v += blockDim.x) dp[v] = sp[v];
  } else {
    for (int v = threadIdx.x; v < heads * run; v += blockDim.x) {
      const int h = v / run, o = h * head_vec + (v - h * run);
      dp[o] = sp[o];
    }
  }
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
  for (int w = tid; w < words; w += blockDim.x) {
    const int lo = w * 32;
    bits[w] = reserved >= lo + 32 ? 0xffffffffu : reserved > lo ? (1u << (reserved - lo)) - 1u : 0u;
  }
  __syncthreads();
  const long n = (long)rows * width;
  for (long e = tid; e < n; e += blockDim.x) {
    const int r = (int)(e / width), c = (int)(e - (long)r * width);
    if (c >= counts[r]) continue;
    const int p = tables[e];
    if (p < 0 || p >= pages)
      record_error(err, ERR_BAD_ARGUMENT);
    else
      atomicOr(&bits[p >> 5], 1u << (p & 31));
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
__global__ void __launch_bounds__(256) kv_compact_move_kernel(uint4* __restrict__ k_pool, uint4* __restrict__ v_pool,
                                                              const int* tables, int* out_tables,
                                                              const int* __restrict__ counts, int rows, int width,
                                                              int layers, long pool_pages, long page_vec,
                                                              const int* __restrict__ remap, const int* __restrict__ src,
                                                              const int* __restrict__ dst,
                                                              const int* __restrict__ n_moves) {
  const long n = (long)rows * width;
  for (long e = (long)blockIdx.x * blockDim.x + threadIdx.x; e < n; e += (long)gridDim.x * blockDim.x) {
    const int r = (int)(e / width), c = (int)(e - (long)r * width);
    const int p = tables[e];
    out_tables[e] = (c < counts[r] && p >= 0 && p < pool_pages) ? remap[p] : p;
  }
  const long blocks = (long)*n_moves * layers * 2;
  for (long b = blockIdx.x; b < blocks; b += gridDim.x) {
    const int which = (int)(b & 1);
    const long x = b >> 1;
    const int layer = (int)(x % layers), i = (int)(x / layers);
    uint4* pool = which == 0 ? k_pool : v_pool;
    const uint4* sp = pool + ((long)layer * pool_pages + src[i]) * page_vec;
    uint4* dp = pool + ((long)layer * pool_pages + dst[i]) * page_vec;
    for (long v = threadIdx.x; v < page_vec; v += blockDim.x) dp[v] = sp[v];
  }
}

cudaError_t launch_kv_move(const KvMoveArgs& a, cudaStream_t st) {
  kv_pages_move_kernel<<<dim3((unsigned)a.n, (unsigned)a.layers, 2), 256, 0, st>>>(
      static_cast<uint4*>(a.k), static_cast<uint4*>(a.v), a.src, a.dst, a.tokens, a.n, a.pool_pages, a.heads, a.page_size,
      a.row_vec, a.err);
  return cudaGetLastError();
}

cudaError_t launch_kv_compact(const KvCompactArgs& a, cudaStream_t st) {
  const size_t smem = kv_compact_smem(a.pool_pages);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kv_compact_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  const int pages = (int)a.pool_pages;
  int *remap = a.ws, *live = a.ws + pages, *moves = a.ws + pages + 1, *src = a.ws + pages + 2, *dst = a.ws + 2 * pages + 2;
  kv_compact_plan_kernel<<<1, 1024, smem, st>>>(a.tables, a.counts, a.rows, a.width, pages, a.reserved, remap, live, src, dst,
                                                moves, a.err);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  kv_compact_move_kernel<<<(unsigned)(8 * a.num_sms), 256, 0, st>>>(
      static_cast<uint4*>(a.k), static_cast<uint4*>(a.v), a.tables, a.out_tables, a.counts, a.rows, a.width, a.layers,
      a.pool_pages, a.page_vec, remap, src, dst, moves);
  return cudaGetLastError();
}

}  // namespace mesh
