// Decode attention of a batch in which groups of sequences share a prefix (sm_100a).
//
// Every sequence b brings T new tokens (1: a decode step; more: drafted tokens to verify) that attend, causally,
// the keys of its block table: o = softmax(q K^T scale) V. Sequences that were forked from one another, or
// that begin with the same prompt, name the same pages for their first keys. Reading those pages once per
// sequence costs B times the traffic they need, so the work is cut differently:
//   prefix items   (group, KV head, up to 256 query rows, key range): the rows (sequence, token, head of the KV group) of
//                  ALL sequences of the group against the shared keys, read once for them (attn_shared_tc.cu);
//   own items      (sequence, KV head, key range): the rows of one sequence against the rest of its keys.
// Every item leaves, per row, the maximum m, the sum l of 2^(s - m) and the unnormalised output in fp32; the
// combine kernel merges a row's partials: out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i. All partials of a row
// are summed in a fixed order, so results do not depend on the schedule.
//
// The item list is made on the host when the groups change (PrefixGroups) and lives in device memory, so a
// captured step follows later changes of groups, lengths and tables.
#include "attn_shared_own.cuh"

namespace mesh {
namespace shared_attn {
namespace {

// Where no sequence shares a prefix: three CTAs of four workers an SM.
template <int D, int HALF>
__global__ void __launch_bounds__(WARPS * 32, CTAS) own_kernel(const __grid_constant__ CUtensorMap tmK,
                                                               const __grid_constant__ CUtensorMap tmV, const Args a) {
  using g = Geo<D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Seq* seqs = reinterpret_cast<Seq*>(base + WARPS * g::SLOTS * g::SLICE_BYTES);  // [B + 1]
  __shared__ uint64_t bars[WARPS][g::SLOTS];
  if (threadIdx.x == 0) {
    for (int i = 0; i < WARPS * g::SLOTS; ++i) mbar_init(&bars[0][0] + i, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  griddep_wait();
  griddep_launch_dependents();
  own_sequences(a, seqs, threadIdx.x, [] { __syncthreads(); });
  // few workers spread over the SMs
  own_worker<D, HALF>(tmK, tmV, a, seqs, base + warp * g::SLOTS * g::SLICE_BYTES, bars[warp], lane,
                      warp * (int)gridDim.x + (int)blockIdx.x, WARPS * (int)gridDim.x);
}

// One warp per row (sequence, token, head): merge its partials, the prefix's first, in order. Lane i holds the (m, l) of
// partial i (of the current 32), so the weights are known before the outputs arrive and eight of those are in flight
// at a time.
template <int D>
__global__ void __launch_bounds__(128) combine_kernel(const Args a) {
  griddep_wait();
  griddep_launch_dependents();
  constexpr int V = D / 32, U = 8;
  const int lane = threadIdx.x & 31, hq = a.hkv * a.G, rows = a.T * a.G;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 5);  // (b * T + t) * hq + head
  if (row >= (long)a.B * a.T * hq) return;
  const int b = (int)(row / (a.T * hq));
  const int x = (int)(row - (long)b * a.T * hq), t = x / hq, head = x - t * hq, h = head / a.G;
  const int before = own_before(a)[b], units = own_before(a)[b + 1] - before, quota = own_before(a)[a.B + 1];
  int n_prefix = seq_prefix_slots(a, b);
  const long base = (long)seq_base(a, b) + (long)x * n_prefix;
  // the workers whose quotas this row's slices fall into
  const int r = t * a.G + (head - h * a.G), tile = r / TILE_ROWS, tiles = (rows + TILE_ROWS - 1) / TILE_ROWS;
  const int u = h * tiles + tile, stride = min(rows, TILE_ROWS);
  const int at = before * a.hkv * tiles + u * units + PIECE_COST;  // its first slice
  const int w0 = at / quota;
  int n_own = units > 0 ? (at + units - PIECE_COST - 1) / quota - w0 + 1 : 0;
  if (n_prefix == 0 && n_own == 1) return;  // already written
  const long own = a.own_at + (long)(w0 + b * a.hkv * tiles + u) * stride + (r - tile * TILE_ROWS);  // pieces are `stride` apart
  if (base < 0 || base + n_prefix > a.own_at || (n_own > 0 && own + (long)(n_own - 1) * stride >= a.slot_cap)) {
    if (lane == 0) record_error(a.err, ERR_BAD_ARGUMENT);
    n_prefix = n_own = 0;
  }
  const int n = n_prefix + n_own;
  auto slot = [&](int i) { return i < n_prefix ? base + i : own + (long)(i - n_prefix) * stride; };
  float acc[V] = {}, den = 0.f, M = -INFINITY;
  for (int i = lane; i < n; i += 32) M = fmaxf(M, a.pml[slot(i)].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  for (int i0 = 0; i0 < n && M > -INFINITY; i0 += 32) {
    const float2 ml = i0 + lane < n ? a.pml[slot(i0 + lane)] : make_float2(-INFINITY, 0.f);
    const float f = ex2_ftz(ml.x - M);  // 0 for a partial that saw nothing; its output may not have been written
    den += ml.x > -INFINITY ? ml.y * f : 0.f;
    for (int i = i0; i < min(n, i0 + 32); i += U) {
      float p[U][V], w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        w[u] = __shfl_sync(0xffffffffu, f, (i + u) & 31);
#pragma unroll
        for (int v = 0; v < V; ++v) p[u][v] = 0.f;
        if (i + u < n && w[u] > 0.f) {
          const float* src = a.po + slot(i + u) * D + lane * V;
          if constexpr (V == 4)
            *reinterpret_cast<float4*>(p[u]) = *reinterpret_cast<const float4*>(src);
          else
            *reinterpret_cast<float2*>(p[u]) = *reinterpret_cast<const float2*>(src);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = fmaf(p[u][v], w[u], acc[v]);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
  const float inv = den > 0.f ? 1.f / den : 0.f;
  __nv_bfloat16* dst = a.out + row * D + lane * V;
#pragma unroll
  for (int v = 0; v < V; v += 2) *reinterpret_cast<uint32_t*>(dst + v) = pack_bf16x2(acc[v] * inv, acc[v + 1] * inv);
}

}  // namespace

template <int D>
static cudaError_t launch(const Args& a, cudaStream_t st) {
  const uint64_t rows = (uint64_t)a.pool_pages * a.hkv * a.page_size;
  const CUtensorMap tk = tma_map_2d_bf16(a.k, D, rows, D, 64, SLICE);
  const CUtensorMap tv = tma_map_2d_bf16(a.v, D, rows, D, 64, SLICE);
  // a slice of 128 columns in one box: two halves of 64 columns, 16 rows each
  auto map3 = [&](const void* p) { return tma_map_3d_bf16(p, 64, rows, 2, D * 2, 128, 64, SLICE, 2); };
  const CUtensorMap ok = D == 128 ? map3(a.k) : tk, ov = D == 128 ? map3(a.v) : tv;
  cudaError_t e;
  if (a.n_prefix > 0) {
    e = launch_prefix<D>(a, tk, tv, ok, ov, st);
  } else {
    auto kern = a.T * a.G <= 8 ? own_kernel<D, 1> : own_kernel<D, 2>;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Geo<D>::smem(SHARED_MAX_BATCH));
    if (e != cudaSuccess) return e;
    e = launch_k(kern, dim3((unsigned)(CTAS * a.num_sms)), dim3(WARPS * 32), Geo<D>::smem(a.B), st, ok, ov, a);
  }
  if (e != cudaSuccess) return e;
  const long out_rows = (long)a.B * a.T * a.hkv * a.G;
  return launch_k(combine_kernel<D>, dim3((unsigned)((out_rows + 3) / 4)), dim3(128), 0, st, a);
}

}  // namespace shared_attn

cudaError_t launch_attn_shared(const SharedAttnArgs& x, int head_dim, double scale, cudaStream_t st) {
  shared_attn::Args a;
  static_cast<SharedAttnArgs&>(a) = x;
  a.slices_per_page = x.page_size / shared_attn::SLICE;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  return head_dim == 128 ? shared_attn::launch<128>(a, st) : shared_attn::launch<64>(a, st);
}

}  // namespace mesh
