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
#include "attn_shared.cuh"

namespace mesh {
namespace shared_attn {
namespace {

constexpr int STAGES = 3;
constexpr int KEYS = 64;  // keys per stage

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
}
// byte offset of (row, 16-byte chunk) inside a [16 x 64] box written with the 128-byte swizzle
__device__ __forceinline__ uint32_t swz(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

template <int D>
struct Geo {
  static constexpr int HALVES = D / 64;
  static constexpr uint32_t BOX = SLICE * 64 * 2;           // one [16 x 64] box
  static constexpr uint32_t SLICE_BYTES = 2 * HALVES * BOX; // K halves then V halves
  static constexpr uint32_t STAGE_BYTES = (KEYS / SLICE) * SLICE_BYTES;
  static constexpr int Q_LD = D + 8;
  static constexpr size_t smem(int rows) { return 1024 + STAGES * STAGE_BYTES + 2 * STAGES * 8 + rows * Q_LD * 2; }
};

// The rows of one sequence and KV head (new tokens x heads of the group, at most 64) against a range of the keys
// behind its shared prefix. With at most 16 rows the four warps split the keys (a 16-key slice each, merged at the
// end); otherwise each warp owns 16 rows and walks all four slices of a stage. Bound by reading K and V.
template <int D>
__global__ void __launch_bounds__(160) own_kernel(const __grid_constant__ CUtensorMap tmK,
                                                      const __grid_constant__ CUtensorMap tmV, const Args a) {
  using g = Geo<D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(stages + STAGES * g::STAGE_BYTES);
  uint64_t* empty = full + STAGES;
  __nv_bfloat16* q_s = reinterpret_cast<__nv_bfloat16*>(empty + STAGES);  // 16 rows, or 64
  __shared__ float red_m[4][16], red_l[4][16];
  __shared__ long row_slot[MAX_ROWS];  // partial slot of each row
  __shared__ int row_pos[MAX_ROWS];    // key position of each row's token
  __shared__ long row_q[MAX_ROWS];     // offset of each row in q

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_launch_dependents();
  // behind a prefix kernel, whose own inputs are complete when it lets this one start, only the end has to wait
  if (a.n_prefix == 0) griddep_wait();
  const int split = blockIdx.x % a.own_splits, y = blockIdx.x / a.own_splits;
  const int h = y % a.hkv, seq = y / a.hkv, hq = a.hkv * a.G, rows = a.T * a.G;
  const int L = min(a.seq_lens[seq], a.max_pages * a.page_size);
  int first = seq_prefix(a, seq);
  if (a.window > 0) first = max(first, L - a.T + 1 - a.window);
  const int n_keys = max(0, L - first);
  // key ranges start on slice boundaries of the table
  const int f0 = first / SLICE;
  const int per = ((first + n_keys + SLICE - 1) / SLICE - f0 + a.own_splits - 1) / a.own_splits;
  const int k0 = max(first, (f0 + split * per) * SLICE);
  const int k1 = min(L, (f0 + (split + 1) * per) * SLICE);
  const int slot = seq_prefix_slots(a, seq) + split;
  const int s0 = k0 / SLICE;                                   // first slice
  const int ns = k1 > k0 ? (k1 + SLICE - 1) / SLICE - s0 : 0;  // slices
  const int nst = (ns + KEYS / SLICE - 1) / (KEYS / SLICE);
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    fence_mbar_init();
  }
  for (int r = threadIdx.x; r < MAX_ROWS; r += blockDim.x) {
    const int t = r / a.G, qh = h * a.G + r % a.G;
    long sl = -1;
    if (r < rows) {
      sl = (long)seq_base(a, seq) + (long)(t * hq + qh) * seq_slots(a, seq) + slot;
      if (sl < 0 || sl >= a.slot_cap || slot >= seq_slots(a, seq)) {
        record_error(a.err, ERR_BAD_ARGUMENT);
        sl = -1;
      }
    }
    row_slot[r] = sl;
    row_pos[r] = r < rows ? L - a.T + t : -1;
    row_q[r] = ((long)(seq * a.T + t) * hq + qh) * D;
  }
  __syncthreads();

  if (warp == 4) {
    if (lane == 0) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
      const uint64_t pol = policy_evict_first();
      const int* bt = a.block_tables + (long)seq * a.max_pages;
      for (int i = 0; i < nst; ++i) {
        const int s = i % STAGES;
        if (!mbar_wait_bounded(&empty[s], ((i / STAGES) & 1) ^ 1, a.err, ERR_MBAR_TIMEOUT_PRODUCER, nullptr, WAIT_NS)) break;
        const int n = min(KEYS / SLICE, ns - i * (KEYS / SLICE));
        mbar_arrive_expect_tx(&full[s], (uint32_t)n * g::SLICE_BYTES);
        for (int p = 0; p < n; ++p) {
          const int sl = s0 + i * (KEYS / SLICE) + p;
          const int pi = sl / a.slices_per_page;
          const int y = (bt[pi] * a.hkv + h) * a.page_size + (sl - pi * a.slices_per_page) * SLICE;
          uint8_t* pb = stages + s * g::STAGE_BYTES + p * g::SLICE_BYTES;
#pragma unroll
          for (int hf = 0; hf < g::HALVES; ++hf) {
            tma_load_2d(pb + hf * g::BOX, &tmK, &full[s], hf * 64, y, pol);
            tma_load_2d(pb + (g::HALVES + hf) * g::BOX, &tmV, &full[s], hf * 64, y, pol);
          }
        }
      }
    }
    if (a.n_prefix != 0) griddep_wait();
    return;
  }
  const bool by_rows = rows > 16;
  for (int i = threadIdx.x; i < (by_rows ? MAX_ROWS : 16) * (D / 8); i += 128) {
    const int r = i / (D / 8), c = i - r * (D / 8);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < rows) v = *reinterpret_cast<const uint4*>(a.q + row_q[r] + c * 8);
    *reinterpret_cast<uint4*>(q_s + r * g::Q_LD + c * 8) = v;
  }
  named_bar_sync(1, 128);
  const int wrow = by_rows ? warp * 16 : 0;  // first row of this warp
  uint32_t qf[D / 16][4];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk)
    ldsm_x4(smem_u32(q_s + (wrow + (lane & 15)) * g::Q_LD + kk * 16 + (lane >> 4) * 8), qf[kk]);
  const int rr[2] = {wrow + (lane >> 2), wrow + (lane >> 2) + 8};
  int hi[2], lo[2];  // keys this lane's two rows may attend: [lo, hi)
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    hi[j] = rr[j] < rows ? min(k1, row_pos[rr[j]] + 1) : 0;
    lo[j] = a.window > 0 ? max(k0, row_pos[rr[j]] + 1 - a.window) : k0;
  }
  float o[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const bool live = !by_rows || wrow < rows;
  for (int i = 0; i < nst; ++i) {
    const int s = i % STAGES;
    int okw = 1;
    if (lane == 0) okw = mbar_wait_bounded(&full[s], (i / STAGES) & 1, a.err, ERR_MBAR_TIMEOUT_MMA, nullptr, WAIT_NS);
    if (!__shfl_sync(0xffffffffu, okw, 0)) break;
    const int n = min(KEYS / SLICE, ns - i * (KEYS / SLICE));
    const int p0 = by_rows ? 0 : warp, p1 = !live ? 0 : by_rows ? n : min(n, warp + 1);
    for (int p = p0; p < p1; ++p) {
      const int key0 = (s0 + i * (KEYS / SLICE) + p) * SLICE;
      uint8_t* base = stages + s * g::STAGE_BYTES + p * g::SLICE_BYTES;
      const uint32_t kb = smem_u32(base), vb = kb + g::HALVES * g::BOX;
      if (key0 + SLICE > k1) {
        // keys past the range may hold anything (a page's unused tail): their values must not reach the
        // products as NaN or infinity times a zero weight
        for (int c = lane; c < SLICE * g::HALVES * 8; c += 32) {
          const int r = c / (g::HALVES * 8), x = c - r * (g::HALVES * 8);
          if (key0 + r >= k1) *reinterpret_cast<uint4*>(base + (g::HALVES + x / 8) * g::BOX + swz(r, x & 7)) = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
      }
      float sc[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; kk += 2) {
          uint32_t bb[4];
          ldsm_x4(kb + (kk >> 2) * g::BOX + swz(t * 8 + (lane & 7), (kk & 3) * 2 + (lane >> 3)), bb);
          mma(sc[t], qf[kk], bb[0], bb[1]);
          mma(sc[t], qf[kk + 1], bb[2], bb[3]);
        }
      }
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + t * 8 + (lane & 3) * 2 + (e & 1), j = e >> 1;
          sc[t][e] = (key < hi[j] && key >= lo[j]) ? sc[t][e] * a.scale_log2 : -INFINITY;
          mx[j] = fmaxf(mx[j], sc[t][e]);
        }
      float pr[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 1));
        mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 2));
        const float mn = fmaxf(m[j], mx[j]);
        const float corr = mn == -INFINITY ? 1.f : exp2f(m[j] - mn);
        float ps = 0.f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float p = mn == -INFINITY ? 0.f : exp2f(sc[t][2 * j + e] - mn);
            pr[t][2 * j + e] = p;
            ps += p;
          }
        l[j] = l[j] * corr + ps;
        m[j] = mn;
#pragma unroll
        for (int x = 0; x < D / 8; ++x) {
          o[x][2 * j] *= corr;
          o[x][2 * j + 1] *= corr;
        }
      }
      // the weights are rounded to bf16 for the product (half a step of 2^-8 each); their sum keeps fp32
      const uint32_t pa[4] = {pack_bf16x2(pr[0][0], pr[0][1]), pack_bf16x2(pr[0][2], pr[0][3]),
                              pack_bf16x2(pr[1][0], pr[1][1]), pack_bf16x2(pr[1][2], pr[1][3])};
#pragma unroll
      for (int x = 0; x < D / 8; x += 2) {
        uint32_t bb[4];
        ldsm_x4_t(vb + (x >> 3) * g::BOX + swz((lane & 7) + ((lane >> 3) & 1) * 8, (x & 7) + (lane >> 4)), bb);
        mma(o[x], pa, bb[0], bb[1]);
        mma(o[x + 1], pa, bb[2], bb[3]);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[s]);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    l[j] += __shfl_xor_sync(0xffffffffu, l[j], 1);
    l[j] += __shfl_xor_sync(0xffffffffu, l[j], 2);
  }
  if (by_rows) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const long sl = row_slot[rr[j]];
      if (sl < 0) continue;
#pragma unroll
      for (int x = 0; x < D / 8; ++x)
        *reinterpret_cast<float2*>(a.po + sl * D + x * 8 + (lane & 3) * 2) = make_float2(o[x][2 * j], o[x][2 * j + 1]);
      if ((lane & 3) == 0) a.pml[sl] = make_float2(m[j], l[j]);
    }
    if (a.n_prefix != 0) griddep_wait();
    return;
  }
  // merge the four warps' keys
  if ((lane & 3) == 0)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      red_m[warp][rr[j]] = m[j];
      red_l[warp][rr[j]] = l[j];
    }
  named_bar_sync(1, 128);  // every warp has left the ring
  float* o_s = reinterpret_cast<float*>(stages);  // [4][16][D]
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int x = 0; x < D / 8; ++x)
      *reinterpret_cast<float2*>(o_s + (warp * 16 + rr[j]) * D + x * 8 + (lane & 3) * 2) = make_float2(o[x][2 * j], o[x][2 * j + 1]);
  named_bar_sync(1, 128);
  for (int i = threadIdx.x; i < rows * D; i += 128) {
    const int r = i / D, d = i - r * D;
    const long sl = row_slot[r];
    if (sl < 0) continue;
    float M = -INFINITY, ls = 0.f, ov = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, red_m[w][r]);
    if (M != -INFINITY) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = exp2f(red_m[w][r] - M);
        ls += red_l[w][r] * f;
        ov += o_s[(w * 16 + r) * D + d] * f;
      }
    }
    a.po[sl * D + d] = ov;
    if (d == 0) a.pml[sl] = make_float2(M, ls);
  }
  if (a.n_prefix != 0) griddep_wait();  // this grid is complete only when the prefix grid is
}

// One warp per row (sequence, token, head): merge its partials in slot order. Lane i holds the (m, l) of slot i (of the
// current 32), so the weights are known before the outputs arrive and eight of those are in flight at a time.
template <int D>
__global__ void __launch_bounds__(128) combine_kernel(const Args a) {
  griddep_wait();
  griddep_launch_dependents();
  constexpr int V = D / 32, U = 8;
  const int lane = threadIdx.x & 31, hq = a.hkv * a.G;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 5);  // (b * T + t) * hq + head
  if (row >= (long)a.B * a.T * hq) return;
  const int b = (int)(row / (a.T * hq));
  const int x = (int)(row - (long)b * a.T * hq);
  const long base = (long)seq_base(a, b) + (long)x * seq_slots(a, b);
  int n = seq_prefix_slots(a, b) + a.own_splits;
  if (base < 0 || base + n > a.slot_cap) {
    if (lane == 0) record_error(a.err, ERR_BAD_ARGUMENT);
    n = 0;
  }
  float acc[V] = {}, den = 0.f, M = -INFINITY;
  for (int i = lane; i < n; i += 32) M = fmaxf(M, a.pml[base + i].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  for (int i0 = 0; i0 < n && M > -INFINITY; i0 += 32) {
    const float2 ml = i0 + lane < n ? a.pml[base + i0 + lane] : make_float2(-INFINITY, 0.f);
    const float f = exp2f(ml.x - M);  // 0 for a slot that saw nothing; its output was not written
    den += ml.x > -INFINITY ? ml.y * f : 0.f;
    for (int i = i0; i < min(n, i0 + 32); i += U) {
      float p[U][V], w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        w[u] = i + u < i0 + 32 ? __shfl_sync(0xffffffffu, f, (i + u) & 31) : 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) p[u][v] = 0.f;
        if (i + u < n && w[u] > 0.f) {
          const float* src = a.po + (base + i + u) * D + lane * V;
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
  cudaError_t e = cudaSuccess;
  if (a.n_prefix > 0 && (e = launch_prefix<D>(a, tk, tv, st)) != cudaSuccess) return e;
  auto kern = own_kernel<D>;
  // up to 16 rows need no more than 16 in shared memory: two CTAs fit an SM
  const size_t smem = Geo<D>::smem(a.T * a.G <= 16 ? 16 : MAX_ROWS);
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Geo<D>::smem(MAX_ROWS));
  if (e != cudaSuccess) return e;
  e = launch_k(kern, dim3((unsigned)(a.B * a.hkv * a.own_splits)), dim3(160), smem, st, tk, tv, a);
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
