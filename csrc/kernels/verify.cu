// Verification of drafted tokens against the target model's probabilities (sm_100a).
//
// A session proposes n <= K tokens x_0..x_{n-1}; the target scored them in one pass, so row k of its
// logits [K+1, V] is the distribution p_k after k drafts, and q_k is the distribution the draft came
// from (none: the draft was a plain guess, q_k(x_k) = 1). With given uniforms u in [0, 1):
//   draft k is accepted while u_k q_k(x_k) < p_k(x_k);
//   at the first one that is not, the new token is drawn from max(p_k - q_k, 0) (without q: from p_k with x_k
//   taken out); after the last draft it is drawn from p_n. The draw is the first index whose running mass
//   exceeds u_K times the whole mass, in vocabulary order.
// Accepted and drawn tokens together are then distributed exactly as the target alone would give them.
// Greedy sessions (inv_t = 0) accept a draft that is the row's first maximum and add the next maximum.
//
// p = e^((x - max) / T) / Z is held in 64 bits: the draw compares running sums over the vocabulary with one
// point, and with V = 128256 tokens of about 1e-5 each, 32-bit sums put the point into a neighbour's share
// about once in a hundred draws. NaN logits have no mass; a row without any mass accepts nothing and
// draws -1; +inf logits share the mass.
//
// Two launches:
//   stats    grid (chunk, row): one CTA reads one chunk of a row once, keeps it in registers, and writes its
//            maximum (first index) and its mass relative to that maximum. Rows past a session's drafts are
//            not read. Bound by reading the logits.
//   resolve  one cluster of 8 CTAs per session: joins the chunks of the session's rows, decides, and for the draw
//            every CTA sums its eighth of the row tile by tile; the sums meet in distributed shared memory and
//            the CTA that holds the point scans the one tile it falls into.
#include <cfloat>
#include <climits>

#include "../include/launch.h"
#include "../include/sharing.h"
#include "../include/sm100.cuh"

namespace mesh {
namespace verify {

constexpr int SNT = 256;                // threads of a stats CTA
constexpr int EPT = 32;                 // logits per thread
constexpr int CHUNK = SNT * EPT;        // logits per stats CTA
constexpr int RNT = 512;                // threads of a resolve CTA
constexpr int CLUSTER = 8;
constexpr int TILE_EPT = 8;
constexpr int TILE = RNT * TILE_EPT;    // logits per tile of the draw
constexpr int MAX_DRAFTS = VERIFY_MAX_DRAFTS;
constexpr int MAX_TILES = 256;          // tiles of one CTA's share of a row

struct Part {
  float m;    // maximum of the chunk (-inf: no selectable token)
  int idx;    // its first index
  double s;   // sum of e^((x - m) inv_t) over the chunk
};

using Args = VerifyArgs;

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }

__device__ __forceinline__ int drafts_of(const Args& a, int b) {
  return a.lens ? max(0, min(a.lens[b], a.K)) : a.K;
}

// mass of logit x in a row with maximum m (m > -inf); equal infinities count as the maximum
__device__ __forceinline__ double mass(float x, float m, double inv_t) {
  if (x == m) return 1.0;
  if (!(x > -INFINITY)) return 0.0;  // -inf or NaN
  return exp(((double)x - (double)m) * inv_t);
}

// larger value first, then the lower index
__device__ __forceinline__ void take(float& m, int& i, float om, int oi) {
  if (om > m || (om == m && oi < i)) {
    m = om;
    i = oi;
  }
}

template <typename T>
__global__ void __launch_bounds__(SNT) stats_kernel(const Args a) {
  __shared__ float red_m[SNT / 32];
  __shared__ int red_i[SNT / 32];
  __shared__ double red_s[SNT / 32];
  griddep_launch_dependents();
  griddep_wait();
  const int row = blockIdx.y, b = row / (a.K + 1), k = row - b * (a.K + 1);
  if (k > drafts_of(a, b)) return;
  const T* x = static_cast<const T*>(a.logits) + (long)b * a.ld_seq + (long)k * a.ld_row;
  const float t = a.inv_t ? a.inv_t[b] : 1.f;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int i0 = blockIdx.x * CHUNK;
  float v[EPT];
  float m = -INFINITY;
  int idx = INT_MAX;
#pragma unroll
  for (int e = 0; e < EPT; ++e) {
    const int i = i0 + e * SNT + tid;
    v[e] = i < a.V ? to_f(x[i]) : -INFINITY;
  }
#pragma unroll
  for (int e = 0; e < EPT; ++e) {
    if (v[e] > m) {
      m = v[e];
      idx = i0 + e * SNT + tid;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    take(m, idx, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, idx, o));
  if (lane == 0) {
    red_m[warp] = m;
    red_i[warp] = idx;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < SNT / 32; ++w) take(m, idx, red_m[w], red_i[w]);
  double s = 0.0;
  if (t > 0.f && m > -INFINITY) {
#pragma unroll 4
    for (int e = 0; e < EPT; ++e) s += mass(v[e], m, (double)t);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) red_s[warp] = s;
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int w = 0; w < SNT / 32; ++w) s += red_s[w];
  }
  if (tid == 0) {
    Part p;
    p.m = m;
    p.idx = idx;
    p.s = s;
    static_cast<Part*>(a.parts)[(long)row * a.chunks + blockIdx.x] = p;
  }
}

// What is drawn from: 0 p, 1 max(p - q, 0), 2 p without one token.
struct Draw {
  int mode, skip;
  float m;
  double inv_t, inv_z;
};

template <typename T, typename Q>
__device__ __forceinline__ double weight(const Draw& d, const T* x, const Q* q, int i) {
  const double p = mass(to_f(x[i]), d.m, d.inv_t) * d.inv_z;
  if (d.mode == 0) return p;
  if (d.mode == 2) return i == d.skip ? 0.0 : p;
  const float f = to_f(q[i]);
  const double r = p - (f > 0.f ? (double)f : 0.0);  // a NaN or negative q counts as none
  return r > 0.0 ? r : 0.0;
}

// sum over the CTA, the same value in every thread
__device__ __forceinline__ double block_sum(double s, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.0;
  for (int w = 0; w < RNT / 32; ++w) s += red[w];
  return s;
}

__device__ __forceinline__ double ld_dsmem_f64(uint32_t cluster_addr) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(cluster_addr) : "memory");
  return v;
}

template <typename T, typename Q>
__global__ void __launch_bounds__(RNT) resolve_kernel(const Args a) {
  __shared__ float row_m[MAX_DRAFTS + 1];
  __shared__ int row_i[MAX_DRAFTS + 1];
  __shared__ double row_z[MAX_DRAFTS + 1], row_p[MAX_DRAFTS + 1];
  __shared__ double tile_sum[MAX_TILES];
  __shared__ double red[RNT / 32];
  __shared__ double share;  // this CTA's mass of the row, read by its cluster
  __shared__ int s_n;
  const int b = blockIdx.x / CLUSTER, rank = blockIdx.x % CLUSTER;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  griddep_wait();
  griddep_launch_dependents();
  const int n = drafts_of(a, b), K = a.K;
  const float t = a.inv_t ? a.inv_t[b] : 1.f;
  const bool greedy = !(t > 0.f);
  const T* xs = static_cast<const T*>(a.logits) + (long)b * a.ld_seq;
  const Q* qs = static_cast<const Q*>(a.probs) + (a.probs ? (long)b * a.lq_seq : 0);

  // every CTA of the cluster joins the chunks of the session's rows: a warp per row
  for (int k = warp; k <= n; k += RNT / 32) {
    const Part* p = static_cast<const Part*>(a.parts) + ((long)b * (K + 1) + k) * a.chunks;
    float m = -INFINITY;
    int idx = INT_MAX;
    for (int c = lane; c < a.chunks; c += 32) take(m, idx, p[c].m, p[c].idx);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      take(m, idx, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, idx, o));
    double z = 0.0;
    if (!greedy && m > -INFINITY)
      for (int c = lane; c < a.chunks; c += 32)
        if (p[c].m > -INFINITY) z += p[c].s * mass(p[c].m, m, (double)t);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    if (lane == 0) {
      row_m[k] = m;
      row_i[k] = m > -INFINITY ? idx : -1;
      row_z[k] = z;
      double px = 0.0;
      if (k < n) {
        const int x = a.ids[(long)b * K + k];
        if (greedy)
          px = (m > -INFINITY && idx == x) ? 1.0 : 0.0;
        else if (x >= 0 && x < a.V && m > -INFINITY)
          px = mass(to_f(xs[(long)k * a.ld_row + x]), m, (double)t) / z;
      }
      row_p[k] = px;
    }
  }
  __syncthreads();
  if (tid == 0) {
    int k = 0;
    for (; k < n; ++k) {
      bool ok = row_p[k] > 0.0;
      if (ok && !greedy) {
        double qx = 1.0;
        if (a.probs) {
          const float f = to_f(qs[(long)k * a.lq_row + a.ids[(long)b * K + k]]);
          qx = f > 0.f ? (double)f : 0.0;
        }
        ok = (double)a.uniforms[(long)b * (K + 1) + k] * qx < row_p[k];
      }
      if (!ok) break;
    }
    s_n = k;
  }
  __syncthreads();
  const int acc = s_n;
  if (rank == 0) {
    for (int k = tid; k <= K; k += RNT) {
      if (k < acc)
        a.tokens[(long)b * (K + 1) + k] = a.ids[(long)b * K + k];
      else if (k > acc)
        a.tokens[(long)b * (K + 1) + k] = -1;
      if (k < K) a.draft_p[(long)b * K + k] = k < n ? (float)row_p[k] : 0.f;
    }
    if (tid == 0) a.accepted[b] = acc;
  }
  int* new_token = a.tokens + (long)b * (K + 1) + acc;
  const float m = row_m[acc];
  if (greedy || !(m > -INFINITY)) {
    if (rank == 0 && tid == 0) *new_token = row_i[acc];
    return;  // the whole cluster takes this branch
  }
  const T* x = xs + (long)acc * a.ld_row;
  const Q* q = qs + (a.probs && acc < n ? (long)acc * a.lq_row : 0);
  Draw d;
  d.m = m;
  d.inv_t = (double)t;
  d.inv_z = 1.0 / row_z[acc];
  d.skip = acc < n ? a.ids[(long)b * K + acc] : -1;
  d.mode = acc == n ? 0 : a.probs ? 1 : 2;
  const int tiles = (a.V + TILE - 1) / TILE, per = (tiles + CLUSTER - 1) / CLUSTER;
  const int t0 = min(tiles, rank * per), t1 = min(tiles, t0 + per);
  double total = 0.0, ahead = 0.0, own = 0.0;
  for (int round = 0; round < 2; ++round) {
    own = 0.0;
    for (int w = t0; w < t1; ++w) {
      double s = 0.0;
#pragma unroll
      for (int e = 0; e < TILE_EPT; ++e) {
        const int i = w * TILE + e * RNT + tid;
        if (i < a.V) s += weight(d, x, q, i);
      }
      s = block_sum(s, red);
      if (tid == 0) tile_sum[w - t0] = s;
      own += s;
    }
    if (tid == 0) share = own;
    cluster_sync();
    total = ahead = 0.0;
    for (int r = 0; r < CLUSTER; ++r) {
      const double s = ld_dsmem_f64(mapa_shared(smem_u32(&share), (uint32_t)r));
      if (r < rank) ahead += s;
      total += s;
    }
    cluster_sync();  // the shares have been read
    if (total > 0.0 || d.mode == 0) break;
    d.mode = 0;  // nothing is left of p: the draft's distribution covers it, so p itself is drawn from
  }
  // the shares' ends are the same sums in every CTA, so the point (below the whole) lies in exactly one share
  const float u = fmaxf(0.f, fminf(a.uniforms[(long)b * (K + 1) + K], 1.f - FLT_EPSILON / 2));
  const double point = (double)u * total;
  if (!(ahead <= point && point < ahead + own)) return;
  // tile, then element
  double run = ahead, before = ahead;  // mass before tile c, and before the chosen tile
  int w = t0;
  for (int c = t0; c < t1; ++c) {
    const double s = tile_sum[c - t0];
    if (s > 0.0) {  // the last tile with mass takes what the rounding of these sums leaves over
      w = c;
      before = run;
      run += s;
      if (run > point) break;
    }
  }
  __shared__ double pre[RNT];
  __shared__ int best, fallback;
  // thread t holds elements t * TILE_EPT .. of the tile, so the scan follows vocabulary order
  double mine = 0.0;
  int top = -1;
  for (int e = 0; e < TILE_EPT; ++e) {
    const int i = w * TILE + tid * TILE_EPT + e;
    if (i < a.V) {
      const double f = weight(d, x, q, i);
      mine += f;
      if (f > 0.0) top = i;
    }
  }
  if (tid == 0) {
    best = INT_MAX;
    fallback = -1;
  }
  pre[tid] = mine;
  __syncthreads();
  for (int o = 1; o < RNT; o <<= 1) {
    const double f = tid >= o ? pre[tid - o] : 0.0;
    __syncthreads();
    pre[tid] += f;
    __syncthreads();
  }
  double c = before + (tid ? pre[tid - 1] : 0.0);
  if (top >= 0) atomicMax(&fallback, top);
  for (int e = 0; e < TILE_EPT; ++e) {
    const int i = w * TILE + tid * TILE_EPT + e;
    if (i >= a.V) break;
    const double f = weight(d, x, q, i);
    c += f;
    if (f > 0.0 && c > point) {
      atomicMin(&best, i);
      break;
    }
  }
  __syncthreads();
  if (tid == 0) *new_token = best != INT_MAX ? best : fallback;
}

}  // namespace verify

int verify_chunks(int64_t V) { return (int)((V + verify::CHUNK - 1) / verify::CHUNK); }
int64_t verify_max_vocab() { return (int64_t)verify::TILE * verify::MAX_TILES * verify::CLUSTER; }
int64_t verify_parts_bytes(int64_t B, int64_t K, int64_t V) {
  return B * (K + 1) * verify_chunks(V) * (int64_t)sizeof(verify::Part);
}

cudaError_t launch_verify(const VerifyArgs& a, cudaStream_t st) {
  using namespace verify;
  const dim3 sg((unsigned)a.chunks, (unsigned)(a.B * (a.K + 1)));
  const cudaError_t e = launch_k(a.logits_bf16 ? stats_kernel<__nv_bfloat16> : stats_kernel<float>, sg, dim3(SNT), 0, st, a);
  if (e != cudaSuccess) return e;
  auto kern = a.logits_bf16 ? (a.probs_bf16 ? resolve_kernel<__nv_bfloat16, __nv_bfloat16> : resolve_kernel<__nv_bfloat16, float>)
                            : (a.probs_bf16 ? resolve_kernel<float, __nv_bfloat16> : resolve_kernel<float, float>);
  return launch_kc(kern, dim3((unsigned)(a.B * CLUSTER)), dim3(RNT), 0, st, CLUSTER, a);
}

}  // namespace mesh
