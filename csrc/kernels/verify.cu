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
//            not read. The 64-bit exponentials cost most: 64 sessions of 5 rows over 128256 tokens (164 MB of fp32) take
//            57 us (fp64 pipe 43 %, issue 64 %, DRAM 35 %); with greedy sessions, which need none, the whole call takes 29,
//            5.6 TB/s. More or fewer warps on an SM, and warps that load ahead of their exponentials, cost more.
//   resolve  one cluster of 8 CTAs per session: joins the chunks of the session's rows and decides. Drawing from p (or
//            p without one token) the chunks' masses are known and one CTA goes on: it picks the chunk, the
//            256-token unit in it, and the token. For max(p - q, 0) every CTA first sums the units of its eighth of the
//            row; the shares meet in distributed shared memory and the CTA whose share holds the point goes on.
#include <cfloat>
#include <climits>

#include "../include/launch.h"
#include "../include/sharing.h"
#include "../include/sm100.cuh"

namespace mesh {
namespace verify {

constexpr int SNT = 256;                // threads of a stats CTA
constexpr int RNT = 256;                // threads of a resolve CTA
constexpr int CLUSTER = 8;
constexpr int MAX_DRAFTS = VERIFY_MAX_DRAFTS;
// Exponentials of a thread side by side. 64 registers keep four CTAs on an SM; under them stats_kernel with 32 logits spills
// 32 to 56 bytes and resolve_kernel 24 to 124.
constexpr int STEP = 4;
constexpr int PER_LANE = 8;            // tokens of a unit per lane
constexpr int UNIT = 32 * PER_LANE;     // tokens whose sum one warp of the resolve kernel makes
constexpr int MAX_SUMS = 4096;          // chunks of a row, units of a CTA's share
// Logits per stats thread, by the CTAs that 32 each would make: 8 below two per SM, 16 below sixteen per SM, else 32, which
// spreads a CTA's fixed work over more logits. Whole calls in captured graphs, us with 8, 16 and 32 each (rows x tokens):
// 8 sessions of 5 x 4096 8.8, 9.2, 10.4; one of 5 x 128256 14.5, 14.2, 15.4; 33 of 8 x 32000 (bf16) 29.1, 26.7, 32.0;
// 64 of 5 x 32000 35.2, 28.9, 29.9; 16 of 5 x 128256 44.7, 37.3, 36.9; 64 of 5 x 128256 110, 82, 75.4, greedy 56, 34, 29.2.
constexpr int EPT_MANY = 32, EPT_SOME = 16, EPT_FEW = 8;
inline int logits_per_thread(int64_t rows, int64_t V) {
  const int64_t ctas = rows * ((V + SNT * EPT_MANY - 1) / (SNT * EPT_MANY));
  return ctas < 2 * 148 ? EPT_FEW : ctas < 16 * 148 ? EPT_SOME : EPT_MANY;
}

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

// 2^(j / 32)
__device__ const double POW2[32] = {
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.6457554781539649,
    1.681792830507429, 1.7186192981224779, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002,
};

// e^((x - m) / T) in 64 bits for one row with a finite maximum m. Reduction by a table (Tang, 1989): with
// z = (x - m) 32 / (T ln 2) = n + f, |f| <= 1/2, it is 2^(n / 32) e^(f ln2 / 32): lane j of the warp holds 2^(j / 32),
// fetched by shuffle, and a polynomial of degree 4 does the rest (its next term, (ln2 / 64)^5 / 120 = 1.2e-12, bounds
// the relative error). Eight 64-bit operations and half as many others; the loops below are bound by their issue,
// and CUDA's exp() made them four times slower. All 32 lanes of a warp must call it together.
// The exponential has to stay a normal number, so tokens below `low` = m - 700 T (masked ones, NaN) are taken
// there, and what is not well above their mass, `least()`, has none. T is taken as at most 1e30 and at least 1e-30.
struct Exp {
  double scale, top;
  float low, m;
  int hi, lo;  // of 2^(j / 32), less j in the exponent's place, so that n adds the whole exponent
  bool only;   // no logit other than m itself is within 700 T (m is infinite, or its neighbours are further): equal shares
  __device__ __forceinline__ Exp(float m_, float inv_t, double pow2) : m(m_) {
    constexpr double PER = 46.166241308446828384;  // 32 / ln 2
    inv_t = fmaxf(fminf(inv_t, 1e30f), 1e-30f);
    low = __fsub_ru(m_, 700.f / inv_t);
    only = low >= m_;
    if (only) {
      low = -700.f;
      inv_t = 1.f;
    }
    scale = (double)inv_t * PER;
    top = only ? 0.0 : (double)m_;
    hi = __double2hiint(pow2) - (int)(threadIdx.x & 31) * 32768;
    lo = __double2loint(pow2);
  }
  // this lane's entry of the table, to be asked for early
  static __device__ __forceinline__ double entry() { return POW2[threadIdx.x & 31]; }
  // what split takes for logit x
  __device__ __forceinline__ float arg(float x) const { return only ? (x == m ? 0.f : -INFINITY) : x; }
  // N logits in step, so that their chains of dependent operations overlap; the masses are w[i] * poly[i]
  template <int N>
  __device__ __forceinline__ void split(const float (&x)[N], double (&w)[N], double (&poly)[N]) const {
    constexpr double MAGIC = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is the nearest integer
    constexpr double L = 0.021660849392498290;     // ln 2 / 32
    constexpr double C2 = L * L / 2, C3 = 0x1.c6b09p-20, C4 = 0x1.3b2abp-27;  // L^3 / 6 and L^4 / 24 to 20 bits, which
    double f[N];                                   // an instruction holds itself: within 2e-14 and 2e-16 of the result
    int n[N];
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = (double)fmaxf(x[i], low) - top;
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = fma(f[i], scale, MAGIC);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      n[i] = __double2loint(w[i]);
      w[i] = MAGIC - w[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = fma(f[i], scale, w[i]);
#pragma unroll
    for (int i = 0; i < N; ++i)  // the low five bits of n choose the lane
      w[i] = __hiloint2double(__shfl_sync(0xffffffffu, hi, n[i]) + n[i] * 32768, __shfl_sync(0xffffffffu, lo, n[i]));
#pragma unroll
    for (int i = 0; i < N; ++i) poly[i] = fma(C4, f[i], C3);
#pragma unroll
    for (int i = 0; i < N; ++i) poly[i] = fma(poly[i], f[i], C2);
#pragma unroll
    for (int i = 0; i < N; ++i) poly[i] = fma(poly[i], f[i], L);
#pragma unroll
    for (int i = 0; i < N; ++i) poly[i] = fma(poly[i], f[i], 1.0);
  }
  __device__ __forceinline__ double operator()(float x) const {
    const float v[1] = {arg(x)};
    double w[1], p[1];
    split(v, w, p);
    return w[0] * p[0];
  }
  __device__ __forceinline__ double least() const {
    const float v[1] = {low};
    double w[1], p[1];
    split(v, w, p);
    return w[0] * p[0] * 1e12;  // above the sum of any chunk of masked tokens
  }
};

// sum over the warp, the same value in every lane
__device__ __forceinline__ double warp_sum(double s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// inclusive sums over the lanes
__device__ __forceinline__ double warp_scan(double s, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double f = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += f;
  }
  return s;
}

// larger value first, then the lower index
__device__ __forceinline__ void take(float& m, int& i, float om, int oi) {
  if (om > m || (om == m && oi < i)) {
    m = om;
    i = oi;
  }
}

// N consecutive elements of a row from index i on, those at or past V as -inf (q: 0). VEC: the row starts
// on a 16-byte boundary, and i is a multiple of N.
template <typename T, int N, bool VEC>
__device__ __forceinline__ void load_run(const T* x, int i, int V, float fill, float (&v)[N]) {
  constexpr int PER = 16 / sizeof(T);
  if constexpr (VEC && N % PER == 0) {
#pragma unroll
    for (int c = 0; c < N; c += PER) {
      if (i + c + PER <= V) {
        const uint4 u = *reinterpret_cast<const uint4*>(x + i + c);
        const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int j = 0; j < PER; ++j) v[c + j] = to_f(e[j]);
      } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) v[c + j] = i + c + j < V ? to_f(x[i + c + j]) : fill;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = i + j < V ? to_f(x[i + j]) : fill;
  }
}

// Logits of a chunk in a stats thread: runs of RUN elements, SNT * RUN apart. A warp takes its mass relative to its own
// maximum, so that the warps of an SM run apart, some loading while others compute; the chunk's is joined from theirs.
template <typename T, int EPT, bool VEC>
__global__ void __launch_bounds__(SNT, 4) stats_kernel(const Args a) {
  constexpr int RUN = VEC ? 16 / (int)sizeof(T) : 1;
  constexpr int CHUNK = SNT * EPT, WARPS = SNT / 32;
  __shared__ float red_m[WARPS];
  __shared__ int first;
  __shared__ double red_s[WARPS];
  const double pow2 = Exp::entry();
  griddep_wait();
  griddep_launch_dependents();
  const int row = blockIdx.y, b = row / (a.K + 1), k = row - b * (a.K + 1);
  if (k > drafts_of(a, b)) return;
  const T* x = static_cast<const T*>(a.logits) + (long)b * a.ld_seq + (long)k * a.ld_row;
  const float t = a.inv_t ? a.inv_t[b] : 1.f;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int i0 = blockIdx.x * CHUNK + tid * RUN;
  float v[EPT / RUN][RUN];
#pragma unroll
  for (int e = 0; e < EPT / RUN; ++e) load_run<T, RUN, VEC>(x, i0 + e * SNT * RUN, a.V, -INFINITY, v[e]);
  float own = -INFINITY;
#pragma unroll
  for (int e = 0; e < EPT / RUN; ++e)
#pragma unroll
    for (int j = 0; j < RUN; ++j) own = fmaxf(own, v[e][j]);
  float wm = own;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, o));
  double s = 0.0, s1 = 0.0;
  if (t > 0.f && wm > -INFINITY) {
    const Exp mass(wm, t, pow2);
    if (mass.only) {
#pragma unroll
      for (int e = 0; e < EPT / RUN; ++e)
#pragma unroll
        for (int j = 0; j < RUN; ++j) s += v[e][j] == wm ? 1.0 : 0.0;
    } else {
#pragma unroll
      for (int k = 0; k < EPT; k += STEP) {
        float x[STEP];
        double w[STEP], p[STEP];
#pragma unroll
        for (int i = 0; i < STEP; ++i) x[i] = v[(k + i) / RUN][(k + i) % RUN];
        mass.split(x, w, p);
#pragma unroll
        for (int i = 0; i < STEP; i += 2) {
          s = fma(w[i], p[i], s);
          s1 = fma(w[i + 1], p[i + 1], s1);
        }
      }
    }
    s = warp_sum(s + s1);
  }
  if (tid == 0) first = INT_MAX;
  if (lane == 0) {
    red_m[warp] = wm;
    red_s[warp] = s;
  }
  __syncthreads();
  float m = red_m[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) m = fmaxf(m, red_m[w]);
  if (own == m && m > -INFINITY) {  // few warps hold the maximum: only they look for its index
    int at = INT_MAX;
#pragma unroll
    for (int e = EPT / RUN - 1; e >= 0; --e)
#pragma unroll
      for (int j = RUN - 1; j >= 0; --j)
        if (v[e][j] == m) at = i0 + e * SNT * RUN + j;
    if (at != INT_MAX) atomicMin(&first, at);
  }
  s = 0.0;
  if (warp == 0 && t > 0.f && m > -INFINITY) {
    const Exp mass(m, t, pow2);
    const double f = mass(lane < WARPS ? red_m[lane] : -INFINITY);
    s = warp_sum(lane < WARPS ? red_s[lane] * f : 0.0);
  }
  __syncthreads();
  if (tid == 0) {
    Part p;
    p.m = m;
    p.idx = first;
    p.s = s;
    static_cast<Part*>(a.parts)[(long)row * a.chunks + blockIdx.x] = p;
  }
}

__device__ __forceinline__ double ld_dsmem_f64(uint32_t cluster_addr) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(cluster_addr) : "memory");
  return v;
}

template <typename T, typename Q, bool VEC>
__global__ void __launch_bounds__(RNT, 4) resolve_kernel(const Args a, int chunk) {
  constexpr int WARPS = RNT / 32;
  constexpr int RUN = VEC ? 16 / (int)sizeof(T) : 1;  // consecutive tokens of a lane
  __shared__ float row_m[MAX_DRAFTS + 1];
  __shared__ int row_i[MAX_DRAFTS + 1], row_x[MAX_DRAFTS + 1], row_ok[MAX_DRAFTS + 1];
  __shared__ double row_z[MAX_DRAFTS + 1], row_p[MAX_DRAFTS + 1];
  __shared__ double sums[MAX_SUMS];
  __shared__ double share;  // this CTA's mass of the row, read by its cluster
  const int b = blockIdx.x / CLUSTER, rank = blockIdx.x % CLUSTER;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int K = a.K, V = a.V;
  const double pow2 = Exp::entry();
  const T* xs = static_cast<const T*>(a.logits) + (long)b * a.ld_seq;
  const Q* qs = static_cast<const Q*>(a.probs) + (a.probs ? (long)b * a.lq_seq : 0);
  // The stats kernel lets this one start once everything before it is complete, so all inputs but its
  // partials may be read already.
  const int n = drafts_of(a, b);
  const float t = a.inv_t ? a.inv_t[b] : 1.f;
  const float u_draw = a.uniforms[(long)b * (K + 1) + K];
  const bool greedy = !(t > 0.f);
  int id = -1;
  float at_x = -INFINITY, at_q = 0.f, u = 0.f;
  auto fetch = [&](int k) {  // of the draft of row k: its token, logit, draft probability and uniform
    id = -1;
    at_x = -INFINITY;
    at_q = 0.f;
    if (k < n) {
      id = a.ids[(long)b * K + k];
      u = a.uniforms[(long)b * (K + 1) + k];
      if (id >= 0 && id < V) {
        at_x = to_f(xs[(long)k * a.ld_row + id]);
        at_q = a.probs ? to_f(qs[(long)k * a.lq_row + id]) : 1.f;
      }
    }
  };
  fetch(warp);
  griddep_wait();
  griddep_launch_dependents();

  // every CTA of the cluster joins the chunks of the session's rows: a warp per row
#pragma unroll 1
  for (int k = warp; k <= n; k += WARPS) {
    if (k != warp) fetch(k);
    const Part* p = static_cast<const Part*>(a.parts) + ((long)b * (K + 1) + k) * a.chunks;
    float m = -INFINITY;
    int idx = INT_MAX;
    for (int c = lane; c < a.chunks; c += 32) take(m, idx, p[c].m, p[c].idx);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      take(m, idx, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, idx, o));
    double z = 0.0, px = 0.0;
    if (!greedy && m > -INFINITY) {
      const Exp mass(m, t, pow2);
#pragma unroll 1
      for (int c = lane; c - lane < a.chunks; c += 32) {
        const double f = mass(c < a.chunks ? p[c].m : -INFINITY);
        if (c < a.chunks) z += p[c].s * f;
      }
      z = warp_sum(z);
      const double w = mass(at_x);
      px = w > mass.least() ? w / z : 0.0;
    } else if (greedy) {
      px = m > -INFINITY && k < n && idx == id ? 1.0 : 0.0;
    }
    if (lane == 0) {
      row_m[k] = m;
      row_i[k] = m > -INFINITY ? idx : -1;
      row_z[k] = z;
      row_x[k] = id;
      row_p[k] = px;
      row_ok[k] = k < n && px > 0.0 && (greedy || (double)u * (at_q > 0.f ? (double)at_q : 0.0) < px);
    }
  }
  __syncthreads();
  int acc = 0;
  while (acc < n && row_ok[acc]) ++acc;
  if (rank == 0) {
    for (int k = tid; k <= K; k += RNT) {
      if (k != acc) a.tokens[(long)b * (K + 1) + k] = k < acc ? row_x[k] : -1;
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
  const Part* parts = static_cast<const Part*>(a.parts) + ((long)b * (K + 1) + acc) * a.chunks;
  const Exp mass(m, t, pow2);
  const double none = mass.least();
  const double inv_z = 1.0 / row_z[acc];
  // what is drawn from: 0 p, 1 max(p - q, 0), 2 p without the token `skip`
  const int skip = acc < n ? row_x[acc] : -1;
  int mode = acc == n ? 0 : a.probs ? 1 : skip >= 0 && skip < V ? 2 : 0;
  const float u_low = fmaxf(0.f, fminf(u_draw, 1.f - FLT_EPSILON / 2));  // the point lies below the whole

  // a lane's tokens of the unit at token i0, in runs of RUN, 32 * RUN apart
  struct Raw {
    float v[PER_LANE / RUN][RUN], f[PER_LANE / RUN][RUN];
  };
  auto fetch_unit = [&](int i0, int end, Raw& r) {
#pragma unroll
    for (int e = 0; e < PER_LANE / RUN; ++e) {
      const int i = i0 + (e * 32 + lane) * RUN;
      load_run<T, RUN, VEC>(x, i, end, -INFINITY, r.v[e]);
      if (mode == 1) load_run<Q, RUN, VEC>(q, i, end, 0.f, r.f[e]);
    }
  };
  // the shares of STEP tokens of a lane, from its k-th of the unit on
  auto weights = [&](const Raw& r, int i0, int k, double (&p)[STEP]) {
    float x[STEP];
    double w[STEP];
#pragma unroll
    for (int i = 0; i < STEP; ++i) x[i] = mass.arg(r.v[(k + i) / RUN][(k + i) % RUN]);
    mass.split(x, w, p);
#pragma unroll
    for (int i = 0; i < STEP; ++i) {
      const int e = (k + i) / RUN, j = (k + i) % RUN;
      p[i] *= w[i];
      if (mode == 1) {
        p[i] = fma(p[i], inv_z, -(double)fmaxf(r.f[e][j], 0.f));  // a NaN or negative q counts as none
      } else {
        p[i] *= inv_z;
        if (mode == 2 && i0 + (e * 32 + lane) * RUN + j == skip) p[i] = 0.0;
      }
      p[i] = p[i] > none ? p[i] : 0.0;
    }
  };
  // sums[] of the units of [i0, end): a warp each, the next unit's loads in flight under this one's exponentials
  auto unit_sums = [&](int i0, int end) {
    Raw r, next;
    int i = i0 + warp * UNIT;
    if (i < end) fetch_unit(i, end, r);
#pragma unroll 1
    for (; i < end; i += WARPS * UNIT) {
      if (i + WARPS * UNIT < end) fetch_unit(i + WARPS * UNIT, end, next);
      double s = 0.0;
#pragma unroll
      for (int k = 0; k < PER_LANE; k += STEP) {
        double p[STEP];
        weights(r, i, k, p);
#pragma unroll
        for (int i = 0; i < STEP; ++i) s += p[i];
      }
      s = warp_sum(s);
      if (lane == 0) sums[(i - i0) / UNIT] = s;
      r = next;
    }
    __syncthreads();
  };
  // Over sums[0, n), 32 at a time: the running sum from `run` on. choose: the entry that holds the point, `run` = the
  // mass before it; the last one with mass takes what the rounding of the sums leaves over.
  auto total_of = [&](int n_sums) {
    double run = 0.0;
    for (int c = 0; c < n_sums; c += 32) run += warp_sum(c + lane < n_sums ? sums[c + lane] : 0.0);
    return run;
  };
  auto choose = [&](int n_sums, double point, double& run) {
    int at = -1;
    double before = run;
    for (int c = 0; c < n_sums; c += 32) {
      const double s = c + lane < n_sums ? sums[c + lane] : 0.0;
      const double incl = warp_scan(s, lane), ahead = run + (incl - s);
      const unsigned some = __ballot_sync(0xffffffffu, s > 0.0);
      const unsigned hit = __ballot_sync(0xffffffffu, s > 0.0 && run + incl > point);
      if (some) {
        const int l = hit ? __ffs(hit) - 1 : 31 - __clz(some);
        at = c + l;
        before = __shfl_sync(0xffffffffu, ahead, l);
        if (hit) break;
      }
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    run = before;
    return at;
  };

  double before = 0.0, point = 0.0;
  int i0 = 0, end = 0;  // tokens whose unit sums are in sums[]
  if (mode == 1) {
    const int units = (V + UNIT - 1) / UNIT, per = (units + CLUSTER - 1) / CLUSTER;
    i0 = min(V, rank * per * UNIT);
    end = min(V, i0 + per * UNIT);
    unit_sums(i0, end);
    const double own = total_of((end - i0 + UNIT - 1) / UNIT);
    double total = 0.0;
    if (tid == 0) share = own;
    cluster_sync();
#pragma unroll
    for (int r = 0; r < CLUSTER; ++r) {
      const double s = ld_dsmem_f64(mapa_shared(smem_u32(&share), (uint32_t)r));
      if (r < rank) before += s;
      total += s;
    }
    cluster_sync();  // the shares have been read
    point = (double)u_low * total;
    if (!(total > 0.0))
      mode = 0;  // nothing is left of p: the draft's distribution covers it, so p itself is drawn from
    else if (!(before <= point && point < before + own))
      return;  // the shares' ends are the same sums in every CTA: the point lies in exactly one share
  }
  if (mode != 1) {
    if (rank != 0) return;
    double without = 0.0;
    if (mode == 2) {
      // the chunk that holds the token left out is summed again without it
      i0 = skip / chunk * chunk;
      end = min(V, i0 + chunk);
      unit_sums(i0, end);
      without = total_of((end - i0 + UNIT - 1) / UNIT);
      __syncthreads();
    }
#pragma unroll 1
    for (int c = warp * 32; c < a.chunks; c += RNT) {
      const int e = c + lane;
      const double f = mass(e < a.chunks ? parts[e].m : -INFINITY);
      if (e < a.chunks) {
        const double s = mode == 2 && e == skip / chunk ? without : parts[e].s * f * inv_z;
        sums[e] = s > none ? s : 0.0;
      }
    }
    __syncthreads();
    const double total = total_of(a.chunks);
    if (mode == 2 && !(total > 0.0)) {  // the token left out had all the mass: it is drawn after all
      if (tid == 0) *new_token = skip;
      return;
    }
    point = (double)u_low * total;
    before = 0.0;
    const int c = choose(a.chunks, point, before);
    __syncthreads();
    i0 = max(c, 0) * chunk;
    end = min(V, i0 + chunk);
    unit_sums(i0, end);
  }
  const int n_units = (end - i0 + UNIT - 1) / UNIT;
  const int y = choose(n_units, point, before);
  if (warp != 0) return;
  i0 += max(y, 0) * UNIT;
  Raw r;
  fetch_unit(i0, end, r);
  int last = -1;
  double all[PER_LANE];
#pragma unroll
  for (int k = 0; k < PER_LANE; k += STEP) {
    double p[STEP];
    weights(r, i0, k, p);
#pragma unroll
    for (int i = 0; i < STEP; ++i) all[k + i] = p[i];
  }
#pragma unroll
  for (int e = 0; e < PER_LANE / RUN; ++e) {  // the runs of step e lie before those of step e + 1
    double w[RUN], mine = 0.0;
#pragma unroll
    for (int j = 0; j < RUN; ++j) {
      w[j] = all[e * RUN + j];
      mine += w[j];
    }
    const double incl = warp_scan(mine, lane);
    double c = before + (incl - mine);
    int hit = INT_MAX;
#pragma unroll
    for (int j = 0; j < RUN; ++j) {
      c += w[j];
      if (w[j] > 0.0) {
        last = i0 + (e * 32 + lane) * RUN + j;
        if (c > point && hit == INT_MAX) hit = last;
      }
    }
    hit = __reduce_min_sync(0xffffffffu, hit);
    if (hit != INT_MAX) {
      if (lane == 0) *new_token = hit;
      return;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  last = __reduce_max_sync(0xffffffffu, last);
  if (lane == 0) *new_token = last;
}

// 16-byte loads where every row of both operands starts on a 16-byte boundary
bool vectors(const VerifyArgs& a) {
  auto ok = [](const void* p, long ld_row, long ld_seq, int size) {
    return (uintptr_t)p % 16 == 0 && ld_row * size % 16 == 0 && ld_seq * size % 16 == 0;
  };
  return ok(a.logits, a.ld_row, a.ld_seq, a.logits_bf16 ? 2 : 4) &&
         (!a.probs || ok(a.probs, a.lq_row, a.lq_seq, a.probs_bf16 ? 2 : 4));
}

template <typename T, typename Q, int EPT, bool VEC>
cudaError_t launch(const VerifyArgs& a, cudaStream_t st) {
  const cudaError_t e =
      launch_k(stats_kernel<T, EPT, VEC>, dim3((unsigned)a.chunks, (unsigned)(a.B * (a.K + 1))), dim3(SNT), 0, st, a);
  if (e != cudaSuccess) return e;
  return launch_kc(resolve_kernel<T, Q, VEC>, dim3((unsigned)(a.B * CLUSTER)), dim3(RNT), 0, st, CLUSTER, a, SNT * EPT);
}

template <typename T, typename Q, bool VEC>
cudaError_t pick(const VerifyArgs& a, cudaStream_t st) {
  switch (logits_per_thread((int64_t)a.B * (a.K + 1), a.V)) {
    case EPT_FEW: return launch<T, Q, EPT_FEW, VEC>(a, st);
    case EPT_SOME: return launch<T, Q, EPT_SOME, VEC>(a, st);
    default: return launch<T, Q, EPT_MANY, VEC>(a, st);
  }
}

template <typename T, typename Q>
cudaError_t pick(const VerifyArgs& a, cudaStream_t st) {
  return vectors(a) ? pick<T, Q, true>(a, st) : pick<T, Q, false>(a, st);
}

}  // namespace verify

int verify_chunks(int64_t B, int64_t K, int64_t V) {
  const int64_t c = verify::SNT * verify::logits_per_thread(B * (K + 1), V);
  return (int)((V + c - 1) / c);
}
int64_t verify_max_vocab() { return (int64_t)verify::SNT * verify::EPT_FEW * verify::MAX_SUMS; }
int64_t verify_parts_bytes(int64_t B, int64_t K, int64_t V) {
  return B * (K + 1) * verify_chunks(B, K, V) * (int64_t)sizeof(verify::Part);
}

cudaError_t launch_verify(const VerifyArgs& a, cudaStream_t st) {
  using namespace verify;
  using bf = __nv_bfloat16;
  if (a.logits_bf16) return a.probs_bf16 ? pick<bf, bf>(a, st) : pick<bf, float>(a, st);
  return a.probs_bf16 ? pick<float, bf>(a, st) : pick<float, float>(a, st);
}

}  // namespace mesh
