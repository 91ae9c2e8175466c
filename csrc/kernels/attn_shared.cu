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
// are summed in a fixed order, so results do not depend on the schedule. NaN in a row's query or in a key it attends makes
// the row NaN however its keys are cut: its sums l are NaN, and only a sum of exactly 0 counts as nothing seen.
//
// Measured (32 query and 8 KV heads of 128): 64 sessions with up to 512 keys of their own behind 8192 shared ones 36.5 us, of
// which reading every key once takes 15.8 at the copy rate; 128 with up to 1024 behind 16384 94 us (52.5); 4 forks of 512
// keys 10.9 us in a captured graph. About 19 us of the large calls do not depend on the shared keys (64 sessions with one key of their
// own, captured: 20.0 us with 64 shared keys for every SM, 27.5 with 512, 53.4 with 2048): first queries and pages (5), partials
// written (3: 256 rows x 128 fp32 from every SM) and merged (5), and three kernels following one another.
//
// The item list is made on the host when the groups change (PrefixGroups) and lives in device memory, so a
// captured step follows later changes of groups, lengths and tables.
#include <type_traits>

#include "attn_shared.cuh"

namespace mesh {
namespace shared_attn {
namespace {

constexpr int WARPS = 4;         // workers of a CTA
// CTAs per SM. Nothing shared: two (64 KB of rings in flight each; 64 sessions of up to 512 keys 19.9 us, one 26.9,
// three 23.3; 128 of up to 2048 keys 99.3, 141, 100).
// Beside the prefix kernel one CTA finds room at a time. Up to LIGHT units an SM one is also the faster: more cut the
// keys into more partials (16 sessions of up to 512 own keys behind 2048 16.1 us, three 20.9; 64 behind 8192, 69 units,
// 36.4 and 36.9). With more to do, those that start when the prefix kernel's leave read the rest faster (96 behind 8192,
// 98 units, 46.9 with one and 45.2 with three; 64 of up to 2048 behind 2048 67.4 and 59.4; 256 of them 274 and 204).
// The lengths are known here, not on the host: three are launched, and two leave at once where one is to do it all,
// which costs less than the timing shows.
constexpr int CTAS_ALONE = 2, CTAS_SHARED = 3, LIGHT = 80;
static_assert(CTAS_SHARED * WARPS <= SHARED_OWN_WORKERS, "partials are reserved for fewer workers");
constexpr int TILE_ROWS = SHARED_OWN_ROWS;
constexpr int PIECE_COST = 2;    // what a piece costs besides its slices, in slices
constexpr int MIN_QUOTA = 4;     // units (slices and piece costs) a worker takes at least

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
// transpose of an 8 x 8 matrix of 16-bit values held by the warp
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// byte offset of (row, 16-byte chunk) inside a [16 x 64] box written with the 128-byte swizzle
__device__ __forceinline__ uint32_t swz(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

template <int D>
struct Geo {
  static constexpr int HALVES = D / 64;
  static constexpr uint32_t BOX = SLICE * 64 * 2;           // one [16 x 64] box
  static constexpr uint32_t SLICE_BYTES = 2 * HALVES * BOX; // K halves then V halves
  static constexpr int SLOTS = 16 * 1024 / SLICE_BYTES;     // slices in flight per worker: 64 KB per CTA
  // rings | what is known of each sequence
  static size_t smem(int B) { return 1024 + WARPS * SLOTS * SLICE_BYTES + 16 * (B + 1); }
};

// A sequence's keys behind its shared prefix (and inside the window).
struct Seq {
  int before;  // units of the sequences before it, for one KV head and tile of rows
  int first;   // first key
  int L;       // end
  int slots;   // partials of its shared prefix per row
  __device__ __forceinline__ int slices() const { return L > first ? (L + SLICE - 1) / SLICE - first / SLICE : 0; }
};

// A value that is the same in all lanes, known to be so (it may live in a uniform register)
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ int uniform_at(int v, int lane) { return __shfl_sync(0xffffffffu, v, lane); }

// All sequences by the WARPS * 32 threads of the workers (tid among them), with the running number of units; seqs [B + 1].
// The loads of all sequences are in flight at once; `sync` is a barrier of these threads.
template <typename Sync>
__device__ __forceinline__ void own_sequences(const Args& a, Seq* seqs, int tid, Sync sync) {
  for (int b = tid; b < a.B; b += WARPS * 32) {
    Seq q;
    q.L = min(a.seq_lens[b], a.max_pages * a.page_size);
    q.first = seq_prefix(a, b);
    q.slots = seq_prefix_slots(a, b);
    if (a.window > 0) q.first = max(q.first, q.L - a.T + 1 - a.window);
    const int n = q.slices();
    q.before = n > 0 ? n + PIECE_COST : 0;
    seqs[b] = q;
  }
  sync();
  if (tid < 32) {
    int run = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      const int b = b0 + tid, n = b < a.B ? seqs[b].before : 0;
      int v = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int w = __shfl_up_sync(0xffffffffu, v, o);
        if (tid >= o) v += w;
      }
      if (b < a.B) seqs[b].before = run + v - n;
      run += __shfl_sync(0xffffffffu, v, 31);
    }
    if (tid == 0) seqs[a.B].before = run;
  }
  sync();
}

// The keys behind the shared prefixes: 8 rows (new tokens x heads of a KV group) of one sequence against that sequence's
// own slices of 16 keys. All of them, in the order (sequence, KV head, tile of rows, slice), are cut into equal quotas,
// one per warp: lengths from one token to long ones then keep every SM as busy. A quota is a run of
// pieces, one for each (sequence, head, tile) it touches; a piece counts as PIECE_COST slices besides its own, about
// what loading its queries and writing its result take. Piece number = worker + (sequence, head, tile), which no other
// piece has. A warp works by itself: it requests slices SLOTS ahead (TMA, 128-byte swizzle), without a barrier between
// warps; four warps that split each piece and merged it took twice as long (64 sessions of up to 512 keys). Bound by
// reading K and V: 128 sessions of up to 1024 keys, 269 MB, take 51.7 us (5.2 TB/s, 0.81 of a copy). Leaving out the rescale and
// the masks where a slice needs neither changed nothing.
// The products run transposed, S^T = K Q^T and O^T = V^T P^T on m16n8k16 fragments, so that the few query rows are the
// narrow side. With the rows on the 16-wide side half of every product and of the accumulators would be padding (168
// registers, so no CTA fitted beside the prefix kernel's). More than 8 rows are cut into tiles, each reading the keys
// again, mostly from L2: one worker for two tiles needs those registers too and was slower at every size (20 rows, 16
// sessions, 8192 shared keys: 46.9 us, tiles 41.9; 16 rows, 64 sessions of 512 keys 36.3 and 31.1).
template <int D>
__device__ __forceinline__ void own_worker(const CUtensorMap& tmK, const CUtensorMap& tmV, const Args& a, const Seq* seqs,
                                           uint8_t* ring, uint64_t* full, int lane, int worker, int workers) {
  using g = Geo<D>;
  constexpr int SLOTS = g::SLOTS;
  const int rows = a.T * a.G, hq = a.hkv * a.G, tiles = (rows + TILE_ROWS - 1) / TILE_ROWS;
  const int per_seq = a.hkv * tiles;
  const int total = seqs[a.B].before * per_seq;
  const int quota = max(MIN_QUOTA, (total + workers - 1) / workers);
  if (worker == 0) {  // for the combine kernel
    for (int b = lane; b <= a.B; b += 32) own_before(a)[b] = seqs[b].before;
    if (lane == 0) own_before(a)[a.B + 1] = quota;
  }
  const int lo = uniform(min(total, worker * quota)), hi = uniform(min(total, lo + quota));

  // a walk over the pieces of [lo, hi)
  struct Piece {
    int b, u, pos;  // sequence; its (KV head, tile); unit the piece starts at
    int sl, n;      // first slice of the own ones, slices
  };
  auto fit = [&](Piece& p, int r) {  // r: units of (b, u) before pos
    const int units = seqs[p.b + 1].before - seqs[p.b].before;
    const int end = min(units, r + hi - p.pos);
    p.sl = max(r, PIECE_COST) - PIECE_COST;
    p.n = max(0, end - PIECE_COST - p.sl);
    p.pos += end - r;  // where the next piece starts
  };
  auto begin = [&](Piece& p) {
    int x = 0, y = a.B - 1;  // last sequence that starts at or before lo
    while (x < y) {
      const int mid = (x + y + 1) >> 1;
      if (seqs[mid].before * per_seq <= lo)
        x = mid;
      else
        y = mid - 1;
    }
    const int units = seqs[x + 1].before - seqs[x].before, off = lo - seqs[x].before * per_seq;
    p.b = x;
    p.u = off / units;
    p.pos = lo;
    fit(p, off - p.u * units);
  };
  auto next = [&](Piece& p) {  // false behind the last piece
    do {
      if (p.pos >= hi) return false;
      if (++p.u == per_seq) {
        p.u = 0;
        do ++p.b;
        while (seqs[p.b + 1].before == seqs[p.b].before);
      }
      fit(p, 0);
    } while (p.n == 0);
    return true;
  };

  if (lo < hi) {
    const uint64_t pol = policy_evict_first();
    // ---- requests: slice ri of the walk's current piece goes to slot rs
    Piece rp, np;  // the piece being requested, the one behind it
    begin(rp);
    bool more = uniform(rp.n > 0 || next(rp)), more2;
    int ri = 0, rs = 0, page = 0, next_page = 0;
    // page that holds slice i0 + lane of a piece; nothing is computed from it here, so the load stays in flight
    auto look_up = [&](const Piece& x, int i0) {
      const int sl = seqs[x.b].first / SLICE + x.sl + i0 + lane;
      return i0 + lane < x.n ? a.block_tables[(long)x.b * a.max_pages + sl / a.slices_per_page] : 0;
    };
    auto look_ahead = [&]() {  // the next piece's first pages are read long before they are needed
      np = rp;
      more2 = uniform(more && next(np));
      if (more2) next_page = look_up(np, 0);
    };
    if (more) page = look_up(rp, 0);
    look_ahead();
    auto request = [&]() {
      if (!more) return;
      const int sl = seqs[rp.b].first / SLICE + rp.sl + ri;
      const int y = uniform((uniform_at(page, ri & 31) * a.hkv + rp.u / tiles) * a.page_size + sl % a.slices_per_page * SLICE);
      if (elect_one()) {
        mbar_arrive_expect_tx(&full[rs], g::SLICE_BYTES);
        uint8_t* dst = ring + rs * g::SLICE_BYTES;
        // both 64-column halves of the 16 rows in one box each of K and V
        if constexpr (g::HALVES == 2) {
          tma_load_3d(dst, &tmK, &full[rs], 0, y, 0, pol);
          tma_load_3d(dst + 2 * g::BOX, &tmV, &full[rs], 0, y, 0, pol);
        } else {
          tma_load_2d(dst, &tmK, &full[rs], 0, y, pol);
          tma_load_2d(dst + g::BOX, &tmV, &full[rs], 0, y, pol);
        }
      }
      __syncwarp();
      if (++rs == SLOTS) rs = 0;
      if (++ri == uniform(rp.n)) {
        ri = 0;
        rp = np;
        page = next_page;
        more = more2;
        look_ahead();
      } else if ((ri & 31) == 0) {
        page = look_up(rp, ri);
      }
    };
#pragma unroll 1
    for (int i = 0; i < SLOTS; ++i) request();

    Piece p;
    begin(p);
    bool todo = p.n > 0 || next(p), ok = true;
    int s = 0;
    uint32_t ph = 0;
    for (; todo; todo = next(p)) {
      const Seq q = seqs[p.b];
      const int h = p.u / tiles, row0 = (p.u - h * tiles) * TILE_ROWS, n_rows = min(TILE_ROWS, rows - row0);
      const int s0 = q.first / SLICE + p.sl;
      const int k0 = max(q.first, s0 * SLICE), k1 = min(q.L, (s0 + p.n) * SLICE);
      // query fragments straight from memory: row lane / 4, columns (lane % 4) * 2 and 8 to the right
      uint32_t qf[D / 16][2];
      const int r = lane >> 2, x = row0 + min(r, n_rows - 1), t = x / a.G;
      const __nv_bfloat16* src = a.q + ((long)(p.b * a.T + t) * hq + h * a.G + x - t * a.G) * D + (lane & 3) * 2;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qf[kk][0] = r < n_rows ? *reinterpret_cast<const uint32_t*>(src + kk * 16) : 0u;
        qf[kk][1] = r < n_rows ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + 8) : 0u;
      }
      int hi_k[2], lo_k[2];  // keys that this lane's rows (lane % 4) * 2 + i may attend: [lo_k, hi_k)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = (lane & 3) * 2 + i, pos = q.L - a.T + (row0 + r) / a.G;
        hi_k[i] = r < n_rows ? min(k1, pos + 1) : 0;
        lo_k[i] = a.window > 0 ? max(k0, pos + 1 - a.window) : k0;
      }
      float o[D / 16][4];  // [16 columns of the head]: columns lane / 4 and 8 below, rows (lane % 4) * 2 + {0, 1}
      float m[2], l[2];
#pragma unroll
      for (int x = 0; x < D / 16; ++x) o[x][0] = o[x][1] = o[x][2] = o[x][3] = 0.f;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
#pragma unroll 1
      for (int i = 0; i < p.n; ++i) {
        ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded(&full[s], ph, a.err, ERR_MBAR_TIMEOUT_MMA, nullptr, WAIT_NS));
        if (!ok) break;
        const int key0 = (s0 + i) * SLICE;
        const uint32_t kb = smem_u32(ring + s * g::SLICE_BYTES), vb = kb + g::HALVES * g::BOX;
        // Keys past the range may hold anything (a page's unused tail), and so may those before it (this sequence's own
        // copy of a prefix that ends inside the slice): their values must not reach the products as NaN or infinity times
        // a zero weight. Clearing them in the fragments costs two masks; clearing them in shared memory needs a proxy
        // fence, which waited for the loads in flight.
        uint32_t keep[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int key = key0 + x * 8 + (lane & 3) * 2, left = k1 - key;  // the first of this lane's two keys
          keep[x] = left >= 2 ? 0xffffffffu : left == 1 ? 0xffffu : 0u;
          if (key < k0) keep[x] &= key + 1 < k0 ? 0u : 0xffff0000u;
        }
        float sc[4], sd[4];  // keys lane / 4 and 8 below; two chains of products each
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[e] = sd[e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t kf[4];
          ldsm_x4(kb + (kk >> 2) * g::BOX + swz((lane & 7) + ((lane >> 3) & 1) * 8, (kk & 3) * 2 + (lane >> 4)), kf);
          mma((kk & 1) ? sd : sc, kf, qf[kk][0], qf[kk][1]);
        }
        uint32_t pf[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int key = key0 + (lane >> 2);
          const bool in0 = key < hi_k[i] && key >= lo_k[i], in1 = key + 8 < hi_k[i] && key + 8 >= lo_k[i];
          const float s0v = in0 ? (sc[i] + sd[i]) * a.scale_log2 : -INFINITY;
          const float s1v = in1 ? (sc[2 + i] + sd[2 + i]) * a.scale_log2 : -INFINITY;
          float mx = fmaxf(s0v, s1v);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
          const float mn = fmaxf(m[i], mx), mb = mn == -INFINITY ? 0.f : mn;
          const float corr = ex2_ftz(m[i] - mb);
          sc[i] = ex2_ftz(s0v - mb);
          sc[2 + i] = ex2_ftz(s1v - mb);
          l[i] = l[i] * corr + (sc[i] + sc[2 + i]);
          m[i] = mn;
#pragma unroll
          for (int x = 0; x < D / 16; ++x) {
            o[x][i] *= corr;
            o[x][2 + i] *= corr;
          }
        }
        // The weights are rounded to bf16 for the product (half a step of 2^-8 each), whose operands are of one type; their
        // sum keeps fp32.
        pf[0] = transposed(pack_bf16x2(sc[0], sc[1]));
        pf[1] = transposed(pack_bf16x2(sc[2], sc[3]));
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {
          uint32_t vf[4];
          ldsm_x4_t(vb + (x >> 2) * g::BOX + swz((lane & 7) + (lane >> 4) * 8, (x & 3) * 2 + ((lane >> 3) & 1)), vf);
          vf[0] &= keep[0];
          vf[1] &= keep[0];
          vf[2] &= keep[1];
          vf[3] &= keep[1];
          mma(o[x], vf, pf[0], pf[1]);
        }
        // the products above have taken every fragment of this slot, so it may be filled again
        __syncwarp();
        request();
        if (++s == SLOTS) {
          s = 0;
          ph ^= 1;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
      // a sequence without a prefix whose keys are all in this piece is done: its rows go out; else a partial
      const bool whole = p.n == q.slices() && q.slots == 0;
      const int stride = min(rows, TILE_ROWS);
      const long part = a.own_at + (long)(worker + p.b * per_seq + p.u) * stride;
      if (part + stride > a.slot_cap) {
        if (lane == 0) record_error(a.err, ERR_BAD_ARGUMENT);
        continue;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = (lane & 3) * 2 + i;
        if (r >= n_rows) continue;
        const int x0 = row0 + r, t = x0 / a.G;
        __nv_bfloat16* out = a.out + ((long)(p.b * a.T + t) * hq + h * a.G + x0 - t * a.G) * D + (lane >> 2);
        float* po = a.po + (part + r) * D + (lane >> 2);
        const float inv = 1.f / l[i];  // a NaN sum stays one; rows without a key give zeros whatever the values hold
#pragma unroll
        for (int x = 0; x < D / 16; ++x)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (whole)
              out[x * 16 + e * 8] = f2bf(l[i] == 0.f ? 0.f : o[x][2 * e + i] * inv);
            else
              po[x * 16 + e * 8] = o[x][2 * e + i];
          }
        if (!whole && lane < 4) a.pml[part + r] = make_float2(m[i], l[i]);
      }
    }
    if (!ok) {
      // the copies still in flight land before the warp goes (bounded)
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 50000000ull) {
      }
    }
  }
}

// 128 registers a thread, so that a CTA fits beside one of the prefix kernel; nothing is spilled.
template <int D>
__global__ void __launch_bounds__(WARPS * 32, 4) own_kernel(const __grid_constant__ CUtensorMap tmK,
                                                            const __grid_constant__ CUtensorMap tmV, const Args a) {
  using g = Geo<D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Seq* seqs = reinterpret_cast<Seq*>(base + WARPS * g::SLOTS * g::SLICE_BYTES);  // [B + 1]
  __shared__ uint64_t bars[WARPS][g::SLOTS];
  if (threadIdx.x == 0) {
    for (int i = 0; i < WARPS * g::SLOTS; ++i) mbar_init(&bars[0][0] + i, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  griddep_launch_dependents();
  // behind a prefix kernel, whose own inputs are complete when it lets this one start, only the end has to wait
  if (a.n_prefix == 0) griddep_wait();
  own_sequences(a, seqs, threadIdx.x, [] { __syncthreads(); });
  const int tiles = (a.T * a.G + TILE_ROWS - 1) / TILE_ROWS;
  const bool light = a.n_prefix != 0 && (long)seqs[a.B].before * a.hkv * tiles < (long)a.num_sms * LIGHT;
  const int ctas = light ? a.num_sms : (int)gridDim.x;
  // few workers spread over the SMs
  if ((int)blockIdx.x < ctas)
    own_worker<D>(tmK, tmV, a, seqs, base + warp * g::SLOTS * g::SLICE_BYTES, bars[warp], lane,
                  warp * ctas + (int)blockIdx.x, WARPS * ctas);
  // this grid is complete only when the prefix grid is; one CTA sees to that, the others make room for the next
  if (a.n_prefix != 0 && blockIdx.x == gridDim.x - 1) griddep_wait();
}

// One warp per row (sequence, token, head): merge its partials, the prefix's first, in order. Bound by latency, not by the
// bytes (5 us for 16.8 MB of partials, all in L2): lane i asks for the (m, l) of partial i and the warp for its first eight
// outputs at once, those of the prefix before it is known which workers had the rest; weights follow. With sixteen at once
// (128 registers instead of 80, fewer warps on an SM) up to 64 sessions gain 0.4 us and 256 lose 2.5.
template <int D>
__global__ void __launch_bounds__(128) combine_kernel(const Args a) {
  constexpr int V = D / 32, U = 8, U_OWN = 2;
  using Vec = typename std::conditional<V == 4, float4, float2>::type;
  const int lane = threadIdx.x & 31, hq = a.hkv * a.G, rows = a.T * a.G;
  const int row = blockIdx.x * 4 + (threadIdx.x >> 5);  // (b * T + t) * hq + head
  const int b = min(row / (a.T * hq), a.B - 1);
  const int x = row - b * a.T * hq, t = x / hq, head = x - t * hq, h = head / a.G;
  // written by the host alone, not by a kernel that this grid may overlap
  int n_prefix = seq_prefix_slots(a, b);
  const int base = seq_base(a, b) + x * n_prefix;
  const bool bad = base < 0 || base + n_prefix > a.own_at;
  if (bad) n_prefix = 0;
  griddep_wait();
  griddep_launch_dependents();
  if (row >= a.B * a.T * hq) return;
  const int before = own_before(a)[b], after = own_before(a)[b + 1], quota = own_before(a)[a.B + 1];
  float acc[V] = {}, den = 0.f, M = -INFINITY;
  auto stats = [&](long first, long step, int n, int i) {
    return i + lane < n ? a.pml[first + (i + lane) * step] : make_float2(-INFINITY, 0.f);
  };
  auto load = [&](long first, long step, int n, int i, auto& p) {
#pragma unroll
    for (int k = 0; k < (int)(sizeof(p) / sizeof(p[0])); ++k)
      if (i + k < n) *reinterpret_cast<Vec*>(p[k]) = *reinterpret_cast<const Vec*>(a.po + (first + (i + k) * step) * D + lane * V);
  };
  // n partials, `step` apart; ml and p: the first of them, already on their way
  auto merge = [&](long first, long step, int n, float2 ml, auto& p) {
    constexpr int N = (int)(sizeof(p) / sizeof(p[0]));
    for (int i0 = 0; i0 < n; i0 += 32) {
      if (i0 > 0) ml = stats(first, step, n, i0);
      float mx = ml.x;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float mn = fmaxf(M, mx), mb = mn == -INFINITY ? 0.f : mn;
      // 0 where nothing was seen: m is -inf and l is 0, or NaN where every score was one, which then stays in the sum
      const float corr = ex2_ftz(M - mb), e = ex2_ftz(ml.x - mb);
      const float f = ml.y == 0.f ? -1.f : e;  // the output of a partial that saw nothing may not have been written
      M = mn;
      den = den * corr + ml.y * e;
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] *= corr;
      for (int i = i0; i < min(n, i0 + 32); i += N) {
        if (i > 0) load(first, step, n, i, p);
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const float w = __shfl_sync(0xffffffffu, f, (i + k) & 31);
          if (i + k < n && w >= 0.f)
#pragma unroll
            for (int v = 0; v < V; ++v) acc[v] = fmaf(p[k][v], w, acc[v]);
        }
      }
    }
  };
  float p[U][V];
  float2 ml = stats(base, 1, n_prefix, 0);
  load(base, 1, n_prefix, 0, p);
  // the workers whose quotas this row's slices fall into
  const int units = after - before, r = t * a.G + (head - h * a.G);
  const int tile = r / TILE_ROWS, tiles = (rows + TILE_ROWS - 1) / TILE_ROWS, u = h * tiles + tile, stride = min(rows, TILE_ROWS);
  const int at = before * a.hkv * tiles + u * units + PIECE_COST;  // its first slice
  const int w0 = at / quota;
  int n_own = units > 0 ? (at + units - PIECE_COST - 1) / quota - w0 + 1 : 0;
  if (n_prefix == 0 && n_own == 1 && !bad) return;  // already written
  const long own = a.own_at + (long)(w0 + b * a.hkv * tiles + u) * stride + (r - tile * TILE_ROWS);  // pieces are `stride` apart
  if (bad || (n_own > 0 && own + (long)(n_own - 1) * stride >= a.slot_cap)) {
    if (lane == 0) record_error(a.err, ERR_BAD_ARGUMENT);
    n_own = 0;
  }
  if (n_prefix > 0) {
    float p_own[U_OWN][V];
    const float2 ml_own = stats(own, stride, n_own, 0);
    load(own, stride, n_own, 0, p_own);
    merge(base, 1, n_prefix, ml, p);
    merge(own, stride, n_own, ml_own, p_own);
  } else {
    ml = stats(own, stride, n_own, 0);
    load(own, stride, n_own, 0, p);
    merge(own, stride, n_own, ml, p);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
  const float inv = den == 0.f ? 0.f : 1.f / den;
  __nv_bfloat16* dst = a.out + (long)row * D + lane * V;
#pragma unroll
  for (int v = 0; v < V; v += 2) *reinterpret_cast<uint32_t*>(dst + v) = pack_bf16x2(acc[v] * inv, acc[v + 1] * inv);
}

}  // namespace

template <int D>
static cudaError_t launch(const Args& a, cudaStream_t st) {
  const uint64_t rows = (uint64_t)a.pool_pages * a.hkv * a.page_size;
  CUtensorMap tk, tv, ok, ov;
  if (a.n_prefix > 0 || D == 64) {
    tk = tma_map_2d_bf16(a.k, D, rows, D, 64, SLICE);
    tv = tma_map_2d_bf16(a.v, D, rows, D, 64, SLICE);
  }
  if (D == 128) {  // a slice of 128 columns in one box: two halves of 64 columns, 16 rows each
    ok = tma_map_3d_bf16(a.k, 64, rows, 2, D * 2, 128, 64, SLICE, 2);
    ov = tma_map_3d_bf16(a.v, 64, rows, 2, D * 2, 128, 64, SLICE, 2);
  } else {
    ok = tk;
    ov = tv;
  }
  cudaError_t e = cudaSuccess;
  if (a.n_prefix > 0 && (e = launch_prefix<D>(a, tk, tv, st)) != cudaSuccess) return e;
  static bool done[MAX_DEVICES] = {};
  e = prepare_kernel(own_kernel<D>, (int)Geo<D>::smem(SHARED_MAX_BATCH), done);
  if (e != cudaSuccess) return e;
  e = launch_k(own_kernel<D>, dim3((unsigned)((a.n_prefix > 0 ? CTAS_SHARED : CTAS_ALONE) * a.num_sms)), dim3(WARPS * 32), Geo<D>::smem(a.B), st, ok, ov, a);
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
