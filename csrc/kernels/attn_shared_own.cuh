// The keys behind the shared prefixes: device code of the warps that read them, for the kernel that does only that
// (attn_shared.cu) and for the prefix kernel, where four warps of every CTA do it beside the tensor cores' work.
#pragma once
#include "attn_shared.cuh"

namespace mesh {
namespace shared_attn {
namespace {

constexpr int WARPS = 4;         // workers of a CTA
constexpr int CTAS = 3;          // per SM, where nothing is shared
constexpr int TILE_ROWS = 16;    // query rows of a worker
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

// The keys behind the shared prefixes: 16 rows (new tokens x heads of a KV group) of one sequence against that sequence's
// own slices of 16 keys. All of them, in the order (sequence, KV head, tile of rows, slice), are cut into equal quotas,
// one per warp: lengths from one token to long ones then keep every SM as busy. A quota is a run of
// pieces, one for each (sequence, head, tile) it touches; a piece counts as PIECE_COST slices besides its own, about
// what loading its queries and writing its result take. Piece number = worker + (sequence, head, tile), which no other
// piece has. A warp works by itself: it requests slices SLOTS ahead (TMA, 128-byte swizzle) and multiplies on m16n8k16
// fragments, without a barrier between warps; four warps that split each piece and merged it took twice as long
// (64 sessions of up to 512 keys). Bound by reading K and V. HALF: 1 for up to 8 rows, whose half of the fragments is the
// only one that counts; else 2.
template <int D, int HALF>
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
      // query fragments straight from memory: rows lane / 4 and 8 below it, columns (lane % 4) * 2 and 8 to the right
      uint32_t qf[D / 16][4];
      int hi_k[2], lo_k[2];  // keys this lane's two rows may attend: [lo_k, hi_k)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = (lane >> 2) + 8 * j, x = row0 + r, t = x / a.G;
        const bool valid = j < HALF && r < n_rows;
        const __nv_bfloat16* src = a.q + ((long)(p.b * a.T + t) * hq + h * a.G + x - t * a.G) * D + (lane & 3) * 2;
        const int pos = q.L - a.T + t;
        hi_k[j] = valid ? min(k1, pos + 1) : 0;
        lo_k[j] = a.window > 0 ? max(k0, pos + 1 - a.window) : k0;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          qf[kk][j] = valid ? *reinterpret_cast<const uint32_t*>(src + kk * 16) : 0u;
          qf[kk][2 + j] = valid ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + 8) : 0u;
        }
      }
      float o[D / 8][4];
#pragma unroll
      for (int x = 0; x < D / 8; ++x) o[x][0] = o[x][1] = o[x][2] = o[x][3] = 0.f;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll 1
      for (int i = 0; i < p.n; ++i) {
        ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded(&full[s], ph, a.err, ERR_MBAR_TIMEOUT_MMA, nullptr, WAIT_NS));
        if (!ok) break;
        const int key0 = (s0 + i) * SLICE;
        const uint32_t kb = smem_u32(ring + s * g::SLICE_BYTES), vb = kb + g::HALVES * g::BOX;
        // Keys past the range may hold anything (a page's unused tail): their values must not reach the products as
        // NaN or infinity times a zero weight. Clearing them in the fragments costs two masks; clearing them in shared
        // memory needs a proxy fence, which waited for the loads in flight.
        uint32_t keep[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int left = k1 - (key0 + x * 8 + (lane & 3) * 2);  // of this lane's two keys
          keep[x] = left >= 2 ? 0xffffffffu : left == 1 ? 0xffffu : 0u;
        }
        float sc[2][4], sd[2][4];  // two chains of products each
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[t][e] = sd[t][e] = 0.f;
#pragma unroll
          for (int kk = 0; kk < D / 16; kk += 2) {
            uint32_t bb[4];
            ldsm_x4(kb + (kk >> 2) * g::BOX + swz(t * 8 + (lane & 7), (kk & 3) * 2 + (lane >> 3)), bb);
            mma(sc[t], qf[kk], bb[0], bb[1]);
            mma(sd[t], qf[kk + 1], bb[2], bb[3]);
          }
        }
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2 * HALF; ++e) {
            const int key = key0 + t * 8 + (lane & 3) * 2 + (e & 1), j = e >> 1;
            sc[t][e] = (key < hi_k[j] && key >= lo_k[j]) ? (sc[t][e] + sd[t][e]) * a.scale_log2 : -INFINITY;
            mx[j] = fmaxf(mx[j], sc[t][e]);
          }
        float pr[2][4] = {};
#pragma unroll
        for (int j = 0; j < HALF; ++j) {
          mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 1));
          mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 2));
          const float mn = fmaxf(m[j], mx[j]), mb = mn == -INFINITY ? 0.f : mn;
          const float corr = ex2_ftz(m[j] - mb);
          float ps = 0.f;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float x = ex2_ftz(sc[t][2 * j + e] - mb);
              pr[t][2 * j + e] = x;
              ps += x;
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
          mma(o[x], pa, bb[0] & keep[0], bb[1] & keep[1]);
          mma(o[x + 1], pa, bb[2] & keep[0], bb[3] & keep[1]);
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
      for (int j = 0; j < HALF; ++j) {
        l[j] += __shfl_xor_sync(0xffffffffu, l[j], 1);
        l[j] += __shfl_xor_sync(0xffffffffu, l[j], 2);
      }
      // a sequence without a prefix whose keys are all in this piece is done: its rows go out; else a partial
      const bool whole = p.n == q.slices() && q.slots == 0;
      const int stride = min(rows, TILE_ROWS);
      const long part = a.own_at + (long)(worker + p.b * per_seq + p.u) * stride;
      if (part + stride > a.slot_cap) {
        if (lane == 0) record_error(a.err, ERR_BAD_ARGUMENT);
        continue;
      }
#pragma unroll
      for (int j = 0; j < HALF; ++j) {
        const int r = (lane >> 2) + 8 * j;
        if (r >= n_rows) continue;
        const int x0 = row0 + r, t = x0 / a.G;
        __nv_bfloat16* out = a.out + ((long)(p.b * a.T + t) * hq + h * a.G + x0 - t * a.G) * D;
        const float inv = l[j] > 0.f ? 1.f / l[j] : 0.f;
#pragma unroll
        for (int x = 0; x < D / 8; ++x) {
          const int d = x * 8 + (lane & 3) * 2;
          if (whole)
            *reinterpret_cast<uint32_t*>(out + d) = pack_bf16x2(o[x][2 * j] * inv, o[x][2 * j + 1] * inv);
          else
            *reinterpret_cast<float2*>(a.po + (part + r) * D + d) = make_float2(o[x][2 * j], o[x][2 * j + 1]);
        }
        if (!whole && (lane & 3) == 0) a.pml[part + r] = make_float2(m[j], l[j]);
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

}  // namespace
}  // namespace shared_attn
}  // namespace mesh
