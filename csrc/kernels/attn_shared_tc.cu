// Shared prefixes on the 5th-generation tensor cores (sm_100a): the rows of all sequences of a group (sequence, new
// token, head of one KV group) against the keys they share, split over the keys so that one wave of CTAs takes it.
//
// An item is up to 256 rows x a range of keys, in two streams of 128 rows that walk the keys in blocks of 64. 64 keys for
// 256 rows are 8.4 MFLOP and 32 KB: tensor cores (11.6 TFLOP/s an SM) and HBM (43 GB/s an SM) take the same 0.73 us.
// Roles (384 threads): warp 0 loads K and warp 10 V (16-key slices of pages, [16 x 64] boxes, 128-byte swizzle) into
// separate rings, so a K block makes room as soon as its scores are done, and because one thread takes 90 ns a box, which
// alone made a block take 1.5 us; warps 1 and 11 issue tcgen05.mma (one thread each) for stream 0 and 1: S = Q K^T into
// TMEM, then O += P V with the bf16 weights P read from TMEM (over the first half of S) and V read MN-major from the page
// layout; warps 2..5 and 6..9 run the softmax of stream 0 and 1, a row per thread, and gather the query rows, which lie
// wherever their sequences do. A stream has two score buffers: the scores of a block are made while the softmax
// of the one before runs, which therefore never waits for a product (with one buffer and blocks of 128 the way from
// weights to the next scores, 1.5 us, stood beside 1.1 us of softmax). The running maximum only moves (and O is rescaled in
// TMEM) when it grows by more than 2^8; sum and output share it, so the result stays exact.
// Measured: 1.0 us a block (128 sessions x 4 heads, 8 KV heads: 28.7 us a call with 8 blocks in every CTA, 53.0 with 32), seven
// tenths of what either bound allows; the chain from scores to weights sets the pace, not a unit: with a half, a quarter or an
// eighth of the exponentials made by multiplications instead, the times stayed within 1 %. Before the first scores go 5.5 us, and 3.3 us into
// writing an item's partials.
// TMEM columns (512): S of stream t, buffer b at t * 128 + b * 64; O_t at 256 + t * 128.
// Every wait is bounded; on a timeout an error is recorded, copies and products in flight are drained, TMEM is freed.
#include "attn_shared.cuh"

namespace mesh {
namespace shared_attn {
namespace {

constexpr int BM = 128, BK = 64, NS = 2;  // rows and keys of a stream's block, streams
constexpr int SLICES = BK / SLICE;
constexpr int THREADS = 128 + NS * BM;
// A thread: 12 warps leave room for the 4 of an own_kernel CTA. prefix_kernel<64> spills 4 bytes under it.
constexpr int MAX_REGS = 128;
constexpr int PRODUCER_V = 10, MMA0 = 1, MMA1 = 11;  // warps
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t S_COLS = 128, O_COL = NS * S_COLS, O_COLS = 128;
constexpr float RESCALE = 8.0f;  // log2 units

template <int D>
struct Cfg {
  static constexpr int HALVES = D / 64;
  static constexpr uint32_t Q_ATOM = BM * 128;            // 128 rows x 64 elements
  static constexpr uint32_t Q_TILE = HALVES * Q_ATOM;     // 128 rows x D
  static constexpr uint32_t ATOM = BK * 128;              // 64 keys x 64 elements
  static constexpr uint32_t TILE = HALVES * ATOM;         // 64 keys x D
  // blocks of K and of V in flight: 80 KB of rings. With the query tiles that leaves room for a CTA of the sequences' own
  // keys on the same SM, which reads while this kernel multiplies.
  static constexpr int K_STAGES = 3 * (128 / D), V_STAGES = 2 * (128 / D);
  static constexpr uint32_t BOX = SLICE * 128;
  static constexpr int STAGED = D * 4 + 16;               // a row of the result on its way out: padded against bank conflicts
};

template <int D>
struct Bars {
  uint64_t q_full;
  uint64_t k_full[Cfg<D>::K_STAGES], k_empty[Cfg<D>::K_STAGES], v_full[Cfg<D>::V_STAGES], v_empty[Cfg<D>::V_STAGES];
  uint64_t s_full[NS][2], p_full[NS][2], o_done[NS], o_last[NS];  // o_last: the item's last product
  uint64_t mma_done;
  uint32_t tmem_base;
  int abort;
};

template <int D>
constexpr size_t smem_bytes() {
  static_assert(NS * BM * Cfg<D>::STAGED <= NS * Cfg<D>::Q_TILE + (Cfg<D>::K_STAGES + Cfg<D>::V_STAGES) * Cfg<D>::TILE, "staged rows fit");
  return 1024 + NS * Cfg<D>::Q_TILE + (Cfg<D>::K_STAGES + Cfg<D>::V_STAGES) * Cfg<D>::TILE + sizeof(Bars<D>);
}

struct Item {
  int table_row, moff, row0, rows, h, k0, k1, slot;
  __device__ __forceinline__ Item(const Args& a, int i) {
    const int4* p = reinterpret_cast<const int4*>(items(a) + (long)i * ITEM);
    const int4 x = p[0], y = p[1];
    table_row = x.x, moff = x.y, row0 = x.z, rows = x.w;
    h = y.x, k0 = y.y, k1 = min(y.z, a.max_pages * a.page_size), slot = y.w;
  }
  __device__ __forceinline__ int blocks() const { return k1 > k0 ? (k1 - k0 + BK - 1) / BK : 0; }
  __device__ __forceinline__ int streams() const { return rows > BM ? 2 : 1; }
};

template <int D>
__global__ void __maxnreg__(MAX_REGS)
    prefix_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Args a) {
  using C = Cfg<D>;
  constexpr int K_STAGES = C::K_STAGES, V_STAGES = C::V_STAGES;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* q_sm = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint8_t* k_sm = q_sm + NS * C::Q_TILE;
  uint8_t* v_sm = k_sm + K_STAGES * C::TILE;
  Bars<D>* bars = reinterpret_cast<Bars<D>*>(v_sm + V_STAGES * C::TILE);
  // broadcast values are known to be the same for the whole warp, so the address arithmetic of the issuing warps stays in
  // uniform registers (a product took 60 ns to issue otherwise, a TMA box 108 instead of 75)
  auto uniform = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, NS * BM);
    for (int i = 0; i < K_STAGES; ++i) {
      mbar_init(&bars->k_full[i], 1);
      mbar_init(&bars->k_empty[i], NS);
    }
    for (int i = 0; i < V_STAGES; ++i) {
      mbar_init(&bars->v_full[i], 1);
      mbar_init(&bars->v_empty[i], NS);
    }
    for (int t = 0; t < NS; ++t) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(&bars->s_full[t][b], 1);
        mbar_init(&bars->p_full[t][b], BM);
      }
      mbar_init(&bars->o_done[t], 1);
      mbar_init(&bars->o_last[t], 1);
    }
    mbar_init(&bars->mma_done, NS);
    bars->abort = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == MMA0) {
    tmem_alloc(&bars->tmem_base, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = (uint32_t)uniform((int)bars->tmem_base);
  volatile int* abort_flag = &bars->abort;
  // The items and members are written by the host alone, never by a kernel that this grid may overlap.
  const int n_items = uniform(min(a.meta[0], a.n_prefix));
  const int TG = a.T * a.G, hq = a.hkv * a.G;
  // softmax threads: stream, TMEM lane (a warp may access those of warp % 4 only), row of the item
  const int st = (warp - 2) >> 2, r = (warp & 3) * 32 + lane, x = st * BM + r;
  int first_b = 0;
  Item it(a, min((int)blockIdx.x, max(0, n_items - 1)));
  if (warp >= 2 && warp < PRODUCER_V && (int)blockIdx.x < n_items) {
    if (x < it.rows) first_b = members(a)[it.moff + (it.row0 + x) / TG];
  }
  griddep_wait();
  // The kernel of the sequences' own keys needs what precedes this grid (complete now) and, at its end only, this
  // grid's partials: it starts beside it.
  griddep_launch_dependents();

  // ring positions of this warp's role: the next block of K (MMA: to score; producer of K) and of V
  int pos = 0, v_pos = 0;
  uint32_t phase = 0, v_phase = 0;
  auto advance = [](int& at, uint32_t& ph, int stages) {
    if (++at == stages) {
      at = 0;
      ph ^= 1u;
    }
  };
  uint32_t cnt = 0;  // blocks this warp's stream has gone through (MMA, softmax)
  uint32_t ic = 0;   // items
  uint32_t lasts = 0;  // items this softmax warp's stream took part in
  for (int i = blockIdx.x; i < n_items; i += gridDim.x, ++ic) {
    if (ic > 0) it = Item(a, i);
    const int nblk = uniform(it.blocks());
    const int ns = uniform(it.streams());
    if (warp == 0 || warp == PRODUCER_V) {
      // ------------------------------------ TMA producers: K, V ------------------------------------
      const uint64_t pol = policy_evict_first();
      const int* bt = a.block_tables + (long)it.table_row * a.max_pages;
      const CUtensorMap* tm = warp == 0 ? &tmK : &tmV;
      uint8_t* ring = warp == 0 ? k_sm : v_sm;
      uint64_t* full = warp == 0 ? bars->k_full : bars->v_full;
      uint64_t* empty = warp == 0 ? bars->k_empty : bars->v_empty;
      const int stages = warp == 0 ? K_STAGES : V_STAGES;
      const int first = it.k0 / SLICE, slices = nblk > 0 ? (it.k1 + SLICE - 1) / SLICE - first : 0;
      int row_y = 0, ok = 1, j = 0;
      for (; j < nblk && ok; ++j) {
        if ((j & (32 / SLICES - 1)) == 0) {  // rows of the pool that hold the next 32 slices, one per lane
          const int c = j * SLICES + lane;
          if (c < slices) {
            const int pi = (first + c) / a.slices_per_page;
            row_y = (bt[pi] * a.hkv + it.h) * a.page_size + (first + c - pi * a.slices_per_page) * SLICE;
          }
        }
        const int s = pos, n = uniform(min(SLICES, slices - j * SLICES));
        int y[SLICES];
#pragma unroll
        for (int p = 0; p < SLICES; ++p) y[p] = __shfl_sync(0xffffffffu, row_y, (j * SLICES + p) & 31);
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&empty[s], phase ^ 1u, a.err, ERR_MBAR_TIMEOUT_PRODUCER,
                                                       abort_flag, WAIT_NS));
        if (ok && elect_one()) {
          mbar_arrive_expect_tx(&full[s], (uint32_t)n * C::HALVES * C::BOX);
#pragma unroll
          for (int p = 0; p < SLICES; ++p)
            if (p < n)
#pragma unroll
              for (int hf = 0; hf < C::HALVES; ++hf)
                tma_load_2d(ring + s * C::TILE + hf * C::ATOM + p * C::BOX, tm, &full[s], hf * 64, y[p], pol);
        }
        __syncwarp();
        if (ok) advance(pos, phase, stages);
      }
      if (!ok && lane == 0) {  // copies already in flight land before the CTA goes on (bounded)
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 1000000ull) {
        }
      }
      __syncwarp();
    } else if (warp == MMA0 || warp == MMA1) {
      // ------------------------------------ MMA issuers: stream 0, 1 ------------------------------------
      // two, because a wait costs the issuing warp about 200 cycles even when it is over, in which the tensor core runs dry
      const int t = warp == MMA0 ? 0 : 1;
      constexpr uint32_t IDESC_QK = make_idesc_bf16(BM, BK);
      constexpr uint32_t IDESC_PV = make_idesc_bf16(BM, D) | IDESC_B_MN_MAJOR;
      // descriptors of the first tile; addresses count in 16 bytes and stay below 2^18, so offsets just add up
      const uint64_t q_desc = make_sdesc_sw128(smem_u32(q_sm)), k_desc = make_sdesc_sw128(smem_u32(k_sm));
      const uint64_t v_desc = make_sdesc_sw128_mn(smem_u32(v_sm), C::ATOM, 1024);
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, a.err, ERR_MBAR_TIMEOUT_MMA, abort_flag, WAIT_NS)) != 0;
      };
      // a block of K or V is free when every stream has given it back
      auto give_back = [&](uint64_t* bar) {
        umma_commit(bar);
        if (ns == 1) umma_commit(bar);
      };
      // scores of the next block of K, the stream's g-th
      auto issue_qk = [&](uint32_t g) {
        const uint64_t qd = q_desc + t * (C::Q_TILE >> 4), kd = k_desc + pos * (C::TILE >> 4);
        const uint32_t st = tmem + t * S_COLS + (g & 1) * BK;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_bf16(st, qd + (kk >> 2) * (C::Q_ATOM >> 4) + 2 * (kk & 3), kd + (kk >> 2) * (C::ATOM >> 4) + 2 * (kk & 3), IDESC_QK,
                      kk > 0 ? 1u : 0u);
          umma_commit(&bars->s_full[t][g & 1]);
          give_back(&bars->k_empty[pos]);
        }
        __syncwarp();
        advance(pos, phase, K_STAGES);
      };
      auto issue_pv = [&](int j, uint32_t g) {
        const uint64_t vd = v_desc + v_pos * (C::TILE >> 4);
        const uint32_t ot = tmem + O_COL + t * O_COLS, pt = tmem + t * S_COLS + (g & 1) * BK;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk)
            umma_bf16_ts(ot, pt + kk * 8, vd + kk * (2048 >> 4), IDESC_PV, (j > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&bars->o_done[t]);
          if (j == nblk - 1) umma_commit(&bars->o_last[t]);
          give_back(&bars->v_empty[v_pos]);
        }
        __syncwarp();
        advance(v_pos, v_phase, V_STAGES);
      };
      // V rows past the range (a page's tail, or a slice that was not loaded) may hold anything; a zero weight times
      // NaN would reach the output, so they are cleared
      auto clear_tail = [&](int j) {
        const int valid = it.k1 - (it.k0 + j * BK);
        if (valid >= BK) return;
        uint8_t* v = v_sm + v_pos * C::TILE;
        for (int c = lane; c < (BK - valid) * C::HALVES * 8; c += 32) {
          const int r = valid + c / (C::HALVES * 8), x = c % (C::HALVES * 8);
          *reinterpret_cast<uint4*>(v + (x >> 3) * C::ATOM + r * 128 + ((x & 7) << 4)) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();
        __syncwarp();
      };
      bool ok = nblk == 0 || wait(&bars->q_full, ic & 1u);
      if (t < ns) {
        // both score buffers
        for (int j = 0; j < min(2, nblk) && ok; ++j) {
          ok = wait(&bars->k_full[pos], phase);
          tc_fence_after();
          if (ok) issue_qk(cnt + j);
        }
        for (int j = 0; j < nblk && ok; ++j) {
          const uint32_t g = cnt + j;
          // V of this block, the softmax's P (and its rescaling of O), K of the next scores
          ok = wait(&bars->v_full[v_pos], v_phase);
          if (!ok) break;
          if (j == nblk - 1) clear_tail(j);
          ok = wait(&bars->p_full[t][g & 1], (g >> 1) & 1u);
          if (!ok) break;
          tc_fence_after();
          issue_pv(j, g);
          if (j + 2 < nblk) {
            // these scores overwrite the columns P was in: one thread's products run in the order of issue
            ok = wait(&bars->k_full[pos], phase);
            tc_fence_after();
            if (ok) issue_qk(g + 2);
          }
        }
        cnt += nblk;
      } else {  // the ring moves on without this stream
        for (int j = 0; j < nblk; ++j) {
          advance(pos, phase, K_STAGES);
          advance(v_pos, v_phase, V_STAGES);
        }
      }
    } else {
      // ------------------------------------ softmax (warps 2..9) ------------------------------------
      const int t = st;
      const bool valid = x < it.rows;
      int b = 0;
      if (valid) b = ic == 0 ? first_b : members(a)[it.moff + (it.row0 + x) / TG];
      const int y = it.row0 + x, tok = (y / a.G) % a.T, head = it.h * a.G + y % a.G;
      // this thread's query row into the tile, all its loads in flight at once
      if (t < ns) {
        constexpr int CH = D / 8;
        uint4 v[CH];
        const uint4* src = reinterpret_cast<const uint4*>(a.q + ((long)(b * a.T + tok) * hq + head) * D);
#pragma unroll
        for (int c = 0; c < CH; ++c) v[c] = valid ? src[c] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < CH; ++c)
          *reinterpret_cast<uint4*>(q_sm + t * C::Q_TILE + (c >> 3) * C::Q_ATOM + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v[c];
        fence_proxy_async();
      }
      mbar_arrive(&bars->q_full);
      long slot = -1;
      int lim = 0, low = 0;  // keys [low, lim) of the range are this row's
      if (valid) {
        const int pos = a.seq_lens[b] - a.T + tok;
        lim = min(it.k1, pos + 1);
        low = a.window > 0 ? pos + 1 - a.window : 0;
        slot = (long)seq_base(a, b) + (long)(tok * hq + head) * seq_prefix_slots(a, b) + it.slot;
        if (slot < 0 || slot >= a.own_at || it.slot >= seq_prefix_slots(a, b)) {
          record_error(a.err, ERR_BAD_ARGUMENT);
          slot = -1;
        }
      }
      const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t o_addr = tmem + lane_off + O_COL + t * O_COLS;
      const bool warp_live = __any_sync(0xffffffffu, valid);
      float m_used = -INFINITY, l = 0.f;
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        int w = 1;
        if (lane == 0) w = mbar_wait_bounded(bar, parity, a.err, ERR_MBAR_TIMEOUT_EPILOGUE, abort_flag, WAIT_NS);
        return __shfl_sync(0xffffffffu, w, 0) != 0;
      };
      for (int j = 0; j < nblk && t < ns; ++j) {
        const uint32_t g = cnt + j;
        if (!(ok = wait(&bars->s_full[t][g & 1], (g >> 1) & 1u))) break;
        tc_fence_after();
        if (warp_live) {
          const uint32_t s_addr = tmem + lane_off + t * S_COLS + (g & 1) * BK;
          uint32_t sv[BK];
#pragma unroll
          for (int c = 0; c < BK / 16; ++c)
            tmem_ld16(s_addr + (uint32_t)(16 * c), *reinterpret_cast<uint32_t(*)[16]>(&sv[16 * c]));
          tmem_ld_wait_tied(sv);
          const int key0 = it.k0 + j * BK;
          if (__any_sync(0xffffffffu, valid && (key0 + BK > lim || key0 < low))) {
#pragma unroll
            for (int c = 0; c < BK; ++c)
              if (key0 + c >= lim || key0 + c < low) sv[c] = __float_as_uint(-INFINITY);
          }
          float mx[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) mx[c] = __uint_as_float(sv[c]);
#pragma unroll
          for (int c = 4; c < BK; ++c) mx[c & 3] = fmaxf(mx[c & 3], __uint_as_float(sv[c]));
          const float mraw = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          const float m_new = fmaxf(m_used, mraw * a.scale_log2);
          const bool resc = m_new > m_used + RESCALE;
          float alpha = 1.f;
          if (resc) {
            alpha = ex2_ftz(m_used - m_new);  // 0 when m_used is -inf
            m_used = m_new;
          }
          const float mb = m_used == -INFINITY ? 0.f : m_used;
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
          // The weights are rounded to bf16 for the product (half a step of 2^-8 each), whose operands are of one type; their
          // sum keeps fp32. Outputs are then 0.0019 to 0.0023 from 64 bits, with fp32 weights and the same last rounding 0.0017.
#pragma unroll
          for (int c = 0; c < BK / 32; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float p0 = ex2_ftz(fmaf(__uint_as_float(sv[32 * c + 2 * e]), a.scale_log2, -mb));
              const float p1 = ex2_ftz(fmaf(__uint_as_float(sv[32 * c + 2 * e + 1]), a.scale_log2, -mb));
              sum[e & 3] += p0 + p1;
              pk[e] = pack_bf16x2(p0, p1);
            }
            tmem_st16(s_addr + (uint32_t)(16 * c), pk);
          }
          l = l * alpha + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
          if (j > 0 && __any_sync(0xffffffffu, resc)) {
            // the product before is complete (the one before that was when these scores were): O is stable
            if (!(ok = wait(&bars->o_done[t], (g - 1) & 1u))) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t ov[16];
              tmem_ld16(o_addr + 16 * c, ov);
              tmem_ld_wait_tied(ov);
#pragma unroll
              for (int e = 0; e < 16; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
              tmem_st16(o_addr + 16 * c, ov);
            }
          }
          tmem_st_wait();
        }
        tc_fence_before();
        mbar_arrive(&bars->p_full[t][g & 1]);
      }
      if (t < ns) {
        cnt += nblk;
        // A barrier of its own: o_done may be one or two products behind, which its parity does not tell apart.
        if (nblk > 0) ok = ok && wait(&bars->o_last[t], lasts++ & 1u);
        tc_fence_after();
        named_bar_sync(1, ns * BM);  // every stream is done with the query tiles and the rings
        if (ok && warp_live) {
          if (slot >= 0) a.pml[slot] = make_float2(m_used, l);
          const long to = slot >= 0 && l != 0.f ? slot : -1;  // NaN too: the merge reads what has a sum
          if (nblk > 0 && __any_sync(0xffffffffu, to >= 0)) {
            // A row is one TMEM lane: the warp lays its 32 rows out in shared memory and writes them row by row.
            uint8_t* rows_sm = q_sm + (x - lane) * C::STAGED;
#pragma unroll 1
            for (int c = 0; c < D / 64; ++c) {
              uint32_t ov[64];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                tmem_ld16(o_addr + 64 * c + 16 * e, *reinterpret_cast<uint32_t(*)[16]>(&ov[16 * e]));
              tmem_ld_wait_tied(ov);
#pragma unroll
              for (int e = 0; e < 16; ++e)
                *reinterpret_cast<uint4*>(rows_sm + lane * C::STAGED + c * 256 + e * 16) =
                    make_uint4(ov[4 * e], ov[4 * e + 1], ov[4 * e + 2], ov[4 * e + 3]);
            }
            __syncwarp();
            constexpr int LANES = D / 4, AT_ONCE = 32 / LANES;  // lanes of a row, rows at once
#pragma unroll 8
            for (int k = 0; k < 32 / AT_ONCE; ++k) {
              const int row = k * AT_ONCE + lane / LANES;
              const long dst = __shfl_sync(0xffffffffu, to, row);
              const float4 v = *reinterpret_cast<const float4*>(rows_sm + row * C::STAGED + (lane % LANES) * 16);
              if (dst >= 0) *reinterpret_cast<float4*>(a.po + dst * D + (lane % LANES) * 4) = v;
            }
          }
        }
      }
      tc_fence_before();
      if (i + (int)gridDim.x < n_items) fence_proxy_async();  // the shared memory is written by TMA again
    }
    __syncthreads();
    tc_fence_after();
    if (bars->abort) break;
  }
  // every product issued above has completed before TMEM is released
  if ((warp == MMA0 || warp == MMA1) && lane == 0) {
    umma_commit(&bars->mma_done);
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(&bars->mma_done, 0) && globaltimer_ns() - t0 < 50000000ull) {
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == MMA0) tmem_dealloc(tmem, TMEM_COLS);
}

}  // namespace

template <int D>
cudaError_t launch_prefix(const Args& a, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t st) {
  auto kern = prefix_kernel<D>;
  static bool done[MAX_DEVICES] = {};
  const cudaError_t e = prepare_kernel(kern, (int)smem_bytes<D>(), done);
  if (e != cudaSuccess) return e;
  return launch_k(kern, dim3((unsigned)min(a.n_prefix, a.num_sms)), dim3(THREADS), smem_bytes<D>(), st, tk, tv, a);
}
template cudaError_t launch_prefix<64>(const Args&, const CUtensorMap&, const CUtensorMap&, cudaStream_t);
template cudaError_t launch_prefix<128>(const Args&, const CUtensorMap&, const CUtensorMap&, cudaStream_t);

}  // namespace shared_attn
}  // namespace mesh
