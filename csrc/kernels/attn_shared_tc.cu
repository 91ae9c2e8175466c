// Shared prefixes on the 5th-generation tensor cores (sm_100a): the rows of all sequences of a group (sequence, new
// token, head of one KV group) against the keys they share, split over the keys so that one wave of CTAs takes it.
//
// An item is up to 256 rows x a range of keys, walked in blocks of 128 keys by two streams of 128 rows x 128 keys that
// keep the tensor cores busy in turn: while one stream's softmax runs, the other's products do.
//   more than 128 rows   stream t takes rows 128 t .. of every block, so each block serves 256 rows: 16.8 MFLOP for
//                        64 KB, where tensor cores (11.6 TFLOP/s an SM) and HBM (43 GB/s an SM) take the same 1.5 us;
//   at most 128          stream t takes every other block with the same rows; bound by reading the keys. The streams'
//                        results are merged in shared memory at the end.
// Roles (320 threads): warp 0 loads K and V (16-key slices of pages, [16 x 64] boxes, 128-byte swizzle) into separate
// rings, so a K block makes room as soon as its scores are done; warp 1 issues tcgen05.mma (one thread): S = Q K^T into
// TMEM, then O += P V with the bf16 weights P read from TMEM (over the first half of S) and V read MN-major from the page
// layout; warps 2..5 and 6..9 run the softmax of stream 0 and 1, a row per thread, and gather the query rows, which lie
// wherever their sequences do. The running maximum only moves (and O is rescaled in TMEM) when it grows by more than
// 2^8; sum and output share it, so the result stays exact.
// TMEM columns (512): S0 [0,128) S1 [128,256) O0 [256,256+D) O1 [384,384+D).
// Every wait is bounded; on a timeout an error is recorded, copies and products in flight are drained, TMEM is freed.
#include "attn_shared.cuh"

namespace mesh {
namespace shared_attn {
namespace {

constexpr int BM = 128, BK = 128, NS = 2;  // rows and keys of a stream's block, streams
constexpr int SLICES = BK / SLICE;
constexpr int THREADS = 64 + NS * BM;
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t O_COL = NS * BK;
constexpr float RESCALE = 8.0f;  // log2 units

template <int D>
struct Cfg {
  static constexpr int HALVES = D / 64;
  static constexpr uint32_t ATOM = BM * 128;           // 128 rows x 64 elements
  static constexpr uint32_t TILE = HALVES * ATOM;      // 128 rows x D
  static constexpr int STAGES = 2 * (128 / D);         // blocks of K, and of V: 128 KB of rings
  static constexpr uint32_t BOX = SLICE * 128;
};

template <int D>
struct Bars {
  uint64_t q_full;
  uint64_t k_full[Cfg<D>::STAGES], v_full[Cfg<D>::STAGES], k_empty[Cfg<D>::STAGES], v_empty[Cfg<D>::STAGES];
  uint64_t s_full[NS], p_full[NS], o_done[NS];
  uint64_t mma_done;
  uint32_t tmem_base;
  int abort;
};

static_assert(BM * (128 * 4 + 16) <= (NS + Cfg<128>::STAGES) * Cfg<128>::TILE && BM * (64 * 4 + 16) <= (NS + Cfg<64>::STAGES) * Cfg<64>::TILE &&
                  NS * BM * (128 * 4 + 16) <= (NS + 2 * Cfg<128>::STAGES) * Cfg<128>::TILE,
              "staged rows fit");

template <int D>
constexpr size_t smem_bytes() {
  return 1024 + (NS + 2 * Cfg<D>::STAGES) * Cfg<D>::TILE + BM * 8 + NS * BM * 8 + sizeof(Bars<D>);
}

// One contiguous copy shared -> global (16-byte aligned, a multiple of 16 bytes).
__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(reinterpret_cast<uint64_t>(dst)),
               "r"(smem_u32(src)), "r"(bytes)
               : "memory");
}
// This thread's bulk copies have read their sources (the shared memory may be used again).
__device__ __forceinline__ void bulk_commit_wait_read() {
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
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
  __device__ __forceinline__ bool two_tiles() const { return rows > BM; }
};

template <int D>
__global__ void __launch_bounds__(THREADS, 1)
    prefix_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Args a) {
  using C = Cfg<D>;
  constexpr int STAGES = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* q_sm = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint8_t* k_sm = q_sm + NS * C::TILE;
  uint8_t* v_sm = k_sm + STAGES * C::TILE;
  float2* ml_sm = reinterpret_cast<float2*>(v_sm + STAGES * C::TILE);
  long* row_sm = reinterpret_cast<long*>(ml_sm + BM);  // offsets of the query rows, then partial slots
  Bars<D>* bars = reinterpret_cast<Bars<D>*>(row_sm + NS * BM);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, NS * BM);
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&bars->k_full[i], 1);
      mbar_init(&bars->v_full[i], 1);
      mbar_init(&bars->k_empty[i], 1);
      mbar_init(&bars->v_empty[i], 1);
    }
    for (int t = 0; t < NS; ++t) {
      mbar_init(&bars->s_full[t], 1);
      mbar_init(&bars->p_full[t], BM);
      mbar_init(&bars->o_done[t], 1);
    }
    mbar_init(&bars->mma_done, 1);
    bars->abort = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  volatile int* abort_flag = &bars->abort;
  griddep_wait();
  // The kernel of the sequences' own keys needs what precedes this grid (complete now) and, at its end only, this
  // grid's partials: it may start as SMs fall free.
  griddep_launch_dependents();
  const int n_items = min(a.meta[0], a.n_prefix);

  uint32_t kvc = 0;               // blocks loaded by this CTA (ring position)
  uint32_t cnt[NS] = {0, 0};      // MMA warp: blocks each stream has gone through; softmax warps: their own in cnt[0]
  uint32_t ic = 0;                // items
  for (int i = blockIdx.x; i < n_items; i += gridDim.x, ++ic) {
    const Item it(a, i);
    const int nblk = it.blocks();
    const bool two = it.two_tiles();
    if (warp == 0) {
      // ------------------------------------ TMA producer ------------------------------------
      if (lane == 0) {
        const uint64_t pol = policy_evict_last();  // other tiles of rows read the same keys
        const int* bt = a.block_tables + (long)it.table_row * a.max_pages;
        bool ok = true;
        int j = 0;
        for (; j < nblk && ok; ++j) {
          const uint32_t c = kvc + j;
          const int s = c % STAGES;
          const uint32_t ph = ((c / STAGES) & 1u) ^ 1u;
          const int key0 = it.k0 + j * BK;
          const int n = min(SLICES, (it.k1 - key0 + SLICE - 1) / SLICE);
          int y[SLICES];
#pragma unroll
          for (int p = 0; p < SLICES; ++p) {
            if (p < n) {
              const int sl = key0 / SLICE + p, pi = sl / a.slices_per_page;
              y[p] = (bt[pi] * a.hkv + it.h) * a.page_size + (sl - pi * a.slices_per_page) * SLICE;
            }
          }
          if (!(ok = mbar_wait_bounded(&bars->k_empty[s], ph, a.err, ERR_MBAR_TIMEOUT_PRODUCER, abort_flag, WAIT_NS))) break;
          mbar_arrive_expect_tx(&bars->k_full[s], (uint32_t)n * C::HALVES * C::BOX);
#pragma unroll
          for (int p = 0; p < SLICES; ++p)
            if (p < n)
#pragma unroll
              for (int hf = 0; hf < C::HALVES; ++hf)
                tma_load_2d(k_sm + s * C::TILE + hf * C::ATOM + p * C::BOX, &tmK, &bars->k_full[s], hf * 64, y[p], pol);
          if (!(ok = mbar_wait_bounded(&bars->v_empty[s], ph, a.err, ERR_MBAR_TIMEOUT_PRODUCER, abort_flag, WAIT_NS))) {
            // the K block just requested lands before the CTA goes on (bounded)
            const uint64_t t0 = globaltimer_ns();
            while (!mbar_try_wait(&bars->k_full[s], ph ^ 1u) && globaltimer_ns() - t0 < 50000000ull) {
            }
            break;
          }
          mbar_arrive_expect_tx(&bars->v_full[s], (uint32_t)n * C::HALVES * C::BOX);
#pragma unroll
          for (int p = 0; p < SLICES; ++p)
            if (p < n)
#pragma unroll
              for (int hf = 0; hf < C::HALVES; ++hf)
                tma_load_2d(v_sm + s * C::TILE + hf * C::ATOM + p * C::BOX, &tmV, &bars->v_full[s], hf * 64, y[p], pol);
        }
        if (!ok) {
          const uint64_t t0 = globaltimer_ns();
          for (int x = max(0, j - STAGES); x < j; ++x) {
            const uint32_t c = kvc + x;
            while (!(mbar_try_wait(&bars->k_full[c % STAGES], (c / STAGES) & 1u) &&
                     mbar_try_wait(&bars->v_full[c % STAGES], (c / STAGES) & 1u)) &&
                   globaltimer_ns() - t0 < 50000000ull) {
            }
          }
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      // ------------------------------------ MMA issuer ------------------------------------
      constexpr uint32_t IDESC_QK = make_idesc_bf16(BM, BK);
      constexpr uint32_t IDESC_PV = make_idesc_bf16(BM, D) | IDESC_B_MN_MAJOR;
      const uint32_t q_addr = smem_u32(q_sm), k_addr = smem_u32(k_sm), v_addr = smem_u32(v_sm);
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        int ok = 1;
        if (lane == 0) ok = mbar_wait_bounded(bar, parity, a.err, ERR_MBAR_TIMEOUT_MMA, abort_flag, WAIT_NS);
        return __shfl_sync(0xffffffffu, ok, 0) != 0;
      };
      auto stage = [&](int j) { return (int)((kvc + j) % STAGES); };
      auto parity = [&](int j) { return ((kvc + j) / STAGES) & 1u; };
      // scores of block j for stream t; `last` = no other stream reads this K block
      auto issue_qk = [&](int t, int j, bool last) {
        if (lane == 0) {
          const uint32_t qa = q_addr + (two ? t : 0) * C::TILE, ka = k_addr + stage(j) * C::TILE;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_bf16(tmem + (uint32_t)(t * BK), make_sdesc_sw128(qa + (kk >> 2) * C::ATOM) + 2 * (kk & 3),
                      make_sdesc_sw128(ka + (kk >> 2) * C::ATOM) + 2 * (kk & 3), IDESC_QK, kk > 0 ? 1u : 0u);
          umma_commit(&bars->s_full[t]);
          if (last) umma_commit(&bars->k_empty[stage(j)]);
        }
        __syncwarp();
      };
      auto issue_pv = [&](int t, int j, bool first, bool last) {
        if (lane == 0) {
          const uint32_t va = v_addr + stage(j) * C::TILE;
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk)
            umma_bf16_ts(tmem + O_COL + (uint32_t)(t * BK), tmem + (uint32_t)(t * BK + kk * 8),
                         make_sdesc_sw128_mn(va + kk * 2048, C::ATOM, 1024), IDESC_PV, (!first || kk > 0) ? 1u : 0u);
          umma_commit(&bars->o_done[t]);
          if (last) umma_commit(&bars->v_empty[stage(j)]);
        }
        __syncwarp();
      };
      // V rows past the range (a page's tail, or a slice that was not loaded) may hold anything; a zero weight times
      // NaN would reach the output, so they are cleared
      auto clear_tail = [&](int j) {
        const int valid = it.k1 - (it.k0 + j * BK);
        if (valid >= BK) return;
        uint8_t* v = v_sm + stage(j) * C::TILE;
        for (int c = lane; c < (BK - valid) * C::HALVES * 8; c += 32) {
          const int r = valid + c / (C::HALVES * 8), x = c % (C::HALVES * 8);
          *reinterpret_cast<uint4*>(v + (x >> 3) * C::ATOM + r * 128 + ((x & 7) << 4)) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();
        __syncwarp();
      };
      bool ok = nblk == 0 || wait(&bars->q_full, ic & 1u);
      tc_fence_after();
      // the first scores of both streams
      for (int t = 0; t < NS && ok; ++t) {
        const int j = two ? 0 : t;
        if (j >= nblk) break;
        ok = wait(&bars->k_full[stage(j)], parity(j));
        tc_fence_after();
        if (ok) issue_qk(t, j, !two || t == NS - 1);
      }
      const int step = two ? 1 : NS;
      for (int j = 0; j < nblk && ok; ++j) {
        ok = wait(&bars->v_full[stage(j)], parity(j));
        if (!ok) break;
        if (j == nblk - 1) clear_tail(j);
#pragma unroll
        for (int t = 0; t < NS; ++t) {
          if (!ok || (!two && t != (j & 1))) continue;
          ok = wait(&bars->p_full[t], cnt[t] & 1u);  // the softmax wrote P and rescaled O
          if (!ok) continue;
          tc_fence_after();
          issue_pv(t, j, j < step, !two || t == NS - 1);
          ++cnt[t];
          if (j + step < nblk) {
            // these scores overwrite the columns P was in: one thread's products run in the order of issue
            ok = wait(&bars->k_full[stage(j + step)], parity(j + step));
            tc_fence_after();
            if (ok) issue_qk(t, j + step, !two || t == NS - 1);
          }
        }
      }
    } else {
      // ------------------------------------ softmax (warps 2..9) ------------------------------------
      const int t = (warp - 2) >> 2;  // stream
      const int quarter = warp & 3;   // TMEM lanes this warp may access
      const int r = quarter * 32 + lane;
      const int x = (two ? t * BM : 0) + r;  // row of the item
      const bool valid = x < it.rows;
      const int TG = a.T * a.G, hq = a.hkv * a.G;
      long slot = -1, src = -1;
      int lim = 0, low = 0;  // keys [low, lim) of the range are this row's
      if (valid) {
        const int y = it.row0 + x;
        const int b = members(a)[it.moff + y / TG];
        const int tok = (y / a.G) % a.T, head = it.h * a.G + y % a.G;
        const int pos = a.seq_lens[b] - a.T + tok;
        src = ((long)(b * a.T + tok) * hq + head) * D;
        lim = min(it.k1, pos + 1);
        low = a.window > 0 ? pos + 1 - a.window : 0;
        slot = (long)seq_base(a, b) + (long)(tok * hq + head) * seq_prefix_slots(a, b) + it.slot;
        if (slot < 0 || slot >= a.own_at || it.slot >= seq_prefix_slots(a, b)) {
          record_error(a.err, ERR_BAD_ARGUMENT);
          slot = -1;
        }
      }
      row_sm[t * BM + r] = src;
      named_bar_sync(1, NS * BM);
      // gather the query rows (one tile, or one per stream): a row's 16-byte pieces by consecutive lanes, eight loads
      // in flight per thread
      {
        constexpr int CH = D / 8, U = 8;
        const int total = (two ? NS * BM : BM) * CH;
        for (int c0 = threadIdx.x - 64; c0 < total; c0 += U * NS * BM) {
          uint4 v[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int c = c0 + u * NS * BM;
            const long from = c < total ? row_sm[c / CH] : -1;
            v[u] = from >= 0 ? *reinterpret_cast<const uint4*>(a.q + from + (c % CH) * 8) : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int c = c0 + u * NS * BM, rr = c / CH, ch = c % CH, tr = rr & (BM - 1);
            if (c < total)
              *reinterpret_cast<uint4*>(q_sm + (rr / BM) * C::TILE + (ch >> 3) * C::ATOM + tr * 128 + (((ch & 7) ^ (tr & 7)) << 4)) = v[u];
          }
        }
        fence_proxy_async();
        mbar_arrive(&bars->q_full);
      }
      const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
      const uint32_t s_addr = tmem + lane_off + (uint32_t)(t * BK);
      const uint32_t o_addr = tmem + lane_off + O_COL + (uint32_t)(t * BK);
      const bool warp_live = __any_sync(0xffffffffu, valid);
      float m_used = -INFINITY, l = 0.f;
      bool ok = true, any = false;
      for (int j = two ? 0 : t; j < nblk; j += two ? 1 : NS, ++cnt[0]) {
        int okw = 1;
        if (lane == 0)
          okw = mbar_wait_bounded(&bars->s_full[t], cnt[0] & 1u, a.err, ERR_MBAR_TIMEOUT_EPILOGUE, abort_flag, WAIT_NS);
        if (!__shfl_sync(0xffffffffu, okw, 0)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (warp_live) {
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
          float mx[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) mx[c] = __uint_as_float(sv[c]);
#pragma unroll
          for (int c = 8; c < BK; ++c) mx[c & 7] = fmaxf(mx[c & 7], __uint_as_float(sv[c]));
          const float mraw =
              fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7])));
          const float m_new = fmaxf(m_used, mraw * a.scale_log2);
          const bool resc = m_new > m_used + RESCALE;
          float alpha = 1.f;
          if (resc) {
            alpha = ex2_ftz(m_used - m_new);  // 0 when m_used is -inf
            m_used = m_new;
          }
          const float mb = m_used == -INFINITY ? 0.f : m_used;
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
          // the weights are rounded to bf16 for the product (half a step of 2^-8 each); their sum keeps fp32
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
          // the product before this block's scores is complete, so O is stable
          if (any && __any_sync(0xffffffffu, resc)) {
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
        any = true;
        tc_fence_before();
        mbar_arrive(&bars->p_full[t]);
      }
      if (ok && any) {
        int okw = 1;
        if (lane == 0)
          okw = mbar_wait_bounded(&bars->o_done[t], (cnt[0] - 1) & 1u, a.err, ERR_MBAR_TIMEOUT_EPILOGUE, abort_flag, WAIT_NS);
        ok = __shfl_sync(0xffffffffu, okw, 0) != 0;
        tc_fence_after();
      }
      // one row: 16 columns at a time, 16-byte pieces rotated by the row so that a warp's rows fall on all banks
      auto piece = [&](int p) {
        return reinterpret_cast<float4*>(v_sm) + r * (D / 4) + ((p + r) & (D / 4 - 1));
      };
      const bool merge = !two && nblk > 1;
      named_bar_sync(1, NS * BM);  // both streams are done with the rings and the query tiles
      if (ok && merge) {
        if (t == 1) {
          if (warp_live) {
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t ov[16];
              tmem_ld16(o_addr + 16 * c, ov);
              tmem_ld_wait_tied(ov);
#pragma unroll
              for (int p = 0; p < 4; ++p)
                *piece(c * 4 + p) = make_float4(__uint_as_float(ov[4 * p]), __uint_as_float(ov[4 * p + 1]),
                                                __uint_as_float(ov[4 * p + 2]), __uint_as_float(ov[4 * p + 3]));
            }
          }
          ml_sm[r] = make_float2(m_used, l);
        }
      }
      if (merge) named_bar_sync(1, NS * BM);
      if (ok && (two || t == 0) && warp_live) {
        float f0 = 1.f, f1 = 0.f, mo = m_used;
        if (merge) {
          const float2 o = ml_sm[r];
          mo = fmaxf(m_used, o.x);
          if (mo > -INFINITY) {
            f0 = ex2_ftz(m_used - mo);
            f1 = ex2_ftz(o.x - mo);
          }
          l = l * f0 + o.y * f1;
        }
        if (slot >= 0) a.pml[slot] = make_float2(mo, l);
        if (any) {
          // A row is 4 D consecutive bytes in memory but one lane here: it is laid out in shared memory (16 bytes of
          // padding a row keep the lanes on different banks) and leaves in one bulk copy. 256 rows reach into the V
          // ring, one stream's 128 end before it, where the other stream's rows wait to be merged.
          float4* mine = reinterpret_cast<float4*>(q_sm + x * (D * 4 + 16));
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t ov[16];
            tmem_ld16(o_addr + 16 * c, ov);
            tmem_ld_wait_tied(ov);
#pragma unroll
            for (int p = 0; p < 4; ++p) {
              float4 v = make_float4(__uint_as_float(ov[4 * p]), __uint_as_float(ov[4 * p + 1]),
                                     __uint_as_float(ov[4 * p + 2]), __uint_as_float(ov[4 * p + 3]));
              if (merge) {
                const float4 w = *piece(c * 4 + p);
                v = make_float4(v.x * f0 + w.x * f1, v.y * f0 + w.y * f1, v.z * f0 + w.z * f1, v.w * f0 + w.w * f1);
              }
              mine[c * 4 + p] = v;
            }
          }
          fence_proxy_async();
          if (slot >= 0 && l > 0.f) {
            bulk_store(a.po + slot * D, mine, D * 4);
            bulk_commit_wait_read();
          }
        }
      }
      tc_fence_before();
      fence_proxy_async();  // the rings are written by TMA again
    }
    kvc += nblk;
    __syncthreads();
    tc_fence_after();
    if (bars->abort) break;
  }
  // every product issued above has completed before TMEM is released
  if (warp == 1 && lane == 0) {
    umma_commit(&bars->mma_done);
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(&bars->mma_done, 0) && globaltimer_ns() - t0 < 50000000ull) {
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, TMEM_COLS);
}

}  // namespace

template <int D>
cudaError_t launch_prefix(const Args& a, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t st) {
  auto kern = prefix_kernel<D>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes<D>());
  if (e != cudaSuccess) return e;
  return launch_k(kern, dim3((unsigned)min(a.n_prefix, a.num_sms)), dim3(THREADS), smem_bytes<D>(), st, tk, tv, a);
}
template cudaError_t launch_prefix<64>(const Args&, const CUtensorMap&, const CUtensorMap&, cudaStream_t);
template cudaError_t launch_prefix<128>(const Args&, const CUtensorMap&, const CUtensorMap&, cudaStream_t);

}  // namespace shared_attn
}  // namespace mesh
