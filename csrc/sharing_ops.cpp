// Tensor front-end of the sharing operators: argument checks, then the kernels' launchers on the current stream.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <climits>
#include <string>
#include <tuple>

#include "include/sharing.h"

namespace mesh {
namespace {

std::string num(int64_t n) { return std::to_string(n); }

void check_pools(const char* what, const at::Tensor& k_pool, const at::Tensor& v_pool) {
  TORCH_CHECK(k_pool.is_cuda() && v_pool.device() == k_pool.device() && k_pool.dim() == 5 &&
                  k_pool.sizes() == v_pool.sizes() && k_pool.is_contiguous() && v_pool.is_contiguous(),
              what, ": contiguous pools [layers, pages, kv_heads, page, D] on one GPU");
  TORCH_CHECK(k_pool.scalar_type() == at::kBFloat16 && v_pool.scalar_type() == at::kBFloat16, what, ": bf16 pools");
  TORCH_CHECK(k_pool.numel() > 0, what, ": empty pools");
  TORCH_CHECK(k_pool.size(4) % 8 == 0, what, ": a token of a head must be a multiple of 16 bytes");
  TORCH_CHECK((uintptr_t)k_pool.data_ptr() % 16 == 0 && (uintptr_t)v_pool.data_ptr() % 16 == 0, what,
              ": pools must be 16-byte aligned");
  TORCH_CHECK(k_pool.size(0) < 65536 && k_pool.size(1) < INT_MAX, what, ": too many layers or pages");
}

std::string dims(at::IntArrayRef shape) {
  std::string s = "[";
  for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + num(shape[i]);
  return s + "]";
}

void check_tensor(const char* what, const char* name, const at::Tensor& x, const at::Tensor& like, at::ScalarType type,
                  at::IntArrayRef shape) {
  TORCH_CHECK(x.device() == like.device() && x.scalar_type() == type && x.sizes() == shape && x.is_contiguous(),
              std::string(what) + ": " + name + " must be contiguous " + c10::toString(type) + " " + dims(shape) + " on " +
                  like.device().str() + ", got " + c10::toString(x.scalar_type()) + " " + dims(x.sizes()) + " on " +
                  x.device().str());
}

}  // namespace

void kv_pages_move(at::Tensor& k_pool, at::Tensor& v_pool, const at::Tensor& src, const at::Tensor& dst,
                   const c10::optional<at::Tensor>& tokens, at::Tensor& err) {
  check_pools("kv_pages_copy", k_pool, v_pool);
  TORCH_CHECK(src.dim() == 1, "kv_pages_copy: page ids [pairs]");
  const int64_t n = src.size(0);
  check_tensor("kv_pages_copy", "src", src, k_pool, at::kInt, {n});
  check_tensor("kv_pages_copy", "dst", dst, k_pool, at::kInt, {n});
  if (tokens.has_value()) check_tensor("kv_pages_copy", "tokens", *tokens, k_pool, at::kInt, {n});
  TORCH_CHECK(n < INT_MAX, "kv_pages_copy: too many pairs");
  if (n == 0) return;
  const c10::cuda::CUDAGuard guard(k_pool.device());
  KvMoveArgs a;
  a.k = k_pool.data_ptr();
  a.v = v_pool.data_ptr();
  a.src = src.data_ptr<int>();
  a.dst = dst.data_ptr<int>();
  a.tokens = tokens.has_value() ? tokens->data_ptr<int>() : nullptr;
  a.n = (int)n;
  a.layers = (int)k_pool.size(0);
  a.heads = (int)k_pool.size(2);
  a.page_size = (int)k_pool.size(3);
  a.row_vec = (int)(k_pool.size(4) / 8);
  a.pool_pages = k_pool.size(1);
  a.err = err.data_ptr<int>();
  C10_CUDA_CHECK(launch_kv_move(a, at::cuda::getCurrentCUDAStream()));
}

// Returns (tables, remap [pages], live [1]).
std::tuple<at::Tensor, at::Tensor, at::Tensor> kv_pages_compact(at::Tensor& k_pool, at::Tensor& v_pool,
                                                                const at::Tensor& tables, const at::Tensor& counts,
                                                                const c10::optional<at::Tensor>& out, int64_t reserved,
                                                                at::Tensor& err) {
  check_pools("kv_pages_compact", k_pool, v_pool);
  TORCH_CHECK(tables.dim() == 2, "kv_pages_compact: block tables [rows, width]");
  const int64_t pages = k_pool.size(1), rows = tables.size(0), width = tables.size(1);
  check_tensor("kv_pages_compact", "block tables", tables, k_pool, at::kInt, {rows, width});
  if (out.has_value()) check_tensor("kv_pages_compact", "out_tables", *out, k_pool, at::kInt, {rows, width});
  check_tensor("kv_pages_compact", "counts", counts, k_pool, at::kInt, {rows});
  TORCH_CHECK(reserved >= 0 && reserved <= pages, "kv_pages_compact: " + num(reserved) + " reserved pages in a pool of " + num(pages));
  TORCH_CHECK(kv_compact_smem(pages) <= 200 * 1024, "kv_pages_compact: at most 819200 pages");
  TORCH_CHECK(rows < INT_MAX && width < INT_MAX, "kv_pages_compact: tables too large");
  const c10::cuda::CUDAGuard guard(k_pool.device());
  at::Tensor out_tables = out.has_value() ? *out : at::empty({rows, width}, tables.options());
  at::Tensor ws = at::empty({3 * pages + 2}, tables.options());
  KvCompactArgs a;
  a.k = k_pool.data_ptr();
  a.v = v_pool.data_ptr();
  a.tables = tables.data_ptr<int>();
  a.counts = counts.data_ptr<int>();
  a.out_tables = out_tables.data_ptr<int>();
  a.ws = ws.data_ptr<int>();
  a.err = err.data_ptr<int>();
  a.rows = (int)rows;
  a.width = (int)width;
  a.layers = (int)k_pool.size(0);
  a.reserved = (int)reserved;
  a.num_sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  a.pool_pages = pages;
  a.page_vec = k_pool.size(2) * k_pool.size(3) * (k_pool.size(4) / 8);
  C10_CUDA_CHECK(launch_kv_compact(a, at::cuda::getCurrentCUDAStream()));
  return {out_tables, ws.narrow(0, 0, pages), ws.narrow(0, pages, 1)};
}

// Returns (tokens [B, K+1] int32, accepted [B] int32, probs [B, K] fp32).
std::tuple<at::Tensor, at::Tensor, at::Tensor> verify_drafts(const at::Tensor& logits, const at::Tensor& ids,
                                                             const at::Tensor& uniforms,
                                                             const c10::optional<at::Tensor>& inv_t,
                                                             const c10::optional<at::Tensor>& probs,
                                                             const c10::optional<at::Tensor>& lens) {
  const char* what = "verify_drafts";
  const at::Tensor& x = logits;
  TORCH_CHECK(x.is_cuda() && x.dim() == 3 && x.size(1) >= 1 && x.size(2) >= 1 && x.stride(2) == 1 &&
                  (x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16),
              what, ": logits [B, K+1, V] fp32 or bf16 on a GPU, vocabulary contiguous");
  const int64_t B = x.size(0), K = x.size(1) - 1, V = x.size(2);
  TORCH_CHECK(K <= VERIFY_MAX_DRAFTS, std::string(what) + ": " + num(K) + " drafts a session, at most " + num(VERIFY_MAX_DRAFTS));
  check_tensor(what, "draft_ids", ids, x, at::kInt, {B, K});
  check_tensor(what, "uniforms", uniforms, x, at::kFloat, {B, K + 1});
  if (inv_t.has_value()) check_tensor(what, "inv_t", *inv_t, x, at::kFloat, {B});
  if (lens.has_value()) check_tensor(what, "draft_lens", *lens, x, at::kInt, {B});
  if (probs.has_value())
    TORCH_CHECK(probs->device() == x.device() && probs->dim() == 3 && probs->size(0) == B && probs->size(1) == K &&
                    probs->size(2) == V && probs->stride(2) == 1 &&
                    (probs->scalar_type() == at::kFloat || probs->scalar_type() == at::kBFloat16),
                what, ": draft_probs [B, K, V] fp32 or bf16 on the logits' device, vocabulary contiguous");
  const bool qs = probs.has_value() && K > 0;
  TORCH_CHECK(V <= verify_max_vocab(), std::string(what) + ": a vocabulary of " + num(V) + ", at most " + num(verify_max_vocab()));
  TORCH_CHECK(B * (K + 1) <= 65535, std::string(what) + ": " + num(B * (K + 1)) + " rows, at most 65535");
  const c10::cuda::CUDAGuard guard(x.device());
  const auto ints = x.options().dtype(at::kInt);
  at::Tensor tokens = at::empty({B, K + 1}, ints), accepted = at::empty({B}, ints);
  at::Tensor draft_p = at::empty({B, K}, x.options().dtype(at::kFloat));
  if (B == 0) return {tokens, accepted, draft_p};
  at::Tensor parts = at::empty({verify_parts_bytes(B, K, V)}, x.options().dtype(at::kByte));
  VerifyArgs a;
  a.logits = x.data_ptr();
  a.ids = ids.data_ptr<int>();
  a.uniforms = uniforms.data_ptr<float>();
  a.inv_t = inv_t.has_value() ? inv_t->data_ptr<float>() : nullptr;
  a.probs = qs ? probs->data_ptr() : nullptr;
  a.lens = lens.has_value() ? lens->data_ptr<int>() : nullptr;
  a.parts = parts.data_ptr();
  a.tokens = tokens.data_ptr<int>();
  a.accepted = accepted.data_ptr<int>();
  a.draft_p = draft_p.data_ptr<float>();
  a.ld_row = x.stride(1);
  a.ld_seq = x.stride(0);
  a.lq_row = qs ? probs->stride(1) : 0;
  a.lq_seq = qs ? probs->stride(0) : 0;
  a.B = (int)B;
  a.K = (int)K;
  a.V = (int)V;
  a.chunks = verify_chunks(B, K, V);
  a.logits_bf16 = x.scalar_type() == at::kBFloat16;
  a.probs_bf16 = qs && probs->scalar_type() == at::kBFloat16;
  C10_CUDA_CHECK(launch_verify(a, at::cuda::getCurrentCUDAStream()));
  return {tokens, accepted, draft_p};
}

// n_items prefix items now; a captured call is launched for item_cap, the most there can be. Returns the kernels launched.
int64_t attn_shared(const at::Tensor& q, const at::Tensor& kcache, const at::Tensor& vcache, const at::Tensor& block_tables,
                    const at::Tensor& seq_lens, at::Tensor& meta, at::Tensor& po, at::Tensor& pml, at::Tensor& out,
                    at::Tensor& err, int64_t n_items, int64_t item_cap, int64_t own_at, double scale, int64_t window) {
  const char* what = "attn_shared_prefix";
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kBFloat16 && q.is_contiguous() && q.dim() == 2, what,
              ": q contiguous bf16 [B * T, hq * D] on a GPU");
  check_tensor(what, "out", out, q, at::kBFloat16, q.sizes());
  TORCH_CHECK((uintptr_t)q.data_ptr() % 16 == 0 && (uintptr_t)out.data_ptr() % 16 == 0, what, ": q and out must be 16-byte aligned");
  TORCH_CHECK(kcache.dim() == 4, what, ": cache [pages, hkv, page, D]");
  check_tensor(what, "kcache", kcache, q, at::kBFloat16, kcache.sizes());
  check_tensor(what, "vcache", vcache, q, at::kBFloat16, kcache.sizes());
  const int64_t hkv = kcache.size(1), ps = kcache.size(2), D = kcache.size(3);
  TORCH_CHECK(D == 64 || D == 128, std::string(what) + ": head_dim " + num(D) + ", must be 64 or 128");
  TORCH_CHECK(ps > 0 && ps % 16 == 0, std::string(what) + ": pages of " + num(ps) + " tokens, must be a multiple of 16");
  TORCH_CHECK(seq_lens.dim() == 1 && block_tables.dim() == 2, what, ": block_tables [B, pages], seq_lens [B]");
  const int64_t B = seq_lens.size(0);
  check_tensor(what, "seq_lens", seq_lens, q, at::kInt, {B});
  check_tensor(what, "block_tables", block_tables, q, at::kInt, {B, block_tables.size(1)});
  if (B == 0) return 0;
  TORCH_CHECK(q.size(0) % B == 0 && q.size(1) % D == 0, std::string(what) + ": q " + dims(q.sizes()) + " for " + num(B) + " sequences of head_dim " + num(D));
  const int64_t T = q.size(0) / B, hq = q.size(1) / D;
  TORCH_CHECK(hkv > 0 && hq % hkv == 0, std::string(what) + ": " + num(hq) + " query heads over " + num(hkv) + " KV heads");
  const int64_t G = hq / hkv;
  TORCH_CHECK(T >= 1 && T * G <= SHARED_MAX_ROWS, std::string(what) + ": " + num(T) + " new tokens x " + num(G) +
              " heads of a KV group, at most " + num(SHARED_MAX_ROWS) + " rows");
  TORCH_CHECK(meta.device() == q.device() && meta.scalar_type() == at::kInt && meta.is_contiguous() &&
                  meta.numel() >= shared_items_at((int)B) + SHARED_ITEM * std::max(n_items, item_cap) && (uintptr_t)meta.data_ptr() % 16 == 0,
              what, ": groups of another batch");
  TORCH_CHECK(po.scalar_type() == at::kFloat && pml.scalar_type() == at::kFloat && po.device() == q.device() &&
                  pml.device() == q.device() && po.numel() / D <= pml.numel() / 2,
              what, ": workspace");
  TORCH_CHECK(B <= SHARED_MAX_BATCH, std::string(what) + ": a batch of " + num(B) + ", at most " + num(SHARED_MAX_BATCH));
  const int64_t own_slots = (SHARED_OWN_WORKERS * at::cuda::getDeviceProperties(q.get_device())->multiProcessorCount +
                             B * hkv * ((T * G + SHARED_OWN_ROWS - 1) / SHARED_OWN_ROWS)) *
                            std::min<int64_t>(SHARED_OWN_ROWS, T * G);
  TORCH_CHECK(own_at >= 0 && (own_at + own_slots) * D <= po.numel(), what, ": workspace too small");
  TORCH_CHECK(kcache.size(0) * hkv * ps < (1ll << 31), what, ": KV pool too large for 32-bit TMA rows");
  TORCH_CHECK(block_tables.size(1) * ps < (1ll << 31), what, ": block tables too wide");
  // the own keys of a call are counted in slices of 16, for every (sequence, KV head, tile of rows), in 32 bits
  const int64_t tiles = (T * G + SHARED_OWN_ROWS - 1) / SHARED_OWN_ROWS;
  TORCH_CHECK(B * hkv * tiles * (block_tables.size(1) * ps / 16 + 4) < (1ll << 30), what,
              ": the block tables hold more keys than one call can attend");
  const c10::cuda::CUDAGuard guard(q.device());
  SharedAttnArgs a;
  a.q = static_cast<const __nv_bfloat16*>(q.data_ptr());
  a.k = kcache.data_ptr();
  a.v = vcache.data_ptr();
  a.block_tables = block_tables.data_ptr<int>();
  a.seq_lens = seq_lens.data_ptr<int>();
  a.meta = meta.data_ptr<int>();
  a.po = po.data_ptr<float>();
  a.pml = reinterpret_cast<float2*>(pml.data_ptr<float>());
  a.out = static_cast<__nv_bfloat16*>(out.data_ptr());
  a.err = err.data_ptr<int>();
  a.B = (int)B;
  a.T = (int)T;
  a.G = (int)G;
  a.hkv = (int)hkv;
  a.max_pages = (int)block_tables.size(1);
  a.page_size = (int)ps;
  a.n_prefix = (int)(c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None ? n_items : item_cap);
  a.own_at = own_at;
  a.window = (int)std::min<int64_t>(window, 1 << 30);  // positions are subtracted from it in 32 bits
  a.slot_cap = po.numel() / D;
  a.num_sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  a.pool_pages = kcache.size(0);
  C10_CUDA_CHECK(launch_attn_shared(a, (int)D, scale, at::cuda::getCurrentCUDAStream()));
  return a.n_prefix > 0 ? 3 : 2;
}

}  // namespace mesh
