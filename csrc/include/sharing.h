// Plain-pointer interfaces between the kernels of the sharing operators (attn_shared.cu, kv_moves.cu, verify.cu) and
// their tensor front-end (sharing_ops.cpp). The kernels' files include no tensor headers, so they build in seconds.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace mesh {

// Copies inside the pools: pairs of pages, optionally their first tokens only.
struct KvMoveArgs {
  void *k, *v;                      // pools, 16-byte aligned
  const int *src, *dst, *tokens;    // [n]; tokens may be null
  int n, layers, heads, page_size, row_vec;  // row_vec: 16-byte vectors of one token of one head
  long pool_pages;
  int* err;
};
cudaError_t launch_kv_move(const KvMoveArgs& a, cudaStream_t st);

// Compaction. ws int32 [3 * pages + 2]: remap, live count, number of moves, then sources and destinations.
struct KvCompactArgs {
  void *k, *v;
  const int *tables, *counts;       // [rows, width], [rows]
  int *out_tables, *ws, *err;
  int rows, width, layers, reserved, num_sms;
  long pool_pages, page_vec;        // page_vec: 16-byte vectors of one page of one layer
};
inline size_t kv_compact_smem(long pages) { return (size_t)((pages + 31) / 32) * 8; }
cudaError_t launch_kv_compact(const KvCompactArgs& a, cudaStream_t st);

// Draft verification.
constexpr int VERIFY_MAX_DRAFTS = 31;
struct VerifyArgs {
  const void* logits;       // [B, K + 1, V] fp32 or bf16
  const int* ids;           // [B, K]
  const float* uniforms;    // [B, K + 1]
  const float* inv_t;       // [B] or null (1)
  const void* probs;        // [B, K, V] fp32 or bf16, or null
  const int* lens;          // [B] or null (K)
  void* parts;              // verify_parts_bytes
  int* tokens;              // [B, K + 1]
  int* accepted;            // [B]
  float* draft_p;           // [B, K]
  long ld_row, ld_seq;      // strides of logits
  long lq_row, lq_seq;      // strides of probs
  int B, K, V, chunks;
  bool logits_bf16, probs_bf16;
};
int verify_chunks(int64_t B, int64_t K, int64_t V);
int64_t verify_max_vocab();
int64_t verify_parts_bytes(int64_t B, int64_t K, int64_t V);
cudaError_t launch_verify(const VerifyArgs& a, cudaStream_t st);

// Attention over shared prefixes.
constexpr int SHARED_OWN_ROWS = 8;   // query rows of one worker on a sequence's own keys
constexpr int SHARED_OWN_WORKERS = 12;  // such workers per SM at most
constexpr int SHARED_MAX_ROWS = 64;  // query rows (new tokens x heads of a KV group) of one sequence
constexpr int SHARED_HDR = 8;        // header ints of meta, [0] = number of prefix items
constexpr int SHARED_ITEM = 8;       // ints per prefix item
inline
#ifdef __CUDACC__
    __host__ __device__
#endif
    int shared_items_at(int batch) { return SHARED_HDR + ((5 * batch + 2 + 3) & ~3); }  // items start on 16 bytes
constexpr int SHARED_MAX_BATCH = 1024;
// meta layout: header | per sequence: prefix length, first partial slot, prefix slots per row | member lists |
// scratch [B + 2] | items {first member, offset of the members, first row, rows, KV head, first key, end key, slot}
struct SharedAttnArgs {
  const __nv_bfloat16* q;   // [B * T, hq, D]
  const void *k, *v;        // [pages, hkv, page_size, D]
  const int* block_tables;  // [B, max_pages]
  const int* seq_lens;      // [B] keys including the new tokens
  int* meta;
  float* po;                // partial outputs [slots, D]
  float2* pml;              // partial (m, l) [slots]
  __nv_bfloat16* out;
  int* err;
  int B, T, G, hkv, max_pages, page_size, n_prefix, window, num_sms;
  long slot_cap, own_at, pool_pages;  // own_at: first slot of the partials of own keys
};
cudaError_t launch_attn_shared(const SharedAttnArgs& a, int head_dim, double scale, cudaStream_t st);

}  // namespace mesh
