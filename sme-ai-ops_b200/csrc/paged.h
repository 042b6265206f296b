// paged.h -- host-side launchers of the paged key/value cache kernels
// (internal; the public C entry points are in include/smeai_paged.h).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace smeai {

// The cache as the kernels see it: byte strides, page number and place of a
// slot by shift and mask.
struct KvView {
  char* k = nullptr;
  char* v = nullptr;
  int64_t page_bytes = 0, head_bytes = 0, token_bytes = 0;
  int64_t n_pages = 0;
  int page_log2 = 0;
  int n_kv = 0, dim = 0;
  bool bf16 = false;
};

int paged_plan(const int32_t* cached_len, const int32_t* new_len, int n_req, int page_log2, const int32_t* free_pages,
               int64_t n_free, const int32_t* n_used, int32_t* n_used_out, int32_t* table, int64_t ld_table,
               int64_t max_blocks, int32_t* q_start, int32_t* kv_len, int64_t* slots, int32_t* positions,
               int64_t n_tokens, cudaStream_t stream);

int paged_append(const KvView& kv, const float* k, int64_t ld_k, const float* v, int64_t ld_v, const float* q,
                 int64_t ld_q, int n_heads, void* q_out, int64_t ld_q_out, int64_t n_tokens, const int64_t* slots,
                 const int32_t* positions, const float* rope, int64_t n_rope, bool halves, cudaStream_t stream);

struct PagedAttention {
  KvView kv;
  const void* q = nullptr;
  int64_t ld_q = 0;
  void* out = nullptr;
  int64_t ld_out = 0;
  int n_heads = 0;
  int64_t n_tokens = 0;
  const int32_t *q_start = nullptr, *kv_len = nullptr, *table = nullptr;
  int n_req = 0;
  int64_t ld_table = 0;
  int max_kv = 0;        // keys that a table row can name
  int64_t max_new = 0;
  float scale = 0.f;
  bool causal = false;
  void* workspace = nullptr;
};
size_t paged_attention_workspace(const PagedAttention& a);
int paged_attention(const PagedAttention& a, cudaStream_t stream);

int sm_count(int* n);   // of the current device

}  // namespace smeai
