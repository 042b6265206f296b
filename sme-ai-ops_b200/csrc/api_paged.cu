// api_paged.cu -- the C-ABI of include/smeai_paged.h.
#include <math.h>

#include <atomic>

#include "common.cuh"
#include "paged.h"
#include "runtime.h"
#include "../../include/smeai_paged.h"

using namespace smeai;

namespace {

cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }

int bad(const char* what, const char* why) {
  set_last_error("%s: %s", what, why);
  return kBadArgument;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int log2_of(int64_t n) {   // -1: not a power of two
  if (n <= 0 || (n & (n - 1))) return -1;
  int l = 0;
  while ((int64_t)1 << l < n) ++l;
  return l;
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr int64_t kMaxStride = (int64_t)1 << 40;   // elements; keeps every byte offset inside 64 bits

int view(const char* what, const smeai_kv_cache* c, KvView* v) {
  if (!c || !c->k || !c->v) return bad(what, "NULL cache");
  if (c->type != SMEAI_KV_F16 && c->type != SMEAI_KV_BF16) return bad(what, "the cache's type is F16 or BF16");
  const int log2 = log2_of(c->page_size);
  if (log2 < 0 || log2 > 16) return bad(what, "page_size is a power of two up to 65536");
  if (c->head_dim <= 0 || c->head_dim % 8 || c->head_dim > 256)
    return bad(what, "head_dim is a multiple of 8 up to 256");
  if (c->n_kv_heads <= 0 || c->n_pages <= 0 || c->n_pages > 0x7fffffff) return bad(what, "no key heads or no pages");
  if (!aligned16(c->k) || !aligned16(c->v)) return bad(what, "k and v are 16-byte aligned");
  const int64_t s[3] = {c->page_stride, c->head_stride, c->token_stride};
  for (int64_t x : s)
    if (x < 0 || x % 8 || x > kMaxStride) return bad(what, "strides are non-negative multiples of 8 elements");
  if ((c->n_pages > 1 && c->page_stride < c->head_dim) || (c->n_kv_heads > 1 && c->head_stride < c->head_dim) ||
      (c->page_size > 1 && c->token_stride < c->head_dim))
    return bad(what, "a stride is smaller than head_dim: rows overlap");
  v->k = static_cast<char*>(c->k);
  v->v = static_cast<char*>(c->v);
  v->page_bytes = c->page_stride * 2;
  v->head_bytes = c->head_stride * 2;
  v->token_bytes = c->token_stride * 2;
  v->n_pages = c->n_pages;
  v->page_log2 = log2;
  v->n_kv = c->n_kv_heads;
  v->dim = c->head_dim;
  v->bf16 = c->type == SMEAI_KV_BF16;
  return kOk;
}

// Whether the current device can run the kernels; what was found is kept, a
// device's compute capability does not change.
int ready(const char* what) {
  static std::atomic<uint64_t> good{0};
  int dev = 0;
  if (good.load() && cudaGetDevice(&dev) == cudaSuccess && dev < 64 && (good.load() >> dev & 1)) return kOk;
  if (device_ready()) {
    if (cudaGetDevice(&dev) == cudaSuccess && dev < 64) good.fetch_or((uint64_t)1 << dev);
    return kOk;
  }
  set_last_error("%s: no compute-capability-10.x device", what);
  return kUnsupported;
}

int attention_args(const char* what, const smeai_kv_cache* cache, int n_heads, int64_t n_tokens, int64_t n_req,
                   int64_t max_blocks, int64_t max_new, PagedAttention* a) {
  const int st = view(what, cache, &a->kv);
  if (st) return st;
  if (n_heads <= 0 || n_heads % a->kv.n_kv) return bad(what, "n_heads is a multiple of n_kv_heads");
  if (n_req <= 0 || n_req > 0x3fffffff || n_tokens < 0 || max_blocks < 0 || max_new < 0)
    return bad(what, "a count is negative, or n_req is 0");
  if (n_tokens > (0x7fffffff - 512) / (int64_t)n_heads) return bad(what, "n_tokens * n_heads passes 2^31");
  a->n_heads = n_heads;
  a->n_tokens = n_tokens;
  a->n_req = (int)n_req;
  a->max_new = max_new < n_tokens ? max_new : n_tokens;
  if (a->max_new < 1) a->max_new = 1;
  const int64_t top = (0x7fffffff - 512) >> a->kv.page_log2;   // table entries that 31-bit positions reach
  a->max_kv = (int)((max_blocks < top ? max_blocks : top) << a->kv.page_log2);
  return kOk;
}

}  // namespace

extern "C" {

int smeai_paged_plan(const int32_t* cached_len, const int32_t* new_len, int64_t n_req, int page_size,
                     const int32_t* free_pages, int64_t n_free, const int32_t* n_used, int32_t* n_used_out,
                     int32_t* block_table, int64_t ld_table, int64_t max_blocks, int32_t* q_start, int32_t* kv_len,
                     int64_t* slots, int32_t* positions, int64_t n_tokens, void* stream) {
  const char* what = "smeai_paged_plan";
  if (!cached_len || !new_len || !n_used || !n_used_out || !block_table || !q_start || !kv_len ||
      (n_free > 0 && !free_pages) || (n_tokens > 0 && (!slots || !positions)))
    return bad(what, "NULL pointer");
  if (n_req <= 0 || n_req > 8192) return bad(what, "n_req is 1 to 8192");
  const int log2 = log2_of(page_size);
  if (log2 < 0 || log2 > 16) return bad(what, "page_size is a power of two up to 65536");
  if (n_free < 0 || n_free > 0x7fffffff || n_tokens < 0 || n_tokens > 0x7fffffff)
    return bad(what, "n_free and n_tokens are 0 to 2^31 - 1");
  if (max_blocks <= 0 || ld_table < max_blocks) return bad(what, "max_blocks is positive and at most ld_table");
  const int st = ready(what);
  if (st) return st;
  return paged_plan(cached_len, new_len, (int)n_req, log2, free_pages, n_free, n_used, n_used_out, block_table,
                    ld_table, max_blocks, q_start, kv_len, slots, positions, n_tokens, as_stream(stream));
}

int smeai_paged_append(const smeai_kv_cache* cache, const float* k, int64_t ld_k, const float* v, int64_t ld_v,
                       const float* q, int64_t ld_q, int n_heads, void* q_out, int64_t ld_q_out, int64_t n_tokens,
                       const int64_t* slots, const int32_t* positions, const float* rope, int64_t n_rope, int halves,
                       void* stream) {
  const char* what = "smeai_paged_append";
  KvView kv;
  int st = view(what, cache, &kv);
  if (st) return st;
  if (n_tokens == 0) return kOk;
  if (!k || !v || !slots) return bad(what, "NULL pointer");
  if (n_tokens < 0 || n_tokens > 0x7fffffff) return bad(what, "n_tokens is 0 to 2^31 - 1");
  const int64_t kv_row = (int64_t)kv.n_kv * kv.dim;
  if (ld_k < kv_row || ld_v < kv_row || ld_k > kMaxStride || ld_v > kMaxStride)
    return bad(what, "a row stride of k or v is smaller than n_kv_heads * head_dim");
  if (!q != !q_out) return bad(what, "q and q_out come together");
  if (q) {
    if (n_heads <= 0) return bad(what, "n_heads is positive");
    const int64_t q_row = (int64_t)n_heads * kv.dim;
    if (ld_q < q_row || ld_q_out < q_row || ld_q > kMaxStride || ld_q_out > kMaxStride)
      return bad(what, "a row stride of q or q_out is smaller than n_heads * head_dim");
    if (!aligned16(q_out) || ld_q_out % 8) return bad(what, "rows of q_out are 16-byte aligned");
    if ((int64_t)n_heads + 2 * (int64_t)kv.n_kv > 0xffff) return bad(what, "too many heads");
  }
  if (rope && (!positions || n_rope <= 0)) return bad(what, "rope needs positions and n_rope rows");
  if (kv.n_kv > 0x7fff) return bad(what, "too many heads");
  st = ready(what);
  if (st) return st;
  return paged_append(kv, k, ld_k, v, ld_v, q, ld_q, n_heads, q_out, ld_q_out, n_tokens, slots, positions, rope,
                      n_rope, halves != 0, as_stream(stream));
}

size_t smeai_paged_attention_workspace(const smeai_kv_cache* cache, int n_heads, int64_t n_tokens, int64_t n_req,
                                       int64_t max_blocks, int64_t max_new) {
  PagedAttention a;
  if (attention_args("smeai_paged_attention_workspace", cache, n_heads, n_tokens, n_req, max_blocks, max_new, &a))
    return 0;
  return paged_attention_workspace(a);
}

int smeai_paged_attention(const smeai_kv_cache* cache, const void* q, int64_t ld_q, int n_heads, int64_t n_tokens,
                          const int32_t* q_start, const int32_t* kv_len, int64_t n_req, const int32_t* block_table,
                          int64_t ld_table, int64_t max_blocks, int64_t max_new, float scale, int causal, void* out,
                          int64_t ld_out, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "smeai_paged_attention";
  PagedAttention a;
  int st = attention_args(what, cache, n_heads, n_tokens, n_req, max_blocks, max_new, &a);
  if (st) return st;
  if (n_tokens == 0) return kOk;
  if (!q || !out || !q_start || !kv_len || !block_table) return bad(what, "NULL pointer");
  const int64_t row = (int64_t)n_heads * a.kv.dim;
  if (ld_q < row || ld_out < row || ld_q > kMaxStride || ld_out > kMaxStride)
    return bad(what, "a row stride of q or out is smaller than n_heads * head_dim");
  if (!aligned16(q) || !aligned16(out) || ld_q % 8 || ld_out % 8) return bad(what, "rows of q and out are 16-byte aligned");
  if (ld_table < max_blocks) return bad(what, "ld_table is at least max_blocks");
  if (!(scale > 0.f) || isinf(scale * kLog2e)) return bad(what, "scale is positive and at most 2e38");
  st = ready(what);
  if (st) return st;
  const size_t need = paged_attention_workspace(a);
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255))) {
    set_last_error("%s: needs a 256-byte aligned workspace of %zu bytes", what, need);
    return !workspace || workspace_bytes < need ? kWorkspaceTooSmall : kBadArgument;
  }
  a.q = q;
  a.ld_q = ld_q;
  a.out = out;
  a.ld_out = ld_out;
  a.q_start = q_start;
  a.kv_len = kv_len;
  a.table = block_table;
  a.ld_table = ld_table;
  a.scale = scale;
  a.causal = causal != 0;
  a.workspace = workspace;
  return paged_attention(a, as_stream(stream));
}

}  // extern "C"
