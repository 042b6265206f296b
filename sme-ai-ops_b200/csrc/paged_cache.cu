// paged_cache.cu -- a serving step's bookkeeping (block table, row offsets,
// slots, positions from the requests' lengths) and the writing of its keys
// and values into their slots.
#include <cuda_bf16.h>

#include <atomic>

#include "common.cuh"
#include "paged.h"

namespace smeai {

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanMaxReq = 8192;
// Tokens that the planning CTA maps to slots itself: 8 a thread.  Above, a
// second kernel maps them with the whole GPU.
constexpr int64_t kPlanOwnTokens = 8 * kPlanThreads;

// Block-wide inclusive scan of (rows, pages); `carry` is added to every lane
// and advanced by the block's sum.
__device__ void scan2(int64_t& a, int64_t& b, int64_t (&carry)[2], int64_t (*warp_sum)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t ta = __shfl_up_sync(0xffffffffu, a, off), tb = __shfl_up_sync(0xffffffffu, b, off);
    if (lane >= off) {
      a += ta;
      b += tb;
    }
  }
  if (lane == 31) {
    warp_sum[warp][0] = a;
    warp_sum[warp][1] = b;
  }
  __syncthreads();
  int64_t la = lane < nw ? warp_sum[lane][0] : 0, lb = lane < nw ? warp_sum[lane][1] : 0;
  int64_t pa = lane < warp ? la : 0, pb = lane < warp ? lb : 0;
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    pa += __shfl_xor_sync(0xffffffffu, pa, off);
    pb += __shfl_xor_sync(0xffffffffu, pb, off);
    la += __shfl_xor_sync(0xffffffffu, la, off);
    lb += __shfl_xor_sync(0xffffffffu, lb, off);
  }
  a += carry[0] + pa;
  b += carry[1] + pb;
  carry[0] += la;
  carry[1] += lb;
  __syncthreads();   // warp_sum is free again
}

// The request of row t: the last r with start[r] <= t, start ascending.
__device__ __forceinline__ int row_request(const int* start, int n_req, int t) {
  int lo = 0, hi = n_req;   // start[lo] <= t < start[hi], start[n_req] taken as past the end
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

struct PlanParams {
  const int32_t *cached, *fresh;
  int n_req, page_log2;
  const int32_t* free_pages;
  int64_t n_free;
  const int32_t* n_used;
  int32_t* n_used_out;
  int32_t* table;
  int64_t ld_table, max_blocks;
  int32_t *q_start, *kv_len;
  int64_t* slots;
  int32_t* positions;
  int64_t n_tokens;
  unsigned* err;
};

// One CTA: two running sums over the requests (rows, pages) decide who is
// served, a thread a page writes the new table entries, and, for a step of up
// to kPlanOwnTokens rows, a thread a row maps rows to slots -- a new page
// straight from the pool, an old one from the table, so nothing waits for the
// table's writes.  The lengths are read once, before anything is written, so
// they may lie where kv_len or q_start go.  A few KB of traffic: bound by the
// latency of its dependent loads.  Measured: 3.4 us for 48 decoding requests,
// 7.7 us for 200 prompts of 51k rows, the second kernel included.
__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PlanParams p) {
  extern __shared__ int plan_smem[];
  int* start = plan_smem;                    // [n_req + 1] first row of each request, cut at n_tokens
  int* first = plan_smem + p.n_req + 1;      // [n_req] pages asked for ahead of it, its own pool index if it is served
  int* held_len = first + p.n_req;           // [n_req] cached tokens; ~ of it for a refused request
  __shared__ int64_t warp_sum[32][2];
  __shared__ long long taken;
  pdl_trigger();
  pdl_wait();
  const int page_mask = (1 << p.page_log2) - 1;
  int64_t used = *p.n_used;
  if (used < 0) used = 0;
  if (threadIdx.x == 0) {
    taken = 0;
    if (*p.n_used < 0) raise_device_error(p.err, kDevErrBadIndex);
  }
  int64_t carry[2] = {0, 0};
  for (int r0 = 0; r0 < p.n_req; r0 += blockDim.x) {
    const int r = r0 + threadIdx.x;
    int c = 0, n = 0;
    if (r < p.n_req) {
      c = p.cached[r];
      n = p.fresh[r];
      if (c < 0 || n < 0) {
        raise_device_error(p.err, kDevErrBadIndex);
        c = c < 0 ? 0 : c;
        n = n < 0 ? 0 : n;
      }
    }
    const int64_t held = ((int64_t)c + page_mask) >> p.page_log2;
    const int64_t want = ((int64_t)c + n + page_mask) >> p.page_log2;
    // rows first: whether they fit decides whether the request takes pages
    int64_t end = n, none = 0;
    int64_t c0[2] = {carry[0], 0};
    scan2(end, none, c0, warp_sum);
    carry[0] = c0[0];
    const bool fits = r < p.n_req && end <= p.n_tokens && want <= p.max_blocks && (int64_t)c + n <= 0x7fffffff;
    const int64_t need = fits ? want - held : 0;
    int64_t upto = need, none2 = 0;
    int64_t c1[2] = {carry[1], 0};
    scan2(upto, none2, c1, warp_sum);
    carry[1] = c1[0];
    if (r < p.n_req) {
      const bool ok = fits && (need == 0 || used + upto <= p.n_free);
      start[r] = (int)min(end - n, p.n_tokens);
      first[r] = (int)min(upto - need, (int64_t)0x7fffffff);
      held_len[r] = ok ? c : ~c;
      if (r == p.n_req - 1) start[p.n_req] = (int)min(end, p.n_tokens);
      if (ok && need > 0) atomicMax(&taken, (long long)upto);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) *p.n_used_out = (int)(used + taken);
  for (int r = threadIdx.x; r <= p.n_req; r += blockDim.x) {
    p.q_start[r] = start[r];
    // a served request's rows all fit: they are its new tokens
    if (r < p.n_req) p.kv_len[r] = held_len[r] < 0 ? 0 : held_len[r] + start[r + 1] - start[r];
  }

  // The pages handed out are the first `taken` asked for; page i belongs to the
  // last request that starts at or before it and asked for some.
  const int32_t* pool = p.free_pages + used;
  for (int i = threadIdx.x; i < (int)taken; i += blockDim.x) {
    const int r = row_request(first, p.n_req, i);
    const int64_t held = ((int64_t)held_len[r] + page_mask) >> p.page_log2;
    p.table[r * p.ld_table + held + i - first[r]] = pool[i];
  }
  if (p.n_tokens > kPlanOwnTokens) return;
  for (int t = threadIdx.x; t < p.n_tokens; t += blockDim.x) {
    int64_t slot = -1;
    int pos = 0;
    if (t < start[p.n_req]) {
      const int r = row_request(start, p.n_req, t);
      const int c = held_len[r];
      if (c >= 0) {
        pos = c + t - start[r];
        const int64_t held = ((int64_t)c + page_mask) >> p.page_log2, b = pos >> p.page_log2;
        const int32_t page = b < held ? p.table[r * p.ld_table + b] : pool[first[r] + b - held];
        slot = ((int64_t)page << p.page_log2) + (pos & page_mask);
      }
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
  }
}

// Rows -> slots of a large step, once the planning kernel has written its
// outputs: each CTA brings the row offsets into shared memory.
__global__ void __launch_bounds__(256) paged_slots_kernel(const PlanParams p) {
  extern __shared__ int plan_smem[];
  pdl_trigger();
  pdl_wait();
  for (int r = threadIdx.x; r <= p.n_req; r += blockDim.x) plan_smem[r] = p.q_start[r];
  __syncthreads();
  const int rows = plan_smem[p.n_req], page_mask = (1 << p.page_log2) - 1;
  for (int64_t t64 = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; t64 < p.n_tokens;
       t64 += (int64_t)gridDim.x * blockDim.x) {
    const int t = (int)t64;
    int64_t slot = -1;
    int pos = 0;
    if (t < rows) {
      const int r = row_request(plan_smem, p.n_req, t);
      if (p.kv_len[r] > 0) {
        pos = p.kv_len[r] - (plan_smem[r + 1] - t);    // the last row is the last key
        const int32_t page = p.table[r * p.ld_table + (pos >> p.page_log2)];
        slot = ((int64_t)page << p.page_log2) + (pos & page_mask);
      }
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
  }
}

}  // namespace

int sm_count(int* n) {
  static std::atomic<int> known[64];
  int dev = 0;
  SMEAI_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 64 && (*n = known[dev].load())) return kOk;
  SMEAI_CUDA_TRY(cudaDeviceGetAttribute(n, cudaDevAttrMultiProcessorCount, dev));
  if (dev < 64) known[dev].store(*n);
  return kOk;
}

int paged_plan(const int32_t* cached_len, const int32_t* new_len, int n_req, int page_log2, const int32_t* free_pages,
               int64_t n_free, const int32_t* n_used, int32_t* n_used_out, int32_t* table, int64_t ld_table,
               int64_t max_blocks, int32_t* q_start, int32_t* kv_len, int64_t* slots, int32_t* positions,
               int64_t n_tokens, cudaStream_t stream) {
  PlanParams p;
  p.cached = cached_len;
  p.fresh = new_len;
  p.n_req = n_req;
  p.page_log2 = page_log2;
  p.free_pages = free_pages;
  p.n_free = n_free;
  p.n_used = n_used;
  p.n_used_out = n_used_out;
  p.table = table;
  p.ld_table = ld_table;
  p.max_blocks = max_blocks;
  p.q_start = q_start;
  p.kv_len = kv_len;
  p.slots = slots;
  p.positions = positions;
  p.n_tokens = n_tokens;
  p.err = device_error_ptr();
  if (!p.err) {
    set_last_error("paged_plan: no device error word");
    return kCudaError;
  }
  const size_t smem = ((size_t)3 * n_req + 1) * sizeof(int);
  constexpr int kMaxSmem = (3 * kPlanMaxReq + 1) * (int)sizeof(int);
  if (smem > 48 * 1024 - 1024)
    SMEAI_CUDA_TRY(cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem));
  // enough threads for the requests, their pages (as many as rows, at most) and, where this CTA maps them, the rows
  int64_t work = n_req;
  if (n_tokens > kPlanOwnTokens) work = kPlanThreads;
  if (n_tokens <= kPlanOwnTokens && n_tokens > work) work = n_tokens;
  const int threads = work >= kPlanThreads ? kPlanThreads : (int)((work + 31) / 32 * 32);
  SMEAI_CUDA_TRY(launch(paged_plan_kernel, dim3(1), dim3(threads < 128 ? 128 : threads), smem, stream, p));
  if (n_tokens > kPlanOwnTokens) {
    int sms = 0;
    const int st = sm_count(&sms);
    if (st) return st;
    int64_t ctas = (n_tokens + 255) / 256;
    if (ctas > 8 * sms) ctas = 8 * sms;
    SMEAI_CUDA_TRY(launch(paged_slots_kernel, dim3((unsigned)ctas), dim3(256), (size_t)(n_req + 1) * sizeof(int),
                          stream, p));
  }
  return kOk;
}

// ---- append -------------------------------------------------------------------

namespace {

template <typename T>
struct Pack;
template <>
struct Pack<__half> {
  static __device__ __forceinline__ uint32_t two(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Pack<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t two(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

struct AppendParams {
  KvView kv;
  const float *k, *v, *q;
  int64_t ld_k, ld_v, ld_q, ld_qo;   // floats, floats, floats, bytes
  char* q_out;
  int n_heads;                       // query heads; 0 without q
  int64_t n_tokens;
  const int64_t* slots;
  const int32_t* positions;
  const float* rope;
  int64_t n_rope;
  unsigned* err;
};

template <bool kVec>
__device__ __forceinline__ float4 load4(const float* p) {
  if (kVec) return __ldcs(reinterpret_cast<const float4*>(p));
  return make_float4(p[0], p[1], p[2], p[3]);
}

enum RopeMode : int { kRopeNone = 0, kRopePairs = 1, kRopeHalves = 2 };

// One CTA per (token, slice of its heads): thread = 8 elements of a head (in
// halves mode 4 and their 4 partners), the same ones in every head it visits,
// so a thread reads its cosines and sines once.  6 bytes a value and nothing
// reused: bound by HBM for a prompt (8191 tokens of 3 x 32 heads of 128: 98.5
// us = 6.2 TB/s), by launch latency for a few tokens (48: 1.9 us).
// Products and sums are fp32, each rounded once; the result is rounded to the
// cache's 16-bit type, the cache's own precision.
template <typename T, int kMode, bool kVec>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendParams p) {
  pdl_trigger();
  pdl_wait();
  const int D = p.kv.dim, lanes = D >> 3;
  const int64_t tok = blockIdx.x;
  const int e = (int)threadIdx.x % lanes;
  const int heads = p.n_heads + 2 * p.kv.n_kv, step = (int)blockDim.x / lanes * gridDim.y;
  // the elements of this thread: 8 from lo, or 4 from lo and 4 from lo + D/2
  const int lo = kMode == kRopeHalves ? 4 * e : 8 * e, hi = kMode == kRopeHalves ? lo + D / 2 : lo + 4;
  const int64_t slot = p.slots[tok];
  const int64_t page = slot >> p.kv.page_log2;
  const bool placed = slot >= 0 && page < p.kv.n_pages;
  if (slot != -1 && !placed && threadIdx.x == 0) raise_device_error(p.err, kDevErrBadIndex);
  const int64_t at = page * p.kv.page_bytes + (slot & ((1 << p.kv.page_log2) - 1)) * p.kv.token_bytes;
  float4 c, s;
  if (kMode != kRopeNone) {
    int pos = p.positions[tok];
    if (pos < 0 || pos >= p.n_rope) {
      if (threadIdx.x == 0) raise_device_error(p.err, kDevErrBadIndex);
      pos = 0;
    }
    const float* row = p.rope + (int64_t)pos * D + 4 * e;   // both modes turn 4 angles a thread, from 4e on
    const float* row2 = row + D / 2;
    c = kVec ? __ldg(reinterpret_cast<const float4*>(row)) : make_float4(row[0], row[1], row[2], row[3]);
    s = kVec ? __ldg(reinterpret_cast<const float4*>(row2)) : make_float4(row2[0], row2[1], row2[2], row2[3]);
  }
  auto source = [&](int h) {
    return h < p.n_heads               ? p.q + tok * p.ld_q + (int64_t)h * D
           : h < p.n_heads + p.kv.n_kv ? p.k + tok * p.ld_k + (int64_t)(h - p.n_heads) * D
                                       : p.v + tok * p.ld_v + (int64_t)(h - p.n_heads - p.kv.n_kv) * D;
  };
  const int h0 = blockIdx.y * ((int)blockDim.x / lanes) + (int)threadIdx.x / lanes;
#pragma unroll 4
  for (int h = h0; h < heads; h += step) {
    const bool is_q = h < p.n_heads, is_v = h >= p.n_heads + p.kv.n_kv;
    if (!is_q && !placed) continue;
    const float* src = source(h);
    const float4 a = load4<kVec>(src + lo), b = load4<kVec>(src + hi);
    uint32_t w[4];
    if (kMode == kRopeNone || is_v) {
      w[0] = Pack<T>::two(a.x, a.y);
      w[1] = Pack<T>::two(a.z, a.w);
      w[2] = Pack<T>::two(b.x, b.y);
      w[3] = Pack<T>::two(b.z, b.w);
    } else if (kMode == kRopePairs) {
      w[0] = Pack<T>::two(a.x * c.x - a.y * s.x, a.x * s.x + a.y * c.x);
      w[1] = Pack<T>::two(a.z * c.y - a.w * s.y, a.z * s.y + a.w * c.y);
      w[2] = Pack<T>::two(b.x * c.z - b.y * s.z, b.x * s.z + b.y * c.z);
      w[3] = Pack<T>::two(b.z * c.w - b.w * s.w, b.z * s.w + b.w * c.w);
    } else {
      w[0] = Pack<T>::two(a.x * c.x - b.x * s.x, a.y * c.y - b.y * s.y);
      w[1] = Pack<T>::two(a.z * c.z - b.z * s.z, a.w * c.w - b.w * s.w);
      w[2] = Pack<T>::two(a.x * s.x + b.x * c.x, a.y * s.y + b.y * c.y);
      w[3] = Pack<T>::two(a.z * s.z + b.z * c.z, a.w * s.w + b.w * c.w);
    }
    char* dst = is_q   ? p.q_out + tok * p.ld_qo + (int64_t)h * D * 2
                : is_v ? p.kv.v + at + (h - p.n_heads - p.kv.n_kv) * p.kv.head_bytes
                       : p.kv.k + at + (h - p.n_heads) * p.kv.head_bytes;
    if (kMode == kRopeHalves) {
      *reinterpret_cast<uint2*>(dst + lo * 2) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(dst + hi * 2) = make_uint2(w[2], w[3]);
    } else {
      *reinterpret_cast<uint4*>(dst + lo * 2) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

template <typename T, bool kVec>
cudaError_t launch_append(const AppendParams& p, int mode, dim3 grid, dim3 block, cudaStream_t stream) {
  switch (mode) {
    case kRopeNone: return launch(paged_append_kernel<T, kRopeNone, kVec>, grid, block, 0, stream, p);
    case kRopePairs: return launch(paged_append_kernel<T, kRopePairs, kVec>, grid, block, 0, stream, p);
    default: return launch(paged_append_kernel<T, kRopeHalves, kVec>, grid, block, 0, stream, p);
  }
}

bool vec16(const void* p, int64_t ld_floats) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld_floats % 4 == 0;
}

}  // namespace

int paged_append(const KvView& kv, const float* k, int64_t ld_k, const float* v, int64_t ld_v, const float* q,
                 int64_t ld_q, int n_heads, void* q_out, int64_t ld_q_out, int64_t n_tokens, const int64_t* slots,
                 const int32_t* positions, const float* rope, int64_t n_rope, bool halves, cudaStream_t stream) {
  AppendParams p;
  p.kv = kv;
  p.k = k;
  p.v = v;
  p.q = q;
  p.ld_k = ld_k;
  p.ld_v = ld_v;
  p.ld_q = ld_q;
  p.ld_qo = ld_q_out * 2;
  p.q_out = static_cast<char*>(q_out);
  p.n_heads = q ? n_heads : 0;
  p.n_tokens = n_tokens;
  p.slots = slots;
  p.positions = positions;
  p.rope = rope;
  p.n_rope = n_rope;
  p.err = device_error_ptr();
  int sms = 0;
  const int st = sm_count(&sms);
  if (st) return st;
  if (!p.err) {
    set_last_error("paged_append: no device error word");
    return kCudaError;
  }
  const int lanes = kv.dim / 8, heads = p.n_heads + 2 * kv.n_kv, per_cta = 256 / lanes;
  // a token's heads over several CTAs while tokens alone do not fill the GPU
  const int most = (heads + per_cta - 1) / per_cta;
  int64_t slices = (4 * (int64_t)sms + n_tokens - 1) / n_tokens;
  if (slices > most) slices = most;
  const dim3 grid((unsigned)n_tokens, (unsigned)slices), block((unsigned)(per_cta * lanes));
  const int mode = !rope ? kRopeNone : halves ? kRopeHalves : kRopePairs;
  const bool vec = vec16(k, ld_k) && vec16(v, ld_v) && (!q || vec16(q, ld_q)) && vec16(rope, 0);
  cudaError_t e;
  if (kv.bf16) e = vec ? launch_append<__nv_bfloat16, true>(p, mode, grid, block, stream)
                       : launch_append<__nv_bfloat16, false>(p, mode, grid, block, stream);
  else e = vec ? launch_append<__half, true>(p, mode, grid, block, stream)
               : launch_append<__half, false>(p, mode, grid, block, stream);
  SMEAI_CUDA_TRY(e);
  return kOk;
}

}  // namespace smeai
