// paged_attn.cuh -- what the paged attention kernels share: parameters, the
// split of a step's work over CTAs, and the partial results of rows whose keys
// several CTAs share.
//
// Work.  The rows of a request that read one key head are its new tokens times
// the query heads of that key head's group, packed as (token, head in group)
// and cut into tiles of TR rows.  A tile is (request, row tile, key head); its
// keys come in blocks of KB.  All key blocks of all tiles of a launch, in a
// fixed order, are one line of units, and every CTA takes an equal piece of
// that line -- whatever the requests' lengths, no CTA has more than its share.
// A piece that ends inside a tile leaves that tile's rows as a partial result
// (running maximum, sum, unnormalized context; all fp32), which a second
// kernel joins in key order, so results do not depend on timing.  Pieces are
// snapped to a tile's edge when one is within kSnap units: short tiles are
// never split and need no joining.  On the line a tile is longer than its
// blocks by what opening and ending it costs (measured: 5000 to 8000 cycles
// against 2500 a block of 64 keys, 8000 against 3000 a block of 128 and up to
// 128 rows), so a CTA that gets many short tiles gets fewer blocks (24 requests
// of 64 rows over 300 to 4096 keys: 1 block 76, 2 blocks 75.5, 3 blocks 67 us).  Where whole tiles dealt out by
// their number take no longer than equal pieces and the splitting (kSplitCost
// blocks), no tile is split: 128 tiles of 5 to 8 blocks on 148 CTAs are one
// each, not none, one or two.
#pragma once

#include <cuda_bf16.h>

#include <atomic>

#include "common.cuh"
#include "paged.h"

namespace smeai {

constexpr int kSnap = 3;
template <int KB>
constexpr int kTileCost = KB == 64 ? 2 : 3;   // in blocks
constexpr int kSplitCost = 4;

struct AttnParams {
  KvView kv;
  const char* q;
  char* out;
  int64_t ld_q, ld_out;   // bytes
  const int32_t *q_start, *kv_len, *table;
  int64_t ld_table;
  int n_req, max_kv, n_tokens;
  int group;              // query heads per key head
  float scale_log2;       // scale * log2(e)
  int causal;
  int rows_lo, rows_hi;   // requests with rows_lo < rows <= rows_hi are this launch's
  float* part_o;          // [2 * CTAs][TR][DP]
  float2* part_ml;        // [2 * CTAs][TR] running maximum (before the scale), sum
  int4* head;             // [CTAs] tile left unfinished at the end {first row of its request or -1, the
                          // request's packed rows, row tile, key head}
  int* state;             // [CTAs] state of slot 0
  unsigned* err;
};

// State of a CTA's partial slot 0, the tile it entered in the middle.
enum : int { kPartNone = 0, kPartGoesOn = 1, kPartEnds = 2 };

struct AttnReq {
  int q0, n_new, kv, rows;   // first row, new tokens, keys, packed rows (0: not this launch's)
};

__device__ __forceinline__ AttnReq attn_req(const AttnParams& p, int b) {
  AttnReq r;
  const int a = p.q_start[b], e = p.q_start[b + 1], kv = p.kv_len[b];
  r.q0 = min(max(a, 0), p.n_tokens);
  r.n_new = min(max(e, r.q0), p.n_tokens) - r.q0;
  r.kv = min(max(kv, 0), p.max_kv);
  if (a != r.q0 || e != r.q0 + r.n_new || kv != r.kv) raise_device_error(p.err, kDevErrBadIndex);
  r.rows = r.n_new * p.group;
  if (r.rows <= p.rows_lo || r.rows > p.rows_hi) r.rows = 0;
  return r;
}

// Keys that packed row `row` sees: j < the result.
__device__ __forceinline__ int attn_limit(const AttnParams& p, const AttnReq& r, int row) {
  return p.causal ? max(0, r.kv - r.n_new + 1 + row / p.group) : r.kv;
}

// Key blocks of row tile rt (at least one: a tile whose rows see nothing still
// has its zeros to write).
template <int TR, int KB>
__device__ __forceinline__ int attn_blocks(const AttnParams& p, const AttnReq& r, int rt) {
  const int end = (rt + 1) * TR;
  const int keys = end >= r.rows ? r.kv : min(r.kv, attn_limit(p, r, end - 1));   // the last row sees them all
  return max(1, (int)((unsigned)(keys + KB - 1) / KB));
}

// The same for every row tile of a request in turn, cheaply: where the group
// divides TR a tile's last row is a fixed number of tokens behind the one
// before's, and no division is left.
template <int TR, int KB>
struct AttnTiles {
  int n_rt, step, keys;      // keys: what the last row of the next tile sees, before clamping
  bool even;
  __device__ __forceinline__ AttnTiles(const AttnParams& p, const AttnReq& r) {
    n_rt = (int)((unsigned)(r.rows + TR - 1) / TR);
    even = !p.causal || n_rt <= 1 || TR % p.group == 0;
    step = !p.causal || n_rt <= 1 ? 0 : TR / p.group;
    keys = step ? r.kv - r.n_new : r.kv;
  }
  // blocks of tile rt; called for rt = 0, 1, ..
  __device__ __forceinline__ int next(const AttnParams& p, const AttnReq& r, int rt) {
    if (!even) return attn_blocks<TR, KB>(p, r, rt);
    keys += step;
    const int k = rt + 1 == n_rt ? r.kv : max(0, min(r.kv, keys));
    return max(1, (int)((unsigned)(k + KB - 1) / KB));
  }
};

// Key blocks of all tiles of a request; `tiles` gets their number, `most` is
// raised to the longest one's blocks.
template <int TR, int KB>
__device__ __forceinline__ int64_t attn_units(const AttnParams& p, const AttnReq& r, int64_t& tiles, int& most) {
  int64_t u = 0;
  AttnTiles<TR, KB> t(p, r);
#pragma unroll 1
  for (int rt = 0; rt < t.n_rt; ++rt) {
    const int nkb = t.next(p, r, rt);
    u += nkb;
    most = max(most, nkb);
  }
  tiles = (int64_t)t.n_rt * p.kv.n_kv;
  return u * p.kv.n_kv;
}

// A place on the line: tile (b, rt, h), key block kb of its nkb.
struct AttnPos {
  int b, rt, h, kb, nkb;
  AttnReq r;
};

template <int TR, int KB>
__device__ __forceinline__ void attn_next_tile(const AttnParams& p, AttnPos& w) {
  w.kb = 0;
  if (++w.h < p.kv.n_kv) return;
  w.h = 0;
  ++w.rt;
  if (w.rt * TR >= w.r.rows) {
    w.rt = 0;
    do {
      if (++w.b >= p.n_req) return;
      w.r = attn_req(p, w.b);
    } while (w.r.rows == 0);
  }
  w.nkb = attn_blocks<TR, KB>(p, w.r, w.rt);
}

struct AttnShare {
  int64_t u0, u1;            // this CTA's units: key blocks, counted along the line
  AttnPos at;                // place of u0
};

// This CTA's piece of the line.  All threads of the block call it; the place
// is in shared memory on return.  warp_sum: [3 * NT / 32] in shared memory.  Each
// thread sums its own run of requests; the one whose run holds an end of the
// piece walks to it.
template <int TR, int KB, int NT>
__device__ void attn_share(const AttnParams& p, AttnShare* s, int64_t* warp_sum) {
  constexpr int kCost = kTileCost<KB>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (p.n_req + NT - 1) / NT;
  const int b0 = min((int)threadIdx.x * per, p.n_req), b1 = min(b0 + per, p.n_req);
  int64_t mine = 0, mine_t = 0;               // blocks, tiles
  int most = 0;                               // blocks of the longest tile
#pragma unroll 1
  for (int b = b0; b < b1; ++b) {
    int64_t t;
    mine += attn_units<TR, KB>(p, attn_req(p, b), t, most);
    mine_t += t;
  }
  int64_t incl = mine, incl_t = mine_t;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t a = __shfl_up_sync(0xffffffffu, incl, off), t = __shfl_up_sync(0xffffffffu, incl_t, off);
    if (lane >= off) {
      incl += a;
      incl_t += t;
    }
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 31) {
    warp_sum[3 * warp] = incl;
    warp_sum[3 * warp + 1] = incl_t;
    warp_sum[3 * warp + 2] = most;
  }
  __syncthreads();
  int64_t lo = incl - mine, lo_t = incl_t - mine_t, total = 0, total_t = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) {
    const int64_t a = warp_sum[3 * w], t = warp_sum[3 * w + 1];
    most = max(most, (int)warp_sum[3 * w + 2]);
    if (w < warp) {
      lo += a;
      lo_t += t;
    }
    total += a;
    total_t += t;
  }
  // 64-bit division is slow, and these numbers are rarely that large
  auto up = [](int64_t n, unsigned d) {
    return n <= 0x7fff0000 ? (int64_t)(((uint32_t)n + d - 1) / d) : (n + d - 1) / d;
  };
  // lengths on the line: the tiles' blocks with their own costs, or 1 a tile
  int64_t line = total + kCost * total_t, per_cta = up(line, gridDim.x);
  const bool whole = up(total_t, gridDim.x) * (most + kCost) <= per_cta + kSplitCost;
  int64_t line_lo = lo + kCost * lo_t, line_hi = line_lo + mine + kCost * mine_t;
  if (whole) {
    line = total_t;
    per_cta = up(line, gridDim.x);
    line_lo = lo_t;
    line_hi = lo_t + mine_t;
  }
  const int64_t cut0 = min(line, per_cta * blockIdx.x), cut1 = min(line, cut0 + per_cta);
  if (threadIdx.x == 0) {
    if (cut0 >= line) s->u0 = total;
    if (cut1 >= line) s->u1 = total;
  }
  // walk to each cut that lies in this run: the tile around it, and the edge it snaps to
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const int64_t cut = which ? cut1 : cut0;
    if (cut < line_lo || cut >= line_hi) continue;
    int64_t at = line_lo, u = lo;
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
      const AttnReq r = attn_req(p, b);
      AttnTiles<TR, KB> t(p, r);
#pragma unroll 1
      for (int rt = 0; rt < t.n_rt; ++rt) {
        const int nkb = t.next(p, r, rt);
        const int one = whole ? 1 : nkb + kCost;
        const int64_t len = (int64_t)one * p.kv.n_kv;
        if (cut >= at + len) {
          at += len;
          u += (int64_t)nkb * p.kv.n_kv;
          continue;
        }
        const int64_t in = cut - at;
        const int h = len <= 0x7fffffff ? (int)((unsigned)in / (unsigned)one) : (int)(in / one);
        int kb = max(0, (int)(in - (int64_t)h * one) - kCost);   // 0 with whole tiles
        if (kb <= kSnap && kb <= nkb - kb) kb = 0;
        else if (nkb - kb <= kSnap) kb = nkb;           // the start of the next tile
        u += (int64_t)h * nkb + kb;
        if (which) s->u1 = u;
        else {
          s->u0 = u;
          s->at = {b, rt, h, kb, nkb, r};
        }
        b = b1;
        break;
      }
    }
  }
  __syncthreads();
}

template <int TR, int KB>
__device__ __forceinline__ void attn_open(const AttnParams& p, const AttnShare& s, AttnPos& w) {
  w = s.at;
  if (w.kb == w.nkb) attn_next_tile<TR, KB>(p, w);
}

// Thread 0 of a CTA: its headers before any tile, and a tile not finished here.
__device__ __forceinline__ void attn_no_parts(const AttnParams& p) {
  if (!p.head) return;       // no tile can be split
  p.head[blockIdx.x] = make_int4(-1, 0, 0, 0);
  p.state[blockIdx.x] = kPartNone;
}
__device__ __forceinline__ void attn_leave_part(const AttnParams& p, const AttnPos& w, bool begun_here, bool ends) {
  if (begun_here) p.head[blockIdx.x] = make_int4(w.r.q0, w.r.rows, w.rt, w.h);
  else p.state[blockIdx.x] = ends ? kPartEnds : kPartGoesOn;
}

// ---- 16-bit types ---------------------------------------------------------------
// kBias: softmax weights are kept as 2^(kBias + s - m).  Half has 14 exponent
// steps below 1; the bias moves the weights up so that ones as small as
// 2^-21 of the largest keep their 11 bits; with the 2^8 by which the maximum may
// lag they stay below 65504.  bfloat16 has fp32's range and needs none.
template <typename T>
struct Num;
template <>
struct Num<__half> {
  static constexpr float kBias = 7.f;
  static constexpr bool kIsBf16 = false;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
};
template <>
struct Num<__nv_bfloat16> {
  static constexpr float kBias = 0.f;
  static constexpr bool kIsBf16 = true;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
};

// Context values rounded to the output's type.  A mean of finite halves is at
// most 65504; the rounding of the weights may have carried it past that, where
// it would round to infinity.  True infinities and NaN stay.
template <typename T>
__device__ __forceinline__ uint32_t pack_mean(float lo, float hi) {
  if constexpr (!Num<T>::kIsBf16) {
    if (fabsf(lo) < INFINITY) lo = fminf(fmaxf(lo, -65504.f), 65504.f);
    if (fabsf(hi) < INFINITY) hi = fminf(fmaxf(hi, -65504.f), 65504.f);
  }
  return Num<T>::pack(lo, hi);
}

// What a row's context is multiplied by in the end: nothing seen gives zeros,
// NaN stays.
__device__ __forceinline__ float row_scale(float sum) { return sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum); }

// A row's weights are 2^(kBias + c (s - m)), c = scale * log2(e): one fused
// multiply-add a score, c s + (kBias - c m), as exact as the second part.  Once
// c m passes 2^22, where fp32 has steps of half and more, the scores are
// subtracted first, which is exact near the maximum.  `base` is what the
// multiply-add subtracts: m, or 0 for such a far row.  A far row's maximum may
// not lag, and any score of it opens the branch in which maxima are raised:
// the subtraction is there and costs other rows nothing.
constexpr float kRaise = 8.f;          // growth of the maximum (log2) that rescales what was gathered
constexpr float kFar = 4194304.f;
__device__ __forceinline__ float row_base(float m, float c) { return fabsf(m) * c < kFar ? m : 0.f; }
__device__ __forceinline__ float raise_lag(float c) { return fminf(kRaise / c, 1e38f); }   // -inf plus it is -inf
template <typename T>
__device__ __forceinline__ float base_offset(float base, float c) {
  return base == -INFINITY ? 0.f : fmaf(-base, c, Num<T>::kBias);
}

// 2^x, the hardware's approximation (2 ulp; 2^-inf = 0).
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Whether any tile can be split: those of up to 2 * kSnap blocks never are.
template <int KB>
constexpr bool attn_splits(int max_kv) {
  return max_kv > 2 * kSnap * KB;
}

// Partial slots and headers of a launch with `ctas` CTAs.
template <int TR, int DP>
constexpr size_t attn_part_bytes(int ctas) {
  return (size_t)2 * ctas * TR * (DP * sizeof(float) + sizeof(float2)) + (size_t)ctas * (sizeof(int4) + sizeof(int));
}
template <int TR, int DP>
void attn_carve(AttnParams& p, void* ws, int ctas) {
  p.part_o = nullptr;
  p.part_ml = nullptr;
  p.head = nullptr;
  p.state = nullptr;
  char* c = static_cast<char*>(ws);
  if (!c) return;
  p.part_o = reinterpret_cast<float*>(c);
  c += (size_t)2 * ctas * TR * DP * sizeof(float);
  p.part_ml = reinterpret_cast<float2*>(c);
  c += (size_t)2 * ctas * TR * sizeof(float2);
  p.head = reinterpret_cast<int4*>(c);
  p.state = reinterpret_cast<int*>(c + (size_t)ctas * sizeof(int4));
}

// The tensor-core kernel of requests with many rows, head_dim up to 128
// (paged_attn_tc.cu): one CTA an SM.
size_t paged_attn_tc_workspace(int padded_dim, int max_kv, int sms);
int paged_attn_tc(const AttnParams& p, int padded_dim, void* workspace, int max_kv, int sms, cudaStream_t stream);

// The kernel's dynamic shared memory limit, set once a device.
template <typename K>
cudaError_t attn_allow_smem(K kernel, size_t bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
  if (done.load() & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) done.fetch_or(bit);
  return e;
}

// Joins the partial results (paged_attn.cu).
template <typename T, int TR, int DP>
cudaError_t attn_join(const AttnParams& p, int ctas, cudaStream_t stream);

}  // namespace smeai
