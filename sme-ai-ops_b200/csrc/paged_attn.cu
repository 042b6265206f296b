// paged_attn.cu -- attention of new tokens over a paged key/value cache for
// requests that bring few rows (a decoding step, drafted tokens, short
// chunks), and the joining of partial results.
//
//   o_r = sum_j p_rj v_j / sum_j p_rj,   p_rj = 2^(c (s_rj - m_r)),
//   s_rj = q_r . k_j,  c = scale log2(e),  m_r = max over the keys seen so far of s_rj
//
// in one pass over the keys: when m_r grows by d, the sum and the context
// gathered so far are multiplied by 2^(-c d).
#include "paged_attn.cuh"

namespace smeai {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kKeys = 64;            // keys a block
constexpr float kNegInf = -INFINITY;

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// d += a b, or d = a b for the first step of a sum.
template <typename T, bool kFirst = false>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  const float z = 0.f;
  if constexpr (kFirst && Num<T>::kIsBf16)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(z));
  else if constexpr (kFirst)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(z));
  else if constexpr (Num<T>::kIsBf16)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Shared-memory layout: [stages][K, V][kKeys rows][DP] 16-bit, the 16-byte
// chunks of a row XORed with the row's index mod 8, so that ldmatrix's eight
// rows fall on different banks; then the query tiles in the same layout.
template <int DP>
struct Shape {
  static constexpr int kRowBytes = DP * 2;
  static constexpr int kTileBytes = kKeys * kRowBytes;
  static constexpr int kStages = DP == 64 ? 6 : 3;      // 96 KB in flight (192 KB at DP 256)
  static constexpr int kPerSm = DP == 256 ? 1 : 2;      // CTAs an SM
};

template <int DP>
__device__ __forceinline__ uint32_t chunk_addr(uint32_t base, int row, int chunk) {
  return base + row * Shape<DP>::kRowBytes + ((chunk ^ (row & 7)) << 4);
}

// Walks a CTA's share ahead of the computation and copies blocks into the
// ring.  Warp w copies rows 16w .. 16w + 15 of a block.  Each lane looks up the
// page of one of these keys a block ahead, so that the table's latency hides
// behind a block, and hands its address to the lanes that copy the row: eight
// lanes take 128 contiguous bytes of it, four rows at a time.
template <int DP, int TR>
struct Loader {
  using S = Shape<DP>;
  AttnPos at;
  int64_t left;
  int page;             // of this lane's key in block `at`; -1: no such key, or a bad page
  uint32_t even, odd;   // place of row i * 4 + lane / 8 of the warp's, for even and odd i, less i
  int bytes[DP / 64];   // 0 past the head's elements

  __device__ __forceinline__ void look_up(const AttnParams& p) {
    const int lane = threadIdx.x & 31, key = at.kb * kKeys + (int)(threadIdx.x >> 5) * 16 + (lane & 15);
    page = key < at.r.kv ? p.table[(int64_t)at.b * p.ld_table + (key >> p.kv.page_log2)] : -1;
    if (key < at.r.kv && (page < 0 || page >= p.kv.n_pages)) {
      raise_device_error(p.err, kDevErrBadIndex);
      page = -1;
    }
  }
  __device__ __forceinline__ void open(const AttnParams& p, const AttnPos& from, int64_t units) {
    const int lane = threadIdx.x & 31, sub = lane >> 3, col = lane & 7, row0 = (int)(threadIdx.x >> 5) * 16;
    at = from;
    left = units;
    even = (row0 + sub) * S::kRowBytes + ((col ^ sub) << 4);
    odd = (row0 + sub) * S::kRowBytes + ((col ^ (sub + 4)) << 4);
#pragma unroll
    for (int cb = 0; cb < DP / 64; ++cb) bytes[cb] = cb * 64 + col * 8 < p.kv.dim ? 16 : 0;
    look_up(p);
  }
  // the next block into `stage` (shared-memory address of its keys); one commit group
  __device__ __forceinline__ void load(const AttnParams& p, uint32_t stage) {
    if (left > 0) {
      const int lane = threadIdx.x & 31, sub = lane >> 3, col = lane & 7;
      const int key = at.kb * kKeys + (int)(threadIdx.x >> 5) * 16 + (lane & 15);
      const int64_t off = page < 0 ? 0
                                   : page * p.kv.page_bytes +
                                         (key & ((1 << p.kv.page_log2) - 1)) * p.kv.token_bytes + at.h * p.kv.head_bytes;
      const unsigned there = __ballot_sync(0xffffffffu, page >= 0);
      const char *k = p.kv.k + col * 16, *v = p.kv.v + col * 16;
      const uint32_t d0 = stage + even, d1 = stage + odd;
      if (there == 0xffffffffu) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t o = __shfl_sync(0xffffffffu, off, i * 4 + sub);
          const uint32_t d = (i & 1 ? d1 : d0) + i * 4 * S::kRowBytes;
#pragma unroll
          for (int cb = 0; cb < DP / 64; ++cb) {
            cp_async16(d + cb * 128, k + o + cb * 128, bytes[cb]);
            cp_async16(d + cb * 128 + S::kTileBytes, v + o + cb * 128, bytes[cb]);
          }
        }
      } else {
        // some keys do not exist: zeros, and nothing is read
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t o = __shfl_sync(0xffffffffu, off, i * 4 + sub);
          const bool ok = there >> (i * 4 + sub) & 1;
          const uint32_t d = (i & 1 ? d1 : d0) + i * 4 * S::kRowBytes;
#pragma unroll
          for (int cb = 0; cb < DP / 64; ++cb) {
            cp_async16(d + cb * 128, k + (ok ? o + cb * 128 : -col * 16), ok ? bytes[cb] : 0);
            cp_async16(d + cb * 128 + S::kTileBytes, v + (ok ? o + cb * 128 : -col * 16), ok ? bytes[cb] : 0);
          }
        }
      }
      if (--left > 0) {
        if (++at.kb == at.nkb) attn_next_tile<TR, kKeys>(p, at);
        look_up(p);
      }
    }
    cp_async_commit();
  }
};

// ---- few rows -----------------------------------------------------------------
// Tiles of 8 * NQ rows: a decode step's query heads of one key head, or those
// of a few drafted tokens.  The products are taken transposed, with the keys
// as the MMA's 16-wide dimension and eight rows as its 8-wide one,
//   S^T = K Q^T,  O^T += V^T P^T
// so eight rows cost DP/8 mma per 16 keys, half of what a 16-row fragment of
// queries would.  All rows meet every key, and each warp takes 16 of a block's
// 64 keys, with its own ring of keys in shared memory: warps never wait for
// one another before the tile's end, where their maxima, sums and contexts
// are merged (through the ring stage that the tile's last block left).  The
// next tile's queries are copied while a tile is worked on.  A row's maximum is
// only raised when a score passes it by more than 2^8, so most blocks need a
// vote and no reduction over the keys.
// Two CTAs an SM with 96 KB of keys and values in flight each cover HBM's
// latency (44 GB/s x ~1 us = 44 KB an SM) through the ends of tiles; bound by
// the cache's bytes.  Measured: 64 requests of 17 to 8192 keys, 32 query and 8
// key heads of 128: 166 us = 6.3 TB/s; one request of 131001 keys, 4 key heads
// of 64: 38 us (28 of them here, 5 until the first block is computed, 10 the
// joining); 24 requests with 2 to 6 drafted tokens (24-row tiles): 54 us =
// 4.3 TB/s, where opening and ending a tile costs 2 to 3 us of a CTA's time.

// 8x8 16-bit transpose across the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <int DP, int NQ>
constexpr size_t few_smem() {
  using S = Shape<DP>;
  return (size_t)S::kStages * 2 * S::kTileBytes + 2 * 8 * NQ * S::kRowBytes;
}

template <typename T, int DP, int NQ>
__global__ void __launch_bounds__(kThreads, Shape<DP>::kPerSm) paged_attn_few_kernel(const AttnParams p) {
  using S = Shape<DP>;
  constexpr int TR = 8 * NQ;
  constexpr int kAhead = 4;          // ldmatrix in flight ahead of the products
  constexpr int kChunks = DP / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ AttnShare share;
  __shared__ int64_t warp_sum[3 * kWarps];
  __shared__ float merge_m[kWarps][TR], merge_l[kWarps][TR];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const uint32_t ring = smem_addr(smem);
  const uint32_t q_tiles = ring + S::kStages * 2 * S::kTileBytes;

  // every CTA is resident: the kernel behind can only take what these free
  pdl_trigger();
  pdl_wait();
  attn_share<TR, kKeys, kThreads>(p, &share, warp_sum);
  const int64_t u0 = share.u0, u1 = share.u1;
  if (threadIdx.x == 0) attn_no_parts(p);
  if (u1 <= u0) return;

  auto out_offset = [&](const AttnPos& at, int row) {   // head and token of a packed row
    const int tok = row / p.group;
    return make_int2(at.r.q0 + tok, at.h * p.group + row - tok * p.group);
  };
  // the query rows of a tile, into one of the two tiles; with the next commit group
  auto load_queries = [&](const AttnPos& at, int which) {
    for (int c = threadIdx.x; c < TR * kChunks; c += kThreads) {
      const int r = c / kChunks, col = c % kChunks, row = at.rt * TR + r;
      const bool there = row < at.r.rows && col * 8 < p.kv.dim;
      const int2 to = out_offset(at, there ? row : 0);
      cp_async16(chunk_addr<DP>(q_tiles + which * TR * S::kRowBytes, r, col),
                 p.q + (there ? (int64_t)to.x * p.ld_q + ((int64_t)to.y * p.kv.dim + col * 8) * 2 : 0), there ? 16 : 0);
    }
  };

  AttnPos w;
  attn_open<TR, kKeys>(p, share, w);
  Loader<DP, TR> ld;
  ld.open(p, w, u1 - u0);
  load_queries(w, 0);
  for (int s = 0; s < S::kStages - 1; ++s) ld.load(p, ring + s * 2 * S::kTileBytes);

  // Q^T fragments: row (n) g of each eight, elements (k) 2 t4 and 2 t4 + 8 on.
  // Scores and contexts of this lane: rows 2 t4 and 2 t4 + 1 of each eight.
  uint32_t qf[DP / 16][NQ][2];
  float o[DP / 16][NQ][4];
  float m[NQ][2], base[NQ][2], l[NQ][2];
  const float lag = raise_lag(p.scale_log2);
  int lim[NQ][2], lim_all = 0;
  AttnPos next = w;
  int tile_kb0 = w.kb, tile = 0;
  bool opened = false, brief = false;  // the tile is set up; the tile before it was so short that copies may be out
  // this lane's ldmatrix rows, four 16-element steps of 128 bytes each
  uint32_t k_off[4], v_off[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    k_off[i] = chunk_addr<DP>(0, warp * 16 + (lane & 15), i * 2 + (lane >> 4));
    v_off[i] = chunk_addr<DP>(0, warp * 16 + (lane & 7) + (lane >> 4) * 8, i * 2 + ((lane >> 3) & 1));
  }

  int stage = 0;
  for (int64_t u = u0; u < u1; ++u) {
    cp_async_wait<S::kStages - 2>();
    if (opened) {
      __syncwarp();
    } else {
      // a new tile: its queries were copied by all warps
      opened = true;
      tile_kb0 = w.kb;
      if (brief) cp_async_wait<0>();
      __syncthreads();
#pragma unroll
      for (int f = 0; f < NQ; ++f) {
#pragma unroll
        for (int ks = 0; ks < DP / 16; ks += 2) {
          uint32_t b[4];
          ldsm4(chunk_addr<DP>(q_tiles + (tile & 1) * TR * S::kRowBytes, f * 8 + (lane & 7), ks * 2 + (lane >> 3)), b);
          qf[ks][f][0] = b[0];
          qf[ks][f][1] = b[1];
          qf[ks + 1][f][0] = b[2];
          qf[ks + 1][f][1] = b[3];
        }
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) o[ks][f][0] = o[ks][f][1] = o[ks][f][2] = o[ks][f][3] = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = w.rt * TR + f * 8 + 2 * t4 + i;
          lim[f][i] = row < w.r.rows ? min(w.r.kv, attn_limit(p, w.r, row)) : 0;
          m[f][i] = base[f][i] = kNegInf;
          l[f][i] = 0.f;
        }
      }
      lim_all = min(w.r.kv, attn_limit(p, w.r, w.rt * TR));
      // the tile after it; its queries' place was last read before the last merge
      const int n = w.nkb - w.kb;
      brief = n < S::kStages;
      if (n < u1 - u) {
        next = w;
        attn_next_tile<TR, kKeys>(p, next);
        load_queries(next, (tile & 1) ^ 1);
      }
      ++tile;
    }
    const uint32_t kt = ring + stage * 2 * S::kTileBytes, vt = kt + S::kTileBytes;
    float* const left = reinterpret_cast<float*>(smem + stage * 2 * S::kTileBytes);   // for the merge
    const int ahead = stage == 0 ? S::kStages - 1 : stage - 1;      // the stage computed with last
    stage = stage + 1 == S::kStages ? 0 : stage + 1;
    ld.load(p, ring + ahead * 2 * S::kTileBytes);

    // S^T; for eight rows in two chains, as one would wait for its own products
    constexpr int kChains = NQ == 1 ? 2 : 1;
    float s[NQ * kChains][4];
    uint32_t a[kAhead][4];             // 16 keys x 16 elements, fetched kAhead steps ahead
#pragma unroll
    for (int ks = 0; ks < kAhead; ++ks) ldsm4(kt + k_off[ks & 3] + (ks >> 2) * 128, a[ks]);
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
#pragma unroll
      for (int f = 0; f < NQ; ++f) {
        if (ks < kChains) mma16816<T, true>(s[f + ks % kChains], a[ks % kAhead], qf[ks][f][0], qf[ks][f][1]);
        else mma16816<T>(s[f + ks % kChains], a[ks % kAhead], qf[ks][f][0], qf[ks][f][1]);
      }
      const int then = ks + kAhead;    // after the keys the values: 16 elements x 16 keys
      if (then < DP / 16) ldsm4(kt + k_off[then & 3] + (then >> 2) * 128, a[ks % kAhead]);
      else ldsm4_t(vt + v_off[(then - DP / 16) & 3], a[ks % kAhead]);
    }
    if (kChains == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[0][i] += s[NQ * kChains - 1][i];
    }
    // element i: row 2 t4 + (i & 1), key g + 8 (i >> 1)
    const int key0 = w.kb * kKeys + warp * 16;
    if (key0 + 16 > lim_all) {
#pragma unroll
      for (int f = 0; f < NQ; ++f)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (key0 + g + 8 * (i >> 1) >= lim[f][i & 1]) s[f][i] = kNegInf;
    }
    bool raise = false;
#pragma unroll
    for (int f = 0; f < NQ; ++f)
#pragma unroll
      for (int i = 0; i < 4; ++i) raise |= s[f][i] > (base[f][i & 1] == m[f][i & 1] ? m[f][i & 1] + lag : kNegInf);
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int f = 0; f < NQ; ++f)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = fmaxf(s[f][i], s[f][i + 2]);
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          if (top > m[f][i]) {
            const float e = exp2_fast((m[f][i] - top) * p.scale_log2);   // m = -inf: 0
            m[f][i] = top;
            base[f][i] = row_base(top, p.scale_log2);
            l[f][i] *= e;
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
              o[d][f][i] *= e;
              o[d][f][i + 2] *= e;
            }
          }
          if (base[f][i] != m[f][i]) {
            s[f][i] -= m[f][i];
            s[f][i + 2] -= m[f][i];
          }
        }
    }
    // P^T, 16 keys x 8 rows: the weights rounded to the cache's type and, up to
    // 16 rows, what the rounding left, rounded again: without it the weights'
    // rounding adds as much error as the result's own.  The second product
    // costs 1% there (the cache's bytes bound the kernel), 3 to 7% with 24 rows.
    constexpr int kParts = NQ <= 2 ? 2 : 1;
    uint32_t b[NQ * kParts][2];
#pragma unroll
    for (int f = 0; f < NQ; ++f) {
      const float plus[2] = {base_offset<T>(base[f][0], p.scale_log2), base_offset<T>(base[f][1], p.scale_log2)};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[f][i] = exp2_fast(fmaf(s[f][i], p.scale_log2, plus[i & 1]));
        l[f][i & 1] += s[f][i];
      }
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t two = Num<T>::pack(s[f][2 * i], s[f][2 * i + 1]);
          b[f * kParts + part][i] = transpose8(two);
          if (part + 1 < kParts) {
            const float2 kept = Num<T>::unpack(two);
            s[f][2 * i] -= kept.x;
            s[f][2 * i + 1] -= kept.y;
          }
        }
      }
    }
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
#pragma unroll
      for (int f = 0; f < NQ * kParts; ++f) mma16816<T>(o[d][f / kParts], a[d % kAhead], b[f][0], b[f][1]);
      const int then = d + kAhead;
      if (then < DP / 16) ldsm4_t(vt + v_off[then & 3] + (then >> 2) * 128, a[d % kAhead]);
    }

    // ---- end of the tile, or of this CTA's share of it
    const bool last = w.kb + 1 == w.nkb;
    if (!last && u + 1 < u1) {
      ++w.kb;
      continue;
    }
    const bool whole = last && tile_kb0 == 0;
    // slot 0: a tile entered in the middle; slot 1: a tile left unfinished
    const int64_t slot = 2 * (int64_t)blockIdx.x + (tile_kb0 == 0 ? 1 : 0);
    // The warps leave maxima, sums and contexts, sixteen rows at a time: eight
    // where each warp's keys were, eight where its values were (16 x DP x 2
    // bytes hold 8 x DP floats).  Columns are XORed with the row so that a
    // store's four rows take different banks.
#pragma unroll
    for (int f0 = 0; f0 < NQ; f0 += 2) {
      const int rows = min(min(16, TR - f0 * 8), w.r.rows - w.rt * TR - f0 * 8);   // of this pass
      if (rows <= 0) break;
#pragma unroll
      for (int f = f0; f < NQ && f < f0 + 2; ++f) {
        float* mine = left + (f - f0) * (S::kTileBytes / 4) + warp * 8 * DP;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) l[f][i] += __shfl_xor_sync(0xffffffffu, l[f][i], off);
#pragma unroll
          for (int d = 0; d < DP / 16; ++d) {
            mine[(2 * t4 + i) * DP + ((d * 16 + g) ^ (t4 * 8))] = o[d][f][i];
            mine[(2 * t4 + i) * DP + ((d * 16 + 8 + g) ^ (t4 * 8))] = o[d][f][i + 2];
          }
        }
        if (g == 0) {
          *reinterpret_cast<float2*>(&merge_m[warp][f * 8 + 2 * t4]) = make_float2(m[f][0], m[f][1]);
          *reinterpret_cast<float2*>(&merge_l[warp][f * 8 + 2 * t4]) = make_float2(l[f][0], l[f][1]);
        }
      }
      __syncthreads();
      for (int c = threadIdx.x; c < rows * kChunks; c += kThreads) {
        const int r = c / kChunks, d8 = c % kChunks;
        float e[kWarps], top = kNegInf, sum = 0.f, v[8] = {};
#pragma unroll
        for (int ww = 0; ww < kWarps; ++ww) top = fmaxf(top, merge_m[ww][f0 * 8 + r]);
#pragma unroll
        for (int ww = 0; ww < kWarps; ++ww) {
          const float mw = merge_m[ww][f0 * 8 + r];
          e[ww] = mw == kNegInf ? 0.f : exp2_fast((mw - top) * p.scale_log2);
          sum = fmaf(merge_l[ww][f0 * 8 + r], e[ww], sum);
          const float4* src = reinterpret_cast<const float4*>(left + (r >> 3) * (S::kTileBytes / 4) + ww * 8 * DP +
                                                              (r & 7) * DP + ((d8 * 8) ^ (((r & 7) >> 1) * 8)));
          const float4 x = src[0], y = src[1];
          v[0] = fmaf(x.x, e[ww], v[0]);
          v[1] = fmaf(x.y, e[ww], v[1]);
          v[2] = fmaf(x.z, e[ww], v[2]);
          v[3] = fmaf(x.w, e[ww], v[3]);
          v[4] = fmaf(y.x, e[ww], v[4]);
          v[5] = fmaf(y.y, e[ww], v[5]);
          v[6] = fmaf(y.z, e[ww], v[6]);
          v[7] = fmaf(y.w, e[ww], v[7]);
        }
        if (whole) {
          const float inv = row_scale(sum);
          const int2 to = out_offset(w, w.rt * TR + f0 * 8 + r);
          if (d8 * 8 < p.kv.dim)
            *reinterpret_cast<uint4*>(p.out + (int64_t)to.x * p.ld_out + ((int64_t)to.y * p.kv.dim + d8 * 8) * 2) =
                make_uint4(pack_mean<T>(v[0] * inv, v[1] * inv), pack_mean<T>(v[2] * inv, v[3] * inv),
                           pack_mean<T>(v[4] * inv, v[5] * inv), pack_mean<T>(v[6] * inv, v[7] * inv));
        } else {
          float4* dst = reinterpret_cast<float4*>(p.part_o + (slot * TR + f0 * 8 + r) * DP + d8 * 8);
          dst[0] = make_float4(v[0], v[1], v[2], v[3]);
          dst[1] = make_float4(v[4], v[5], v[6], v[7]);
          if (d8 == 0) p.part_ml[slot * TR + f0 * 8 + r] = make_float2(top, sum);
        }
      }
      __syncthreads();
    }
    if (!whole && threadIdx.x == 0) attn_leave_part(p, w, tile_kb0 == 0, last);
    w = next;
    opened = false;
  }
  cp_async_wait<0>();
}

// ---- more rows, head_dim above 128 ----------------------------------------------
// Tiles of 64 rows, 16 a warp, every warp through all keys of a block; the
// query tile stays in shared memory (its fragments would take the registers
// that the context needs).  Weights are rounded once to the cache's type: the
// products bound it, and the remainder would add half as many again.  Measured:
// 2 x 1024 new tokens over 4096 keys, 16 query and 4 key heads of 256: 664 us =
// 181 TFLOP/s.
template <int DP>
constexpr size_t mid_smem() {
  using S = Shape<DP>;
  return (size_t)S::kStages * 2 * S::kTileBytes + 64 * DP * 2;
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, Shape<DP>::kPerSm) paged_attn_mid_kernel(const AttnParams p) {
  using S = Shape<DP>;
  constexpr int TR = 64, kChunks = DP / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ AttnShare share;
  __shared__ int64_t warp_sum[3 * kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t ring = smem_addr(smem);
  uint8_t* q_tile = smem + (size_t)S::kStages * 2 * S::kTileBytes;
  const uint32_t q_smem = smem_addr(q_tile);

  pdl_wait();
  attn_share<TR, kKeys, kThreads>(p, &share, warp_sum);
  const int64_t u0 = share.u0, u1 = share.u1;
  if (threadIdx.x == 0) attn_no_parts(p);
  if (u1 <= u0) return;

  AttnPos w;
  attn_open<TR, kKeys>(p, share, w);
  Loader<DP, TR> ld;
  ld.open(p, w, u1 - u0);
  for (int s = 0; s < S::kStages - 1; ++s) ld.load(p, ring + s * 2 * S::kTileBytes);

  const int g = lane >> 2, t4 = lane & 3;
  float o[DP / 8][4];
  float m[2], base[2], l[2];
  int lim[2], lim_all = 0;
  int tile_kb0 = w.kb;
  auto open_tile = [&]() {
    tile_kb0 = w.kb;
    lim_all = min(w.r.kv, attn_limit(p, w.r, w.rt * TR));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = w.rt * TR + warp * 16 + g + 8 * i;
      lim[i] = row < w.r.rows ? min(w.r.kv, attn_limit(p, w.r, row)) : 0;
      m[i] = base[i] = kNegInf;
      l[i] = 0.f;
    }
#pragma unroll
    for (int d = 0; d < DP / 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
    // the query tile, in the layout of the keys
    __syncthreads();
    for (int c = threadIdx.x; c < TR * kChunks; c += kThreads) {
      const int r = c / kChunks, col = c % kChunks, row = w.rt * TR + r;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (row < w.r.rows && col * 8 < p.kv.dim) {
        const int tok = row / p.group, hd = w.h * p.group + row % p.group;
        v = *reinterpret_cast<const uint4*>(p.q + (int64_t)(w.r.q0 + tok) * p.ld_q + ((int64_t)hd * p.kv.dim + col * 8) * 2);
      }
      *reinterpret_cast<uint4*>(q_tile + chunk_addr<DP>(0, r, col)) = v;
    }
    __syncthreads();
  };
  open_tile();

  int stage = 0;
  for (int64_t u = u0; u < u1; ++u) {
    cp_async_wait<S::kStages - 2>();
    __syncthreads();
    const uint32_t kt = ring + stage * 2 * S::kTileBytes, vt = kt + S::kTileBytes;
    const int ahead = stage == 0 ? S::kStages - 1 : stage - 1;
    stage = stage + 1 == S::kStages ? 0 : stage + 1;
    ld.load(p, ring + ahead * 2 * S::kTileBytes);

    float s[kKeys / 8][4];
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      uint32_t a[4];
      ldsm4(chunk_addr<DP>(q_smem, warp * 16 + (lane & 15), ks * 2 + (lane >> 4)), a);
#pragma unroll
      for (int n2 = 0; n2 < kKeys / 16; ++n2) {
        uint32_t b[4];
        ldsm4(chunk_addr<DP>(kt, n2 * 16 + (lane & 7) + (lane >> 4) * 8, ks * 2 + ((lane >> 3) & 1)), b);
        mma16816<T>(s[2 * n2], a, b[0], b[1]);
        mma16816<T>(s[2 * n2 + 1], a, b[2], b[3]);
      }
    }
    const int key0 = w.kb * kKeys;
    const bool masked = key0 + kKeys > lim_all;
    float mx[2] = {kNegInf, kNegInf};
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (masked && key0 + n * 8 + 2 * t4 + (i & 1) >= lim[i >> 1]) s[n][i] = kNegInf;
        mx[i >> 1] = fmaxf(mx[i >> 1], s[n][i]);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
    }
    if (__any_sync(0xffffffffu, mx[0] > (base[0] == m[0] ? m[0] : kNegInf) || mx[1] > (base[1] == m[1] ? m[1] : kNegInf))) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float e = mx[i] > m[i] ? exp2_fast((m[i] - mx[i]) * p.scale_log2) : 1.f;   // m = -inf: 0
        m[i] = fmaxf(m[i], mx[i]);
        base[i] = m[i] == kNegInf ? m[i] : row_base(m[i], p.scale_log2);
        l[i] *= e;
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) {
          o[d][2 * i] *= e;
          o[d][2 * i + 1] *= e;
        }
        const float less = base[i] == m[i] ? 0.f : m[i];
#pragma unroll
        for (int n = 0; n < kKeys / 8; ++n) {
          s[n][2 * i] -= less;
          s[n][2 * i + 1] -= less;
        }
      }
    }
    const float plus[2] = {base_offset<T>(base[0], p.scale_log2), base_offset<T>(base[1], p.scale_log2)};
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[n][i] = exp2_fast(fmaf(s[n][i], p.scale_log2, plus[i >> 1]));
        l[i >> 1] += s[n][i];
      }
#pragma unroll
    for (int k2 = 0; k2 < kKeys / 16; ++k2) {
      uint32_t a[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = Num<T>::pack(s[2 * k2 + (i >> 1)][2 * (i & 1)], s[2 * k2 + (i >> 1)][2 * (i & 1) + 1]);
#pragma unroll
      for (int d2 = 0; d2 < DP / 16; ++d2) {
        uint32_t b[4];
        ldsm4_t(chunk_addr<DP>(vt, k2 * 16 + (lane & 15), d2 * 2 + (lane >> 4)), b);
        mma16816<T>(o[2 * d2], a, b[0], b[1]);
        mma16816<T>(o[2 * d2 + 1], a, b[2], b[3]);
      }
    }

    // ---- end of the tile, or of this CTA's share of it
    const bool last = w.kb + 1 == w.nkb;
    if (!last && u + 1 < u1) {
      ++w.kb;
      continue;
    }
    const bool whole = last && tile_kb0 == 0;
    const int64_t slot = 2 * (int64_t)blockIdx.x + (tile_kb0 == 0 ? 1 : 0);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      const int r = warp * 16 + g + 8 * i, row = w.rt * TR + r;
      if (row < w.r.rows && whole) {
        const float inv = row_scale(l[i]);
        const int tok = row / p.group, hd = w.h * p.group + row % p.group;
        char* dst = p.out + (int64_t)(w.r.q0 + tok) * p.ld_out + (int64_t)hd * p.kv.dim * 2;
#pragma unroll
        for (int d = 0; d < DP / 8; ++d)
          if (d * 8 < p.kv.dim)
            *reinterpret_cast<uint32_t*>(dst + (d * 8 + 2 * t4) * 2) = pack_mean<T>(o[d][2 * i] * inv, o[d][2 * i + 1] * inv);
      } else if (row < w.r.rows) {
        float* dst = p.part_o + (slot * TR + r) * DP;
#pragma unroll
        for (int d = 0; d < DP / 8; ++d)
          *reinterpret_cast<float2*>(dst + d * 8 + 2 * t4) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
        if (t4 == 0) p.part_ml[slot * TR + r] = make_float2(m[i], l[i]);
      }
      __syncwarp();
    }
    if (!whole && threadIdx.x == 0) attn_leave_part(p, w, tile_kb0 == 0, last);
    if (u + 1 < u1) {
      attn_next_tile<TR, kKeys>(p, w);
      open_tile();
    }
  }
  cp_async_wait<0>();
  pdl_trigger();
}

constexpr int kJoinWarps = 32;

// Joins the pieces of the tiles that CTAs left unfinished: CTA c's slot 1, then
// slot 0 of the CTAs after it up to the one where the tile ends.  One CTA per
// c (and slice of a tall tile's rows): its warps are dealt to the rows, several
// a row when there are fewer rows, each taking every w-th piece with a running
// maximum of its own; a row's warps meet in shared memory in warp order.  The
// pieces were just written, so they come from L2; bound by the latency of
// three dependent reads (7 to 8 us alone, 10 for 8 rows of 74 pieces).  Two CTAs
// an SM: all of the few-row kernel's CTAs are joined at once (a second round
// cost a prompt beside decoding requests 7 of 99 us).
template <typename T, int TR, int DP>
__global__ void __launch_bounds__(32 * kJoinWarps, DP <= 128 ? 2 : 1) paged_attn_join_kernel(const AttnParams p, int ctas) {
  constexpr int kRows = TR < kJoinWarps ? TR : kJoinWarps;    // rows a CTA joins
  constexpr int kCols = DP >= 128 ? 4 : 2;                    // consecutive columns a lane
  constexpr int kN = DP / 32;                                 // columns a lane
  __shared__ float acc[kJoinWarps][DP];
  __shared__ float2 wml[kJoinWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x;
  pdl_wait();
  const int4 hd = p.head[c];
  // the state of every CTA after c, 32 at a time, all loads in flight together
  constexpr int kLook = 10;
  int st[kLook];
#pragma unroll
  for (int i = 0; i < kLook; ++i) {
    const int o = c + 1 + i * 32 + lane;
    st[i] = o < ctas ? p.state[o] : kPartEnds;                // the last CTA ends the line
  }
  pdl_trigger();
  if (hd.x < 0) return;
  int n = 0;
#pragma unroll
  for (int i = 0; i < kLook; ++i) {
    const unsigned ends = __ballot_sync(0xffffffffu, st[i] == kPartEnds);
    if (n == 0 && ends) n = 1 + i * 32 + __ffs(ends);
  }
  for (int i = kLook; n == 0; ++i) {                          // GPUs with more SMs than that
    const int o = c + 1 + i * 32 + lane;
    const unsigned ends = __ballot_sync(0xffffffffu, o >= ctas || p.state[o] == kPartEnds);
    if (ends) n = 1 + i * 32 + __ffs(ends);
  }
  n = min(n, ctas - c);
  const int row0 = hd.z * TR + blockIdx.y * kRows;
  const int rows = min(kRows, hd.y - row0);                   // of this CTA's
  if (rows <= 0) return;
  int share = 1;                                              // warps a row
  while (share * 2 * rows <= kJoinWarps) share *= 2;
  const int row_t = warp / share, part = warp % share;
  float m = kNegInf, l = 0.f, a[kN] = {};
  if (row_t < rows) {
#pragma unroll 8
    for (int i = part; i < n; i += share) {
      const int64_t at = (i == 0 ? 2 * (int64_t)c + 1 : 2 * (int64_t)(c + i)) * TR + blockIdx.y * kRows + row_t;
      const float2 ml = p.part_ml[at];
      const float* src = p.part_o + at * DP + lane * kCols;
      float v[kN];
#pragma unroll
      for (int s = 0; s < kN / kCols; ++s) {
        if (kCols == 4) *reinterpret_cast<float4*>(v + 4 * s) = *reinterpret_cast<const float4*>(src + s * 128);
        else *reinterpret_cast<float2*>(v + 2 * s) = *reinterpret_cast<const float2*>(src + s * 64);
      }
      const bool some = ml.y != 0.f;    // or it saw no key, and its context may not have been written
      const bool up = some && ml.x > m;
      const float t = exp2_fast(-fabsf((m - ml.x) * p.scale_log2));   // of the lower maximum
      const float f = up ? t : 1.f, e = up ? 1.f : some ? t : 0.f;
      if (up) m = ml.x;
      l = fmaf(ml.y, e, l * f);
#pragma unroll
      for (int k = 0; k < kN; ++k) a[k] = fmaf(some ? v[k] : 0.f, e, a[k] * f);
    }
  }
  if (share > 1) {
    if (lane == 0) wml[warp] = make_float2(m, l);
#pragma unroll
    for (int k = 0; k < kN; ++k) acc[warp][(k / kCols) * 32 * kCols + lane * kCols + k % kCols] = a[k];
    __syncthreads();
    if (part || row_t >= rows) return;
    float top = m;
    for (int w = 1; w < share; ++w) top = fmaxf(top, wml[warp + w].x);
    const float f = m == kNegInf ? 0.f : exp2_fast((m - top) * p.scale_log2);
    l *= f;
#pragma unroll
    for (int k = 0; k < kN; ++k) a[k] *= f;
    for (int w = 1; w < share; ++w) {
      const float2 ml = wml[warp + w];
      if (ml.y == 0.f) continue;
      const float e = exp2_fast((ml.x - top) * p.scale_log2);
      l = fmaf(ml.y, e, l);
#pragma unroll
      for (int k = 0; k < kN; ++k)
        a[k] = fmaf(acc[warp + w][(k / kCols) * 32 * kCols + lane * kCols + k % kCols], e, a[k]);
    }
  }
  if (row_t >= rows) return;
  const float inv = row_scale(l);
  const int row = row0 + row_t, tok = row / p.group, head = hd.w * p.group + row % p.group;
  char* dst = p.out + (int64_t)(hd.x + tok) * p.ld_out + (int64_t)head * p.kv.dim * 2;
#pragma unroll
  for (int k = 0; k < kN; k += 2) {
    const int d = (k / kCols) * 32 * kCols + lane * kCols + k % kCols;
    if (d < p.kv.dim) *reinterpret_cast<uint32_t*>(dst + d * 2) = pack_mean<T>(a[k] * inv, a[k + 1] * inv);
  }
}

// TR rows a tile: 8 to 24 on the few-row kernel, 64 on the other.  The joining
// comes behind all kernels of a call (run_join).
template <typename T, int DP, int TR>
int run_class(AttnParams& p, void* workspace, bool splits, int sms, cudaStream_t stream) {
  const int ctas = sms * Shape<DP>::kPerSm;
  attn_carve<TR, DP>(p, splits ? workspace : nullptr, ctas);
  void (*kernel)(AttnParams);
  size_t smem;
  if constexpr (TR == 64) {
    kernel = paged_attn_mid_kernel<T, DP>;
    smem = mid_smem<DP>();
  } else {
    kernel = paged_attn_few_kernel<T, DP, TR / 8>;
    smem = few_smem<DP, TR / 8>();
  }
  static std::atomic<uint64_t> allowed{0};
  SMEAI_CUDA_TRY(attn_allow_smem(kernel, smem, allowed));
  SMEAI_CUDA_TRY(launch(kernel, dim3((unsigned)ctas), dim3(kThreads), smem, stream, p));
  return kOk;
}
template <typename T, int DP, int TR>
int run_join(const AttnParams& p, int sms, cudaStream_t stream) {
  if (p.head) SMEAI_CUDA_TRY((attn_join<T, TR, DP>(p, sms * Shape<DP>::kPerSm, stream)));
  return kOk;
}

// Which kernels a call needs, from what the host knows: the largest request's
// packed rows and the total.
//   up to 8, 16, 24 rows  tiles of so many: one reading of the keys for all
//   more                  the tensor-core kernel, and beside it the 8-row tiles
//                         (16 with more than 8 heads a key head) for requests
//                         of so few rows (a step that mixes prompts and
//                         decoding) unless the total says that there are none:
//                         one row costs the tensor-core kernel's tile as much
//                         as 128, and 8 requests, one of 860 rows, took 148 us
//                         without the second kernel and 104 us with it.  Rows
//                         behind the last request count into the total: padded
//                         up to n_req * max_new, a step's few rows take the
//                         tensor-core kernel
// head_dim above 128: up to 16 rows as above, more the 64-row tiles for all.
struct Classes {
  int few;      // rows a tile of the few-row kernel; 0: not needed
  bool mid, many;
};
Classes classes(const PagedAttention& a) {
  const int64_t group = a.n_heads / a.kv.n_kv, most = a.max_new * group;
  Classes c = {0, false, false};
  if (most <= 16) c.few = most <= 8 ? 8 : 16;
  else if (a.kv.dim > 128) c.mid = true;
  else if (most <= 24) c.few = 24;
  else {
    c.many = true;
    // with one request of so few rows the others, of max_new at most, could not make up more tokens
    const int tile = group <= 8 ? 8 : 16;
    if (group <= tile && a.n_tokens <= (a.n_req - 1) * a.max_new + tile / group) c.few = tile;
  }
  return c;
}

int padded_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// Workspace of the few-row kernel, whichever its tile, a multiple of 256 bytes.
size_t few_part_bytes(int dp, int max_kv, int sms) {
  if (!attn_splits<kKeys>(max_kv)) return 0;
  const size_t n = dp == 64    ? attn_part_bytes<24, 64>(2 * sms)
                   : dp == 128 ? attn_part_bytes<24, 128>(2 * sms)
                               : attn_part_bytes<16, 256>(sms);
  return (n + 255) / 256 * 256;
}

template <typename T, int DP, int TR>
int run_few(AttnParams p, const PagedAttention& a, const Classes& c, int sms, cudaStream_t stream) {
  if (c.many) p.rows_hi = TR;
  const bool splits = attn_splits<kKeys>(a.max_kv);
  int st = run_class<T, DP, TR>(p, a.workspace, splits, sms, stream);
  if (st) return st;
  if constexpr (DP <= 128 && TR <= 16) {
    if (c.many) {
      // the tensor-core kernel in between: it has nothing to do with these
      // partial results, and its set-up hides behind the first kernel's end
      AttnParams q = p;
      q.rows_hi = 0x7fffffff;
      q.rows_lo = TR;
      st = paged_attn_tc(q, DP, static_cast<char*>(a.workspace) + few_part_bytes(DP, a.max_kv, sms), a.max_kv, sms, stream);
      if (st) return st;
    }
  }
  return run_join<T, DP, TR>(p, sms, stream);
}

template <typename T, int DP>
int run_dim(const AttnParams& p, const PagedAttention& a, int sms, cudaStream_t stream) {
  const Classes c = classes(a);
  if (c.few == 8) return run_few<T, DP, 8>(p, a, c, sms, stream);
  if (c.few == 16) return run_few<T, DP, 16>(p, a, c, sms, stream);
  if constexpr (DP > 128) {
    AttnParams q = p;
    const int st = run_class<T, DP, 64>(q, a.workspace, attn_splits<kKeys>(a.max_kv), sms, stream);
    return st ? st : run_join<T, DP, 64>(q, sms, stream);
  } else {
    if (c.few == 24) return run_few<T, DP, 24>(p, a, c, sms, stream);
    return paged_attn_tc(p, DP, a.workspace, a.max_kv, sms, stream);
  }
}

}  // namespace

template <typename T, int TR, int DP>
cudaError_t attn_join(const AttnParams& p, int ctas, cudaStream_t stream) {
  return launch(paged_attn_join_kernel<T, TR, DP>, dim3((unsigned)ctas, (unsigned)((TR + kJoinWarps - 1) / kJoinWarps)),
                dim3(32 * kJoinWarps), 0, stream, p, ctas);
}
template cudaError_t attn_join<__half, 256, 64>(const AttnParams&, int, cudaStream_t);
template cudaError_t attn_join<__half, 256, 128>(const AttnParams&, int, cudaStream_t);
template cudaError_t attn_join<__nv_bfloat16, 256, 64>(const AttnParams&, int, cudaStream_t);
template cudaError_t attn_join<__nv_bfloat16, 256, 128>(const AttnParams&, int, cudaStream_t);

size_t paged_attention_workspace(const PagedAttention& a) {
  int sms = 0;
  if (sm_count(&sms)) return 0;
  const Classes c = classes(a);
  const int dp = padded_dim(a.kv.dim);
  size_t need = 0;
  if (c.few) need += few_part_bytes(dp, a.max_kv, sms);
  if (c.mid && attn_splits<kKeys>(a.max_kv)) need += attn_part_bytes<64, 256>(sms);
  if (c.many) need += paged_attn_tc_workspace(dp, a.max_kv, sms);
  return need;
}

int paged_attention(const PagedAttention& a, cudaStream_t stream) {
  AttnParams p;
  p.kv = a.kv;
  p.q = static_cast<const char*>(a.q);
  p.out = static_cast<char*>(a.out);
  p.ld_q = a.ld_q * 2;
  p.ld_out = a.ld_out * 2;
  p.q_start = a.q_start;
  p.kv_len = a.kv_len;
  p.table = a.table;
  p.ld_table = a.ld_table;
  p.n_req = a.n_req;
  p.max_kv = a.max_kv;
  p.n_tokens = (int)a.n_tokens;
  p.group = a.n_heads / a.kv.n_kv;
  p.scale_log2 = a.scale * 1.4426950408889634f;   // finite: the entry point checks it
  p.causal = a.causal ? 1 : 0;
  p.rows_lo = 0;
  p.rows_hi = 0x7fffffff;
  p.err = device_error_ptr();
  int sms = 0;
  const int st = sm_count(&sms);
  if (st) return st;
  if (!p.err) {
    set_last_error("paged_attention: no device error word");
    return kCudaError;
  }
  const int dp = padded_dim(a.kv.dim);
  if (a.kv.bf16)
    return dp == 64    ? run_dim<__nv_bfloat16, 64>(p, a, sms, stream)
           : dp == 128 ? run_dim<__nv_bfloat16, 128>(p, a, sms, stream)
                       : run_dim<__nv_bfloat16, 256>(p, a, sms, stream);
  return dp == 64    ? run_dim<__half, 64>(p, a, sms, stream)
         : dp == 128 ? run_dim<__half, 128>(p, a, sms, stream)
                     : run_dim<__half, 256>(p, a, sms, stream);
}

}  // namespace smeai
