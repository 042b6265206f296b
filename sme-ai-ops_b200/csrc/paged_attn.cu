// paged_attn.cu -- attention of new tokens over a paged key/value cache for
// requests that bring few rows (a decoding step, drafted tokens, short
// chunks), and the joining of partial results.
//
//   o_r = sum_j p_rj v_j / sum_j p_rj,   p_rj = 2^(c s_rj - m_r),
//   s_rj = q_r . k_j,  c = scale log2(e),  m_r = max over the keys seen so far of c s_rj
//
// in one pass over the keys: when m_r grows by d, the sum and the context
// gathered so far are multiplied by 2^-d.
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
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Shared-memory layout: [stages][K, V][kKeys rows][DP] 16-bit, the 16-byte
// chunks of a row XORed with the row's index mod 8, so that ldmatrix's eight
// rows fall on different banks; then the merge buffer.
template <int DP>
struct Shape {
  static constexpr int kRowBytes = DP * 2;
  static constexpr int kTileBytes = kKeys * kRowBytes;
  static constexpr int kStages = DP == 64 ? 6 : 3;      // 96 KB in flight (192 KB at DP 256)
  static constexpr int kPerSm = DP == 256 ? 1 : 2;      // CTAs an SM
};
template <int DP, int MT>
constexpr size_t smem_bytes() {
  using S = Shape<DP>;
  return (size_t)S::kStages * 2 * S::kTileBytes + (MT == 0 ? 64 * DP * 2 : 2 * 16 * DP * 4);
}

template <int DP>
__device__ __forceinline__ uint32_t chunk_addr(uint32_t base, int row, int chunk) {
  return base + row * Shape<DP>::kRowBytes + ((chunk ^ (row & 7)) << 4);
}

// MT 1, 2: tiles of 16 or 32 rows (a decode step's query heads of one key
//   head, or those of a few drafted tokens).  All rows meet every key, and each
//   warp takes 16 of a block's 64 keys, with its own ring of keys in shared
//   memory: warps never wait for one another before the tile's end, where
//   their maxima, sums and contexts are merged.  Per 16 keys, 16 rows and 128
//   elements a warp issues 32 mma for 8 KB of cache; HBM's share of an SM (44
//   GB/s) leaves five times the issue slots that this takes, so the kernel is
//   bound by the cache's bytes.
// MT 0: tiles of 64 rows, 16 a warp, every warp through all keys (head_dim
//   above 128 with many rows).
//
// Two CTAs an SM with 96 KB of keys and values in flight each cover HBM's
// latency (44 GB/s x ~1 us = 44 KB an SM) through the ends of tiles.
// Each lane looks up the page of one key a block ahead and hands the address
// to the lanes that copy the row, so the table's latency hides behind a block.
template <typename T, int DP, int MT>
__global__ void __launch_bounds__(kThreads, Shape<DP>::kPerSm) paged_attn_kernel(const AttnParams p) {
  using S = Shape<DP>;
  constexpr bool kRowSplit = MT == 0;
  constexpr int M = kRowSplit ? 1 : MT;          // 16-row fragments a warp computes with
  constexpr int TR = kRowSplit ? 64 : 16 * MT;
  constexpr int NK = kRowSplit ? 64 : 16;        // keys a warp computes with per block
  constexpr int kChunks = DP / 8;                // 16-byte chunks a row
  constexpr bool kQRegs = DP * M <= 128;         // query fragments live in registers, or the tile in shared memory
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ AttnShare share;
  __shared__ int64_t warp_sum[kWarps];
  __shared__ float merge_m[kWarps][16], merge_l[kWarps][16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t ring = smem_addr(smem);
  float* merge = reinterpret_cast<float*>(smem + (size_t)S::kStages * 2 * S::kTileBytes);
  const uint32_t q_smem = smem_addr(merge);      // the query tile, while nothing is merged

  pdl_wait();
  attn_share<TR, kKeys, kThreads>(p, &share, warp_sum);
  const int64_t u0 = share.u0, u1 = share.u1;
  if (threadIdx.x == 0) attn_no_parts(p);
  if (u1 <= u0) return;

  // ---- loading: `ld` walks ahead of the computation
  AttnPos ld;
  attn_open<TR, kKeys>(p, share, ld);
  AttnPos w = ld;
  int64_t to_load = u1 - u0;
  const int page_mask = (1 << p.kv.page_log2) - 1;
  int page = -1;                                  // page of this lane's key in block `ld`
  auto look_up = [&]() {
    const int key = ld.kb * kKeys + warp * 16 + (lane & 15);
    page = key < ld.r.kv ? p.table[(int64_t)ld.b * p.ld_table + (key >> p.kv.page_log2)] : -1;
    if (key < ld.r.kv && (page < 0 || page >= p.kv.n_pages)) {
      raise_device_error(p.err, kDevErrBadIndex);
      page = -1;
    }
  };
  auto load_block = [&](int stage) {
    if (to_load > 0) {
      const int key = ld.kb * kKeys + warp * 16 + (lane & 15);
      // byte offset of this lane's key row, or -1: nothing there, zeros instead
      const int64_t off = page < 0 ? -1
                                   : page * p.kv.page_bytes + (key & page_mask) * p.kv.token_bytes +
                                         ld.h * p.kv.head_bytes;
      const uint32_t kt = ring + (stage * 2) * S::kTileBytes, vt = kt + S::kTileBytes;
      constexpr int kPer = 16 * kChunks / 32;     // chunks a lane copies of K, and of V
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int c = i * 32 + lane, row = c / kChunks, col = c % kChunks;
        const int64_t o = __shfl_sync(0xffffffffu, off, row);
        const int n = o >= 0 && col * 8 < p.kv.dim ? 16 : 0;
        const int64_t at = n ? o + col * 16 : 0;
        const int r = warp * 16 + row;
        cp_async16(chunk_addr<DP>(kt, r, col), p.kv.k + at, n);
        cp_async16(chunk_addr<DP>(vt, r, col), p.kv.v + at, n);
      }
      if (--to_load > 0) {
        if (++ld.kb == ld.nkb) attn_next_tile<TR, kKeys>(p, ld);
        look_up();
      }
    }
    cp_async_commit();
  };
  look_up();
  for (int s = 0; s < S::kStages - 1; ++s) load_block(s);

  // ---- computing
  const int g = lane >> 2, t4 = lane & 3;
  uint32_t qf[kQRegs ? DP / 16 : 1][M][4];
  float o[M][DP / 8][4];
  float m[M][2], l[M][2];
  int lim[M][2], lim_all = 0;
  int tile_kb0 = w.kb;
  // rows of this lane in fragment f: f * 16 + g and f * 16 + g + 8 of the warp's
  const int row_in = (kRowSplit ? warp * 16 : 0) + g;
  auto open_tile = [&]() {
    tile_kb0 = w.kb;
    lim_all = min(w.r.kv, attn_limit(p, w.r, w.rt * TR));
#pragma unroll
    for (int f = 0; f < M; ++f) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = w.rt * TR + row_in + f * 16 + 8 * i;
        lim[f][i] = row < w.r.rows ? min(w.r.kv, attn_limit(p, w.r, row)) : 0;
        m[f][i] = kNegInf;
        l[f][i] = 0.f;
      }
#pragma unroll
      for (int d = 0; d < DP / 8; ++d) o[f][d][0] = o[f][d][1] = o[f][d][2] = o[f][d][3] = 0.f;
    }
    auto q_row = [&](int row) -> const char* {
      const int tok = row / p.group, hd = w.h * p.group + row % p.group;
      return p.q + (int64_t)(w.r.q0 + tok) * p.ld_q + (int64_t)hd * p.kv.dim * 2;
    };
    if (kQRegs) {
#pragma unroll
      for (int f = 0; f < M; ++f)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = w.rt * TR + row_in + f * 16 + 8 * i;
          const bool live = row < w.r.rows;
          const char* src = q_row(live ? row : 0);
#pragma unroll
          for (int ks = 0; ks < DP / 16; ++ks) {
            const int d = ks * 16 + 2 * t4;
            qf[kQRegs ? ks : 0][f][i] = live && d < p.kv.dim ? *reinterpret_cast<const uint32_t*>(src + d * 2) : 0u;
            qf[kQRegs ? ks : 0][f][i + 2] =
                live && d + 8 < p.kv.dim ? *reinterpret_cast<const uint32_t*>(src + d * 2 + 16) : 0u;
          }
        }
    } else {
      // the query tile in shared memory, in the layout of the keys
      __syncthreads();
      for (int c = threadIdx.x; c < TR * kChunks; c += kThreads) {
        const int r = c / kChunks, col = c % kChunks, row = w.rt * TR + r;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (row < w.r.rows && col * 8 < p.kv.dim) v = *reinterpret_cast<const uint4*>(q_row(row) + col * 16);
        *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(merge) + (chunk_addr<DP>(0, r, col))) = v;
      }
      __syncthreads();
    }
  };
  open_tile();

  for (int64_t u = u0; u < u1; ++u) {
    const int stage = (int)((u - u0) % S::kStages);
    cp_async_wait<S::kStages - 2>();
    if (kRowSplit) __syncthreads();
    else __syncwarp();
    load_block((int)((u - u0 + S::kStages - 1) % S::kStages));

    const uint32_t kt = ring + (stage * 2) * S::kTileBytes, vt = kt + S::kTileBytes;
    const int krow0 = kRowSplit ? 0 : warp * 16;    // first of this warp's keys in the block
    float s[M][NK / 8][4];
#pragma unroll
    for (int f = 0; f < M; ++f)
#pragma unroll
      for (int n = 0; n < NK / 8; ++n) s[f][n][0] = s[f][n][1] = s[f][n][2] = s[f][n][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      uint32_t a[M][4];
#pragma unroll
      for (int f = 0; f < M; ++f) {
        if (kQRegs) {
#pragma unroll
          for (int i = 0; i < 4; ++i) a[f][i] = qf[kQRegs ? ks : 0][f][i];
        } else {
          const int r = (kRowSplit ? warp * 16 : f * 16) + (lane & 7) + ((lane >> 3) & 1) * 8;
          ldsm4(chunk_addr<DP>(q_smem, r, ks * 2 + (lane >> 4)), a[f]);
        }
      }
#pragma unroll
      for (int n2 = 0; n2 < NK / 16; ++n2) {
        uint32_t b[4];
        const int r = krow0 + n2 * 16 + (lane & 7) + ((lane >> 4) & 1) * 8;
        ldsm4(chunk_addr<DP>(kt, r, ks * 2 + ((lane >> 3) & 1)), b);
#pragma unroll
        for (int f = 0; f < M; ++f) {
          mma16816<T>(s[f][2 * n2], a[f], b[0], b[1]);
          mma16816<T>(s[f][2 * n2 + 1], a[f], b[2], b[3]);
        }
      }
    }
    const int key0 = w.kb * kKeys + krow0;
    const bool masked = key0 + NK > lim_all;
#pragma unroll
    for (int f = 0; f < M; ++f) {
      float mx[2] = {kNegInf, kNegInf};
#pragma unroll
      for (int n = 0; n < NK / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (masked && key0 + n * 8 + 2 * t4 + (i & 1) >= lim[f][i >> 1]) s[f][n][i] = kNegInf;
          mx[i >> 1] = fmaxf(mx[i >> 1], s[f][n][i]);
        }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
        mx[i] = fmaxf(m[f][i], mx[i] * p.scale_log2);
      }
      if (__any_sync(0xffffffffu, mx[0] > m[f][0] || mx[1] > m[f][1])) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float e = mx[i] > m[f][i] ? exp2_fast(m[f][i] - mx[i]) : 1.f;   // m = -inf: 0
          m[f][i] = mx[i];
          l[f][i] *= e;
#pragma unroll
          for (int d = 0; d < DP / 8; ++d) {
            o[f][d][2 * i] *= e;
            o[f][d][2 * i + 1] *= e;
          }
        }
      }
      const float sub[2] = {m[f][0] == kNegInf ? 0.f : Num<T>::kBias - m[f][0],
                            m[f][1] == kNegInf ? 0.f : Num<T>::kBias - m[f][1]};
#pragma unroll
      for (int n = 0; n < NK / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[f][n][i] = exp2_fast(fmaf(s[f][n][i], p.scale_log2, sub[i >> 1]));
          l[f][i >> 1] += s[f][n][i];
        }
    }
#pragma unroll
    for (int k2 = 0; k2 < NK / 16; ++k2) {
      uint32_t a[M][4];
#pragma unroll
      for (int f = 0; f < M; ++f)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          a[f][i] = Num<T>::pack(s[f][2 * k2 + (i >> 1)][2 * (i & 1)], s[f][2 * k2 + (i >> 1)][2 * (i & 1) + 1]);
#pragma unroll
      for (int d2 = 0; d2 < DP / 16; ++d2) {
        uint32_t b[4];
        const int r = krow0 + k2 * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
        ldsm4_t(chunk_addr<DP>(vt, r, d2 * 2 + (lane >> 4)), b);
#pragma unroll
        for (int f = 0; f < M; ++f) {
          mma16816<T>(o[f][2 * d2], a[f], b[0], b[1]);
          mma16816<T>(o[f][2 * d2 + 1], a[f], b[2], b[3]);
        }
      }
    }

    // ---- end of the tile, or of this CTA's share of it
    const bool last = w.kb + 1 == w.nkb;
    if (last || u + 1 == u1) {
      const bool whole = last && tile_kb0 == 0;
      // slot 0: a tile entered in the middle; slot 1: a tile left unfinished
      const int64_t slot = 2 * (int64_t)blockIdx.x + (tile_kb0 == 0 ? 1 : 0);
      auto out_row = [&](int row) -> char* {
        const int tok = row / p.group, hd = w.h * p.group + row % p.group;
        return p.out + (int64_t)(w.r.q0 + tok) * p.ld_out + (int64_t)hd * p.kv.dim * 2;
      };
#pragma unroll
      for (int f = 0; f < M; ++f) {
        const int frag_rows = w.r.rows - w.rt * TR - f * 16;   // rows from this fragment on
        if (!kRowSplit && frag_rows <= 0) break;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          l[f][i] += __shfl_xor_sync(0xffffffffu, l[f][i], 1);
          l[f][i] += __shfl_xor_sync(0xffffffffu, l[f][i], 2);
        }
        if (kRowSplit) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = row_in + 8 * i, row = w.rt * TR + r;
            if (row >= w.r.rows) continue;
            if (whole) {
              const float inv = l[f][i] > 0.f ? 1.f / l[f][i] : (l[f][i] == 0.f ? 0.f : l[f][i]);
              char* dst = out_row(row);
#pragma unroll
              for (int d = 0; d < DP / 8; ++d)
                if (d * 8 < p.kv.dim)
                  *reinterpret_cast<uint32_t*>(dst + (d * 8 + 2 * t4) * 2) =
                      Num<T>::pack(o[f][d][2 * i] * inv, o[f][d][2 * i + 1] * inv);
            } else {
              float* dst = p.part_o + (slot * TR + r) * DP;
#pragma unroll
              for (int d = 0; d < DP / 8; ++d)
                *reinterpret_cast<float2*>(dst + d * 8 + 2 * t4) = make_float2(o[f][d][2 * i], o[f][d][2 * i + 1]);
              if (t4 == 0) p.part_ml[slot * TR + r] = make_float2(m[f][i], l[f][i]);
            }
          }
          continue;
        }
        // merge the warps: their common maximum, then the contexts added up in
        // a fixed order
        if (t4 == 0) {
          merge_m[warp][g] = m[f][0];
          merge_m[warp][g + 8] = m[f][1];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = merge_m[0][g + 8 * i];
#pragma unroll
          for (int ww = 1; ww < kWarps; ++ww) top = fmaxf(top, merge_m[ww][g + 8 * i]);
          const float e = m[f][i] == kNegInf ? 0.f : exp2_fast(m[f][i] - top);
          l[f][i] *= e;
#pragma unroll
          for (int d = 0; d < DP / 8; ++d) {
            o[f][d][2 * i] *= e;
            o[f][d][2 * i + 1] *= e;
          }
        }
        if (t4 == 0) {
          merge_l[warp][g] = l[f][0];
          merge_l[warp][g + 8] = l[f][1];
        }
        // warps 2 and 3 leave theirs in a buffer each, warps 0 and 1 add their own
        static_assert(kWarps == 4, "merge order");
#pragma unroll
        for (int step = 0; step < 2; ++step) {
          if ((warp >> 1) != step) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int d = 0; d < DP / 8; ++d) {
                // columns XORed with the row, so that the eight rows of a store take different banks
                float2* dst = reinterpret_cast<float2*>(merge + (warp & 1) * 16 * DP + (g + 8 * i) * DP +
                                                        ((d * 8 + 2 * t4) ^ (g * 8)));
                float2 v = make_float2(o[f][d][2 * i], o[f][d][2 * i + 1]);
                if (step) {
                  const float2 old = *dst;
                  v.x = old.x + v.x;
                  v.y = old.y + v.y;
                }
                *dst = v;
              }
          }
          __syncthreads();
        }
        for (int c = threadIdx.x; c < 16 * (DP / 8); c += kThreads) {
          const int r = c / (DP / 8), d8 = c % (DP / 8);
          if (r >= frag_rows) break;
          const float4* src = reinterpret_cast<const float4*>(merge + r * DP + ((d8 * 8) ^ ((r & 7) * 8)));
          float4 a = src[0], b = src[1];
          const float4 a1 = src[16 * DP / 4], b1 = src[16 * DP / 4 + 1];
          a = make_float4(a.x + a1.x, a.y + a1.y, a.z + a1.z, a.w + a1.w);
          b = make_float4(b.x + b1.x, b.y + b1.y, b.z + b1.z, b.w + b1.w);
          const float sum = merge_l[0][r] + merge_l[1][r] + merge_l[2][r] + merge_l[3][r];
          if (whole) {
            const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
            if (d8 * 8 < p.kv.dim)
              *reinterpret_cast<uint4*>(out_row(w.rt * TR + f * 16 + r) + d8 * 16) =
                  make_uint4(Num<T>::pack(a.x * inv, a.y * inv), Num<T>::pack(a.z * inv, a.w * inv),
                             Num<T>::pack(b.x * inv, b.y * inv), Num<T>::pack(b.z * inv, b.w * inv));
          } else {
            float4* dst = reinterpret_cast<float4*>(p.part_o + (slot * TR + f * 16 + r) * DP + d8 * 8);
            dst[0] = a;
            dst[1] = b;
            if (d8 == 0) {
              const float top_m = fmaxf(fmaxf(merge_m[0][r], merge_m[1][r]), fmaxf(merge_m[2][r], merge_m[3][r]));
              p.part_ml[slot * TR + f * 16 + r] = make_float2(top_m, sum);
            }
          }
        }
        __syncthreads();
      }
      if (!whole && threadIdx.x == 0) attn_leave_part(p, w, tile_kb0 == 0, last);
      if (u + 1 < u1) {
        attn_next_tile<TR, kKeys>(p, w);
        open_tile();
      }
    } else {
      ++w.kb;
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
// three dependent reads.
template <typename T, int TR, int DP>
__global__ void __launch_bounds__(32 * kJoinWarps) paged_attn_join_kernel(const AttnParams p, int ctas) {
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
      const float top = some ? fmaxf(m, ml.x) : m;
      const float f = m == top ? 1.f : exp2_fast(m - top), e = some ? exp2_fast(ml.x - top) : 0.f;
      m = top;
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
    const float f = m == kNegInf ? 0.f : exp2_fast(m - top);
    l *= f;
#pragma unroll
    for (int k = 0; k < kN; ++k) a[k] *= f;
    for (int w = 1; w < share; ++w) {
      const float2 ml = wml[warp + w];
      if (ml.y == 0.f) continue;
      const float e = exp2_fast(ml.x - top);
      l = fmaf(ml.y, e, l);
#pragma unroll
      for (int k = 0; k < kN; ++k)
        a[k] = fmaf(acc[warp + w][(k / kCols) * 32 * kCols + lane * kCols + k % kCols], e, a[k]);
    }
  }
  if (row_t >= rows) return;
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  const int row = row0 + row_t, tok = row / p.group, head = hd.w * p.group + row % p.group;
  char* dst = p.out + (int64_t)(hd.x + tok) * p.ld_out + (int64_t)head * p.kv.dim * 2;
#pragma unroll
  for (int k = 0; k < kN; k += 2) {
    const int d = (k / kCols) * 32 * kCols + lane * kCols + k % kCols;
    if (d < p.kv.dim) *reinterpret_cast<uint32_t*>(dst + d * 2) = Num<T>::pack(a[k] * inv, a[k + 1] * inv);
  }
}

template <typename T, int DP, int MT>
int run_class(AttnParams p, const PagedAttention& a, int sms, cudaStream_t stream) {
  constexpr int TR = MT == 0 ? 64 : 16 * MT;
  const int ctas = sms * Shape<DP>::kPerSm;
  attn_carve<TR, DP>(p, a.workspace, ctas);
  constexpr size_t smem = smem_bytes<DP, MT>();
  auto kernel = paged_attn_kernel<T, DP, MT>;
  SMEAI_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  SMEAI_CUDA_TRY(launch(kernel, dim3((unsigned)ctas), dim3(kThreads), smem, stream, p));
  // a tile of up to 2 * kSnap blocks is never split
  if (a.max_kv > 2 * kSnap * kKeys) SMEAI_CUDA_TRY((attn_join<T, TR, DP>(p, ctas, stream)));
  return kOk;
}

// Which kernels a call needs, from what the host knows: the largest request's
// packed rows and the total.
//   up to 16 rows   16-row tiles
//   up to 32        32-row tiles: one reading of the keys for all rows
//   more            the tensor-core kernel, and the 16-row tiles beside it for
//                   requests of up to 16 rows (a step that mixes prompts and
//                   decoding) unless the total says that there are none: one
//                   row costs the tensor-core kernel's tile as much as 256,
//                   and 8 requests, one of 860 rows, took 148 us without the
//                   second kernel and 104 us with it
// head_dim above 128: up to 16 rows as above, more the 64-row tiles for all.
struct Classes {
  bool few, mid, many;
};
Classes classes(const PagedAttention& a) {
  const int64_t group = a.n_heads / a.kv.n_kv, most = a.max_new * group;
  Classes c = {false, false, false};
  if (most <= 16) c.few = true;
  else if (most <= 32 || a.kv.dim > 128) c.mid = true;
  else {
    c.many = true;
    // with one request of r <= 16 / group rows the others, of max_new at most, could not make up n_tokens
    c.few = a.n_tokens <= (a.n_req - 1) * a.max_new + 16 / group;
  }
  return c;
}

int padded_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

template <typename T, int DP>
int run_dim(const AttnParams& p, const PagedAttention& a, int sms, cudaStream_t stream) {
  const Classes c = classes(a);
  if (c.few) {
    AttnParams q = p;
    if (c.many) q.rows_hi = 16;
    const int st = run_class<T, DP, 1>(q, a, sms, stream);
    if (st) return st;
  }
  if (c.mid) return run_class<T, DP, DP <= 128 ? 2 : 0>(p, a, sms, stream);
  if constexpr (DP <= 128) {
    if (c.many) {
      AttnParams q = p;
      if (c.few) q.rows_lo = 16;
      return paged_attn_tc(q, DP, a.workspace, a.max_kv, sms, stream);
    }
  }
  return kOk;
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
  if (c.many) return paged_attn_tc_workspace(dp, sms);   // the 16-row tiles' need is smaller
  if (c.mid)
    return dp == 64    ? attn_part_bytes<32, 64>(2 * sms)
           : dp == 128 ? attn_part_bytes<32, 128>(2 * sms)
                       : attn_part_bytes<64, 256>(sms);
  return dp == 64    ? attn_part_bytes<16, 64>(2 * sms)
         : dp == 128 ? attn_part_bytes<16, 128>(2 * sms)
                     : attn_part_bytes<16, 256>(sms);
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
  p.scale_log2 = a.scale * 1.4426950408889634f;
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
