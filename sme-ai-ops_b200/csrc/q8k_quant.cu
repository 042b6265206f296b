// q8k_quant.cu -- standalone activation quantizer (fp32 -> ggml block_q8_K),
// optionally preceded by an RMSNorm of the whole row
// (sme_ai_library/src/sme_ai_ops.c:1060-1092: x / sqrt(mean(x^2) + eps), then
// times weight[j] when a weight is given -- two roundings, as there).
// The arithmetic lives in q8k_device.cuh; one warp quantizes one block.
#include "common.cuh"
#include "kernels.h"
#include "q8k_device.cuh"

namespace smeai {

// Plain quantization: warp per block over rows x blocks.
__global__ void q8k_quantize_kernel(const float* __restrict__ x, int64_t ld_x, int nb, int64_t total_blocks,
                                    uint8_t* __restrict__ y) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warp = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int64_t nwarps = (int64_t)gridDim.x * (blockDim.x >> 5);
  for (int64_t blk = warp; blk < total_blocks; blk += nwarps) {
    const int64_t row = blk / nb, b = blk % nb;
    float v[8];
    load8(x + row * ld_x + b * QK_K + lane * 8, v);
    q8k_store_global(q8k_quantize_lane(v), y + blk * Q8K_BLOCK_BYTES);
  }
}

// RMSNorm + quantization, one CTA per row.
__global__ void rms_q8k_quantize_kernel(const float* __restrict__ x, int64_t ld_x, int nb, float eps,
                                        const float* __restrict__ norm_w, uint8_t* __restrict__ y) {
  extern __shared__ float sm_gsum[];  // 8 group sums per block, then 1/rms
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  const int64_t row = blockIdx.x;
  const float* xr = x + row * ld_x;
  for (int b = warp; b < nb; b += nwarps) {
    float v[8];
    load8(xr + b * QK_K + lane * 8, v);
    const float s = group_sumsq_load8(v);
    if ((lane & 3) == 0) sm_gsum[b * 8 + (lane >> 2)] = s;
  }
  __syncthreads();
  if (warp == 0) {
    const float total = rms_fold_groups(sm_gsum, nb * 8);
    if (lane == 0) sm_gsum[nb * 8] = rms_inv_from_sum(total, nb * QK_K, eps);
  }
  __syncthreads();
  const float inv = sm_gsum[nb * 8];
  for (int b = warp; b < nb; b += nwarps) {
    float v[8];
    load8(xr + b * QK_K + lane * 8, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], inv);
    if (norm_w) {
      float g[8];
      load8(norm_w + b * QK_K + lane * 8, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], g[i]);
    }
    q8k_store_global(q8k_quantize_lane(v), y + (row * nb + b) * Q8K_BLOCK_BYTES);
  }
}

template <bool kAligned>
__device__ __forceinline__ void load8_row(const float* p, float (&v)[8]) {
  if (!kAligned) {
    load8(p, v);
    return;
  }
  const float4 a = *reinterpret_cast<const float4*>(p);
  const float4 b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

// A lane's 8 values of a block: times 1/rms, times the weight (when there is
// one), quantized and stored.
template <bool kWeight>
__device__ __forceinline__ void norm_quantize_store(float (&t)[8], const float (&w)[8], float inv, uint8_t* out) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    t[j] = __fmul_rn(t[j], inv);
    if (kWeight) t[j] = __fmul_rn(t[j], w[j]);
  }
  q8k_store_global(q8k_quantize_lane(t), out);
}

// Residual addition + RMSNorm + quantization, one CTA per row: h = x + resid
// is formed once and kept in registers (kKeep 256-value blocks a warp) between
// the two passes that the norm needs, so a row costs one read of x and of
// resid, one write of h and one of the blocks: 13.1 bytes a value.  All loads
// of a warp (the weight's too) go out together before anything waits; blocks
// past kKeep a warp are read back from h by the lanes that wrote it.  Measured:
// 2048 x 4096 27 us = 4.1 TB/s, one row 3.2 us; the quantization's
// instructions (issue slots 53% busy, mostly waiting between the two barriers)
// bound it, not the bytes.  No __restrict__ on h: it may be x or resid.
template <int kKeep, bool kWeight, bool kAligned>
__global__ void __launch_bounds__(512) add_rms_q8k_quantize_kernel(const float* x, int64_t ld_x, const float* resid,
                                                                   int64_t ld_r, int nb, float eps,
                                                                   const float* __restrict__ norm_w, float* h,
                                                                   int64_t ld_h, uint8_t* __restrict__ y) {
  extern __shared__ float sm_gsum[];  // 8 group sums per block, then 1/rms
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  const int64_t row = blockIdx.x;
  const float *xr = x + row * ld_x + lane * 8, *rr = resid + row * ld_r + lane * 8, *wr = norm_w + lane * 8;
  float* hr = h + row * ld_h + lane * 8;
  uint8_t* yr = y + row * nb * Q8K_BLOCK_BYTES;
  auto add_store = [&](float (&t)[8], const float (&u)[8], int b) {
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = __fadd_rn(t[j], u[j]);
    if (kAligned) {
      *reinterpret_cast<float4*>(hr + b * QK_K) = make_float4(t[0], t[1], t[2], t[3]);
      *reinterpret_cast<float4*>(hr + b * QK_K + 4) = make_float4(t[4], t[5], t[6], t[7]);
    } else {
      store8(hr + b * QK_K, t);
    }
    const float s = group_sumsq_load8(t);
    if ((lane & 3) == 0) sm_gsum[b * 8 + (lane >> 2)] = s;
  };
  float v[kKeep][8], a[kKeep][8], g[kKeep][8];
#pragma unroll
  for (int i = 0; i < kKeep; ++i) {
    const int b = warp + i * nwarps;
    if (b < nb) {
      load8_row<kAligned>(xr + b * QK_K, v[i]);
      load8_row<kAligned>(rr + b * QK_K, a[i]);
      if (kWeight) load8_row<kAligned>(wr + b * QK_K, g[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kKeep; ++i) {
    const int b = warp + i * nwarps;
    if (b < nb) add_store(v[i], a[i], b);
  }
  for (int b = warp + kKeep * nwarps; b < nb; b += nwarps) {
    float t[8], u[8];
    load8_row<kAligned>(xr + b * QK_K, t);
    load8_row<kAligned>(rr + b * QK_K, u);
    add_store(t, u, b);
  }
  __syncthreads();
  if (warp == 0) {
    const float total = rms_fold_groups(sm_gsum, nb * 8);
    if (lane == 0) sm_gsum[nb * 8] = rms_inv_from_sum(total, nb * QK_K, eps);
  }
  __syncthreads();
  const float inv = sm_gsum[nb * 8];
#pragma unroll
  for (int i = 0; i < kKeep; ++i) {
    const int b = warp + i * nwarps;
    if (b < nb) norm_quantize_store<kWeight>(v[i], g[i], inv, yr + (size_t)b * Q8K_BLOCK_BYTES);
  }
  for (int b = warp + kKeep * nwarps; b < nb; b += nwarps) {
    float t[8], w[8];
    load8_row<kAligned>(hr + b * QK_K, t);
    if (kWeight) load8_row<kAligned>(wr + b * QK_K, w);
    norm_quantize_store<kWeight>(t, w, inv, yr + (size_t)b * Q8K_BLOCK_BYTES);
  }
}

int q8k_quantize(const float* x, int64_t ld_x, int64_t n_rows, int64_t k, void* y, cudaStream_t stream) {
  if (k <= 0 || k % QK_K != 0 || n_rows <= 0 || ld_x < k) {
    set_last_error("q8k_quantize: k must be a positive multiple of 256 (k=%lld rows=%lld ld=%lld)",
                   (long long)k, (long long)n_rows, (long long)ld_x);
    return kBadArgument;
  }
  const int nb = (int)(k / QK_K);
  const int64_t total = n_rows * nb;
  const int warps_per_cta = 4;
  int64_t ctas = (total + warps_per_cta - 1) / warps_per_cta;
  if (ctas > 148 * 32) ctas = 148 * 32;
  SMEAI_CUDA_TRY(launch(q8k_quantize_kernel, dim3((unsigned)ctas), dim3(32 * warps_per_cta), 0, stream, x, ld_x,
                        nb, total, static_cast<uint8_t*>(y)));
  return kOk;
}

int rms_q8k_quantize(const float* x, int64_t ld_x, int64_t n_rows, int64_t k, float eps, void* y,
                     cudaStream_t stream, const float* norm_w) {
  if (k <= 0 || k % QK_K != 0 || n_rows <= 0 || ld_x < k || n_rows > 0x7fffffff) {
    set_last_error("rms_q8k_quantize: k must be a positive multiple of 256");
    return kBadArgument;
  }
  const int nb = (int)(k / QK_K);
  const int threads = nb >= 16 ? 512 : (nb >= 8 ? 256 : 128);
  SMEAI_CUDA_TRY(launch(rms_q8k_quantize_kernel, dim3((unsigned)n_rows), dim3(threads), (size_t)(8 * nb + 1) * 4,
                        stream, x, ld_x, nb, eps, norm_w, static_cast<uint8_t*>(y)));
  return kOk;
}

int add_rms_q8k_quantize(const float* x, int64_t ld_x, const float* resid, int64_t ld_r, int64_t n_rows, int64_t k,
                         float eps, const float* norm_w, float* h, int64_t ld_h, void* y, cudaStream_t stream) {
  if (k <= 0 || k % QK_K != 0 || k > 65536 || n_rows <= 0 || n_rows > 0x7fffffff || ld_x < k || ld_r < k ||
      ld_h < k) {
    set_last_error("add_rms_q8k_quantize: k must be a multiple of 256 from 256 to 65536, the row strides at least k "
                   "(k=%lld rows=%lld)", (long long)k, (long long)n_rows);
    return kBadArgument;
  }
  const int nb = (int)(k / QK_K);
  const size_t smem = (size_t)(8 * nb + 1) * 4;
  uint8_t* out = static_cast<uint8_t*>(y);
  auto wide = [](const void* p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 4 == 0; };
  const bool aligned = wide(x, ld_x) && wide(resid, ld_r) && wide(h, ld_h) && wide(norm_w, 0);
  // One block a warp up to 16 warps: 2048 rows of 4096 take 27 us, with two
  // blocks a warp they took 32.5 us (84 registers a thread leave room for half
  // the rows).  Wider rows have no choice: 2048 rows of 5120, 8192, 11008 take
  // 53, 67 and 92 us (2.6 to 3.3 TB/s).
  const int warps = nb < 16 ? nb : 16;
  auto run = [&](auto kernel) {
    return launch(kernel, dim3((unsigned)n_rows), dim3(32 * warps), smem, stream, x, ld_x, resid, ld_r, nb, eps, norm_w,
                  h, ld_h, out);
  };
  cudaError_t e;
  if (nb <= warps && aligned)
    e = norm_w ? run(add_rms_q8k_quantize_kernel<1, true, true>) : run(add_rms_q8k_quantize_kernel<1, false, true>);
  else if (aligned)
    e = norm_w ? run(add_rms_q8k_quantize_kernel<2, true, true>) : run(add_rms_q8k_quantize_kernel<2, false, true>);
  else
    e = norm_w ? run(add_rms_q8k_quantize_kernel<2, true, false>) : run(add_rms_q8k_quantize_kernel<2, false, false>);
  SMEAI_CUDA_TRY(e);
  return kOk;
}

}  // namespace smeai
