// RMS norm of the residual stream, both directions.
//
//   h = bf16(x + r)      rstd = 1 / sqrt(mean h^2 + eps)      y = bf16(h * rstd * w)      MXFP8 of y in blocks of 32
//   g = dy * w           dh = rstd * (g - n * mean(g * n)) + d_hidden, n = h * rstd       dw = sum over rows of dy * n
//
// What is normalised is h as it is stored, so the backward pass sees the numbers the forward pass used. Sums and
// the statistics are fp32; y is rounded to bf16 before it is quantised, so the bytes are those of
// plb_mxfp8_quantize on y.
#include "kernels.h"
#include "mxfp8.cuh"

namespace plb {

namespace {

constexpr int kNormThreads = 256;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
// Sum over the CTA, the same bits in every thread.
__device__ __forceinline__ float block_sum(float v) {
  __shared__ float part[kNormThreads / 32];
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < kNormThreads / 32; ++i) s += part[i];
  __syncthreads();
  return s;
}
__device__ __forceinline__ float round_bf16(float v) { return __bfloat162float(__float2bfloat16_rn(v)); }

// One CTA per row, any width and alignment: the row is read twice, the second time from the cache.
__global__ void __launch_bounds__(kNormThreads)
rmsnorm_fwd_kernel(const NormFwdArgs a) {
  const int64_t row = blockIdx.x;
  const int64_t width = a.width;
  const bool live = row < a.rows;             // rows up to a multiple of 128 exist in the MXFP8 output only: zeros
  const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(a.x) + row * a.ld_x;
  const __nv_bfloat16* r = a.residual ? static_cast<const __nv_bfloat16*>(a.residual) + row * a.ld_residual : nullptr;
  const __nv_bfloat16* w = static_cast<const __nv_bfloat16*>(a.weight);
  auto hidden = [&](int64_t c) {
    const float v = __bfloat162float(x[c]);
    return r ? round_bf16(v + __bfloat162float(r[c])) : v;
  };
  float sq = 0.0f;
  if (live)
    for (int64_t c = threadIdx.x; c < width; c += kNormThreads) {
      const float h = hidden(c);
      sq = fmaf(h, h, sq);
    }
  const float rstd = rsqrtf(block_sum(sq) / static_cast<float>(width) + a.eps);
  if (live && threadIdx.x == 0) a.rstd[row] = rstd;
  for (int64_t c = threadIdx.x; c < (width + 31) / 32 * 32; c += kNormThreads) {     // whole warps: a warp is one block of 32
    const bool in = live && c < width;
    const float h = in ? hidden(c) : 0.0f;
    const float y = in ? round_bf16(h * rstd * __bfloat162float(w[c])) : 0.0f;
    if (in && r) static_cast<__nv_bfloat16*>(a.hidden)[row * width + c] = __float2bfloat16_rn(h);
    if (in && a.y) static_cast<__nv_bfloat16*>(a.y)[row * width + c] = __float2bfloat16_rn(y);
    if (a.fp8 != nullptr) {
      float amax = fabsf(y);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
      const uint32_t e = e8m0_from_amax(amax);
      static_cast<uint8_t*>(a.fp8)[row * width + c] = static_cast<uint8_t>(cvt_e4m3x4(y * e8m0_inverse(e), 0.0f, 0.0f, 0.0f));
      if ((threadIdx.x & 31) == 0) static_cast<uint8_t*>(a.sc)[scale_offset(row, c >> 5, width >> 7)] = static_cast<uint8_t>(e);
    }
  }
}

__global__ void __launch_bounds__(kNormThreads)
rmsnorm_bwd_kernel(const NormBwdArgs a) {
  const int64_t row = blockIdx.x;
  const __nv_bfloat16* dy = static_cast<const __nv_bfloat16*>(a.d_y) + row * a.ld_d_y;
  const __nv_bfloat16* h = static_cast<const __nv_bfloat16*>(a.hidden) + row * a.ld_hidden;
  const __nv_bfloat16* w = static_cast<const __nv_bfloat16*>(a.weight);
  const float rstd = a.rstd[row];
  float dot = 0.0f;
  for (int64_t c = threadIdx.x; c < a.width; c += kNormThreads)
    dot = fmaf(__bfloat162float(dy[c]) * __bfloat162float(w[c]), __bfloat162float(h[c]) * rstd, dot);
  const float mean = block_sum(dot) / static_cast<float>(a.width);
  for (int64_t c = threadIdx.x; c < a.width; c += kNormThreads) {
    const float n = __bfloat162float(h[c]) * rstd;
    float d = rstd * (__bfloat162float(dy[c]) * __bfloat162float(w[c]) - n * mean);
    if (a.d_hidden) d += __bfloat162float(static_cast<const __nv_bfloat16*>(a.d_hidden)[row * a.ld_d_hidden + c]);
    static_cast<__nv_bfloat16*>(a.d_x)[row * a.width + c] = __float2bfloat16_rn(d);
  }
}

// Column sums of dy * n over one strip of rows: partial[strip][c].
__global__ void __launch_bounds__(kNormThreads)
rmsnorm_dw_kernel(const NormBwdArgs a, int64_t rows_per_strip) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kNormThreads + threadIdx.x;
  const int64_t r0 = blockIdx.y * rows_per_strip, r1 = r0 + rows_per_strip < a.rows ? r0 + rows_per_strip : a.rows;
  if (c >= a.width) return;
  float s = 0.0f;
  for (int64_t r = r0; r < r1; ++r)
    s = fmaf(__bfloat162float(static_cast<const __nv_bfloat16*>(a.d_y)[r * a.ld_d_y + c]),
             __bfloat162float(static_cast<const __nv_bfloat16*>(a.hidden)[r * a.ld_hidden + c]) * a.rstd[r], s);
  a.workspace[blockIdx.y * a.width + c] = s;
}

// d_weight = sum over the strips, in their order.
__global__ void __launch_bounds__(kNormThreads)
rmsnorm_dw_sum_kernel(const float* __restrict__ partial, int strips, int64_t width, float* __restrict__ d_weight) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kNormThreads + threadIdx.x;
  if (c >= width) return;
  float s = 0.0f;
  for (int i = 0; i < strips; ++i) s += partial[i * width + c];
  d_weight[c] = s;
}

}  // namespace

int64_t norm_bwd_strips(int64_t rows) { return rows < kNormMaxStrips ? (rows > 0 ? rows : 1) : kNormMaxStrips; }

cudaError_t launch_rmsnorm_fwd(const NormFwdArgs& a, cudaStream_t stream) {
  const int64_t rows = a.fp8 != nullptr ? (a.rows + 127) / 128 * 128 : a.rows;
  if (rows == 0) return cudaSuccess;
  rmsnorm_fwd_kernel<<<static_cast<unsigned>(rows), kNormThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_rmsnorm_bwd(const NormBwdArgs& a, cudaStream_t stream) {
  const int64_t strips = norm_bwd_strips(a.rows), per = (a.rows + strips - 1) / strips;
  const unsigned columns = static_cast<unsigned>((a.width + kNormThreads - 1) / kNormThreads);
  if (a.rows > 0) {
    rmsnorm_bwd_kernel<<<static_cast<unsigned>(a.rows), kNormThreads, 0, stream>>>(a);
    cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return err;
  }
  rmsnorm_dw_kernel<<<dim3(columns, static_cast<unsigned>(strips)), kNormThreads, 0, stream>>>(a, per > 0 ? per : 1);
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  rmsnorm_dw_sum_kernel<<<columns, kNormThreads, 0, stream>>>(a.workspace, static_cast<int>(strips), a.width, a.d_weight);
  return cudaGetLastError();
}

}  // namespace plb
