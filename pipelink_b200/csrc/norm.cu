// RMS norm of the residual stream, both directions.
//
//   h = bf16(x + r)      rstd = 1 / sqrt(mean h^2 + eps)      y = bf16(h * rstd * w)      MXFP8 of y in blocks of 32
//   g = dy * w           dh = rstd * (g - n * mean(g * n)) + d_hidden, n = h * rstd       dw = sum over rows of dy * n
//
// What is normalised is h as it is stored, so the backward pass sees the numbers the forward pass used. Sums and
// the statistics are fp32; y is rounded to bf16 before it is quantised, so the bytes are those of
// plb_mxfp8_quantize on y.
//
// Both directions are bound by memory: a row is read once into registers, reduced by the threads that hold it
// and written from there. VEC is the elements a thread moves at a time: 8 (16 bytes) where width, strides and
// addresses allow, else 1. Rows too wide for registers (16384 elements, 8192 unaligned) are read twice.
#include <type_traits>

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
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&t);
}

// VEC bf16 numbers as they travel.
template <int VEC>
struct Chunk;
template <>
struct Chunk<8> {
  uint4 raw;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { raw = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = raw; }
  __device__ __forceinline__ void zero() { raw = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ float get(int i) const {
    const uint32_t w = i < 2 ? raw.x : i < 4 ? raw.y : i < 6 ? raw.z : raw.w;
    return i & 1 ? bf16_hi(w) : bf16_lo(w);
  }
  __device__ __forceinline__ Pair pair(int i) const {      // numbers 2 i and 2 i + 1
    const uint32_t w = i == 0 ? raw.x : i == 1 ? raw.y : i == 2 ? raw.z : raw.w;
    return make_pair(bf16_lo(w), bf16_hi(w));
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    raw = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
  }
};
template <>
struct Chunk<1> {
  __nv_bfloat16 raw;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { raw = *p; }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const { *p = raw; }
  __device__ __forceinline__ void zero() { raw = __float2bfloat16_rn(0.0f); }
  __device__ __forceinline__ float get(int) const { return __bfloat162float(raw); }
  __device__ __forceinline__ void set(const float (&f)[1]) { raw = __float2bfloat16_rn(f[0]); }
};

// Two by two, the numbers of a thread's chunks: of one chunk, or of two chunks of one.
template <int NV>
__device__ __forceinline__ Pair pair_of(const Chunk<8> (&c)[NV], int i) { return c[i >> 2].pair(i & 3); }
template <int NV>
__device__ __forceinline__ Pair pair_of(const Chunk<1> (&c)[NV], int i) { return make_pair(c[2 * i].get(0), c[2 * i + 1].get(0)); }

// The SIZE threads of a row: a warp (eight rows a CTA, no barriers) or a whole CTA. A compile-time size: with the
// exact number of warps a width needs, known at run time only, 16384 x 4096 takes 94 us instead of 91.
template <int SIZE>
struct RowTeam {
  static constexpr int kThreads = SIZE == 32 ? kNormThreads : SIZE, kRows = kThreads / SIZE;
  __device__ static __forceinline__ int thread() { return threadIdx.x % SIZE; }
  __device__ static __forceinline__ int row() { return threadIdx.x / SIZE; }
  // Sum over a row's threads, the same bits in each; `round` alternates the buffers of consecutive sums.
  __device__ static __forceinline__ float sum(float v, int round) {
    v = warp_sum(v);
    if constexpr (SIZE > 32) {
      __shared__ float part[2][32];
      const int lane = threadIdx.x & 31;
      if (lane == 0) part[round & 1][threadIdx.x >> 5] = v;
      __syncthreads();
      v = warp_sum(lane < SIZE / 32 ? part[round & 1][lane] : 0.0f);
    }
    return v;
  }
};

// NV chunks of VEC elements a thread. Threads per SM by what a thread holds, with the registers that suffice but for a
// few words (8 bytes a thread of 32 elements in a warp's row, 6 to 10 of single ones): 2048 for 8 elements (16384 x 2048: 44
// us with one register more, 41 so), 1280 for 16 (16384 x 4096 with both outputs: 100 us with 1024, 91 so), 1024 for 32.
template <int VEC, int SIZE, int NV>
__global__ void __launch_bounds__(RowTeam<SIZE>::kThreads, (NV * VEC <= 8 ? 2048 : NV * VEC <= 16 ? 1280 : 1024) / RowTeam<SIZE>::kThreads)
rmsnorm_fwd_rows(const __grid_constant__ NormFwdArgs a) {
  using Team = RowTeam<SIZE>;
  const int t = Team::thread();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * Team::kRows + Team::row();
  const bool live = row < a.rows;
  const int width = static_cast<int>(a.width);
  const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(a.x) + row * a.ld_x;
  const __nv_bfloat16* residual = static_cast<const __nv_bfloat16*>(a.residual) + row * a.ld_residual;
  const __nv_bfloat16* weight = static_cast<const __nv_bfloat16*>(a.weight);
  __nv_bfloat16* hidden = static_cast<__nv_bfloat16*>(a.hidden) + row * width;
  __nv_bfloat16* y_out = static_cast<__nv_bfloat16*>(a.y) + row * width;
  Chunk<VEC> h[NV], w[NV];
  float sq = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * SIZE) * VEC;
    h[i].zero();
    w[i].zero();
    if (c < width) {
      if (live) h[i].load(x + c);
      w[i].load(weight + c);
    }
  }
  if (a.residual != nullptr && live) {
    Chunk<VEC> r[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * SIZE) * VEC;
      if (c < width) r[i].load(residual + c);
      else r[i].zero();
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * SIZE) * VEC;
      float f[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = h[i].get(e) + r[i].get(e);
      h[i].set(f);
      if (c < width) h[i].store(hidden + c);
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) sq = fmaf(h[i].get(e), h[i].get(e), sq);
  const float rstd = rsqrtf(Team::sum(sq, 0) / static_cast<float>(width) + a.eps);
  if (live && t == 0) a.rstd[row] = rstd;
  const bool quantise = a.fp8 != nullptr;
  if (!live && !(quantise && row < (a.rows + 127) / 128 * 128)) return;     // MXFP8 rows up to a multiple of 128 are zeros
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * SIZE) * VEC;
    const bool in = c < width;
    if (i * SIZE * VEC >= width) break;            // the same for every thread of the row
    float f[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = h[i].get(e) * rstd * w[i].get(e);
    Chunk<VEC> y;
    y.set(f);
    if (live && in && a.y != nullptr) y.store(y_out + c);
    if (!quantise) continue;
    // 32 / VEC adjacent lanes hold a block; width is a multiple of 128, so a block is wholly inside the row or outside
    float amax = 0.0f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      f[e] = live ? y.get(e) : 0.0f;
      amax = fmaxf(amax, fabsf(f[e]));
    }
#pragma unroll
    for (int o = 1; o < 32 / VEC; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
    const uint32_t s = e8m0_from_amax(amax);
    const float inv = e8m0_inverse(s);
    uint8_t* fp8 = static_cast<uint8_t*>(a.fp8) + row * width + c;
    uint8_t* sc = static_cast<uint8_t*>(a.sc) + scale_offset(row, c >> 5, width >> 7);
    if constexpr (VEC == 8) {
      uint32_t word = s;                          // the four scales of 128 columns are one word
      word |= __shfl_down_sync(0xFFFFFFFFu, s, 4) << 8;
      word |= __shfl_down_sync(0xFFFFFFFFu, s, 8) << 16;
      word |= __shfl_down_sync(0xFFFFFFFFu, s, 12) << 24;
      if (in) {
        *reinterpret_cast<uint2*>(fp8) = make_uint2(cvt_e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                                                    cvt_e4m3x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
        if ((t & 15) == 0) *reinterpret_cast<uint32_t*>(sc) = word;
      }
    } else {
      if (in) {
        *fp8 = static_cast<uint8_t>(cvt_e4m3x4(f[0] * inv, 0.0f, 0.0f, 0.0f));
        if ((t & 31) == 0) *sc = static_cast<uint8_t>(s);
      }
    }
  }
}

// The gradient of x, and this CTA's share of the weight's: a thread keeps the sums of its columns over the rows
// the CTA walks, so dy and h are read once for both.
//
// CTAs per SM: 1024 threads where a thread holds 8 elements, 512 (128 registers) where it holds more or loads ahead; 768
// threads of 16 elements spill (16384 x 4096: 114 us, with 512 threads 104). Rows of 8200 to 16384 (32 elements and their sums a
// thread) spill 280 bytes a thread, rows of 520 to 1024 in a warp 108 (4096 x 16384: 125 us, 0.66 of the copy rate).
template <int VEC, int SIZE, int NV>
constexpr int kBwdResident = SIZE == 1024 ? 1 : (SIZE == 32 || NV * VEC > 8 ? 512 : 1024) / RowTeam<SIZE>::kThreads;
template <int VEC, int SIZE, int NV>
__global__ void __launch_bounds__(RowTeam<SIZE>::kThreads, kBwdResident<VEC, SIZE, NV>)
rmsnorm_bwd_rows(const __grid_constant__ NormBwdArgs a) {
  using Team = RowTeam<SIZE>;
  const int t = Team::thread(), team = Team::row();
  const int width = static_cast<int>(a.width);
  const int64_t sets = (a.rows + Team::kRows - 1) / Team::kRows;
  const float inv_width = 1.0f / static_cast<float>(width);
  constexpr int kPairs = NV * VEC / 2;
  Pair dw[kPairs];
#pragma unroll
  for (int i = 0; i < kPairs; ++i) dw[i] = make_pair(0.0f, 0.0f);
  // the weight's columns of this thread: kept in registers, or read again (from L1) where those are short
  constexpr bool kKeepWeight = NV * VEC < 32;
  Chunk<VEC> w[NV];
  auto load_weight = [&](int i) {
    const int c = (t + i * SIZE) * VEC;
    w[i].zero();
    if (c < width) w[i].load(static_cast<const __nv_bfloat16*>(a.weight) + c);
  };
  if (kKeepWeight)
#pragma unroll
    for (int i = 0; i < NV; ++i) load_weight(i);
  struct Row { Chunk<VEC> g[NV], h[NV], r[NV]; float rstd; };
  auto fetch = [&](Row& v, int64_t set) {
    const int64_t row = set * Team::kRows + team;
    const bool live = row < a.rows;
    const __nv_bfloat16* g = static_cast<const __nv_bfloat16*>(a.d_y) + row * a.ld_d_y;
    const __nv_bfloat16* h = static_cast<const __nv_bfloat16*>(a.hidden) + row * a.ld_hidden;
    const __nv_bfloat16* r = static_cast<const __nv_bfloat16*>(a.d_hidden) + row * a.ld_d_hidden;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * SIZE) * VEC;
      v.g[i].zero();
      v.h[i].zero();
      v.r[i].zero();
      if (live && c < width) {
        v.g[i].load(g + c);
        v.h[i].load(h + c);
        if (a.d_hidden != nullptr) v.r[i].load(r + c);
      }
    }
    v.rstd = live ? a.rstd[row] : 0.0f;
  };
  // the next row's loads are in flight while this one is summed, where registers allow (16384 x 4096: 102 us without,
  // 86 with)
  constexpr bool kAhead = SIZE <= 512 && NV * VEC <= (VEC == 8 ? 16 : 8);
  Row next;
  if (kAhead) fetch(next, blockIdx.x);
  int round = 0;
  for (int64_t set = blockIdx.x; set < sets; set += gridDim.x, ++round) {
    const int64_t row = set * Team::kRows + team;
    const bool live = row < a.rows;
    Row now;
    if (kAhead) {
      now = next;
      if (set + gridDim.x < sets) fetch(next, set + gridDim.x);
    } else {
      fetch(now, set);
    }
    const float rstd = now.rstd;
    // n and g of the row in fp32, packed: unpacking the operands once, two numbers to an instruction
    Pair n[kPairs], gw[kPairs];
    Pair dot = make_pair(0.0f, 0.0f);
    const Pair rstd2 = make_pair(rstd, rstd);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      if (!kKeepWeight && 2 * i % VEC == 0) load_weight(2 * i / VEC);
      const Pair g = pair_of(now.g, i);
      n[i] = mul2(pair_of(now.h, i), rstd2);
      dw[i] = fma2(g, n[i], dw[i]);
      gw[i] = mul2(g, pair_of(w, i));
      dot = fma2(gw[i], n[i], dot);
    }
    float dot_lo, dot_hi;
    split(dot, dot_lo, dot_hi);
    const float mean = Team::sum(dot_lo + dot_hi, round) * inv_width;
    if (!live) continue;
    __nv_bfloat16* d_x = static_cast<__nv_bfloat16*>(a.d_x) + row * width;
    const Pair minus_mean = make_pair(-mean, -mean);
    float d[NV][VEC];
#pragma unroll
    for (int i = 0; i < kPairs; ++i)
      split(fma2(fma2(n[i], minus_mean, gw[i]), rstd2, pair_of(now.r, i)), d[2 * i / VEC][2 * i % VEC], d[(2 * i + 1) / VEC][(2 * i + 1) % VEC]);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * SIZE) * VEC;
      if (c >= width) continue;
      Chunk<VEC> out;
      out.set(d[i]);
      out.store(d_x + c);
    }
  }
  float sums[NV * VEC];
#pragma unroll
  for (int i = 0; i < kPairs; ++i) split(dw[i], sums[2 * i], sums[2 * i + 1]);
  if constexpr (Team::kRows > 1) {                 // the CTA's rows of each column, in their order
    __shared__ float part[kNormThreads][NV * VEC];
#pragma unroll
    for (int i = 0; i < NV * VEC; ++i) part[threadIdx.x][i] = sums[i];
    __syncthreads();
    if (team != 0) return;
#pragma unroll
    for (int i = 0; i < NV * VEC; ++i)
      for (int k = 1; k < Team::kRows; ++k) sums[i] += part[k * 32 + t][i];
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * SIZE) * VEC;
    if (c >= width) continue;
    float* dst = a.workspace + static_cast<int64_t>(blockIdx.x) * width + c;
    if constexpr (VEC == 8) {
      reinterpret_cast<float4*>(dst)[0] = make_float4(sums[i * 8], sums[i * 8 + 1], sums[i * 8 + 2], sums[i * 8 + 3]);
      reinterpret_cast<float4*>(dst)[1] = make_float4(sums[i * 8 + 4], sums[i * 8 + 5], sums[i * 8 + 6], sums[i * 8 + 7]);
    } else {
      *dst = sums[i];
    }
  }
}

// ---- any width: one CTA per row, the row read a second time from the cache
__global__ void __launch_bounds__(kNormThreads)
rmsnorm_fwd_wide(const NormFwdArgs a) {
  const int64_t row = blockIdx.x;
  const int64_t width = a.width;
  const bool live = row < a.rows;
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
rmsnorm_bwd_wide(const NormBwdArgs a) {
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
rmsnorm_dw_wide(const NormBwdArgs a, int64_t rows_per_strip) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kNormThreads + threadIdx.x;
  const int64_t r0 = blockIdx.y * rows_per_strip, r1 = r0 + rows_per_strip < a.rows ? r0 + rows_per_strip : a.rows;
  if (c >= a.width) return;
  float s = 0.0f;
  for (int64_t r = r0; r < r1; ++r)
    s = fmaf(__bfloat162float(static_cast<const __nv_bfloat16*>(a.d_y)[r * a.ld_d_y + c]),
             __bfloat162float(static_cast<const __nv_bfloat16*>(a.hidden)[r * a.ld_hidden + c]) * a.rstd[r], s);
  a.workspace[blockIdx.y * a.width + c] = s;
}

// d_weight = sum over the strips: 32 columns a CTA, a strip a warp, the warps' sums joined in their order. 32 warps
// so that a few loads in flight per thread cover all strips (296 strips of 4096: 3 us; 8 warps took 10).
constexpr int kSumThreads = 1024;
__global__ void __launch_bounds__(kSumThreads)
rmsnorm_dw_sum(const float* __restrict__ partial, int strips, int64_t width, float* __restrict__ d_weight) {
  __shared__ float part[kSumThreads / 32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float s = 0.0f;
  if (c < width)
#pragma unroll 8
    for (int i = warp; i < strips; i += kSumThreads / 32) s += partial[i * width + c];
  part[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || c >= width) return;
#pragma unroll
  for (int i = 1; i < kSumThreads / 32; ++i) s += part[i][lane];
  d_weight[c] = s;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int V, int S, int N>
struct RowShape {
  static constexpr int kVec = V, kSize = S, kNv = N;
};
// Calls f with the row shape for a width, false where rows do not fit in registers. Rows that a warp can hold get a
// warp, wider ones a CTA of 256 threads as long as those can hold them, and few rows as many threads as they fill,
// since the time of one row is what counts there (1 x 4096: 2.4 us with 512 threads).
template <bool kBack, class F>
bool by_row_shape(bool vec, int64_t width, bool few, F&& f) {
  if (vec) {
    const int64_t n = width / 8;
    if (n <= 32) f(RowShape<8, 32, 1>{});
    else if (n <= 64) f(RowShape<8, 32, 2>{});
    else if (n <= 128) f(RowShape<8, 32, 4>{});
    else if (n <= 256) f(RowShape<8, 256, 1>{});
    else if (few && n <= 512) f(RowShape<8, 512, 1>{});
    else if (few && n <= 1024) f(RowShape<8, 1024, 1>{});
    else if (n <= 512) f(RowShape<8, 256, 2>{});
    else if (n <= 1024) {
      if constexpr (kBack) f(RowShape<8, 512, 2>{});          // 32 elements a thread and their sums spill (8192 x 8192: 119 us, so 88)
      else f(RowShape<8, 256, 4>{});
    }
    else if (n <= 2048) f(RowShape<8, 512, 4>{});
    else return false;
  } else {
    if (width <= 128) f(RowShape<1, 32, 4>{});
    else if (width <= 1024) f(RowShape<1, 256, 4>{});
    else if (width <= 4096) f(RowShape<1, 256, 16>{});
    else if (width <= 8192) f(RowShape<1, 1024, 8>{});
    else return false;
  }
  return true;
}

}  // namespace

int64_t norm_bwd_strips(int64_t rows) { return rows < kNormMaxStrips ? (rows > 0 ? rows : 1) : kNormMaxStrips; }

cudaError_t launch_rmsnorm_fwd(const NormFwdArgs& a, cudaStream_t stream) {
  const int64_t rows = a.fp8 != nullptr ? (a.rows + 127) / 128 * 128 : a.rows;
  if (rows == 0) return cudaSuccess;
  const bool vec = a.width % 8 == 0 && a.ld_x % 8 == 0 && a.ld_residual % 8 == 0 && aligned16(a.x) && aligned16(a.residual) &&
                   aligned16(a.weight) && aligned16(a.hidden) && aligned16(a.y);
  const bool done = by_row_shape<false>(vec, a.width, a.rows <= a.num_sms, [&](auto s) {
    using S = decltype(s);
    using Team = RowTeam<S::kSize>;
    rmsnorm_fwd_rows<S::kVec, S::kSize, S::kNv><<<static_cast<unsigned>((rows + Team::kRows - 1) / Team::kRows), Team::kThreads, 0, stream>>>(a);
  });
  if (!done) rmsnorm_fwd_wide<<<static_cast<unsigned>(rows), kNormThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_rmsnorm_bwd(const NormBwdArgs& a, cudaStream_t stream) {
  const bool vec = a.width % 8 == 0 && a.ld_d_y % 8 == 0 && a.ld_hidden % 8 == 0 && a.ld_d_hidden % 8 == 0 && aligned16(a.d_y) &&
                   aligned16(a.hidden) && aligned16(a.d_hidden) && aligned16(a.weight) && aligned16(a.d_x);
  int64_t strips = norm_bwd_strips(a.rows);
  const bool done = by_row_shape<true>(vec, a.width, a.rows <= a.num_sms, [&](auto s) {
    using S = decltype(s);
    using Team = RowTeam<S::kSize>;
    const int64_t sets = (a.rows + Team::kRows - 1) / Team::kRows;
    const int64_t most = static_cast<int64_t>(a.num_sms) * kBwdResident<S::kVec, S::kSize, S::kNv>;
    strips = sets < 1 ? 1 : sets;
    if (strips > most) strips = most;
    if (strips > kNormMaxStrips) strips = kNormMaxStrips;
    rmsnorm_bwd_rows<S::kVec, S::kSize, S::kNv><<<static_cast<unsigned>(strips), Team::kThreads, 0, stream>>>(a);
  });
  if (!done) {
    const int64_t per = (a.rows + strips - 1) / strips;
    if (a.rows > 0) rmsnorm_bwd_wide<<<static_cast<unsigned>(a.rows), kNormThreads, 0, stream>>>(a);
    cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return err;
    rmsnorm_dw_wide<<<dim3(static_cast<unsigned>((a.width + kNormThreads - 1) / kNormThreads), static_cast<unsigned>(strips)), kNormThreads, 0,
                      stream>>>(a, per > 0 ? per : 1);
  }
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  rmsnorm_dw_sum<<<static_cast<unsigned>((a.width + 31) / 32), kSumThreads, 0, stream>>>(a.workspace, static_cast<int>(strips), a.width, a.d_weight);
  return cudaGetLastError();
}

}  // namespace plb
