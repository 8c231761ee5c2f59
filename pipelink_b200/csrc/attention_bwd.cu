// Gradients of causal attention (bf16, head_dim 128) from the saved output and log-sum-exp, on tcgen05.
//
//   x = scale * q.k        y = x, or cap * tanh(x / cap)        P = exp(y - lse) on visible keys, 0 elsewhere
//   delta = sum_d dO * O   dP = dO V^T                          dX = P * (dP - delta) [* (1 - tanh^2)]
//   dV = P^T dO            dQ = scale * dX K                    dK = scale * dX^T Q
//
// The probabilities are recomputed tile by tile, so nothing of size seq^2 exists in memory. Two kernels:
//   dq    one CTA per 128-query tile and query head, keys streamed past it (S, dP, then dQ += dX K); it also
//         writes delta and the base-2 log-sum-exp the second kernel reads
//   dkdv  one CTA per 128-key tile and KV head, the queries of every head of the group streamed past it
//         (S^T, dP^T, then dV += P^T dO and dK += dX^T Q)
// Computing S and dP in both costs seven tile products where one kernel would need five, and buys that every
// sum has one owner: no atomics, no fp32 gradient buffer in memory and its conversion pass, the same bits in
// every run, and gradients of shared KV heads summed in fp32 in tensor memory.
//
// Roundings: P and dX go to bf16 (the tensor cores' operand type, half a step 2^-9 of the value); every sum,
// the exponent, delta and the accumulators are fp32; the gradients are rounded once when they are stored.
//
// Tensor maps are 3-D (column, position, batch): rows past a sequence's end read as zeros and never as the
// next sequence's, and their probabilities are forced to 0 (log-sum-exp +inf), so any length works.
#include <math.h>

#include <cstddef>

#include "attention_bwd.h"
#include "attention_roles.cuh"

namespace plb {

using namespace attn;

namespace {

constexpr int kBwdThreads = 384;      // warp 0 TMA, warp 1 MMA, warps 4-11 compute
constexpr int kCompute = 256;
constexpr uint32_t kFullMask = 0xFFFFFFFFu;
constexpr float kLog2e = 1.4426950408889634f;

// ---- shared-memory maps (offsets from a 1024-byte aligned base)
constexpr int kDqK = 2 * kTileBytes, kDqKStages = 3;                  // after Q and dO
constexpr int kDqV = kDqK + kDqKStages * kTileBytes, kDqVStages = 2;
constexpr int kDqRed = kDqV + kDqVStages * kTileBytes;                // [2][2][128] floats
constexpr int kDqBar = kDqRed + 2048;
constexpr int kDqSmem = kDqBar + 256;

constexpr int kKvQ = 2 * kTileBytes, kKvQStages = 3;                  // after K and V
constexpr int kKvDo = kKvQ + kKvQStages * kTileBytes, kKvDoStages = 2;
constexpr int kKvStat = kKvDo + kKvDoStages * kTileBytes, kKvStatStages = 2;   // 128 lse2, 128 delta
constexpr int kKvBar = kKvStat + kKvStatStages * 1024;
constexpr int kKvSmem = kKvBar + 256;
static_assert(kDqSmem <= 232448 && kKvSmem <= 232448, "227 KB of shared memory per CTA");

struct DqBars {
  uint64_t q_full, q_empty, k_full[kDqKStages], k_empty[kDqKStages], v_full[kDqVStages], v_empty[kDqVStages];
  uint64_t s_full[2], dp_full, ds_full, dq_full, dq_free, red, drain;
  uint32_t tmem_base, pad;
};
struct KvBars {
  uint64_t kv_full, kv_empty, q_full[kKvQStages], q_empty[kKvQStages], do_full[kKvDoStages], do_empty[kKvDoStages];
  uint64_t stat_full[kKvStatStages], stat_empty[kKvStatStages];
  uint64_t s_full, p_full, dp_full, ds_full, acc_full, acc_free, drain;
  uint32_t tmem_base, pad;
};
static_assert(sizeof(DqBars) <= 256 && sizeof(KvBars) <= 256, "barrier block");

// Work lists are sorted heavy first; walking them forth and back evens out what a CTA gets.
__device__ __forceinline__ int snake(int wave) {
  return wave * gridDim.x + ((wave & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

struct DqItem { int b, h, q0, first, blocks; };
__device__ __forceinline__ DqItem dq_item(const AttnBwdParams& p, int w) {
  const int bh = p.batch * p.q_heads;
  DqItem t;
  const int back = w / bh, r = w - back * bh;
  const int qb = p.tiles - 1 - back;
  t.b = r / p.q_heads;
  t.h = r - t.b * p.q_heads;
  t.q0 = qb * kBlk;
  t.first = p.window > 0 ? max(0, (t.q0 - p.window + 1) / kBlk) : 0;
  t.blocks = qb + 1 - t.first;
  return t;
}
struct KvItem { int b, h, k0, first, tiles, n; };
__device__ __forceinline__ KvItem kv_item(const AttnBwdParams& p, int w) {
  const int bh = p.batch * p.kv_heads;
  KvItem t;
  const int kb = w / bh, r = w - kb * bh;
  t.b = r / p.kv_heads;
  t.h = r - t.b * p.kv_heads;
  t.k0 = kb * kBlk;
  t.first = kb;
  int last = p.tiles - 1;
  if (p.window > 0) last = min(static_cast<int64_t>(last), (static_cast<int64_t>(t.k0) + kBlk - 1 + p.window - 1) / kBlk);
  t.tiles = last + 1 - kb;
  t.n = t.tiles * p.group;
  return t;
}

// A role's wait: the warp's lanes agree on the outcome.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, Status* st, int code, int what) {
  return __all_sync(kFullMask, mbar_wait(bar, parity, st, code, what)) != 0;
}
__device__ __forceinline__ void warp_commit(uint32_t bar) {
  if (elect_one_sync()) tc_commit(bar);
  __syncwarp();
}
// D = A B^T over 128 columns of the contraction, both operands K-major tiles in shared memory, then the barrier.
__device__ __forceinline__ void mma_tiles(uint32_t d, uint32_t a, uint32_t b, uint32_t bar) {
  const uint64_t ad = smem_desc(a, kDescSw128KMajor), bd = smem_desc(b, kDescSw128KMajor);
  if (elect_one_sync()) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t off = ((k >> 2) * kAtomBytes + (k & 3) * 32) >> 4;
      tc_mma_f16(d, ad + off, bd + off, kIdescQK, k != 0 ? 1u : 0u);
    }
    tc_commit(bar);
  }
  __syncwarp();
}
// D += A B with A bf16 in tensor memory (its two 64-column halves at a and a + 64) and B's rows along the contraction.
__device__ __forceinline__ void mma_from_tmem(uint32_t d, uint32_t a, uint32_t b, bool accumulate, uint32_t bar) {
  const uint64_t bd = smem_desc(b, kDescVMn);
  if (elect_one_sync()) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      tc_mma_f16_ts(d, a + (k >> 2) * 64 + (k & 3) * 8, bd + ((k * 2048) >> 4), kIdescPV, k != 0 || accumulate ? 1u : 0u);
    tc_commit(bar);
  }
  __syncwarp();
}
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint32_t bar, int col, int row, int batch) {
  tma_load_3d(dst, map, bar, col, row, batch);
  tma_load_3d(dst + kAtomBytes, map, bar, col + 64, row, batch);
}
__device__ __forceinline__ void drain_mma(uint32_t bar) {
  if ((threadIdx.x & 31) == 0) {
    tc_commit(bar);
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, 0)) {
      if (clock64() - t0 > 20000000LL) break;
    }
  }
  __syncwarp();
}
__device__ __forceinline__ void linger() {   // copies in flight land before the CTA's shared memory is given up
  const long long t0 = clock64();
  while (clock64() - t0 < 200000LL) {
  }
}

// Base-2 exponent of a raw score and, with a cap, the cap's slope. tanh from exp2 and a division rather than
// tanh.approx: the slope and the exponent both see its error, scaled by the cap.
template <bool kCap>
__device__ __forceinline__ float probability(float s, float lse2, const AttnBwdParams& p, float& slope) {
  if (kCap) {
    const float t = 1.0f - __fdividef(2.0f, 1.0f + ex2_approx(fminf(s * p.cap_in, 60.0f)));   // tanh(x) = 1 - 2 / (1 + 2^(2 x log2 e))
    slope = fmaf(-t, t, 1.0f);
    return ex2_approx(fmaf(t, p.cap_out, -lse2));
  }
  return ex2_approx(fmaf(s, p.scale_log2, -lse2));
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&t);
}
// 64 fp32 accumulator columns of this lane, scaled, as bf16 to 128 contiguous bytes.
__device__ __forceinline__ void store_half_row(const uint32_t (&a)[32], const uint32_t (&b)[32], float scale, __nv_bfloat16* dst) {
  uint4* out = reinterpret_cast<uint4*>(dst);
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = (g & 3) * 8 + e * 2;
      w[e] = g < 4 ? pack_bf16(__uint_as_float(a[i]) * scale, __uint_as_float(a[i + 1]) * scale)
                   : pack_bf16(__uint_as_float(b[i]) * scale, __uint_as_float(b[i + 1]) * scale);
    }
    out[g] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

#define PLB_BAR(type, base, name) (sb + (base) + offsetof(type, name))

// ------------------------------------------------------------------------------------------ dQ
// TMEM columns: dQ 0-127, S 128-255 and 256-383 (two buffers), dP 384-511. dX overwrites the S buffer it came
// from, as the A operand of dQ += dX K. Issue order: S(j+1), dQ(j), dP(j+1); S(j+1) runs while the compute warps
// finish dX(j), dQ(j) and dP(j+1) while they exponentiate S(j+1).
template <bool kCap>
__global__ void __launch_bounds__(kBwdThreads, 1)
attention_bwd_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                        const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        const AttnBwdParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sb = smem_u32(smem);
  if ((sb & 1023u) != 0) {          // the swizzle pattern repeats every 1024 bytes
    if (threadIdx.x == 0) report_failure(p.status, ST_BAD_ARGUMENT, 499, sb, 1024);
    return;
  }
  DqBars* bars = reinterpret_cast<DqBars*>(smem + kDqBar);
  const int warp = __shfl_sync(kFullMask, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
#define BAR(name) PLB_BAR(DqBars, kDqBar, name)
  if (threadIdx.x == 0) {
    mbar_init(BAR(q_full), 1);
    mbar_init(BAR(q_empty), 1);
    for (int s = 0; s < kDqKStages; ++s) { mbar_init(BAR(k_full) + 8 * s, 1); mbar_init(BAR(k_empty) + 8 * s, 1); }
    for (int s = 0; s < kDqVStages; ++s) { mbar_init(BAR(v_full) + 8 * s, 1); mbar_init(BAR(v_empty) + 8 * s, 1); }
    mbar_init(BAR(s_full), 1);
    mbar_init(BAR(s_full) + 8, 1);
    mbar_init(BAR(dp_full), 1);
    mbar_init(BAR(ds_full), kCompute);
    mbar_init(BAR(dq_full), 1);
    mbar_init(BAR(dq_free), kCompute);
    mbar_init(BAR(red), kCompute);
    mbar_init(BAR(drain), 1);
    fence_mbar_init();
    prefetch_tensormap(&map_q);
    prefetch_tensormap(&map_do);
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&bars->tmem_base), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(kFullMask, *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base), 0);
  const uint32_t t_dq = tmem, t_s = tmem + 128, t_dp = tmem + 384;
  const int items = p.tiles * p.batch * p.q_heads;

  if (warp == 0) {
    uint32_t it = 0, kv = 0;
    bool ok = true;
    for (int wave = 0; ok && wave * static_cast<int>(gridDim.x) < items; ++wave) {
      const int w = snake(wave);
      if (w >= items) continue;
      const DqItem t = dq_item(p, w);
      const int col = t.h * kD, kv_col = t.h / p.group * kD;
      if (!warp_wait(BAR(q_empty), (it & 1u) ^ 1u, p.status, ST_TIMEOUT_EMPTY, 400)) { ok = false; break; }
      if (elect_one_sync()) {
        mbar_arrive_expect_tx(BAR(q_full), 2 * kTileBytes);
        load_tile(sb, &map_q, BAR(q_full), col, t.q0, t.b);
        load_tile(sb + kTileBytes, &map_do, BAR(q_full), col, t.q0, t.b);
      }
      __syncwarp();
      ++it;
      for (int j = 0; j < t.blocks; ++j, ++kv) {
        const int row = (t.first + j) * kBlk;
        const uint32_t ks = kv % kDqKStages, vs = kv % kDqVStages;
        if (!warp_wait(BAR(k_empty) + 8 * ks, ((kv / kDqKStages) & 1u) ^ 1u, p.status, ST_TIMEOUT_EMPTY, 401)) { ok = false; break; }
        if (elect_one_sync()) {
          mbar_arrive_expect_tx(BAR(k_full) + 8 * ks, kTileBytes);
          load_tile(sb + kDqK + ks * kTileBytes, &map_k, BAR(k_full) + 8 * ks, kv_col, row, t.b);
        }
        __syncwarp();
        if (!warp_wait(BAR(v_empty) + 8 * vs, ((kv / kDqVStages) & 1u) ^ 1u, p.status, ST_TIMEOUT_EMPTY, 402)) { ok = false; break; }
        if (elect_one_sync()) {
          mbar_arrive_expect_tx(BAR(v_full) + 8 * vs, kTileBytes);
          load_tile(sb + kDqV + vs * kTileBytes, &map_v, BAR(v_full) + 8 * vs, kv_col, row, t.b);
        }
        __syncwarp();
      }
    }
    if (!ok) linger();
  } else if (warp == 1) {
    uint32_t it = 0, blk = 0;   // items, blocks since the start
    bool ok = true;
    auto issue_s = [&](uint32_t n) {   // block n of the CTA's stream
      const uint32_t ks = n % kDqKStages;
      if (!warp_wait(BAR(k_full) + 8 * ks, (n / kDqKStages) & 1u, p.status, ST_TIMEOUT_FULL, 410)) return false;
      tc_fence_after();
      mma_tiles(t_s + (n & 1u) * 128, sb, sb + kDqK + ks * kTileBytes, BAR(s_full) + 8 * (n & 1u));
      return true;
    };
    auto issue_dp = [&](uint32_t n) {
      const uint32_t vs = n % kDqVStages;
      if (!warp_wait(BAR(v_full) + 8 * vs, (n / kDqVStages) & 1u, p.status, ST_TIMEOUT_FULL, 411)) return false;
      tc_fence_after();
      mma_tiles(t_dp, sb + kTileBytes, sb + kDqV + vs * kTileBytes, BAR(dp_full));
      warp_commit(BAR(v_empty) + 8 * vs);
      return true;
    };
    for (int wave = 0; ok && wave * static_cast<int>(gridDim.x) < items; ++wave) {
      const int w = snake(wave);
      if (w >= items) continue;
      const int n = __shfl_sync(kFullMask, dq_item(p, w).blocks, 0);
      if (!warp_wait(BAR(q_full), it & 1u, p.status, ST_TIMEOUT_FULL, 412)) { ok = false; break; }
      tc_fence_after();
      if (!issue_s(blk) || !issue_dp(blk)) { ok = false; break; }
      for (int j = 0; j < n && ok; ++j, ++blk) {
        const bool more = j + 1 < n;
        if (more && !issue_s(blk + 1)) { ok = false; break; }
        if (!warp_wait(BAR(ds_full), blk & 1u, p.status, ST_TIMEOUT_FULL, 413)) { ok = false; break; }
        if (j == 0 && !warp_wait(BAR(dq_free), (it & 1u) ^ 1u, p.status, ST_TIMEOUT_TMEM_EMPTY, 414)) { ok = false; break; }
        tc_fence_after();
        const uint32_t ks = blk % kDqKStages;
        mma_from_tmem(t_dq, t_s + (blk & 1u) * 128, sb + kDqK + ks * kTileBytes, j != 0, BAR(k_empty) + 8 * ks);
        if (more && !issue_dp(blk + 1)) { ok = false; break; }
      }
      if (!ok) break;
      warp_commit(BAR(q_empty));
      warp_commit(BAR(dq_full));
      ++it;
    }
    if (!ok) drain_mma(BAR(drain));
  } else if (warp >= 4) {
    const int half = (warp - 4) >> 2, quad = warp & 3, row = quad * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quad * 32) << 16;
    float* red = reinterpret_cast<float*>(smem + kDqRed);
    uint32_t it = 0, blk = 0;
    bool ok = true;
    for (int wave = 0; ok && wave * static_cast<int>(gridDim.x) < items; ++wave) {
      const int w = snake(wave);
      if (w >= items) continue;
      const DqItem t = dq_item(p, w);
      const int q_pos = t.q0 + row;
      const bool live = q_pos < p.seq;
      const int64_t bh = static_cast<int64_t>(t.b) * p.q_heads + t.h;
      const size_t at = ((static_cast<size_t>(t.b) * p.seq + (live ? q_pos : 0)) * p.q_heads + t.h) * kD + half * 64;
      // delta: each thread half of its row, the two halves exchanged through shared memory
      float part = 0.0f;
      if (live) {
        const uint4* o = reinterpret_cast<const uint4*>(p.out + at);
        const uint4* g = reinterpret_cast<const uint4*>(p.d_out + at);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint4 a = o[i], c = g[i];
          part = fmaf(bf16_lo(a.x), bf16_lo(c.x), part); part = fmaf(bf16_hi(a.x), bf16_hi(c.x), part);
          part = fmaf(bf16_lo(a.y), bf16_lo(c.y), part); part = fmaf(bf16_hi(a.y), bf16_hi(c.y), part);
          part = fmaf(bf16_lo(a.z), bf16_lo(c.z), part); part = fmaf(bf16_hi(a.z), bf16_hi(c.z), part);
          part = fmaf(bf16_lo(a.w), bf16_lo(c.w), part); part = fmaf(bf16_hi(a.w), bf16_hi(c.w), part);
        }
      }
      float* red_it = red + (it & 1u) * 256;     // two buffers: the barrier below orders reuse
      red_it[half * kBlk + row] = part;
      mbar_arrive(BAR(red));
      if (!warp_wait(BAR(red), it & 1u, p.status, ST_TIMEOUT_FULL, 423)) { ok = false; break; }
      const float delta = red_it[row] + red_it[kBlk + row];
      float lse2 = INFINITY;                     // rows past the end, and rows that saw no key, have no probabilities
      if (live) {
        const float l = p.lse[bh * p.seq + q_pos];
        if (l > -INFINITY) lse2 = l * kLog2e;
      }
      if (half == 0) {
        p.lse2[bh * p.seq_pad + q_pos] = lse2;
        p.delta[bh * p.seq_pad + q_pos] = delta;
      }
      for (int j = 0; j < t.blocks; ++j, ++blk) {
        const int key0 = (t.first + j) * kBlk + half * 64;
        const uint32_t s_addr = t_s + (blk & 1u) * 128 + lane_addr + half * 64;
        if (!warp_wait(BAR(s_full) + 8 * (blk & 1u), (blk >> 1) & 1u, p.status, ST_TIMEOUT_TMEM_FULL, 420)) { ok = false; break; }
        tc_fence_after();
        const int hi = live ? q_pos - key0 + 1 : 0;      // visible keys of this row: [lo, hi) of the 64
        const int lo = p.window > 0 ? q_pos - key0 - p.window + 1 : 0;
        const bool masked = __any_sync(kFullMask, hi < 64 || lo > 0);
        float pr[64];
        uint32_t v[32], pk[32];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          tc_ld_32x32b_x32(s_addr + c * 32, v);
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float slope;
            const float pi = probability<kCap>(__uint_as_float(v[i]), lse2, p, slope);
            pr[c * 32 + i] = kCap ? pi * slope : pi;
          }
        }
        if (!warp_wait(BAR(dp_full), blk & 1u, p.status, ST_TIMEOUT_TMEM_FULL, 421)) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          tc_ld_32x32b_x32(t_dp + lane_addr + half * 64 + c * 32, v);
          tc_wait_ld();
          // one branch per tile: the tests of a masked tile cost as much as the arithmetic
          if (masked) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const int n = c * 32 + i;
              pr[n] = n < hi && n >= lo ? pr[n] * (__uint_as_float(v[i]) - delta) : 0.0f;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) pr[c * 32 + i] *= __uint_as_float(v[i]) - delta;
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) pk[c * 16 + i] = pack_bf16(pr[c * 32 + 2 * i], pr[c * 32 + 2 * i + 1]);
        }
        tc_st_32x32b_x32(s_addr, pk);
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(BAR(ds_full));
      }
      if (!ok) break;
      if (!warp_wait(BAR(dq_full), it & 1u, p.status, ST_TIMEOUT_TMEM_FULL, 422)) { ok = false; break; }
      tc_fence_after();
      uint32_t a[32], b[32];
      tc_ld_32x32b_x32(t_dq + lane_addr + half * 64, a);
      tc_ld_32x32b_x32(t_dq + lane_addr + half * 64 + 32, b);
      tc_wait_ld();
      tc_fence_before();
      mbar_arrive(BAR(dq_free));
      ++it;
      if (live) store_half_row(a, b, p.scale, p.dq + at);
    }
  }
#undef BAR
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------------------------------ dK, dV
// TMEM columns: dV 0-127, dK 128-255, S^T 256-383, dP^T 384-511 (lane = key, column = query). P^T overwrites
// S^T and dX^T overwrites dP^T as the A operands of the two accumulating products. Issue order: dV(i), S(i+1),
// dK(i), dP(i+1): the first pair runs while the compute warps form dX(i), the second while they exponentiate.
template <bool kCap>
__global__ void __launch_bounds__(kBwdThreads, 1)
attention_bwd_dkdv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                          const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                          const AttnBwdParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sb = smem_u32(smem);
  if ((sb & 1023u) != 0) {          // the swizzle pattern repeats every 1024 bytes
    if (threadIdx.x == 0) report_failure(p.status, ST_BAD_ARGUMENT, 499, sb, 1024);
    return;
  }
  KvBars* bars = reinterpret_cast<KvBars*>(smem + kKvBar);
  const int warp = __shfl_sync(kFullMask, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
#define BAR(name) PLB_BAR(KvBars, kKvBar, name)
  if (threadIdx.x == 0) {
    mbar_init(BAR(kv_full), 1);
    mbar_init(BAR(kv_empty), 1);
    for (int s = 0; s < kKvQStages; ++s) { mbar_init(BAR(q_full) + 8 * s, 1); mbar_init(BAR(q_empty) + 8 * s, 1); }
    for (int s = 0; s < kKvDoStages; ++s) { mbar_init(BAR(do_full) + 8 * s, 1); mbar_init(BAR(do_empty) + 8 * s, 1); }
    for (int s = 0; s < kKvStatStages; ++s) { mbar_init(BAR(stat_full) + 8 * s, 1); mbar_init(BAR(stat_empty) + 8 * s, kCompute / 32); }
    mbar_init(BAR(s_full), 1);
    mbar_init(BAR(p_full), kCompute);
    mbar_init(BAR(dp_full), 1);
    mbar_init(BAR(ds_full), kCompute);
    mbar_init(BAR(acc_full), 1);
    mbar_init(BAR(acc_free), kCompute);
    mbar_init(BAR(drain), 1);
    fence_mbar_init();
    prefetch_tensormap(&map_q);
    prefetch_tensormap(&map_do);
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&bars->tmem_base), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(kFullMask, *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base), 0);
  const uint32_t t_dv = tmem, t_dk = tmem + 128, t_s = tmem + 256, t_dp = tmem + 384;
  const int items = p.tiles * p.batch * p.kv_heads;

  if (warp == 0) {
    uint32_t it = 0, n = 0;
    bool ok = true;
    for (int wave = 0; ok && wave * static_cast<int>(gridDim.x) < items; ++wave) {
      const int w = snake(wave);
      if (w >= items) continue;
      const KvItem t = kv_item(p, w);
      if (!warp_wait(BAR(kv_empty), (it & 1u) ^ 1u, p.status, ST_TIMEOUT_EMPTY, 430)) { ok = false; break; }
      if (elect_one_sync()) {
        mbar_arrive_expect_tx(BAR(kv_full), 2 * kTileBytes);
        load_tile(sb, &map_k, BAR(kv_full), t.h * kD, t.k0, t.b);
        load_tile(sb + kTileBytes, &map_v, BAR(kv_full), t.h * kD, t.k0, t.b);
      }
      __syncwarp();
      ++it;
      int g = 0, qt = 0;
      for (int i = 0; i < t.n; ++i, ++n) {
        const int h = t.h * p.group + g, row = (t.first + qt) * kBlk;
        const uint32_t qs = n % kKvQStages, ds = n % kKvDoStages, ss = n % kKvStatStages;
        if (!warp_wait(BAR(q_empty) + 8 * qs, ((n / kKvQStages) & 1u) ^ 1u, p.status, ST_TIMEOUT_EMPTY, 431)) { ok = false; break; }
        if (elect_one_sync()) {
          mbar_arrive_expect_tx(BAR(q_full) + 8 * qs, kTileBytes);
          load_tile(sb + kKvQ + qs * kTileBytes, &map_q, BAR(q_full) + 8 * qs, h * kD, row, t.b);
        }
        __syncwarp();
        if (!warp_wait(BAR(stat_empty) + 8 * ss, ((n / kKvStatStages) & 1u) ^ 1u, p.status, ST_TIMEOUT_EMPTY, 432)) { ok = false; break; }
        if (elect_one_sync()) {
          const int64_t at = (static_cast<int64_t>(t.b) * p.q_heads + h) * p.seq_pad + row;
          mbar_arrive_expect_tx(BAR(stat_full) + 8 * ss, 1024);
          bulk_load(sb + kKvStat + ss * 1024, p.lse2 + at, 512, BAR(stat_full) + 8 * ss);
          bulk_load(sb + kKvStat + ss * 1024 + 512, p.delta + at, 512, BAR(stat_full) + 8 * ss);
        }
        __syncwarp();
        if (!warp_wait(BAR(do_empty) + 8 * ds, ((n / kKvDoStages) & 1u) ^ 1u, p.status, ST_TIMEOUT_EMPTY, 433)) { ok = false; break; }
        if (elect_one_sync()) {
          mbar_arrive_expect_tx(BAR(do_full) + 8 * ds, kTileBytes);
          load_tile(sb + kKvDo + ds * kTileBytes, &map_do, BAR(do_full) + 8 * ds, h * kD, row, t.b);
        }
        __syncwarp();
        if (++qt == t.tiles) { qt = 0; ++g; }
      }
    }
    if (!ok) linger();
  } else if (warp == 1) {
    uint32_t it = 0, n = 0;
    bool ok = true;
    auto issue_s = [&](uint32_t i) {
      const uint32_t qs = i % kKvQStages;
      if (!warp_wait(BAR(q_full) + 8 * qs, (i / kKvQStages) & 1u, p.status, ST_TIMEOUT_FULL, 440)) return false;
      tc_fence_after();
      mma_tiles(t_s, sb, sb + kKvQ + qs * kTileBytes, BAR(s_full));
      return true;
    };
    auto issue_dp = [&](uint32_t i) {
      const uint32_t ds = i % kKvDoStages;
      if (!warp_wait(BAR(do_full) + 8 * ds, (i / kKvDoStages) & 1u, p.status, ST_TIMEOUT_FULL, 441)) return false;
      tc_fence_after();
      mma_tiles(t_dp, sb + kTileBytes, sb + kKvDo + ds * kTileBytes, BAR(dp_full));
      return true;
    };
    for (int wave = 0; ok && wave * static_cast<int>(gridDim.x) < items; ++wave) {
      const int w = snake(wave);
      if (w >= items) continue;
      const int steps = __shfl_sync(kFullMask, kv_item(p, w).n, 0);
      if (!warp_wait(BAR(kv_full), it & 1u, p.status, ST_TIMEOUT_FULL, 442)) { ok = false; break; }
      tc_fence_after();
      if (!issue_s(n) || !issue_dp(n)) { ok = false; break; }
      for (int i = 0; i < steps && ok; ++i, ++n) {
        const bool more = i + 1 < steps;
        const uint32_t qs = n % kKvQStages, ds = n % kKvDoStages;
        if (!warp_wait(BAR(p_full), n & 1u, p.status, ST_TIMEOUT_FULL, 443)) { ok = false; break; }
        if (i == 0 && !warp_wait(BAR(acc_free), (it & 1u) ^ 1u, p.status, ST_TIMEOUT_TMEM_EMPTY, 444)) { ok = false; break; }
        tc_fence_after();
        mma_from_tmem(t_dv, t_s, sb + kKvDo + ds * kTileBytes, i != 0, BAR(do_empty) + 8 * ds);
        if (more && !issue_s(n + 1)) { ok = false; break; }
        if (!warp_wait(BAR(ds_full), n & 1u, p.status, ST_TIMEOUT_FULL, 445)) { ok = false; break; }
        tc_fence_after();
        mma_from_tmem(t_dk, t_dp, sb + kKvQ + qs * kTileBytes, i != 0, BAR(q_empty) + 8 * qs);
        if (more && !issue_dp(n + 1)) { ok = false; break; }
      }
      if (!ok) break;
      warp_commit(BAR(kv_empty));
      warp_commit(BAR(acc_full));
      ++it;
    }
    if (!ok) drain_mma(BAR(drain));
  } else if (warp >= 4) {
    const int half = (warp - 4) >> 2, quad = warp & 3, row = quad * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t s_addr = t_s + lane_addr + half * 64, dp_addr = t_dp + lane_addr + half * 64;
    uint32_t it = 0, n = 0;
    bool ok = true;
    for (int wave = 0; ok && wave * static_cast<int>(gridDim.x) < items; ++wave) {
      const int w = snake(wave);
      if (w >= items) continue;
      const KvItem t = kv_item(p, w);
      const int k_pos = t.k0 + row;
      int qt = 0;
      for (int i = 0; i < t.n; ++i, ++n) {
        const int q0 = (t.first + qt) * kBlk + half * 64;
        if (++qt == t.tiles) qt = 0;
        const uint32_t ss = n % kKvStatStages;
        const float4* stat = reinterpret_cast<const float4*>(smem + kKvStat + ss * 1024 + half * 256);
        // visible queries of this key: [lo, hi) of the 64
        const int lo = k_pos - q0;
        const int hi = min(p.seq - q0, p.window > 0 ? min(lo, 64) + p.window : 64);
        const bool masked = __any_sync(kFullMask, lo > 0 || hi < 64);
        if (!warp_wait(BAR(stat_full) + 8 * ss, (n / kKvStatStages) & 1u, p.status, ST_TIMEOUT_FULL, 450)) { ok = false; break; }
        if (!warp_wait(BAR(s_full), n & 1u, p.status, ST_TIMEOUT_TMEM_FULL, 451)) { ok = false; break; }
        tc_fence_after();
        float pr[64];
        uint32_t v[32], pk[32];
        auto probabilities = [&](auto m, int c) {
#pragma unroll
          for (int i4 = 0; i4 < 8; ++i4) {
            const float4 l = stat[c * 8 + i4];
            const float ls[4] = {l.x, l.y, l.z, l.w};
            float last = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int q = c * 32 + i4 * 4 + e;
              float slope;
              float v1 = probability<kCap>(__uint_as_float(v[i4 * 4 + e]), ls[e], p, slope);
              if (decltype(m)::value && (q < lo || q >= hi)) v1 = 0.0f;
              if (e & 1) pk[q >> 1] = pack_bf16(last, v1);
              last = v1;
              pr[q] = kCap ? v1 * slope : v1;
            }
          }
        };
        auto gradients = [&](auto m, int c) {
#pragma unroll
          for (int i4 = 0; i4 < 8; ++i4) {
            const float4 l = stat[32 + c * 8 + i4];
            const float dl[4] = {l.x, l.y, l.z, l.w};
            float last = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int q = c * 32 + i4 * 4 + e;
              float d = pr[q] * (__uint_as_float(v[i4 * 4 + e]) - dl[e]);
              if (decltype(m)::value && (q < lo || q >= hi)) d = 0.0f;
              if (e & 1) pk[q >> 1] = pack_bf16(last, d);
              last = d;
            }
          }
        };
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          tc_ld_32x32b_x32(s_addr + c * 32, v);
          tc_wait_ld();
          // one branch per tile: the tests of a masked tile cost as much as the arithmetic
          if (masked) probabilities(TrueTag{}, c);
          else probabilities(FalseTag{}, c);
        }
        tc_st_32x32b_x32(s_addr, pk);
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(BAR(p_full));
        if (!warp_wait(BAR(dp_full), n & 1u, p.status, ST_TIMEOUT_TMEM_FULL, 452)) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          tc_ld_32x32b_x32(dp_addr + c * 32, v);
          tc_wait_ld();
          if (masked) gradients(TrueTag{}, c);
          else gradients(FalseTag{}, c);
        }
        tc_st_32x32b_x32(dp_addr, pk);
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(BAR(ds_full));
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR(stat_empty) + 8 * ss);
      }
      if (!ok) break;
      if (!warp_wait(BAR(acc_full), it & 1u, p.status, ST_TIMEOUT_TMEM_FULL, 453)) { ok = false; break; }
      tc_fence_after();
      const size_t at = ((static_cast<size_t>(t.b) * p.seq + k_pos) * p.kv_heads + t.h) * kD + half * 64;
      uint32_t a[32], b[32];
      tc_ld_32x32b_x32(t_dv + lane_addr + half * 64, a);
      tc_ld_32x32b_x32(t_dv + lane_addr + half * 64 + 32, b);
      tc_wait_ld();
      if (k_pos < p.seq) store_half_row(a, b, 1.0f, p.dv + at);
      tc_ld_32x32b_x32(t_dk + lane_addr + half * 64, a);
      tc_ld_32x32b_x32(t_dk + lane_addr + half * 64 + 32, b);
      tc_wait_ld();
      tc_fence_before();
      mbar_arrive(BAR(acc_free));
      ++it;
      if (k_pos < p.seq) store_half_row(a, b, p.scale, p.dk + at);
    }
  }
#undef BAR
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                             const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                             CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// [batch, seq, cols] bf16, contiguous; box = 64 columns x 128 positions of one sequence, 128-byte swizzle.
bool encode_sequences(CUtensorMap* map, const void* base, uint64_t batch, uint64_t seq, uint64_t cols) {
  static EncodeFn fn = nullptr;
  if (fn == nullptr) {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return false;
    fn = reinterpret_cast<EncodeFn>(sym);
  }
  const cuuint64_t dims[3] = {cols, seq, batch};
  const cuuint64_t strides[2] = {cols * 2, seq * cols * 2};
  const cuuint32_t box[3] = {64, kBlk, 1};
  const cuuint32_t elem[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, elem,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

cudaError_t launch_attention_bwd(const AttnBwdArgs& a, cudaStream_t stream) {
  CUtensorMap mq, mdo, mk, mv;
  if (!encode_sequences(&mq, a.q, a.batch, a.seq, static_cast<uint64_t>(a.q_heads) * kD) ||
      !encode_sequences(&mdo, a.d_out, a.batch, a.seq, static_cast<uint64_t>(a.q_heads) * kD) ||
      !encode_sequences(&mk, a.k, a.batch, a.seq, static_cast<uint64_t>(a.kv_heads) * kD) ||
      !encode_sequences(&mv, a.v, a.batch, a.seq, static_cast<uint64_t>(a.kv_heads) * kD))
    return cudaErrorInvalidValue;
  AttnBwdParams p;
  p.out = static_cast<const __nv_bfloat16*>(a.out);
  p.d_out = static_cast<const __nv_bfloat16*>(a.d_out);
  p.lse = a.lse;
  p.dq = static_cast<__nv_bfloat16*>(a.dq);
  p.dk = static_cast<__nv_bfloat16*>(a.dk);
  p.dv = static_cast<__nv_bfloat16*>(a.dv);
  p.batch = a.batch;
  p.seq = a.seq;
  p.tiles = (a.seq + kBlk - 1) / kBlk;
  p.seq_pad = static_cast<int64_t>(p.tiles) * kBlk;
  p.q_heads = a.q_heads;
  p.kv_heads = a.kv_heads;
  p.group = a.q_heads / a.kv_heads;
  p.window = a.window < a.seq ? a.window : 0;     // a window no shorter than the sequence hides nothing
  p.lse2 = a.workspace;
  p.delta = a.workspace + static_cast<int64_t>(a.batch) * a.q_heads * p.seq_pad;
  p.scale = a.scale;
  p.scale_log2 = a.scale * kLog2e;
  const bool cap = a.softcap > 0.0f;
  p.cap_in = cap ? 2.0f * kLog2e * a.scale / a.softcap : 0.0f;
  p.cap_out = a.softcap * kLog2e;
  p.status = a.status;
  const int64_t q_items = static_cast<int64_t>(p.tiles) * a.batch * a.q_heads;
  const int64_t kv_items = static_cast<int64_t>(p.tiles) * a.batch * a.kv_heads;
  auto dq = cap ? attention_bwd_dq_kernel<true> : attention_bwd_dq_kernel<false>;
  auto dkdv = cap ? attention_bwd_dkdv_kernel<true> : attention_bwd_dkdv_kernel<false>;
  cudaError_t err = cudaFuncSetAttribute(dq, cudaFuncAttributeMaxDynamicSharedMemorySize, kDqSmem);
  if (err != cudaSuccess) return err;
  err = cudaFuncSetAttribute(dkdv, cudaFuncAttributeMaxDynamicSharedMemorySize, kKvSmem);
  if (err != cudaSuccess) return err;
  dq<<<static_cast<int>(q_items < a.num_sms ? q_items : a.num_sms), kBwdThreads, kDqSmem, stream>>>(mq, mdo, mk, mv, p);
  err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  dkdv<<<static_cast<int>(kv_items < a.num_sms ? kv_items : a.num_sms), kBwdThreads, kKvSmem, stream>>>(mq, mdo, mk, mv, p);
  return cudaGetLastError();
}

}  // namespace plb
