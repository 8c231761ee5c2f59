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
// Roundings: P and dX go to bf16 (the tensor cores' operand type, off by at most 2^-8 of the value); every sum,
// the exponent, delta and the accumulators are fp32; the gradients are rounded once when they are stored. Two roundings
// of the same size on the way, so the error of a gradient is sqrt(2) times what rounding the exact one leaves, 2.3e-3 to
// 2.4e-3 of its norm against 1.7e-3, at any length: the errors of a sum's terms add up as the terms do.
//
// Tensor maps are 3-D (column, position, batch): rows past a sequence's end read as zeros and never as the
// next sequence's, and their probabilities are forced to 0 (log-sum-exp +inf), so any length works.
#include <math.h>

#include <atomic>
#include <cstddef>

#include "attention_bwd.h"
#include "attention_roles.cuh"

namespace plb {

using namespace attn;

namespace {

constexpr int kBwdThreads = 384;      // warp 0 TMA, warp 1 MMA, warps 2-3 the rows' constants (dq), warps 4-11 compute
constexpr int kComputeWarps = 8;
constexpr uint32_t kFullMask = 0xFFFFFFFFu;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kBwdRuns = 148;         // runs of steps: a CTA on every SM; no run waits for another, so fewer SMs only take longer

// ---- shared-memory maps (offsets from a 1024-byte aligned base)
constexpr int kDqK = 2 * kTileBytes, kDqKStages = 3;                  // after Q and dO
constexpr int kDqV = kDqK + kDqKStages * kTileBytes, kDqVStages = 2;
constexpr int kDqStat = kDqV + kDqVStages * kTileBytes;               // [2][2][128] floats: log-sum-exp and delta of two tiles
constexpr int kDqRed = kDqStat + 2048;                                // [128] floats
constexpr int kDqBar = kDqRed + 512;
constexpr int kDqSmem = kDqBar + 256;

// dK, dV: K and V, then the streamed tiles with their rows' constants behind them (see kAuxBytes)
constexpr int kAuxBytes = kBlk * 32;                                  // 128 rows of 16 bf16
constexpr int kKvStage = kTileBytes + kAuxBytes;
constexpr int kKvQ = 2 * kTileBytes, kKvQStages = 2;
constexpr int kKvDo = kKvQ + kKvQStages * kKvStage, kKvDoStages = 2;
constexpr int kKvOnes = kKvDo + kKvDoStages * kKvStage;
constexpr int kKvBar = kKvOnes + kAuxBytes;
constexpr int kKvSmem = kKvBar + 256;
static_assert(kDqSmem <= 232448 && kKvSmem <= 232448, "227 KB of shared memory per CTA");

struct DqBars {
  uint64_t q_full, q_empty, k_full[kDqKStages], k_empty[kDqKStages], v_full[kDqVStages], v_empty[kDqVStages];
  uint64_t s_full[2], dp_full, dp_read, ds_full[2], dq_full, dq_free, red, stat_full[2], stat_empty[2], drain;
  uint32_t tmem_base, pad;
};
struct KvBars {
  uint64_t kv_full, kv_empty, q_full[kKvQStages], q_empty[kKvQStages], do_full[kKvDoStages], do_empty[kKvDoStages];
  uint64_t s_full, p_full[2], dp_full, ds_full, acc_full, acc_free, drain;
  uint32_t tmem_base, pad;
};
static_assert(sizeof(DqBars) <= 256 && sizeof(KvBars) <= 256, "barrier block");

// Work lists are sorted heavy first; walking them forth and back evens out what a CTA gets.
__device__ __forceinline__ int snake(int wave) {
  return wave * gridDim.x + ((wave & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

// A tile of queries that see one or two key tiles (`measure`) goes over them twice, first for delta = sum P dP: where a
// row sees few keys the rounding of the saved output is not averaged out of delta = sum dO O, and with it the error of
// dQ and dK would be larger (sequences of 20: 2.6e-3 of the norm instead of 2.3e-3, of 77: 2.5e-3 instead of 2.3e-3; a window
// of 32 in 1024 positions: 2.44e-3 instead of 2.35e-3). It costs 0.3 us of 14 there, and where a window of at most 129 leaves
// no other tiles, 4 to 7 % (8192 positions of 32 / 8 heads, window 64: 177 us, 165.5 without; window 128: 172 and 165).
struct DqItem { int b, h, q0, first, blocks, steps; bool measure; };
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
  t.measure = t.blocks <= 2;
  t.steps = t.measure ? 2 * t.blocks : t.blocks;
  return t;
}
// Query tiles that see key tile kb.
__host__ __device__ __forceinline__ int kv_query_tiles(int tiles, int window, int kb) {
  const int64_t last = window > 0 ? (static_cast<int64_t>(kb) * kBlk + kBlk - 1 + window - 1) / kBlk : tiles;
  return (last < tiles - 1 ? static_cast<int>(last) : tiles - 1) + 1 - kb;
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
  t.tiles = kv_query_tiles(p.tiles, p.window, kb);
  t.n = t.tiles * p.group;
  return t;
}
// The key tiles' steps (a step: one query tile of one head) in one line, heaviest tiles first, cut into equal runs,
// where a tile counts kTileSteps more than it has, for its loads and stores: run r begins at step[r] of tile w[r].
constexpr int kTileSteps = 2;
struct Runs { int count, w[kBwdRuns + 1], step[kBwdRuns + 1]; };
// What a CTA works through: whole tiles (no runs, the list walked forth and back) or its run, steps [i0, i1) of tile w.
struct KvWalk {
  int w, i0, i1, wave, end_w, end_step;
  KvItem t;
  bool whole;
  __device__ __forceinline__ bool begin(const AttnBwdParams& p, const Runs& runs, int items) {
    wave = 0;
    i0 = 0;
    end_w = items;
    end_step = 0;
    whole = runs.count == 0;
    if (!whole) {
      w = runs.w[blockIdx.x];
      i0 = runs.step[blockIdx.x];
      end_w = runs.w[blockIdx.x + 1];
      end_step = runs.step[blockIdx.x + 1];
    } else {
      w = snake(0);
    }
    return set(p);
  }
  __device__ __forceinline__ bool next(const AttnBwdParams& p) {
    if (!whole) {
      ++w;
      i0 = 0;
    } else {
      w = snake(++wave);
    }
    return set(p);
  }
  __device__ __forceinline__ bool set(const AttnBwdParams& p) {
    if (w > end_w || (w == end_w && i0 >= end_step)) return false;     // only the last wave of whole tiles is short
    t = kv_item(p, w);
    i1 = w == end_w ? end_step : t.n;
    return true;
  }
};

// The second kernel is launched while the first one ends: its CTAs set up on SMs that are free and wait for the first
// one's results where they first read them (4 us of two sequences of 77's 20).
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_first() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// The waiting itself, out of the way of the roles' code. A launch finds none of its code in the instruction caches, and
// what does not fit there is fetched again in every step: this and one copy of each product and epilogue took 2048
// positions of 32 / 8 heads from 122 to 111 us, 2 x 4001 with a cap from 305 to 260.
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity, Status* st, int code, int what) {
  const long long t0 = clock64();
  for (uint32_t it = 1; !mbar_try_wait(bar, parity); ++it) {
    if ((it & 63u) != 0u) continue;
    if (st != nullptr && ld_volatile_i32(&st->code) != 0) return false;
    if (clock64() - t0 > kWaitBudgetCycles) {
      if (st != nullptr) report_failure(st, code, what, parity, bar);
      return false;
    }
  }
  return true;
}
// A role's bounded wait; the warp's lanes agree on the outcome. Without a status record a wait that runs out goes
// unreported, and the CTA's others run out by themselves.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, Status* st, int code, int what) {
  const bool ok = mbar_try_wait(bar, parity) || wait_long(bar, parity, st, code, what);
  return __all_sync(kFullMask, ok) != 0;
}
// A compute warp's arrival: one for its 32 lanes (32 arrivals on one barrier are 32 shared-memory atomics in a row,
// and with two barriers a tile those took a quarter of the compute warps' time).
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}
__device__ __forceinline__ void warp_commit(uint32_t bar) {
  if (elect_one_sync()) tc_commit(bar);
  __syncwarp();
}
// A constant c_q of every row q of B, added to column q of A B^T by the tensor core: one more step of the contraction
// whose A is all ones and whose B row holds c_q as three bf16 numbers (24 bits, an fp32 number) and zeros. In the
// transposed products the constants belong to columns, and every thread would read all 128 of them from shared
// memory, 665 cycles of its bandwidth a tile next to the 2048 the products take.
constexpr uint64_t kDescAux = smem_desc_hi(256, 0, 6);                // rows of 32 bytes, 32-byte swizzle
__device__ __forceinline__ void store_constant(uint8_t* tile, int row, float c) {
  const __nv_bfloat16 hi = __float2bfloat16_rn(c);
  const float r = fabsf(c) < INFINITY ? c - __bfloat162float(hi) : 0.0f;
  const __nv_bfloat16 mid = __float2bfloat16_rn(r);
  const __nv_bfloat16 lo = __float2bfloat16_rn(r - __bfloat162float(mid));
  const uint32_t w0 = static_cast<uint32_t>(__bfloat16_as_ushort(hi)) | static_cast<uint32_t>(__bfloat16_as_ushort(mid)) << 16;
  uint4* dst = reinterpret_cast<uint4*>(tile + row * 32);
  const int first = (row >> 2) & 1;                                   // the swizzle exchanges the two 16-byte chunks of rows 4-7 of 8
  dst[first] = make_uint4(w0, __bfloat16_as_ushort(lo), 0, 0);
  dst[first ^ 1] = make_uint4(0, 0, 0, 0);
}
// D = A B^T over 128 columns of the contraction, both operands K-major tiles in shared memory, then the barrier. With
// aux, B's rows' constants are added (ones: the tile of ones).
__device__ __forceinline__ void mma_tiles(uint32_t d, uint32_t a, uint32_t b, uint32_t bar, uint32_t ones = 0, uint32_t aux = 0) {
  const uint64_t ad = smem_desc(a, kDescSw128KMajor), bd = smem_desc(b, kDescSw128KMajor);
  const uint64_t od = smem_desc(ones, kDescAux), cd = smem_desc(aux, kDescAux);
  if (elect_one_sync()) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t off = ((k >> 2) * kAtomBytes + (k & 3) * 32) >> 4;
      tc_mma_f16(d, ad + off, bd + off, kIdescQK, k != 0 ? 1u : 0u);
    }
    if (aux != 0) tc_mma_f16(d, od, cd, kIdescQK, 1u);
    tc_commit(bar);
  }
  __syncwarp();
}
// D += A B with A bf16 in tensor memory (its two 64-column halves at a and a + 64) and B's rows along the contraction.
// Steps k0, k0 + 1 of each half if `part`, else all eight; the barrier may be 0.
__device__ __forceinline__ void mma_from_tmem(uint32_t d, uint32_t a, uint32_t b, bool accumulate, uint32_t bar, bool part = false, int k0 = 0) {
  const uint64_t bd = smem_desc(b, kDescVMn);
  if (elect_one_sync()) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (!part || (k & 2) == k0)
        tc_mma_f16_ts(d, a + (k >> 2) * 64 + (k & 3) * 8, bd + ((k * 2048) >> 4), kIdescPV, k != k0 || accumulate ? 1u : 0u);
    if (bar != 0) tc_commit(bar);
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

__device__ __forceinline__ Pair exp2_pair(Pair x) {
  float a, b;
  split(x, a, b);
  return make_pair(ex2_approx(a), ex2_approx(b));
}

// tanh(x) for |x| <= kSmallCap as x times a polynomial of degree 4 in x^2, fitted here for the least largest relative
// error (its extremes over the range alternate at six points): 2^-23.4 with the coefficients as written, rounded to fp32,
// 2^-22.4 as evaluated in fp32. Where all scores of a warp's tile are that small against
// the cap it leaves the special-function unit to the exponential: with tanh from exp2 and a division it has three
// results to give per score. 2 x 4096 positions of 16 heads, window 1024, cap 30: 255 us with scores of deviation 1, all of
// them small, and 678 us with deviation 16, which the other path takes; 8192 of 32 / 8 heads without a window 1.73 and 5.2 ms.
// The forward pass takes tanh.approx, 2^-16.4 of its value as measured: its log-sum-exp is off by at most 4e-4 at a cap of
// 50 with scores at it, and errors of the gradients by norm are larger by at most 4 % than with the exact one.
constexpr float kSmallCap = 0.6f;
__device__ __forceinline__ Pair tanh_small(Pair x) {
  const Pair u = mul2(x, x);
  Pair y = fma2(make_pair(0.015475427731871605f, 0.015475427731871605f), u, make_pair(-0.05210148170590401f, -0.05210148170590401f));
  y = fma2(y, u, make_pair(0.13310173153877258f, 0.13310173153877258f));
  y = fma2(y, u, make_pair(-0.33332309126853943f, -0.33332309126853943f));
  y = fma2(y, u, make_pair(0.9999999403953552f, 0.9999999403953552f));
  return mul2(x, y);
}
// Any x: 1 - 2 / (1 + 2^(2 x log2 e)) rather than tanh.approx, whose error the slope 1 - tanh^2 would see. A function of
// its own: 64 copies of it would lie between the code of the tiles whose scores are small.
__device__ __noinline__ float tanh_any(float x) {
  return 1.0f - __fdividef(2.0f, 1.0f + ex2_approx(fminf(x * (2.0f * kLog2e), 60.0f)));
}
// Probabilities of two raw scores; with a cap also its slope. minus_lse2: the rows' negated base-2 log-sum-exp; small:
// whether every score of the warp's tile is within the polynomial's range.
template <bool kCap>
__device__ __forceinline__ Pair probability(Pair s, Pair minus_lse2, const AttnBwdParams& p, bool small, Pair& slope) {
  if (kCap) {
    const Pair x = mul2(s, make_pair(p.cap_in, p.cap_in));
    Pair t;
    if (small) {
      t = tanh_small(x);
    } else {
      float a, b;
      split(x, a, b);
      t = make_pair(tanh_any(a), tanh_any(b));
    }
    slope = fma2(mul2(t, t), make_pair(-1.0f, -1.0f), make_pair(1.0f, 1.0f));
    return exp2_pair(fma2(t, make_pair(p.cap_out, p.cap_out), minus_lse2));
  }
  return exp2_pair(fma2(s, make_pair(p.scale_log2, p.scale_log2), minus_lse2));
}
// Whether no score of the 64 a lane holds, or of its warp's other lanes', leaves the polynomial's range.
__device__ __forceinline__ bool all_small(const uint32_t (&v)[32], const uint32_t (&u)[32], const AttnBwdParams& p) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 32; ++i) m = fmaxf(m, fmaxf(fabsf(__uint_as_float(v[i])), fabsf(__uint_as_float(u[i]))));
  return __all_sync(kFullMask, m * p.cap_in <= kSmallCap) != 0;
}
__device__ __forceinline__ uint32_t pack_bf16(Pair p) {
  float a, b;
  split(p, a, b);
  const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&t);
}
// Zeroes a pair's members outside [lo, hi); i is the first one's index.
__device__ __forceinline__ Pair keep_range(Pair p, int i, int lo, int hi) {
  float a, b;
  split(p, a, b);
  return make_pair(i >= lo && i < hi ? a : 0.0f, i + 1 >= lo && i + 1 < hi ? b : 0.0f);
}
// 64 fp32 accumulator columns of each lane's row, scaled, as bf16 to 128 bytes of the row; `rows` of the warp's rows
// exist, `stride` elements apart from dst on. Eight lanes first exchange their 16-byte chunks so that each store
// writes whole 128-byte pieces of four rows; a lane storing its own row would touch 32 lines with every store, some
// 8000 cycles of the store path a tile.
__device__ __forceinline__ void store_half_rows(const uint32_t (&a)[32], const uint32_t (&b)[32], float scale, __nv_bfloat16* dst,
                                                int64_t stride, int rows) {
  const int lane = threadIdx.x & 31;
  uint32_t w[8][4];
#pragma unroll
  for (int g = 0; g < 8; ++g)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = (g & 3) * 8 + e * 2;
      w[g][e] = g < 4 ? pack_bf16(mul2(make_pair(a[i], a[i + 1]), make_pair(scale, scale)))
                      : pack_bf16(mul2(make_pair(b[i], b[i + 1]), make_pair(scale, scale)));
    }
  // chunk g of lane l goes to chunk l of lane g of its eight: exchange across one bit of both at a time
#pragma unroll
  for (int bit = 1; bit < 8; bit <<= 1) {
    const bool up = lane & bit;
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      if (g & bit) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t got = __shfl_xor_sync(kFullMask, up ? w[g][e] : w[g | bit][e], bit);
        if (up) w[g][e] = got;
        else w[g | bit][e] = got;
      }
    }
  }
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    const int row = (lane & ~7) + g;
    if (row < rows) reinterpret_cast<uint4*>(dst + row * stride)[lane & 7] = make_uint4(w[g][0], w[g][1], w[g][2], w[g][3]);
  }
}

// A part's slot: dV then dK, [32 column quadruples][128 rows].
constexpr int kPartVecs = 2 * 32 * kBlk;
__device__ __forceinline__ void store_part(const uint32_t (&a)[32], const uint32_t (&b)[32], float4* dst) {
#pragma unroll
  for (int g = 0; g < 16; ++g) {
    const int i = (g & 7) * 4;
    dst[g * kBlk] = g < 8 ? make_float4(__uint_as_float(a[i]), __uint_as_float(a[i + 1]), __uint_as_float(a[i + 2]), __uint_as_float(a[i + 3]))
                          : make_float4(__uint_as_float(b[i]), __uint_as_float(b[i + 1]), __uint_as_float(b[i + 2]), __uint_as_float(b[i + 3]));
  }
}

#define PLB_BAR(type, base, name) (sb + (base) + offsetof(type, name))

// ------------------------------------------------------------------------------------------ dQ
// TMEM columns: dQ 0-127, S 128-255 and 256-383 (two buffers), dP 384-511. dX overwrites the S buffer it came
// from, as the A operand of dQ += dX K. dP(j+1) is issued as soon as dP(j) has been read into registers, S(j+2) as
// soon as dQ(j) has released its buffer, so the compute warps find their next operands ready. A warp that is done with
// dX(j) may therefore finish dX(j+1) before another is done with dX(j) (a warp without masked pairs before one with some):
// consecutive blocks report on two barriers, or its second arrival would count for the other warp's first.
template <bool kCap>
__global__ void __launch_bounds__(kBwdThreads, 1)
attention_bwd_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                        const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        const AttnBwdParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sb = smem_u32(smem);
  if ((sb & 1023u) != 0) {          // the swizzle pattern repeats every 1024 bytes
    if (threadIdx.x == 0 && p.status != nullptr) report_failure(p.status, ST_BAD_ARGUMENT, 499, sb, 1024);
    return;
  }
  launch_dependents();
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
    mbar_init(BAR(dp_read), kComputeWarps);
    mbar_init(BAR(ds_full), kComputeWarps);
    mbar_init(BAR(ds_full) + 8, kComputeWarps);
    mbar_init(BAR(dq_full), 1);
    mbar_init(BAR(dq_free), kComputeWarps);
    mbar_init(BAR(red), kComputeWarps);
    for (int s = 0; s < 2; ++s) { mbar_init(BAR(stat_full) + 8 * s, 2); mbar_init(BAR(stat_empty) + 8 * s, kComputeWarps); }
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
      for (int j = 0; j < t.steps; ++j, ++kv) {
        const int row = (t.first + (j < t.blocks ? j : j - t.blocks)) * kBlk;
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
      const DqItem t = dq_item(p, w);
      const int n = __shfl_sync(kFullMask, t.steps, 0), from = __shfl_sync(kFullMask, t.steps - t.blocks, 0);
      if (!warp_wait(BAR(q_full), it & 1u, p.status, ST_TIMEOUT_FULL, 412)) { ok = false; break; }
      tc_fence_after();
      // dP(j+1), dQ(j), S(j+2), from one copy of each product's code
      blk -= 2;
#pragma unroll 1
      for (int j = -2; j < n; ++j, ++blk) {
        if (j >= 0 && !warp_wait(BAR(dp_read), blk & 1u, p.status, ST_TIMEOUT_FULL, 415)) { ok = false; break; }
        if (j >= -1 && j + 1 < n && !issue_dp(blk + 1)) { ok = false; break; }
        if (j + 2 == n) warp_commit(BAR(q_empty));       // the last products that read Q and dO are issued: both may be replaced
        if (j >= 0) {
          if (!warp_wait(BAR(ds_full) + 8 * (blk & 1u), (blk >> 1) & 1u, p.status, ST_TIMEOUT_FULL, 413)) { ok = false; break; }
          if (j == from && !warp_wait(BAR(dq_free), (it & 1u) ^ 1u, p.status, ST_TIMEOUT_TMEM_EMPTY, 414)) { ok = false; break; }
          tc_fence_after();
          const uint32_t ks = blk % kDqKStages;
          if (j < from) warp_commit(BAR(k_empty) + 8 * ks);
          else mma_from_tmem(t_dq, t_s + (blk & 1u) * 128, sb + kDqK + ks * kTileBytes, j != from, BAR(k_empty) + 8 * ks);
        }
        if (j + 2 < n && !issue_s(blk + 2)) { ok = false; break; }
      }
      if (!ok) break;
      warp_commit(BAR(dq_full));
      ++it;
    }
    if (!ok) drain_mma(BAR(drain));
  } else if (warp < 4) {
    // base-2 log-sum-exp and delta of the rows, a tile ahead of the compute warps: 64 rows a warp, 16 lanes a row
    uint32_t it = 0;
    for (int wave = 0; wave * static_cast<int>(gridDim.x) < items; ++wave) {
      const int w = snake(wave);
      if (w >= items) continue;
      const DqItem t = dq_item(p, w);
      if (!warp_wait(BAR(stat_empty) + 8 * (it & 1u), ((it >> 1) & 1u) ^ 1u, p.status, ST_TIMEOUT_EMPTY, 404)) break;
      float* stat = reinterpret_cast<float*>(smem + kDqStat) + (it & 1u) * 256;
      const int row0 = (warp - 2) * 64;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = row0 + 32 * i + lane;
        float lse2 = INFINITY;                   // rows past the end, and rows that saw no key, have no probabilities
        if (t.q0 + row < p.seq) {
          const float l = p.lse[(static_cast<int64_t>(t.b) * p.q_heads + t.h) * p.seq + t.q0 + row];
          if (l > -INFINITY) lse2 = l * kLog2e;
        }
        stat[row] = lse2;
      }
      if (!t.measure) {
        const size_t at = ((static_cast<size_t>(t.b) * p.seq + t.q0) * p.q_heads + t.h) * kD;
        const size_t stride = static_cast<size_t>(p.q_heads) * kD;
#pragma unroll 1                            // code that runs once a tile is fetched as it runs: four copies took 4 us more
        for (int r0 = row0; r0 < row0 + 64; r0 += 16) {
          uint4 o[8], g[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int row = r0 + 2 * i + (lane >> 4);
            o[i] = make_uint4(0, 0, 0, 0);
            g[i] = make_uint4(0, 0, 0, 0);
            if (t.q0 + row < p.seq) {
              o[i] = reinterpret_cast<const uint4*>(p.out + at + row * stride)[lane & 15];
              g[i] = reinterpret_cast<const uint4*>(p.d_out + at + row * stride)[lane & 15];
            }
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            Pair sum = mul2(make_pair(bf16_lo(o[i].x), bf16_hi(o[i].x)), make_pair(bf16_lo(g[i].x), bf16_hi(g[i].x)));
            sum = fma2(make_pair(bf16_lo(o[i].y), bf16_hi(o[i].y)), make_pair(bf16_lo(g[i].y), bf16_hi(g[i].y)), sum);
            sum = fma2(make_pair(bf16_lo(o[i].z), bf16_hi(o[i].z)), make_pair(bf16_lo(g[i].z), bf16_hi(g[i].z)), sum);
            sum = fma2(make_pair(bf16_lo(o[i].w), bf16_hi(o[i].w)), make_pair(bf16_lo(g[i].w), bf16_hi(g[i].w)), sum);
            float lo, hi;
            split(sum, lo, hi);
            lo += hi;
#pragma unroll
            for (int k = 8; k > 0; k >>= 1) lo += __shfl_xor_sync(kFullMask, lo, k);
            if ((lane & 15) == 0) stat[kBlk + r0 + 2 * i + (lane >> 4)] = lo;
          }
        }
      }
      warp_arrive(BAR(stat_full) + 8 * (it & 1u));
      ++it;
    }
  } else {
    const int half = (warp - 4) >> 2, quad = warp & 3, row = quad * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quad * 32) << 16;
    float* red = reinterpret_cast<float*>(smem + kDqRed);
    uint32_t it = 0, blk = 0, measured = 0;
    bool ok = true;
    for (int wave = 0; ok && wave * static_cast<int>(gridDim.x) < items; ++wave) {
      const int w = snake(wave);
      if (w >= items) continue;
      const DqItem t = dq_item(p, w);
      const int q_pos = t.q0 + row;
      const bool live = q_pos < p.seq;
      float* stat = reinterpret_cast<float*>(smem + kDqStat) + (it & 1u) * 256;
      if (!warp_wait(BAR(stat_full) + 8 * (it & 1u), (it >> 1) & 1u, p.status, ST_TIMEOUT_FULL, 424)) { ok = false; break; }
      const float lse2 = stat[row];
      const Pair minus_lse2 = make_pair(-lse2, -lse2);
      float delta = t.measure ? 0.0f : stat[kBlk + row];
      Pair minus_delta = make_pair(-delta, -delta);
      // for the second kernel: -delta, and the log-sum-exp as it enters S (with a cap: as it is subtracted from y)
      const int64_t tile = ((static_cast<int64_t>(t.b) * p.q_heads + t.h) * p.seq_pad + t.q0) * 32;
      auto leave = [&]() {
        warp_arrive(BAR(stat_empty) + 8 * (it & 1u));
        if (half != 0) store_constant(p.delta + tile, row, -delta);
        else if (kCap) *reinterpret_cast<float*>(p.lse2 + tile / 8 + row * 4) = -lse2;
        else store_constant(p.lse2 + tile, row, -lse2 * p.inv_scale_log2);
      };
      if (!t.measure) leave();
      const int from = t.steps - t.blocks;
      Pair sum = make_pair(0.0f, 0.0f);
      for (int j = 0; j < t.steps; ++j, ++blk) {
        const int key0 = (t.first + (j < from ? j : j - from)) * kBlk + half * 64;
        const uint32_t s_addr = t_s + (blk & 1u) * 128 + lane_addr + half * 64;
        if (!warp_wait(BAR(s_full) + 8 * (blk & 1u), (blk >> 1) & 1u, p.status, ST_TIMEOUT_TMEM_FULL, 420)) { ok = false; break; }
        tc_fence_after();
        const int hi = live ? q_pos - key0 + 1 : 0;      // visible keys of this row: [lo, hi) of the 64
        const int lo = p.window > 0 ? q_pos - key0 - p.window + 1 : 0;
        const bool masked = __any_sync(kFullMask, hi < 64 || lo > 0);
        Pair pr[32];
        uint32_t v[32], u[32], pk[32];
        tc_ld_32x32b_x32(s_addr, v);
        tc_ld_32x32b_x32(s_addr + 32, u);
        tc_wait_ld();
        auto probabilities = [&](auto small) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            Pair slope;
            pr[i] = probability<kCap>(i < 16 ? make_pair(v[(2 * i) & 31], v[(2 * i + 1) & 31]) : make_pair(u[(2 * i) & 31], u[(2 * i + 1) & 31]),
                                      minus_lse2, p, decltype(small)::value, slope);
            if (kCap && j >= from) pr[i] = mul2(pr[i], slope);
          }
        };
        if (!kCap || all_small(v, u, p)) probabilities(TrueTag{});
        else probabilities(FalseTag{});
        if (!warp_wait(BAR(dp_full), blk & 1u, p.status, ST_TIMEOUT_TMEM_FULL, 421)) { ok = false; break; }
        tc_fence_after();
        tc_ld_32x32b_x32(t_dp + lane_addr + half * 64, v);
        tc_ld_32x32b_x32(t_dp + lane_addr + half * 64 + 32, u);
        tc_wait_ld();
        tc_fence_before();
        warp_arrive(BAR(dp_read));
        auto dp = [&](int i) { return i < 16 ? make_pair(v[(2 * i) & 31], v[(2 * i + 1) & 31]) : make_pair(u[(2 * i) & 31], u[(2 * i + 1) & 31]); };
        if (j < from) {                            // the first time over: the row's sum of P dP
#pragma unroll
          for (int i = 0; i < 32; ++i) sum = add2(sum, keep_range(mul2(pr[i], dp(i)), 2 * i, lo, hi));
          warp_arrive(BAR(ds_full) + 8 * (blk & 1u));
          if (j == from - 1) {                     // the two halves of the row
            float a, b;
            split(sum, a, b);
            (half == 0 ? stat + kBlk : red)[row] = a + b;
            warp_arrive(BAR(red));
            if (!warp_wait(BAR(red), measured & 1u, p.status, ST_TIMEOUT_FULL, 423)) { ok = false; break; }
            ++measured;
            delta = stat[kBlk + row] + red[row];
            minus_delta = make_pair(-delta, -delta);
            leave();
          }
          continue;
        }
        // one branch per tile: the tests of a masked tile cost as much as the arithmetic
        auto gradients = [&](auto m) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            Pair d = mul2(pr[i], add2(dp(i), minus_delta));
            if (decltype(m)::value) d = keep_range(d, 2 * i, lo, hi);
            pk[i] = pack_bf16(d);
          }
        };
        if (masked) gradients(TrueTag{});
        else gradients(FalseTag{});
        tc_st_32x32b_x32(s_addr, pk);
        tc_wait_st();
        tc_fence_before();
        warp_arrive(BAR(ds_full) + 8 * (blk & 1u));
      }
      if (!ok) break;
      if (!warp_wait(BAR(dq_full), it & 1u, p.status, ST_TIMEOUT_TMEM_FULL, 422)) { ok = false; break; }
      tc_fence_after();
      uint32_t a[32], b[32];
      tc_ld_32x32b_x32(t_dq + lane_addr + half * 64, a);
      tc_ld_32x32b_x32(t_dq + lane_addr + half * 64 + 32, b);
      tc_wait_ld();
      tc_fence_before();
      warp_arrive(BAR(dq_free));
      ++it;
      const int row0 = t.q0 + quad * 32;
      store_half_rows(a, b, p.scale, p.dq + ((static_cast<size_t>(t.b) * p.seq + row0) * p.q_heads + t.h) * kD + half * 64,
                      static_cast<int64_t>(p.q_heads) * kD, p.seq - row0);
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
                          const __grid_constant__ AttnBwdParams p, const __grid_constant__ Runs runs) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sb = smem_u32(smem);
  if ((sb & 1023u) != 0) {          // the swizzle pattern repeats every 1024 bytes
    if (threadIdx.x == 0 && p.status != nullptr) report_failure(p.status, ST_BAD_ARGUMENT, 499, sb, 1024);
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
    mbar_init(BAR(s_full), 1);
    mbar_init(BAR(p_full), kComputeWarps);
    mbar_init(BAR(p_full) + 8, kComputeWarps);
    mbar_init(BAR(dp_full), 1);
    mbar_init(BAR(ds_full), kComputeWarps);
    mbar_init(BAR(acc_full), 1);
    mbar_init(BAR(acc_free), kComputeWarps);
    mbar_init(BAR(drain), 1);
    fence_mbar_init();
    prefetch_tensormap(&map_q);
    prefetch_tensormap(&map_do);
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  for (int i = threadIdx.x; i < kAuxBytes / 4; i += kBwdThreads) reinterpret_cast<uint32_t*>(smem + kKvOnes)[i] = 0x3F803F80u;
  fence_proxy_async_smem();
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
    KvWalk walk;
    for (bool go = walk.begin(p, runs, items); go && ok; go = walk.next(p)) {
      const KvItem& t = walk.t;
      if (!warp_wait(BAR(kv_empty), (it & 1u) ^ 1u, p.status, ST_TIMEOUT_EMPTY, 430)) { ok = false; break; }
      if (elect_one_sync()) {
        mbar_arrive_expect_tx(BAR(kv_full), 2 * kTileBytes);
        load_tile(sb, &map_k, BAR(kv_full), t.h * kD, t.k0, t.b);
        load_tile(sb + kTileBytes, &map_v, BAR(kv_full), t.h * kD, t.k0, t.b);
      }
      __syncwarp();
      ++it;
      if (it == 1) wait_for_first();     // K and V are on their way; the queries' constants are the first kernel's
      int g = walk.i0 / t.tiles, qt = walk.i0 % t.tiles;
      for (int i = walk.i0; i < walk.i1; ++i, ++n) {
        const int h = t.h * p.group + g, row = (t.first + qt) * kBlk;
        const uint32_t qs = n % kKvQStages, ds = n % kKvDoStages;
        const uint32_t q_dst = sb + kKvQ + qs * kKvStage, do_dst = sb + kKvDo + ds * kKvStage;
        const int64_t at = ((static_cast<int64_t>(t.b) * p.q_heads + h) * p.seq_pad + row) * 32;
        if (!warp_wait(BAR(q_empty) + 8 * qs, ((n / kKvQStages) & 1u) ^ 1u, p.status, ST_TIMEOUT_EMPTY, 431)) { ok = false; break; }
        if (elect_one_sync()) {
          constexpr int kLseBytes = kCap ? kBlk * 4 : kAuxBytes;
          mbar_arrive_expect_tx(BAR(q_full) + 8 * qs, kTileBytes + kLseBytes);
          load_tile(q_dst, &map_q, BAR(q_full) + 8 * qs, h * kD, row, t.b);
          bulk_load(q_dst + kTileBytes, p.lse2 + (kCap ? at / 8 : at), kLseBytes, BAR(q_full) + 8 * qs);
        }
        __syncwarp();
        if (!warp_wait(BAR(do_empty) + 8 * ds, ((n / kKvDoStages) & 1u) ^ 1u, p.status, ST_TIMEOUT_EMPTY, 433)) { ok = false; break; }
        if (elect_one_sync()) {
          mbar_arrive_expect_tx(BAR(do_full) + 8 * ds, kTileBytes + kAuxBytes);
          load_tile(do_dst, &map_do, BAR(do_full) + 8 * ds, h * kD, row, t.b);
          bulk_load(do_dst + kTileBytes, p.delta + at, kAuxBytes, BAR(do_full) + 8 * ds);
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
      const uint32_t q = sb + kKvQ + qs * kKvStage;
      mma_tiles(t_s, sb, q, BAR(s_full), sb + kKvOnes, kCap ? 0 : q + kTileBytes);
      return true;
    };
    auto issue_dp = [&](uint32_t i) {
      const uint32_t ds = i % kKvDoStages;
      if (!warp_wait(BAR(do_full) + 8 * ds, (i / kKvDoStages) & 1u, p.status, ST_TIMEOUT_FULL, 441)) return false;
      tc_fence_after();
      const uint32_t g = sb + kKvDo + ds * kKvStage;
      mma_tiles(t_dp, sb + kTileBytes, g, BAR(dp_full), sb + kKvOnes, g + kTileBytes);
      return true;
    };
    KvWalk walk;
    for (bool go = walk.begin(p, runs, items); go && ok; go = walk.next(p)) {
      const int steps = __shfl_sync(kFullMask, walk.i1 - walk.i0, 0);
      if (!warp_wait(BAR(kv_full), it & 1u, p.status, ST_TIMEOUT_FULL, 442)) { ok = false; break; }
      tc_fence_after();
      // dV(i), S(i+1), dK(i), dP(i+1), from one copy of each product's code
      --n;
#pragma unroll 1
      for (int i = -1; i < steps; ++i, ++n) {
        const bool more = i + 1 < steps;
        const uint32_t qs = n % kKvQStages, ds = n % kKvDoStages;
        if (i >= 0) {
          if (!warp_wait(BAR(p_full), n & 1u, p.status, ST_TIMEOUT_FULL, 443)) { ok = false; break; }
          if (i == 0 && !warp_wait(BAR(acc_free), (it & 1u) ^ 1u, p.status, ST_TIMEOUT_TMEM_EMPTY, 444)) { ok = false; break; }
          tc_fence_after();
          // dV's product starts on the half of P that is ready first
          mma_from_tmem(t_dv, t_s, sb + kKvDo + ds * kKvStage, i != 0, 0, true, 0);
          if (!warp_wait(BAR(p_full) + 8, n & 1u, p.status, ST_TIMEOUT_FULL, 446)) { ok = false; break; }
          tc_fence_after();
          mma_from_tmem(t_dv, t_s, sb + kKvDo + ds * kKvStage, true, BAR(do_empty) + 8 * ds, true, 2);
        }
        if (more && !issue_s(n + 1)) { ok = false; break; }
        if (i >= 0) {
          if (!warp_wait(BAR(ds_full), n & 1u, p.status, ST_TIMEOUT_FULL, 445)) { ok = false; break; }
          tc_fence_after();
          mma_from_tmem(t_dk, t_dp, sb + kKvQ + qs * kKvStage, i != 0, BAR(q_empty) + 8 * qs);
        }
        if (more && !issue_dp(n + 1)) { ok = false; break; }
        if (i + 2 == steps) warp_commit(BAR(kv_empty));      // the last products that read K and V are issued: both may be replaced
      }
      if (!ok) break;
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
    KvWalk walk;
    for (bool go = walk.begin(p, runs, items); go && ok; go = walk.next(p)) {
      const KvItem& t = walk.t;
      const int k_pos = t.k0 + row;
      int qt = walk.i0 % t.tiles;
      for (int i = walk.i0; i < walk.i1; ++i, ++n) {
        const int q0 = (t.first + qt) * kBlk + half * 64;
        if (++qt == t.tiles) qt = 0;
        // visible queries of this key: [lo, hi) of the 64
        const int lo = k_pos - q0;
        const int hi = min(p.seq - q0, p.window > 0 ? min(lo, 64) + p.window : 64);
        const bool masked = __any_sync(kFullMask, lo > 0 || hi < 64);
        const uint32_t qs = n % kKvQStages;
        const float4* lse2 = reinterpret_cast<const float4*>(smem + kKvQ + qs * kKvStage + kTileBytes + half * 256);
        if (kCap && !warp_wait(BAR(q_full) + 8 * qs, (n / kKvQStages) & 1u, p.status, ST_TIMEOUT_FULL, 450)) { ok = false; break; }
        if (!warp_wait(BAR(s_full), n & 1u, p.status, ST_TIMEOUT_TMEM_FULL, 451)) { ok = false; break; }
        tc_fence_after();
        Pair pr[32];
        uint32_t v[32], u[32], pk[32];
        // one branch per tile: the tests of a masked tile cost as much as the arithmetic
        auto raw = [&](int i) { return i < 16 ? make_pair(v[(2 * i) & 31], v[(2 * i + 1) & 31]) : make_pair(u[(2 * i) & 31], u[(2 * i + 1) & 31]); };
        auto probabilities = [&](auto m, auto small, int from) {
#pragma unroll
          for (int i = from; i < from + 16; ++i) {
            Pair slope;
            if (kCap) {
              const float4 l = lse2[i >> 1];
              pr[i] = probability<true>(raw(i), i & 1 ? make_pair(l.z, l.w) : make_pair(l.x, l.y), p, decltype(small)::value, slope);
            } else {
              pr[i] = exp2_pair(mul2(raw(i), make_pair(p.scale_log2, p.scale_log2)));     // the log-sum-exp is in S already
            }
            if (decltype(m)::value) pr[i] = keep_range(pr[i], 2 * i, lo, hi);
            pk[i] = pack_bf16(pr[i]);
            if (kCap) pr[i] = mul2(pr[i], slope);
          }
        };
        tc_ld_32x32b_x32(s_addr, v);
        tc_ld_32x32b_x32(s_addr + 32, u);
        tc_wait_ld();
        const bool small = !kCap || all_small(v, u, p);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (!small) probabilities(TrueTag{}, FalseTag{}, 16 * c);          // rare: masked or not
          else if (masked) probabilities(TrueTag{}, TrueTag{}, 16 * c);
          else probabilities(FalseTag{}, TrueTag{}, 16 * c);
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = pk[16 * c + i];
          tc_st_32x32b_x16(s_addr + 16 * c, w);
          tc_wait_st();
          tc_fence_before();
          warp_arrive(BAR(p_full) + 8 * c);
        }
        if (!warp_wait(BAR(dp_full), n & 1u, p.status, ST_TIMEOUT_TMEM_FULL, 452)) { ok = false; break; }
        tc_fence_after();
        tc_ld_32x32b_x32(dp_addr, v);
        tc_ld_32x32b_x32(dp_addr + 32, u);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) pk[i] = pack_bf16(mul2(pr[i], raw(i)));      // delta is in dP already, masked places are 0 in pr
        tc_st_32x32b_x32(dp_addr, pk);
        tc_wait_st();
        tc_fence_before();
        warp_arrive(BAR(ds_full));
      }
      if (!ok) break;
      if (!warp_wait(BAR(acc_full), it & 1u, p.status, ST_TIMEOUT_TMEM_FULL, 453)) { ok = false; break; }
      tc_fence_after();
      // dV, then dK: of a whole tile, or a part's fp32 sums for the joining kernel, 4 columns of all rows together. One
      // copy of the code for both, as it is fetched for the first time where nothing else is left to do.
      const bool all = walk.i0 == 0 && walk.i1 == t.n;
      const int row0 = t.k0 + quad * 32;
      const size_t at = ((static_cast<size_t>(t.b) * p.seq + row0) * p.kv_heads + t.h) * kD + half * 64;
      float4* part = p.partial + (2 * static_cast<size_t>(blockIdx.x) + (walk.i0 == 0 ? 1 : 0)) * kPartVecs + half * 16 * kBlk + row;
#pragma unroll 1
      for (int m = 0; m < 2; ++m) {
        uint32_t a[32], b[32];
        tc_ld_32x32b_x32(t_dv + m * 128 + lane_addr + half * 64, a);
        tc_ld_32x32b_x32(t_dv + m * 128 + lane_addr + half * 64 + 32, b);
        tc_wait_ld();
        if (m == 1) {
          tc_fence_before();
          warp_arrive(BAR(acc_free));
        }
        if (all) store_half_rows(a, b, m == 1 ? p.scale : 1.0f, (m == 1 ? p.dk : p.dv) + at, static_cast<int64_t>(p.kv_heads) * kD, p.seq - row0);
        else store_part(a, b, part + m * (kPartVecs / 2));
      }
      ++it;
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

// Tiles that more than one run worked on: block (c, y) takes the tile whose first cut is where run c begins, and an
// eighth of its columns; the parts are added in the order of their runs.
__global__ void __launch_bounds__(256)
attention_bwd_join_kernel(const __grid_constant__ AttnBwdParams p, const __grid_constant__ Runs runs) {
  const int c = blockIdx.x + 1, w = runs.w[c];
  if (runs.step[c] == 0 || (runs.w[c - 1] == w && runs.step[c - 1] > 0)) return;     // no cut, or not the tile's first
  const KvItem t = kv_item(p, w);
  int last = c;                                              // the last run with steps of this tile
  while (runs.w[last + 1] == w) ++last;
  const int row = threadIdx.x & (kBlk - 1);
  if (t.k0 + row >= p.seq) return;
  // 64 column groups of 4 (dV, dK) over 8 blocks and two halves of the CTA: 4 a thread, stored in pairs
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int group = blockIdx.y * 8 + (threadIdx.x >> 7) * 4 + k * 2;
    float s[8];
    const float4* part = p.partial + (2 * static_cast<size_t>(c - 1) + 1) * kPartVecs + group * kBlk + row;
    float4 u = part[0], v = part[kBlk];
    s[0] = u.x; s[1] = u.y; s[2] = u.z; s[3] = u.w; s[4] = v.x; s[5] = v.y; s[6] = v.z; s[7] = v.w;
    for (int r = c; r <= last; ++r) {
      part = p.partial + 2 * static_cast<size_t>(r) * kPartVecs + group * kBlk + row;
      u = part[0];
      v = part[kBlk];
      s[0] += u.x; s[1] += u.y; s[2] += u.z; s[3] += u.w; s[4] += v.x; s[5] += v.y; s[6] += v.z; s[7] += v.w;
    }
    const bool dk = group >= 32;
    const float scale = dk ? p.scale : 1.0f;
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const __nv_bfloat162 x = __floats2bfloat162_rn(s[2 * e] * scale, s[2 * e + 1] * scale);
      o[e] = *reinterpret_cast<const uint32_t*>(&x);
    }
    __nv_bfloat16* dst = (dk ? p.dk : p.dv) + ((static_cast<size_t>(t.b) * p.seq + t.k0 + row) * p.kv_heads + t.h) * kD + (group & 31) * 4;
    *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// How the second kernel shares its work out. Whole tiles to CTAs leave SMs idle when there are few tiles (causal
// tiles differ in length by their number) or the last wave is short; equal runs of steps leave none idle and cost
// the parts' fp32 sums and the joining kernel, about ten steps' time and an eighth of what is shared out. Both kernels
// together, whole and in runs: 2048 positions of 32 / 8 heads 145 and 110 us, 1024 of 8 / 1 heads 106 and 36 us, 4096 of
// 32 / 8 heads 361 and 369 us.
constexpr int kLeastSteps = 4;        // of a run: 512 positions of 8 / 2 heads take 26.9 us with 6, 25.5 with 4, 25.1 with 3
Runs kv_runs(int batch, int seq, int kv_heads, int group, int window) {
  const int tiles = (seq + kBlk - 1) / kBlk, bh = batch * kv_heads;
  auto length = [&](int kb) { return static_cast<int64_t>(kv_query_tiles(tiles, window, kb)) * group + kTileSteps; };
  int64_t steps = 0;
  for (int kb = 0; kb < tiles; ++kb) steps += length(kb);
  steps *= bh;
  Runs runs;
  runs.count = 0;
  const int64_t items = static_cast<int64_t>(tiles) * bh, longest = length(0);
  const int64_t even = steps / kBwdRuns, waves = (items + kBwdRuns - 1) / kBwdRuns;
  int64_t whole = even + longest / 8;
  if (whole < longest) whole = longest;
  if (window > 0 && whole < waves * steps / items) whole = waves * steps / items;      // tiles of about the same length
  if (whole <= even + even / 8 + 10 || steps < 2 * kLeastSteps) return runs;
  runs.count = static_cast<int>(steps / kLeastSteps < kBwdRuns ? steps / kLeastSteps : kBwdRuns);
  int64_t before = 0;                                        // where tile row kb begins
  int r = 0;
  for (int kb = 0; kb < tiles; ++kb) {
    const int64_t n = length(kb);
    for (; r < runs.count; ++r) {
      const int64_t at = steps * r / runs.count - before;
      if (at >= n * bh) break;
      const int64_t step = at % n - kTileSteps;
      runs.w[r] = kb * bh + static_cast<int>(at / n);
      runs.step[r] = step > 0 ? static_cast<int>(step) : 0;
    }
    before += n * bh;
  }
  runs.w[r] = static_cast<int>(items);
  runs.step[r] = 0;
  return runs;
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

size_t attention_bwd_workspace_bytes(int batch, int seq, int q_heads, int kv_heads, int window) {
  const size_t rows = static_cast<size_t>(batch) * q_heads * ((static_cast<size_t>(seq) + kBlk - 1) / kBlk * kBlk);
  const Runs runs = kv_runs(batch, seq, kv_heads, q_heads / kv_heads, window < seq ? window : 0);
  return 2 * rows * 32 + static_cast<size_t>(runs.count) * 2 * kPartVecs * sizeof(float4);
}

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
  p.lse2 = static_cast<uint8_t*>(a.workspace);
  p.delta = p.lse2 + static_cast<int64_t>(a.batch) * a.q_heads * p.seq_pad * 32;
  p.partial = reinterpret_cast<float4*>(p.delta + static_cast<int64_t>(a.batch) * a.q_heads * p.seq_pad * 32);
  const Runs runs = kv_runs(a.batch, a.seq, a.kv_heads, p.group, p.window);
  p.scale = a.scale;
  p.scale_log2 = a.scale * kLog2e;
  p.inv_scale_log2 = 1.0f / p.scale_log2;
  const bool cap = a.softcap > 0.0f;
  p.cap_in = cap ? a.scale / a.softcap : 0.0f;
  p.cap_out = a.softcap * kLog2e;
  p.status = a.status;
  const int64_t q_items = static_cast<int64_t>(p.tiles) * a.batch * a.q_heads;
  const int64_t kv_items = static_cast<int64_t>(p.tiles) * a.batch * a.kv_heads;
  auto dq = cap ? attention_bwd_dq_kernel<true> : attention_bwd_dq_kernel<false>;
  auto dkdv = cap ? attention_bwd_dkdv_kernel<true> : attention_bwd_dkdv_kernel<false>;
  // shared-memory limits of the two kernels, once per device
  static std::atomic<bool> ready[2][64];
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) return err;
  if (device >= 64 || !ready[cap][device].load(std::memory_order_relaxed)) {
    err = cudaFuncSetAttribute(dq, cudaFuncAttributeMaxDynamicSharedMemorySize, kDqSmem);
    if (err != cudaSuccess) return err;
    err = cudaFuncSetAttribute(dkdv, cudaFuncAttributeMaxDynamicSharedMemorySize, kKvSmem);
    if (err != cudaSuccess) return err;
    if (device < 64) ready[cap][device].store(true, std::memory_order_relaxed);
  }
  dq<<<static_cast<int>(q_items < a.num_sms ? q_items : a.num_sms), kBwdThreads, kDqSmem, stream>>>(mq, mdo, mk, mv, p);
  err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  const int grid = runs.count > 0 ? runs.count : static_cast<int>(kv_items < a.num_sms ? kv_items : a.num_sms);
  // a launch that may begin while the one before it ends
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(kBwdThreads);
  config.dynamicSmemBytes = kKvSmem;
  config.stream = stream;
  config.attrs = &early;
  config.numAttrs = 1;
  err = cudaLaunchKernelEx(&config, dkdv, mq, mdo, mk, mv, p, runs);
  if (err != cudaSuccess || runs.count < 2) return err;
  // launched the same way the joining kernel's blocks get in the way of the last runs (2048 positions: 127 -> 131 us)
  attention_bwd_join_kernel<<<dim3(runs.count - 1, 8), 256, 0, stream>>>(p, runs);
  return cudaGetLastError();
}

}  // namespace plb
