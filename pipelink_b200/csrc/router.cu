// Routing of tokens to experts, and the gradient of the weights.
//
//   s = softmax(x) or sigmoid(x)        choice c = s + bias, masked experts (x = -inf) -inf
//   group score = max of c or the sum of its two best unmasked c; the topk_groups best groups are kept
//   the topk best c of the kept groups, ties to the lowest index; w = scale * s [/ sum of the chosen s]
//   dS_j = scale / S * (g_j - sum_i g_i s_i / S) or scale * g_j;  dx = s (dS - sum s dS) or dS s (1 - s)
//
// One warp per token, NV consecutive experts to a lane. The topk-th largest of the 32 lanes' maxima bounds the topk-th
// value from below: what is not under it, some 10 to 20 candidates, is put one to a lane and ranked by comparing each
// with each (16384 tokens, 256 experts, 8 chosen: 11.6 us; rounds of maxima took 7 us more). Where that leaves
// more than 32 (many ties, a large topk), topk rounds of a warp-wide maximum choose. Without a bias the scores are
// ordered as the logits are, and those are compared as they stand. With one (or with sums of two scores over groups) the
// order is that of numbers fp32 may not tell apart. Every comparison that matters is checked against the bound of the
// fp32 scores' error; candidates closer than that are put in order by their fp64 values (some 2 tokens of 1000 at 256
// experts).
#include <math.h>

#include <type_traits>

#include "kernels.h"

namespace plb {

namespace {

constexpr int kRouteWarps = 4;
constexpr uint32_t kAll = 0xFFFFFFFFu;
constexpr int kMostRanked = 16;       // topk up to which the lanes' maxima leave few candidates

// A warp's shared memory: a word per expert and 32 more, in 16-byte pieces.
__host__ __device__ constexpr int scratch_words(int experts) { return (experts + 33) & ~1; }

__device__ __forceinline__ float load_logit(const void* p, int64_t i, bool bf16) {
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i];
}
// A lane's NV consecutive logits (of the row at index `row`); past the experts -inf. Whole rows in 16-byte pieces where
// `wide`: row starts and lengths are multiples of a lane's share.
template <int NV>
__device__ __forceinline__ void load_logits(const void* p, int64_t row, int experts, bool bf16, bool wide, float (&x)[NV]) {
  const int first = (threadIdx.x & 31) * NV;
#pragma unroll
  for (int i = 0; i < NV; ++i) x[i] = -INFINITY;
  if (first >= experts) return;
  if (!wide) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (first + i < experts) x[i] = load_logit(p, row + first + i, bf16);
  } else if (bf16) {
    const uint32_t* q = reinterpret_cast<const uint32_t*>(static_cast<const __nv_bfloat16*>(p) + row + first);
    uint32_t w[NV / 2];
    if constexpr (NV == 2) w[0] = *q;
    else if constexpr (NV == 4) { const uint2 v = *reinterpret_cast<const uint2*>(q); w[0] = v.x; w[1] = v.y; }
    else {
#pragma unroll
      for (int i = 0; i < NV / 8; ++i) {
        const uint4 v = reinterpret_cast<const uint4*>(q)[i];
        w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
      }
    }
#pragma unroll
    for (int i = 0; i < NV / 2; ++i) { x[2 * i] = bf16_lo(w[i]); x[2 * i + 1] = bf16_hi(w[i]); }
  } else {
    const float* q = static_cast<const float*>(p) + row + first;
    if constexpr (NV == 2) { const float2 v = *reinterpret_cast<const float2*>(q); x[0] = v.x; x[1] = v.y; }
    else {
#pragma unroll
      for (int i = 0; i < NV / 4; ++i) {
        const float4 v = reinterpret_cast<const float4*>(q)[i];
        x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
      }
    }
  }
}
// Sigmoid for a choice, whose error the comparisons allow for (see slack); weights are computed with expf.
__device__ __forceinline__ float choice_sigmoid(float x) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.4426950408889634f));
  return __fdividef(1.0f, 1.0f + e);
}
// Unsigned integers in the order of the numbers; NaN below every number, 0 is left for "not a candidate".
__device__ __forceinline__ uint64_t order_key(double v) {
  if (v != v) return 1;
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v == 0.0 ? 0.0 : v));
  return (b >> 63) ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);            // -0 becomes 0
  return v != v ? 1u : b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {   // the number of a key that is one
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
template <class T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
template <class T>
__device__ __forceinline__ T warp_max(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const T u = __shfl_xor_sync(kAll, v, o);
    v = u > v ? u : v;
  }
  return v;
}

// Below this sum the scores of the chosen are not divided by it: they come near the end of fp32's range, or are past it,
// where their ratios still are of order 1. Ratios of scores are then taken from the logits, exp(x - m) with m the
// largest chosen one (a sigmoid's 1 + exp(x) is 1 there). Above it a score that underflows is under 2^-86 of the sum.
// Scores of exp(-700) and less, next to nothing in 64 bits too, are 0: a type's lowest number as a logit masks.
constexpr float kFarSum = 0x1p-40f, kNoScore = -700.0f;
// The slots' shares of their sum, from their logits and the logarithms of their scores (lane j: slot j, `in` or 0).
__device__ __forceinline__ float far_shares(float x, float log_score, bool in) {
  in = in && log_score > kNoScore;
  const float m = warp_max(in ? x : -INFINITY);
  if (m == -INFINITY) return 0.0f;
  const float t = in ? expf(x - m) : 0.0f;
  return t / warp_sum(t);
}

// Scaled weights of the chosen (lane j: slot j) with their logits x and scores; top: what a softmax's logits are taken from.
__device__ __forceinline__ void store_choice(const RouteArgs& a, int64_t token, int lane, int pick, float x, float top, float weight) {
  if (a.renormalize) {
    const float total = warp_sum(lane < a.topk ? weight : 0.0f);
    weight = total < kFarSum ? far_shares(x, a.sigmoid ? x : x - top, lane < a.topk) : __fdividef(weight, total);
  }
  if (lane < a.topk) {
    a.experts_out[token * a.topk + lane] = pick;
    a.weights_out[token * a.topk + lane] = weight * a.scale;
  }
}

// A token's scores in fp64.
struct ExactScores {
  const RouteArgs& a;
  int64_t token;
  double top, sum;
  __device__ __forceinline__ ExactScores(const RouteArgs& args, int64_t t) : a(args), token(t), top(0.0), sum(1.0) {
    if (a.sigmoid) return;
    const int lane = threadIdx.x & 31;
    top = -INFINITY;
    for (int e = lane; e < a.experts; e += 32) top = fmax(top, logit(e));
    top = warp_max(top);
    if (top == -INFINITY) top = 0.0;
    sum = 0.0;
    for (int e = lane; e < a.experts; e += 32) sum += exp(logit(e) - top);
    sum = warp_sum(sum);
  }
  __device__ __forceinline__ double logit(int e) const { return static_cast<double>(load_logit(a.logits, token * a.ld_logits + e, a.bf16)); }
  __device__ __forceinline__ double score(double x) const { return a.sigmoid ? 1.0 / (1.0 + exp(-x)) : sum == 0.0 ? 0.0 : exp(x - top) / sum; }
  __device__ __forceinline__ double choice(int e) const {
    const double x = logit(e);
    return x == -INFINITY ? x : a.bias != nullptr ? score(x) + static_cast<double>(a.bias[e]) : score(x);
  }
};

// The groups a token keeps (bit g * group_share: group g), from fp64 scores. `choice`: the warp's shared memory, a word per expert.
__device__ __noinline__ uint32_t exact_groups(const RouteArgs& a, int64_t token, double* choice) {
  const int lane = threadIdx.x & 31, size = a.experts / a.groups;
  const ExactScores s(a, token);
  __syncwarp();
  for (int e = lane; e < a.experts; e += 32) choice[e] = s.choice(e);
  __syncwarp();
  double first = -INFINITY, second = -INFINITY;
  if (lane < a.groups)
    for (int e = lane * size; e < (lane + 1) * size; ++e) {
      const double c = choice[e];
      if (c > first) { second = first; first = c; }
      else if (c > second) second = c;
    }
  const uint64_t mine = order_key(a.group_top2 && second > -INFINITY ? first + second : first);
  int better = 0;
  for (int g = 0; g < a.groups; ++g) {
    const uint64_t other = __shfl_sync(kAll, mine, g);
    better += other > mine || (other == mine && g < lane);
  }
  __syncwarp();
  const uint32_t groups = __ballot_sync(kAll, lane < a.groups && better < a.topk_groups);
  uint32_t kept = 0;
  for (int g = 0; g < a.groups; ++g) kept |= ((groups >> g) & 1u) << (g * a.group_share);
  return kept;
}

// Lanes 0 .. count - 1 hold candidates, among them all that may be chosen: in their order by fp64 choice values.
__device__ __noinline__ int exact_order(const RouteArgs& a, int64_t token, int pick, int count) {
  const int lane = threadIdx.x & 31;
  const ExactScores s(a, token);
  const uint64_t mine = lane < count ? order_key(s.choice(pick)) : 0;
  int rank = 0;
  for (int i = 0; i < count; ++i) {
    const uint64_t other = __shfl_sync(kAll, mine, i);
    const int e = __shfl_sync(kAll, pick, i);
    rank += other > mine || (other == mine && e < pick);
  }
  int at = 0;
  for (int i = 0; i < count; ++i) {
    const int r = __shfl_sync(kAll, rank, i), e = __shfl_sync(kAll, pick, i);
    if (r == lane) at = e;
  }
  return at;
}

// The whole choice in fp64, for more close candidates than a warp has lanes.
__device__ __noinline__ int exact_choice(const RouteArgs& a, int64_t token, uint32_t kept, uint64_t* key) {
  const int lane = threadIdx.x & 31, size = a.experts / a.groups;
  const ExactScores s(a, token);
  __syncwarp();
  for (int e = lane; e < a.experts; e += 32) key[e] = !((kept >> (a.groups > 1 ? e / size * a.group_share : 0)) & 1u) ? 0 : order_key(s.choice(e));
  __syncwarp();
  int pick = 0;
  for (int j = 0; j < a.topk; ++j) {
    uint64_t best = 0;
    int at = 0x7FFFFFFF;
    for (int e = lane; e < a.experts; e += 32)
      if (key[e] > best) { best = key[e]; at = e; }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t b = __shfl_xor_sync(kAll, best, o);
      const int e = __shfl_xor_sync(kAll, at, o);
      if (b > best || (b == best && e < at)) { best = b; at = e; }
    }
    if (lane == (at & 31)) key[at] = 0;
    if (lane == j) pick = at;
    __syncwarp();
  }
  return pick;
}

// kScored: the choice needs the scores, for a bias or the sums of two; without them no comparison is ever close, and the
// kernel has neither the tests nor the fp64 paths (65536 x 128: 37.7 us with them, 31.6 without).
//
// CTAs per SM: what hides the latencies of a token's steps is other tokens, at the price of registers where a lane
// holds few experts (256 experts in groups with a bias: 18.1 us with 40 warps an SM, 18.5 with 48; by logits alone 48 are
// as good or better).
template <int NV, bool kScored>
__global__ void __launch_bounds__(kRouteWarps * 32, NV <= 8 ? (kScored ? 10 : 12) : NV <= 16 ? 8 : 4)
route_topk_kernel(const __grid_constant__ RouteArgs a) {
  extern __shared__ __align__(16) uint64_t shared[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t token = static_cast<int64_t>(blockIdx.x) * kRouteWarps + warp;
  if (token >= a.tokens) return;
  uint64_t* scratch = shared + warp * scratch_words(a.experts);
  const int e0 = lane * NV;              // the lane's first expert
  float c[NV];                           // logits, then what a choice goes by
  uint32_t key[NV];
  float top = -INFINITY;
  load_logits<NV>(a.logits, token * a.ld_logits, a.experts, a.bf16, a.wide, c);
  const bool by_score = kScored && a.bias != nullptr;             // else by logits
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    key[i] = !by_score && e0 + i < a.experts ? order_key(c[i]) : 0;
    top = fmaxf(top, c[i]);
  }
  const bool by_sum = kScored && a.groups > 1 && a.group_top2;
  float inv_sum = 1.0f;
  if (!a.sigmoid) {
    top = warp_max(top);
    if (top == -INFINITY) top = 0.0f;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float e = expf(c[i] - top);
      sum += e;
      if (by_score || by_sum) c[i] = c[i] == -INFINITY ? -1.0f : e;      // a masked one stays known
    }
    sum = warp_sum(sum);
    inv_sum = sum == 0.0f ? 0.0f : __fdividef(1.0f, sum);
  }
  auto score = [&](float x) { return a.sigmoid ? __fdividef(1.0f, 1.0f + expf(-x)) : expf(x - top) * inv_sum; };
  // How far two fp32 choice values must lie apart to be in the order of the exact ones: twice the error of a score,
  // and the roundings of the sums (under 2^-23 of |c| + 1/4 each). A sigmoid is off by s (1 - s) times e's relative error
  // (2^-22 of exp2, and under 2^-23.7 |x| of its argument's roundings), by the sum's half step and the quotient's two steps:
  // with s (1 - s) at most 1/4, and |x| s (1 - s) 0.224, 2^-24 + 2^-25.8 + 2^-24 + 2^-22, twice that under 2^-20.3. A softmax by two steps of expf, the sum's NV + 5
  // roundings, six more, and half a step of |x - top|, which is largest against exp(top - x) at 1: under (NV + 16) 2^-23
  // of the largest.
  const float slack = a.sigmoid ? 1.1e-6f : (NV + 16) * 2.4e-7f * inv_sum;
  auto near = [&](float high, float low) { return high - low <= slack + 2.4e-7f * (fabsf(high) + 0.25f); };   // NaN and inf - inf: not near
  if (by_score || by_sum) {
    float bias[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) bias[i] = 0.0f;
    if (by_score) load_logits<NV>(a.bias, 0, a.experts, false, a.wide_bias, bias);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const bool masked = c[i] == (a.sigmoid ? -INFINITY : -1.0f);
      const float s = a.sigmoid ? choice_sigmoid(c[i]) : c[i] * inv_sum;
      c[i] = masked ? -INFINITY : s + bias[i];
      if (by_score) key[i] = e0 + i < a.experts ? order_key(c[i]) : 0;
    }
  }
  uint32_t kept = kAll;                                           // bit g * share: group g takes part
  if (a.groups > 1) {
    const int size = a.experts / a.groups, log_share = 31 - __clz(a.group_share), share = a.group_share;
    float first = -INFINITY, second = -INFINITY;
    auto take = [&](float v) {
      second = fmaxf(second, fminf(first, v));                    // fminf, fmaxf pass NaN over
      first = fmaxf(first, v);
    };
    const int g = lane >> log_share;
    if (share * NV == size) {                                     // a group is `share` lanes' registers
#pragma unroll
      for (int i = 0; i < NV; ++i) take(c[i]);
    } else {
      // `share` adjacent lanes look through a group in shared memory, where each group starts `share` words on, so that
      // the groups' lanes meet different banks
      float* choice = reinterpret_cast<float*>(scratch);
      const float inv_size = 1.0f / static_cast<float>(size);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = e0 + i;
        if (e < a.experts) choice[e + (static_cast<int>((static_cast<float>(e) + 0.5f) * inv_size) << log_share)] = c[i];
      }
      __syncwarp();
      if (g < a.groups)
        for (int e = lane & (share - 1); e < size; e += share) take(choice[g * (size + share) + e]);
    }
    for (int o = 1; o < share; o <<= 1) {
      const float f = __shfl_xor_sync(kAll, first, o), h = __shfl_xor_sync(kAll, second, o);
      second = fmaxf(fmaxf(second, h), fminf(first, f));
      first = fmaxf(first, f);
    }
    // a sum of two as half of it, which does not overflow where a bias is near the type's end
    if (by_sum) first = 0.5f * first + (second > -INFINITY ? 0.5f * second : 0.0f);
    const uint32_t mine = order_key(first);
    int better = 0;
    for (int h = 0; h < a.groups; ++h) {
      const uint32_t other = __shfl_sync(kAll, mine, h << log_share);
      better += other > mine || (other == mine && h < g);
    }
    const bool keep = g < a.groups && better < a.topk_groups;
    kept = __ballot_sync(kAll, keep);
    if (by_score || by_sum) {
      const uint32_t worst_kept = __reduce_min_sync(kAll, keep ? mine : 0xFFFFFFFFu);
      const uint32_t best_dropped = __reduce_max_sync(kAll, g < a.groups && !keep ? mine : 0u);
      // half a sum of two is off as much as one score
      if (near(key_value(worst_kept), key_value(best_dropped))) kept = exact_groups(a, token, reinterpret_cast<double*>(scratch));
    }
    if (share * NV == size) {
      if (!((kept >> (g << log_share)) & 1u))
#pragma unroll
        for (int i = 0; i < NV; ++i) key[i] = 0;
    } else {
      const float inv_size = 1.0f / static_cast<float>(size);
#pragma unroll
      for (int i = 0; i < NV; ++i) {        // (e + 1/2) / size is exact enough up to 1024
        const int of = static_cast<int>((static_cast<float>(e0 + i) + 0.5f) * inv_size);
        if (e0 + i < a.experts && !((kept >> (of << log_share)) & 1u)) key[i] = 0;
      }
    }
  }
  uint32_t best = 0;                       // the lane's best candidate
#pragma unroll
  for (int i = 0; i < NV; ++i) best = max(best, key[i]);
  int pick = 0;          // lane j: the j-th candidate, best first
  int count = 33;
  bool close = false;
  if (a.topk <= kMostRanked) {
    uint32_t bound = 0, v = best;
    for (int j = 0; j < a.topk; ++j) {                               // equal maxima go together, which only lowers the bound
      bound = __reduce_max_sync(kAll, v);
      if (v == bound) v = 0;
    }
    // with scores: also what may change places with a chosen one
    if (by_score && bound > 1u) {
      const float x = key_value(bound);
      const float low = x - (slack + 2.4e-7f * (fabsf(x) + 0.25f)) * 1.001f;
      if (low == low) bound = order_key(low);
    }
    if (bound == 0) bound = 1;
    uint32_t* list = reinterpret_cast<uint32_t*>(scratch);           // 32 keys, then their experts
    int mine_in = 0, n = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) mine_in += key[i] >= bound;
    int at = mine_in;                                                // where the lane's candidates go
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int before = __shfl_up_sync(kAll, at, o);
      if (lane >= o) at += before;
    }
    n = __shfl_sync(kAll, at, 31);
    if (n <= 32) {
      at -= mine_in;
      __syncwarp();
      list[lane] = 0;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (key[i] >= bound) {
          list[at] = key[i];
          list[32 + at] = e0 + i;
          ++at;
        }
      __syncwarp();
      // the list is in the order of the experts, so among equal keys the earlier place is the lower index
      const uint32_t mine = lane < n ? list[lane] : 0;
      const int e = lane < n ? list[32 + lane] : 0;
      int rank = 0;
      for (int j = 0; j < n; j += 4) {
        const uint4 other = *reinterpret_cast<const uint4*>(list + j);
        rank += other.x + (j < lane) > mine;                         // no key is 2^32 - 1
        rank += other.y + (j + 1 < lane) > mine;
        rank += other.z + (j + 2 < lane) > mine;
        rank += other.w + (j + 3 < lane) > mine;
      }
      __syncwarp();
      if (lane < n) {
        list[rank] = mine;
        list[32 + rank] = e;
      }
      __syncwarp();
      count = n;
      pick = lane < n ? list[32 + lane] : 0;
      if (by_score) {
        // neighbours that near are in order only if they are the same number: the same logit under the same bias
        const bool follows = lane > 0 && lane < n && lane <= a.topk && list[lane] > 1u && near(key_value(list[lane - 1]), key_value(list[lane]));
        bool differ = false;
        if (follows) {
          const int before = list[32 + lane - 1];
          differ = a.bias[pick] != a.bias[before] ||
                   load_logit(a.logits, token * a.ld_logits + pick, a.bf16) != load_logit(a.logits, token * a.ld_logits + before, a.bf16);
        }
        close = __any_sync(kAll, differ);
      }
    }
  }
  if (count > 32) {
    int slot = 0;          // of the lane's best, and the key chosen before with its expert
    uint32_t last = 0;
    int last_at = 0;
    auto look = [&]() {
      best = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (key[i] > best) { best = key[i]; slot = i; }
    };
    look();
    for (count = 0;; ++count) {
      const uint32_t m = __reduce_max_sync(kAll, best);
      // past topk as long as a candidate may still change places with a chosen one
      const bool follows = by_score && count > 0 && m > 1u && near(key_value(last), key_value(m));
      if (count >= a.topk && (!follows || count == 32)) {
        if (follows) count = 33;
        break;
      }
      const int at = __reduce_min_sync(kAll, best == m ? e0 + slot : 0x7FFFFFFF);
      if (follows)
        close = close || a.bias[at] != a.bias[last_at] ||
                load_logit(a.logits, token * a.ld_logits + at, a.bf16) != load_logit(a.logits, token * a.ld_logits + last_at, a.bf16);
      last = m;
      last_at = at;
      if (lane == at / NV) {
#pragma unroll
        for (int i = 0; i < NV; ++i) key[i] = at == e0 + i ? 0 : key[i];
        look();
      }
      if (lane == count) pick = at;
    }
  }
  if (count > 32) pick = exact_choice(a, token, kept, scratch);
  else if (close) pick = exact_order(a, token, pick, count);
  const float x = lane < a.topk ? load_logit(a.logits, token * a.ld_logits + pick, a.bf16) : 0.0f;
  store_choice(a, token, lane, pick, x, top, score(x));
}

template <int NV>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_topk_bwd_kernel(const __grid_constant__ RouteBwdArgs a) {
  extern __shared__ float ds_all[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t token = static_cast<int64_t>(blockIdx.x) * kRouteWarps + warp;
  if (token >= a.tokens) return;
  const int e0 = lane * NV;
  float s[NV];
  float top = -INFINITY;
  // lane j holds slot j: its expert, that expert's logit and the gradient of its weight
  const int at = lane < a.topk ? a.experts_in[token * a.topk + lane] : -1;
  const bool valid = at >= 0 && at < a.experts;
  float g = lane < a.topk ? a.d_weights[token * a.topk + lane] : 0.0f;
  load_logits<NV>(a.logits, token * a.ld_logits, a.experts, a.bf16, a.wide, s);
  const float x = valid ? load_logit(a.logits, token * a.ld_logits + at, a.bf16) : 0.0f;
  g = valid ? g * a.scale : 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) top = fmaxf(top, s[i]);
  top = warp_max(top);
  if (top == -INFINITY) top = 0.0f;
  float sum = 0.0f, inv_sum = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (a.sigmoid) {               // the slope s (1 - s), without the difference that cancels where s is near 1
      const float e = expf(-fabsf(s[i]));
      s[i] = __fdividef(e, (1.0f + e) * (1.0f + e));
    } else {
      s[i] = expf(s[i] - top);
      sum += s[i];
    }
  }
  if (!a.sigmoid) {
    sum = warp_sum(sum);
    inv_sum = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < NV; ++i) s[i] *= inv_sum;
  }
  float mine = 0.0f;                     // the score of the slot's expert
  if (valid) mine = a.sigmoid ? 1.0f / (1.0f + expf(-x)) : expf(x - top) * inv_sum;
  if (a.renormalize) {
    const float total = warp_sum(mine), inner = warp_sum(g * mine);
    if (total < kFarSum) {
      // dx_j = w_j (g_j - sum g w) from the shares themselves (times 1 - s for a sigmoid, which is 1), 0 for the others
      const float w = far_shares(x, a.sigmoid ? x : x - top, valid);
      g = w * (g - warp_sum(g * w));
      mine = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i) s[i] = s[i] * 0.0f + 1.0f;      // a NaN stays one
    } else {
      g = !valid ? 0.0f : (g - inner / total) / total;
    }
  }
  const float dot = a.sigmoid ? 0.0f : warp_sum(g * mine);
  // slots to experts, in the slots' order (an expert may be named twice, which the slots' numbers find out)
  float* ds = ds_all + warp * 32 * NV;
  int* tag = reinterpret_cast<int*>(ds);
  if (valid) tag[at] = lane;
  __syncwarp();
  const bool alone = __all_sync(kAll, !valid || tag[at] == lane);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < NV; ++i) ds[e0 + i] = 0.0f;
  __syncwarp();
  if (alone) {
    if (valid) ds[at] = g;
  } else {
    for (int j = 0; j < a.topk; ++j) {
      if (lane == j && valid) ds[at] += g;
      __syncwarp();
    }
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < NV; ++i) s[i] = a.sigmoid ? ds[e0 + i] * s[i] : s[i] * (ds[e0 + i] - dot);
  if (e0 >= a.experts) return;
  const int64_t out = token * a.experts + e0;
  if (a.bf16) {
    __nv_bfloat16* d = static_cast<__nv_bfloat16*>(a.d_logits) + out;
    if (a.wide_out) {
#pragma unroll
      for (int i = 0; i < NV / 2; ++i) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(s[2 * i], s[2 * i + 1]);
        reinterpret_cast<__nv_bfloat162*>(d)[i] = v;
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (e0 + i < a.experts) d[i] = __float2bfloat16_rn(s[i]);
    }
  } else {
    float* d = static_cast<float*>(a.d_logits) + out;
    if (a.wide_out) {
      if constexpr (NV == 2) *reinterpret_cast<float2*>(d) = make_float2(s[0], s[1]);
      else {
#pragma unroll
        for (int i = 0; i < NV / 4; ++i) reinterpret_cast<float4*>(d)[i] = make_float4(s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (e0 + i < a.experts) d[i] = s[i];
    }
  }
}

template <class F>
cudaError_t by_width(int experts, F&& f) {
  const int n = (experts + 31) / 32;
  if (n <= 2) f(std::integral_constant<int, 2>{});
  else if (n <= 4) f(std::integral_constant<int, 4>{});
  else if (n <= 8) f(std::integral_constant<int, 8>{});
  else if (n <= 16) f(std::integral_constant<int, 16>{});
  else if (n <= 32) f(std::integral_constant<int, 32>{});
  else return cudaErrorInvalidValue;
  return cudaGetLastError();
}

}  // namespace

// Rows of `experts` numbers from p on, `ld` apart, whose lanes' shares are whole, aligned pieces.
static bool whole_pieces(const void* p, int64_t ld, int experts, int nv, bool bf16) {
  const int bytes = nv * (bf16 ? 2 : 4);
  return experts % nv == 0 && ld % nv == 0 && reinterpret_cast<uintptr_t>(p) % (bytes < 16 ? bytes : 16) == 0;
}

cudaError_t launch_route_topk(const RouteArgs& args, cudaStream_t stream) {
  RouteArgs a = args;
  if (a.tokens == 0) return cudaSuccess;
  const unsigned grid = static_cast<unsigned>((a.tokens + kRouteWarps - 1) / kRouteWarps);
  return by_width(a.experts, [&](auto n) {
    constexpr int kNv = decltype(n)::value;
    a.wide = whole_pieces(a.logits, a.ld_logits, a.experts, kNv, a.bf16);
    a.wide_bias = whole_pieces(a.bias, 0, a.experts, kNv, false);
    auto kernel = a.bias != nullptr || (a.groups > 1 && a.group_top2) ? route_topk_kernel<kNv, true> : route_topk_kernel<kNv, false>;
    kernel<<<grid, kRouteWarps * 32, kRouteWarps * scratch_words(a.experts) * sizeof(uint64_t), stream>>>(a);
  });
}

cudaError_t launch_route_topk_bwd(const RouteBwdArgs& args, cudaStream_t stream) {
  RouteBwdArgs a = args;
  if (a.tokens == 0) return cudaSuccess;
  const unsigned grid = static_cast<unsigned>((a.tokens + kRouteWarps - 1) / kRouteWarps);
  return by_width(a.experts, [&](auto n) {
    constexpr int kNv = decltype(n)::value;
    a.wide = whole_pieces(a.logits, a.ld_logits, a.experts, kNv, a.bf16);
    a.wide_out = whole_pieces(a.d_logits, a.experts, a.experts, kNv, a.bf16);
    route_topk_bwd_kernel<kNv><<<grid, kRouteWarps * 32, kRouteWarps * 32 * kNv * sizeof(float), stream>>>(a);
  });
}

}  // namespace plb
