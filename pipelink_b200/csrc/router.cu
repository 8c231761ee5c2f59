// Routing of tokens to experts, and the gradient of the weights.
//
//   s = softmax(x) or sigmoid(x)        choice c = s + bias, masked experts (x = -inf) -inf
//   group score = max of c or the sum of its two best unmasked c; the topk_groups best groups are kept
//   the topk best c of the kept groups, ties to the lowest index; w = scale * s [/ sum of the chosen s]
//   dS_j = scale / S * (g_j - sum_i g_i s_i / S) or scale * g_j;  dx = s (dS - sum s dS) or dS s (1 - s)
//
// One warp per token, expert e in register e / 32 of lane e % 32. The topk-th largest of the 32 lanes' maxima bounds
// the topk-th value from below: what is not under it, some 10 to 20 candidates, is put one to a lane and ranked by
// comparing each with each (16384 tokens, 256 experts, 8 chosen: kRouteNote). Where that leaves more than 32 (many
// ties, a large topk), topk rounds of a warp-wide maximum choose. Without a bias the scores are ordered as the logits are, and those are compared as they
// stand. With one (or with sums of two scores over groups) the order is that of numbers fp32 may not tell apart.
// Every comparison that matters is checked against the bound of the fp32 scores' error; candidates closer than that
// are put in order by their fp64 values (some 2 tokens of 1000 at 256 experts).
#include <math.h>

#include <type_traits>

#include "kernels.h"

namespace plb {

namespace {

constexpr int kRouteWarps = 4;
constexpr uint32_t kAll = 0xFFFFFFFFu;
constexpr int kMostRanked = 16;       // topk up to which the lanes' maxima leave few candidates

__device__ __forceinline__ float load_logit(const void* p, int64_t i, bool bf16) {
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i];
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

// Scaled weights of the chosen (lane j: slot j).
__device__ __forceinline__ void store_choice(const RouteArgs& a, int64_t token, int lane, int pick, float weight) {
  if (a.renormalize) {
    const float total = warp_sum(lane < a.topk ? weight : 0.0f);
    weight = total == 0.0f ? 0.0f : weight / total;
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

// CTAs per SM: what hides the latencies of a token's steps is other tokens, at the price of registers where a lane
// holds few experts (256 experts in groups: 32 us with 24 warps an SM, 27 with 48).
template <int NV>
__global__ void __launch_bounds__(kRouteWarps * 32, NV <= 8 ? 12 : NV <= 16 ? 8 : 4)
route_topk_kernel(const __grid_constant__ RouteArgs a) {
  extern __shared__ uint64_t shared[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t token = static_cast<int64_t>(blockIdx.x) * kRouteWarps + warp;
  if (token >= a.tokens) return;
  uint64_t* scratch = shared + warp * (a.experts + 32);
  float c[NV];           // logits, then what a choice goes by
  uint32_t key[NV];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = lane + 32 * i;
    c[i] = e < a.experts ? load_logit(a.logits, token * a.ld_logits + e, a.bf16) : -INFINITY;
    key[i] = e < a.experts ? order_key(c[i]) : 0;
    top = fmaxf(top, c[i]);
  }
  const bool by_score = a.bias != nullptr;                        // else by logits
  const bool by_sum = a.groups > 1 && a.group_top2;
  float inv_sum = 1.0f;
  if (!a.sigmoid) {
    top = warp_max(top);
    if (top == -INFINITY) top = 0.0f;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) sum += expf(c[i] - top);
    sum = warp_sum(sum);
    inv_sum = sum == 0.0f ? 0.0f : 1.0f / sum;
  }
  auto score = [&](float x) { return a.sigmoid ? __fdividef(1.0f, 1.0f + expf(-x)) : expf(x - top) * inv_sum; };
  // How far two fp32 choice values must lie apart to be in the order of the exact ones: twice the error of a score,
  // and the roundings of the sums (under 2^-23 of |c| + 1/4 each). A sigmoid is off by the two steps of expf (2^-23
  // each), the sum's half step and the quotient's two: 2^-20.8 at most. A softmax by two steps of expf, the sum's NV + 5 roundings, two
  // more, and half a step of |x - top|, which is largest against exp(top - x) at 1: under (NV + 12) 2^-23 of the largest.
  const float slack = a.sigmoid ? 1.1e-6f : (NV + 12) * 2.4e-7f * inv_sum;
  auto near = [&](float high, float low) { return high - low <= slack + 2.4e-7f * (fabsf(high) + 0.25f); };   // NaN and inf - inf: not near
  if (by_score || by_sum) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = lane + 32 * i;
      if (e >= a.experts) continue;
      const float s = score(c[i]);
      c[i] = c[i] == -INFINITY ? c[i] : by_score ? s + a.bias[e] : s;
      if (by_score) key[i] = order_key(c[i]);
    }
  }
  uint32_t kept = kAll;                                           // bit g * share: group g takes part
  if (a.groups > 1) {
    // `share` adjacent lanes look through a group; in shared memory each group starts `share` words on, so that the
    // groups' lanes meet different banks
    const int size = a.experts / a.groups;
    const float inv_size = 1.0f / static_cast<float>(size);
    const int share = a.group_share, log_share = 31 - __clz(share);
    float* choice = reinterpret_cast<float*>(scratch);
    int first_lane[NV];                                            // of an expert's group
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = lane + 32 * i;
      first_lane[i] = static_cast<int>((static_cast<float>(e) + 0.5f) * inv_size) << log_share;      // the quotient is exact up to 1024
      if (e < a.experts) choice[e + first_lane[i]] = c[i];
    }
    __syncwarp();
    const int g = lane >> log_share, sub = lane & (share - 1);
    float first = -INFINITY, second = -INFINITY;
    if (g < a.groups)
      for (int e = sub; e < size; e += share) {
        const float v = choice[g * (size + share) + e];
        second = fmaxf(second, fminf(first, v));     // fminf, fmaxf pass NaN over
        first = fmaxf(first, v);
      }
    for (int o = 1; o < share; o <<= 1) {
      const float f = __shfl_xor_sync(kAll, first, o), h = __shfl_xor_sync(kAll, second, o);
      second = fmaxf(fmaxf(second, h), fminf(first, f));
      first = fmaxf(first, f);
    }
    const uint32_t mine = order_key(by_sum && second > -INFINITY ? first + second : first);
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
      // sums of two have twice the error
      if (near(key_value(worst_kept) * 0.5f, key_value(best_dropped) * 0.5f)) kept = exact_groups(a, token, reinterpret_cast<double*>(scratch));
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (lane + 32 * i < a.experts && !((kept >> first_lane[i]) & 1u)) key[i] = 0;
  }
  uint32_t best = 0;     // this lane's best candidate and its register
  int slot = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (key[i] > best) { best = key[i]; slot = i; }
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
    uint32_t* list = reinterpret_cast<uint32_t*>(scratch);           // keys, then experts
    int n = 0;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const bool in = key[i] >= bound;
      const uint32_t lanes = __ballot_sync(kAll, in);
      const int at = n + __popc(lanes & ((1u << lane) - 1u));
      if (in && at < 32) {
        list[at] = key[i];
        list[32 + at] = lane + 32 * i;
      }
      n += __popc(lanes);
    }
    __syncwarp();
    if (n <= 32) {
      // the list is in the order of the experts, so among equal keys the earlier place is the lower index
      const uint32_t mine = lane < n ? list[lane] : 0;
      const int e = lane < n ? list[32 + lane] : 0;
      int rank = 0;
      for (int j = 0; j < n; ++j) {
        const uint32_t other = list[j];
        rank += other > mine || (other == mine && j < lane);
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
    uint32_t last = 0;     // the key chosen before, and its expert
    int last_at = 0;
    for (count = 0;; ++count) {
      const uint32_t m = __reduce_max_sync(kAll, best);
      // past topk as long as a candidate may still change places with a chosen one
      const bool follows = by_score && count > 0 && m > 1u && near(key_value(last), key_value(m));
      if (count >= a.topk && (!follows || count == 32)) {
        if (follows) count = 33;
        break;
      }
      const int at = __reduce_min_sync(kAll, best == m ? lane + 32 * slot : 0x7FFFFFFF);
      if (follows)
        close = close || a.bias[at] != a.bias[last_at] ||
                load_logit(a.logits, token * a.ld_logits + at, a.bf16) != load_logit(a.logits, token * a.ld_logits + last_at, a.bf16);
      last = m;
      last_at = at;
      if (lane == (at & 31)) {
        best = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          key[i] = at == lane + 32 * i ? 0 : key[i];
          if (key[i] > best) { best = key[i]; slot = i; }
        }
      }
      if (lane == count) pick = at;
    }
  }
  if (count > 32) pick = exact_choice(a, token, kept, scratch);
  else if (close) pick = exact_order(a, token, pick, count);
  store_choice(a, token, lane, pick, lane < a.topk ? score(load_logit(a.logits, token * a.ld_logits + pick, a.bf16)) : 0.0f);
}

template <int NV>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_topk_bwd_kernel(const __grid_constant__ RouteBwdArgs a) {
  extern __shared__ float ds_all[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t token = static_cast<int64_t>(blockIdx.x) * kRouteWarps + warp;
  if (token >= a.tokens) return;
  float s[NV];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = lane + 32 * i;
    s[i] = e < a.experts ? load_logit(a.logits, token * a.ld_logits + e, a.bf16) : -INFINITY;
    top = fmaxf(top, s[i]);
  }
  top = warp_max(top);
  if (top == -INFINITY) top = 0.0f;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    s[i] = a.sigmoid ? 1.0f / (1.0f + expf(-s[i])) : expf(s[i] - top);
    if (!a.sigmoid) sum += s[i];
  }
  if (!a.sigmoid) {
    sum = warp_sum(sum);
#pragma unroll
    for (int i = 0; i < NV; ++i) s[i] = sum == 0.0f ? 0.0f : s[i] / sum;
  }
  // lane j holds slot j: its expert, that expert's score and the gradient of its weight
  const int at = lane < a.topk ? a.experts_in[token * a.topk + lane] : -1;
  const bool valid = at >= 0 && at < a.experts;
  float g = valid ? a.d_weights[token * a.topk + lane] * a.scale : 0.0f;
  float mine = 0.0f;
  if (valid) {
    const float x = load_logit(a.logits, token * a.ld_logits + at, a.bf16);
    mine = a.sigmoid ? 1.0f / (1.0f + expf(-x)) : sum == 0.0f ? 0.0f : expf(x - top) / sum;
  }
  if (a.renormalize) {
    const float total = warp_sum(mine), inner = warp_sum(g * mine);
    g = !valid || total == 0.0f ? 0.0f : (g - inner / total) / total;
  }
  const float dot = a.sigmoid ? 0.0f : warp_sum(g * mine);
  // slots to experts, in the slots' order (an expert may be named twice)
  float* ds = ds_all + warp * a.experts;
  for (int e = lane; e < a.experts; e += 32) ds[e] = 0.0f;
  __syncwarp();
  const uint32_t peers = __match_any_sync(kAll, valid ? at : -1 - lane);
  const bool alone = __all_sync(kAll, peers == 1u << lane);
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
  for (int i = 0; i < NV; ++i) {
    const int e = lane + 32 * i;
    if (e >= a.experts) continue;
    const float d = a.sigmoid ? ds[e] * s[i] * (1.0f - s[i]) : s[i] * (ds[e] - dot);
    const int64_t o = token * a.experts + e;
    if (a.bf16) static_cast<__nv_bfloat16*>(a.d_logits)[o] = __float2bfloat16_rn(d);
    else static_cast<float*>(a.d_logits)[o] = d;
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

cudaError_t launch_route_topk(const RouteArgs& a, cudaStream_t stream) {
  if (a.tokens == 0) return cudaSuccess;
  const unsigned grid = static_cast<unsigned>((a.tokens + kRouteWarps - 1) / kRouteWarps);
  return by_width(a.experts, [&](auto n) {
    route_topk_kernel<decltype(n)::value><<<grid, kRouteWarps * 32, kRouteWarps * (a.experts + 32) * sizeof(uint64_t), stream>>>(a);
  });
}

cudaError_t launch_route_topk_bwd(const RouteBwdArgs& a, cudaStream_t stream) {
  if (a.tokens == 0) return cudaSuccess;
  const unsigned grid = static_cast<unsigned>((a.tokens + kRouteWarps - 1) / kRouteWarps);
  return by_width(a.experts, [&](auto n) { route_topk_bwd_kernel<decltype(n)::value><<<grid, kRouteWarps * 32, kRouteWarps * a.experts * sizeof(float), stream>>>(a); });
}

}  // namespace plb
