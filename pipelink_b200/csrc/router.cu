// Routing of tokens to experts, and the gradient of the weights.
//
//   s = softmax(x) or sigmoid(x)        choice c = s + bias, masked experts (x = -inf) -inf
//   group score = max of c or the sum of its two best unmasked c; the topk_groups best groups are kept
//   the topk best c of the kept groups, ties to the lowest index; w = scale * s [/ sum of the chosen s]
//   dS_j = scale / S * (g_j - sum_i g_i s_i / S) or scale * g_j;  dx = s (dS - sum s dS) or dS s (1 - s)
//
// One warp per token, expert e in register e / 32 of lane e % 32; a choice is topk rounds of a warp-wide maximum
// over the lanes' best. Without a bias the scores are ordered as the logits are, and those are compared as they
// stand. With one (or with sums of two scores over groups) the order is that of numbers fp32 may not tell apart:
// each comparison that matters is checked against the bound of the fp32 scores' error, and a token that fails is
// done again in fp64 (about 3 of 1000 at 256 experts).
#include <math.h>

#include <type_traits>

#include "kernels.h"

namespace plb {

namespace {

constexpr int kRouteWarps = 4;
constexpr uint32_t kAll = 0xFFFFFFFFu;

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

// One token with every score in fp64. `key` is the warp's shared memory, one word per expert.
__device__ __noinline__ void route_exact(const RouteArgs& a, int64_t token, uint64_t* key) {
  const int lane = threadIdx.x & 31, size = a.experts / a.groups;
  double top = -INFINITY, sum = 0.0;
  auto logit = [&](int e) { return static_cast<double>(load_logit(a.logits, token * a.ld_logits + e, a.bf16)); };
  if (!a.sigmoid) {
    for (int e = lane; e < a.experts; e += 32) top = fmax(top, logit(e));
    top = warp_max(top);
    if (top == -INFINITY) top = 0.0;
    for (int e = lane; e < a.experts; e += 32) sum += exp(logit(e) - top);
    sum = warp_sum(sum);
  }
  auto score = [&](double x) { return a.sigmoid ? 1.0 / (1.0 + exp(-x)) : sum == 0.0 ? 0.0 : exp(x - top) / sum; };
  double* choice = reinterpret_cast<double*>(key);
  __syncwarp();
  for (int e = lane; e < a.experts; e += 32) {
    const double x = logit(e);
    choice[e] = x == -INFINITY ? x : a.bias != nullptr ? score(x) + static_cast<double>(a.bias[e]) : score(x);
  }
  __syncwarp();
  uint32_t kept = kAll;
  if (a.groups > 1) {
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
    kept = __ballot_sync(kAll, lane < a.groups && better < a.topk_groups);
  }
  __syncwarp();
  for (int e = lane; e < a.experts; e += 32)
    key[e] = !((kept >> (a.groups > 1 ? e / size : 0)) & 1u) ? 0 : order_key(a.bias != nullptr ? choice[e] : logit(e));
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
  store_choice(a, token, lane, pick, lane < a.topk ? static_cast<float>(score(logit(pick))) : 0.0f);
}

template <int NV>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_topk_kernel(const __grid_constant__ RouteArgs a) {
  extern __shared__ uint64_t shared[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t token = static_cast<int64_t>(blockIdx.x) * kRouteWarps + warp;
  if (token >= a.tokens) return;
  uint64_t* scratch = shared + warp * a.experts;
  float s[NV];
  uint32_t key[NV];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = lane + 32 * i;
    s[i] = e < a.experts ? load_logit(a.logits, token * a.ld_logits + e, a.bf16) : -INFINITY;
    key[i] = e < a.experts ? order_key(s[i]) : 0;                 // the logits' order, for now
    top = fmaxf(top, s[i]);
  }
  const bool by_score = a.bias != nullptr;                        // else by logits
  const bool by_sum = a.groups > 1 && a.group_top2;
  float inv_sum = 1.0f;
  if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < NV; ++i) s[i] = __fdividef(1.0f, 1.0f + expf(-s[i]));       // expf is at most 3e38 above: 1 / inf = 0
  } else {
    top = warp_max(top);
    if (top == -INFINITY) top = 0.0f;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      s[i] = expf(s[i] - top);
      sum += s[i];
    }
    sum = warp_sum(sum);
    inv_sum = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < NV; ++i) s[i] *= inv_sum;
  }
  // How far two fp32 choice values must lie apart to be in the order of the exact ones: twice the error of a score
  // (expf 2 steps of 2^-23, sums and quotients at most NV + 8 half steps, |x - top| half steps where the score is
  // exp(top - x) times smaller: together under (NV + 16) * 2^-23 of the largest score), and the rounding of the sums.
  const float slack = (NV + 16) * 2.4e-7f * inv_sum;
  auto near = [&](float high, float low) { return high - low <= slack + 4.8e-7f * (fabsf(high) + 0.25f); };   // NaN and inf - inf: not near
  bool exact = true;
  if (by_score || by_sum) {
    float c[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = lane + 32 * i;
      c[i] = e < a.experts ? (key[i] == 0x007FFFFFu ? -INFINITY : by_score ? s[i] + a.bias[e] : s[i]) : -INFINITY;
      if (by_score && e < a.experts) key[i] = order_key(c[i]);
    }
    if (a.groups > 1) {
      float* choice = reinterpret_cast<float*>(scratch);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (lane + 32 * i < a.experts) choice[lane + 32 * i] = c[i];
    }
  } else if (a.groups > 1) {
    float* choice = reinterpret_cast<float*>(scratch);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (lane + 32 * i < a.experts) choice[lane + 32 * i] = key[i] == 1u ? NAN : key_value(key[i]);
  }
  if (a.groups > 1) {
    const int size = a.experts / a.groups;
    const float inv_size = 1.0f / static_cast<float>(size);
    const float* choice = reinterpret_cast<const float*>(scratch);
    __syncwarp();
    float first = -INFINITY, second = -INFINITY;
    if (lane < a.groups)
      for (int e = lane * size; e < (lane + 1) * size; ++e) {
        const float c = choice[e];
        second = fmaxf(second, fminf(first, c));     // fminf, fmaxf pass NaN over
        first = fmaxf(first, c);
      }
    const float value = by_sum && second > -INFINITY ? first + second : first;
    const uint32_t mine = order_key(value);
    int better = 0;
    for (int g = 0; g < a.groups; ++g) {
      const uint32_t other = __shfl_sync(kAll, mine, g);
      better += other > mine || (other == mine && g < lane);
    }
    const bool keep = lane < a.groups && better < a.topk_groups;
    const uint32_t kept = __ballot_sync(kAll, keep);
    if (by_score || by_sum) {
      const uint32_t worst_kept = __reduce_min_sync(kAll, keep ? mine : 0xFFFFFFFFu);
      const uint32_t best_dropped = __reduce_max_sync(kAll, lane < a.groups && !keep ? mine : 0u);
      exact = !near(key_value(worst_kept) * 0.5f, key_value(best_dropped) * 0.5f);       // sums of two have twice the error
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = lane + 32 * i;
      const int g = static_cast<int>((static_cast<float>(e) + 0.5f) * inv_size);
      if (e < a.experts && !((kept >> g) & 1u)) key[i] = 0;
    }
  }
  int pick = 0;          // lane j: the j-th chosen expert
  uint32_t best = 0;     // this lane's best candidate and its register
  int slot = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (key[i] > best) { best = key[i]; slot = i; }
  uint32_t last = 0;     // the key chosen before, and its expert
  int last_at = 0;
  const int rounds = by_score ? a.topk + 1 : a.topk;               // one more value is looked at than chosen
  for (int j = 0; j < rounds; ++j) {
    const uint32_t m = __reduce_max_sync(kAll, best);
    const int at = __reduce_min_sync(kAll, best == m ? lane + 32 * slot : 0x7FFFFFFF);
    // near values are in order only if they are the same number: the same logit under the same bias
    if (by_score && j > 0 && m > 1u && near(key_value(last), key_value(m)))
      exact = exact && a.bias[at] == a.bias[last_at] &&
              load_logit(a.logits, token * a.ld_logits + at, a.bf16) == load_logit(a.logits, token * a.ld_logits + last_at, a.bf16);
    last = m;
    last_at = at;
    if (j == a.topk) break;
    if (lane == (at & 31)) {
      best = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        key[i] = at == lane + 32 * i ? 0 : key[i];
        if (key[i] > best) { best = key[i]; slot = i; }
      }
    }
    if (lane == j) pick = at;
  }
  if (!exact) {
    route_exact(a, token, scratch);
    return;
  }
  float weight = 0.0f;
  if (lane < a.topk) {
    const float x = load_logit(a.logits, token * a.ld_logits + pick, a.bf16);
    weight = a.sigmoid ? __fdividef(1.0f, 1.0f + expf(-x)) : expf(x - top) * inv_sum;
  }
  store_choice(a, token, lane, pick, weight);
}

template <int NV>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_topk_bwd_kernel(const RouteBwdArgs a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t token = static_cast<int64_t>(blockIdx.x) * kRouteWarps + warp;
  if (token >= a.tokens) return;
  float s[NV], ds[NV];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = lane + 32 * i;
    s[i] = e < a.experts ? load_logit(a.logits, token * a.ld_logits + e, a.bf16) : -INFINITY;
    top = fmaxf(top, s[i]);
    ds[i] = 0.0f;
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
  for (int j = 0; j < a.topk; ++j) {
    const int e = __shfl_sync(kAll, at, j);
    const float v = __shfl_sync(kAll, g, j);
    if ((e & 31) == lane) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (e == lane + 32 * i) ds[i] += v;
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = lane + 32 * i;
    if (e >= a.experts) continue;
    const float d = a.sigmoid ? ds[i] * s[i] * (1.0f - s[i]) : s[i] * (ds[i] - dot);
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
    route_topk_kernel<decltype(n)::value><<<grid, kRouteWarps * 32, kRouteWarps * a.experts * sizeof(uint64_t), stream>>>(a);
  });
}

cudaError_t launch_route_topk_bwd(const RouteBwdArgs& a, cudaStream_t stream) {
  if (a.tokens == 0) return cudaSuccess;
  const unsigned grid = static_cast<unsigned>((a.tokens + kRouteWarps - 1) / kRouteWarps);
  return by_width(a.experts, [&](auto n) { route_topk_bwd_kernel<decltype(n)::value><<<grid, kRouteWarps * 32, 0, stream>>>(a); });
}

}  // namespace plb
