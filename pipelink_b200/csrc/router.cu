// Routing of tokens to experts, and the gradient of the weights.
//
//   s = softmax(x) or sigmoid(x)        choice c = s + bias, masked experts (x = -inf) -inf
//   group score = max of c or the sum of its two best unmasked c; the topk_groups best groups are kept
//   the topk best c of the kept groups, ties to the lowest index; w = scale * s [/ sum of the chosen s]
//   dS_j = scale / S * (g_j - sum_i g_i s_i / S) or scale * g_j;  dx = s (dS - sum s dS) or dS s (1 - s)
//
// One warp per token, expert e in register e / 32 of lane e % 32. A choice is an order of scores that may lie
// closer together than fp32 resolves, so they are compared in fp64; without a bias the scores are ordered as the
// logits are, and those are compared as they stand.
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
__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(kAll, v, o));
  return v;
}
__device__ __forceinline__ double warp_add(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

template <int NV>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_topk_kernel(const RouteArgs a) {
  extern __shared__ double shared[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t token = static_cast<int64_t>(blockIdx.x) * kRouteWarps + warp;
  if (token >= a.tokens) return;
  double* choice = shared + warp * a.experts;
  double s[NV];
  uint64_t key[NV];
  double top = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = lane + 32 * i;
    s[i] = e < a.experts ? static_cast<double>(load_logit(a.logits, token * a.ld_logits + e, a.bf16)) : -INFINITY;
    top = fmax(top, s[i]);
  }
  top = warp_max(top);
  if (top == -INFINITY) top = 0.0;
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = lane + 32 * i;
    const double x = s[i];
    if (a.sigmoid) s[i] = 1.0 / (1.0 + exp(-x));
    else { s[i] = exp(x - top); sum += s[i]; }
    key[i] = __double_as_longlong(x);
    (void)e;
  }
  if (!a.sigmoid) {
    sum = warp_add(sum);
#pragma unroll
    for (int i = 0; i < NV; ++i) s[i] = sum == 0.0 ? 0.0 : s[i] / sum;
  }
  uint32_t kept = kAll;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = lane + 32 * i;
    const double x = __longlong_as_double(static_cast<long long>(key[i]));
    double c = a.bias != nullptr && e < a.experts ? s[i] + static_cast<double>(a.bias[e]) : s[i];
    if (x == -INFINITY) c = -INFINITY;
    if (e < a.experts) choice[e] = c;
    key[i] = e < a.experts ? order_key(a.bias != nullptr ? c : x) : 0;
    if (x == -INFINITY && e < a.experts) key[i] = order_key(-INFINITY);
  }
  const int size = a.experts / a.groups;
  if (a.groups > 1) {
    __syncwarp();
    double score = -INFINITY;
    if (lane < a.groups) {
      double first = -INFINITY, second = -INFINITY;
      for (int e = lane * size; e < (lane + 1) * size; ++e) {
        const double c = choice[e];
        if (c > first) { second = first; first = c; }
        else if (c > second) second = c;
      }
      score = a.group_top2 && second > -INFINITY ? first + second : first;
    }
    const uint64_t mine = order_key(score);
    int better = 0;
    for (int g = 0; g < a.groups; ++g) {
      const uint64_t other = __shfl_sync(kAll, mine, g);
      better += other > mine || (other == mine && g < lane);
    }
    kept = __ballot_sync(kAll, lane < a.groups && better < a.topk_groups);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = lane + 32 * i;
      if (e < a.experts && !((kept >> (e / size)) & 1u)) key[i] = 0;
    }
  }
  int pick = 0;          // lane j: the j-th chosen expert and its score
  float weight = 0.0f;
  for (int j = 0; j < a.topk; ++j) {
    uint64_t best = 0;
    int at = 0x7FFFFFFF;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (key[i] > best) { best = key[i]; at = lane + 32 * i; }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t b = __shfl_xor_sync(kAll, best, o);
      const int e = __shfl_xor_sync(kAll, at, o);
      if (b > best || (b == best && e < at)) { best = b; at = e; }
    }
    float w = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (at == lane + 32 * i) { key[i] = 0; w = static_cast<float>(s[i]); }
    w = __shfl_sync(kAll, w, at & 31);
    if (lane == j) { pick = at; weight = w; }
  }
  if (a.renormalize) {
    float total = lane < a.topk ? weight : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(kAll, total, o);
    weight = total == 0.0f ? 0.0f : weight / total;
  }
  if (lane < a.topk) {
    a.experts_out[token * a.topk + lane] = pick;
    a.weights_out[token * a.topk + lane] = weight * a.scale;
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
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
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
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
  // lane j holds slot j
  const int at = lane < a.topk ? a.experts_in[token * a.topk + lane] : -1;
  float g = lane < a.topk ? a.d_weights[token * a.topk + lane] * a.scale : 0.0f;
  float mine = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    for (int j = 0; j < a.topk; ++j) {
      const int e = __shfl_sync(kAll, at, j);
      const float v = __shfl_sync(kAll, s[i], e & 31);
      if (lane == j && e >= 0 && e < a.experts && (e >> 5) == i) mine = v;
    }
  if (a.renormalize) {
    const float total = warp_sum(mine), dot = warp_sum(g * mine);
    g = total == 0.0f ? 0.0f : (g - dot / total) / total;
  }
  for (int j = 0; j < a.topk; ++j) {
    const int e = __shfl_sync(kAll, at, j);
    const float v = __shfl_sync(kAll, g, j);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (e == lane + 32 * i) ds[i] += v;
  }
  float dot = 0.0f;
  if (!a.sigmoid) {
#pragma unroll
    for (int i = 0; i < NV; ++i) dot = fmaf(s[i], ds[i], dot);
    dot = warp_sum(dot);
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
    route_topk_kernel<decltype(n)::value><<<grid, kRouteWarps * 32, kRouteWarps * a.experts * sizeof(double), stream>>>(a);
  });
}

cudaError_t launch_route_topk_bwd(const RouteBwdArgs& a, cudaStream_t stream) {
  if (a.tokens == 0) return cudaSuccess;
  const unsigned grid = static_cast<unsigned>((a.tokens + kRouteWarps - 1) / kRouteWarps);
  return by_width(a.experts, [&](auto n) { route_topk_bwd_kernel<decltype(n)::value><<<grid, kRouteWarps * 32, 0, stream>>>(a); });
}

}  // namespace plb
