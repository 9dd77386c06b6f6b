// Choice of experts from router logits: per token the top-k of E scores, and their weights.
//
//   s_e = softmax(l)_e  or  1 / (1 + exp(-l_e));   c_e = s_e + bias_e, which chooses but does not weigh
//   with groups: the E experts are equal runs; a run's score is the sum of its two largest c; only the best runs stay
//   idx = the k largest c, largest first, ties to the lowest index;   w = s[idx] (/ their sum) * scale
//
// One warp per token, the logits in its registers (expert i * 32 + lane in lane `lane`), k rounds of a warp maximum over
// order-preserving integer keys. Without bias and groups the order of c is that of l, so the keys are the logits' own bits
// and nothing is rounded before the choice. With them, scores and sums are computed in 64 bits: two experts whose scores
// differ by less than an fp32 rounding are told apart, and the choice does not depend on the order of a sum.
// A logit or bias of -inf or NaN takes its expert out; where fewer than k are left, the rest of the row is (-1, 0).
// The weights of the chosen few are computed in 64 bits either way; of 32 bits is only the sum of a softmax without bias and groups.
// Bound by latency: a token is a chain of k warp maxima; the reads (1 KiB per token at E = 256) are never the limit. With groups the
// 64-bit exponentials and quotients of all experts are in front of it, a warp's steps one after the other; no pipe is full (46 % of the issue
// slots). Measured in a graph, 256 experts, top-8: one token 4.2 us; 4096 tokens 8.2 us, within 4 of 8 groups 16.3 us.
#include <type_traits>

#include "eux_device.cuh"

namespace eux {

constexpr int kRouteWarps = 4;

__device__ __forceinline__ uint32_t order_key(float v) {  // larger value, larger key; never 0 for a number
  const uint32_t u = __float_as_uint(v + 0.f);            // -0 counts as 0
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ uint64_t order_key(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);
  return u ^ ((u >> 63) ? ~0ull : 0x8000000000000000ull);
}
__device__ __forceinline__ double key_value(uint64_t k) {
  return __longlong_as_double((long long)(k ^ ((k >> 63) ? 0x8000000000000000ull : ~0ull)));
}

__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ double warp_sum(double v) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float route_logit(const eux_route_desc& d, int64_t t, int e) {
  const int64_t at = t * d.logits_stride + e;
  return d.dtype == EUX_DT_F32 ? reinterpret_cast<const float*>(d.logits)[at]
                               : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(d.logits)[at]);
}

// A lane's largest key and where it is, from its registers.
template <int NV, typename Key>
__device__ __forceinline__ void lane_best(const Key (&key)[NV], Key& mine, int& at) {
  mine = 0, at = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (key[i] > mine) mine = key[i], at = i;
}
// The warp's largest key, of equal ones that of the lowest expert, is taken out; its expert, -1 if there is none. `mine` and `at` are the
// lanes' largest.
template <int NV>
__device__ __forceinline__ int take_best(uint32_t (&key)[NV], uint32_t& mine, int& at, int lane) {
  const uint32_t top = warp_max(mine);
  const uint32_t e = __reduce_min_sync(0xffffffffu, mine == top ? (uint32_t)(at * 32 + lane) : 0xffffffffu);
  if (top == 0) return -1;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((uint32_t)(i * 32 + lane) == e) key[i] = 0;
  lane_best<NV>(key, mine, at);
  return (int)e;
}
// With 64-bit keys the upper halves nearly always tell; only where they do not are the lower ones, and then the experts, asked, and only
// the lane that had it looks for its next one.
template <int NV>
__device__ __forceinline__ int take_best(uint64_t (&key)[NV], uint64_t& mine, int& at, int lane) {
  const uint32_t top = warp_max((uint32_t)(mine >> 32));
  uint32_t who = __ballot_sync(0xffffffffu, mine != 0 && (uint32_t)(mine >> 32) == top);
  if (who == 0) return -1;
  if (who & (who - 1)) {
    const uint32_t low = warp_max((who >> lane) & 1u ? (uint32_t)mine : 0u);
    who = __ballot_sync(0xffffffffu, ((who >> lane) & 1u) && (uint32_t)mine == low);
    who = 1u << (__reduce_min_sync(0xffffffffu, (who >> lane) & 1u ? (uint32_t)(at * 32 + lane) : 0xffffffffu) & 31u);
  }
  const int winner = __ffs(who) - 1, e = __shfl_sync(0xffffffffu, at, winner) * 32 + winner;
  if (lane == winner) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i == at) key[i] = 0;
    lane_best<NV>(key, mine, at);
  }
  return e;
}

// WIDE: scores and keys in 64 bits (bias or groups). Without, only a softmax's sum is of 32.
template <int NV, bool WIDE>
__global__ void __launch_bounds__(kRouteWarps * 32) moe_route_kernel(eux_route_desc d) {
  using Key = typename std::conditional<WIDE, uint64_t, uint32_t>::type;
  using Real = typename std::conditional<WIDE, double, float>::type;
  wait_for_launch_before();
  __shared__ uint64_t keys[WIDE ? kRouteWarps : 1][WIDE ? NV * 32 : 1];
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
  if (t < d.n_tokens) {
    const int E = d.n_experts;
    float l[NV];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = i * 32 + lane;
      const float v = e < E ? route_logit(d, t, e) : -INFINITY;
      // an infinite logit weighs as the largest number does
      l[i] = v > -INFINITY ? fminf(v, 3.402823466e38f) : -INFINITY;  // NaN too
      if (l[i] > -INFINITY) top = max(top, order_key(l[i]));
    }
    top = warp_max(top);
    // the largest logit, and the sum of exponentials above it
    const float peak = top ? __uint_as_float(top ^ ((top >> 31) ? 0x80000000u : 0xffffffffu)) : 0.f;
    Real sum = 1;
    Real ex[WIDE ? NV : 1];
    if (!d.sigmoid) {
      Real part = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const Real v = l[i] > -INFINITY ? (WIDE ? (Real)exp((double)l[i] - (double)peak) : (Real)expf(l[i] - peak)) : (Real)0;
        if (WIDE) ex[WIDE ? i : 0] = v;
        part += v;
      }
      sum = warp_sum(part);
    }
    Key key[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = i * 32 + lane;
      key[i] = 0;
      if (l[i] > -INFINITY) {
        if constexpr (WIDE) {
          const float b = d.bias ? d.bias[e] : 0.f;
          const double s = d.sigmoid ? __drcp_rn(1.0 + exp(-(double)l[i])) : ex[i] / sum;
          if (b > -INFINITY) key[i] = order_key(s + (double)b);
        } else {
          key[i] = order_key(route_logit(d, t, e));  // with +inf above the largest number
        }
      }
    }
    if constexpr (WIDE) {
      if (d.groups > 1) {
        // As many lanes as there are for each group look through its experts, in shared memory, for the two largest.
        const int size = E / d.groups, per = 32 / d.groups, lanes = per >= 16 ? 16 : per >= 8 ? 8 : per >= 4 ? 4 : per >= 2 ? 2 : 1;
        uint64_t* const mine = keys[threadIdx.x >> 5];
#pragma unroll
        for (int i = 0; i < NV; ++i) mine[i * 32 + lane] = key[i];
        __syncwarp();
        const int g0 = lane / lanes;
        uint64_t b1 = 0, b2 = 0;
        if (g0 < d.groups)
          for (int e = lane % lanes; e < size; e += lanes) {
            const uint64_t k = mine[g0 * size + e], low = min(k, b1);
            b1 = max(k, b1), b2 = max(low, b2);
          }
        for (int o = 1; o < lanes; o <<= 1) {
          const uint64_t o1 = __shfl_xor_sync(0xffffffffu, b1, o), o2 = __shfl_xor_sync(0xffffffffu, b2, o);
          b2 = max(min(b1, o1), max(b2, o2)), b1 = max(b1, o1);
        }
        const double of_mine = b1 ? key_value(b1) + (b2 ? key_value(b2) : 0.0) : -INFINITY;
        const double score = __shfl_sync(0xffffffffu, of_mine, min(lane, d.groups - 1) * lanes);  // of the group with this lane's number
        int ahead = 0;
        for (int g = 0; g < d.groups; ++g) {
          const double other = __shfl_sync(0xffffffffu, score, g);
          ahead += other > score || (other == score && g < lane);
        }
        const uint32_t open = __ballot_sync(0xffffffffu, lane < d.groups && ahead < d.topk_groups);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int e = i * 32 + lane;
          if (e < E && !((open >> (e / size)) & 1u)) key[i] = 0;
        }
      }
    }
    int mine = -1, at;  // lane j: the expert in place j
    Key best;
    lane_best<NV>(key, best, at);
    for (int j = 0; j < d.topk; ++j) {
      const int e = take_best<NV>(key, best, at, lane);
      if (lane == j) mine = e;
    }
    // The weights of the few that are chosen, one per lane, in 64 bits: sigmoids and quotients of them that 32 bits have no number for count.
    double s = 0;
    if (mine >= 0) {
      const double v = fminf(route_logit(d, t, mine), 3.402823466e38f);
      s = d.sigmoid ? __drcp_rn(1.0 + exp(-v)) : exp(v - (double)peak) / (double)sum;
    }
    if (d.renormalize) {
      const double all = warp_sum(s);
      s = all > 0 ? s / all : 0.0;  // none taken, or every score too small for a number: no weight
    }
    if (lane < d.topk) {
      d.topk_idx[t * d.topk + lane] = mine;
      d.topk_w[t * d.topk + lane] = (float)(s * (double)d.scale);
    }
  }
  allow_next_launch();
}

template <int NV>
static int route_launch(const eux_route_desc& d, cudaStream_t st) {
  const int grid = (d.n_tokens + kRouteWarps - 1) / kRouteWarps;
  return d.bias || d.groups > 1 ? launch_early(moe_route_kernel<NV, true>, grid, kRouteWarps * 32, 0, st, d)
                                : launch_early(moe_route_kernel<NV, false>, grid, kRouteWarps * 32, 0, st, d);
}

template <int NV>
static int route_preload() {
  cudaFuncAttributes a;
  if (cudaError_t e = cudaFuncGetAttributes(&a, moe_route_kernel<NV, true>); e != cudaSuccess) return (int)e;
  return (int)cudaFuncGetAttributes(&a, moe_route_kernel<NV, false>);
}

}  // namespace eux

using namespace eux;

extern "C" int eux_route_launch(const eux_route_desc* d, void* stream) {
  if (!d || d->n_tokens < 0 || d->n_experts < 1 || d->n_experts > EUX_ROUTE_MAX_EXPERTS) return EUX_ERR_BAD_ARG;
  if (d->topk < 1 || d->topk > 32 || d->topk > d->n_experts) return EUX_ERR_BAD_ARG;
  if (d->groups < 1 || d->groups > 32 || d->n_experts % d->groups || d->topk_groups < 1 || d->topk_groups > d->groups) return EUX_ERR_BAD_ARG;
  if (d->dtype != EUX_DT_F32 && d->dtype != EUX_DT_BF16) return EUX_ERR_BAD_ARG;
  if (d->n_tokens == 0) return 0;
  if (!d->logits || !d->topk_idx || !d->topk_w) return EUX_ERR_BAD_ARG;
  const cudaStream_t st = (cudaStream_t)stream;
  const int nv = (d->n_experts + 31) / 32;
  if (nv <= 1) return route_launch<1>(*d, st);
  if (nv <= 2) return route_launch<2>(*d, st);
  if (nv <= 4) return route_launch<4>(*d, st);
  if (nv <= 8) return route_launch<8>(*d, st);
  if (nv <= 16) return route_launch<16>(*d, st);
  return route_launch<32>(*d, st);
}

extern "C" int eux_route_preload(void) {
  for (int rc : {route_preload<1>(), route_preload<2>(), route_preload<4>(), route_preload<8>(), route_preload<16>(), route_preload<32>()})
    if (rc) return rc;
  return 0;
}
