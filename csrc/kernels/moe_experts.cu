// A whole mixture-of-experts layer for a few tokens, in two launches:
//
//   h_j = silu(W_gate[e] x_t) * (W_up[e] x_t)      for every entry j = (t, slot) whose expert e is here
//   out_t = sum over the entries of t of w_j * (W_down[e] h_j)
//
// One warp per row of a weight and entry: 16 bytes per lane and step, sums in fp32.
#include <algorithm>

#include "eux_bulk.cuh"
#include "eux_device.cuh"

namespace eux {

constexpr int kExpertThreads = 256;

// The dot product of a weight row of n elements with n bf16 values, by a warp.
template <bool FP8>
__device__ __forceinline__ float row_dot(const void* w, const float* scale, const __nv_bfloat16* v, int n, int lane) {
  float acc = 0.f;
  for (int k = lane * 8; k < n; k += 256) {
    const uint4 xv = *reinterpret_cast<const uint4*>(v + k);
    const __nv_bfloat162* x2 = reinterpret_cast<const __nv_bfloat162*>(&xv);
    float part = 0.f;
    if (FP8) {
      const uint2 wv = *reinterpret_cast<const uint2*>((const uint8_t*)w + k);
      const __nv_fp8_e4m3* w8 = reinterpret_cast<const __nv_fp8_e4m3*>(&wv);
      for (int i = 0; i < 4; ++i) {
        const float2 a = __bfloat1622float2(x2[i]);
        part += float(w8[2 * i]) * a.x + float(w8[2 * i + 1]) * a.y;
      }
      acc += part * scale[k / 128];
    } else {
      const uint4 wv = *reinterpret_cast<const uint4*>((const __nv_bfloat16*)w + k);
      const __nv_bfloat162* w2 = reinterpret_cast<const __nv_bfloat162*>(&wv);
      for (int i = 0; i < 4; ++i) {
        const float2 a = __bfloat1622float2(x2[i]), b = __bfloat1622float2(w2[i]);
        part += a.x * b.x + a.y * b.y;
      }
      acc += part;
    }
  }
  for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  return acc;
}

template <bool FP8>
__global__ void __launch_bounds__(kExpertThreads) experts_up_kernel(eux_experts_desc d) {
  const int lane = threadIdx.x & 31, j = blockIdx.y, i = blockIdx.x * (kExpertThreads / 32) + (threadIdx.x >> 5);
  const int e = d.topk_idx[j];
  if (e < 0 || e >= d.n_experts || i >= d.inner) return;
  const __nv_bfloat16* x = (const __nv_bfloat16*)d.x + (int64_t)(j / d.topk) * d.x_stride;
  const size_t elem = FP8 ? 1 : 2, sr = (2 * d.inner + 127) / 128, sc = (d.hidden + 127) / 128;
  float v[2];
  for (int half = 0; half < 2; ++half) {
    const size_t r = (size_t)i + (size_t)half * d.inner;
    v[half] = row_dot<FP8>((const char*)d.w_gate_up + ((size_t)e * 2 * d.inner + r) * d.hidden * elem,
                           d.gate_up_scale + (e * sr + r / 128) * sc, x, d.hidden, lane);
  }
  if (lane == 0) ((__nv_bfloat16*)d.workspace)[(size_t)j * d.inner + i] = __float2bfloat16_rn(v[0] / (1.f + __expf(-v[0])) * v[1]);
}

template <bool FP8>
__global__ void __launch_bounds__(kExpertThreads) experts_down_kernel(eux_experts_desc d) {
  const int lane = threadIdx.x & 31, t = blockIdx.y, r = blockIdx.x * (kExpertThreads / 32) + (threadIdx.x >> 5);
  if (r >= d.hidden) return;
  const size_t elem = FP8 ? 1 : 2, sr = (d.hidden + 127) / 128, sc = (d.inner + 127) / 128;
  float y = 0.f;
  for (int s = 0; s < d.topk; ++s) {
    const int j = t * d.topk + s, e = d.topk_idx[j];
    if (e < 0 || e >= d.n_experts) continue;
    y += d.topk_w[j] * row_dot<FP8>((const char*)d.w_down + ((size_t)e * d.hidden + r) * d.inner * elem,
                                    d.down_scale + (e * sr + r / 128) * sc, (const __nv_bfloat16*)d.workspace + (size_t)j * d.inner,
                                    d.inner, lane);
  }
  if (lane == 0) ((__nv_bfloat16*)d.out)[(int64_t)t * d.out_stride + r] = __float2bfloat16_rn(y);
}

static int experts_check(const eux_experts_desc* d) {
  if (!d || d->n_tokens < 0 || d->n_tokens > EUX_EXPERTS_MAX_TOKENS || d->topk < 1 || d->topk > 32) return EUX_ERR_BAD_ARG;
  if (d->n_experts < 1 || d->n_experts > EUX_EXPERTS_MAX_EXPERTS || d->hidden < 1 || d->inner < 1) return EUX_ERR_BAD_ARG;
  const int unit = d->fp8 ? 16 : 8;  // rows of weights begin on 16 bytes
  if (d->hidden % unit || d->inner % unit || d->x_stride % 8 || d->out_stride % 8) return EUX_ERR_BAD_ARG;
  return 0;
}

}  // namespace eux

using namespace eux;

extern "C" size_t eux_experts_workspace_bytes(const eux_experts_desc* d) {
  return experts_check(d) ? 0 : (size_t)d->n_tokens * d->topk * d->inner * 2;
}
extern "C" size_t eux_experts_counter_words(const eux_experts_desc* d) { return experts_check(d) ? 0 : 1; }

extern "C" int eux_experts_launch(const eux_experts_desc* d, void* stream) {
  if (int rc = experts_check(d)) return rc;
  if (d->n_tokens == 0) return 0;
  if (!d->x || !d->topk_idx || !d->topk_w || !d->out || !d->w_gate_up || !d->w_down || !d->workspace) return EUX_ERR_BAD_ARG;
  if (d->fp8 && (!d->gate_up_scale || !d->down_scale)) return EUX_ERR_BAD_ARG;
  if (((uintptr_t)d->x | (uintptr_t)d->out | (uintptr_t)d->w_gate_up | (uintptr_t)d->w_down | (uintptr_t)d->workspace) & 15) return EUX_ERR_BAD_ARG;
  const cudaStream_t st = (cudaStream_t)stream;
  const int w = kExpertThreads / 32;
  const dim3 up((d->inner + w - 1) / w, d->n_tokens * d->topk), down((d->hidden + w - 1) / w, d->n_tokens);
  if (d->fp8) {
    experts_up_kernel<true><<<up, kExpertThreads, 0, st>>>(*d);
    experts_down_kernel<true><<<down, kExpertThreads, 0, st>>>(*d);
  } else {
    experts_up_kernel<false><<<up, kExpertThreads, 0, st>>>(*d);
    experts_down_kernel<false><<<down, kExpertThreads, 0, st>>>(*d);
  }
  return (int)cudaGetLastError();
}

extern "C" int eux_experts_preload(void) {
  cudaFuncAttributes a;
  const void* kernels[] = {(const void*)experts_up_kernel<false>, (const void*)experts_up_kernel<true>,
                           (const void*)experts_down_kernel<false>, (const void*)experts_down_kernel<true>};
  for (const void* k : kernels)
    if (cudaError_t e = cudaFuncGetAttributes(&a, k); e != cudaSuccess) return (int)e;
  return 0;
}
