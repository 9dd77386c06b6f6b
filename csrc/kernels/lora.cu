// Low-rank adapters of many requests at once, added to what a shared projection gave:
//
//   v_t = A[i] x_t,   out_t = y_t + scale[i] * (B[i] v_t),   i = ids[t]
//
// One CTA per token.
#include <algorithm>

#include "eux_device.cuh"

namespace eux {

constexpr int kLoraThreads = 256;

__global__ void __launch_bounds__(kLoraThreads) lora_kernel(eux_lora_desc d) {
  __shared__ float v[EUX_LORA_MAX_RANK];
  const int64_t t = blockIdx.x;
  const int id = d.ids[t], lane = threadIdx.x & 31;
  const bool has = id >= 0 && id < d.n_adapters;
  if (has) {
    const __nv_bfloat16* x = (const __nv_bfloat16*)d.x + t * d.x_stride;
    for (int r = threadIdx.x >> 5; r < d.rank; r += kLoraThreads / 32) {
      const __nv_bfloat16* a = (const __nv_bfloat16*)d.a + ((int64_t)id * d.rank + r) * d.k;
      float acc = 0.f;
      for (int k = lane; k < d.k; k += 32) acc += __bfloat162float(a[k]) * __bfloat162float(x[k]);
      for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
      if (lane == 0) v[r] = acc;
    }
  }
  __syncthreads();
  const float s = has ? d.scale[id] : 0.f;
  for (int n = threadIdx.x; n < d.n; n += kLoraThreads) {
    float acc = 0.f;
    if (has) {
      const __nv_bfloat16* b = (const __nv_bfloat16*)d.b + ((int64_t)id * d.n + n) * d.rank;
      for (int r = 0; r < d.rank; ++r) acc += __bfloat162float(b[r]) * v[r];
    }
    const __nv_bfloat16 y = ((const __nv_bfloat16*)d.y)[t * d.y_stride + n];
    ((__nv_bfloat16*)d.out)[t * d.out_stride + n] = has ? __float2bfloat16_rn(__bfloat162float(y) + s * acc) : y;
  }
}

static int lora_check(const eux_lora_desc* d) {
  if (!d || d->n_tokens < 0 || d->k < 8 || d->n < 8 || d->rank < 8 || d->rank > EUX_LORA_MAX_RANK || d->n_adapters < 1) return EUX_ERR_BAD_ARG;
  if (d->k % 8 || d->n % 8 || d->rank % 8 || d->x_stride % 8 || d->y_stride % 8 || d->out_stride % 8) return EUX_ERR_BAD_ARG;
  return 0;
}

}  // namespace eux

using namespace eux;

extern "C" size_t eux_lora_workspace_bytes(const eux_lora_desc* d) { return lora_check(d) ? 0 : 16; }

extern "C" int eux_lora_launch(const eux_lora_desc* d, void* stream) {
  if (int rc = lora_check(d)) return rc;
  if (d->n_tokens == 0) return 0;
  if (!d->x || !d->ids || !d->y || !d->out || !d->a || !d->b || !d->scale || !d->workspace) return EUX_ERR_BAD_ARG;
  if (((uintptr_t)d->x | (uintptr_t)d->y | (uintptr_t)d->out | (uintptr_t)d->a | (uintptr_t)d->b | (uintptr_t)d->workspace) & 15) return EUX_ERR_BAD_ARG;
  lora_kernel<<<d->n_tokens, kLoraThreads, 0, (cudaStream_t)stream>>>(*d);
  return (int)cudaGetLastError();
}

extern "C" int eux_lora_preload(void) {
  cudaFuncAttributes a;
  return (int)cudaFuncGetAttributes(&a, lora_kernel);
}
