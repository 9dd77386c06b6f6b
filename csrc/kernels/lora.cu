// Low-rank adapters of many requests at once, added to what a shared projection gave:
//
//   v_t = A[i] x_t,   out_t = y_t + scale[i] * (B[i] v_t),   i = ids[t]
//
// What bounds it: with many tokens x, y and out go through HBM once, 2 (K + 2N) bytes per token for 2 r (K + N) operations, at
// ranks up to 128 still less than the tensor cores do in that time; with few tokens the adapters that are named, and latency.
// Two kernels, `shrink` (x to v) and `expand` (v to out), and for many tokens one in front:
//
// * Few tokens each stand for themselves: nothing is sorted, and requests that share an adapter read it again from the L2.
//   lora_shrink_one: a warp has some rows of A and a part of K, both straight into registers; its CTA adds up four parts, and expand up to
//   eight of these (with all parts added up by expand 16 tokens, 4096 x 4096, rank 64, took 9.8 us, 6.0 to 6.9 so).
//   lora_expand_one: a row of B is read by as many lanes as it has 16-byte pieces; a lane group makes eight columns side by side.
//   All in float32, no shared memory in the way: the chain id, A, v, B is four round trips to memory, and that is the time.
// * With more, lora_order orders the tokens by adapter, in one CTA, and cuts them into tiles of up to kLoraTile that share one.
//   lora_shrink: a cluster of CTAs has a tile, each a part of K; x and A go through a ring of stages with cp.async, four warps have
//   16 rows each. The parts are added up through the cluster's shared memory, in order: v is written once, nothing is added with
//   atomics.
//   lora_expand: a warp has 16 tokens and runs over a part of N. v is its first operand, two bfloat16 numbers that add up to it (what is
//   lost is 2^-16 of it, nothing beside the result's rounding), made in registers. y and B go through a ring of stages with cp.async: B
//   for all four warps, of y a lane fetches what it will need itself. Sums that are no numbers are made again in float32, so that an adapter's
//   infinities give with tiles what they give without.
//
// Measured, in a graph: one token, 4096 x 4096, rank 16: 4.1 us; 64 tokens, 8192 x 8192, rank 16, about 40 adapters: 9.9 us, with an adapter each
// 11.5 (most of expand's CTAs find no room beside shrink's, and fetch B only then); 777 tokens, 7168 x 2056, rank 40: 17.6 us (3.8 at the
// measured copy rate; order 2.5, the rest the two kernels' latency); 8192 tokens, 8192 x 8192, rank 16: 86.7 us (62 at the copy rate); 4096 x
// 4096, rank 64: 67.5 us (32), rank 128: 108.6 (32): A and B come through the L2 for every tile of 64 tokens, and expand multiplies twice.
#include <algorithm>
#include <mutex>

#include "eux_device.cuh"

namespace eux {

constexpr int kLoraPlain = 512;       // tokens up to which each may stand for itself ...
constexpr int64_t kLoraPlainBytes = int64_t(128) << 20;  // ... if the adapters that they read then come to no more than this,
constexpr int64_t kLoraSharedBytes = int64_t(48) << 20;  // or this where more than four tokens must share one on average
constexpr int kLoraTile = 64;         // tokens of a tile, with more
constexpr int kLoraThreads = 128;
constexpr int kLoraColumns = 128;     // of N in a stage of expand (8192 tokens, 4096 x 4096, rank 64: 67.5 us, 3 more with 64 columns and three or four stages)
constexpr int kLoraMaxSlices = 8;     // parts of K of a token, each of a CTA
constexpr int kLoraCluster = 8;       // parts of K of a tile at most

struct LoraParams {
  eux_lora_desc d;
  float* v;          // [slices][n_tokens][rank]; with tiles [n_tokens][rank] in the order of the tokens' places
  int4* tiles;       // {adapter, first place in order, tokens, -} of each tile
  int* order;        // tokens, those of an adapter side by side
  int* n_tiles;
  int slices;        // parts of K
  int per_slice;     // of K, a multiple of 256; without tiles of each warp
  int per_cta;       // of N, a multiple of 64; with tiles of 128
};

__device__ __forceinline__ uint32_t lora_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void lora_cp_16(uint32_t dst, const void* src, bool some) {  // zero if not
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(some ? 16 : 0) : "memory");
}
__device__ __forceinline__ void lora_cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void lora_cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void lora_ldsm_x4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void lora_ldsm_x2(uint32_t& a, uint32_t& b, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];" : "=r"(a), "=r"(b) : "r"(at) : "memory");
}
__device__ __forceinline__ void lora_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

constexpr int kOrderThreads = 1024;
constexpr size_t kOrderSmem = 200 * 1024;  // for the counts, where they fit

__device__ __forceinline__ int lora_adapter(const eux_lora_desc& d, int64_t token) {  // n_adapters: none
  const int id = __ldcg(d.ids + token);
  return (uint32_t)id < (uint32_t)d.n_adapters ? id : d.n_adapters;
}

// ---- a token at a time ----

__device__ __forceinline__ void lora_floats(const uint4& v, float (&f)[8]) {
  const __nv_bfloat162* const h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __bfloat1622float2(h[i]);
    f[2 * i] = t.x, f[2 * i + 1] = t.y;
  }
}

// Grid: tokens, and the CTAs that a token takes, each with eight rows of A and a part of K, a quarter of it for each warp.
__global__ void __launch_bounds__(kLoraThreads) lora_shrink_one_kernel(const __grid_constant__ LoraParams p) {
  const eux_lora_desc& d = p.d;
  constexpr int WARPS = kLoraThreads / 32;
  __shared__ float sums[WARPS][8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t token = blockIdx.x;
  const int slice = blockIdx.y % p.slices, r0 = blockIdx.y / p.slices * 8;
  wait_for_launch_before();
  allow_next_launch();  // expand's CTAs find room beside these, and have much to fetch that does not come from here
  const int adapter = lora_adapter(d, token);
  const int k0 = (slice * WARPS + warp) * p.per_slice, k1 = min(d.k, k0 + p.per_slice);
  if (adapter < d.n_adapters) {
    const __nv_bfloat16* const x = (const __nv_bfloat16*)d.x + token * d.x_stride;
    const __nv_bfloat16* const a = (const __nv_bfloat16*)d.a + ((int64_t)adapter * d.rank + r0) * d.k;
    float acc[8] = {};
    for (int k = k0 + lane * 8; k < k1; k += 256) {
      const uint4 xv = __ldg(reinterpret_cast<const uint4*>(x + k));
      uint4 av[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) av[r] = __ldg(reinterpret_cast<const uint4*>(a + (int64_t)r * d.k + k));
      float xf[8];
      lora_floats(xv, xf);
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        float af[8];
        lora_floats(av[r], af);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[r] = fmaf(af[i], xf[i], acc[r]);
      }
    }
    // row `lane & 7` is added up in the lanes that have this number, halving what each has
#pragma unroll
    for (int o = 4; o; o >>= 1)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (r < o) {
          const bool upper = lane & o;
          const float give = upper ? acc[r] : acc[r + o], keep = upper ? acc[r + o] : acc[r];
          acc[r] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    float v = acc[0];
    v += __shfl_xor_sync(0xffffffffu, v, 8);
    v += __shfl_xor_sync(0xffffffffu, v, 16);
    if (lane < 8) sums[warp][lane] = v;
    __syncthreads();
    if (threadIdx.x < 8) p.v[((int64_t)slice * d.n_tokens + token) * d.rank + r0 + lane] = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
  }
}

// A CTA's results, a column at a time.
__device__ __noinline__ void lora_one_plainly(const LoraParams& p, int64_t token, int adapter, float scale, const float (*parts)[EUX_LORA_MAX_RANK]) {
  const eux_lora_desc& d = p.d;
  const int n1 = min(d.n, (blockIdx.y + 1) * p.per_cta);
  for (int n = blockIdx.y * p.per_cta + threadIdx.x; n < n1; n += kLoraThreads) {
    const __nv_bfloat16* const b = (const __nv_bfloat16*)d.b + ((int64_t)adapter * d.n + n) * d.rank;
    float sum = 0.f;
    for (int r = 0; r < d.rank; ++r) {
      float v = 0.f;
      for (int s = 0; s < p.slices; ++s) v += parts[s][r];
      sum = fmaf(v, __bfloat162float(b[r]), sum);
    }
    const __nv_bfloat16* const y = (const __nv_bfloat16*)d.y + token * d.y_stride + n;
    ((__nv_bfloat16*)d.out)[token * d.out_stride + n] = __float2bfloat16_rn(fmaf(scale, sum, __bfloat162float(*y)));
  }
}

// Grid: tokens, parts of N. LANES: that share a row of B, a power of two of at least rank / 8.
template <int LANES>
__global__ void __launch_bounds__(kLoraThreads) lora_expand_one_kernel(const __grid_constant__ LoraParams p) {
  const eux_lora_desc& d = p.d;
  __shared__ float parts[kLoraMaxSlices][EUX_LORA_MAX_RANK];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t token = blockIdx.x;
  const int sub = lane % LANES, group = lane / LANES;
  constexpr int GROUPS = 32 / LANES;
  const int n0 = blockIdx.y * p.per_cta + (warp * GROUPS + group) * 8, n1 = min(d.n, blockIdx.y * p.per_cta + p.per_cta);
  // Shrink was through with its wait for whatever is in front when it let this in: all but v is there, in the L2 (an L1 may hold what
  // was there before).
  const int adapter = lora_adapter(d, token);
  const bool has = adapter < d.n_adapters, some = has && sub * 8 < d.rank;
  const __nv_bfloat16* const b = (const __nv_bfloat16*)d.b + (int64_t)(has ? adapter : 0) * d.n * d.rank + sub * 8;
  uint4 y, w[8];
  auto fetch = [&](int n) {  // n1 is a multiple of 8: eight columns are all there or not at all
    if (n < n1) {
      if (sub == 0) y = ld_cg_u4((const __nv_bfloat16*)d.y + token * d.y_stride + n);
      if (some)
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = ld_cg_u4(b + (int64_t)(n + i) * d.rank);
    }
  };
  fetch(n0);
  const float scale = has ? __ldcg(d.scale + adapter) : 0.f;
  wait_for_launch_before();
  float v[8] = {};
  if (has) {
    for (int i = threadIdx.x; i < p.slices * d.rank; i += kLoraThreads) {
      const int s = i / d.rank, r = i - s * d.rank;
      parts[s][r] = __ldcg(p.v + ((int64_t)s * d.n_tokens + token) * d.rank + r);
    }
    __syncthreads();
    if (!isfinite(scale)) {  // times each product's terms it would make NaN of signs that differ: behind their sum
      lora_one_plainly(p, token, adapter, scale, parts);
      allow_next_launch();
      return;
    }
    if (some)
      for (int s = 0; s < p.slices; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += parts[s][sub * 8 + i];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= scale;
  }
  for (int n = n0; n < n1; n += 4 * GROUPS * 8) {
    if (n != n0) fetch(n);
    float acc[8] = {};
    if (some) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float f[8];
        lora_floats(w[i], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i] = fmaf(f[j], v[j], acc[i]);
      }
    }
    const uint32_t mask = ((1u << LANES) - 1u) << (group * LANES);
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += __shfl_xor_sync(mask, acc[i], o);
    if (sub == 0) {
      if (has) {
        __nv_bfloat162* const y2 = reinterpret_cast<__nv_bfloat162*>(&y);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = __bfloat1622float2(y2[i]);
          y2[i] = __floats2bfloat162_rn(f.x + acc[2 * i], f.y + acc[2 * i + 1]);
        }
      }
      st_u4((__nv_bfloat16*)d.out + token * d.out_stride + n, y);
    }
  }
  allow_next_launch();
}

// ---- tiles of tokens that share an adapter ----

// Tokens ordered by adapter, those without one behind all (as adapter n_adapters: expand copies their rows), and the tiles, by one CTA.
// `counts` [n_adapters + 1]: null if they lie in shared memory. The order of an adapter's tokens is left to chance: a token's result
// does not depend on its place.
__global__ void __launch_bounds__(kOrderThreads) lora_order_kernel(const __grid_constant__ LoraParams p, int* counts) {
  extern __shared__ int order_smem[];
  __shared__ int sums[kOrderThreads / 32], tile_sums[kOrderThreads / 32];
  if (!counts) counts = order_smem;
  const eux_lora_desc& d = p.d;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, A = d.n_adapters + 1;
  // Behind the wait: counts that do not fit shared memory lie in the workspace, which may still be another call's until then.
  wait_for_launch_before();
  for (int i = threadIdx.x; i < A; i += kOrderThreads) counts[i] = 0;
  constexpr int KEPT = 8;  // a thread's first adapters, fetched at once
  int kept[KEPT];
#pragma unroll
  for (int q = 0; q < KEPT; ++q) {
    const int i = q * kOrderThreads + threadIdx.x;
    kept[q] = i < d.n_tokens ? lora_adapter(d, i) : -1;
  }
  __syncthreads();
  // A warp's neighbours with the same adapter count, and are placed, as one: prompts are runs of one adapter.
  auto add = [&](int a, bool place, int token) {
    const int before = __shfl_up_sync(0xffffffffu, a, 1);
    const uint32_t heads = __ballot_sync(0xffffffffu, lane == 0 || a != before);
    const int head = 31 - __clz(heads & (0xffffffffu >> (31 - lane)));
    const uint32_t behind = heads & ~(0xffffffffu >> (31 - lane));
    int at = 0;
    if (head == lane && a >= 0) at = atomicAdd(counts + a, (behind ? __ffs(behind) - 1 : 32) - lane);
    if (place) {
      at = __shfl_sync(0xffffffffu, at, head) + lane - head;
      if (a >= 0) p.order[at] = token;
    }
  };
  auto over_tokens = [&](bool place) {
#pragma unroll
    for (int q = 0; q < KEPT; ++q)
      if (q * kOrderThreads < d.n_tokens) add(kept[q], place, q * kOrderThreads + threadIdx.x);
    for (int i0 = KEPT * kOrderThreads; i0 < d.n_tokens; i0 += kOrderThreads) {
      const int i = i0 + threadIdx.x;
      add(i < d.n_tokens ? lora_adapter(d, i) : -1, place, i);
    }
  };
  over_tokens(false);
  __syncthreads();
  int all = 0, tiles = 0;
  for (int a0 = 0; a0 < A; a0 += kOrderThreads) {
    const int a = a0 + threadIdx.x, c = a < A ? counts[a] : 0, t = (c + kLoraTile - 1) / kLoraTile;
    int sum = c, tsum = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, sum, o), v = __shfl_up_sync(0xffffffffu, tsum, o);
      if (lane >= o) sum += u, tsum += v;
    }
    if (lane == 31) sums[warp] = sum, tile_sums[warp] = tsum;
    __syncthreads();
    const int u = sums[lane], v = tile_sums[lane];  // as many warps as lanes
    const int at = all + __reduce_add_sync(0xffffffffu, lane < warp ? u : 0) + sum - c;
    const int tile = tiles + __reduce_add_sync(0xffffffffu, lane < warp ? v : 0) + tsum - t;
    all += __reduce_add_sync(0xffffffffu, u), tiles += __reduce_add_sync(0xffffffffu, v);
    if (c) {
      const int n = (c + t - 1) / t;  // tiles of equal size
      for (int i = 0; i < t; ++i) p.tiles[tile + i] = make_int4(a, at + i * n, min(n, c - i * n), 0);
      counts[a] = at;  // from counts to places
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) *p.n_tiles = tiles;
  over_tokens(true);
  allow_next_launch();
}

struct LoraTile {
  int adapter, first, n;
};
__device__ __forceinline__ bool lora_tile(const LoraParams& p, int i, LoraTile* t) {
  const int4 v = __ldcg(p.tiles + i);  // there is room for one per CTA: fetched together with the number that are filled
  if (i >= __ldcg(p.n_tiles)) return false;
  t->adapter = v.x, t->first = v.y, t->n = v.z;
  return true;
}

__device__ __forceinline__ void lora_cluster_meets() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 lora_ld_cluster(uint32_t at, uint32_t cta) {
  uint32_t there;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(cta));
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(there) : "memory");
  return v;
}

// R8: ranks in eights, rounded up to a power of two. WIDE: stages of twice the size, half as many rounds of the CTA, for two CTAs of an SM.
template <int R8, bool WIDE>
struct LoraShrink {
  static constexpr int STEP = WIDE ? 128 : 64;  // of K in a stage
  static constexpr int STAGE = (kLoraTile + R8 * 8) * STEP * 2, STAGES = WIDE ? (R8 >= 16 ? 2 : 3) : (R8 >= 8 ? 3 : 4);
  static constexpr int RING = STAGES * STAGE, SUM = kLoraTile * (R8 * 8 + 4) * 4, BYTES = RING > SUM ? RING : SUM;
};
template <int R8, bool WIDE>
__global__ void __launch_bounds__(kLoraThreads) lora_shrink_kernel(const __grid_constant__ LoraParams p) {
  using S = LoraShrink<R8, WIDE>;
  constexpr int STEP = S::STEP, PIECES = STEP / 8;  // 16-byte pieces of a row
  constexpr int X = kLoraTile * STEP * 2, STAGE = S::STAGE, STAGES = S::STAGES;
  constexpr int LD = R8 * 8 + 4;               // floats between the tile's rows when it is added up
  extern __shared__ __align__(1024) unsigned char lora_smem_raw[];
  const eux_lora_desc& d = p.d;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  wait_for_launch_before();
  LoraTile t;
  if (!lora_tile(p, blockIdx.x, &t) || t.adapter == d.n_adapters) {  // all CTAs of the cluster
    allow_next_launch();
    return;
  }
  const int k0 = blockIdx.y * p.per_slice, k1 = min(d.k, k0 + p.per_slice), steps = max(0, (k1 - k0 + STEP - 1) / STEP);
  const uint32_t smem = lora_smem(lora_smem_raw);
  auto place = [](int row, int piece) { return row * (STEP * 2) + ((piece ^ (row & 7)) << 4); };
  // What this thread fetches of every stage: a piece of some rows of x and of A.
  constexpr int ROWS = kLoraThreads / PIECES, XR = kLoraTile / ROWS, AR = (R8 * 8 + ROWS - 1) / ROWS;
  const int row = threadIdx.x / PIECES, piece = threadIdx.x % PIECES;
  const __nv_bfloat16 *x[XR], *a[AR];
#pragma unroll
  for (int i = 0; i < XR; ++i) {
    const int r = row + ROWS * i;
    x[i] = r < t.n ? (const __nv_bfloat16*)d.x + p.order[t.first + r] * d.x_stride : nullptr;
  }
#pragma unroll
  for (int i = 0; i < AR; ++i) {
    const int r = row + ROWS * i;
    a[i] = r < d.rank ? (const __nv_bfloat16*)d.a + ((int64_t)t.adapter * d.rank + r) * d.k : nullptr;
  }
  auto fetch = [&](int step) {
    if (step < steps) {
      const uint32_t at = smem + step % STAGES * STAGE;
      const int k = k0 + step * STEP + piece * 8;
#pragma unroll
      for (int i = 0; i < XR; ++i) {
        const bool some = x[i] && k < k1;
        lora_cp_16(at + place(row + ROWS * i, piece), some ? x[i] + k : (const __nv_bfloat16*)d.x, some);
      }
#pragma unroll
      for (int i = 0; i < AR; ++i) {
        const bool some = a[i] && k < k1;
        if (row + ROWS * i < R8 * 8) lora_cp_16(at + X + place(row + ROWS * i, piece), some ? a[i] + k : (const __nv_bfloat16*)d.a, some);
      }
    }
    lora_cp_commit();
  };
  for (int s = 0; s < STAGES - 1; ++s) fetch(s);
  // Expand's CTAs fetch their first y and B beside this (2048 tokens, 4096 x 4096, rank 64: 29.0 us, 30.8 without); with ranks above 64 the
  // few that find room beside these hold it unevenly until the end (8192 tokens, rank 128: 139 us, 115 without).
  if (R8 < 16) allow_next_launch();
  float acc[R8][4] = {};
  for (int s = 0; s < steps; ++s) {
    lora_cp_wait<STAGES - 2>();
    __syncthreads();
    fetch(s + STAGES - 1);
    const uint32_t xs = smem + s % STAGES * STAGE, w = xs + X;
    if (warp * 16 < t.n) {
#pragma unroll
      for (int ks = 0; ks < STEP / 16; ++ks) {
        uint32_t av[4];
        lora_ldsm_x4(av, xs + place(warp * 16 + (lane & 15), ks * 2 + (lane >> 4)));
#pragma unroll
        for (int j = 0; j < R8; j += 2) {
          if (R8 > 1) {
            uint32_t b[4];
            lora_ldsm_x4(b, w + place(j * 8 + (lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)));
            lora_mma(acc[j], av, b[0], b[1]);
            lora_mma(acc[j + (R8 > 1)], av, b[2], b[3]);
          } else {
            uint32_t b0, b1;
            lora_ldsm_x2(b0, b1, w + place(lane & 7, ks * 2 + ((lane >> 3) & 1)));
            lora_mma(acc[j], av, b0, b1);
          }
        }
      }
    }
  }
  lora_cp_wait<0>();
  __syncthreads();
  float* const tile = reinterpret_cast<float*>(lora_smem_raw);
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int j = 0; j < R8; ++j)
      *reinterpret_cast<float2*>(tile + (warp * 16 + g + 8 * h) * LD + j * 8 + 2 * c) = make_float2(acc[j][2 * h], acc[j][2 * h + 1]);
  lora_cluster_meets();
  // each CTA adds up its share of the tile's rows, by the parts of K in their order; rows lie by place, not by token
  const int slices = p.slices, q = d.rank / 4;
  for (int i = threadIdx.x + blockIdx.y * kLoraThreads; i < t.n * q; i += kLoraThreads * slices) {
    const int r = i / q, e = i % q * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float4 o[kLoraCluster];  // all under way at once
#pragma unroll
    for (int s = 0; s < kLoraCluster; ++s)
      if (s < slices) o[s] = lora_ld_cluster(smem + (r * LD + e) * 4, s);
#pragma unroll
    for (int s = 0; s < kLoraCluster; ++s)
      if (s < slices) v.x += o[s].x, v.y += o[s].y, v.z += o[s].z, v.w += o[s].w;
    *reinterpret_cast<float4*>(p.v + (int64_t)(t.first + r) * d.rank + e) = v;
  }
  lora_cluster_meets();  // the others have read this one's
  if (R8 >= 16) allow_next_launch();
}

__device__ __forceinline__ float2 lora_times_zero(float x, float y, float2 to) {  // to + 0 * (x, y)
  asm("{\n\t.reg .b64 a, b, z;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%0, %1};\n\tmov.b64 z, 0;\n\t"
      "fma.rn.f32x2 b, a, z, b;\n\tmov.b64 {%0, %1}, b;\n\t}"
      : "+f"(to.x), "+f"(to.y)
      : "f"(x), "f"(y));
  return to;
}
// Of eight results those that are no numbers, made again of v in float32: as two bfloat16 numbers v is an infinity where it is above their
// largest, and the second of them, zero or of the other sign, makes NaN of an infinity of B. `y` lies in shared memory.
__device__ __forceinline__ void lora_again(__nv_bfloat16* out, uint32_t y, const float* v, const __nv_bfloat16* b, int rank, float scale) {
#pragma unroll 1
  for (int i = 0; i < 8; ++i) {
    if (isfinite(__bfloat162float(out[i]))) continue;
    float sum = 0.f;
#pragma unroll 1
    for (int r = 0; r < rank; ++r) sum = fmaf(__ldcg(v + r), __bfloat162float(b[(int64_t)i * rank + r]), sum);
    unsigned short of_y;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(of_y) : "r"(y + 2 * i) : "memory");
    out[i] = __float2bfloat16_rn(fmaf(scale, sum, __bfloat162float(__ushort_as_bfloat16(of_y))));
  }
}

// K16: ranks in 16s, rounded up to a power of two. Columns go 128 at a time, in runs of 32. A lane's eight columns of a run lie side
// by side, so that y and out are moved 16 bytes at a time: column 2c + i of the product's j-th eight is column 8c + 2j + i of the run,
// and the rows of B lie in shared memory in the product's order.
template <int K16>
struct LoraExpand {
  static constexpr int PITCH = K16 * 32 + 16;  // bytes between rows of B: eight rows on different banks
  static constexpr int B = kLoraColumns * PITCH, Y = kLoraTile * kLoraColumns * 2, STAGE = B + Y, STAGES = 2, BYTES = STAGES * STAGE;
};
template <int K16>
__global__ void __launch_bounds__(kLoraThreads) lora_expand_kernel(const __grid_constant__ LoraParams p) {
  using S = LoraExpand<K16>;
  extern __shared__ __align__(1024) unsigned char lora_smem_raw[];
  const eux_lora_desc& d = p.d;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  // Shrink was through with its wait for whatever is in front when it let this in: all but v is there, in the L2.
  LoraTile t;
  if (!lora_tile(p, blockIdx.x, &t)) return;  // the others, there are some, wait for what is in front: whatever follows may rely on that
  const bool has = t.adapter < d.n_adapters;
  const int row0 = warp * 16, n0 = blockIdx.y * p.per_cta, n1 = min(d.n, n0 + p.per_cta), steps = (n1 - n0 + kLoraColumns - 1) / kLoraColumns;
  // this lane's rows: g and g + 8 of the warp's
  const __nv_bfloat16* y_row[2];
  __nv_bfloat16* out_row[2];
  bool row[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = row0 + g + 8 * h;
    row[h] = r < t.n;
    const int64_t token = row[h] ? __ldcg(p.order + t.first + r) : 0;
    y_row[h] = (const __nv_bfloat16*)d.y + token * d.y_stride, out_row[h] = (__nv_bfloat16*)d.out + token * d.out_stride;
  }
  const __nv_bfloat16* const b = (const __nv_bfloat16*)d.b + (int64_t)(has ? t.adapter : 0) * d.n * d.rank;
  const uint32_t smem = lora_smem(lora_smem_raw);
  auto fetch = [&](int step) {
    if (step < steps) {
      const uint32_t at = smem + step % S::STAGES * S::STAGE;
      const int n = n0 + step * kLoraColumns;
      if (has) {
        constexpr int PIECES = K16 * 2;
#pragma unroll
        for (int i = threadIdx.x; i < kLoraColumns * PIECES; i += kLoraThreads) {
          const int place = i / PIECES, piece = i % PIECES, in = place & 7, eight = place >> 3 & 3;
          const int col = n + (place & ~31) + (in >> 1) * 8 + eight * 2 + (in & 1);
          const bool some = col < n1 && piece * 8 < d.rank;
          lora_cp_16(at + place * S::PITCH + piece * 16, some ? b + (int64_t)col * d.rank + piece * 8 : b, some);
        }
      }
      // y: what this lane needs itself
#pragma unroll
      for (int q = 0; q < kLoraColumns / 16; ++q) {
        const int h = q & 1, col = n + (q >> 1) * 32 + c * 8;
        if (row[h] && col < n1) lora_cp_16(at + S::B + (q * kLoraThreads + threadIdx.x) * 16, y_row[h] + col, true);
      }
    }
    lora_cp_commit();
  };
  for (int i = 0; i < S::STAGES - 1; ++i) fetch(i);
  uint32_t hi[K16][4], lo[K16][4];  // first operands
  const float scale = has ? __ldcg(d.scale + t.adapter) : 0.f;
  wait_for_launch_before();
#pragma unroll
  for (int k = 0; k < K16; ++k)
#pragma unroll
    for (int q = 0; q < 4; ++q) {  // row g + 8 (q & 1), columns 2c + 8 (q >> 1) and the next
      const int at = k * 16 + 2 * c + 8 * (q >> 1);
      float2 v = make_float2(0.f, 0.f);
      if (has && row[q & 1] && at < d.rank) v = __ldcg(reinterpret_cast<const float2*>(p.v + (int64_t)(t.first + row0 + g + 8 * (q & 1)) * d.rank + at));
      const __nv_bfloat162 u = __floats2bfloat162_rn(v.x, v.y);
      const float2 f = __bfloat1622float2(u);
      // nothing is lost of an infinity; what else is no number here is made again (lora_again)
      const __nv_bfloat162 l = __floats2bfloat162_rn(isinf(f.x) ? 0.f : v.x - f.x, isinf(f.y) ? 0.f : v.y - f.y);
      hi[k][q] = *reinterpret_cast<const uint32_t*>(&u), lo[k][q] = *reinterpret_cast<const uint32_t*>(&l);
    }
  float2 none = make_float2(0.f, 0.f);  // zero, or NaN where one of the last step's sums is no number
  auto again = [&](int step) {
    none = make_float2(0.f, 0.f);
#pragma unroll 1
    for (int q = 0; q < kLoraColumns / 16; ++q) {
      const int h = q & 1, col = n0 + step * kLoraColumns + (q >> 1) * 32 + c * 8;
      if ((h ? row[1] : row[0]) && col < n1)
        lora_again((h ? out_row[1] : out_row[0]) + col, smem + step % S::STAGES * S::STAGE + S::B + (q * kLoraThreads + threadIdx.x) * 16,
                   p.v + (int64_t)(t.first + row0 + g + 8 * h) * d.rank, b + (int64_t)col * d.rank, d.rank, scale);
    }
  };
  for (int s = 0; s < steps; ++s) {
    lora_cp_wait<S::STAGES - 2>();
    __syncthreads();
    if (none.x != 0.f || none.y != 0.f) again(s - 1);  // y is still there, until the fetch
    fetch(s + S::STAGES - 1);
    const uint32_t at = smem + s % S::STAGES * S::STAGE;
    if (row0 < t.n) {
#pragma unroll
      for (int run = 0; run < kLoraColumns / 32; ++run) {
        float acc[4][4] = {};
        if (has) {
#pragma unroll
          for (int k = 0; k < K16; ++k)
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
              uint32_t w[4];
              lora_ldsm_x4(w, at + (run * 32 + j * 8 + (lane & 7) + ((lane >> 4) << 3)) * S::PITCH + k * 32 + ((lane >> 3) & 1) * 16);
              lora_mma(acc[j], hi[k], w[0], w[1]), lora_mma(acc[j + 1], hi[k], w[2], w[3]);
              lora_mma(acc[j], lo[k], w[0], w[1]), lora_mma(acc[j + 1], lo[k], w[2], w[3]);
            }
        }
        const int col = n0 + s * kLoraColumns + run * 32 + c * 8;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (row[h] && col < n1) {
            uint4 y;
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(y.x), "=r"(y.y), "=r"(y.z), "=r"(y.w)
                         : "r"(at + S::B + ((run * 2 + h) * kLoraThreads + threadIdx.x) * 16)
                         : "memory");
            if (has) {
              __nv_bfloat162* const y2 = reinterpret_cast<__nv_bfloat162*>(&y);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float2 f = __bfloat1622float2(y2[j]);
                y2[j] = __floats2bfloat162_rn(fmaf(scale, acc[j][2 * h], f.x), fmaf(scale, acc[j][2 * h + 1], f.y));
                none = lora_times_zero(acc[j][2 * h], acc[j][2 * h + 1], none);
              }
            }
            st_u4(out_row[h] + col, y);
          }
      }
    }
  }
  if (none.x != 0.f || none.y != 0.f) again(steps - 1);
  lora_cp_wait<0>();
  allow_next_launch();
}

// ---- host ----

static int lora_check(const eux_lora_desc* d) {
  if (!d || d->n_tokens < 0 || d->k < 8 || d->n < 8 || d->rank < 8 || d->rank > EUX_LORA_MAX_RANK || d->n_adapters < 1) return EUX_ERR_BAD_ARG;
  if (d->k % 8 || d->n % 8 || d->rank % 8 || d->x_stride % 8 || d->y_stride % 8 || d->out_stride % 8) return EUX_ERR_BAD_ARG;
  if (d->n_adapters > (1 << 20) || d->k > (1 << 24) || d->n > (1 << 24)) return EUX_ERR_BAD_ARG;
  return 0;
}

struct LoraShape {
  bool one, wide;
  int tiles, slices, per_slice, parts, per_cta;
  size_t v_bytes, tile_bytes, order_bytes, count_bytes;
};
// Columns that a CTA of lora_expand_one makes at a time.
static int lora_width(int rank) { return rank <= 8 ? 1024 : rank <= 16 ? 512 : rank <= 32 ? 256 : rank <= 64 ? 128 : 64; }
static LoraShape lora_shape(const eux_lora_desc* d) {
  LoraShape s;
  constexpr int kSms = 148;
  // Each token for itself, or tiles of those that share an adapter. 64 adapters: 60 tokens, 8192 x 8192, rank 64, 126 MB, 27.2 and 39.4 us; 200
  // tokens, rank 16, 105 MB, 23.4 and 27.3; 256, 134 MB, 28.3 and 27.9. 16 adapters, rank 16: 128 tokens, 4096 x 4096, 34 MB, 8.9 and 9.9; 240
  // tokens, 63 MB, 12.9 and 10.2; 500 tokens, 131 MB, 22.8 and 11.5.
  s.one = d->n_tokens <= kLoraPlain &&
          (int64_t)d->n_tokens * d->rank * ((int64_t)d->k + d->n) * 2 <= (d->n_adapters >= d->n_tokens / 4 ? kLoraPlainBytes : kLoraSharedBytes);
  s.tiles = s.one ? d->n_tokens : (int)std::min<int64_t>(d->n_tokens, d->n_tokens / kLoraTile + (int64_t)d->n_adapters + 1);
  if (s.one) {
    // As many warps as the SMs have places for about, each with 256 of K or a multiple; expand once over its columns, likewise.
    const int64_t units = (int64_t)d->n_tokens * (d->rank / 8);
    constexpr int warps = kLoraThreads / 32;
    const int want = (int)std::max<int64_t>(1, std::min<int64_t>(warps * kLoraMaxSlices, 32 * kSms / units));
    s.per_slice = ((d->k + want - 1) / want + 255) / 256 * 256;
    s.slices = ((d->k + s.per_slice - 1) / s.per_slice + warps - 1) / warps;
    const int width = lora_width(d->rank), passes = (int)std::max<int64_t>(1, (int64_t)d->n_tokens * ((d->n + width - 1) / width) / (16 * kSms));
    s.per_cta = width * passes;
  } else {
    // Parts of K and of N that the SMs have places for at once: a second wave that is half empty costs as much as a full one.
    // How many tiles there will be is not known here: the tokens', and half a tile for each adapter, taken to be a dozen at most (1500 tokens of
    // 16 adapters, 2048 x 6144, rank 32: 21.2 us, 24.0 without; with every adapter that is there counted 4096 tokens of 9 of 64, 8192 x 8192, rank
    // 16, took 58 us, 49 so; it costs where few tokens name many: 256 tokens of 64 adapters, 8192 x 8192, rank 16, in tiles 27.6 us, 24.2 with 16
    // for the dozen).
    const int likely = (d->n_tokens + kLoraTile - 1) / kLoraTile + std::min({d->n_adapters, d->n_tokens / 16, 12}) / 2, r = d->rank;
    auto places = [](int smem) { return kSms * (227 * 1024 / (smem + 1024)); };
    const int shrink = places(r <= 8 ? LoraShrink<1, false>::BYTES : r <= 16 ? LoraShrink<2, false>::BYTES : r <= 32 ? LoraShrink<4, false>::BYTES
                              : r <= 64 ? LoraShrink<8, false>::BYTES : LoraShrink<16, false>::BYTES);
    const int expand = places(r <= 16 ? LoraExpand<1>::BYTES : r <= 32 ? LoraExpand<2>::BYTES : r <= 64 ? LoraExpand<4>::BYTES : LoraExpand<8>::BYTES);
    auto cluster = [&](int all) {
      int n = std::max(1, std::min({kLoraCluster, all / likely, (d->k + 255) / 256}));
      while (n & (n - 1)) n &= n - 1;
      return n;
    };
    // Wide stages where the tiles have places for them even if every adapter has one that is not full (777 tokens, 7168 x 2056, rank 40,
    // 24 adapters: 19.4 us, 22.5 with narrow ones; 8192 tokens, 4096 x 4096, rank 128: 110 and 113; but 256 tokens with 64 adapters
    // of rank 64: 33.8 and 31.1). Up to rank 32 a stage is mostly x, and narrow ones are as fast.
    s.wide = r > 32 && s.tiles * cluster(2 * kSms) <= 2 * kSms;
    const int want = cluster(s.wide ? 2 * kSms : shrink);
    s.per_slice = ((d->k + want - 1) / want + 255) / 256 * 256;
    s.slices = want;
    const int parts = std::max(1, std::min(expand / likely, (d->n + 127) / 128));
    s.per_cta = ((d->n + parts - 1) / parts + 127) / 128 * 128;
  }
  s.parts = (d->n + s.per_cta - 1) / s.per_cta;
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  s.v_bytes = up((size_t)(s.one ? s.slices : 1) * d->n_tokens * d->rank * 4);
  s.tile_bytes = s.one ? 0 : up(((size_t)s.tiles + 1) * 16);
  s.order_bytes = s.one ? 0 : up((size_t)d->n_tokens * 4);
  s.count_bytes = s.one ? 0 : up(((size_t)d->n_adapters + 1) * 4);
  return s;
}

// A launch that may begin while the kernel before it ends, of clusters of `cluster` CTAs along y.
static int lora_launch(void (*kernel)(LoraParams), dim3 grid, int cluster, size_t smem, cudaStream_t st, const LoraParams& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid, cfg.blockDim = dim3(kLoraThreads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1, attr[1].val.clusterDim.y = (unsigned)cluster, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = cluster > 1 ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, kernel, p);
}
template <int R8, bool WIDE>
static int lora_shrink(const LoraParams& p, const LoraShape& s, int dev, cudaStream_t st) {
  constexpr size_t smem = LoraShrink<R8, WIDE>::BYTES;
  if (smem > 48 * 1024)
    if (cudaError_t e = allow_smem<lora_shrink_kernel<R8, WIDE>>(dev, smem); e != cudaSuccess) return (int)e;
  return lora_launch(lora_shrink_kernel<R8, WIDE>, dim3(s.tiles, s.slices), s.slices, smem, st, p);
}

template <int K16>
static int lora_expand(const LoraParams& p, const LoraShape& s, int dev, cudaStream_t st) {
  constexpr size_t smem = LoraExpand<K16>::BYTES;
  if (smem > 48 * 1024)
    if (cudaError_t e = allow_smem<lora_expand_kernel<K16>>(dev, smem); e != cudaSuccess) return (int)e;
  return lora_launch(lora_expand_kernel<K16>, dim3(s.tiles, s.parts), 1, smem, st, p);
}

static int lora_run_one(const LoraParams& p, const LoraShape& s, cudaStream_t st) {
  const int r = p.d.rank;
  if (int rc = lora_launch(lora_shrink_one_kernel, dim3(s.tiles, s.slices * (r / 8)), 1, 0, st, p)) return rc;
  return lora_launch(r <= 8 ? lora_expand_one_kernel<1> : r <= 16 ? lora_expand_one_kernel<2> : r <= 32 ? lora_expand_one_kernel<4>
                     : r <= 64 ? lora_expand_one_kernel<8> : lora_expand_one_kernel<16>, dim3(s.tiles, s.parts), 1, 0, st, p);
}
static int lora_run_tiles(const LoraParams& p, const LoraShape& s, int dev, cudaStream_t st) {
  const int r = p.d.rank;
  const int rc = r <= 8 ? lora_shrink<1, false>(p, s, dev, st) : r <= 16 ? lora_shrink<2, false>(p, s, dev, st)
                 : r <= 32 ? lora_shrink<4, false>(p, s, dev, st)
                 : r <= 64 ? (s.wide ? lora_shrink<8, true>(p, s, dev, st) : lora_shrink<8, false>(p, s, dev, st))
                           : (s.wide ? lora_shrink<16, true>(p, s, dev, st) : lora_shrink<16, false>(p, s, dev, st));
  if (rc) return rc;
  return r <= 16 ? lora_expand<1>(p, s, dev, st) : r <= 32 ? lora_expand<2>(p, s, dev, st) : r <= 64 ? lora_expand<4>(p, s, dev, st) : lora_expand<8>(p, s, dev, st);
}

}  // namespace eux

using namespace eux;

extern "C" size_t eux_lora_workspace_bytes(const eux_lora_desc* d) {
  if (lora_check(d)) return 0;
  if (d->n_tokens == 0) return 16;
  const LoraShape s = lora_shape(d);
  return s.v_bytes + s.tile_bytes + s.order_bytes + s.count_bytes;
}

extern "C" int eux_lora_launch(const eux_lora_desc* d, void* stream) {
  if (int rc = lora_check(d)) return rc;
  if (d->n_tokens == 0) return 0;
  if (!d->x || !d->ids || !d->y || !d->out || !d->a || !d->b || !d->scale || !d->workspace) return EUX_ERR_BAD_ARG;
  if (((uintptr_t)d->x | (uintptr_t)d->y | (uintptr_t)d->out | (uintptr_t)d->a | (uintptr_t)d->b | (uintptr_t)d->workspace) & 15) return EUX_ERR_BAD_ARG;
  const cudaStream_t st = (cudaStream_t)stream;
  // Threads that share a stream share a workspace: their launches must not mix.
  static std::mutex launching;
  std::lock_guard<std::mutex> lock(launching);
  const LoraShape s = lora_shape(d);
  char* at = (char*)d->workspace;
  LoraParams p = {};
  p.d = *d;
  p.v = (float*)at, at += s.v_bytes;
  p.slices = s.slices, p.per_slice = s.per_slice, p.per_cta = s.per_cta;
  int dev = 0;
  cudaGetDevice(&dev);
  if (s.one) return lora_run_one(p, s, st);
  p.n_tiles = (int*)at, p.tiles = (int4*)at + 1, at += s.tile_bytes;
  p.order = (int*)at, at += s.order_bytes;
  const size_t count_bytes = ((size_t)d->n_adapters + 1) * 4;
  const bool in_smem = count_bytes <= kOrderSmem;
  if (cudaError_t e = allow_smem<lora_order_kernel>(dev, kOrderSmem); e != cudaSuccess) return (int)e;
  if (int rc = launch_early(lora_order_kernel, 1, kOrderThreads, in_smem ? count_bytes : 0, st, p, in_smem ? (int*)nullptr : (int*)at)) return rc;
  return lora_run_tiles(p, s, dev, st);
}

extern "C" int eux_lora_preload(void) {
  cudaFuncAttributes a;
  const void* kernels[] = {(const void*)lora_shrink_one_kernel, (const void*)lora_expand_one_kernel<1>, (const void*)lora_expand_one_kernel<2>,
                           (const void*)lora_expand_one_kernel<4>, (const void*)lora_expand_one_kernel<8>, (const void*)lora_expand_one_kernel<16>,
                           (const void*)lora_order_kernel, (const void*)lora_shrink_kernel<1, false>, (const void*)lora_shrink_kernel<2, false>,
                           (const void*)lora_shrink_kernel<4, false>, (const void*)lora_shrink_kernel<8, false>, (const void*)lora_shrink_kernel<8, true>,
                           (const void*)lora_shrink_kernel<16, false>, (const void*)lora_shrink_kernel<16, true>,
                           (const void*)lora_expand_kernel<1>, (const void*)lora_expand_kernel<2>, (const void*)lora_expand_kernel<4>, (const void*)lora_expand_kernel<8>};
  for (const void* k : kernels)
    if (cudaError_t e = cudaFuncGetAttributes(&a, k); e != cudaSuccess) return (int)e;
  return 0;
}
