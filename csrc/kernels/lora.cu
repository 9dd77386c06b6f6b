// Low-rank adapters of many requests at once, added to what a shared projection gave:
//
//   v_t = A[i] x_t,   out_t = y_t + scale[i] * (B[i] v_t),   i = ids[t]
//
// What bounds it: with many tokens x, y and out go through HBM once, 2 (K + 2N) bytes per token for 2 r (K + N) operations, at
// ranks up to 128 still less than the tensor cores do in that time; with few tokens the adapters that are named, and latency.
// Two kernels, `shrink` (x to v) and `expand` (v to out):
//
// * Tokens come in tiles that share an adapter. Up to kLoraPlain tokens each token is a tile: nothing is sorted, and requests that
//   share an adapter read it again from the L2. With more, a third kernel in front orders the tokens by adapter, in one CTA.
// * shrink: a CTA has a tile and a part of K. x and A go through a ring of stages with cp.async; its four warps share the tile's
//   rows (16 each) or, where the tile is one row, the part's K. v stays float32, one slice per part of K: nothing is added with
//   atomics, expand adds the slices in their order.
// * expand: a warp has 16 tokens and runs over a part of N, 32 columns at a time. v is its first operand, two bfloat16 numbers that add
//   up to it (what is lost is 2^-16 of it, nothing beside the result's rounding), made in registers; B comes from L1 and L2 straight
//   into registers, y is fetched before the product and out written behind it, 16 bytes per lane.
#include <algorithm>

#include "eux_device.cuh"

namespace eux {

constexpr int kLoraPlain = 64;        // tokens up to which each is a tile of its own
constexpr int kLoraTile = 64;         // tokens of a tile, with more
constexpr int kLoraThreads = 128;
constexpr int kLoraStages = 4;
constexpr int kLoraMaxSlices = 32;

struct LoraParams {
  eux_lora_desc d;
  float* v;          // [slices][n_tokens][rank]
  int4* tiles;       // {adapter, first place in order, tokens, -} of each tile; null: tile t is token t
  int* order;        // tokens, those of an adapter side by side
  int* n_tiles;
  int slices;        // parts of K
  int per_slice;     // of K, a multiple of 64
  int per_cta;       // of N, a multiple of 32
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
constexpr int kOrderWarps = kOrderThreads / 32;
constexpr size_t kOrderSmem = 200 * 1024;  // for the counts, where they fit

// Where a tile's tokens are.
struct LoraTile {
  int adapter, first, n;
};
__device__ __forceinline__ bool lora_tile(const LoraParams& p, int i, LoraTile* t) {
  const eux_lora_desc& d = p.d;
  if (!p.tiles) {
    const int id = d.ids[i];
    t->adapter = (uint32_t)id < (uint32_t)d.n_adapters ? id : d.n_adapters, t->first = i, t->n = 1;
    return true;
  }
  if (i >= *p.n_tiles) return false;
  const int4 v = p.tiles[i];
  t->adapter = v.x, t->first = v.y, t->n = v.z;
  return true;
}

// Tokens ordered by adapter, those without one behind all (as adapter n_adapters: expand copies their rows), and the tiles. One CTA,
// whose warps each count a run of tokens per adapter, `counts` [n_adapters + 1][warps]: null if they lie in shared memory.
__global__ void __launch_bounds__(kOrderThreads) lora_order_kernel(const __grid_constant__ LoraParams p, int* counts) {
  extern __shared__ int order_smem[];
  if (!counts) counts = order_smem;
  __shared__ int sums[kOrderWarps], tile_sums[kOrderWarps];
  const eux_lora_desc& d = p.d;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, A = d.n_adapters + 1;
  const int each = ((d.n_tokens + kOrderWarps - 1) / kOrderWarps + 31) & ~31, lo = min(d.n_tokens, warp * each), hi = min(d.n_tokens, lo + each);
  const uint32_t below = (1u << lane) - 1u;
  wait_for_launch_before();
  for (int i = threadIdx.x; i < A * kOrderWarps; i += kOrderThreads) counts[i] = 0;
  __syncthreads();
  auto adapter = [&](int i) {
    const int id = i < hi ? d.ids[i] : -1;
    return (uint32_t)id < (uint32_t)d.n_adapters ? id : d.n_adapters;
  };
  for (int i = lo + lane; i < hi; i += 32) atomicAdd(counts + adapter(i) * kOrderWarps + warp, 1);
  __syncthreads();
  int all = 0, tiles = 0;
  for (int a0 = 0; a0 < A; a0 += kOrderThreads) {
    const int a = a0 + threadIdx.x;
    int c = 0;
    if (a < A)
      for (int w = 0; w < kOrderWarps; ++w) c += counts[a * kOrderWarps + w];
    const int t = (c + kLoraTile - 1) / kLoraTile;
    int sum = c, tsum = t;
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, sum, o), v = __shfl_up_sync(0xffffffffu, tsum, o);
      if (lane >= o) sum += u, tsum += v;
    }
    if (lane == 31) sums[warp] = sum, tile_sums[warp] = tsum;
    __syncthreads();
    int at = all, tile = tiles;
    for (int w = 0; w < kOrderWarps; ++w) {
      if (w < warp) at += sums[w], tile += tile_sums[w];
      all += sums[w], tiles += tile_sums[w];
    }
    at += sum - c, tile += tsum - t;
    if (c) {
      // tiles of equal size
      const int n = (c + t - 1) / t;
      for (int i = 0; i < t; ++i) p.tiles[tile + i] = make_int4(a, at + i * n, min(n, c - i * n), 0);
      for (int w = 0; w < kOrderWarps; ++w) {  // from counts to places
        const int m = counts[a * kOrderWarps + w];
        counts[a * kOrderWarps + w] = at;
        at += m;
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) *p.n_tiles = tiles;
  for (int i0 = lo; i0 < hi; i0 += 32) {
    const int i = i0 + lane, a = adapter(i);
    const uint32_t same = __match_any_sync(0xffffffffu, i < hi ? a : -1);
    const int before = __popc(same & below);
    if (i < hi) p.order[counts[a * kOrderWarps + warp] + before] = i;
    __syncwarp();
    if (i < hi && before == 0) counts[a * kOrderWarps + warp] += __popc(same);
    __syncwarp();
  }
  allow_next_launch();
}

// What a stage of shrink holds.
template <int R8, bool ONE>
struct LoraStage {
  static constexpr int KS = ONE && R8 == 16 ? 2 : 4;           // of K: 16s per warp
  static constexpr int STEP = ONE ? KS * 64 : KS * 16;         // of K: a token's is shared by the warps
  static constexpr int ROWS = ONE ? 1 : kLoraTile;             // of x
  static constexpr int X = ROWS * STEP * 2, BYTES = X + R8 * 8 * STEP * 2;
};

// R8: ranks in eights, rounded up to a power of two. ONE: tiles of one token, whose warps share K.
template <int R8, bool ONE>
__global__ void __launch_bounds__(kLoraThreads) lora_shrink_kernel(const __grid_constant__ LoraParams p) {
  using S = LoraStage<R8, ONE>;
  constexpr int STEP = S::STEP, ROWS = S::ROWS, X = S::X, PIECES = STEP / 8;  // 16-byte pieces of a row
  extern __shared__ __align__(1024) unsigned char lora_smem_raw[];
  const eux_lora_desc& d = p.d;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  wait_for_launch_before();
  LoraTile t;
  if (!lora_tile(p, blockIdx.x, &t) || t.adapter == d.n_adapters) {
    allow_next_launch();
    return;
  }
  const int k0 = blockIdx.y * p.per_slice, k1 = min(d.k, k0 + p.per_slice), steps = (k1 - k0 + STEP - 1) / STEP;
  const uint32_t smem = lora_smem(lora_smem_raw);
  const __nv_bfloat16* const a = (const __nv_bfloat16*)d.a + (int64_t)t.adapter * d.rank * d.k;
  // a row's pieces are swizzled within 128 bytes
  auto place = [](int row, int piece) { return row * (STEP * 2) + (piece & ~7) * 16 + (((piece ^ row) & 7) << 4); };
  auto fetch = [&](int step) {
    if (step < steps) {
      const uint32_t at = smem + step % kLoraStages * S::BYTES;
      const int k = k0 + step * STEP;
      for (int i = threadIdx.x; i < ROWS * PIECES; i += kLoraThreads) {
        const int row = i / PIECES, piece = i % PIECES;
        const bool some = row < t.n && k + piece * 8 < k1;
        const int64_t token = some ? (p.tiles ? p.order[t.first + row] : t.first) : 0;
        lora_cp_16(at + place(row, piece), (const __nv_bfloat16*)d.x + token * d.x_stride + (some ? k + piece * 8 : 0), some);
      }
      for (int i = threadIdx.x; i < R8 * 8 * PIECES; i += kLoraThreads) {
        const int row = i / PIECES, piece = i % PIECES;
        const bool some = row < d.rank && k + piece * 8 < k1;
        lora_cp_16(at + X + place(row, piece), a + (some ? (int64_t)row * d.k + k + piece * 8 : 0), some);
      }
    }
    lora_cp_commit();
  };
  for (int s = 0; s < kLoraStages - 1; ++s) fetch(s);
  float acc[R8][4] = {};
  for (int s = 0; s < steps; ++s) {
    lora_cp_wait<kLoraStages - 2>();
    __syncthreads();
    fetch(s + kLoraStages - 1);
    const uint32_t x = smem + s % kLoraStages * S::BYTES, w = x + X;
    if (ONE || warp * 16 < t.n) {
#pragma unroll
      for (int ks = 0; ks < S::KS; ++ks) {
        const int piece = (ONE ? warp * S::KS * 2 : 0) + ks * 2;
        uint32_t av[4];
        if (ONE) {
          // the token is row 0, which lanes 0 to 3 hold; the others hold zeros
          av[0] = av[1] = av[2] = av[3] = 0;
          if (g == 0) {
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(av[0]) : "r"(x + place(0, piece) + 4 * c) : "memory");
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(av[2]) : "r"(x + place(0, piece + 1) + 4 * c) : "memory");
          }
        } else {
          lora_ldsm_x4(av, x + place(warp * 16 + (lane & 15), piece + (lane >> 4)));
        }
#pragma unroll
        for (int j = 0; j < R8; j += 2) {
          if (R8 > 1) {
            uint32_t b[4];
            lora_ldsm_x4(b, w + place(j * 8 + (lane & 7) + ((lane >> 4) << 3), piece + ((lane >> 3) & 1)));
            lora_mma(acc[j], av, b[0], b[1]);
            lora_mma(acc[j + (R8 > 1)], av, b[2], b[3]);
          } else {
            uint32_t b0, b1;
            lora_ldsm_x2(b0, b1, w + place(lane & 7, piece + ((lane >> 3) & 1)));
            lora_mma(acc[j], av, b0, b1);
          }
        }
      }
    }
  }
  lora_cp_wait<0>();
  float* const v = p.v + (int64_t)blockIdx.y * d.n_tokens * d.rank;
  if (ONE) {
    __shared__ float part[4][R8 * 8];
    if (g == 0)
#pragma unroll
      for (int j = 0; j < R8; ++j) part[warp][j * 8 + 2 * c] = acc[j][0], part[warp][j * 8 + 2 * c + 1] = acc[j][1];
    __syncthreads();
    for (int i = threadIdx.x; i < d.rank; i += kLoraThreads) v[(int64_t)t.first * d.rank + i] = (part[0][i] + part[1][i]) + (part[2][i] + part[3][i]);
  } else {
    // by place, not by token: expand reads a tile's rows side by side
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = warp * 16 + g + 8 * h;
      if (row < t.n)
#pragma unroll
        for (int j = 0; j < R8; ++j)
          if (j * 8 < d.rank) *reinterpret_cast<float2*>(v + (int64_t)(t.first + row) * d.rank + j * 8 + 2 * c) = make_float2(acc[j][2 * h], acc[j][2 * h + 1]);
    }
  }
  allow_next_launch();
}

// K32: ranks in 32s. A lane's eight values of K are side by side (the order of K is the product's own affair), and so are its eight
// columns of 32 (column 2c + i of the product's n-th eight is 8c + 2n + i of the 32).
template <int K32, bool ONE>
__global__ void __launch_bounds__(kLoraThreads) lora_expand_kernel(const __grid_constant__ LoraParams p) {
  const eux_lora_desc& d = p.d;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  wait_for_launch_before();
  LoraTile t;
  if (!lora_tile(p, blockIdx.x, &t)) {
    allow_next_launch();
    return;
  }
  const bool has = t.adapter < d.n_adapters;
  // a tile of one token: the warps share the columns
  const int row0 = ONE ? 0 : warp * 16, n0 = blockIdx.y * p.per_cta, n1 = min(d.n, n0 + p.per_cta);
  if (row0 < t.n) {
    // this lane's rows: g and g + 8 of the warp's
    int64_t token[2];
    bool row[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = row0 + g + 8 * h;
      row[h] = r < t.n;
      token[h] = row[h] ? (p.tiles ? p.order[t.first + r] : t.first) : 0;
    }
    uint32_t hi[K32][2][4], lo[K32][2][4];  // first operands of 16 of K
    if (has) {
      const float scale = d.scale[t.adapter];
#pragma unroll
      for (int k = 0; k < K32; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[8] = {};
          if (row[h] && k * 32 + c * 8 < d.rank) {
            const float* at = p.v + (int64_t)(t.first + row0 + g + 8 * h) * d.rank + k * 32 + c * 8;
            for (int s = 0; s < p.slices; ++s, at += (int64_t)d.n_tokens * d.rank) {
              const float4 q0 = __ldcg(reinterpret_cast<const float4*>(at)), q1 = __ldcg(reinterpret_cast<const float4*>(at) + 1);
              v[0] += q0.x, v[1] += q0.y, v[2] += q0.z, v[3] += q0.w, v[4] += q1.x, v[5] += q1.y, v[6] += q1.z, v[7] += q1.w;
            }
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float v0 = v[2 * q] * scale, v1 = v[2 * q + 1] * scale;
            const __nv_bfloat162 u = __floats2bfloat162_rn(v0, v1);
            const float2 f = __bfloat1622float2(u);
            // nothing is lost of an infinity
            const __nv_bfloat162 w = __floats2bfloat162_rn(isinf(f.x) ? 0.f : v0 - f.x, isinf(f.y) ? 0.f : v1 - f.y);
            // pairs 0 and 1 are the first 16's k = 2c and 2c + 8, pairs 2 and 3 the second's
            hi[k][q >> 1][(q & 1) * 2 + h] = *reinterpret_cast<const uint32_t*>(&u);
            lo[k][q >> 1][(q & 1) * 2 + h] = *reinterpret_cast<const uint32_t*>(&w);
          }
        }
    }
    const __nv_bfloat16* const b = (const __nv_bfloat16*)d.b + (int64_t)(has ? t.adapter : 0) * d.n * d.rank;
    for (int n = n0 + (ONE ? warp * 32 : 0); n < n1; n += ONE ? 128 : 32) {
      uint4 y[2];
      const int col = n + c * 8;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (row[h] && col < d.n) y[h] = *reinterpret_cast<const uint4*>((const __nv_bfloat16*)d.y + token[h] * d.y_stride + col);
      if (has) {
        float acc[4][4] = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = n + (g >> 1) * 8 + j * 2 + (g & 1);  // the row of B for this lane's column
#pragma unroll
          for (int k = 0; k < K32; ++k) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (at < d.n && k * 32 + c * 8 < d.rank) w = __ldg(reinterpret_cast<const uint4*>(b + (int64_t)at * d.rank + k * 32 + c * 8));
            lora_mma(acc[j], hi[k][0], w.x, w.y), lora_mma(acc[j], hi[k][1], w.z, w.w);
            lora_mma(acc[j], lo[k][0], w.x, w.y), lora_mma(acc[j], lo[k][1], w.z, w.w);
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          __nv_bfloat162* const y2 = reinterpret_cast<__nv_bfloat162*>(&y[h]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = __bfloat1622float2(y2[j]);
            y2[j] = __floats2bfloat162_rn(f.x + acc[j][2 * h], f.y + acc[j][2 * h + 1]);
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (row[h] && col < d.n) st_u4((__nv_bfloat16*)d.out + token[h] * d.out_stride + col, y[h]);
    }
  }
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
  bool one;
  int tiles, slices, per_slice, parts, per_cta;
  size_t v_bytes, tile_bytes, order_bytes, count_bytes;
};
static LoraShape lora_shape(const eux_lora_desc* d) {
  LoraShape s;
  constexpr int kSms = 148;
  s.one = d->n_tokens <= kLoraPlain;
  s.tiles = s.one ? d->n_tokens : (int)std::min<int64_t>(d->n_tokens, d->n_tokens / kLoraTile + (int64_t)d->n_adapters + 1);
  const int likely = s.one ? d->n_tokens : (d->n_tokens + kLoraTile - 1) / kLoraTile;
  // Parts of K for about four CTAs per SM, of 256 (512: a token's) at least
  const int step = s.one ? 512 : 256;
  int want = std::max(1, std::min(kLoraMaxSlices, 4 * kSms / likely));
  want = std::min(want, (d->k + step - 1) / step);
  s.per_slice = ((d->k + want - 1) / want + 255) / 256 * 256;
  s.slices = (d->k + s.per_slice - 1) / s.per_slice;
  // Parts of N likewise, of 128 at least
  int parts = std::max(1, std::min(4 * kSms / likely, (d->n + 127) / 128));
  s.per_cta = ((d->n + parts - 1) / parts + 127) / 128 * 128;
  s.parts = (d->n + s.per_cta - 1) / s.per_cta;
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  s.v_bytes = up((size_t)s.slices * d->n_tokens * d->rank * 4);
  s.tile_bytes = s.one ? 0 : up(((size_t)s.tiles + 1) * 16);
  s.order_bytes = s.one ? 0 : up((size_t)d->n_tokens * 4);
  s.count_bytes = s.one ? 0 : up(((size_t)d->n_adapters + 1) * kOrderWarps * 4);
  return s;
}

template <int R8, bool ONE>
static int lora_shrink(const LoraParams& p, const LoraShape& s, int dev, cudaStream_t st) {
  constexpr size_t smem = (size_t)kLoraStages * LoraStage<R8, ONE>::BYTES;
  if (smem > 48 * 1024)
    if (cudaError_t e = allow_smem<lora_shrink_kernel<R8, ONE>>(dev, smem); e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(s.tiles, s.slices), cfg.blockDim = dim3(kLoraThreads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr, cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, lora_shrink_kernel<R8, ONE>, p);
}
template <int K32, bool ONE>
static int lora_expand(const LoraParams& p, const LoraShape& s, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(s.tiles, s.parts), cfg.blockDim = dim3(kLoraThreads), cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr, cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, lora_expand_kernel<K32, ONE>, p);
}

template <bool ONE>
static int lora_run(const LoraParams& p, const LoraShape& s, int dev, cudaStream_t st) {
  const int r = p.d.rank;
  int rc = r <= 8 ? lora_shrink<1, ONE>(p, s, dev, st) : r <= 16 ? lora_shrink<2, ONE>(p, s, dev, st) : r <= 32 ? lora_shrink<4, ONE>(p, s, dev, st)
           : r <= 64 ? lora_shrink<8, ONE>(p, s, dev, st) : lora_shrink<16, ONE>(p, s, dev, st);
  if (rc) return rc;
  return r <= 32 ? lora_expand<1, ONE>(p, s, st) : r <= 64 ? lora_expand<2, ONE>(p, s, st) : lora_expand<4, ONE>(p, s, st);
}

template <bool ONE>
static int lora_preload() {
  cudaFuncAttributes a;
  const void* kernels[] = {(const void*)lora_shrink_kernel<1, ONE>, (const void*)lora_shrink_kernel<2, ONE>, (const void*)lora_shrink_kernel<4, ONE>,
                           (const void*)lora_shrink_kernel<8, ONE>, (const void*)lora_shrink_kernel<16, ONE>, (const void*)lora_expand_kernel<1, ONE>,
                           (const void*)lora_expand_kernel<2, ONE>, (const void*)lora_expand_kernel<4, ONE>, (const void*)lora_order_kernel};
  for (const void* k : kernels)
    if (cudaError_t e = cudaFuncGetAttributes(&a, k); e != cudaSuccess) return (int)e;
  return 0;
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
  const LoraShape s = lora_shape(d);
  char* at = (char*)d->workspace;
  LoraParams p = {};
  p.d = *d;
  p.v = (float*)at, at += s.v_bytes;
  p.slices = s.slices, p.per_slice = s.per_slice, p.per_cta = s.per_cta;
  int dev = 0;
  cudaGetDevice(&dev);
  if (s.one) return lora_run<true>(p, s, dev, st);
  p.n_tiles = (int*)at, p.tiles = (int4*)at + 1, at += s.tile_bytes;
  p.order = (int*)at, at += s.order_bytes;
  const size_t count_bytes = ((size_t)d->n_adapters + 1) * kOrderWarps * 4;
  const bool in_smem = count_bytes <= kOrderSmem;
  if (cudaError_t e = allow_smem<lora_order_kernel>(dev, kOrderSmem); e != cudaSuccess) return (int)e;
  if (int rc = launch_early(lora_order_kernel, 1, kOrderThreads, in_smem ? count_bytes : 0, st, p, in_smem ? (int*)nullptr : (int*)at)) return rc;
  return lora_run<false>(p, s, dev, st);
}

extern "C" int eux_lora_preload(void) {
  if (int rc = lora_preload<true>()) return rc;
  return lora_preload<false>();
}
