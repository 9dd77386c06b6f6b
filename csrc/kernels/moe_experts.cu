// A whole mixture-of-experts layer for a few tokens, in two launches of one kernel's two forms:
//
//   up:    h_j = silu(W_gate[e] x_t) * (W_up[e] x_t)   for every entry j = (t, slot) whose expert e is here
//   down:  out_t = sum over the entries of t of w_j * (W_down[e] h_j)
//
// What bounds it: the weights of the named experts have to come from HBM once, 2 (or 1) bytes for 2 operations per token of
// the expert; everything else is small. So the kernel is a stream of weights with the products hung on:
//
// * The weights of a form are cut into segments, 128 rows of an expert by all of K (up: 64 gate rows and the 64 up rows that
//   belong to them, with up to 64 of the expert's tokens), and these into blocks of 128 rows x 128 bytes, 16 KiB. All blocks of
//   all segments stand in one line, and each SM gets the same number of them, one after the other: no SM has more to read
//   than another, whatever the number of experts and their sizes. Where an SM's share begins or ends inside a tile of
//   results, it leaves its part in a workspace, and the last to come adds the parts up, in the order of the SMs. For the down
//   form a tile is 128 rows of the output with all experts, so the weighted sum over a token's experts is made in shared
//   memory, and only what an SM's share cuts goes through the workspace.
// * One thread fetches blocks with TMA into a ring of up to a dozen stages, one warp the tokens' values beside them, others
//   multiply, and others again make results of the sums while those go on. The ring runs on over the borders of segments; the
//   down form's starts before the up form has ended (programmatic dependent launch), since weights wait for nobody.
// * An expert's tokens lie side by side, so that one copy takes them: up to eight tokens of the call do as they are (every
//   token is a column of every product), more are put into the experts' order by a kernel in front, once for both forms.
// * The weights are the first operand, 128 rows of them, and the tokens the second: a token costs a column and not a row.
//   With few tokens, and with e4m3 weights, that is mma.sync m16n8k16, whose 8 columns are the smallest padding for one token and whose
//   operands go through registers, where e4m3 weights are widened to the tokens' bfloat16, exactly (see widen). With bfloat16 weights, where
//   an expert of the call has more than kXpFewColumns tokens, it is tcgen05 for all of them, straight from the stages into TMEM.
//
// At 16 KiB per 0.37 us and SM (the share of the measured copy bandwidth) an SM has 700 clocks for a block. Measured, in a graph, of
// the measured copy bandwidth (6550 GB/s): 128 tokens, 31 of 32 experts of 7168 x 2048: bf16 426 us (0.98), e4m3 266 us (0.78); one
// token, 8 experts of that size: 117 us (0.92) and 79 us (0.68); one token, 8 experts of 2048 x 768, bf16: 27 us (0.43: two launches'
// beginnings and ends are half of it, since the down form's CTAs, which ask for all of an SM's shared memory, find no room beside the up form's);
// 128 tokens, top-4 of 16 experts of 4096 x 2048: bf16 160 us (0.77), e4m3 193 us (0.32: widening and mma.sync are the bound, 32 tokens to an
// expert).
//
// Sums are float32 throughout. h is rounded to bfloat16, which its product takes: a relative error of up to 2^-8 in each term of a sum, on
// average as much as the result's own rounding. With few tokens the product has columns to spare, and h is two such numbers (xp_pairs). So a
// token's last bits depend on what else is in the call.
#include <cuda.h>

#include <algorithm>
#include <mutex>

#include "eux_bulk.cuh"
#include "eux_device.cuh"

namespace eux {

constexpr int kXpThreads = 512;
// Two ways to multiply. With mma.sync three groups of warps do it, each takes the blocks of every third stage, and each of its four
// warps 32 rows of them; two warps see to the results. With tcgen05 one warp does it, four see to the results, the others help at both
// ends.
constexpr int kXpGroups = 3;
constexpr int kXpWarps = kXpGroups * 4;
template <bool TC>
constexpr int kXpEndThreads = TC ? 128 : 64;
constexpr int kXpAccColumns = 64;                   // of TMEM: the tokens of a segment at most
constexpr int kXpFewTokens = 8;                     // of a call: used where they lie if their rows allow it, and h may be two numbers (xp_pairs)
constexpr int kXpFewColumns = 16;                   // bfloat16 weights: calls with up to so many tokens of any expert are multiplied with mma.sync
constexpr int kXpRows = 128;                        // rows of weights in a block
constexpr int kXpBlock = kXpRows * 128;             // bytes of a block: 128 of K per row
constexpr int kXpMaxStages = 13;
constexpr int kXpSumBars = 96;                      // bytes: for each of two sums, each group's and the results' barrier, and of tcgen05 two
constexpr int kXpLd = kXpRows + 4;                  // floats between tokens in shared memory: no bank conflicts, 16-byte rows
constexpr int kXpMaxGrid = 160;
constexpr size_t kXpDynamic = 226 * 1024;           // shared memory of a launch; the kernel declares a little more itself
constexpr int64_t kXpMaxLine = 1 << 30;             // places on it are 32 bits, and some lie a little behind its end
constexpr int kXpMinBlocks = 4;                     // of an SM's share: fewer cost more to add up than they save; none may cost more than all of these (xp_cost)

struct XpParams {
  eux_experts_desc d;
  __nv_bfloat16* x;      // [entries, x_pitch]: the tokens' values in the order of the entries; null: used where they lie
  __nv_bfloat16* h;      // [entries, h_pitch], in the same order, or two rows for each (xp_pairs); zeros behind inner
  int x_pitch, h_pitch;
  uint32_t* tables;      // what moe_experts_sort_kernel found (XpTables), with `named`, `cap` and `most` in front; null: found by every CTA
  float* part;           // [grid][2][part_rows][128]
  int part_rows;
  int token_of;          // ceil(2^20 / topk): entry * token_of >> 20 is entry / topk, for less than 2^20 / topk entries
};

// Shared memory: the ring of weights (128-byte swizzle: on 1024 bytes), behind it the tokens' values of each stage, the sums
// of a segment (tcgen05) or of two; from the end the parts whose sizes the launch knows. How many tokens a segment takes (`cap`), and with it how
// many stages there is room for, is known when the entries have been counted.
__host__ __device__ inline int xp_table_bytes(int n_experts, int entries) { return ((n_experts + 1) * 10 + entries * 8 + 31) & ~15; }
struct XpLayout {
  int acc, scales, bars, tables;  // from the beginning
  int room;                       // bytes in front of these
};
__host__ __device__ inline XpLayout xp_layout(bool down, int n_tokens, int n_experts, int entries) {
  XpLayout l;
  int at = (int)kXpDynamic;
  at -= xp_table_bytes(n_experts, entries), l.tables = at;
  at -= kXpMaxStages * 32 + kXpSumBars, l.bars = at;
  at -= kXpMaxStages * 16, l.scales = at;
  at -= down ? n_tokens * kXpLd * 4 : 0, l.acc = at;
  l.room = at;
  return l;
}
__host__ __device__ inline bool xp_tc(bool fp8, int columns) { return !fp8 && columns > kXpFewColumns; }
__host__ __device__ inline int xp_sums(bool fp8, int columns) { return xp_tc(fp8, columns) ? 1 : 2; }
__host__ __device__ inline int xp_x_bytes(bool fp8, int columns) { return columns * (fp8 ? 256 : 128); }
__host__ __device__ inline int xp_stages(bool fp8, int room, int columns) {
  const int n = (room - xp_sums(fp8, columns) * columns * kXpLd * 4) / (kXpBlock + xp_x_bytes(fp8, columns));
  return n < kXpMaxStages ? n : kXpMaxStages;
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
               "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
               : "memory");
}
// mbar_wait by a warp that has nothing else to do: it asks to be left asleep until the phase ends, for up to 20 us, instead of
// asking again and again, which takes issue slots from the warps that multiply.
__device__ __forceinline__ bool mbar_sleep(uint32_t bar, uint32_t parity, volatile int* abort, uint64_t timeout_ns) {
  uint64_t t0 = 0;
  for (uint32_t it = 0; it < 0x7fffffffu; ++it) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(20000u)
        : "memory");
    if (ok) return true;
    if ((it & 15u) == 15u) {
      if (*abort) return false;
      const uint64_t now = globaltimer_ns();
      if (t0 == 0) t0 = now;
      if (now - t0 > (timeout_ns ? timeout_ns : 2000000000ull)) break;
    }
  }
  *abort = 1;
  return false;
}
__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void lds_64(uint32_t& a, uint32_t& b, uint32_t at) {
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(a), "=r"(b) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <bool TC>
__device__ __forceinline__ void end_warps_meet() { asm volatile("bar.sync 1, %0;" ::"n"(kXpEndThreads<TC>) : "memory"); }

// ---- tcgen05 (bfloat16 weights, many tokens): the weights' 128 rows are the first operand, the tokens the second, the accumulators lie in TMEM ----
__device__ __forceinline__ uint64_t xp_operand(uint32_t at) {  // rows of 128 bytes, swizzled, eight of them 1024 bytes apart from the next
  return (uint64_t)((at >> 4) & 0x3fffu) | (uint64_t)(1024u >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ void xp_multiply(uint32_t acc, uint64_t a, uint64_t b, int columns, bool add) {
  // float32 += bfloat16 x bfloat16, 128 rows
  const uint32_t what = 1u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(columns >> 3) << 17 | (uint32_t)(kXpRows >> 4) << 24;
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(acc), "l"(a), "l"(b), "r"(what), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void xp_multiplied(uint32_t bar) {  // arrives when the products so far are through
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void xp_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void xp_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void xp_acc_16(uint32_t at, float (&v)[16]) {  // of this lane's row
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]),
        "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(at)
      : "memory");
}

// Four e4m3 values as bfloat16, bytes 0 and 2 in `even` and 1 and 3 in `odd`: sign, exponent and mantissa are moved to their places,
// which gives the value times 2^-120 (the exponents' biases are 7 and 127; subnormal ones stay subnormal), and multiplied by
// 2^120. Both steps are exact. NaN (0x7f) would become 480: weights with NaN are refused when they are given.
// The shifts to the left are written as products, which the pipe that multiplies takes: integer logic has half its rate.
__device__ __forceinline__ void widen(uint32_t w, uint32_t& even, uint32_t& odd) {
  const uint32_t w4 = w * 16u, w8 = w * 256u, r4 = w >> 4;
  const uint32_t e = (w4 & 0x07f007f0u) | (w8 & 0x80008000u), o = (r4 & 0x07f007f0u) | (w & 0x80008000u);
  const __nv_bfloat162 big = __floats2bfloat162_rn(0x1p120f, 0x1p120f);
  const __nv_bfloat162 a = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&e), big), b = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&o), big);
  even = *reinterpret_cast<const uint32_t*>(&a), odd = *reinterpret_cast<const uint32_t*>(&b);
}

// Which entries go to which expert, and the line of segments. The tables lie in shared memory and are the same in all CTAs:
//   start[a]   where the entries of the a-th named expert begin in `order` (the experts in order, entries of one in order)
//   first[a]   number of the first chunk (of up to `cap` entries) of that expert; first[named] is their number
//   expert[a]
//   cost[a]    what the chunks in front of that expert cost; only where they are made uneven (XpLine)
struct XpTables {
  int* start;        // [named + 1]
  uint16_t* first;   // [named + 1]
  uint16_t* expert;  // [named]
  uint16_t* cost;    // [named + 1]
  uint16_t* order;   // [entries]
  uint16_t* token;   // [entries]: of order
  float* weight;     // [entries]: of order
  int named;
  int most;          // entries of an expert
  __device__ XpTables(unsigned char* at, int n_experts, int entries) {
    start = reinterpret_cast<int*>(at);
    first = reinterpret_cast<uint16_t*>(start + n_experts + 1);
    expert = first + n_experts + 1;
    cost = expert + n_experts + 1;
    order = cost + n_experts + 1;
    token = order + entries;
    weight = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(token + entries) + 3) & ~(uintptr_t)3);
  }
};

// What a block of e4m3 weights costs an SM with so many eights of tokens, in quarters of what its bytes take; with more than one it is
// the products that count. Tried: 4, 4, 7, 9 and 4, 5, 8, 11 and 4, 4, 6, 8 (2 to 4 % slower over the sizes below).
__device__ __forceinline__ int xp_cost(int eights) { return eights <= 1 ? 4 : eights == 2 ? 5 : eights == 3 ? 7 : 9; }
__device__ __forceinline__ void xp_costs(XpTables& r, int lane) {  // by a warp
  int all = 0;
  for (int a0 = 0; a0 < r.named; a0 += 32) {
    const int a = a0 + lane;
    int c = 0;
    if (a < r.named) {
      const int count = r.start[a + 1] - r.start[a], chunks = r.first[a + 1] - r.first[a];
      c = chunks * xp_cost(((count + chunks - 1) / chunks + 7) >> 3);
    }
    int sum = c;
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += u;
    }
    if (a < r.named) r.cost[a] = (uint16_t)(all + sum - c);
    all += __shfl_sync(0xffffffffu, sum, 31);
  }
  if (lane == 0) r.cost[r.named] = (uint16_t)all;
}

struct XpSegment {
  int expert, tile, pos, n;
};

// With few tokens, of which no expert has more than four, h is kept as two bfloat16 numbers that add up to it, in two rows: the product has
// eight columns either way.
__device__ __forceinline__ bool xp_pairs(const XpParams& p, const XpTables& r) { return p.d.n_tokens <= kXpFewTokens && r.most <= 4; }

__device__ __forceinline__ void xp_locate(const XpTables& r, int a, int chunk, XpSegment* s) {
  const int count = r.start[a + 1] - r.start[a], chunks = r.first[a + 1] - r.first[a];
  const int each = (count + chunks - 1) / chunks;
  s->expert = r.expert[a];
  s->pos = r.start[a] + chunk * each;
  s->n = min(each, count - chunk * each);
}

// Segments one after the other; `a` is where the last one was found, which is near.
template <bool DOWN>
struct XpWalk {
  const XpTables& r;
  int tiles;  // up: row tiles of an expert
  int a = 0;
  __device__ XpWalk(const XpTables& r_, int tiles_) : r(r_), tiles(tiles_) {}
  __device__ XpSegment at(int segment) {
    XpSegment s;
    const int all = r.first[r.named];
    if (DOWN) {
      s.tile = segment / all;
      const int q = segment - s.tile * all;
      if (q < r.first[a]) a = 0;
      while (q >= r.first[a + 1]) ++a;
      xp_locate(r, a, q - r.first[a], &s);
    } else {
      while (segment >= tiles * r.first[a + 1]) ++a;
      const int in = segment - tiles * r.first[a], chunks = r.first[a + 1] - r.first[a];
      s.tile = in / chunks;
      xp_locate(r, a, in - s.tile * chunks, &s);
    }
    return s;
  }
};

// The tables. Returns the tokens that a segment takes at most: 8, 16, 32 or 64, as the expert with the most needs and `most`
// allows. `counts` is scratch, [warps][n_experts]; `out` has room for 4 and two words per warp. Entries are counted per warp and
// expert, and their places follow: by expert and then by entry, the same in every CTA.
__device__ __forceinline__ int xp_route(const eux_experts_desc& d, int token_of, int most, XpTables& r, int* counts, int* out) {
  const int E = d.n_experts, n = d.n_tokens * d.topk, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int W = kXpThreads / 32;
  const uint32_t below = (1u << lane) - 1u;
  int *const sums = out + 4, *const heads = sums + W;
  if (n <= 32) {  // one warp, by comparing
    if (warp == 0) {
      const int e0 = lane < n ? __ldcg(d.topk_idx + lane) : -1, e = (uint32_t)e0 < (uint32_t)E ? e0 : E;  // not here: behind all others
      int at = 0;
#pragma unroll 1
      for (int j = 0; j < n; ++j) {
        const int o = __shfl_sync(0xffffffffu, e, j);
        at += o < e || (o == e && j < lane);
      }
      const uint32_t same = __match_any_sync(0xffffffffu, lane < n ? e : -1);
      const bool head = lane < n && e < E && (same & below) == 0;
      const int count = head ? __popc(same) : 0;
      if (lane < n && e < E) {
        r.order[at] = (uint16_t)lane, r.token[at] = (uint16_t)((uint32_t)lane * token_of >> 20);
        r.weight[at] = __ldcg(d.topk_w + lane);
      }
      // heads in the order of their places
      int named = 0, chunks = 0, top = __reduce_max_sync(0xffffffffu, count), cap = 8;
      while (cap < top && cap < most) cap *= 2;
      const int ch = (count + cap - 1) >> (31 - __clz(cap));
      uint32_t all = __ballot_sync(0xffffffffu, head);
      int before = 0, first = 0;
#pragma unroll 1
      for (uint32_t m = all; m; m &= m - 1) {
        const int j = __ffs(m) - 1, oe = __shfl_sync(0xffffffffu, e, j), oc = __shfl_sync(0xffffffffu, ch, j);
        before += oe < e, first += oe < e ? oc : 0;
        ++named, chunks += oc;
      }
      if (head) r.expert[before] = (uint16_t)e, r.start[before] = at, r.first[before] = (uint16_t)first;
      const int here = __popc(__ballot_sync(0xffffffffu, lane < n && e < E));
      if (lane == 0) r.start[named] = here, r.first[named] = (uint16_t)chunks, out[0] = named, out[1] = cap, out[2] = top;
    }
    __syncthreads();
    r.named = out[0], r.most = out[2];
    return out[1];
  }
  const int used = min(W, (n + 31) / 32);  // warps that have entries
  const int each = ((n + used - 1) / used + 31) & ~31, lo = min(n, warp * each), hi = min(n, lo + each);
  const int e_first = lo + lane < hi ? __ldcg(d.topk_idx + lo + lane) : -1;
  for (int i = threadIdx.x; i < used * E; i += kXpThreads) counts[i] = 0;
  if (threadIdx.x == 0) out[0] = 0;
  __syncthreads();
  for (int i = lo + lane; i < hi; i += 32) {
    const int e = i == lo + lane ? e_first : __ldcg(d.topk_idx + i);
    if ((uint32_t)e < (uint32_t)E) atomicAdd(&counts[warp * E + e], 1);
  }
  __syncthreads();
  int top = 0;
  for (int e = threadIdx.x; e < E; e += kXpThreads) {
    int c = 0;
    for (int w = 0; w < used; ++w) c += counts[w * E + e];
    top = max(top, c);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0 && top) atomicMax(out, top);
  __syncthreads();
  int cap = 8;
  while (cap < out[0] && cap < most) cap *= 2;
  int named = 0, all = 0;  // of the experts so far; `all`: entries, and chunks from bit 16
  for (int e0 = 0; e0 < E; e0 += kXpThreads) {
    const int e = e0 + threadIdx.x;
    int c = 0;
    if (e < E)
      for (int w = 0; w < used; ++w) c += counts[w * E + e];
    const uint32_t has = __ballot_sync(0xffffffffu, c > 0);
    const int v = c | ((c + cap - 1) >> (31 - __clz(cap))) << 16;
    int sum = v;
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += u;
    }
    if (lane == 31) sums[warp] = sum, heads[warp] = __popc(has);
    __syncthreads();
    int before = all, a = named + __popc(has & below);
    for (int w = 0; w < W; ++w) {
      if (w < warp) before += sums[w], a += heads[w];
      all += sums[w], named += heads[w];
    }
    if (c > 0) {
      before += sum - v;
      int p = before & 0xffff;
      r.expert[a] = (uint16_t)e, r.start[a] = p, r.first[a] = (uint16_t)(before >> 16);
      for (int w = 0; w < used; ++w) {  // from counts to places
        const int m = counts[w * E + e];
        counts[w * E + e] = p;
        p += m;
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) r.start[named] = all & 0xffff, r.first[named] = (uint16_t)(all >> 16);
  for (int i0 = lo; i0 < hi; i0 += 32) {
    const int i = i0 + lane;
    const int e = i0 == lo ? e_first : i < hi ? __ldcg(d.topk_idx + i) : -1;
    const bool here = (uint32_t)e < (uint32_t)E;
    const uint32_t same = __match_any_sync(0xffffffffu, here ? e : -1);
    const int before = __popc(same & below);
    if (here) {
      const int at = counts[warp * E + e] + before;
      r.order[at] = (uint16_t)i, r.token[at] = (uint16_t)((uint32_t)i * token_of >> 20);
      r.weight[at] = __ldcg(d.topk_w + i);
    }
    __syncwarp();
    if (here && before == 0) counts[warp * E + e] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  r.named = named, r.most = out[0];
  return cap;
}

// Equal shares of a line, the first `more` of them one longer. (A line is no longer than kXpMaxLine, which the host sees to.)
struct XpShares {
  int each, more;
  __device__ XpShares(int length, int grid) : each(length / grid), more(length % grid) {}
  __device__ int begin(int i) const { return i * each + min(i, more); }
  __device__ int owner(int at) const { return at < more * (each + 1) ? at / (each + 1) : more + (at - more * (each + 1)) / each; }
};

// The line that is shared out: of blocks, or where e4m3 weights meet experts of more than 8 tokens, of what the blocks cost. An expert's
// blocks stand side by side, so that in equal numbers a few SMs would get all the dear ones, and the others wait (128 tokens, top-8 of 256
// experts of 7168 x 2048, of which 23 to 25 of this GPU's 32: one has 17 tokens, 225 us, 289 by number; two have 9 or 10, 210 and 221; 64
// tokens, top-2 of 8 experts of 4096 x 8192: 196 and 209). A block belongs to the share in which it begins; with kXpMinBlocks to a share
// each has one.
template <bool FP8, bool DOWN>
struct XpLine {
  const XpTables& r;
  int tiles, nk;
  bool by_cost;
  __device__ int each(int a) const { return (r.cost[a + 1] - r.cost[a]) / (r.first[a + 1] - r.first[a]); }
  __device__ int length() const { return tiles * nk * (FP8 && by_cost ? r.cost[r.named] : r.first[r.named]); }
  // The first block that begins at `at` or behind it. By whole warps.
  __device__ int block(int at) const {
    if (!FP8 || !by_cost) return at;
    const int all = r.first[r.named], lane = threadIdx.x & 31;
    if (at >= length()) return tiles * nk * all;
    const int of_tile = nk * r.cost[r.named], tile = DOWN ? at / of_tile : 0, unit = DOWN ? nk : nk * tiles;
    at -= tile * of_tile;
    int a = 0;
    for (;; a += 32) {
      const uint32_t behind = __ballot_sync(0xffffffffu, a + lane < r.named && unit * r.cost[min(a + lane, r.named - 1) + 1] > at);
      if (behind) {
        a += __ffs(behind) - 1;
        break;
      }
    }
    const int c = each(a);
    return nk * tile * all + unit * r.first[a] + (at - unit * r.cost[a] + c - 1) / c;
  }
  // Where the first and the last block of a tile of results begin; up: a tile is a segment, of the a-th expert.
  __device__ int tile_first(int tile, int a) const {
    if (!FP8 || !by_cost) return tile * nk * (DOWN ? r.first[r.named] : 1);
    return DOWN ? tile * nk * r.cost[r.named] : nk * (tiles * r.cost[a] + (tile - tiles * r.first[a]) * each(a));
  }
  __device__ int tile_last(int tile, int a) const {
    if (!FP8 || !by_cost) return (tile + 1) * nk * (DOWN ? r.first[r.named] : 1) - 1;
    return DOWN ? (tile + 1) * nk * r.cost[r.named] - each(r.named - 1) : tile_first(tile, a) + (nk - 1) * each(a);
  }
};

// Of the tokens' values (up) or h (down), by the rows of a copy: 8, 16, 32 and 64.
struct XpMaps {
  CUtensorMap of[4];
};

// What the warps that multiply share.
struct XpRing {
  uint32_t w, x, scales, full, empty;
  int stages, x_bytes;
  int s = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void next() {
    if (++s == stages) s = 0, ph ^= 1u;
  }
  // Of a group, which has the stages group, group + kXpGroups, ... A stage must not change hands: its barrier tells two phases
  // apart, and a group that came to it from elsewhere, ahead of a load that is late, would take the phase before the last for it.
  __device__ __forceinline__ void next_of_group(int group, int& block) {
    block += kXpGroups;
    if ((s += kXpGroups) >= stages) block += group + stages - s, s = group, ph ^= 1u;
  }
};

// The blocks of a segment up to number `end` of this SM's line times the segment's tokens: those in this group's stages, `mine`
// the next of them, and this warp's 32 rows. The groups' sums are added up in `sum` [token][row], one group after the other: each
// waits for the barrier in front of its own in `bars` (the first for the last, that the results made of an earlier segment's
// sums are done), and the warps that see to the results for the last group's. Groups by blocks and not by parts of one: a block
// takes a warp some hundred clocks from its arrival to its release, one thing after the other, and so three are under way at once.
template <bool FP8, bool DOWN, int NB>
__device__ __forceinline__ void xp_segment(XpRing& ring, int& mine, int end, int up_border, float* sum, uint32_t bars, uint32_t bars_ph, int warp, int lane,
                                           volatile int* abort, uint64_t timeout_ns) {
  const int rows = (warp & 3) * 32, group = warp >> 2, g = lane >> 2, c = lane & 3;
  // Which of eight tokens a column of the product is. With e4m3 weights a half of a warp reads 32 bytes of four tokens at a time: of
  // every second one, whose places differ under the swizzle.
  auto column = [](int j) { return FP8 ? (j & 3) * 2 + (j >> 2) : j; };
  float acc[2][NB][4] = {};
  while (mine < end) {
    // A wait that ran out raises `abort`; the warps then finish on whatever lies there, so that they meet at every barrier, and the
    // status word says that the result is none.
    mbar_sleep(ring.full + 32 * ring.s, ring.ph, abort, timeout_ns);
    __syncwarp();
    const uint32_t w = ring.w + ring.s * kXpBlock, x = ring.x + ring.s * ring.x_bytes;
    if constexpr (!FP8) {
#pragma unroll
      for (int kp = 0; kp < 2; ++kp) {  // 32 of K
        uint32_t b1[4];
        if (NB == 1) ldsm_x4(b1, x + (lane & 7) * 128 + (((kp * 4 + (lane >> 3)) ^ (lane & 7)) << 4));
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const int step = kp * 2 + ks;
          uint32_t a[2][4], b[NB > 1 ? NB / 2 : 1][4];
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const int row = rows + m * 16 + (lane & 15);
            ldsm_x4(a[m], w + row * 128 + (((step * 2 + (lane >> 4)) ^ (row & 7)) << 4));
          }
          if (NB == 1) {
            b[0][0] = b1[2 * ks], b[0][1] = b1[2 * ks + 1];
          } else {
#pragma unroll
            for (int j = 0; j < NB / 2; ++j) {
              const int row = j * 16 + (lane & 7) + ((lane >> 4) << 3);
              ldsm_x4(b[j], x + row * 128 + (((step * 2 + ((lane >> 3) & 1)) ^ (row & 7)) << 4));
            }
          }
#pragma unroll
          for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int m = 0; m < 2; ++m)
              mma_bf16(acc[m][j], a[m][0], a[m][1], a[m][2], a[m][3], b[j / 2][(j & 1) * 2], b[j / 2][(j & 1) * 2 + 1]);
        }
      }
    } else {
      // A 16-byte piece of a row is 16 values of K. ldmatrix gives lane (g, c) the four at 4c: the first and the third are the product's k = 2c
      // and 2c + 1, the others 2c + 8 and 2c + 9, and the tokens' values are paired likewise (the order of K is the product's own affair).
      float part[2][NB][4] = {};
#pragma unroll
      for (int kp = 0; kp < 4; ++kp) {
        const int step = kp * 2;
        uint32_t a[2][4];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const int row = rows + m * 16 + (lane & 15);
          ldsm_x4(a[m], w + row * 128 + (((step + (lane >> 4)) ^ (row & 7)) << 4));
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          uint32_t wa[2][4];
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const uint32_t r0 = a[m][2 * ks], r1 = a[m][2 * ks + 1];
            widen(r0, wa[m][0], wa[m][2]), widen(r1, wa[m][1], wa[m][3]);
          }
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            uint32_t x0, x1;
            const int st = step + ks;
            lds_64(x0, x1, x + (st >> 2) * ((NB == 3 ? 4 : NB) * 1024) + (j * 8 + column(g)) * 128 + ((((st & 3) * 2 + (c >> 1)) ^ column(g)) << 4) + (c & 1) * 8);
            const uint32_t b0 = __byte_perm(x0, x1, 0x5410), b1 = __byte_perm(x0, x1, 0x7632);
#pragma unroll
            for (int m = 0; m < 2; ++m) mma_bf16(part[m][j], wa[m][0], wa[m][1], wa[m][2], wa[m][3], b0, b1);
          }
        }
      }
      // a block of K is a block of scales; of the rows, the up half may lie in two
      float sc[3];
      asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(sc[0]), "=f"(sc[1]) : "r"(ring.scales + 16 * ring.s) : "memory");
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(sc[2]) : "r"(ring.scales + 16 * ring.s + 8) : "memory");
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        float lo = sc[0], hi = sc[0];
        if (!DOWN && rows >= 64) {
          const int row = rows - 64 + m * 16 + g;
          lo = row < up_border ? sc[1] : sc[2], hi = row + 8 < up_border ? sc[1] : sc[2];
        }
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          acc[m][j][0] = fmaf(part[m][j][0], lo, acc[m][j][0]), acc[m][j][1] = fmaf(part[m][j][1], lo, acc[m][j][1]);
          acc[m][j][2] = fmaf(part[m][j][2], hi, acc[m][j][2]), acc[m][j][3] = fmaf(part[m][j][3], hi, acc[m][j][3]);
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(ring.empty + 32 * ring.s);
    ring.next_of_group(group, mine);
  }
  mbar_sleep(bars + (group ? 8 * (group - 1) : 8 * kXpGroups), group ? bars_ph : bars_ph ^ 1u, abort, timeout_ns);
  __syncwarp();
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float* at = sum + (j * 8 + column(2 * c + (q & 1))) * kXpLd + rows + m * 16 + g + (q >> 1) * 8;
        *at = group ? *at + acc[m][j][q] : acc[m][j][q];
      }
  __syncwarp();
  if (lane == 0) mbar_arrive(bars + 8 * group);
}

__device__ __forceinline__ float4 ldcg_f4(const float* p) { return __ldcg(reinterpret_cast<const float4*>(p)); }
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}

__device__ __forceinline__ void cta_meets() { __syncthreads(); }

// The end of a tile of results, or of this SM's part of it: the sums `from` [token][row], which THREADS threads have, that meet with
// `meet`. The parts of a tile that begin in the middle of it come early in their SMs' shares, and the first part comes last in its
// own: where the others are there already, which it sees from their count, it need not leave its part in the workspace and count itself.
template <bool DOWN, int THREADS, typename Meet>
__device__ __forceinline__ void xp_tile_end(const XpParams& p, const XpTables& r, const XpSegment& s, int first, int last, int me, const float* from,
                                            bool in_place, int tid, int* s_last, Meet meet) {
  const eux_experts_desc& d = p.d;
  auto sum_row = [&](int j) { return (in_place ? r.token[s.pos + j] : j) * kXpLd; };
  const int rows = DOWN ? d.n_tokens : s.n;
  uint32_t* const counter = d.counters + (DOWN ? kXpMaxGrid : 0) + first;
  constexpr int Q = DOWN ? kXpRows / 4 : 16;  // four rows of results per thread and step
  bool own_here = first == last;
  if (first != last && me == first) {
    if (tid == 0) {
      *s_last = ld_acquire_gpu(counter) == (unsigned)(last - first);
      if (*s_last) *counter = 0;
    }
    meet();
    own_here = *s_last != 0;
    meet();
  }
  if (!own_here) {
    float* const part = p.part + ((int64_t)me * 2 + (me == first)) * p.part_rows * kXpRows;
    for (int i = tid; i < rows * (kXpRows / 4); i += THREADS)
      __stcg(reinterpret_cast<float4*>(part) + i, *reinterpret_cast<const float4*>(from + sum_row(i / (kXpRows / 4)) + (i % (kXpRows / 4)) * 4));
    __threadfence();
    meet();
    // counts up to the number of parts and starts again: ready for the next launch
    if (tid == 0) *s_last = atomicInc(counter, (unsigned)(last - first)) == (unsigned)(last - first);
    meet();
    const bool all_there = *s_last != 0;
    meet();
    if (!all_there) return;
    __threadfence();
  }
  for (int i = tid; i < rows * Q; i += THREADS) {
    const int j = i / Q, q = (i % Q) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f), u = v;
    auto add = [](float4& to, const float4& a) { to.x += a.x, to.y += a.y, to.z += a.z, to.w += a.w; };
    int k = first;
    if (own_here) {
      add(v, *reinterpret_cast<const float4*>(from + sum_row(j) + q));
      if (!DOWN) add(u, *reinterpret_cast<const float4*>(from + sum_row(j) + 64 + q));
      ++k;
    }
    constexpr int AT_ONCE = DOWN ? 6 : 3;
    for (; k <= last; k += AT_ONCE) {  // in the order of the SMs, several loads under way
      float4 a[AT_ONCE], o[AT_ONCE];
#pragma unroll
      for (int n = 0; n < AT_ONCE; ++n) {
        const int c = min(k + n, last);
        const float* const part = p.part + (((int64_t)c * 2 + (c == first)) * p.part_rows + j) * kXpRows + q;
        a[n] = ldcg_f4(part);
        if (!DOWN) o[n] = ldcg_f4(part + 64);
      }
#pragma unroll
      for (int n = 0; n < AT_ONCE; ++n)
        if (k + n <= last) {
          add(v, a[n]);
          if (!DOWN) add(u, o[n]);
        }
    }
    if (DOWN) {
      const int at = s.tile * kXpRows + q;
      if (at < d.hidden) *reinterpret_cast<uint2*>((__nv_bfloat16*)d.out + j * d.out_stride + at) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
    } else {
      const int at = s.tile * 64 + q;
      auto gated = [](float g, float w) { return g / (1.f + expf(-g)) * w; };
      // what bfloat16 loses; of an infinity nothing
      auto rest = [](float f) {
        const float b = __bfloat162float(__float2bfloat16_rn(f));
        return isinf(b) ? 0.f : f - b;
      };
      const bool pairs = xp_pairs(p, r), last = s.tile * 64 + 64 >= d.inner && s.tile * 64 + 64 < p.h_pitch;
      float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
      if (at < d.inner) f = make_float4(gated(v.x, u.x), gated(v.y, u.y), gated(v.z, u.z), gated(v.w, u.w));
      __nv_bfloat16* h = p.h + (int64_t)(s.pos + j) * (pairs ? 2 : 1) * p.h_pitch + at;
      *reinterpret_cast<uint2*>(h) = make_uint2(pack_bf16(f.x, f.y), pack_bf16(f.z, f.w));
      if (last) *reinterpret_cast<uint2*>(h + 64) = make_uint2(0, 0);
      if (pairs) {
        h += p.h_pitch;
        *reinterpret_cast<uint2*>(h) = make_uint2(pack_bf16(rest(f.x), rest(f.y)), pack_bf16(rest(f.z), rest(f.w)));
        if (last) *reinterpret_cast<uint2*>(h + 64) = make_uint2(0, 0);
      }
    }
  }
}

// What the warps that see to the results do.
template <bool FP8, bool DOWN>
struct XpResults {
  const XpParams& p;
  const XpTables& r;
  const XpLine<FP8, DOWN>& line;
  const XpShares& shares;
  int b0, b1, seg0, nk, chunks, me;
  bool in_place;
  int columns;
  float *sums, *acc;
  int* s_last;
  volatile int* abort;

  template <bool TC>
  __device__ __forceinline__ void make(XpWalk<DOWN>& walk, uint32_t all_bars, uint32_t tmem, int tid) const {
    const eux_experts_desc& d = p.d;
    constexpr int THREADS = kXpEndThreads<TC>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile_segs = DOWN ? chunks : 1;  // segments of a tile of results
    const int tile_blocks = tile_segs * nk;
    if (DOWN && chunks == 0) {  // no expert is named: the result is zero
      for (int i = blockIdx.x * THREADS + tid; i < d.n_tokens * (d.hidden / 8); i += gridDim.x * THREADS)
        st_u4((__nv_bfloat16*)d.out + (int64_t)(i / (d.hidden / 8)) * d.out_stride + (i % (d.hidden / 8)) * 8, make_uint4(0, 0, 0, 0));
    }
    int buf = 0, tile = b0 < b1 ? seg0 / tile_segs : 0;
    uint32_t buf_ph = 0;
    for (int b = b0, seg = seg0; b < b1; ++seg) {
      const XpSegment s = walk.at(seg);
      const int tile0 = tile * tile_blocks, tile1 = tile0 + tile_blocks;
      float* const sum = sums + (TC ? 0 : buf * columns * kXpLd);
      const uint32_t bars = all_bars + buf * 8 * (TC ? 2 : kXpGroups + 1), free_bar = bars + 8 * (TC ? 1 : kXpGroups);
      if (DOWN && b == tile0 && b != b0) {
        for (int i = tid; i < d.n_tokens * (kXpLd / 4); i += THREADS) reinterpret_cast<float4*>(acc)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        end_warps_meet<TC>();
      }
      mbar_sleep(bars + (TC ? 0 : 8 * (kXpGroups - 1)), buf_ph, abort, d.wait_timeout_ns);
      __syncwarp();
      b = min((seg + 1) * nk, b1);
      // Down: entries of the same token, also twice of the same expert, are added by one thread, which has one or two rows, in order.
      if (TC) {
        // A thread has a row, which is a lane of TMEM.
        xp_fence_after();
        for (int j0 = 0; j0 < s.n; j0 += 16) {
          float v[16];
          xp_acc_16(tmem + buf * kXpAccColumns + j0 + ((uint32_t)(warp * 32) << 16), v);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (j0 + i < s.n) {
              if (DOWN) {
                float* const at = acc + r.token[s.pos + j0 + i] * kXpLd + tid;
                *at = fmaf(r.weight[s.pos + j0 + i], v[i], *at);
              } else {
                sum[(j0 + i) * kXpLd + tid] = v[i];
              }
            }
        }
        xp_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(free_bar);
      } else if (DOWN) {
        const bool pairs = xp_pairs(p, r);
        for (int j0 = 0; j0 < s.n; j0 += 4) {
          float2 v[4];
          float w[4];
          int t[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = min(j0 + i, s.n - 1);
            v[i] = reinterpret_cast<const float2*>(sum + (pairs ? 2 * j : j) * kXpLd)[tid], w[i] = r.weight[s.pos + j], t[i] = r.token[s.pos + j];
            if (pairs) {
              const float2 u = reinterpret_cast<const float2*>(sum + (2 * j + 1) * kXpLd)[tid];
              // an infinite weight is met by the first of the two: zero, or the other sign, in the second would make it NaN
              v[i].x += isfinite(u.x) ? u.x : 0.f, v[i].y += isfinite(u.y) ? u.y : 0.f;
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (j0 + i < s.n) {
              float2* const at = reinterpret_cast<float2*>(acc + t[i] * kXpLd) + tid;
              *at = make_float2(fmaf(w[i], v[i].x, at->x), fmaf(w[i], v[i].y, at->y));
            }
        }
      }
      if (!DOWN || b == b1 || b == tile1) {
        // the end of a tile, or of this SM's part of it
        end_warps_meet<TC>();  // what they have put together is complete
        if (b == b1) break;    // the end of the share is everybody's
        xp_tile_end<DOWN, THREADS>(p, r, s, shares.owner(line.tile_first(tile, walk.a)), shares.owner(line.tile_last(tile, walk.a)), me, DOWN ? acc : sum, in_place, tid, s_last,
                                     end_warps_meet<TC>);
        end_warps_meet<TC>();  // and is written over next
        if (b == tile1) ++tile;
      }
      if (!TC) {
        __syncwarp();
        if (lane == 0) mbar_arrive(free_bar);
      }
      if ((buf ^= 1) == 0) buf_ph ^= 1u;
    }
  }
};

template <bool FP8, bool DOWN>
__global__ void __launch_bounds__(kXpThreads, 1) moe_experts_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ XpMaps x_maps, const __grid_constant__ XpParams p) {
  extern __shared__ __align__(1024) unsigned char xp_smem[];
  __shared__ int s_abort, s_last, s_route[4 + 2 * kXpThreads / 32];
  __shared__ uint32_t s_acc;
  const eux_experts_desc& d = p.d;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int entries = d.n_tokens * d.topk;
  const XpLayout l = xp_layout(DOWN, d.n_tokens, d.n_experts, entries);
  const uint32_t smem = smem_u32(xp_smem);
  XpRing ring;
  ring.w = smem, ring.scales = smem + l.scales, ring.full = smem + l.bars, ring.empty = smem + l.bars + 8;  // tcgen05: + 16
  const uint32_t sum_bars = smem + l.bars + kXpMaxStages * 32, tc_bars = sum_bars + 2 * (kXpGroups + 1) * 8;
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < kXpMaxStages; ++i) {
      mbar_init(ring.full + 32 * i, 2);       // weights and tokens
      mbar_init(ring.empty + 32 * i, 4);      // the warps of a group
      mbar_init(ring.empty + 32 * i + 8, 1);
    }
    for (int i = 0; i < 2 * (kXpGroups + 1); ++i) mbar_init(sum_bars + 8 * i, i % (kXpGroups + 1) < kXpGroups ? 4 : kXpEndThreads<false> / 32);
    for (int i = 0; i < 4; ++i) mbar_init(tc_bars + 8 * i, i % 2 ? kXpEndThreads<true> / 32 : 1);  // full and free, of two accumulators
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&x_maps.of[0]) : "memory");
  }
  constexpr int kProducts = 4, kWeights = kXpThreads / 32 - 2, kTokens = kWeights + 1;  // warps
  // The up form waits here for whatever wrote the tokens and their experts. The down form was let in by the up form, behind its
  // wait: what both read is there, in the L2, and only what the up form writes is waited for (below).
  if (!DOWN) wait_for_launch_before();
  XpTables r(xp_smem + l.tables, d.n_experts, entries);
  int cap;
  if (p.tables) {
    const uint4* const from = reinterpret_cast<const uint4*>(p.tables + 4);
    for (int i = threadIdx.x; i < xp_table_bytes(d.n_experts, entries) / 16; i += kXpThreads) reinterpret_cast<uint4*>(xp_smem + l.tables)[i] = __ldcg(from + i);
    const uint4 head = ld_cg_u4(p.tables);
    r.named = (int)head.x, cap = (int)head.y, r.most = (int)head.z;
    __syncthreads();
  } else {
    cap = xp_route(d, p.token_of, FP8 ? 32 : kXpAccColumns, r, reinterpret_cast<int*>(xp_smem), s_route);
  }
  // Up to eight tokens lie where they are: each is a column of every product, whichever of them an expert has.
  const bool in_place = !DOWN && !p.x;
  const int columns = in_place ? 8 : cap;
  // Few tokens take a tensor core little time either way, and tcgen05 draws more power for its padding to 16: the memory clock's share of
  // it is what counts then (16 tokens, 32 experts of 7168 x 2048: 421 us with mma.sync, 439 with tcgen05; one token 115.5 and 120). With
  // more, operands through registers are what an SM waits for (128 tokens, top-4 of 16 experts of 4096 x 2048: 187 and 160).
  const bool tc = xp_tc(FP8, columns);
  if (!FP8 && tc && warp == kProducts) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_acc)), "r"(2u * kXpAccColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tc) ring.empty += 8;
  ring.x_bytes = xp_x_bytes(FP8, columns);
  ring.stages = xp_stages(FP8, l.room, columns);
  ring.x = smem + ring.stages * kXpBlock;
  const int K = DOWN ? d.inner : d.hidden, per_block = FP8 ? 128 : 64;
  const int nk = (K + per_block - 1) / per_block;
  const int tiles = DOWN ? (d.hidden + kXpRows - 1) / kXpRows : (d.inner + 63) / 64;
  const int chunks = r.first[r.named];
  const int blocks = tiles * chunks * nk;
  const int grid = min((int)gridDim.x, max(1, blocks / kXpMinBlocks));
  const int me = blockIdx.x;
  const XpLine<FP8, DOWN> line{r, tiles, nk, FP8 && p.tables && cap > 8};
  const XpShares shares(line.length(), grid);
  const int b0 = me < grid ? line.block(shares.begin(me)) : blocks, b1 = me < grid ? line.block(shares.begin(me + 1)) : blocks;
  const int seg0 = b0 / nk, kb0 = b0 - seg0 * nk;  // the segment that the share begins in, and where
  float* const sums = reinterpret_cast<float*>(xp_smem + ring.stages * (kXpBlock + ring.x_bytes));
  const int n_sums = xp_sums(FP8, columns);
  float* const acc = reinterpret_cast<float*>(xp_smem + l.acc);
  if (DOWN)
    for (int i = threadIdx.x; i < d.n_tokens * (kXpLd / 4); i += kXpThreads) reinterpret_cast<float4*>(acc)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  // the counts lay where weights are about to land
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  xp_fence_before();
  __syncthreads();
  xp_fence_after();
  volatile int* abort = &s_abort;
  XpWalk<DOWN> walk(r, tiles);

  if (warp == kWeights) {
    // ---- weights ----
    if (lane == 0) {
      for (int b = b0, seg = seg0, kb = kb0; b < b1 && !*abort; ++seg, kb = 0) {
        const int end = min(nk, kb + (b1 - b));
        const XpSegment s = walk.at(seg);
        for (int k = kb; k < end; ++k) {
          if (!mbar_sleep(ring.empty + 32 * ring.s, ring.ph ^ 1u, abort, d.wait_timeout_ns)) break;
          const uint32_t bar = ring.full + 32 * ring.s, dst = ring.w + ring.s * kXpBlock;
          mbar_expect_tx(bar, kXpBlock);
          if (DOWN) tma_load_3d(dst, &map, bar, k * per_block, s.tile * kXpRows, s.expert);
          else tma_load_3d(dst, &map, bar, k * per_block, s.tile * 64, s.expert * 2);  // 64 gate rows, and 64 up rows behind them
          ring.next();
        }
        b += end - kb;
      }
      if (*abort) {  // loads that were issued still write shared memory: give them time to land
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
      }
      allow_next_launch();
    }
  } else if (warp == kTokens) {
    // ---- the tokens' values (down: their h) and the scales ----
    if (DOWN) wait_for_launch_before();
    asm volatile("fence.proxy.async;" ::: "memory");  // written by ordinary stores, read by copies
    const int sr = ((DOWN ? d.hidden : 2 * d.inner) + 127) / 128, sk = (K + 127) / 128;
    bool gone = false;
    for (int b = b0, seg = seg0, kb = kb0; b < b1 && !gone; ++seg, kb = 0) {
      const int end = min(nk, kb + (b1 - b));
      const XpSegment s = walk.at(seg);
      const int nb = in_place ? 1 : (s.n + 7) >> 3, size = nb <= 1 ? 0 : nb <= 2 ? 1 : nb <= 4 ? 2 : 3, row = in_place ? 0 : DOWN && xp_pairs(p, r) ? 2 * s.pos : s.pos;
      // the scales of 32 blocks at a time, one per lane. Down: of the rows. Up: of the gate rows, of the first up rows, of the up rows
      // that lie in the next block.
      const float* const scale = FP8 ? (DOWN ? d.down_scale : d.gate_up_scale) + (int64_t)s.expert * sr * sk : nullptr;
      float sc[DOWN ? 1 : 3];
      for (int k = kb; k < end; ++k) {
        if (FP8 && (k - kb) % 32 == 0) {
#pragma unroll
          for (int q = 0; q < (DOWN ? 1 : 3); ++q) {
            const int block = DOWN ? s.tile : q == 0 ? s.tile * 64 / 128 : min((d.inner + s.tile * 64) / 128 + q - 1, sr - 1);
            sc[q] = k + lane < end ? __ldg(scale + (int64_t)block * sk + k + lane) : 0.f;
          }
        }
        gone = __any_sync(0xffffffffu, !mbar_sleep(ring.empty + 32 * ring.s, ring.ph ^ 1u, abort, d.wait_timeout_ns));
        if (gone) break;
        const uint32_t bar = ring.full + 32 * ring.s, dst = ring.x + ring.s * ring.x_bytes;
        if (FP8) {
          float v[3];
#pragma unroll
          for (int q = 0; q < 3; ++q) v[q] = __shfl_sync(0xffffffffu, sc[DOWN ? 0 : q], (k - kb) % 32);
          if (lane == 0) asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %3};" ::"r"(ring.scales + 16 * ring.s), "f"(v[0]), "f"(v[1]), "f"(v[2]) : "memory");
        }
        if (lane == 0) {
          mbar_expect_tx(bar, (8u << size) * (FP8 ? 256 : 128));
          tma_load_3d(dst, &x_maps.of[size], bar, 0, row, FP8 ? 2 * k : k);  // rows behind the expert's are multiplied and not used
        }
        ring.next();
      }
      b += end - kb;
    }
    if (gone && lane == 0) {  // as above
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
  } else if (!tc && warp < kXpWarps) {
    // ---- products with mma.sync ----
    int mine = b0 + (warp >> 2), sum_at = 0;
    uint32_t sum_ph = 0;
    ring.s = warp >> 2;
    for (int b = b0, seg = seg0; b < b1; ++seg) {
      const int end = min((seg + 1) * nk, b1);
      const XpSegment s = walk.at(seg);
      const int up_border = 128 - (d.inner + s.tile * 64) % 128;
      const int nb = in_place ? 1 : (s.n + 7) >> 3;
      float* const sum = sums + sum_at * columns * kXpLd;
      const uint32_t bars = sum_bars + sum_at * 8 * (kXpGroups + 1);
      if (nb <= 1) xp_segment<FP8, DOWN, 1>(ring, mine, end, up_border, sum, bars, sum_ph, warp, lane, abort, d.wait_timeout_ns);
      else if (!FP8 || nb <= 2) xp_segment<FP8, DOWN, 2>(ring, mine, end, up_border, sum, bars, sum_ph, warp, lane, abort, d.wait_timeout_ns);
      else if constexpr (FP8) {  // 32 tokens at most; three eights are worth a form of their own (64 tokens, top-2 of 8 experts of 4096 x 8192: 209 us, 231 without)
        if (nb == 3) xp_segment<FP8, DOWN, 3>(ring, mine, end, up_border, sum, bars, sum_ph, warp, lane, abort, d.wait_timeout_ns);
        else xp_segment<FP8, DOWN, 4>(ring, mine, end, up_border, sum, bars, sum_ph, warp, lane, abort, d.wait_timeout_ns);
      }
      if (++sum_at == n_sums) sum_at = 0, sum_ph ^= 1u;
      b = end;
    }
  } else if (!FP8 && tc && warp == kProducts) {
    // ---- products with tcgen05 ----
    if (lane == 0) {
      int buf = 0;
      uint32_t buf_ph = 0;
      bool gone = false;
      for (int b = b0, seg = seg0; b < b1 && !gone; ++seg) {
        const int end = min((seg + 1) * nk, b1);
        const XpSegment s = walk.at(seg);
        const int n = s.n <= 16 ? 16 : s.n <= 32 ? 32 : 64;  // 16 are the fewest
        const uint32_t bars = tc_bars + buf * 16, acc = s_acc + buf * kXpAccColumns;
        gone = !mbar_sleep(bars + 8, buf_ph ^ 1u, abort, d.wait_timeout_ns);
        xp_fence_after();
        for (int k = b; k < end && !gone; ++k) {
          if ((gone = !mbar_sleep(ring.full + 32 * ring.s, ring.ph, abort, d.wait_timeout_ns))) break;
          xp_fence_after();
          const uint64_t w = xp_operand(ring.w + ring.s * kXpBlock), x = xp_operand(ring.x + ring.s * ring.x_bytes);
#pragma unroll
          for (int i = 0; i < 4; ++i) xp_multiply(acc, w + 2 * i, x + 2 * i, n, k > b || i > 0);  // 16 of K, 32 bytes, each
          xp_multiplied(ring.empty + 32 * ring.s);
          ring.next();
        }
        if (!gone) xp_multiplied(bars);
        if ((buf ^= 1) == 0) buf_ph ^= 1u;
        b = end;
      }
      if (gone) {  // products that were begun still write TMEM and read shared memory
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
      }
    }
  } else if (!tc || warp < kXpEndThreads<true> / 32) {
    if (DOWN) wait_for_launch_before();
    const XpResults<FP8, DOWN> results{p, r, line, shares, b0, b1, seg0, nk, chunks, me, in_place, columns, sums, acc, &s_last, abort};
    if (!tc) results.template make<false>(walk, sum_bars, 0, threadIdx.x - kXpWarps * 32);
    else if constexpr (!FP8) results.template make<true>(walk, tc_bars, s_acc, threadIdx.x);
  }
  xp_fence_before();
  __syncthreads();
  if (b0 < b1) {
    const int seg = (b1 - 1) / nk, tile = DOWN ? seg / chunks : seg;
    const XpSegment s = walk.at(seg);
    xp_tile_end<DOWN, kXpThreads>(p, r, s, shares.owner(line.tile_first(tile, walk.a)), shares.owner(line.tile_last(tile, walk.a)), me,
                                  DOWN ? acc : sums + (seg - seg0) % n_sums * columns * kXpLd, in_place, threadIdx.x, &s_last, cta_meets);
  }
  if (!FP8 && tc && warp == kProducts) {
    xp_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s_acc), "r"(2u * kXpAccColumns) : "memory");
  }
  if (threadIdx.x == 0 && s_abort) set_status(d.status, EUX_ST_TIMEOUT, DOWN ? 2 : 1);
}

// With more than eight tokens: finds the tables, once for both launches, and puts the tokens' values into the order of the entries, so
// that an expert's lie side by side and one copy takes them (gathered four rows at a time they cost an SM up to a sixth of its time:
// 128 tokens, top-4 of 16 experts of 4096 x 2048, bf16: 205 us, 179 from one place; 16 tokens, 32 experts of 7168 x 2048, e4m3: 313 and 268).
__global__ void __launch_bounds__(kXpThreads) moe_experts_sort_kernel(const __grid_constant__ XpParams p, int most) {
  extern __shared__ __align__(1024) unsigned char xp_smem[];
  __shared__ int s_route[4 + 2 * kXpThreads / 32];
  const eux_experts_desc& d = p.d;
  const int entries = d.n_tokens * d.topk, bytes = xp_table_bytes(d.n_experts, entries);
  wait_for_launch_before();
  XpTables r(xp_smem, d.n_experts, entries);
  const int cap = xp_route(d, p.token_of, most, r, reinterpret_cast<int*>(xp_smem + bytes), s_route);
  if (blockIdx.x == 0) {
    if (d.fp8 && cap > 8) {
      if (threadIdx.x < 32) xp_costs(r, threadIdx.x);
      __syncthreads();
    }
    for (int i = threadIdx.x; i < bytes / 16; i += kXpThreads) reinterpret_cast<uint4*>(p.tables + 4)[i] = reinterpret_cast<const uint4*>(xp_smem)[i];
    if (threadIdx.x == 0) p.tables[0] = (uint32_t)r.named, p.tables[1] = (uint32_t)cap, p.tables[2] = (uint32_t)r.most;
  }
  const int here = r.start[r.named], pieces = p.x_pitch / 8;
  for (int i = blockIdx.x * kXpThreads + threadIdx.x; i < here * pieces; i += gridDim.x * kXpThreads) {
    const int pos = i / pieces, at = (i - pos * pieces) * 8;
    const uint4 v = at < d.hidden ? ld_cg_u4((const __nv_bfloat16*)d.x + r.token[pos] * d.x_stride + at) : make_uint4(0, 0, 0, 0);
    st_u4(p.x + (int64_t)pos * p.x_pitch + at, v);
  }
  allow_next_launch();
}

// Whether one of n 16-byte pieces holds an e4m3 NaN (0x7f or 0xff).
__global__ void __launch_bounds__(512) moe_experts_nan_kernel(const uint4* q, size_t n, uint32_t* found) {
  uint32_t any = 0;
  for (size_t i = (size_t)blockIdx.x * 512 + threadIdx.x; i < n; i += (size_t)gridDim.x * 512) {
    const uint4 v = ld_stream_u4(q + i);
    any |= ((v.x & 0x7f7f7f7fu) + 0x01010101u) | ((v.y & 0x7f7f7f7fu) + 0x01010101u) | ((v.z & 0x7f7f7f7fu) + 0x01010101u) | ((v.w & 0x7f7f7f7fu) + 0x01010101u);
  }
  if (any & 0x80808080u) *found = 1;
}

// ---- host ----

typedef CUresult (*XpEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                               const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static XpEncodeFn xp_encode() {
  static const XpEncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess
               ? (XpEncodeFn)p
               : nullptr;
  }();
  return fn;
}
// Rows of bfloat16 `pitch` elements apart, cols a multiple of 64: copies of 8 to 64 rows by `runs` times 64 columns, one run behind the other
static int xp_map_rows(XpMaps* m, const void* base, uint64_t rows, uint64_t cols, uint64_t pitch, int runs, int most) {
  const XpEncodeFn fn = xp_encode();
  if (!fn) return EUX_ERR_UNSUPPORTED;
  for (int i = 0; i < 4 && (i == 0 || (4 << i) < most); ++i) {  // up to `most` rows
    const cuuint64_t dims[3] = {64, rows, cols / 64}, strides[2] = {pitch * 2, 128};
    const cuuint32_t box[3] = {64, 8u << i, (cuuint32_t)runs}, step[3] = {1, 1, 1};
    const CUresult rc = fn(m->of + i, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return EUX_ERR_BAD_ARG;
  }
  return 0;
}
// [slices][rows][cols], boxes of box_rows x 128 bytes, 128-byte swizzle; what lies outside is read as zero
static int xp_map(CUtensorMap* m, const void* base, bool fp8, uint64_t slices, uint64_t rows, uint64_t cols, uint32_t box_rows, uint32_t box_slices) {
  const XpEncodeFn fn = xp_encode();
  if (!fn) return EUX_ERR_UNSUPPORTED;
  const uint64_t elem = fp8 ? 1 : 2;
  const cuuint64_t dims[3] = {cols, rows, slices}, strides[2] = {cols * elem, rows * cols * elem};
  const cuuint32_t box[3] = {(cuuint32_t)(128 / elem), box_rows, box_slices}, step[3] = {1, 1, 1};
  const CUresult rc = fn(m, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, step,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? 0 : EUX_ERR_BAD_ARG;
}

// The longest line that a pass can have, of blocks or of what they cost: each named expert has a chunk of up to `most` entries that is not
// full, the others are.
static int64_t xp_longest_line(const eux_experts_desc* d) {
  const int64_t entries = (int64_t)d->n_tokens * d->topk, chunks = std::min<int64_t>(d->n_experts, entries) + entries / (d->fp8 ? 32 : kXpAccColumns);
  auto runs = [](int64_t n, int64_t of) { return (n + of - 1) / of; };
  const int64_t per_block = d->fp8 ? 128 : 64;
  const int64_t blocks = std::max(runs(d->inner, 64) * runs(d->hidden, per_block), runs(d->hidden, kXpRows) * runs(d->inner, per_block));
  return blocks * chunks * (d->fp8 ? 9 : 1);  // xp_cost
}

static int experts_check(const eux_experts_desc* d) {
  if (!d || d->n_tokens < 0 || d->n_tokens > EUX_EXPERTS_MAX_TOKENS || d->topk < 1 || d->topk > 32) return EUX_ERR_BAD_ARG;
  if (d->n_experts < 1 || d->n_experts > EUX_EXPERTS_MAX_EXPERTS || d->hidden < 1 || d->inner < 1) return EUX_ERR_BAD_ARG;
  if (d->hidden > (1 << 20) || d->inner > (1 << 20)) return EUX_ERR_BAD_ARG;
  const int unit = d->fp8 ? 16 : 8;  // rows of weights begin on 16 bytes
  if (d->hidden % unit || d->inner % unit || d->x_stride % 8 || d->out_stride % 8 || d->x_stride < 0 || d->out_stride < 0) return EUX_ERR_BAD_ARG;
  if (xp_longest_line(d) > kXpMaxLine) return EUX_ERR_TOO_LARGE;
  return 0;
}
static int xp_part_rows(const eux_experts_desc* d) { return std::max(64, d->n_tokens); }
// Where what lies in a workspace: h, the tokens' values in order, the tables, parts of tiles.
struct XpSpace {
  int x_pitch, h_pitch;
  bool sorted;
  size_t h_rows, h, x, tables, parts;
};
static XpSpace xp_space(const eux_experts_desc* d) {
  XpSpace s;
  const size_t entries = (size_t)d->n_tokens * d->topk;
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  s.x_pitch = (d->hidden + 127) & ~127, s.h_pitch = (d->inner + 127) & ~127;
  s.sorted = d->n_tokens > kXpFewTokens || d->hidden != s.x_pitch;  // copies take whole runs of columns
  s.h_rows = (d->n_tokens > kXpFewTokens ? 1 : 2) * entries;  // xp_pairs
  s.h = up(s.h_rows * s.h_pitch * 2);
  s.x = s.sorted ? up(entries * s.x_pitch * 2) : 0;
  s.tables = s.sorted ? up(16 + xp_table_bytes(d->n_experts, (int)entries)) : 0;
  s.parts = (size_t)kXpMaxGrid * 2 * xp_part_rows(d) * kXpRows * 4;
  return s;
}

static int xp_sms(int* dev) {
  int sms = 148;
  cudaGetDevice(dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, *dev);
  return std::min(sms, kXpMaxGrid);
}

template <bool FP8, bool DOWN>
static int xp_launch(const CUtensorMap& map, const XpMaps& x_maps, const XpParams& p, int dev, int sms, cudaStream_t st) {
  const eux_experts_desc& d = p.d;
  // the ring holds a block of every group; the routing's counts lie where the ring will be
  const int room = xp_layout(DOWN, d.n_tokens, d.n_experts, d.n_tokens * d.topk).room;
  if (xp_stages(FP8, room, FP8 ? 32 : kXpAccColumns) < kXpGroups || xp_stages(FP8, room, kXpFewColumns) < kXpGroups || kXpThreads / 32 * d.n_experts * 4 > room) return EUX_ERR_TOO_LARGE;
  if (cudaError_t e = allow_smem<moe_experts_kernel<FP8, DOWN>>(dev, kXpDynamic); e != cudaSuccess) return (int)e;
  return launch_early(moe_experts_kernel<FP8, DOWN>, sms, kXpThreads, kXpDynamic, st, map, x_maps, p);
}

}  // namespace eux

using namespace eux;

extern "C" size_t eux_experts_workspace_bytes(const eux_experts_desc* d) {
  if (experts_check(d)) return 0;
  const XpSpace s = xp_space(d);
  return s.h + s.x + s.tables + s.parts;
}
extern "C" int eux_experts_maps(const eux_experts_desc* d, void* maps) {
  if (int rc = experts_check(d)) return rc;
  if (!d->w_gate_up || !d->w_down || !maps || ((uintptr_t)d->w_gate_up | (uintptr_t)d->w_down) & 15 || (uintptr_t)maps & 63) return EUX_ERR_BAD_ARG;
  CUtensorMap* const m = (CUtensorMap*)maps;
  if (int rc = xp_map(m, d->w_gate_up, d->fp8, 2 * (uint64_t)d->n_experts, d->inner, d->hidden, 64, 2)) return rc;
  return xp_map(m + 1, d->w_down, d->fp8, d->n_experts, d->hidden, d->inner, kXpRows, 1);
}
extern "C" size_t eux_experts_counter_words(const eux_experts_desc* d) { return experts_check(d) ? 0 : 2 * kXpMaxGrid; }

extern "C" int eux_experts_find_nan(const void* e4m3, size_t bytes, uint32_t* found, void* stream) {
  if (!e4m3 || !found || (uintptr_t)e4m3 & 15 || bytes % 16) return EUX_ERR_BAD_ARG;
  if (bytes == 0) return 0;
  int dev = 0;
  const size_t n = bytes / 16;
  moe_experts_nan_kernel<<<(int)std::min<size_t>((n + 511) / 512, 8 * xp_sms(&dev)), 512, 0, (cudaStream_t)stream>>>((const uint4*)e4m3, n, found);
  return (int)cudaGetLastError();
}

extern "C" int eux_experts_launch(const eux_experts_desc* d, void* stream) {
  if (int rc = experts_check(d)) return rc;
  if (d->n_tokens == 0) return 0;
  if (!d->x || !d->topk_idx || !d->topk_w || !d->out || !d->w_gate_up || !d->w_down || !d->workspace || !d->counters || !d->maps) return EUX_ERR_BAD_ARG;
  if (d->fp8 && (!d->gate_up_scale || !d->down_scale)) return EUX_ERR_BAD_ARG;
  if (((uintptr_t)d->x | (uintptr_t)d->out | (uintptr_t)d->w_gate_up | (uintptr_t)d->w_down | (uintptr_t)d->workspace) & 15 || (uintptr_t)d->maps & 63) return EUX_ERR_BAD_ARG;
  const cudaStream_t st = (cudaStream_t)stream;
  // Threads that share a stream share a workspace: their launches must not mix.
  static std::mutex launching;
  std::lock_guard<std::mutex> lock(launching);
  const CUtensorMap *up = (const CUtensorMap*)d->maps, *down = up + 1;
  XpParams p = {};
  p.d = *d;
  const XpSpace space = xp_space(d);
  char* at = (char*)d->workspace;
  p.h = (__nv_bfloat16*)at, at += space.h;
  p.h_pitch = space.h_pitch, p.x_pitch = space.x_pitch;
  if (space.sorted) {
    p.x = (__nv_bfloat16*)at, at += space.x;
    p.tables = (uint32_t*)at, at += space.tables;
  }
  p.part = (float*)at;
  p.part_rows = xp_part_rows(d);
  p.token_of = ((1 << 20) + d->topk - 1) / d->topk;
  int dev = 0;
  const int sms = xp_sms(&dev), entries = d->n_tokens * d->topk, runs = d->fp8 ? 2 : 1;
  XpMaps x = {}, h = {};
  if (int rc = space.sorted ? xp_map_rows(&x, p.x, entries, p.x_pitch, p.x_pitch, runs, entries)
                            : xp_map_rows(&x, d->x, d->n_tokens, d->hidden, std::max<int64_t>(d->x_stride, d->hidden), runs, 8)) return rc;
  if (int rc = xp_map_rows(&h, p.h, space.h_rows, p.h_pitch, p.h_pitch, runs, entries)) return rc;
  if (space.sorted) {
    const size_t smem = xp_table_bytes(d->n_experts, entries) + std::max<size_t>((size_t)kXpThreads / 32 * d->n_experts * 4, 16 * kXpThreads);
    if (cudaError_t e = allow_smem<moe_experts_sort_kernel>(dev, 200 * 1024); e != cudaSuccess) return (int)e;
    const int64_t pieces = (int64_t)entries * (p.x_pitch / 8);
    const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(sms, pieces / kXpThreads));
    if (int rc = launch_early(moe_experts_sort_kernel, grid, kXpThreads, smem, st, p, d->fp8 ? 32 : kXpAccColumns)) return rc;
  }
  if (int rc = d->fp8 ? xp_launch<true, false>(*up, x, p, dev, sms, st) : xp_launch<false, false>(*up, x, p, dev, sms, st)) return rc;
  return d->fp8 ? xp_launch<true, true>(*down, h, p, dev, sms, st) : xp_launch<false, true>(*down, h, p, dev, sms, st);
}

extern "C" int eux_experts_preload(void) {
  cudaFuncAttributes a;
  const void* kernels[] = {(const void*)moe_experts_kernel<false, false>, (const void*)moe_experts_kernel<false, true>,
                           (const void*)moe_experts_kernel<true, false>, (const void*)moe_experts_kernel<true, true>,
                           (const void*)moe_experts_sort_kernel, (const void*)moe_experts_nan_kernel};
  for (const void* k : kernels)
    if (cudaError_t e = cudaFuncGetAttributes(&a, k); e != cudaSuccess) return (int)e;
  return 0;
}
