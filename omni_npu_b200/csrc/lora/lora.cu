// Low-rank adapters of many requests beside a shared projection.
//
//   z[t, n]   = y[t, n] + scale[s] * sum_j B[s][n, j] * h[t, p(n), j],   h[t, p, j] = sum_k A[s][p, j, k] * x[t, k]
//   out[t, n] = z[t, n],   or   act(z[t, gate n]) * z[t, up n]
//
// for tokens t with adapter s = slots[t] (none: z = y).  y is the shared product; p(n) is the slice of column n (query, key and
// value of a joined projection have factors of their own).  Ranks are multiples of 16 (zero padded), 0 for a slice without an
// adapter; the slices' A of a slot are joined along the rank.  The padded ranks' h is 0 also where x holds an infinity.
//
// The factors lie in the order in which the matrix instructions take them, so that they are read in whole kilobytes and need no
// shuffling: as 8 x 8 matrices (rows of ldmatrix, unswizzled operands of tcgen05), B of stacks up to rank 32, whose products all are
// mma.sync's, as lanes hold it (g = lane / 4, q = lane % 4):
//   A  [K / 32][rank / 8][4][rank % 8][8]        8 of K each of eight ranks, four times
//   B  [N / 64][rank / 8][2][4][8][8]            (interleaved columns: [N / 32][rank / 8][1]...) 8 ranks each of eight columns,
//                                                the columns of matrix j of a block of 32: 8 (i / 2) + 2 j + i % 2
//   or [N / 32][rank / 16][v = 0, 1][lane][8]    columns 8 (g / 2) + 2 j + g % 2 of 32 for j = 2 v, 2 v + 1 times
//                                                k = 2 q, 2 q + 1, 2 q + 8, 2 q + 9 of 16
// K and N padded with zeros.  So the columns of a lane's results are eight neighbours.
//
// Tokens are grouped by adapter once a step (lora_plan_kernel: a stable counting sort, then tiles of up to `rows` tokens of one
// adapter).  Two launches apply the adapters, both bound by what they read and write:
//   lora_shrink_*_kernel  h: CTAs that share K per (tile, some of the joined ranks)
//   lora_expand_*_kernel  z: a CTA per (tile, run of column groups)
// so that many small pieces of work even out adapters of unlike ranks (one cluster per tile for both, h in distributed shared
// memory, took 56 us where this takes 15: 128 tokens of 31 adapters of ranks 8 to 64).  The second is launched while the first
// runs and has its first y and factors at hand by the time h is there.  Measured (us, and the time of the bytes at 6.56 TB/s):
// one token 4.5; 128 tokens of 128 adapters of rank 16, 14336 to 4096 18.1 / 12.4; 8192 tokens of 8, 4096 to 6144 56 / 42;
// the same to 2 x 14336 with silu, rank 32 166 / 121 in a short graph at 1.97 GHz, 185 called without a pause, which reaches the
// power limit (1.70 GHz); 8192 tokens of rank 64, 4096 to 6144 72 / 42, of rank 128 102.

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../common/device_once.h"
#include "../common/pdl.cuh"
#include "../common/ptx.cuh"
#include "../common/tensormap.h"
#include "../gemm/gated_act.cuh"

namespace b200 {

static constexpr int kLoraMaxSlices = 4;
static constexpr int kLanesRank = 32;            // up to this largest rank B lies in the order of lanes
static constexpr int kFewChunk = 4, kManyChunk = 16;  // 8-wide tiles of h that a CTA computes
static constexpr int kPlanThreads = 1024;

// ----------------------------------------------------------------------------------------------- grouping
struct LoraTile {
  int slot, start, count, pad;
};

// order: tokens by adapter (those without one last), in their own order within an adapter.
__global__ void __launch_bounds__(kPlanThreads)
lora_plan_kernel(const int* __restrict__ slots, int T, int L, int rows, int* __restrict__ order,
                 LoraTile* __restrict__ tiles, int* __restrict__ num_tiles, int* __restrict__ status) {
  extern __shared__ int counts[];                // [warps][L + 1], then totals and tile bases [L + 1] each
  const int groups = L + 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = kPlanThreads / 32;
  int* total = counts + warps * groups;
  int* tile_base = total + groups;
  pdl_trigger();
  pdl_wait();
  for (int i = threadIdx.x; i < warps * groups; i += kPlanThreads) counts[i] = 0;
  __syncthreads();
  const int chunk = ((T + warps - 1) / warps + 31) / 32 * 32;
  const long long lo = static_cast<long long>(warp) * chunk;
  const int hi = static_cast<int>(lo + chunk < T ? lo + chunk : T);
  int* mine = counts + warp * groups;
  for (int t0 = static_cast<int>(lo < T ? lo : T); t0 < hi; t0 += 32) {
    const int t = t0 + lane;
    int s = -2 - lane;                           // lanes past the end match nobody
    if (t < hi) {
      s = slots[t];
      if (s < -1 || s >= L) {
        atomicExch(status, kStatusBadArgument);
        s = -1;
      }
      if (s < 0) s = L;
    }
    const unsigned same = __match_any_sync(0xffffffffu, s);
    if (t < hi && __ffs(same) - 1 == lane) mine[s] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int g = threadIdx.x; g < groups; g += kPlanThreads) {
    int sum = 0;
    for (int w = 0; w < warps; ++w) {
      const int c = counts[w * groups + g];
      counts[w * groups + g] = sum;
      sum += c;
    }
    total[g] = sum;
  }
  __syncthreads();
  if (warp == 0) {                               // first token and first tile of every group
    int tok = 0, til = 0;
    for (int g0 = 0; g0 < groups; g0 += 32) {
      const int g = g0 + lane;
      const int c = g < groups ? total[g] : 0, n = (c + rows - 1) / rows;
      int a = c, b = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int ua = __shfl_up_sync(0xffffffffu, a, o), ub = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) a += ua, b += ub;
      }
      if (g < groups) {
        const int first = tok + a - c, tile = til + b - n;
        total[g] = first;
        tile_base[g] = tile;
        for (int i = 0; i < n; ++i)
          tiles[tile + i] = LoraTile{g < L ? g : -1, first + i * rows, min(rows, c - i * rows), 0};
      }
      tok += __shfl_sync(0xffffffffu, a, 31);
      til += __shfl_sync(0xffffffffu, b, 31);
    }
    if (lane == 0) *num_tiles = til;
  }
  __syncthreads();
  for (int t0 = static_cast<int>(lo < T ? lo : T); t0 < hi; t0 += 32) {
    const int t = t0 + lane;
    int s = -2 - lane;
    if (t < hi) {
      s = slots[t];
      if (s < 0 || s >= L) s = L;
    }
    const unsigned same = __match_any_sync(0xffffffffu, s);
    if (t < hi) order[total[s] + mine[s] + __popc(same & ((1u << lane) - 1))] = t;
    __syncwarp();
    if (t < hi && __ffs(same) - 1 == lane) mine[s] += __popc(same);
    __syncwarp();
  }
}

// ---------------------------------------------------------------------------------------------- the adapters
struct LoraParams {
  const __nv_bfloat16* x;
  const __nv_bfloat16* y;
  __nv_bfloat16* out;
  long long x_stride, y_stride, out_stride;
  const __nv_bfloat16* a;                        // [L, a_slot]
  const __nv_bfloat16* b;                        // [L, b_slot]
  long long a_slot, b_slot;
  const int* ranks;                              // [L, slices + 1]: of each slice, not padded, then the scale's bits
  const int* order;
  const LoraTile* tiles;
  const int* num_tiles;
  // h, rows in the order of the plan: few rows fp32 [parts][T][h_width], to be summed; many rows bf16 [2][h_width / 8][T][8], h
  // times the scale rounded and what that leaves
  void* h;
  long long h_plane;                             // T * h_width
  int h_width;                                   // slices * largest rank
  int T, K, slices, parts;
  int stages, stage_bytes;                       // many rows: the first kernel's ring
  int groups, buffers, max_rank;                 // many rows, tcgen05: column groups of all slices, groups in flight, bound of the ranks
  int boxes;                                     // 1: rows of x that follow one another are copied as a box
  int* status;
  int per;                                       // column groups of a CTA of the second kernel
  int n[kLoraMaxSlices];
  int h_pitch;                                   // elements between rows of h in shared memory
  float act_alpha, act_limit;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float lo_f(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float hi_f(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
__device__ __forceinline__ constexpr int padded_rank(int r) { return (r + 15) & ~15; }
// The slices' ranks of an adapter together.
__device__ __forceinline__ int joined_ranks(const LoraParams& p, int slot) {
  int sum = 0;
  for (int s = 0; s < p.slices; ++s) sum += padded_rank(p.ranks[slot * (p.slices + 1) + s]);
  return sum;
}
__device__ __forceinline__ float lora_scale(const LoraParams& p, int slot) {
  return __int_as_float(p.ranks[slot * (p.slices + 1) + p.slices]);
}

// The tile of a CTA, or false when there is none.  (Entries behind the last tile lie in the buffer.)
__device__ __forceinline__ bool lora_tile(const LoraParams& p, int tile, LoraTile& tl) {
  const int4 v = *reinterpret_cast<const int4*>(p.tiles + tile);
  if (tile >= *p.num_tiles) return false;
  tl = LoraTile{v.x, v.y, v.z, 0};
  return true;
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp16_or_zero(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// Whether joined rank `col` is a rank, not padding.  An infinity or NaN in x times the zeros of a padded rank is NaN, which would
// go on to every column: the padded ranks' h is taken as 0.
__device__ __forceinline__ bool is_rank(const LoraParams& p, int slot, int col) {
  const int* ranks = p.ranks + slot * (p.slices + 1);
  for (int s = 0; s < p.slices; ++s) {
    const int pad = padded_rank(ranks[s]);
    if (col < pad) return col < ranks[s];
    col -= pad;
  }
  return false;
}
__device__ __forceinline__ void keep_ranks(float4& v, int left) {
  v.x = left > 0 ? v.x : 0.f;
  v.y = left > 1 ? v.y : 0.f;
  v.z = left > 2 ? v.z : 0.f;
  v.w = left > 3 ? v.w : 0.f;
}

// Four of h times the scale as the sum of two bf16 (17 bits of the fp32 values), so that the product with B adds no rounding
// beside that of its result.
__device__ __forceinline__ void split_h(const float4& s, float scale, uint2& hi, uint2& lo) {
  const float f[4] = {s.x * scale, s.y * scale, s.z * scale, s.w * scale};
  float up[4], rest[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    up[e] = __bfloat162float(__float2bfloat16(f[e]));
    rest[e] = f[e] - up[e];
    if (!(rest[e] - rest[e] == 0.f)) rest[e] = 0.f;                    // beside an infinity
  }
  hi = make_uint2(pack_bf16x2(up[0], up[1]), pack_bf16x2(up[2], up[3]));
  lo = make_uint2(pack_bf16x2(rest[0], rest[1]), pack_bf16x2(rest[2], rest[3]));
}

// ---- h of few rows: 16 at most, K dealt to the parts and, in steps of 32, to the warps.  The factors are what is read: every
// lane has a ring of its own in shared memory for what it alone uses of A and x (no barrier between copy and product), 12 KB a
// warp however many ranks there are, so that four CTAs are resident (128 adapters of rank 16, K 14336: 13.2 us, with 24 KB
// and two CTAs 15.8).  A CTA computes 32 of the joined ranks: with 64, a ring of 12 KB has two stages only (both kernels, one
// token, three slices, rank 16: 4.5 us, 4.7 with 64 ranks; over ranks 8 to 64 and 1 to 128 tokens 4% more); with a ring of 9 KB
// 128 adapters take 20.1 us for both kernels, 18.4 so.
static constexpr int kFewThreads = 128, kFewWarps = kFewThreads / 32, kFewRing = 12 * 1024;

template <int NT>
__device__ __forceinline__ void shrink_rows(const LoraParams& p, const LoraTile& tl, int n0, int sum_r, int s_lo, int s_hi,
                                            uint32_t ring, float* d) {
  constexpr int STAGE = (NT + 2) * 512, D = kFewRing / STAGE;          // NT pieces of A, two rows of x
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const __nv_bfloat16* a = p.a + tl.slot * p.a_slot + (n0 / 8) * 256 + lane * 8;
  const long long a_step = sum_r * 32;
  const int swap = g >> 1 & 3;                                         // places of the pieces of x: ldmatrix without bank conflicts
  const bool ok0 = g < tl.count, ok1 = g + 8 < tl.count;               // (the other rows of h are not used)
  const __nv_bfloat16* x0 = p.x + (ok0 ? p.order[tl.start + g] : 0) * p.x_stride + t4 * 8;
  const __nv_bfloat16* x1 = p.x + (ok1 ? p.order[tl.start + g + 8] : 0) * p.x_stride + t4 * 8;
  const uint32_t at = ring + lane * 16, x_put = ring + NT * 512 + (g * 4 + (t4 ^ swap)) * 16;
  // 16 rows of x as four matrices: rows 0 - 7 and 8 - 15 of one piece of 8 of K, then of the next
  const uint32_t x_get = ring + NT * 512 + (lane >> 3 & 1) * 512 + ((lane & 7) * 4 + (lane >> 4 ^ (lane >> 1 & 3))) * 16;
  int put = 0;
  auto copy = [&](int s) {
    if (s < s_hi) {
      const uint32_t st = put * STAGE;
      put = put + 1 == D ? 0 : put + 1;
#pragma unroll
      for (int u = 0; u < NT; ++u) cp16(at + st + u * 512, a + s * a_step + u * 256);
      const bool in = s * 32 + t4 * 8 < p.K;                           // K is a multiple of 8
      const int k = in ? s * 32 : 0;
      if (ok0) cp16_or_zero(x_put + st, x0 + k, in);
      if (ok1) cp16_or_zero(x_put + st + 512, x1 + k, in);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int i = 0; i < D - 1; ++i) copy(s_lo + i * kFewWarps);
  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
  int get = 0;
  for (int s = s_lo; s < s_hi; s += kFewWarps) {
    asm volatile("cp.async.wait_group %0;" ::"n"(D - 2) : "memory");
    __syncwarp();
    const uint32_t st = get * STAGE;
    get = get + 1 == D ? 0 : get + 1;
    uint32_t v[4], w[4];
    ldmatrix4(v, x_get + st);
    ldmatrix4(w, x_get + st ^ 32);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      uint32_t b[4];                                                   // eight ranks, 32 of K
      ldmatrix4(b, at + st + j * 512);
      mma_bf16(acc[j], v[0], v[1], v[2], v[3], b[0], b[1]);
      mma_bf16(acc[j], w[0], w[1], w[2], w[3], b[2], b[3]);
    }
    copy(s + (D - 1) * kFewWarps);                                     // where the stage before this one was
  }
  __syncwarp();
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    *reinterpret_cast<float2*>(d + j * 8) = make_float2(acc[j][0], acc[j][1]);
    *reinterpret_cast<float2*>(d + 8 * kFewChunk * 8 + j * 8) = make_float2(acc[j][2], acc[j][3]);
  }
}

__global__ void __launch_bounds__(kFewThreads) lora_shrink_few_kernel(const LoraParams p) {
  constexpr int W = kFewChunk * 8;
  extern __shared__ __align__(128) char smem[];
  pdl_wait();
  pdl_trigger();                                                       // (the second kernel reads what was there before this one)
  LoraTile tl;
  if (!lora_tile(p, blockIdx.z, tl) || tl.slot < 0) return;
  const int sum_r = joined_ranks(p, tl.slot);
  const int n0 = blockIdx.y * W;
  if (n0 >= sum_r) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int nt = min(kFewChunk, (sum_r - n0) / 8);                     // even: ranks are multiples of 16
  const int steps = (p.K + 31) / 32;
  const int s_lo = static_cast<int>(static_cast<long long>(steps) * blockIdx.x / p.parts) + warp;
  const int s_hi = static_cast<int>(static_cast<long long>(steps) * (blockIdx.x + 1) / p.parts);
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * kFewRing;
  // (a warp's part of h goes where its ring was)
  const auto red = [&](int w) { return reinterpret_cast<float*>(smem + w * kFewRing); };
  float* d = red(warp) + g * W + t4 * 2;
  if (nt == 2) shrink_rows<2>(p, tl, n0, sum_r, s_lo, s_hi, ring, d);
  else shrink_rows<4>(p, tl, n0, sum_r, s_lo, s_hi, ring, d);
  __syncthreads();
  // the warps' parts in order, four columns a thread
  float* h = static_cast<float*>(p.h) + blockIdx.x * p.h_plane + static_cast<long long>(tl.start) * p.h_width + n0;
  for (int i = threadIdx.x; i < tl.count * nt * 2; i += kFewThreads) {
    const int row = i / (nt * 2), col = i % (nt * 2) * 4;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      const float4 v = *reinterpret_cast<const float4*>(red(w) + row * W + col);
      sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    *reinterpret_cast<float4*>(h + static_cast<long long>(row) * p.h_width + col) = sum;
  }
}

// ---- h of many rows: 128 rows of x and up to 128 of the joined ranks on tcgen05, the sum in tensor memory, in slabs of 64 of K
// through a ring of stages.  Rows of x that follow one another (a prompt's) are one TMA box a slab; others are gathered by eight
// warps in copies of 16 bytes (rows behind the tile's last are not copied: what lies there only reaches rows of h that nobody
// reads).  The factors lie in the order of unswizzled operands, so a slab of them is two bulk copies.  The parts of K, a CTA of
// the cluster each, meet in distributed shared memory.  Alone, 8192 tokens, K 4096: 20 us for 48 joined ranks, 27 for 192, 42 for
// 384 (x's bytes alone 10; some 8 us are the start, the first copies and the joining); with mma.sync, where every warp reads x
// from shared memory again for 32 of the ranks, 25 for 48 and 60 for 192.  Also slower: the fence between copies and products
// issued by the copying threads, which then wait for all their copies (384 ranks: 80), and TMA's gathers of four rows (85
// cycles each; both kernels 66 us for 56).
static constexpr int kManyCopies = 256, kManyThreads = kManyCopies + 64, kManyRows = 128, kSlab = 64, kManyRing = 208 * 1024;
static constexpr int kManyStages = 8, kXBytes = kManyRows * kSlab * 2;

// Arrive on an mbarrier once all of this thread's copies so far have landed (the arrival is one of the expected).
__device__ __forceinline__ void arrive_when_copied(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Words of descriptors of unswizzled operands: 128 bytes from eight rows to the next eight (high word, SBO) or `rows` times that
// of 16 bytes of a row to the next 16 (low word, LBO).  Above 18 bits, an address holds the CTA's rank in its cluster.
__device__ __forceinline__ constexpr uint32_t plain_hi(uint32_t sbo) { return sbo >> 4 | 1u << 14; }
__device__ __forceinline__ uint32_t plain_lo(uint32_t addr, uint32_t lbo) { return (addr & 0x3FFFF) >> 4 | (lbo >> 4) << 16; }

// A product of 16 of K.  HA, HB: the descriptors' high words; ACC: added to what is there.
template <uint32_t HA, uint32_t HB, bool ACC>
__device__ __forceinline__ void umma_words(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc) {
  asm volatile(
      "{\n\t"
      ".reg .b64 da, db;\n\t"
      ".reg .pred p;\n\t"
      "mov.b64 da, {%1, %3};\n\t"
      "mov.b64 db, {%2, %4};\n\t"
      "setp.eq.u32 p, %6, 1;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t"
      "}"
      :
      : "r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(HA), "r"(HB), "r"(idesc), "n"(ACC ? 1 : 0)
      : "memory");
}

__global__ void __launch_bounds__(kManyThreads, 2)
lora_shrink_many_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ LoraParams p) {
  constexpr int W = kManyChunk * 8;
  extern __shared__ __align__(128) char smem[];
  __shared__ uint64_t full[kManyStages], empty[kManyStages], done;
  __shared__ uint32_t tmem_slot, ranks_are[W / 32];                    // bits: not padding
  __shared__ int gave_up;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = (smem_u32(smem) + 1023) & ~1023u;
  char* ring_ptr = smem + (ring - smem_u32(smem));
  pdl_wait();
  LoraTile tl;
  if (!lora_tile(p, blockIdx.z, tl) || tl.slot < 0) return;
  const int first = p.order[tl.start];
  const bool box = p.boxes && p.order[tl.start + tl.count - 1] - first == tl.count - 1;   // (the order is ascending)
  // copies: eight lanes a row of 128 bytes, 32 rows at once
  const int crow = threadIdx.x >> 3, piece = threadIdx.x & 7;
  int order[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) order[i] = crow < 32 && crow + 32 * i < tl.count ? p.order[tl.start + crow + 32 * i] : 0;
  const int sum_r = joined_ranks(p, tl.slot);
  const float scale = lora_scale(p, tl.slot);
  const int n0 = blockIdx.y * W;
  if (n0 >= sum_r) return;
  const int width = min(W, sum_r - n0);                                // a multiple of 16
  const int slabs = (p.K + kSlab - 1) / kSlab, blocks = (p.K + 31) / 32;
  const int s_lo = static_cast<int>(static_cast<long long>(slabs) * blockIdx.x / p.parts);
  const int count = static_cast<int>(static_cast<long long>(slabs) * (blockIdx.x + 1) / p.parts) - s_lo;   // one at least
  const uint32_t tmem_cols = width > 64 ? 128 : width > 32 ? 64 : 32;
  // a slab's factors, and its rows of x where these are a box
  const char* a = reinterpret_cast<const char*>(p.a + tl.slot * p.a_slot) + n0 * 64;
  const long long a_step = static_cast<long long>(sum_r) * 64;
  int loaded = 0;
  auto load = [&](int i, int put) {
    const int s = (s_lo + i) * 2, steps = min(2, blocks - s);
    char* st = ring_ptr + put * p.stage_bytes;
    mbar_arrive_expect_tx(&full[put], steps * width * 64 + (box ? kXBytes : 0));
    if (box) tma_load_2d(st, &tm_x, &full[put], (s_lo + i) * kSlab, first);
    for (int u = 0; u < steps; ++u) bulk_load_1d(st + kXBytes + u * width * 64, a + (s + u) * a_step, width * 64, &full[put]);
  };
  if (threadIdx.x == kManyCopies + 32) {
    tma_prefetch_desc(&tm_x);
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&full[i], box ? 1 : kManyCopies + 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(&done, 1);
    gave_up = 0;
    fence_barrier_init();
    fence_proxy_async();
    for (; loaded < min(count, p.stages); ++loaded) load(loaded, loaded);   // (this thread's barriers, and places nobody has used)
  }
  if (warp == kManyCopies / 32) {
    tmem_alloc(&tmem_slot, tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  pdl_trigger();                                                       // (not before tensor memory is held: the second kernel takes some too)

  if (warp < kManyCopies / 32 && !box) {
    const __nv_bfloat16* xs[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) xs[i] = p.x + order[i] * p.x_stride + s_lo * kSlab + piece * 8;
    const uint32_t dst = ring + crow * 128 + ((piece ^ (crow & 7)) << 4);
    int put = 0;
    uint32_t phase = 1;                                                // (the first pass over the ring does not wait)
    for (int i = 0; i < count; ++i) {
      if (!__shfl_sync(0xffffffffu, lane > 0 || mbar_wait(&empty[put], phase), 0)) {
        if (lane == 0) atomicCAS(p.status, 0, kStatusTimeoutEmptyBarrier);
        break;
      }
      const bool in = (s_lo + i) * kSlab + piece * 8 < p.K;            // K is a multiple of 8
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (crow + 32 * u < tl.count) cp16_or_zero(dst + put * p.stage_bytes + u * 4096, in ? xs[u] + i * kSlab : p.x, in);
      arrive_when_copied(&full[put]);
      if (++put == p.stages) put = 0, phase ^= 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == kManyCopies / 32 + 1 && lane == 0) {
    // (the first pass over the ring went before)
    int put = loaded == p.stages ? 0 : loaded, i = loaded;
    uint32_t phase = loaded == p.stages ? 0 : 1;
    for (; i < count; ++i) {
      if (!mbar_wait(&empty[put], phase)) {
        atomicCAS(p.status, 0, kStatusTimeoutEmptyBarrier);
        break;
      }
      load(i, put);
      if (++put == p.stages) put = 0, phase ^= 1;
    }
  } else if (warp == kManyCopies / 32 && lane == 0) {
    const uint32_t idesc = make_idesc(1, 1, kManyRows, width);
    // x in rows of 128 bytes in the 128-byte swizzle; the factors: 128 bytes to the next eight of K, 512 to the next eight ranks
    constexpr uint32_t HX = kSmemDescHiSw128, HF = plain_hi(512);
    const uint32_t lo = plain_lo(ring, 0), stage_lo = p.stage_bytes >> 4, f_at = (kXBytes >> 4) + ((128u >> 4) << 16);
    int get = 0;
    uint32_t phase = 0;
    for (int i = 0; i < count; ++i) {
      if (!mbar_wait(&full[get], phase)) {
        atomicCAS(p.status, 0, kStatusTimeoutFullBarrier);
        gave_up = 1;
        break;
      }
      // Gathered rows were written through another proxy than the products read them.  (Here: a fence of the copying threads would
      // wait for all of their copies in flight.)
      if (!box) fence_proxy_async();
      tc_fence_after_sync();
      const uint32_t x_lo = lo + get * stage_lo, f_lo = x_lo + f_at, f_next = f_lo + width * 4;
      if ((s_lo + i) * 2 + 1 < blocks) {
        if (i == 0) umma_words<HX, HF, false>(tmem, x_lo, f_lo, idesc);
        else umma_words<HX, HF, true>(tmem, x_lo, f_lo, idesc);
        umma_words<HX, HF, true>(tmem, x_lo + 2, f_lo + 16, idesc);
        umma_words<HX, HF, true>(tmem, x_lo + 4, f_next, idesc);
        umma_words<HX, HF, true>(tmem, x_lo + 6, f_next + 16, idesc);
      } else {                                                         // the last 32 of K
        if (i == 0) umma_words<HX, HF, false>(tmem, x_lo, f_lo, idesc);
        else umma_words<HX, HF, true>(tmem, x_lo, f_lo, idesc);
        umma_words<HX, HF, true>(tmem, x_lo + 2, f_lo + 16, idesc);
      }
      tc_commit(&empty[get]);
      if (++get == p.stages) get = 0, phase ^= 1;
    }
    tc_commit(&done);
    if (!mbar_wait(&done, 0)) atomicCAS(p.status, 0, kStatusTimeoutTmemFull);
    tc_fence_before_sync();
  }
  if (warp < W / 32) {                                                 // (while the last products run)
    const uint32_t bits = __ballot_sync(0xffffffffu, is_rank(p, tl.slot, n0 + threadIdx.x));
    if (lane == 0) ranks_are[warp] = bits;
  }
  // Every product is through, and the ring free.  (The other warps wait here and not at the mbarrier: eight warps that poll it
  // slow down the two that work.)
  __syncthreads();
  if (*static_cast<volatile int*>(&gave_up)) {                         // what is in flight ends first (bounded waits)
    if (threadIdx.x == 0)
      for (int i = 0; i < p.stages; ++i) mbar_wait(&full[i], 0), mbar_wait(&full[i], 1);
    __syncthreads();
  }
  tc_fence_after_sync();
  float* part = reinterpret_cast<float*>(ring_ptr);
  const int pitch = width + 4;
  if (warp < kManyCopies / 32 && (warp & 3) * 32 < tl.count) {         // a quarter of the rows, every other 32 columns
    const int row = (warp & 3) * 32 + lane;
    for (int c = (warp >> 2) * 32; c < width; c += 64) {
      uint32_t v[32];
      tmem_ld_32x32b_x32(tmem + ((warp & 3) << 21) + c, v);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 32; j += 4)
        if (c + j < width)
          *reinterpret_cast<uint4*>(part + row * pitch + c + j) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    }
  }
  tc_fence_before_sync();
  // The cluster's CTAs have summed a part of K each.  Every one adds up its share of the elements in the order of the parts and
  // leaves them ready for the second kernel, whose many CTAs then need no more than copy them.
  cluster_arrive_release();
  cluster_wait_acquire();
  if (warp == kManyCopies / 32) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, tmem_cols);
  }
  // A warp takes four rows x 32 ranks: 128 bytes of a row at once from every part, 64 of h for eight ranks.  (With eight rows x 16
  // ranks, whole 16 bytes of h a lane but half as much of a part's row at once, the kernel takes 2 to 4 us more.)
  const int C = p.parts, rank = blockIdx.x, across = (width + 31) / 32, units = (tl.count + 3) / 4 * across;
  __nv_bfloat16* h = static_cast<__nv_bfloat16*>(p.h) + (static_cast<long long>(n0 / 8) * p.T + tl.start) * 8;
  for (int i = rank * (kManyThreads / 32) + warp; i < units; i += C * (kManyThreads / 32)) {
    const int row = i / across * 4 + (lane >> 3), v = i % across * 32 + (lane & 7) * 4;
    if (row >= tl.count || v >= width) continue;
    const uint32_t at = smem_u32(part + row * pitch + v);
    float4 q[8];                                                       // (8 parts at most)
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < C) q[c] = ld_shared_cluster_f4(mapa_shared(at, c));
    float4 sum = q[0];
#pragma unroll
    for (int c = 1; c < 8; ++c)
      if (c < C) sum.x += q[c].x, sum.y += q[c].y, sum.z += q[c].z, sum.w += q[c].w;
    const uint32_t is = ranks_are[v >> 5] >> (v & 31);                 // (ranks behind a padded one of the four are padded)
    keep_ranks(sum, __popc(is & 15));
    uint2 hi, lo;
    split_h(sum, scale, hi, lo);
    __nv_bfloat16* dst = h + (static_cast<long long>(v / 8) * p.T + row) * 8 + (v & 4);
    *reinterpret_cast<uint2*>(dst) = hi;
    *reinterpret_cast<uint2*>(dst + p.h_plane) = lo;
  }
  cluster_arrive_release();                                            // no CTA leaves while its part is read
  cluster_wait_acquire();
}

// ---- z: a CTA has a tile's rows and a run of column groups of one slice, 64 columns of y each (gated: 32 of gate and their 32 of
// up).  A warp takes 16 rows of a group at a time.  y comes through a ring of the lane's own; a lane's results are eight
// neighbouring columns twice, so y and the result move 16 bytes a lane.
static constexpr int kExpandThreads = 128;

// What both kernels find out first: the CTA's slice and groups in it.
struct LoraRun {
  int h0, first, r0, r1, N, groups, ga, gb;      // first rank in h, first column of y, padded ranks (of gate and of up), columns
  int real0, real1;                              // the ranks that are not padding
  const __nv_bfloat16 *b, *b_up;                 // factors, in blocks of 64 columns (gated: 32)
};

// per > 0: `at` is a CTA's number among the slices' runs of `per` groups; 0: the run starts at group `at` of all of the slices'.
template <bool GATED, bool LANES>
__device__ __forceinline__ LoraRun lora_run(const LoraParams& p, int slot, int at, int per) {
  constexpr int GW = GATED ? 32 : 64, BC = GATED || LANES ? 32 : 64;   // columns of a group, of a block of B
  LoraRun c;
  int slice = 0;
  c.h0 = c.first = 0;
  c.b = p.b + max(slot, 0) * p.b_slot;
  const int* ranks = p.ranks + max(slot, 0) * (p.slices + 1);
  if constexpr (GATED) {
    c.real0 = slot >= 0 ? ranks[0] : 0;
    c.real1 = slot >= 0 ? ranks[1] : 0;
    c.r0 = padded_rank(c.real0);
    c.r1 = padded_rank(c.real1);
  } else {
    for (;; ++slice) {
      c.real0 = slot >= 0 ? ranks[slice] : 0;
      c.r0 = padded_rank(c.real0);
      const int groups = (p.n[slice] + 63) / 64, steps = per ? (groups + per - 1) / per : groups;
      if (at < steps) break;
      at -= steps;
      c.h0 += c.r0;
      c.first += p.n[slice];
      c.b += static_cast<long long>((p.n[slice] + BC - 1) / BC) * c.r0 * BC;
    }
    c.r1 = c.r0;
    c.real1 = c.real0;
  }
  c.N = p.n[slice];
  c.groups = (c.N + GW - 1) / GW;
  c.b_up = c.b + (GATED ? static_cast<long long>(c.groups) * c.r0 * 32 : 0);
  c.ga = per ? at * per : at;
  c.gb = per ? min(c.groups, c.ga + per) : c.groups;
  return c;
}

// 16 rows (g, g + 8 of a lane) x 64 columns of y: into a ring's stage, `st` this lane's place of four of 512 bytes.  Columns behind
// the slice's last eight are read there; their results are not stored.
// Gated: the eight pieces of 16 bytes of a row are gate and up in turn, and a lane needs two neighbours; copied so, every request
// would be for halves of sectors, twice.  So lane q copies pieces q and 4 + q, the latter one place off, and finds its own without
// bank conflicts (other lanes' copies: a __syncwarp).
template <bool GATED>
__device__ __forceinline__ void copy_y(uint32_t st, const __nv_bfloat16* y, int group, int N, int t4, long long at0, long long at1) {
  const int col = group * 64 + t4 * 8, end = (GATED ? 2 : 1) * N - 8;
  const __nv_bfloat16 *src0 = y + min(col, end), *src1 = y + min(col + 32, end);
  constexpr uint32_t swap = GATED ? 16 : 0;
  cp16(st, src0 + at0);
  cp16((st + 512) ^ swap, src1 + at0);
  cp16(st + 1024, src0 + at1);
  cp16((st + 1536) ^ swap, src1 + at1);
}
template <bool GATED>
__device__ __forceinline__ void get_y(float (&v)[8][4], uint32_t st, int t4) {
  const uint32_t own = GATED ? (t4 >> 1) * 512 + ((t4 & 1) * 2 ^ t4 >> 1) * 16 - t4 * 16 : 0;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint4 u = lds16(GATED ? (st + own + i * 1024) ^ s * 16 : st + i * 1024 + s * 512);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[4 * s + j][2 * i] = lo_f(w[j]);
        v[4 * s + j][2 * i + 1] = hi_f(w[j]);
      }
    }
}

// A lane's results; out_row -1: not a row of the tile.
template <int ACT>
__device__ __forceinline__ void store_z(const LoraParams& p, const float (&acc)[8][4], __nv_bfloat16* out, int group, int left,
                                        long long at0, long long at1) {
  constexpr bool GATED = ACT != kActNone;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = 2 * i;
    const long long at = i ? at1 : at0;
    uint32_t o0[4], o1[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (GATED) {
        o0[j] = pack_bf16x2(gated_act(ACT, acc[j][e], acc[4 + j][e], p.act_alpha, p.act_limit),
                            gated_act(ACT, acc[j][e + 1], acc[4 + j][e + 1], p.act_alpha, p.act_limit));
      } else {
        o0[j] = pack_bf16x2(acc[j][e], acc[j][e + 1]);
        o1[j] = pack_bf16x2(acc[4 + j][e], acc[4 + j][e + 1]);
      }
    }
    __nv_bfloat16* row = out + at + group * (GATED ? 32 : 64);
    if (at >= 0 && left > 0) *reinterpret_cast<uint4*>(row) = make_uint4(o0[0], o0[1], o0[2], o0[3]);
    if (!GATED && at >= 0 && left > 32) *reinterpret_cast<uint4*>(row + 32) = make_uint4(o1[0], o1[1], o1[2], o1[3]);
  }
}

// ---- few rows: a warp has every fourth group.  B comes through the ring as well, 32 ranks a stage; y starts the accumulators.
template <int ACT, bool LANES>
__global__ void __launch_bounds__(kExpandThreads, 4) lora_expand_few_kernel(const LoraParams p) {
  constexpr bool GATED = ACT != kActNone;
  constexpr int BM = 16, STEP = 4, D = 4, STAGE = 2048 + 4096;
  constexpr int GW = GATED ? 32 : 64;                                  // columns of a slice in a group
  extern __shared__ __align__(128) char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const bool in_place = !GATED && p.out == p.y;
  // Everything but h is older than the first kernel, which has started only behind it: no wait yet.
  LoraTile tl;
  if (!lora_tile(p, blockIdx.y, tl)) {
    pdl_wait();
    return;
  }
  // where a lane's two rows start (rows behind the last read what the first does, and are not stored)
  const int t0 = p.order[tl.start + (g < tl.count ? g : 0)], t1 = p.order[tl.start + (g + 8 < tl.count ? g + 8 : 0)];
  const long long y0 = t0 * p.y_stride, y1 = t1 * p.y_stride;
  const long long o0 = g < tl.count ? t0 * p.out_stride : -1, o1 = g + 8 < tl.count ? t1 * p.out_stride : -1;
  const LoraRun c = lora_run<GATED, LANES>(p, tl.slot, blockIdx.x, p.per);
  const int k0 = c.r0 / 16, k1 = c.r1 / 16, ks = max(k0, k1);
  if (ks == 0 && in_place) {
    pdl_wait();
    return;
  }
  const float scale = tl.slot >= 0 ? lora_scale(p, tl.slot) : 0.f;
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * D * STAGE + lane * 16;
  const __nv_bfloat16* y = p.y + c.first;
  __nv_bfloat16* out = p.out + c.first + t4 * 8;
  // the ring's next stage: group cg, steps ck, ck + 1 of 16 ranks
  int cg = c.ga + warp, ck = 0;
  uint32_t put = ring;
  auto copy = [&]() {
    if (cg < c.gb) {
      const uint32_t st = put;
      put = put + STAGE == ring + D * STAGE ? ring : put + STAGE;
      if (ck == 0) copy_y<GATED>(st, y, cg, c.N, t4, y0, y1);
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (ck + k < ks) {
#pragma unroll
          for (int s = 0; s < 2; ++s) {                                // gated: gate and up; past the end of one, its last
            const int steps = GATED && s ? k1 : k0;
            const __nv_bfloat16* src =
                GATED   ? (s ? c.b_up : c.b) + (static_cast<long long>(cg) * steps + min(ck + k, max(steps - 1, 0))) * 512
                : LANES ? c.b + (static_cast<long long>(min(2 * cg + s, (c.N - 1) / 32)) * k0 + ck + k) * 512
                        : c.b + (static_cast<long long>(cg) * k0 + ck + k) * 1024 + s * 512;
            cp16(st + 2048 + k * 2048 + s * 1024, src + lane * 8);
            cp16(st + 2048 + k * 2048 + s * 1024 + 512, src + lane * 8 + 256);
          }
        }
      ck += 2;
      if (ck >= ks) {
        ck = 0;
        cg += STEP;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < D - 1; ++i) copy();
  pdl_wait();
  pdl_trigger();

  // h of this slice (gated: of both) into shared memory, [2][BM][h_pitch]
  const uint32_t h_at = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + 4 * D * STAGE;
  {
    const float* h = static_cast<const float*>(p.h) + static_cast<long long>(tl.start) * p.h_width + c.h0;
    __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(smem + 4 * D * STAGE);
    const int vecs = (GATED ? c.r0 + c.r1 : c.r0) / 4;
    for (int i = threadIdx.x; i < tl.count * vecs; i += kExpandThreads) {
      const int row = i / vecs, v = i % vecs * 4;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      const float* src = h + static_cast<long long>(row) * p.h_width + v;
#pragma unroll 4
      for (int part = 0; part < p.parts; ++part) {
        const float4 q = *reinterpret_cast<const float4*>(src + part * p.h_plane);
        sum.x += q.x, sum.y += q.y, sum.z += q.z, sum.w += q.w;
      }
      keep_ranks(sum, GATED && v >= c.r0 ? c.real1 - (v - c.r0) : c.real0 - v);
      uint2 hi, lo;
      split_h(sum, scale, hi, lo);
      *reinterpret_cast<uint2*>(dst + row * p.h_pitch + v) = hi;
      *reinterpret_cast<uint2*>(dst + (BM + row) * p.h_pitch + v) = lo;
    }
  }
  __syncthreads();
  const uint32_t hf = h_at + ((lane & 15) * p.h_pitch + (lane >> 4) * 8) * 2, lo_at = 2 * BM * p.h_pitch;
  // two tiles of eight columns, 16 ranks of each as two matrices
  const uint32_t b_lane = 2048 + (lane >> 3 & 1) * (GATED ? 512 : 1024) + (lane >> 4) * 128 + (lane & 7) * 16 - lane * 16;
  uint32_t get = ring;
  auto next = [&]() {
    asm volatile("cp.async.wait_group %0;" ::"n"(D - 2) : "memory");
    __syncwarp();
    const uint32_t st = get;
    get = get + STAGE == ring + D * STAGE ? ring : get + STAGE;
    return st;
  };
  for (int gi = c.ga + warp; gi < c.gb; gi += STEP) {
    float acc[8][4];
    uint32_t st = next();
    get_y<GATED>(acc, st, t4);
    for (int k = 0;;) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (k + u < ks) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (GATED && k + u >= (s ? k1 : k0)) continue;
            if (GATED || s == 0) {
              const uint32_t at = hf + (k + u) * 32 + (GATED && s ? c.r0 * 2 : 0);
              ldmatrix4(hi, at);
              ldmatrix4(lo, at + lo_at);
            }
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
              uint32_t b[4];
              if constexpr (LANES) {
                const uint4 v = lds16(st + 2048 + u * 2048 + s * 1024 + j * 256);
                b[0] = v.x, b[1] = v.y, b[2] = v.z, b[3] = v.w;
              } else {
                ldmatrix4(b, st + b_lane + u * 2048 + (GATED ? s * 1024 + j * 128 : (4 * s + j) * 128));
              }
              mma_bf16(acc[4 * s + j], hi[0], hi[1], hi[2], hi[3], b[0], b[1]);
              mma_bf16(acc[4 * s + j + 1], hi[0], hi[1], hi[2], hi[3], b[2], b[3]);
              mma_bf16(acc[4 * s + j], lo[0], lo[1], lo[2], lo[3], b[0], b[1]);
              mma_bf16(acc[4 * s + j + 1], lo[0], lo[1], lo[2], lo[3], b[2], b[3]);
            }
          }
        }
      copy();
      k += 2;
      if (k >= ks) break;
      st = next();
    }
    store_z<ACT>(p, acc, out, gi, c.N - gi * GW - t4 * 8, o0, o1);
  }
}

// ---- many rows, up to 32 ranks: mma.sync, half a tile's rows, a warp has every fourth group.  y starts the accumulators, and B stays
// in registers for the 64 rows: little to compute, so that four CTAs an SM keep memory busy (8192 tokens of rank 16, 4096 to
// 6144: 33 us for 31 of bytes; the tcgen05 kernel takes 4 to 10 more, gated 9 to 35).
// Gated, rank 32, 14336 columns: 147 us, issue slots half busy; four CTAs are too few warps (14.6 counted) for the chain of loads,
// products, activation and store, whose fixed latencies are what they wait for first.
// PAIRS: gated ranks above 144, whose h the tcgen05 kernel has no room for.  Every step of 16 ranks is used for 32 rows, and the
// registers take the step after next meanwhile.
template <int ACT, bool PAIRS>
__global__ void __launch_bounds__(kExpandThreads, PAIRS ? 3 : 4) lora_expand_many_kernel(const LoraParams p) {
  constexpr bool GATED = ACT != kActNone, LANES = !PAIRS;
  static_assert(GATED || LANES, "without an activation, ranks above 32 take the tcgen05 kernel");
  constexpr int BM = 64, STEP = 4, D = PAIRS ? 6 : 4, STAGE = 2048;
  constexpr int GW = GATED ? 32 : 64;                                  // columns of a slice in a group
  extern __shared__ __align__(128) char smem[];
  __shared__ long long y_row[BM], out_row[BM];                         // where a row of the tile starts; out_row -1: none
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const bool in_place = !GATED && p.out == p.y;
  // Everything but h is older than the first kernel, which has started only behind it: no wait yet.
  LoraTile tl;
  const int from = (blockIdx.y & 1) * BM;
  if (!lora_tile(p, blockIdx.y >> 1, tl) || from >= tl.count) {
    pdl_wait();
    return;
  }
  tl.start += from;
  tl.count = min(BM, tl.count - from);
  if (threadIdx.x < BM) {
    const bool ok = threadIdx.x < tl.count;
    const int t = p.order[tl.start + (ok ? threadIdx.x : 0)];          // (rows behind the last read what the first does)
    y_row[threadIdx.x] = t * p.y_stride;
    out_row[threadIdx.x] = ok ? t * p.out_stride : -1;
  }
  const LoraRun c = lora_run<GATED, LANES>(p, tl.slot, blockIdx.x, p.per);
  const int k0 = c.r0 / 16, k1 = c.r1 / 16, ks = max(k0, k1);
  if (ks == 0 && in_place) {
    pdl_wait();
    return;
  }
  const int ga = c.ga + warp, gb = c.gb, ms = (tl.count + 15) / 16;
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * D * STAGE + lane * 16;
  const __nv_bfloat16* y = p.y + c.first;
  __nv_bfloat16* out = p.out + c.first + t4 * 8;
  __syncthreads();
  int cg = ga, cm = 0;                                                 // the ring's next stage: group cg and its rows cm
  uint32_t put = ring;
  auto copy = [&]() {
    if (cg < gb) {
      copy_y<GATED>(put, y, cg, c.N, t4, y_row[cm * 16 + g], y_row[cm * 16 + g + 8]);
      put = put + STAGE == ring + D * STAGE ? ring : put + STAGE;
      if (++cm == ms) {
        cm = 0;
        cg += STEP;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < D - 1; ++i) copy();
  // B of two steps: eight times eight columns.  Gated, past the end of one of the two: its last, not used
  uint2 bv[2][8];
  auto load_b = [&](uint2 (&v)[8], int gi, int k) {
    if constexpr (LANES) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int steps = GATED && s ? k1 : k0, block = GATED ? gi : min(2 * gi + s, (c.N - 1) / 32);
        const __nv_bfloat16* src =
            (s && GATED ? c.b_up : c.b) + (static_cast<long long>(block) * steps + min(k, max(steps - 1, 0))) * 512 + lane * 8;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint4 q = *reinterpret_cast<const uint4*>(src + j * 256);
          v[4 * s + 2 * j] = make_uint2(q.x, q.y);
          v[4 * s + 2 * j + 1] = make_uint2(q.z, q.w);
        }
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int steps = j >= 4 ? k1 : k0;
      const __nv_bfloat16* src =
          (j >= 4 ? c.b_up : c.b) + (static_cast<long long>(gi) * steps + min(k, max(steps - 1, 0))) * 512 + (j & 3) * 64;
      v[j].x = *reinterpret_cast<const uint32_t*>(src + lane * 2);
      v[j].y = *reinterpret_cast<const uint32_t*>(src + lane * 2 + 256);
    }
  };
  if (ks > 0 && ga < gb) {
    load_b(bv[0], ga, 0);
    if (ks > 1) load_b(bv[1], ga, 1);
  }
  pdl_wait();
  pdl_trigger();

  // h of this slice (gated: of both) into shared memory, [2][BM][h_pitch]
  const uint32_t h_at = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + 4 * D * STAGE;
  {
    const __nv_bfloat16* h = static_cast<const __nv_bfloat16*>(p.h) + (static_cast<long long>(c.h0 / 8) * p.T + tl.start) * 8;
    const int pieces = (GATED ? c.r0 + c.r1 : c.r0) / 8;
    for (int i = threadIdx.x; i < 2 * tl.count * pieces; i += kExpandThreads) {
      const int row = i % tl.count, q = i / tl.count, rest = q >= pieces, piece = q - rest * pieces;
      cp16(h_at + ((rest * BM + row) * p.h_pitch + piece * 8) * 2,
           h + rest * p.h_plane + (static_cast<long long>(piece) * p.T + row) * 8);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  __syncthreads();
  const uint32_t hf = h_at + ((lane & 15) * p.h_pitch + (lane >> 4) * 8) * 2;
  const uint32_t lo_at = 2 * BM * p.h_pitch, m_step = 32 * p.h_pitch;
  uint32_t get = ring;
  // the accumulators of 16 rows, from a stage of the ring
  auto start = [&](float (&acc)[8][4]) {
    asm volatile("cp.async.wait_group %0;" ::"n"(D - 2) : "memory");
    if (GATED) __syncwarp();
    get_y<GATED>(acc, get, t4);
    get = get + STAGE == ring + D * STAGE ? ring : get + STAGE;
    copy();
  };
  // step k of h of rows m times its B
  auto multiply = [&](float (&acc)[8][4], int m, int k, const uint2 (&b)[8]) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (GATED && k >= (s ? k1 : k0)) continue;
      if (GATED || s == 0) {
        const uint32_t at = hf + m * m_step + k * 32 + (GATED && s ? c.r0 * 2 : 0);
        ldmatrix4(hi, at);
        ldmatrix4(lo, at + lo_at);
      }
#pragma unroll
      for (int j = 4 * s; j < 4 * s + 4; ++j) mma_bf16(acc[j], hi[0], hi[1], hi[2], hi[3], b[j].x, b[j].y);
#pragma unroll
      for (int j = 4 * s; j < 4 * s + 4; ++j) mma_bf16(acc[j], lo[0], lo[1], lo[2], lo[3], b[j].x, b[j].y);
    }
  };
  auto store = [&](const float (&acc)[8][4], int gi, int m) {
    store_z<ACT>(p, acc, out, gi, c.N - gi * GW - t4 * 8, out_row[m * 16 + g], out_row[m * 16 + g + 8]);
  };
  for (int gi = ga; gi < gb; gi += STEP) {
    const bool more = gi + STEP < gb;
    if constexpr (PAIRS) {
      // 32 rows at a time for every step's B, whose registers take the steps after it as soon as it has been used
      for (int m = 0; m < ms; m += 2) {
        const bool two = m + 1 < ms, last = m + 2 >= ms;
        float acc[2][8][4];
        start(acc[0]);
        if (two) start(acc[1]);
        for (int k = 0; k < ks; k += 2) {
          const bool tail = k + 2 >= ks;
          const int ng = tail && last && more ? gi + STEP : gi, nk = tail ? 0 : k + 2;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if (k + u < ks) {
              multiply(acc[0], m, k + u, bv[u]);
              if (two) multiply(acc[1], m + 1, k + u, bv[u]);
            }
            load_b(bv[u], ng, nk + u);
          }
        }
        store(acc[0], gi, m);
        if (two) store(acc[1], gi, m + 1);
      }
    } else {
      for (int m = 0; m < ms; ++m) {
        float acc[8][4];
        start(acc);
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (u < ks) multiply(acc, m, u, bv[u]);
        if (m + 1 == ms && more)
#pragma unroll
          for (int u = 0; u < 2; ++u)
            if (u < ks) load_b(bv[u], gi + STEP, u);
        store(acc, gi, m);
      }
    }
  }
}

// ---- many rows, more than 32 ranks: the products on tcgen05 (h's two parts one after the other along K), 64 columns of tensor
// memory a group, NB groups in flight.  CTAs stay for the whole kernel and share out (tiles x groups) evenly.  Four warps add y to
// what they read from tensor memory, 32 rows each; one thread issues the products, one warp copies h and, in bulk, B of each
// group.  Both kernels, 4096 to 6144: 8192 tokens of rank 64 72 us (94 with mma.sync), of rank 128 100 (149); 4096 tokens of rank
// 64 to 2 x 14336 with silu 103 (196); 1024 tokens of rank 64 22 (28).  Two CTAs an SM even if the ring of y is short for it: 2847
// tokens of ranks 33 to 128 40 us, 44 with one.
static constexpr int kExpandTcThreads = 192;

__device__ __forceinline__ void tmem_ld_16x256b_x8(uint32_t taddr, float (&v)[8][4]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(v[0][0]), "=f"(v[0][1]), "=f"(v[0][2]), "=f"(v[0][3]), "=f"(v[1][0]), "=f"(v[1][1]), "=f"(v[1][2]), "=f"(v[1][3]),
        "=f"(v[2][0]), "=f"(v[2][1]), "=f"(v[2][2]), "=f"(v[2][3]), "=f"(v[3][0]), "=f"(v[3][1]), "=f"(v[3][2]), "=f"(v[3][3]),
        "=f"(v[4][0]), "=f"(v[4][1]), "=f"(v[4][2]), "=f"(v[4][3]), "=f"(v[5][0]), "=f"(v[5][1]), "=f"(v[5][2]), "=f"(v[5][3]),
        "=f"(v[6][0]), "=f"(v[6][1]), "=f"(v[6][2]), "=f"(v[6][3]), "=f"(v[7][0]), "=f"(v[7][1]), "=f"(v[7][2]), "=f"(v[7][3])
      : "r"(taddr)
      : "memory");
}

// Products of one group: `steps` of 16 ranks, for both parts of h.
template <int ROWS, int BW>
__device__ __forceinline__ void expand_group(uint32_t d, uint32_t h_lo, uint32_t h_part, uint32_t b_lo, int steps) {
  constexpr uint32_t HI = plain_hi(128), idesc = make_idesc(1, 1, ROWS, BW);
  constexpr uint32_t h_step = ROWS * 32 / 16, b_step = BW * 32 / 16;
  umma_words<HI, HI, false>(d, h_lo, b_lo, idesc);
  umma_words<HI, HI, true>(d, h_lo + h_part, b_lo, idesc);
  for (int k = 1; k < steps; ++k) {
    umma_words<HI, HI, true>(d, h_lo + k * h_step, b_lo + k * b_step, idesc);
    umma_words<HI, HI, true>(d, h_lo + h_part + k * h_step, b_lo + k * b_step, idesc);
  }
}

template <int ACT, int D>
__global__ void __launch_bounds__(kExpandTcThreads, D == 8 ? 1 : 2)
lora_expand_tc_kernel(const __grid_constant__ LoraParams p) {
  constexpr bool GATED = ACT != kActNone;
  constexpr int ROWS = 128, STAGE = 2048, GW = GATED ? 32 : 64;
  extern __shared__ __align__(128) char smem[];
  __shared__ uint64_t b_full[4], d_full[4], d_empty[4], h_full;
  __shared__ uint32_t tmem_slot;
  __shared__ int token[ROWS], gave_up;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const bool in_place = !GATED && p.out == p.y;
  // Everything but h is older than the first kernel, which has started only behind it: no wait yet.
  const long long work = static_cast<long long>(*p.num_tiles) * p.groups;
  long long pos = work * blockIdx.x / gridDim.x;
  const long long end = work * (blockIdx.x + 1) / gridDim.x;
  const int NB = p.buffers;
  if (threadIdx.x == 160) {
    for (int i = 0; i < NB; ++i) {
      mbar_init(&b_full[i], 1);
      mbar_init(&d_full[i], 1);
      mbar_init(&d_empty[i], 4);
    }
    mbar_init(&h_full, 1);
    gave_up = 0;
    fence_barrier_init();
  }
  // shared memory: rings of the four warps, NB times B of a group, h [2][ranks / 8][ROWS][8]
  char* b_ptr = smem + 4 * D * STAGE;
  const int b_bytes = p.max_rank * 128;
  char* h_ptr = b_ptr + NB * b_bytes;
  bool started = false;
  // (no kernel behind this one starts before tensor memory is held: it may take some too)
  auto ready = [&]() {
    if (started) return;
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    pdl_wait();
    pdl_trigger();
  };
  // each role's place among the NB, and in the warps' rings
  int buf = 0;
  uint32_t phase = warp == 5 ? 1 : 0, h_phase = 0, tmem = 0;
  const uint32_t ring = smem_u32(smem) + warp * D * STAGE + lane * 16;
  uint32_t put = ring, get = ring;

  while (pos < end) {
    // a stretch: one tile, one slice
    const int tile = static_cast<int>(pos / p.groups);
    const int4 entry = *reinterpret_cast<const int4*>(p.tiles + tile);
    const int slot = entry.x, start = entry.y, rows = entry.z;
    LoraRun c = lora_run<GATED, false>(p, slot, static_cast<int>(pos % p.groups), 0);
    const int n = static_cast<int>(min(static_cast<long long>(c.gb - c.ga), end - pos));
    pos += n;
    const int k0 = c.r0 / 16, k1 = c.r1 / 16;
    const bool products = k0 + k1 > 0;
    if (!products && in_place) continue;
    const int hk = GATED ? c.r0 + c.r1 : c.r0;
    __syncthreads();                                                   // the stretch before is through
    if (threadIdx.x < ROWS) token[threadIdx.x] = p.order[start + (threadIdx.x < rows ? threadIdx.x : 0)];
    if (warp < 4) {
      asm volatile("bar.sync 1, 128;" ::: "memory");
      const int row0 = warp * (ROWS / 4), ms = min(ROWS / 64, max(0, (rows - row0 + 15) / 16));
      const __nv_bfloat16* y = p.y + c.first;
      __nv_bfloat16* out = p.out + c.first + t4 * 8;
      int cg = ms ? 0 : n, cm = 0;
      auto copy = [&]() {
        if (cg < n) {
          const int row = row0 + cm * 16 + g;
          copy_y<GATED>(put, y, c.ga + cg, c.N, t4, token[row] * p.y_stride, token[row + 8] * p.y_stride);
          put = put + STAGE == ring + D * STAGE ? ring : put + STAGE;
          if (++cm == ms) cm = 0, ++cg;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
#pragma unroll
      for (int i = 0; i < D - 1; ++i) copy();
      ready();
      tmem = tmem_slot;
      for (int i = 0; i < n; ++i) {
        if (products) {
          if (!*static_cast<volatile int*>(&gave_up) && !mbar_wait(&d_full[buf], phase)) {
            atomicCAS(p.status, 0, kStatusTimeoutTmemFull);
            gave_up = 1;
          }
          tc_fence_after_sync();
          __syncwarp();
          if (ms == 0 && lane == 0) mbar_arrive(&d_empty[buf]);
        }
#pragma unroll 1
        for (int m = 0; m < ms; ++m) {
          float acc[8][4], v[8][4];
          if (products) {
            tmem_ld_16x256b_x8(tmem + ((warp * 32 + m * 16) << 16) + buf * 64, acc);
            tmem_ld_wait();
            if (m + 1 == ms) {
              tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) mbar_arrive(&d_empty[buf]);
            }
          }
          asm volatile("cp.async.wait_group %0;" ::"n"(D - 2) : "memory");
          if (GATED) __syncwarp();
          get_y<GATED>(v, get, t4);
          get = get + STAGE == ring + D * STAGE ? ring : get + STAGE;
          copy();
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              acc[j][e] = (GATED ? (j < 4 ? k0 : k1) != 0 : products) ? acc[j][e] + v[j][e] : v[j][e];
          const int row = row0 + m * 16 + g;
          store_z<ACT>(p, acc, out, c.ga + i, c.N - (c.ga + i) * GW - t4 * 8, row < rows ? token[row] * p.out_stride : -1,
                       row + 8 < rows ? token[row + 8] * p.out_stride : -1);
        }
        if (products && ++buf == NB) buf = 0, phase ^= 1;
      }
    } else if (warp == 4) {
      if (!started) {
        tmem_alloc(&tmem_slot, NB * 64);
        tmem_relinquish();
      }
      ready();
      tmem = tmem_slot;
      if (products && lane == 0) {
        const uint32_t h_lo = plain_lo(smem_u32(h_ptr), ROWS * 16), b_base = plain_lo(smem_u32(b_ptr), GW * 16);
        const uint32_t h_part = hk / 8 * ROWS;                         // (in 16 bytes)
        const uint32_t h_up = h_lo + c.r0 / 8 * ROWS, b_up = c.r0 * 4; // gated: r0 / 8 times 32 columns
        bool ok = !*static_cast<volatile int*>(&gave_up) && mbar_wait(&h_full, h_phase);
        for (int i = 0; i < n && ok; ++i) {
          ok = mbar_wait(&b_full[buf], phase) && mbar_wait(&d_empty[buf], phase ^ 1);
          if (!ok) break;
          tc_fence_after_sync();
          const uint32_t d = tmem + buf * 64, b_lo = b_base + buf * (b_bytes >> 4);
          if (k0) expand_group<ROWS, GW>(d, h_lo, h_part, b_lo, k0);
          if (GATED && k1) expand_group<ROWS, GW>(d + 32, h_up, h_part, b_lo + b_up, k1);
          tc_commit(&d_full[buf]);
          if (++buf == NB) buf = 0, phase ^= 1;
        }
        if (!ok) {
          atomicCAS(p.status, 0, kStatusTimeoutFullBarrier);
          gave_up = 1;
        }
      }
      h_phase ^= products;
    } else {
      int i = 0;
      // B of a group (gated: of gate and of up), when the products that were before in its place are through
      auto load = [&]() {
        if (*static_cast<volatile int*>(&gave_up) || !mbar_wait(&d_full[buf], phase)) return false;
        char* dst = b_ptr + buf * b_bytes;
        mbar_arrive_expect_tx(&b_full[buf], (GATED ? hk * 32 : hk * 64) * 2);
        const long long at = c.ga + i;
        if (GATED) {
          if (c.r0) bulk_load_1d(dst, c.b + at * c.r0 * 32, c.r0 * 64, &b_full[buf]);
          if (c.r1) bulk_load_1d(dst + c.r0 * 64, c.b_up + at * c.r1 * 32, c.r1 * 64, &b_full[buf]);
        } else {
          bulk_load_1d(dst, c.b + at * c.r0 * 64, c.r0 * 128, &b_full[buf]);
        }
        if (++buf == NB) buf = 0, phase ^= 1;
        return true;
      };
      bool ok = true;
      if (products && lane == 0)
        for (; i < min(n, NB) && ok; ++i) ok = load();
      __syncwarp();
      ready();
      if (products) {
        const int pieces = hk / 8;
        if (lane == 0) mbar_arrive_expect_tx(&h_full, 2 * pieces * rows * 16);
        __syncwarp();
        const __nv_bfloat16* h = static_cast<const __nv_bfloat16*>(p.h) + (static_cast<long long>(c.h0 / 8) * p.T + start) * 8;
        for (int q = lane; q < 2 * pieces; q += 32)
          bulk_load_1d(h_ptr + q * ROWS * 16, h + q / pieces * p.h_plane + static_cast<long long>(q % pieces) * p.T * 8,
                       rows * 16, &h_full);
        __syncwarp();
        if (lane == 0) {
          for (; i < n && ok; ++i) ok = load();
          if (!ok) {
            atomicCAS(p.status, 0, kStatusTimeoutEmptyBarrier);
            gave_up = 1;
          }
        }
        __syncwarp();
      }
    }
    started = true;
  }
  if (!started) {
    pdl_wait();
    return;
  }
  __syncthreads();
  if (*static_cast<volatile int*>(&gave_up)) {                         // what is in flight ends first (bounded waits)
    if (threadIdx.x == 0)
      for (int q = 0; q < 2; ++q) {
        mbar_wait(&h_full, q);
        for (int i = 0; i < NB; ++i) mbar_wait(&b_full[i], q), mbar_wait(&d_full[i], q);
      }
    __syncthreads();
  }
  if (warp == 4) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, NB * 64);
  }
}

static constexpr int kShrinkFewSmem = kFewWarps * kFewRing, kExpandFewSmem = 140 * 1024, kExpandManySmem = 184 * 1024, kExpandTcSmem = 224 * 1024;

template <int ACT, bool LANES>
static int launch_few(const LoraParams& p, unsigned tiles, unsigned chunks, unsigned blocks, cudaStream_t stream) {
  auto expand = lora_expand_few_kernel<ACT, LANES>;
  static DeviceOnce once;
  int dev;
  if (once.needed(&dev)) {
    const auto attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
    if (cudaFuncSetAttribute(lora_shrink_few_kernel, attr, kShrinkFewSmem) != cudaSuccess ||
        cudaFuncSetAttribute(expand, attr, kExpandFewSmem) != cudaSuccess)
      return -3;
    once.mark(dev);
  }
  const size_t smem = 4 * 4 * 6144 + 2 * sizeof(__nv_bfloat16) * 16 * p.h_pitch;
  if (smem > kExpandFewSmem || tiles > 65535) return -2;
  if (launch_pdl(lora_shrink_few_kernel, dim3(p.parts, chunks, tiles), dim3(kFewThreads), kShrinkFewSmem, stream, 1, p) != cudaSuccess ||
      launch_pdl(expand, dim3(blocks, tiles), dim3(kExpandThreads), smem, stream, 1, p) != cudaSuccess)
    return -3;
  return 0;
}

template <int ACT, typename Kernel>
static int launch_many(const LoraParams& p, Kernel expand, int attr_smem, unsigned tiles, unsigned chunks, dim3 grid, int threads,
                       size_t smem, DeviceOnce& once, cudaStream_t stream) {
  int dev;
  if (once.needed(&dev)) {
    const auto attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
    if (cudaFuncSetAttribute(lora_shrink_many_kernel, attr, kManyRing + 1024) != cudaSuccess ||
        cudaFuncSetAttribute(expand, attr, attr_smem) != cudaSuccess)
      return -3;
    once.mark(dev);
  }
  if (smem > static_cast<size_t>(attr_smem) || tiles > 32767) return -2;
  CUtensorMap tm_x = {};
  if (p.boxes && make_tensormap_2d(&tm_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.x, p.T, p.K, p.x_stride, kManyRows, kSlab,
                                   CU_TENSOR_MAP_SWIZZLE_128B) != 0)
    return -4;
  if (launch_pdl(lora_shrink_many_kernel, dim3(p.parts, chunks, tiles), dim3(kManyThreads), p.stages * p.stage_bytes + 1024, stream,
                 p.parts, tm_x, p) != cudaSuccess ||
      launch_pdl(expand, grid, dim3(threads), smem, stream, 1, p) != cudaSuccess)
    return -3;
  return 0;
}

// Shared memory of the tcgen05 kernel: h of 128 rows, two or four groups' B, and a ring of y; two CTAs an SM, or one with a ring of
// twice the depth.  ctas 0: too much.
struct TcPlan {
  int buffers, depth, ctas;
  size_t smem;
};
static TcPlan tc_plan(bool gated, int max_rank) {
  const size_t h = (gated ? 2 : 1) * max_rank * 128 * 4, b = max_rank * 128, ring = 4 * 2048;
  const size_t half = 114 * 1024 - 1792;
  for (int depth = 4; depth > 1; depth /= 2)
    for (int buffers = 4; buffers > 1; buffers /= 2)
      if (h + buffers * b + depth * ring <= half) return {buffers, depth, 2, h + buffers * b + depth * ring};
  for (int depth = 8; depth > 2; depth /= 2)
    if (h + 2 * b + depth * ring <= kExpandTcSmem) return {2, depth, 1, h + 2 * b + depth * ring};
  return {2, 0, 0, 0};
}

template <int ACT>
static int launch_lora(LoraParams& p, bool many, int max_tiles, unsigned chunks, int slices, int groups, cudaStream_t stream) {
  constexpr bool GATED = ACT != kActNone;
  const unsigned tiles = static_cast<unsigned>(max_tiles);
  const TcPlan tc = tc_plan(GATED, p.max_rank);
  const long long work = static_cast<long long>(groups) * max_tiles;
  if (many && p.max_rank > kLanesRank && tc.ctas) {
    static DeviceOnce once2, once4, once8;
    p.buffers = tc.buffers;
    const auto launch = [&](auto kernel, DeviceOnce& once) {
      return launch_many<ACT>(p, kernel, kExpandTcSmem, tiles, chunks, dim3(sm_count() * tc.ctas), kExpandTcThreads, tc.smem, once, stream);
    };
    return tc.depth == 2   ? launch(lora_expand_tc_kernel<ACT, 2>, once2)
           : tc.depth == 4 ? launch(lora_expand_tc_kernel<ACT, 4>, once4)
                           : launch(lora_expand_tc_kernel<ACT, 8>, once8);
  }
  // column groups of a CTA: two rounds of the resident CTAs in all, or for few rows one, where a CTA's start is most of its
  // time (128 adapters of rank 16, 4096 columns: 7.7 us, with two rounds 9.6); a group a warp at least
  const long long want = many ? static_cast<long long>(groups) * (max_tiles + p.T / kManyRows) / (148 * 8) : work / (148 * 2);
  p.per = static_cast<int>(std::max(1LL, (want + 3) / 4)) * 4;
  unsigned blocks = 0;
  for (int s = 0; s < (GATED ? 1 : slices); ++s) blocks += ((GATED ? (p.n[s] + 31) / 32 : (p.n[s] + 63) / 64) + p.per - 1) / p.per;
  if (!many)
    return p.max_rank > kLanesRank ? launch_few<ACT, false>(p, tiles, chunks, blocks, stream)
                                   : launch_few<ACT, true>(p, tiles, chunks, blocks, stream);
  static DeviceOnce once;
  const size_t smem = 4 * (p.max_rank > kLanesRank ? 6 : 4) * 2048 + 2 * sizeof(__nv_bfloat16) * 64 * p.h_pitch;
  const dim3 grid(blocks, 2 * tiles);
  if constexpr (GATED)
    if (p.max_rank > kLanesRank) {
      static DeviceOnce pairs;
      return launch_many<ACT>(p, lora_expand_many_kernel<ACT, true>, kExpandManySmem, tiles, chunks, grid, kExpandThreads, smem, pairs, stream);
    }
  return launch_many<ACT>(p, lora_expand_many_kernel<ACT, false>, kExpandManySmem, tiles, chunks, grid, kExpandThreads, smem, once, stream);
}

// Parts of K that a step's h is summed from, a CTA each (many rows: of a cluster).  They set the order of the sums, so they follow
// from the step and the stack's bounds alone, not from the adapters that happen to be loaded beside a token's own.  Few rows (tiles
// of 16): as many as the slots let be resident, whatever the number of tokens, so that a row does not depend on it.  Many rows: as
// many as fill the SMs, given the pieces of 128 ranks that a tile may have, in a power of two (clusters of seven: 2048 tokens to
// 2 x 14336 of a stack of rank 128 79 us, of four or eight 73).  Going by the ranks that are loaded, 8192 tokens of rank 16 in a
// stack of 128 took 81 us for 84, and with the stack's own rank the same.
static int lora_parts(int K, int rows, int max_tiles, int num_slots, int chunks) {
  if (rows < kManyRows) return std::min(std::max(std::min((K + 511) / 512, 592 / num_slots), 1), 16);
  const int pieces = max_tiles * chunks, want = std::min((K + 127) / 128, (296 + pieces / 2) / pieces);
  return want >= 8 ? 8 : want >= 4 ? 4 : want >= 2 ? 2 : 1;
}

}  // namespace b200

// Bytes of scratch for a step's h.
extern "C" long long b200_lora_scratch_bytes(int T, int K, int rows, int max_tiles, int num_slots, int slices, int max_rank) {
  return 4LL * T * slices * max_rank * (rows < b200::kManyRows ? b200::lora_parts(K, rows, max_tiles, num_slots, 1) : 1);
}

// Groups tokens by adapter.  tiles: at least T / rows + min(T, L + 1) of four ints.
extern "C" int b200_lora_plan(const int* slots, int T, int L, int rows, int* order, int* tiles, int* num_tiles, int* status,
                              cudaStream_t stream) {
  using namespace b200;
  if (L < 1 || L > 512 || rows < 1) return -1;
  const size_t smem = sizeof(int) * (kPlanThreads / 32 + 2) * (L + 1);
  static DeviceOnce once;
  int dev;
  if (once.needed(&dev)) {
    if (cudaFuncSetAttribute(lora_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(sizeof(int) * (kPlanThreads / 32 + 2) * 513)) != cudaSuccess)
      return -3;
    once.mark(dev);
  }
  return launch_pdl(lora_plan_kernel, dim3(1), dim3(kPlanThreads), smem, stream, 1, slots, T, L, rows, order,
                    reinterpret_cast<LoraTile*>(tiles), num_tiles, status) == cudaSuccess ? 0 : -3;
}

// ranks: [L, slices + 1], a slot's ranks and the bits of its scale.  max_tiles: tiles that the plan may have, of `rows` (16 or 128)
// tokens each.  h: scratch of b200_lora_scratch_bytes.  n: columns of each slice.  max_rank: bound of the ranks; mean_rank: about
// what a tile's joined ranks are (16 at least).  act: 0 adds, a gated kind of gemm/gated_act.cuh joins gate and up (alternating
// groups of eight columns of y).
extern "C" int b200_lora(const void* x, long long x_stride, const void* y, long long y_stride, void* out, long long out_stride,
                         const void* a, long long a_slot, const void* b, long long b_slot, const int* ranks, const int* order,
                         const int* tiles, const int* num_tiles, int max_tiles, int rows, void* h, int T, int num_slots, int K,
                         int slices, const int* n, int max_rank, int mean_rank, int act, float act_alpha, float act_limit,
                         int* status, cudaStream_t stream) {
  using namespace b200;
  if (slices < 1 || slices > kLoraMaxSlices || (K & 7) || max_rank < 16 || mean_rank < 16 || (max_rank & 15) || max_tiles < 1 ||
      (rows != 16 && rows != kManyRows))
    return -1;
  if (act != kActNone && (!act_is_gated(act) || slices != 2 || n[0] != n[1])) return -1;
  LoraParams p;
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.y = static_cast<const __nv_bfloat16*>(y);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.x_stride = x_stride;
  p.y_stride = y_stride;
  p.out_stride = out_stride;
  p.a = static_cast<const __nv_bfloat16*>(a);
  p.b = static_cast<const __nv_bfloat16*>(b);
  p.a_slot = a_slot;
  p.b_slot = b_slot;
  p.ranks = ranks;
  p.order = order;
  p.tiles = reinterpret_cast<const LoraTile*>(tiles);
  p.num_tiles = num_tiles;
  p.h = h;
  p.h_width = slices * max_rank;
  p.h_plane = static_cast<long long>(T) * p.h_width;
  p.T = T;
  p.K = K;
  p.boxes = x_stride >= K;                       // (not where rows overlap)
  p.slices = slices;
  p.status = status;
  const bool many = rows == kManyRows, gated = act != kActNone;
  p.act_alpha = act_alpha;
  p.act_limit = act_limit;
  const int width = (many ? kManyChunk : kFewChunk) * 8;
  const unsigned chunks = (p.h_width + width - 1) / width;
  p.parts = lora_parts(K, rows, max_tiles, num_slots, chunks);
  // the first kernel's ring: two CTAs an SM, or all of it for one where there are too few
  const long long ctas = static_cast<long long>(p.parts) * max_tiles * ((mean_rank + width - 1) / width);
  p.stage_bytes = kXBytes + std::min(p.h_width, width) * kSlab * 2;
  p.stages = std::min((ctas > 148 ? kManyRing / 2 : kManyRing) / p.stage_bytes, kManyStages);
  p.h_pitch = (gated ? 2 : 1) * max_rank + 8;    // eight rows of 16 bytes are in banks of their own
  int groups = 0;
  for (int s = 0; s < kLoraMaxSlices; ++s) {
    p.n[s] = s < slices ? n[s] : 0;
    if (p.n[s] & 7) return -1;
    if (!gated || s == 0) groups += gated ? (p.n[s] + 31) / 32 : (p.n[s] + 63) / 64;
  }
  p.groups = groups;
  p.max_rank = max_rank;
  switch (act) {
    case kActNone: return launch_lora<kActNone>(p, many, max_tiles, chunks, slices, groups, stream);
    case kActSilu: return launch_lora<kActSilu>(p, many, max_tiles, chunks, slices, groups, stream);
    case kActClampedGlu: return launch_lora<kActClampedGlu>(p, many, max_tiles, chunks, slices, groups, stream);
    case kActGeluTanh: return launch_lora<kActGeluTanh>(p, many, max_tiles, chunks, slices, groups, stream);
    default: return launch_lora<kActReluGate>(p, many, max_tiles, chunks, slices, groups, stream);
  }
}
