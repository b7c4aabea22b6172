// Low-rank adapters of many requests beside a shared projection.
//
//   z[t, n]   = y[t, n] + scale[s] * sum_j B[s][n, j] * h[t, p(n), j],   h[t, p, j] = sum_k A[s][p, j, k] * x[t, k]
//   out[t, n] = z[t, n],   or   act(z[t, gate n]) * z[t, up n]
//
// for tokens t with adapter s = slots[t] (none: z = y).  y is the shared product; p(n) is the slice of column n (query, key and
// value of a joined projection have factors of their own).  A slot's factors lie packed: A as [sum of ranks, K], B as one
// [N_p, rank_p] after another; ranks are multiples of 16 (zero padded), 0 for a slice without an adapter.
//
// Tokens are grouped by adapter once a step (lora_plan_kernel: a stable counting sort, then tiles of up to `rows` tokens of one
// adapter).  Two launches apply the adapters, both bound by what they read and write:
//   lora_shrink_kernel  parts of h in fp32: a CTA per (tile, 64 of the joined ranks, part of K)
//   lora_expand_kernel  h as the sum of its parts, then z: a CTA per (tile, 256 columns of y)
// so that many small pieces of work even out adapters of unlike ranks.  The second is launched while the first runs and
// has y and its first factors in registers by the time h is there.

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../common/device_once.h"
#include "../common/pdl.cuh"
#include "../common/ptx.cuh"
#include "../gemm/gated_act.cuh"

namespace b200 {

static constexpr int kLoraThreads = 256;
static constexpr int kLoraWarps = kLoraThreads / 32;
static constexpr int kLoraMaxSlices = 4;
static constexpr int kLoraChunk = 8;             // 8-wide tiles of h in a piece of work
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
  const int* ranks;                              // [L, slices]
  const float* scales;                           // [L]
  const int* order;
  const LoraTile* tiles;
  const int* num_tiles;
  float* h;                                      // [parts][T][h_width], rows in the order of the plan
  long long h_part;                              // T * h_width
  int h_width;                                   // slices * largest rank
  int K, slices, parts;
  int subs_shrink, subs;                         // pieces of a plan's tile, each with CTAs of its own
  int per;                                       // column groups of a CTA of the second kernel
  int chunk;                                     // ranks in a stage of its ring
  int n[kLoraMaxSlices];
  int h_pitch;                                   // elements between rows of h in shared memory
  float act_alpha, act_limit;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float lo_f(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float hi_f(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
// The tile of a CTA, or false when there is none.  (Entries behind the last tile lie in the buffer.)
__device__ __forceinline__ bool lora_tile(const LoraParams& p, int item, int subs, int rows, LoraTile& tl) {
  const int tile = item / subs, sub = item % subs;
  const int4 v = *reinterpret_cast<const int4*>(p.tiles + tile);
  if (tile >= *p.num_tiles) return false;
  tl = LoraTile{v.x, v.y + sub * rows, min(rows, v.z - sub * rows), 0};
  return tl.count > 0;
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// ---- h of few rows: 16 at most, K dealt to the parts and within one to the warps.  The factors are what is read: every warp has a
// ring of its own in shared memory (no barrier between copy and product), with some 4 KB of A a stage however many ranks there
// are: 128 of K for 16 of them, 64 for 32, 32 for 48 or 64.  Rows lie 16 bytes past their length apart, so that eight of them
// are in banks of their own.
static constexpr int kFewThreads = 128, kFewWarps = kFewThreads / 32, kFewStages = 3, kFewStageBytes = 2 * 16 * 272;

template <int NT>
__device__ __forceinline__ void shrink_rows(const LoraParams& p, const LoraTile& tl, const int* tok, int n0, int k_lo, int k_hi,
                                            uint32_t ring, float* d) {
  constexpr int KT = NT == 2 ? 128 : NT == 4 ? 64 : 32, PIECES = KT / 8, PITCH = KT * 2 + 16;
  constexpr int X_AT = NT * 8 * PITCH;
  static_assert(X_AT + 16 * PITCH <= kFewStageBytes, "stage");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const __nv_bfloat16* a = p.a + tl.slot * p.a_slot + static_cast<long long>(n0) * p.K;
  auto copy = [&](int i) {
    const int k0 = k_lo + (i * kFewWarps + warp) * KT;
    if (k0 < k_hi) {
      const uint32_t st = ring + i % kFewStages * kFewStageBytes;
#pragma unroll
      for (int u = 0; u < NT * 8 * PIECES / 32; ++u) {
        const int row = (lane + 32 * u) / PIECES, k = k0 + (lane + 32 * u) % PIECES * 8;
        cp16(st + row * PITCH + (k - k0) * 2, a + static_cast<long long>(row) * p.K + (k < k_hi ? k : 0), k < k_hi);
      }
#pragma unroll
      for (int u = 0; u < 16 * PIECES / 32; ++u) {
        const int row = (lane + 32 * u) / PIECES, k = k0 + (lane + 32 * u) % PIECES * 8;
        if (row < tl.count)                                            // (the other rows of h are not used)
          cp16(st + X_AT + row * PITCH + (k - k0) * 2, p.x + tok[row] * p.x_stride + (k < k_hi ? k : 0), k < k_hi);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kFewStages - 1; ++i) copy(i);
  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
  const uint32_t xf = X_AT + (lane & 15) * PITCH + (lane >> 4) * 16;
  const uint32_t af = ((lane & 7) + (lane >> 4) * 8) * PITCH + (lane >> 3 & 1) * 16;
  for (int i = 0; k_lo + (i * kFewWarps + warp) * KT < k_hi; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kFewStages - 2) : "memory");
    __syncwarp();
    copy(i + kFewStages - 1);
    const uint32_t st = ring + i % kFewStages * kFewStageBytes;
#pragma unroll
    for (int k = 0; k < KT; k += 16) {
      uint32_t x[4];
      ldmatrix4(x, st + xf + k * 2);
#pragma unroll
      for (int j = 0; j < NT; j += 2) {
        uint32_t b[4];
        ldmatrix4(b, st + af + j * 8 * PITCH + k * 2);
        mma_bf16(acc[j], x[0], x[1], x[2], x[3], b[0], b[1]);
        mma_bf16(acc[j + 1], x[0], x[1], x[2], x[3], b[2], b[3]);
      }
    }
    __syncwarp();
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    *reinterpret_cast<float2*>(d + j * 8) = make_float2(acc[j][0], acc[j][1]);
    *reinterpret_cast<float2*>(d + 8 * kLoraChunk * 8 + j * 8) = make_float2(acc[j][2], acc[j][3]);
  }
}

__global__ void __launch_bounds__(kFewThreads) lora_shrink_few_kernel(const LoraParams p) {
  constexpr int BM = 16, W = kLoraChunk * 8;
  extern __shared__ __align__(128) char smem[];
  __shared__ int tok[BM];
  pdl_wait();
  pdl_trigger();                                                       // (the second kernel reads what was there before this one)
  LoraTile tl;
  if (!lora_tile(p, blockIdx.z, p.subs_shrink, BM, tl) || tl.slot < 0) return;
  int sum_r = 0;
  for (int s = 0; s < p.slices; ++s) sum_r += p.ranks[tl.slot * p.slices + s];
  const int n0 = blockIdx.y * W;
  if (n0 >= sum_r) return;
  if (threadIdx.x < tl.count) tok[threadIdx.x] = p.order[tl.start + threadIdx.x];
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int nt = min(kLoraChunk, (sum_r - n0) / 8);                    // even: ranks are multiples of 16
  const int steps = (p.K + 31) / 32;
  const int k_lo = static_cast<int>(static_cast<long long>(steps) * blockIdx.x / p.parts) * 32;
  const int k_hi = min(p.K, static_cast<int>(static_cast<long long>(steps) * (blockIdx.x + 1) / p.parts) * 32);
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * kFewStages * kFewStageBytes;
  // (a warp's part of h goes where its ring was)
  const auto red = [&](int w) { return reinterpret_cast<float*>(smem + w * kFewStages * kFewStageBytes); };
  float* d = red(warp) + g * W + t4 * 2;
  if (nt == 2) shrink_rows<2>(p, tl, tok, n0, k_lo, k_hi, ring, d);
  else if (nt == 4) shrink_rows<4>(p, tl, tok, n0, k_lo, k_hi, ring, d);
  else if (nt == 6) shrink_rows<6>(p, tl, tok, n0, k_lo, k_hi, ring, d);
  else shrink_rows<8>(p, tl, tok, n0, k_lo, k_hi, ring, d);
  __syncthreads();
  // the warps' parts in order, four columns a thread
  float* h = p.h + blockIdx.x * p.h_part + static_cast<long long>(tl.start) * p.h_width + n0;
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

// ---- h of many rows: 64 rows of x and 64 of the joined ranks, in slabs of 64 of K through a ring in shared memory, so that
// what is in flight does not depend on registers.  Warps: two halves of every slab's K, then 32 rows x 32 ranks each (a fragment
// of x and one of A serve two and two pairs of matrix instructions).
static constexpr int kSlab = 64, kStages = 5, kStageBytes = 2 * 64 * kSlab * 2;

__global__ void __launch_bounds__(kLoraThreads, 2) lora_shrink_many_kernel(const LoraParams p) {
  constexpr int BM = 64, W = kLoraChunk * 8;
  extern __shared__ __align__(128) char smem[];
  pdl_wait();
  pdl_trigger();
  LoraTile tl;
  if (!lora_tile(p, blockIdx.z, p.subs_shrink, BM, tl) || tl.slot < 0) return;
  int sum_r = 0;
  for (int s = 0; s < p.slices; ++s) sum_r += p.ranks[tl.slot * p.slices + s];
  const int n0 = blockIdx.y * W;
  if (n0 >= sum_r) return;
  const int width = min(W, sum_r - n0);                                // a multiple of 16
  const int slabs = (p.K + kSlab - 1) / kSlab;
  const int s_lo = static_cast<int>(static_cast<long long>(slabs) * blockIdx.x / p.parts);
  const int s_hi = static_cast<int>(static_cast<long long>(slabs) * (blockIdx.x + 1) / p.parts);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // copies: eight lanes a row of 128 bytes, its 16-byte pieces at (piece ^ row % 8); two rows of x and of A each
  const int crow = threadIdx.x >> 3, piece = threadIdx.x & 7;
  const __nv_bfloat16 *xs[2], *as[2];
  bool xok[2], aok[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = crow + 32 * i;
    xok[i] = row < tl.count;
    aok[i] = row < width;
    xs[i] = p.x + (xok[i] ? p.order[tl.start + row] : 0) * p.x_stride + piece * 8;
    as[i] = p.a + tl.slot * p.a_slot + static_cast<long long>(n0 + (aok[i] ? row : 0)) * p.K + piece * 8;
  }
  const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  const uint32_t cdst = base + crow * 128 + ((piece ^ (crow & 7)) << 4);
  auto copy = [&](int s) {
    if (s < s_hi) {
      const uint32_t dst = cdst + (s - s_lo) % kStages * kStageBytes;
      const bool in = s * kSlab + piece * 8 < p.K;                     // K is a multiple of 8
      const int k = in ? s * kSlab : -piece * 8;                       // (nothing is read there)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        cp16(dst + i * 4096, xs[i] + k, in && xok[i]);
        cp16(dst + 8192 + i * 4096, as[i] + k, in && aok[i]);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int i = 0; i < kStages - 1; ++i) copy(s_lo + i);

  const int kw = warp >> 2, m0 = (warp & 1) * 32, j0 = (warp >> 1 & 1) * 32;
  const bool live = j0 < width && m0 < tl.count;
  float acc[2][4][4];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[m][j][e] = 0.f;
  // rows of the four 8 x 8 matrices of a fragment: x rows 0-7, 8-15 at k, then at k + 8; A ranks 0-7 at k, k + 8, then 8-15
  const int xr = m0 + (lane & 15), xk = lane >> 4;
  const int arow = j0 + (lane & 7) + (lane >> 4) * 8, ak = lane >> 3 & 1;
  for (int s = s_lo; s < s_hi; ++s) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncthreads();
    copy(s + kStages - 1);
    if (!live) continue;
    const uint32_t st = base + (s - s_lo) % kStages * kStageBytes;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int kc = (kw * 2 + q) * 2;                                 // its first 16-byte piece
      uint32_t xf[2][4], af[2][4];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const int row = xr + m * 16;
        ldmatrix4(xf[m], st + row * 128 + (((kc + xk) ^ (row & 7)) << 4));
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = arow + j * 16;
        ldmatrix4(af[j], st + 8192 + row * 128 + (((kc + ak) ^ (row & 7)) << 4));
      }
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          mma_bf16(acc[m][j], xf[m][0], xf[m][1], xf[m][2], xf[m][3], af[j >> 1][(j & 1) * 2], af[j >> 1][(j & 1) * 2 + 1]);
    }
  }
  // the two halves of K in order
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);                         // [4 warps][32][32]
  const int g = lane >> 2, t4 = lane & 3;
  float* mine = red + (warp & 3) * 32 * 36;
  if (kw == 1 && live) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        *reinterpret_cast<float2*>(mine + (m * 16 + g) * 36 + j * 8 + t4 * 2) = make_float2(acc[m][j][0], acc[m][j][1]);
        *reinterpret_cast<float2*>(mine + (m * 16 + g + 8) * 36 + j * 8 + t4 * 2) = make_float2(acc[m][j][2], acc[m][j][3]);
      }
  }
  __syncthreads();
  if (kw == 0 && live) {
    float* h = p.h + blockIdx.x * p.h_part + static_cast<long long>(tl.start) * p.h_width + n0;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = m * 16 + g + e * 8, col = j0 + j * 8 + t4 * 2;
          const float2 o = *reinterpret_cast<const float2*>(mine + r * 36 + j * 8 + t4 * 2);
          if (m0 + r < tl.count && col < width)
            *reinterpret_cast<float2*>(h + static_cast<long long>(m0 + r) * p.h_width + col) =
                make_float2(acc[m][j][2 * e] + o.x, acc[m][j][2 * e + 1] + o.y);
        }
  }
}

// ---- z: a CTA has a tile's rows and a run of column groups of one slice, 64 columns of y each (gated: 32 of gate and their 32 of
// up).  A team of RW warps, 16 rows each, takes a group; y and B come through a ring in shared memory (many rows: one team of
// four, so that a group's B is read once for 64 rows; few rows: four teams of a warp).  Columns of B are dealt to the matrix
// instructions so that a lane ends up with eight neighbouring columns twice: y and the result move 16 bytes a lane, 128 of a
// row at once.
static constexpr int kExpandThreads = 128, kExpandStages = 3;

template <int RW, int ACT>
__global__ void __launch_bounds__(kExpandThreads, 4) lora_expand_kernel(const LoraParams p) {
  constexpr int BM = 16 * RW, TEAMS = kExpandThreads / 32 / RW, TEAM = 32 * RW;
  constexpr bool GATED = ACT != kActNone;
  extern __shared__ __align__(128) char smem[];
  __shared__ int tok[BM];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int team = warp / RW, member = threadIdx.x % TEAM, rows0 = warp % RW * 16;
  const bool in_place = !GATED && p.out == p.y;
  // Everything but h is older than the first kernel, which has started only behind it: no wait yet.
  LoraTile tl;
  if (!lora_tile(p, blockIdx.y, p.subs, BM, tl)) {
    pdl_wait();
    return;
  }
  // this CTA's slice and groups in it; of the slice: first rank in h, first column of y, factors
  int slice = 0, block = blockIdx.x, h0 = 0, first = 0, r0 = 0, r1 = 0;
  const __nv_bfloat16* b = p.b + (tl.slot >= 0 ? tl.slot * p.b_slot : 0);
  const int* ranks = p.ranks + max(tl.slot, 0) * p.slices;
  if constexpr (GATED) {
    r0 = tl.slot >= 0 ? ranks[0] : 0;
    r1 = tl.slot >= 0 ? ranks[1] : 0;
  } else {
    for (;; ++slice) {
      r0 = tl.slot >= 0 ? ranks[slice] : 0;
      const int blocks = ((p.n[slice] + 63) / 64 + p.per - 1) / p.per;
      if (block < blocks) break;
      block -= blocks;
      h0 += r0;
      first += p.n[slice];
      b += static_cast<long long>(p.n[slice]) * r0;
    }
    r1 = r0;
  }
  const int rank = max(r0, r1), N = p.n[slice];
  if (rank == 0 && in_place) {
    pdl_wait();
    return;
  }
  constexpr int GW = GATED ? 32 : 64;                                  // columns of a slice in a group
  const int ga = block * p.per + team, gb = min((N + GW - 1) / GW, (block + 1) * p.per);
  const float scale = tl.slot >= 0 ? p.scales[tl.slot] : 0.f;
  if (threadIdx.x < BM) tok[threadIdx.x] = threadIdx.x < tl.count ? p.order[tl.start + threadIdx.x] : -1;
  __syncthreads();

  const int b_pitch = p.chunk * 2 + 16;                                // bytes; eight rows are in banks of their own
  const int stage_bytes = 64 * b_pitch + RW * 2048;
  const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  const uint32_t ring = base + team * kExpandStages * stage_bytes;
  const uint32_t h_at = base + TEAMS * kExpandStages * stage_bytes;
  __nv_bfloat16* h_hi = reinterpret_cast<__nv_bfloat16*>(smem + TEAMS * kExpandStages * stage_bytes);   // [BM][h_pitch]
  __nv_bfloat16* h_lo = h_hi + BM * p.h_pitch;
  const uint32_t y_slot = 64 * b_pitch + (warp % RW * 128 + lane) * 16;
  const int tok0 = tok[rows0 + g], tok1 = tok[rows0 + g + 8];
  const int chunks = max(1, (rank + p.chunk - 1) / p.chunk);
  // the ring's next item: chunk of ranks cc of group cg
  int cg = ga, cc = 0, cs = 0;
  auto copy = [&]() {
    if (cg < gb) {
      const uint32_t st = ring + cs * stage_bytes;
      const int c0 = cg * GW;
#pragma unroll
      for (int s = 0; s < (GATED ? 2 : 1); ++s) {
        const int rs = s ? r1 : r0, kc = min(p.chunk, rs - cc * p.chunk), pieces = kc >> 3;
        if (kc <= 0) continue;
        const __nv_bfloat16* src = b + (s ? static_cast<long long>(N) * r0 : 0) + static_cast<long long>(c0) * rs + cc * p.chunk;
        const uint32_t inv = 65536u / pieces + 1;                      // i / pieces for i < 512
        for (int i = member; i < GW * pieces; i += TEAM) {
          const int col = (i * inv) >> 16, piece = i - col * pieces, c = col & 31;
          const int row = s * 32 + (col & 32) + ((c & 7) >> 1) * 8 + (c >> 3) * 2 + (c & 1);
          if (c0 + col < N) cp16(st + row * b_pitch + piece * 16, src + col * rs + piece * 8, true);
        }
      }
      if (cc == 0) {
        const int col = c0 + t4 * 8;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int t = i ? tok1 : tok0;
          const __nv_bfloat16* row = p.y + t * p.y_stride + first + (GATED ? 2 : 1) * col;
          if (t >= 0 && col < N) cp16(st + y_slot + i * 1024, row, true);
          if (t >= 0 && col + (GATED ? 0 : 32) < N) cp16(st + y_slot + i * 1024 + 512, row + (GATED ? 8 : 32), true);
        }
      }
      if (++cc == chunks) {
        cc = 0;
        cg += TEAMS;
      }
      cs = cs + 1 == kExpandStages ? 0 : cs + 1;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kExpandStages - 1; ++i) copy();
  pdl_wait();
  pdl_trigger();

  // h: the parts in order, times the scale, as the sum of two bf16 (17 bits of the fp32 value), so that the product below adds
  // no rounding beside that of its result
  const int sum_r = GATED ? r0 + r1 : r0;
  if (sum_r > 0) {
    const float* h = p.h + static_cast<long long>(tl.start) * p.h_width + h0;
    const int vecs = sum_r / 4;
    for (int i = threadIdx.x; i < BM * vecs; i += kExpandThreads) {
      const int row = i / vecs, v = i % vecs * 4;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < tl.count) {
        const float* src = h + static_cast<long long>(row) * p.h_width + v;
#pragma unroll 4
        for (int c = 0; c < p.parts; ++c) {
          const float4 q = *reinterpret_cast<const float4*>(src + c * p.h_part);
          sum.x += q.x, sum.y += q.y, sum.z += q.z, sum.w += q.w;
        }
      }
      const float f[4] = {sum.x * scale, sum.y * scale, sum.z * scale, sum.w * scale};
      float up[4], rest[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        up[e] = __bfloat162float(__float2bfloat16(f[e]));
        rest[e] = f[e] - up[e];
        if (!(rest[e] - rest[e] == 0.f)) rest[e] = 0.f;                // beside an infinity
      }
      *reinterpret_cast<uint2*>(h_hi + row * p.h_pitch + v) = make_uint2(pack_bf16x2(up[0], up[1]), pack_bf16x2(up[2], up[3]));
      *reinterpret_cast<uint2*>(h_lo + row * p.h_pitch + v) = make_uint2(pack_bf16x2(rest[0], rest[1]), pack_bf16x2(rest[2], rest[3]));
    }
  }
  __syncthreads();
  const uint32_t hf = h_at + ((rows0 + (lane & 15)) * p.h_pitch + (lane >> 4) * 8) * 2, lo_at = 2 * BM * p.h_pitch;
  const uint32_t bf = ((lane & 7) + (lane >> 4) * 8) * b_pitch + (lane >> 3 & 1) * 16;
  const bool live = rows0 < tl.count;
  __nv_bfloat16* out0 = p.out + tok0 * p.out_stride + first + t4 * 8;
  __nv_bfloat16* out1 = p.out + tok1 * p.out_stride + first + t4 * 8;
  int rs = 0;                                                          // the ring's stage that is read
  for (int gi = ga; gi < gb; gi += TEAMS) {
    float acc[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
    uint4 yv[4];
    for (int c = 0; c < chunks; ++c) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kExpandStages - 2) : "memory");
      if constexpr (RW > 1) __syncthreads();
      else __syncwarp();
      copy();
      const uint32_t st = ring + rs * stage_bytes;
      rs = rs + 1 == kExpandStages ? 0 : rs + 1;
      if (!live) continue;
      if (c == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(yv[i].x), "=r"(yv[i].y), "=r"(yv[i].z), "=r"(yv[i].w)
                       : "r"(st + y_slot + i * 512)
                       : "memory");
      }
      const int k0 = c * p.chunk;
      for (int k = 0; k < min(p.chunk, rank - k0); k += 16) {
#pragma unroll
        for (int s = 0; s < (GATED ? 2 : 1); ++s) {
          if (GATED && k0 + k >= (s ? r1 : r0)) continue;
          uint32_t hi[4], lo[4];
          const uint32_t at = hf + (k0 + k + (s ? r0 : 0)) * 2;
          ldmatrix4(hi, at);
          ldmatrix4(lo, at + lo_at);
#pragma unroll
          for (int j = 0; j < (GATED ? 4 : 8); j += 2) {
            uint32_t v[4];
            const int o = 4 * s + j;
            ldmatrix4(v, st + bf + o * 8 * b_pitch + k * 2);
            mma_bf16(acc[o], hi[0], hi[1], hi[2], hi[3], v[0], v[1]);
            mma_bf16(acc[o + 1], hi[0], hi[1], hi[2], hi[3], v[2], v[3]);
            mma_bf16(acc[o], lo[0], lo[1], lo[2], lo[3], v[0], v[1]);
            mma_bf16(acc[o + 1], lo[0], lo[1], lo[2], lo[3], v[2], v[3]);
          }
        }
      }
    }
    if (!live) continue;
    const int c0 = gi * GW, left = N - c0 - t4 * 8;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int e = 2 * i;
      const uint32_t w0[4] = {yv[2 * i].x, yv[2 * i].y, yv[2 * i].z, yv[2 * i].w};
      const uint32_t w1[4] = {yv[2 * i + 1].x, yv[2 * i + 1].y, yv[2 * i + 1].z, yv[2 * i + 1].w};
      uint32_t o0[4], o1[4];
      if constexpr (GATED) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o0[j] = pack_bf16x2(gated_act(ACT, lo_f(w0[j]) + acc[j][e], lo_f(w1[j]) + acc[4 + j][e], p.act_alpha, p.act_limit),
                              gated_act(ACT, hi_f(w0[j]) + acc[j][e + 1], hi_f(w1[j]) + acc[4 + j][e + 1], p.act_alpha,
                                        p.act_limit));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          o0[j] = pack_bf16x2(lo_f(w0[j]) + acc[j][e], hi_f(w0[j]) + acc[j][e + 1]);
          o1[j] = pack_bf16x2(lo_f(w1[j]) + acc[4 + j][e], hi_f(w1[j]) + acc[4 + j][e + 1]);
        }
      }
      __nv_bfloat16* row = (i ? out1 : out0) + c0;
      const bool ok = (i ? tok1 : tok0) >= 0;
      if (ok && left > 0) *reinterpret_cast<uint4*>(row) = make_uint4(o0[0], o0[1], o0[2], o0[3]);
      if (!GATED && ok && left > 32) *reinterpret_cast<uint4*>(row + 32) = make_uint4(o1[0], o1[1], o1[2], o1[3]);
    }
  }
}

static constexpr int kShrinkFewSmem = kFewWarps * kFewStages * kFewStageBytes, kShrinkSmem = kStages * kStageBytes,
                     kExpandSmem = 200 * 1024;

template <int ACT>
static int launch_lora(const LoraParams& p, bool many, unsigned tiles, unsigned chunks, unsigned blocks, cudaStream_t stream) {
  auto expand = many ? lora_expand_kernel<4, ACT> : lora_expand_kernel<1, ACT>;
  static DeviceOnce once;
  int dev;
  if (once.needed(&dev)) {
    const auto attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
    if (cudaFuncSetAttribute(lora_shrink_few_kernel, attr, kShrinkFewSmem) != cudaSuccess ||
        cudaFuncSetAttribute(lora_shrink_many_kernel, attr, kShrinkSmem) != cudaSuccess ||
        cudaFuncSetAttribute(lora_expand_kernel<4, ACT>, attr, kExpandSmem) != cudaSuccess ||
        cudaFuncSetAttribute(lora_expand_kernel<1, ACT>, attr, kExpandSmem) != cudaSuccess)
      return -3;
    once.mark(dev);
  }
  const int rw = many ? 4 : 1;
  const size_t smem = static_cast<size_t>(4 / rw) * kExpandStages * (64 * (p.chunk * 2 + 16) + rw * 2048) +
                      2 * sizeof(__nv_bfloat16) * rw * 16 * p.h_pitch;
  if (smem > kExpandSmem) return -2;
  const dim3 grid(p.parts, chunks, tiles * p.subs_shrink);
  if (grid.z > 65535 || tiles * p.subs > 65535) return -1;
  const cudaError_t e =
      many ? launch_pdl(lora_shrink_many_kernel, grid, dim3(kLoraThreads), kShrinkSmem, stream, 1, p)
           : launch_pdl(lora_shrink_few_kernel, grid, dim3(kFewThreads), kShrinkFewSmem, stream, 1, p);
  if (e != cudaSuccess) return -3;
  return launch_pdl(expand, dim3(blocks, tiles * p.subs), dim3(kExpandThreads), smem, stream, 1, p) == cudaSuccess ? 0 : -3;
}

}  // namespace b200

// Parts of K that a step's h is summed from.  Few rows (tiles of 16): as many as the slots let be resident, whatever the number of
// tokens, so that a row does not depend on it; many rows: as many as fill the SMs.
extern "C" int b200_lora_parts(int K, int rows, int max_tiles, int num_slots) {
  const int want = rows < 64 ? std::min((K + 511) / 512, 592 / num_slots) : std::min((K + 255) / 256, 296 / max_tiles);
  return std::min(std::max(want, 1), 16);
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

// n: columns of each slice.  h: fp32 [b200_lora_parts][T][slices * max_rank].  max_tiles: tiles that the plan may have, of `rows`
// tokens each.  max_rank: bound of the ranks.  act: 0 adds, a gated kind of gemm/gated_act.cuh joins gate and up (alternating
// groups of eight columns of y).
extern "C" int b200_lora(const void* x, long long x_stride, const void* y, long long y_stride, void* out, long long out_stride,
                         const void* a, long long a_slot, const void* b, long long b_slot, const int* ranks,
                         const float* scales, const int* order, const int* tiles, const int* num_tiles, int max_tiles, int rows,
                         float* h, int T, int num_slots, int K, int slices, const int* n, int max_rank, int act,
                         float act_alpha, float act_limit, cudaStream_t stream) {
  using namespace b200;
  if (slices < 1 || slices > kLoraMaxSlices || (K & 7) || max_rank < 16 || (max_rank & 15) || max_tiles < 1 || (rows & 15)) return -1;
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
  p.scales = scales;
  p.order = order;
  p.tiles = reinterpret_cast<const LoraTile*>(tiles);
  p.num_tiles = num_tiles;
  p.h = h;
  p.h_width = slices * max_rank;
  p.h_part = static_cast<long long>(T) * p.h_width;
  p.K = K;
  p.slices = slices;
  const bool many = rows >= 64, gated = act != kActNone;
  p.act_alpha = act_alpha;
  p.act_limit = act_limit;
  p.subs_shrink = p.subs = many ? rows / 64 : rows / 16;
  p.parts = b200_lora_parts(K, rows, max_tiles, num_slots);
  p.chunk = std::min(max_rank, many ? 64 : 32);
  p.h_pitch = (gated ? 2 : 1) * max_rank + 8;    // eight rows of 16 bytes are in banks of their own
  const unsigned chunks = (p.h_width + kLoraChunk * 8 - 1) / (kLoraChunk * 8), tiles_n = static_cast<unsigned>(max_tiles);
  // column groups of a CTA: a few rounds of the resident CTAs in all, a group a team at least
  int groups = 0;
  for (int s = 0; s < kLoraMaxSlices; ++s) {
    p.n[s] = s < slices ? n[s] : 0;
    if (p.n[s] & 7) return -1;
    if (!gated || s == 0) groups += gated ? (p.n[s] + 31) / 32 : (p.n[s] + 63) / 64;
  }
  const int team = many ? 1 : 4;
  const long long want = static_cast<long long>(groups) * max_tiles * p.subs / (148 * 8);
  p.per = static_cast<int>(std::max(1LL, (want + team - 1) / team)) * team;
  unsigned blocks = 0;
  for (int s = 0; s < slices; ++s)
    if (!gated || s == 0) blocks += ((gated ? (n[s] + 31) / 32 : (n[s] + 63) / 64) + p.per - 1) / p.per;
  switch (act) {
    case kActNone: return launch_lora<kActNone>(p, many, tiles_n, chunks, blocks, stream);
    case kActSilu: return launch_lora<kActSilu>(p, many, tiles_n, chunks, blocks, stream);
    case kActClampedGlu: return launch_lora<kActClampedGlu>(p, many, tiles_n, chunks, blocks, stream);
    case kActGeluTanh: return launch_lora<kActGeluTanh>(p, many, tiles_n, chunks, blocks, stream);
    default: return launch_lora<kActReluGate>(p, many, tiles_n, chunks, blocks, stream);
  }
}
