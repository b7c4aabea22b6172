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
// adapter).  A cluster takes a tile: its CTAs share out K for h, sum their parts over distributed shared memory in rank order,
// and share out the columns for z, so that x, y, A and B are read once per tile, in one launch, and h never leaves the SMs.

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../common/device_once.h"
#include "../common/pdl.cuh"
#include "../common/ptx.cuh"
#include "../gemm/gated_act.cuh"

namespace b200 {

static constexpr int kLoraThreads = 256;
static constexpr int kLoraWarps = kLoraThreads / 32;
static constexpr int kLoraMaxSlices = 4;
static constexpr int kLoraChunk = 8;             // 8-wide tiles of h that are summed at a time
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
  int K, slices, subs;                           // subs: parts of a plan's tile, each for a cluster of its own
  int n[kLoraMaxSlices];
  int h_pitch;                                   // elements between rows of h in shared memory
  int act;
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
__device__ __forceinline__ uint4 load16(const void* p, bool ok) {
  return ok ? *static_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ uint2 load8(const void* p, bool ok) {
  return ok ? *static_cast<const uint2*>(p) : make_uint2(0, 0);
}

// MT 16-row tiles a warp, MW warps side by side on rows in the first product: 16 * MT * MW rows a cluster.  The second
// product gives every warp all rows and its own columns.  In the first, a lane's 16 bytes of a row of x and of A stand for
// the k of two matrix instructions: both operands use the same permutation of k, which the sum does not see.
template <int MT, int MW, bool GATED>
__global__ void __launch_bounds__(kLoraThreads) lora_kernel(const LoraParams p) {
  constexpr int BM = 16 * MT * MW, KW = kLoraWarps / MW, NT = kLoraChunk, M2 = MT * MW;
  extern __shared__ __align__(16) char smem[];
  float* red = reinterpret_cast<float*>(smem);                         // [KW][BM][NT * 8] parts of the warps
  float* part = red + KW * BM * NT * 8;                                // [2][BM][NT * 8] of this CTA
  __nv_bfloat16* h_hi = reinterpret_cast<__nv_bfloat16*>(part + 2 * BM * NT * 8);
  __nv_bfloat16* h_lo = h_hi + BM * p.h_pitch;
  __shared__ int tok[BM];

  pdl_trigger();
  pdl_wait();
  uint32_t C;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(C));
  const int rank = static_cast<int>(cluster_ctarank());
  const int item = blockIdx.x / C;
  const int tile = item / p.subs;
  if (tile >= *p.num_tiles) return;                                    // the whole cluster alike
  LoraTile tl = p.tiles[tile];
  tl.start += (item % p.subs) * BM;
  tl.count = min(BM, tl.count - (item % p.subs) * BM);
  if (tl.count <= 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  int r[kLoraMaxSlices], sum_r = 0;
#pragma unroll
  for (int s = 0; s < kLoraMaxSlices; ++s) {
    r[s] = tl.slot >= 0 && s < p.slices ? p.ranks[tl.slot * p.slices + s] : 0;
    sum_r += r[s];
  }
  const bool in_place = !GATED && p.out == p.y;
  if (sum_r == 0 && in_place) return;
  if (threadIdx.x < BM) tok[threadIdx.x] = threadIdx.x < tl.count ? p.order[tl.start + threadIdx.x] : -1;
  __syncthreads();

  // ---- h: this CTA's part of K, in chunks of 64 of the joined ranks
  if (sum_r > 0) {
    const int steps = (p.K + 31) / 32;
    const int s_lo = static_cast<int>(static_cast<long long>(steps) * rank / C);
    const int s_hi = static_cast<int>(static_cast<long long>(steps) * (rank + 1) / C);
    const int mw = warp % MW, kw = warp / MW;
    const __nv_bfloat16* xr[2 * MT];
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
      const int t = tok[mw * 16 * MT + i * 8 + g];
      xr[i] = t >= 0 ? p.x + t * p.x_stride : nullptr;
    }
    const __nv_bfloat16* a = p.a + tl.slot * p.a_slot;
    const float scale = p.scales[tl.slot];
    int buf = 0;
    for (int n0 = 0; n0 < sum_r; n0 += NT * 8, buf ^= 1) {
      const int nt = min(NT, (sum_r - n0) / 8), width = nt * 8;
      float acc[MT][NT][4];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[m][j][e] = 0.f;
      const __nv_bfloat16* ar = a + static_cast<long long>(n0 + g) * p.K;
#pragma unroll 2
      for (int s = s_lo + kw; s < s_hi; s += KW) {
        const int k = s * 32 + t4 * 8;
        const bool in = k < p.K;                                       // K is a multiple of 8
        uint4 xv[2 * MT];
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) xv[i] = load16(xr[i] + k, in && xr[i] != nullptr);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          if (j >= nt) break;
          const uint4 av = load16(ar + static_cast<long long>(j) * 8 * p.K + k, in);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            mma_bf16(acc[m][j], xv[2 * m].x, xv[2 * m + 1].x, xv[2 * m].y, xv[2 * m + 1].y, av.x, av.y);
            mma_bf16(acc[m][j], xv[2 * m].z, xv[2 * m + 1].z, xv[2 * m].w, xv[2 * m + 1].w, av.z, av.w);
          }
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          if (j >= nt) break;
          float* d = red + (kw * BM + (mw * MT + m) * 16 + g) * (NT * 8) + j * 8 + t4 * 2;
          *reinterpret_cast<float2*>(d) = make_float2(acc[m][j][0], acc[m][j][1]);
          *reinterpret_cast<float2*>(d + 8 * NT * 8) = make_float2(acc[m][j][2], acc[m][j][3]);
        }
      __syncthreads();
      float* pt = part + buf * BM * NT * 8;
      for (int i = threadIdx.x; i < BM * width; i += kLoraThreads) {
        const int row = i / width, col = i % width;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < KW; ++w) sum += red[(w * BM + row) * (NT * 8) + col];
        pt[row * (NT * 8) + col] = sum;
      }
      cluster_arrive_release();
      cluster_wait_acquire();
      // the parts of all CTAs in rank order; h as the sum of two bf16 (17 bits of the fp32 sum), so that the second
      // product adds no rounding beside that of its result
      const uint32_t base = smem_u32(pt);
      for (int i = threadIdx.x; i < BM * width; i += kLoraThreads) {
        const int row = i / width, col = i % width;
        float sum = 0.f;
        for (uint32_t c = 0; c < C; ++c) {
          float v;
          asm volatile("ld.shared::cluster.f32 %0, [%1];"
                       : "=f"(v)
                       : "r"(mapa_shared(base + (row * (NT * 8) + col) * 4, c))
                       : "memory");
          sum += v;
        }
        sum *= scale;
        const __nv_bfloat16 hi = __float2bfloat16(sum);
        h_hi[row * p.h_pitch + n0 + col] = hi;
        const float rest = sum - __bfloat162float(hi);
        h_lo[row * p.h_pitch + n0 + col] = __float2bfloat16(rest - rest == 0.f ? rest : 0.f);      // (0 beside an infinity)
      }
      // (the buffer is written again two chunks on, behind the next chunk's barrier)
    }
    cluster_arrive_release();                                          // waited for before this CTA's memory goes
    __syncthreads();
  }

  // ---- z: groups of 32 columns of y, each to one warp for all rows
  int groups = 0;
  if constexpr (GATED) {
    groups = p.n[0] / 16 + (p.n[0] % 16 != 0);
  } else {
    for (int s = 0; s < p.slices; ++s) groups += (p.n[s] + 31) / 32;
  }
  const __nv_bfloat16* b0 = p.b + (tl.slot >= 0 ? tl.slot * p.b_slot : 0);
  for (int gi = rank * kLoraWarps + warp; gi < groups; gi += C * kLoraWarps) {
    float acc[M2][4][4];
#pragma unroll
    for (int m = 0; m < M2; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[m][j][e] = 0.f;
    if constexpr (!GATED) {
      int s = 0, c0 = gi, h0 = 0, first = 0;                           // slice, its group, first rank and first column
      long long off = 0;
      while (s + 1 < p.slices && c0 >= (p.n[s] + 31) / 32) {
        c0 -= (p.n[s] + 31) / 32;
        h0 += r[s];
        off += static_cast<long long>(p.n[s]) * r[s];
        first += p.n[s];
        ++s;
      }
      const int rs = r[s], N = p.n[s];
      if (rs == 0 && in_place) continue;
      c0 *= 32;
      const int col = c0 + t4 * 8;
      uint4 yv[2 * M2];
#pragma unroll
      for (int i = 0; i < 2 * M2; ++i) {
        const int t = tok[i * 8 + g];
        yv[i] = load16(p.y + t * p.y_stride + first + col, t >= 0 && col < N);
      }
      // columns 8 t + 2 j + e of the group are column 2 t + e of matrix tile j: a lane ends up with eight neighbours
      const int bc = c0 + (g >> 1) * 8 + (g & 1);
      const __nv_bfloat16* br = b0 + off + static_cast<long long>(bc) * rs + t4 * 4;
      const bool bin = (c0 + (g >> 1) * 8) < N;
      for (int k = 0; k < rs; k += 16) {
        uint2 bv[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) bv[j] = load8(br + 2 * j * rs + k, bin);
#pragma unroll
        for (int m = 0; m < M2; ++m) {
          const int at = (m * 16 + g) * p.h_pitch + h0 + k + t4 * 4;
          const uint2 p0 = *reinterpret_cast<const uint2*>(h_hi + at), p1 = *reinterpret_cast<const uint2*>(h_hi + at + 8 * p.h_pitch);
          const uint2 q0 = *reinterpret_cast<const uint2*>(h_lo + at), q1 = *reinterpret_cast<const uint2*>(h_lo + at + 8 * p.h_pitch);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            mma_bf16(acc[m][j], p0.x, p1.x, p0.y, p1.y, bv[j].x, bv[j].y);
            mma_bf16(acc[m][j], q0.x, q1.x, q0.y, q1.y, bv[j].x, bv[j].y);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 2 * M2; ++i) {
        const int t = tok[i * 8 + g], m = i >> 1, e = (i & 1) * 2;
        if (t < 0 || col >= N) continue;
        const uint32_t w[4] = {yv[i].x, yv[i].y, yv[i].z, yv[i].w};
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = pack_bf16x2(lo_f(w[j]) + acc[m][j][e], hi_f(w[j]) + acc[m][j][e + 1]);
        *reinterpret_cast<uint4*>(p.out + t * p.out_stride + first + col) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    } else {
      // 16 columns of the result: matrix tiles 0, 1 are their gate columns 4 t + 2 j + e, tiles 2, 3 the up columns
      const int N = p.n[0], c0 = gi * 16, col = c0 + t4 * 4;
      const int phys = col / 8 * 16 + col % 8;
      uint2 gv[2 * M2], uv[2 * M2];
#pragma unroll
      for (int i = 0; i < 2 * M2; ++i) {
        const int t = tok[i * 8 + g];
        const __nv_bfloat16* yr = p.y + t * p.y_stride + phys;
        gv[i] = load8(yr, t >= 0 && col < N);
        uv[i] = load8(yr + 8, t >= 0 && col < N);
      }
      const int bc = c0 + (g >> 1) * 4 + (g & 1);
      const bool bin = bc < N;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int rs = r[s], h0 = s ? r[0] : 0;
        const __nv_bfloat16* br = b0 + (s ? static_cast<long long>(N) * r[0] : 0) + static_cast<long long>(bc) * rs + t4 * 4;
        for (int k = 0; k < rs; k += 16) {
          uint2 bv[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) bv[j] = load8(br + 2 * j * rs + k, bin);
#pragma unroll
          for (int m = 0; m < M2; ++m) {
            const int at = (m * 16 + g) * p.h_pitch + h0 + k + t4 * 4;
            const uint2 p0 = *reinterpret_cast<const uint2*>(h_hi + at), p1 = *reinterpret_cast<const uint2*>(h_hi + at + 8 * p.h_pitch);
            const uint2 q0 = *reinterpret_cast<const uint2*>(h_lo + at), q1 = *reinterpret_cast<const uint2*>(h_lo + at + 8 * p.h_pitch);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              mma_bf16(acc[m][2 * s + j], p0.x, p1.x, p0.y, p1.y, bv[j].x, bv[j].y);
              mma_bf16(acc[m][2 * s + j], q0.x, q1.x, q0.y, q1.y, bv[j].x, bv[j].y);
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 2 * M2; ++i) {
        const int t = tok[i * 8 + g], m = i >> 1, e = (i & 1) * 2;
        if (t < 0 || col >= N) continue;
        const uint32_t gw[2] = {gv[i].x, gv[i].y}, uw[2] = {uv[i].x, uv[i].y};
        uint32_t o[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
          o[j] = pack_bf16x2(gated_act(p.act, lo_f(gw[j]) + acc[m][j][e], lo_f(uw[j]) + acc[m][2 + j][e], p.act_alpha, p.act_limit),
                             gated_act(p.act, hi_f(gw[j]) + acc[m][j][e + 1], hi_f(uw[j]) + acc[m][2 + j][e + 1], p.act_alpha,
                                       p.act_limit));
        *reinterpret_cast<uint2*>(p.out + t * p.out_stride + col) = make_uint2(o[0], o[1]);
      }
    }
  }
  if (sum_r > 0) cluster_wait_acquire();
}

template <int MT, int MW, bool GATED>
static int launch_lora(const LoraParams& p, int clusters, int C, cudaStream_t stream) {
  constexpr int BM = 16 * MT * MW, KW = kLoraWarps / MW;
  const size_t smem = sizeof(float) * (KW + 2) * BM * kLoraChunk * 8 + 2 * sizeof(__nv_bfloat16) * BM * p.h_pitch;
  if (smem > 227 * 1024 - 1024) return -2;
  auto kern = lora_kernel<MT, MW, GATED>;
  static DeviceOnce once;
  int dev;
  if (once.needed(&dev)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024) != cudaSuccess) return -3;
    once.mark(dev);
  }
  return launch_pdl(kern, dim3(static_cast<unsigned>(clusters) * C), dim3(kLoraThreads), smem, stream, C, p) == cudaSuccess ? 0 : -3;
}

}  // namespace b200

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

// n: columns of each slice.  max_tiles: tiles that the plan may have, of `rows` tokens each.  max_rank: bound of the ranks.
// act: 0 adds, a gated kind of gemm/gated_act.cuh joins gate and up (alternating groups of eight columns of y).
extern "C" int b200_lora(const void* x, long long x_stride, const void* y, long long y_stride, void* out, long long out_stride,
                         const void* a, long long a_slot, const void* b, long long b_slot, const int* ranks,
                         const float* scales, const int* order, const int* tiles, const int* num_tiles, int max_tiles, int rows,
                         int K, int slices, const int* n, int max_rank, int act, float act_alpha, float act_limit,
                         cudaStream_t stream) {
  using namespace b200;
  if (slices < 1 || slices > kLoraMaxSlices || (K & 7) || max_rank < 16 || (max_rank & 15) || max_tiles < 1) return -1;
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
  p.K = K;
  p.slices = slices;
  for (int s = 0; s < kLoraMaxSlices; ++s) {
    p.n[s] = s < slices ? n[s] : 0;
    if (p.n[s] & 7) return -1;
  }
  p.act = act;
  p.act_alpha = act_alpha;
  p.act_limit = act_limit;
  // rows of h are 32 or 96 bytes past a multiple of 128 apart: the eight-byte reads of a half warp touch every bank once
  const int width = slices * max_rank;
  p.h_pitch = width + (width % 32 ? 0 : 16);
  const bool wide = rows >= 64 && p.h_pitch <= 400;
  p.subs = wide ? rows / 64 : (rows + 15) / 16;
  const long long clusters = static_cast<long long>(max_tiles) * p.subs;
  if (clusters > (1 << 24)) return -1;
  const int C = wide ? 4 : 8;
  const int cl = static_cast<int>(clusters);
  if (act != kActNone) return wide ? launch_lora<2, 2, true>(p, cl, C, stream) : launch_lora<1, 1, true>(p, cl, C, stream);
  return wide ? launch_lora<2, 2, false>(p, cl, C, stream) : launch_lora<1, 1, false>(p, cl, C, stream);
}
