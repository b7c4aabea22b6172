// An adapter's factors into the order that lora.cu reads them in, in one launch for all slices of a projection.
//
// Every thread makes 16 bytes of the packed factors: eight of K of one rank of A, or of B eight ranks of one column (in the order
// of lanes: four ranks of two columns), zeros behind the ranks, K and the columns.  Bound by what it reads and writes, or rather by
// the launch: 16 ranks of 4096 to 6144 in three slices are 0.6 MB (14 us a load, the host's time; with a copy a factor and the ranks
// from the host 103).

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../common/pdl.cuh"
#include "../common/ptx.cuh"

namespace b200 {

static constexpr int kPackThreads = 256, kPackSlices = 4;

struct PackParams {
  const void* a[kPackSlices];                    // [r, K]
  const void* b[kPackSlices];                    // [n, r]
  long long a_row[kPackSlices], a_col[kPackSlices], b_row[kPackSlices], b_col[kPackSlices];
  int a_type[kPackSlices], b_type[kPackSlices];  // 0 bf16, 1 fp16, 2 fp32
  int r[kPackSlices], rank[kPackSlices], n[kPackSlices];   // ranks, the same in whole 16, columns
  __nv_bfloat16 *out_a, *out_b;
  int* out_ranks;
  long long a_units, units;                      // of 16 bytes: of A, of both
  int slices, K, sum_r, block, scale;
  bool lanes;
};

__device__ __forceinline__ float pack_value(const void* p, int type, long long at) {
  if (type == 0) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
  if (type == 1) return __half2float(static_cast<const __half*>(p)[at]);
  return static_cast<const float*>(p)[at];
}

// `count` neighbours along a row from element `at` on, zeros behind them
__device__ __forceinline__ uint4 pack_eight(const void* p, int type, long long at, long long step, int count) {
  if (type == 0 && step == 1 && count >= 8 && (reinterpret_cast<uintptr_t>(static_cast<const __nv_bfloat16*>(p) + at) & 15) == 0)
    return *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + at);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < count ? pack_value(p, type, at + i * step) : 0.f;
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

__global__ void __launch_bounds__(kPackThreads) lora_pack_kernel(const __grid_constant__ PackParams p) {
  pdl_wait();
  pdl_trigger();
  const long long u = static_cast<long long>(blockIdx.x) * kPackThreads + threadIdx.x;
  if (u <= p.slices) p.out_ranks[u] = u < p.slices ? p.r[u] : p.scale;
  if (u >= p.units) return;
  if (u < p.a_units) {
    // [K / 32][rank / 8][4][8][8]
    const long long step = u / (p.sum_r * 4);
    const int rest = static_cast<int>(u - step * p.sum_r * 4);
    int j = rest / 32 * 8 + rest % 8, s = 0;
    while (j >= p.rank[s]) j -= p.rank[s++];
    const long long k = step * 32 + rest / 8 % 4 * 8;
    const bool in = j < p.r[s] && k < p.K;                             // K is a multiple of 8
    reinterpret_cast<uint4*>(p.out_a)[u] = in ? pack_eight(p.a[s], p.a_type[s], j * p.a_row[s] + k * p.a_col[s], p.a_col[s], 8)
                                              : make_uint4(0, 0, 0, 0);
    return;
  }
  long long v = u - p.a_units;
  int s = 0;
  for (;; ++s) {
    const long long here = static_cast<long long>((p.n[s] + p.block - 1) / p.block) * p.block * p.rank[s] / 8;
    if (v < here) break;
    v -= here;
  }
  const int per = p.block * p.rank[s] / 8, rest = static_cast<int>(v % per);
  const long long first = v / per * p.block;                           // column of the block's first
  uint4 w;
  if (p.lanes) {
    // [rank / 16][v][lane][8]: columns 8 (g / 2) + 2 j + g % 2 for j = 2 v, 2 v + 1 times k = 2 q, 2 q + 1, 2 q + 8, 2 q + 9
    const int lane = rest % 32, g = lane / 4, q = lane % 4, k0 = rest / 64 * 16 + 2 * q;
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long long col = first + g / 2 * 8 + 2 * (rest / 32 % 2 * 2 + i / 4) + g % 2;
      const int k = k0 + (i / 2 % 2) * 8 + i % 2;
      f[i] = col < p.n[s] && k < p.r[s] ? pack_value(p.b[s], p.b_type[s], col * p.b_row[s] + k * p.b_col[s]) : 0.f;
    }
    w = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  } else {
    // [rank / 8][block / 32][4][8][8]
    const int i = rest % 8, j = rest / 8 % 4, half = rest / 32 % (p.block / 32), k = rest / p.block * 8;
    const long long col = first + half * 32 + i / 2 * 8 + 2 * j + i % 2;
    w = col < p.n[s] && k < p.r[s]
            ? pack_eight(p.b[s], p.b_type[s], col * p.b_row[s] + k * p.b_col[s], p.b_col[s], min(8, p.r[s] - k))
            : make_uint4(0, 0, 0, 0);
  }
  reinterpret_cast<uint4*>(p.out_b)[u - p.a_units] = w;
}

}  // namespace b200

// Per slice (rank 0: none): a, b and their strides in elements, types (0 bf16, 1 fp16, 2 fp32), rank r, columns n.
extern "C" int b200_lora_pack(const void* const* a, const void* const* b, const long long* a_strides, const long long* b_strides,
                              const int* a_types, const int* b_types, const int* r, const int* n, int slices, int K, bool lanes,
                              int block, float scale, void* out_a, void* out_b, int* out_ranks, cudaStream_t stream) {
  using namespace b200;
  if (slices < 1 || slices > kPackSlices || (K & 7) || (block != 32 && block != 64) || (lanes && block != 32)) return -1;
  PackParams p = {};
  long long b_units = 0;
  for (int s = 0; s < slices; ++s) {
    p.a[s] = a[s], p.b[s] = b[s];
    p.a_row[s] = a_strides[2 * s], p.a_col[s] = a_strides[2 * s + 1];
    p.b_row[s] = b_strides[2 * s], p.b_col[s] = b_strides[2 * s + 1];
    p.a_type[s] = a_types[s], p.b_type[s] = b_types[s];
    p.r[s] = r[s], p.rank[s] = (r[s] + 15) / 16 * 16, p.n[s] = n[s];
    p.sum_r += p.rank[s];
    b_units += static_cast<long long>((n[s] + block - 1) / block) * block * p.rank[s] / 8;
  }
  p.out_a = static_cast<__nv_bfloat16*>(out_a);
  p.out_b = static_cast<__nv_bfloat16*>(out_b);
  p.out_ranks = out_ranks;
  p.a_units = static_cast<long long>((K + 31) / 32) * p.sum_r * 4;
  p.units = p.a_units + b_units;
  p.slices = slices, p.K = K, p.block = block, p.lanes = lanes;
  union { float f; int i; } bits = {scale};
  p.scale = bits.i;
  const long long blocks = std::max<long long>(1, (p.units + kPackThreads - 1) / kPackThreads);
  return launch_pdl(lora_pack_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kPackThreads), 0, stream, 1, p) == cudaSuccess ? 0 : -3;
}
