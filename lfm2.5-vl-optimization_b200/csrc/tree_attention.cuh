// Shared pieces of the drafted-token attention kernels (tree_attention.cu, tree_attention_tc.cu).
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "common.cuh"

namespace lfm2q {

constexpr int TA_KEYS = 64;  // keys per tile

// Pairs of cache elements
template <class T>
struct Pair;
template <>
struct Pair<bf16> {
  static __device__ __forceinline__ float2 up(uint32_t u) { return make_float2(bf_lo(u), bf_hi(u)); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static __device__ __forceinline__ bool finite(uint32_t u) {
    return (u & 0x7f80u) != 0x7f80u && (u & 0x7f800000u) != 0x7f800000u;
  }
};
template <>
struct Pair<__half> {
  static __device__ __forceinline__ float2 up(uint32_t u) { return __half22float2(*reinterpret_cast<__half2 *>(&u)); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  static __device__ __forceinline__ bool finite(uint32_t u) {
    return (u & 0x7c00u) != 0x7c00u && (u & 0x7c000000u) != 0x7c000000u;
  }
};

// 2^x, to about 2 ulp (results below 2^-126 are 0)
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

struct TreeArgs {
  const void *q, *kc, *vc;
  const int *table, *ctx, *cu;
  const unsigned long long *mask;
  void *out;
  float *ws;
  float scale_log2;  // scale * log2 e
  int N, B, NQ, NKV, G, page, width, num_pages, S, max_q;
};

// Lengths of request b, held inside what the tensors have: queries within [0, N) and at most max_q, positions within
// the table.
struct Request {
  int n0, T, ctx, len;
  __device__ __forceinline__ Request(const TreeArgs &a, int b) {
    const int c0 = __ldcg(a.cu + b), c1 = __ldcg(a.cu + b + 1);
    n0 = min(max(c0, 0), a.N);
    T = max(0, min(min(c1, a.N) - n0, a.max_q));
    const long long room = (long long)a.width * a.page;
    ctx = (int)min((long long)max(0, __ldcg(a.ctx + b)), room);
    len = (int)min((long long)ctx + T, room);
  }
};

// Keys per split, the same for every request (so that splits of long and short requests take the same time): the
// longest request cut into S, in whole tiles. For a whole block; `red` is one int of its shared memory.
__device__ __forceinline__ int split_chunk(const TreeArgs &a, int *red) {
  if (threadIdx.x == 0) *red = 1;
  __syncthreads();
  int longest = 1;
  for (int b = threadIdx.x; b < a.B; b += blockDim.x) longest = max(longest, Request(a, b).len);
  longest = __reduce_max_sync(0xffffffffu, longest);
  if ((threadIdx.x & 31) == 0) atomicMax(red, longest);
  __syncthreads();
  return ((*red + a.S - 1) / a.S + TA_KEYS - 1) / TA_KEYS * TA_KEYS;
}

// tree_attention_tc.cu
cudaError_t launch_tree_tc(const TreeArgs &a, int D, bool half, bool pdl, cudaStream_t st);

}  // namespace lfm2q
