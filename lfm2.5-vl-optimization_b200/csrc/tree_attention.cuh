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
  __device__ __forceinline__ Request() {}
  __device__ __forceinline__ Request(const TreeArgs &a, int b) {
    const int c0 = __ldcg(a.cu + b), c1 = __ldcg(a.cu + b + 1);
    n0 = min(max(c0, 0), a.N);
    T = max(0, min(min(c1, a.N) - n0, a.max_q));
    const long long room = (long long)a.width * a.page;
    ctx = (int)min((long long)max(0, __ldcg(a.ctx + b)), room);
    len = (int)min((long long)ctx + T, room);
  }
};

// Keys per split of the kernel for pages that are not multiples of 8, the same for every request (so that splits of long
// and short requests take the same time): the longest request cut into S, in whole tiles. For a whole block; `red` is one
// int of its shared memory.
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

// How the tensor-core kernel deals out work. A unit is one KV head and up to `rows` rows of one request; the tiles of all
// units, in the order (request, KV head, row tile, position), are one line that is cut into equal stretches of `quota`
// tiles, one a block: every block has the same work whatever the lengths, and a unit is split only where a stretch ends.
// Every unit counts TA_UNIT_COST tiles more than it has, for its beginning and end in a block: by a fit over blocks of one
// to four units 3.9 us, where a tile takes 0.6 us (32 requests x 16 drafts: 50 us with 3 tiles, 47 with 5 to 9; 100
// requests x 4: 89 and 80; heads of 128, 32 x 16: 92 us with 3, 82 with 5 and 8). No unit may fall into more than S
// stretches: quota >= longest / (S - 1). With S = 1 whole units are dealt out. The entry point holds the line below 2^31
// tiles. Every division here is on the way to the block's first load (with 64 bits and three more of them: one token
// 10.8 us, 10.2 so).
constexpr int TA_UNIT_COST = 5;
struct TreePlan {
  int rows;        // of a unit
  int quota;
  int x0, count;   // the block's stretch of the line
  int b;           // request of its first tile
  int base;        // tiles before that request
  int r_n0, r_T, r_ctx, r_len;  // lane i: request i (of the first 32)
  static __device__ __forceinline__ int tiles(const Request &rq) { return (rq.len + TA_KEYS - 1) / TA_KEYS; }
  // what a unit of n tiles takes of the line
  static __device__ __forceinline__ int span(const TreeArgs &a, int n) { return a.S == 1 ? 1 : n + TA_UNIT_COST; }
  // units of a KV head
  __device__ __forceinline__ int per_head(const TreeArgs &a, const Request &rq) const {
    return rq.T * a.G <= rows ? 1 : (rq.T * a.G + rows - 1) / rows;
  }
  __device__ __forceinline__ int weight(const TreeArgs &a, const Request &rq, int &n) const {
    n = 0;
    if (rq.T == 0) return 0;
    n = tiles(rq);
    return a.NKV * per_head(a, rq) * span(a, n);
  }
  // request i, for a whole warp: of the first 32 without another load
  __device__ __forceinline__ Request request(const TreeArgs &a, int i) const {
    if (i >= 32) return Request(a, i);
    Request rq;
    rq.n0 = __shfl_sync(0xffffffffu, r_n0, i);
    rq.T = __shfl_sync(0xffffffffu, r_T, i);
    rq.ctx = __shfl_sync(0xffffffffu, r_ctx, i);
    rq.len = __shfl_sync(0xffffffffu, r_len, i);
    return rq;
  }
  // For a whole warp: the stretch of block c of `blocks`.
  __device__ __forceinline__ TreePlan(const TreeArgs &a, int rows_, int blocks, int c)
      : rows(rows_), x0(0), count(0), b(a.B), base(0) {
    const int lane = threadIdx.x & 31;
    int longest = 1, total = 0, first = 0;
    r_n0 = r_T = r_ctx = r_len = 0;
#pragma unroll 4
    for (int i = lane; i < a.B; i += 32) {
      int n;
      const Request rq(a, i);
      const int w = weight(a, rq, n);
      if (i == lane) {
        first = w;
        r_n0 = rq.n0;
        r_T = rq.T;
        r_ctx = rq.ctx;
        r_len = rq.len;
      }
      total += w;
      longest = max(longest, n);
    }
    total = (int)__reduce_add_sync(0xffffffffu, (unsigned)total);
    longest = __reduce_max_sync(0xffffffffu, longest);
    quota = (total + blocks - 1) / blocks;
    if (a.S > 1 && (long long)quota * (a.S - 1) < longest) quota = (longest + a.S - 2) / (a.S - 1);
    // A part of few tiles and many rows writes, and the joining kernel reads, more than it loads: a tile for every 64 rows
    // (5 requests x 13 drafts, 104 rows of 128: 21.6 us with a tile a part, 19.3 with two).
    if (a.S > 1) quota = max(quota, (min(rows, a.max_q * a.G) + 63) / 64);
    if ((long long)quota * c >= total) return;
    x0 = quota * c;
    count = min(quota, total - x0);
    int run = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      int n;
      const int w = b0 == 0 ? first : b0 + lane < a.B ? weight(a, Request(a, b0 + lane), n) : 0;
      int s = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int s2 = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += s2;
      }
      s += run;
      const uint32_t here = __ballot_sync(0xffffffffu, s - w <= x0 && x0 < s);
      if (here) {  // one lane
        const int at = __ffs(here) - 1;
        b = b0 + at;
        base = __shfl_sync(0xffffffffu, s - w, at);
        break;
      }
      run = __shfl_sync(0xffffffffu, s, 31);
    }
  }
};

// The workspace of a call with S > 1 splits: for every part of every row its accumulator divided by its sum, [S][N NQ]
// [D], then per row 1 + S words: the number of parts, and each part's log2 of the sum of 2^score.
__device__ __forceinline__ float *ws_acc(const TreeArgs &a, int D, int part, size_t row) {
  return a.ws + ((size_t)part * a.N * a.NQ + row) * D;
}
__device__ __forceinline__ float *ws_row(const TreeArgs &a, int D, size_t row) {
  return a.ws + (size_t)a.S * a.N * a.NQ * D + row * (1 + a.S);
}

// tree_attention_tc.cu
cudaError_t launch_tree_tc(const TreeArgs &a, int D, bool half, bool pdl, cudaStream_t st);

}  // namespace lfm2q
