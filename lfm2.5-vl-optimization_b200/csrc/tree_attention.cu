// Attention of drafted tokens over a paged KV cache: every request b brings T_b = cu[b + 1] - cu[b] query tokens
// (a tree of drafts, a chain, or the one token of an ordinary decode step), whose keys and values already lie in the
// cache behind its ctx[b] cached positions. Query i sees every position t < ctx[b], and position ctx[b] + j (draft j)
// where bit j of its mask is set (mask NULL: j <= i). out = softmax(scale q.k) v per head; a query that sees nothing
// gives zeros. Heads are grouped: G = NQ / NKV query heads share a KV head.
//
// Mathematics: the rows of one (request, KV head) are its T_b G queries, so K and V are read once for all of them;
// the online softmax keeps a running maximum m and sum l per row in fp32 (base 2: scores times scale log2 e) and
// rescales the fp32 accumulator when m grows. The probabilities are rounded to the cache's type for the second
// product, which 16-bit operands of the tensor cores ask for, and l sums the unrounded ones: each p is off by at most half
// a step, which leaves out within one rounding of that type. In fp16, whose steps are fixed below 2^-14, they are raised
// by a power of two before the rounding (here 2^15, and m stands for the maximum less 15): half a step of each holds down
// to 2^-29 of the largest, and below that each is off by 2^-40 at most (tree_attention_tc.cu: 2^-25 and 2^-36).
//
// Two kernels: tree_attention_tc.cu has the one for pages that are multiples of 8 positions (a TMA box of rows never
// crosses a page, and eight rows are the swizzle's period); this file the one for other pages, and the join of both.
// 32 requests x 16 drafts x 500 to 4000 positions, 32 heads over 8 KV heads of 64: 111 us here with pages of 20 or 36,
// 44 us there with pages of 16 or 64, 49 us with pages of 8.
//
// Here a block takes a tile of 64 keys at a time through a ring of cp.async stages, 16 bytes a lane, each with its own
// page (rows swizzled in 16-byte units, so ldmatrix reads are conflict-free), mma.sync m16n8k16 for both products. What
// bounds it is the instructions: some 950 a warp and tile, the address of every 16 bytes among them. Long caches are cut
// into S splits of one length for all requests (split_chunk); the accumulator of a split, divided by its sum, and log2 of
// that sum go to ws, and tree_combine_kernel joins them in split order: the same result in every run. Rows behind the
// request's length, and positions whose table entry is not a page of the pool, are filled with zeros in shared memory
// and masked: nothing outside the pool is read.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "launch.h"
#include "tree_attention.cuh"

namespace lfm2q {
namespace {

template <class T>
struct Mma;
template <>
struct Mma<bf16> {
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct Mma<__half> {
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ uint32_t saddr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
// 16 bytes global -> shared; bytes = 0 writes zeros and reads nothing
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// WM x WK warps: WM row groups of 16 MT rows, WK groups of 64 / WK keys of every tile (joined at the end).
template <class T, int D, int WM, int WK, int MT, int STAGES>
__global__ void __launch_bounds__(32 * WM * WK) tree_kernel(const TreeArgs a) {
  constexpr int THREADS = 32 * WM * WK, ROWS = 16 * WM * MT;
  constexpr int CH = D / 8;              // 16-byte units per row
  constexpr int KW = TA_KEYS / WK;       // keys of a tile per warp
  constexpr int NB = KW / 8;             // 8-key column blocks per warp
  constexpr int TILE = TA_KEYS * D * 2;  // bytes of a K (or V) tile
  constexpr float RAISE = std::is_same<T, __half>::value ? 15.f : 0.f;
  extern __shared__ __align__(128) uint8_t ta_smem[];
  __shared__ int bad_pages;  // a page outside the pool was met
  __shared__ int red;
  uint8_t *sk = ta_smem, *sv = ta_smem + STAGES * TILE, *sq = ta_smem + 2 * STAGES * TILE;
  pdl_trigger();
  pdl_wait();
  const int kvh = blockIdx.x % a.NKV, b = blockIdx.x / a.NKV, split = blockIdx.y, r_base = blockIdx.z * ROWS;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wm = warp / WK, wk = warp % WK;
  const Request rq(a, b);
  const int rows = rq.T * a.G;
  if (r_base >= rows) return;
  const int chunk = split_chunk(a, &red);
  const int t0 = (int)min((long long)split * chunk, (long long)rq.len), t1 = t0 + min(rq.len - t0, chunk);
  const int tiles = (t1 - t0 + TA_KEYS - 1) / TA_KEYS;
  if (tid == 0) bad_pages = 0;
  __syncthreads();

  // queries: row r = token r / G, head kvh G + r % G, swizzled like the keys; rows past the end are zeros
  for (int i = tid; i < ROWS * CH; i += THREADS) {
    const int r = i / CH, c = i % CH, gr = r_base + r;
    const bool in = gr < rows;
    const T *src = reinterpret_cast<const T *>(a.q) +
                   ((size_t)(rq.n0 + (in ? gr / a.G : 0)) * a.NQ + kvh * a.G + (in ? gr % a.G : 0)) * D + 8 * c;
    cp16(saddr(sq + (r * CH + (c ^ (r & 7))) * 16), src, in ? 16 : 0);
  }
  cp_commit();

  const int *table = a.table + (size_t)b * a.width;
  auto page_of = [&](int t) { return __ldcg(table + t / a.page); };
  auto load_tile = [&](int i) {
    const int base = t0 + i * TA_KEYS, slot = i % STAGES;
    constexpr int RPP = THREADS / CH;  // rows per pass
    static_assert(THREADS % CH == 0 && TA_KEYS % RPP == 0, "whole passes");
    const int c = tid % CH;
#pragma unroll
    for (int p = 0; p < TA_KEYS / RPP; ++p) {
      const int r = p * RPP + tid / CH, t = base + r;
      bool in = t < t1;
      size_t off = 0;
      if (in) {
        const int pg = page_of(t);
        in = pg >= 0 && pg < a.num_pages;
        if (!in) bad_pages = 1;
        else off = (((size_t)pg * a.NKV + kvh) * a.page + t % a.page) * D + 8 * c;
      }
      const uint32_t d = (r * CH + (c ^ (r & 7))) * 16;
      cp16(saddr(sk + slot * TILE + d), reinterpret_cast<const T *>(a.kc) + off, in ? 16 : 0);
      cp16(saddr(sv + slot * TILE + d), reinterpret_cast<const T *>(a.vc) + off, in ? 16 : 0);
    }
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    if (i < tiles) load_tile(i);
    cp_commit();
  }

  float o[MT][D / 8][4], m[MT][2], l[MT][2];
  unsigned long long see[MT][2];  // the drafts that the lane's rows see
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int j = 0; j < D / 8; ++j) o[mt][j][0] = o[mt][j][1] = o[mt][j][2] = o[mt][j][3] = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m[mt][h] = -INFINITY;
      l[mt][h] = 0.f;
      const int gr = r_base + wm * 16 * MT + mt * 16 + (lane >> 2) + 8 * h;
      see[mt][h] = 0;
      if (gr < rows) {
        const int i = gr / a.G;
        see[mt][h] = a.mask ? __ldcg(a.mask + rq.n0 + i) : (i >= 63 ? ~0ull : (2ull << i) - 1);
      }
    }
  }

  unsigned long long apart = 0;  // this warp's drafts that were taken out of the second product
  for (int it = 0; it < tiles; ++it) {
    cp_wait<STAGES - 2>();
    __syncthreads();  // the tile has landed for every warp, and the slot of tile it - 1 is free
    if (it + STAGES - 1 < tiles) load_tile(it + STAGES - 1);
    cp_commit();
    const int slot = it % STAGES, base = t0 + it * TA_KEYS;
    const uint32_t kb = saddr(sk + slot * TILE), vb = saddr(sv + slot * TILE), qb = saddr(sq);
    const int k0 = wk * KW;  // this warp's keys of the tile

    // ---------------------------------------------------------------- scores
    float s[MT][NB][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < NB; ++j) s[mt][j][0] = s[mt][j][1] = s[mt][j][2] = s[mt][j][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      uint32_t qa[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int r = wm * 16 * MT + mt * 16 + (lane & 15), c = 2 * kk + (lane >> 4);
        ldsm4(qa[mt], qb + (r * CH + (c ^ (r & 7))) * 16);
      }
#pragma unroll
      for (int jp = 0; jp < NB / 2; ++jp) {  // two 8-key blocks per ldmatrix.x4
        uint32_t kf[4];
        const int r = k0 + jp * 16 + (lane & 7) + ((lane >> 4) << 3), c = 2 * kk + ((lane >> 3) & 1);
        ldsm4(kf, kb + (r * CH + (c ^ (r & 7))) * 16);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          Mma<T>::run(s[mt][2 * jp], qa[mt], kf[0], kf[1]);
          Mma<T>::run(s[mt][2 * jp + 1], qa[mt], kf[2], kf[3]);
        }
      }
    }
    // ---------------------------------------------------------------- masks
    const bool edge = base + TA_KEYS > rq.ctx || base + TA_KEYS > t1;
    const bool bad = *(volatile int *)&bad_pages != 0;
    if (edge || bad) {
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int t = base + k0 + 8 * j + 2 * (lane & 3) + e;
          bool in = t < t1;
          if (in && bad) {
            const int pg = page_of(t);
            in = pg >= 0 && pg < a.num_pages;
          }
          const int d = t - rq.ctx;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (!in || (d >= 0 && !((see[mt][h] >> d) & 1))) s[mt][j][2 * h + e] = -INFINITY;
        }
    }
    // ---------------------------------------------------------------- online softmax
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < NB; ++j) mx = fmaxf(mx, fmaxf(s[mt][j][2 * h], s[mt][j][2 * h + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m[mt][h], mx * a.scale_log2 - RAISE);
        const float ms = mn == -INFINITY ? 0.f : mn;
        const float corr = ex2(m[mt][h] - ms);  // 2^-inf = 0 while nothing was seen
        m[mt][h] = mn;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float p = ex2(fmaf(s[mt][j][2 * h + e], a.scale_log2, -ms));
            s[mt][j][2 * h + e] = p;
            sum += p;
          }
        l[mt][h] = l[mt][h] * corr + sum;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          o[mt][j][2 * h] *= corr;
          o[mt][j][2 * h + 1] *= corr;
        }
      }
    // ---------------------------------------------------------------- values
    // A draft that a row does not see has p = 0 there, but 0 times an infinity or a NaN is a NaN: drafts whose value
    // row holds one are taken out of the product, and added at the end to the rows that see them.
    unsigned long long weird = 0;
    if (base + TA_KEYS > rq.ctx) {
#pragma unroll
      for (int g = 0; g < (KW + 31) / 32; ++g) {
        bool w = false;
        const int r = k0 + g * 32 + lane;
        if (g * 32 + lane < KW && base + r >= rq.ctx) {
#pragma unroll 4
          for (int c = 0; c < CH; ++c) {
            const uint4 u = *reinterpret_cast<const uint4 *>(sv + slot * TILE + (r * CH + c) * 16);
            w = w || !(Pair<T>::finite(u.x) && Pair<T>::finite(u.y) && Pair<T>::finite(u.z) && Pair<T>::finite(u.w));
          }
        }
        weird |= (unsigned long long)__ballot_sync(0xffffffffu, w) << (32 * g);
      }
      const int d0 = base + k0 - rq.ctx;  // draft of the warp's first key (> -64)
      apart |= d0 >= 0 ? weird << d0 : weird >> -d0;
    }
#pragma unroll
    for (int kk = 0; kk < KW / 16; ++kk) {
      uint32_t pa[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        pa[mt][0] = Pair<T>::pack(s[mt][2 * kk][0], s[mt][2 * kk][1]);
        pa[mt][1] = Pair<T>::pack(s[mt][2 * kk][2], s[mt][2 * kk][3]);
        pa[mt][2] = Pair<T>::pack(s[mt][2 * kk + 1][0], s[mt][2 * kk + 1][1]);
        pa[mt][3] = Pair<T>::pack(s[mt][2 * kk + 1][2], s[mt][2 * kk + 1][3]);
      }
#pragma unroll
      for (int jp = 0; jp < D / 16; ++jp) {
        uint32_t vf[4];
        const int r = k0 + kk * 16 + (lane & 15), c = 2 * jp + (lane >> 4);
        ldsm4t(vf, vb + (r * CH + (c ^ (r & 7))) * 16);
        if (weird) {  // a lane's registers hold keys 2 (lane % 4), + 1 of each eight
          const uint32_t w = (uint32_t)(weird >> (16 * kk + 2 * (lane & 3)));
          const uint32_t k0m = ((w & 1) ? 0u : 0xffffu) | ((w & 2) ? 0u : 0xffff0000u);
          const uint32_t k8m = ((w & 0x100) ? 0u : 0xffffu) | ((w & 0x200) ? 0u : 0xffff0000u);
          vf[0] &= k0m;
          vf[1] &= k8m;
          vf[2] &= k0m;
          vf[3] &= k8m;
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          Mma<T>::run(o[mt][2 * jp], pa[mt], vf[0], vf[1]);
          Mma<T>::run(o[mt][2 * jp + 1], pa[mt], vf[2], vf[3]);
        }
      }
    }
  }
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[mt][h] += __shfl_xor_sync(0xffffffffu, l[mt][h], 1);
      l[mt][h] += __shfl_xor_sync(0xffffffffu, l[mt][h], 2);
    }

  for (; apart; apart &= apart - 1) {  // rare: the score again from global memory, and p v added where it is seen
    const int d = __ffsll(apart) - 1, t = rq.ctx + d;
    const size_t at = (((size_t)page_of(t) * a.NKV + kvh) * a.page + t % a.page) * D;  // a page of the pool: it held
    const T *kr = reinterpret_cast<const T *>(a.kc) + at, *vr = reinterpret_cast<const T *>(a.vc) + at;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int gr = r_base + wm * 16 * MT + mt * 16 + (lane >> 2) + 8 * h;
        const T *qr = reinterpret_cast<const T *>(a.q) +
                      ((size_t)(rq.n0 + (gr < rows ? gr / a.G : 0)) * a.NQ + kvh * a.G + (gr < rows ? gr % a.G : 0)) * D;
        float dot = 0.f;
        for (int j = lane & 3; j < D / 2; j += 4) {
          const float2 x = Pair<T>::up(__ldcg(reinterpret_cast<const uint32_t *>(qr) + j));
          const float2 y = Pair<T>::up(__ldcg(reinterpret_cast<const uint32_t *>(kr) + j));
          dot += x.x * y.x + x.y * y.y;
        }
        dot += __shfl_xor_sync(0xffffffffu, dot, 1);
        dot += __shfl_xor_sync(0xffffffffu, dot, 2);
        if (gr < rows && ((see[mt][h] >> d) & 1)) {
          const float p = ex2(fmaf(dot, a.scale_log2, m[mt][h] == -INFINITY ? 0.f : -m[mt][h]));
#pragma unroll
          for (int j = 0; j < D / 8; ++j) {
            const float2 v = Pair<T>::up(__ldcg(reinterpret_cast<const uint32_t *>(vr) + 4 * j + (lane & 3)));
            o[mt][j][2 * h] += p * v.x;
            o[mt][j][2 * h + 1] += p * v.y;
          }
        }
      }
  }

  // ---------------------------------------------------------------- join the WK key groups of a row group
  if (WK > 1) {
    constexpr int PITCH = D + 4;  // floats per row: m, l, acc (4 floats apart from a bank multiple)
    static_assert(WM * WK * 16 * MT * PITCH * 4 <= 2 * STAGES * TILE, "the partials fit in the ring");
    float *part = reinterpret_cast<float *>(ta_smem);
    cp_wait<0>();
    __syncthreads();
    if (wk > 0) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float *p = part + ((wm * WK + wk) * 16 * MT + mt * 16 + (lane >> 2) + 8 * h) * PITCH;
          if ((lane & 3) == 0) {
            p[D] = m[mt][h];
            p[D + 1] = l[mt][h];
          }
#pragma unroll
          for (int j = 0; j < D / 8; ++j)
            *reinterpret_cast<float2 *>(p + 8 * j + 2 * (lane & 3)) = make_float2(o[mt][j][2 * h], o[mt][j][2 * h + 1]);
        }
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        for (int w = 1; w < WK; ++w) {
          const float *p = part + ((wm * WK + w) * 16 * MT + mt * 16 + (lane >> 2) + 8 * h) * PITCH;
          const float m2 = p[D], l2 = p[D + 1], mn = fmaxf(m[mt][h], m2), ms = mn == -INFINITY ? 0.f : mn;
          const float c1 = ex2(m[mt][h] - ms), c2 = ex2(m2 - ms);
          m[mt][h] = mn;
          l[mt][h] = l[mt][h] * c1 + l2 * c2;
#pragma unroll
          for (int j = 0; j < D / 8; ++j) {
            const float2 v = *reinterpret_cast<const float2 *>(p + 8 * j + 2 * (lane & 3));
            o[mt][j][2 * h] = o[mt][j][2 * h] * c1 + v.x * c2;
            o[mt][j][2 * h + 1] = o[mt][j][2 * h + 1] * c1 + v.y * c2;
          }
        }
  }

  // ---------------------------------------------------------------- out, or this split's partial
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int gr = r_base + wm * 16 * MT + mt * 16 + (lane >> 2) + 8 * h;
      if (gr >= rows) continue;
      const size_t row = (size_t)(rq.n0 + gr / a.G) * a.NQ + kvh * a.G + gr % a.G;
      if (a.S == 1) {
        const float inv = l[mt][h] == 0.f ? 0.f : 1.f / l[mt][h];
        uint32_t *dst = reinterpret_cast<uint32_t *>(reinterpret_cast<T *>(a.out) + row * D) + (lane & 3);
#pragma unroll
        for (int j = 0; j < D / 8; ++j) dst[4 * j] = Pair<T>::pack(o[mt][j][2 * h] * inv, o[mt][j][2 * h + 1] * inv);
      } else {
        const float inv = l[mt][h] == 0.f ? 0.f : 1.f / l[mt][h];
        float *w = ws_acc(a, D, split, row), *info = ws_row(a, D, row);
        if ((lane & 3) == 0) {
          info[1 + split] = l[mt][h] == 0.f ? -INFINITY : m[mt][h] + log2f(l[mt][h]);
          if (split == 0) reinterpret_cast<int *>(info)[0] = a.S;
        }
#pragma unroll
        for (int j = 0; j < D / 8; ++j)
          *reinterpret_cast<float2 *>(w + 8 * j + 2 * (lane & 3)) =
              make_float2(o[mt][j][2 * h] * inv, o[mt][j][2 * h + 1] * inv);
      }
    }
}

// D / 4 lanes per (query, head): the parts joined in order. A row of one part has been written by its block. What bounds
// it is a chain of loads (lengths, the parts' sums, the parts), so the sums come in one go, UNR parts are in flight
// together and, at D = 64, two rows share a warp (32 requests x 16 drafts in all: 47.4 us with a row a warp, 44.3 so). UNR
// 16 where there may be many parts, which are few rows (one token: 10.8 us, 11.1 with 8), else 8, which leaves room for
// more warps (32 x 16 drafts: 44.3 us, 46.6 with 16, 44.3 with 4).
constexpr int TC_WARPS = 4;
template <class T, int D, int UNR>
__global__ void __launch_bounds__(32 * TC_WARPS) tree_combine_kernel(const TreeArgs a) {
  constexpr int LANES = D / 4, ROWS = 32 / LANES;  // of a row; rows of a warp
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, sub = lane % LANES;
  const int unit = (blockIdx.x * TC_WARPS + (threadIdx.x >> 5)) * ROWS + lane / LANES;
  const int b = blockIdx.y, i = unit / a.NQ, h = unit - i * a.NQ;
  const Request rq(a, b);
  const bool live = i < rq.T;
  const size_t row = live ? (size_t)(rq.n0 + i) * a.NQ + h : 0;
  const float *info = ws_row(a, D, row);
  // two loads at once bring the number of parts (lane 0) and the first parts' logarithms (word 1 + part)
  const float first = live && sub <= a.S ? __ldcg(info + sub) : -INFINITY;
  const float second = live && LANES + sub <= a.S ? __ldcg(info + LANES + sub) : -INFINITY;
  // (held to S: after a wait that gave up the words were never written)
  int parts = min(__shfl_sync(0xffffffffu, __float_as_int(first), 0, LANES), a.S);
  if (!live || parts <= 1) parts = 0;
  const int most = __reduce_max_sync(0xffffffffu, parts);
  if (most == 0) return;
  float M = sub > 0 && sub <= parts ? first : -INFINITY;
  if (LANES + sub <= parts) M = fmaxf(M, second);
  for (int s = 2 * LANES - 1 + sub; s < parts; s += LANES) M = fmaxf(M, __ldcg(info + 1 + s));
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  const float ms = M == -INFINITY ? 0.f : M;
  float L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < most; s0 += UNR) {  // UNR parts in flight
    float4 v[UNR];
#pragma unroll
    for (int u = 0; u < UNR; ++u)
      v[u] = s0 + u < parts ? __ldcg(reinterpret_cast<const float4 *>(ws_acc(a, D, s0 + u, row) + 4 * sub))
                            : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int u = 0; u < UNR; ++u) {
      const int s = s0 + u;
      float lse = __shfl_sync(0xffffffffu, s + 1 < LANES ? first : second, (s + 1) & (LANES - 1), LANES);
      if (s + 1 >= 2 * LANES && s < parts) lse = __ldcg(info + 1 + s);
      const float c = s < parts ? ex2(lse - ms) : 0.f;
      L += c;
      acc.x += v[u].x * c;
      acc.y += v[u].y * c;
      acc.z += v[u].z * c;
      acc.w += v[u].w * c;
    }
  }
  if (parts == 0) return;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  *reinterpret_cast<uint2 *>(reinterpret_cast<T *>(a.out) + row * D + 4 * sub) =
      make_uint2(Pair<T>::pack(acc.x * inv, acc.y * inv), Pair<T>::pack(acc.z * inv, acc.w * inv));
}

template <class T, int D>
cudaError_t launch_combine(const TreeArgs &a, bool pdl, cudaStream_t st) {
  auto kernel = a.S <= 8 ? tree_combine_kernel<T, D, 8> : tree_combine_kernel<T, D, 16>;
  constexpr int ROWS = TC_WARPS * 128 / D;  // of a block
  cudaLaunchAttribute attr;
  const cudaLaunchConfig_t cfg =
      pdl_config(dim3((a.max_q * a.NQ + ROWS - 1) / ROWS, a.B), dim3(32 * TC_WARPS), pdl, st, &attr);
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <class T, int D, int WM, int WK, int MT, int STAGES>
cudaError_t launch_tile(const TreeArgs &a, int B, bool pdl, cudaStream_t st) {
  constexpr int ROWS = 16 * WM * MT, SMEM = 2 * STAGES * TA_KEYS * D * 2 + ROWS * D * 2;
  auto kernel = tree_kernel<T, D, WM, WK, MT, STAGES>;
  static std::atomic<int> attr_set[64];  // the shared-memory opt-in, once per device
  int dev = 0;
  if (const cudaError_t e = cudaGetDevice(&dev)) return e;
  if (dev < 64 && !attr_set[dev].load(std::memory_order_acquire)) {
    if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM)) return e;
    attr_set[dev].store(1, std::memory_order_release);
  }
  cudaLaunchAttribute attr;
  cudaLaunchConfig_t cfg = pdl_config(dim3(B * a.NKV, a.S, (a.max_q * a.G + ROWS - 1) / ROWS), dim3(32 * WM * WK), pdl,
                                      st, &attr);
  cfg.dynamicSmemBytes = SMEM;
  if (const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a)) return e;
  return a.S == 1 ? cudaSuccess : launch_combine<T, D>(a, pdl, st);
}

template <class T, int D>
cudaError_t launch_rows(const TreeArgs &a, int B, bool pdl, cudaStream_t st) {
  const int rows = a.max_q * a.G;
  if (rows <= 16) return launch_tile<T, D, 1, 4, 1, 4>(a, B, pdl, st);
  if (rows <= 32) return launch_tile<T, D, 2, 2, 1, 4>(a, B, pdl, st);
  if (rows <= 64) return launch_tile<T, D, 4, 1, 1, 3>(a, B, pdl, st);
  if constexpr (D == 64) return launch_tile<T, D, 4, 1, 2, 3>(a, B, pdl, st);
  else return launch_tile<T, D, 8, 1, 1, 3>(a, B, pdl, st);  // 128-wide accumulators of 32 rows would spill
}

}  // namespace

int tree_attention_splits(int B, int NQ, int NKV, int D, int max_q, long long max_len) {
  // As many parts as the equal stretches of the blocks cut a unit into, were all requests half as long as the longest; no
  // more than a part a tile.
  const int per_tile = std::max(1, 128 / (NQ / NKV)), tiles_q = max_q <= per_tile ? 1 : 2;  // of a unit
  const long long blocks = (tiles_q == 1 && D == 64 ? 2LL : 1LL) * device_sm_count();
  const long long units = (long long)B * NKV * ((max_q + tiles_q * per_tile - 1) / (tiles_q * per_tile));
  const long long parts = 2 + (2 * blocks + units - 1) / units, tiles = (max_len + TA_KEYS - 1) / TA_KEYS;
  return tiles <= 1 ? 1 : (int)std::min(std::min(parts, tiles + 1), 64LL);
}

cudaError_t launch_tree_attention(const void *q, const void *kc, const void *vc, const int *table, const int *ctx,
                                  const int *cu, const int64_t *mask, void *out, float *ws, int N, int B, int NQ,
                                  int NKV, int D, int num_pages, int page, int width, int S, int max_q, float scale,
                                  bool half, bool pdl, cudaStream_t st) {
  const TreeArgs a{q, kc, vc, table, ctx, cu, reinterpret_cast<const unsigned long long *>(mask), out, ws,
                   scale * 1.4426950408889634f, N, B, NQ, NKV, NQ / NKV, page, width, num_pages, S, max_q};
  if (page % 8 == 0) {
    if (const cudaError_t e = launch_tree_tc(a, D, half, pdl, st)) return e;
    if (S == 1) return cudaSuccess;
    if (half) return D == 64 ? launch_combine<__half, 64>(a, pdl, st) : launch_combine<__half, 128>(a, pdl, st);
    return D == 64 ? launch_combine<bf16, 64>(a, pdl, st) : launch_combine<bf16, 128>(a, pdl, st);
  }
  if (half) return D == 64 ? launch_rows<__half, 64>(a, B, pdl, st) : launch_rows<__half, 128>(a, B, pdl, st);
  return D == 64 ? launch_rows<bf16, 64>(a, B, pdl, st) : launch_rows<bf16, 128>(a, B, pdl, st);
}

}  // namespace lfm2q
