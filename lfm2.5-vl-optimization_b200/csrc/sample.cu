// Sampling from given uniforms: sample_next, the batched counterpart of argmax_next.
//
// Row x of V logits, temperature T > 0: w_i = e^((x_i - max) / T), the tokens ordered by (x descending, index
// ascending). Kept: the first top_k; of those the shortest prefix whose mass reaches top_p of theirs (at least one);
// of those w_i >= min_p. Every filter keeps a prefix of the one order, so the kept set is "all keys above a threshold
// key, and the first t of the keys equal to it". The token is the first one, in index order, whose running kept mass
// exceeds u times the kept mass. T <= 0 (or a NaN among the logits) takes the argmax, as argmax_next does.
//
// A sum decides which token comes out, so sums are integers: w in steps of 2^-44 (max w = 1, V <= 2^18, so a sum
// stays below 2^62), exact and the same in any order; the weight is computed in fp64. A cumulative sum is off by at
// most V 2^-45 from the real one: a draw differs from exact arithmetic with a probability of some 10^-9.
//
// A cluster of C thread blocks holds one row in shared memory (read once); selections run as histograms over the
// cluster: 1024 bins linear in x first (so that a peaked row spreads over the bins), then 1024 bins of the order-
// preserving integer key inside the chosen bin until a bin is one key. Every block reads all the cluster's bins and
// finds the same crossing, so nothing is broadcast.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "common.cuh"
#include "launch.h"

namespace cg = cooperative_groups;

namespace lfm2q {
namespace {

constexpr int SA_T = 512;               // threads per block
constexpr int SA_W = SA_T / 32;
constexpr int SA_BINS = 1024;
constexpr int SA_MAX_C = 8;             // blocks per cluster (the portable limit)
constexpr int SA_MAX_STAGE = 160 * 1024;  // bytes of a row that one block stages
constexpr double SA_ONE = 17592186044416.0;  // 2^44

// Element types: raw storage, an order-preserving key (equal keys <=> equal values: -0 takes +0's) and its inverse.
// Key 0 is a filler, below every value (it would be a negative NaN; rows with a NaN never get here).
struct B16 {
  typedef unsigned short raw;
  static constexpr int KEY_BITS = 16;
  static __device__ __forceinline__ float up(raw r) { return __uint_as_float((uint32_t)r << 16); }
};
struct H16 {
  typedef unsigned short raw;
  static constexpr int KEY_BITS = 16;
  static __device__ __forceinline__ float up(raw r) { return __half2float(__ushort_as_half(r)); }
};
struct F32 {
  typedef uint32_t raw;
  static constexpr int KEY_BITS = 32;
  static __device__ __forceinline__ float up(raw r) { return __uint_as_float(r); }
};
template <class E>
__device__ __forceinline__ uint32_t key_of(typename E::raw r) {
  constexpr uint32_t SIGN = 1u << (E::KEY_BITS - 1), ALL = SIGN | (SIGN - 1);
  uint32_t u = r;
  if (u == SIGN) u = 0;
  return (u & SIGN) ? (~u & ALL) : (u | SIGN);
}
template <class E>
__device__ __forceinline__ float value_of(uint32_t key) {
  constexpr uint32_t SIGN = 1u << (E::KEY_BITS - 1), ALL = SIGN | (SIGN - 1);
  return E::up((typename E::raw)((key & SIGN) ? (key & ~SIGN) : (~key & ALL)));
}

struct SampleArgs {
  const void *logits;
  long long stride;
  const float *temperature;
  const int *top_k;
  const float *top_p, *min_p, *u;
  int64_t *tok, *pos;
  int V;
};

__device__ __forceinline__ bool better(float a, int ia, float b, int ib) {
  const bool na = a != a, nb = b != b;
  if (na || nb) return na && (!nb || ia < ib);
  return a > b || (a == b && ia < ib);
}

struct SampleShared {
  float best_v[SA_W];
  int best_i[SA_W];
  float row_v;  // this block's maximum and its index: read by the cluster
  int row_i;
  uint32_t cnt[2][SA_BINS], lo[2][SA_BINS], hi[2][SA_BINS];
  uint32_t kmin[2], kmax[2];  // [0] the selection by count, [1] by mass
  unsigned long long scan[SA_W];
  unsigned long long mass[SA_W];  // per warp: kept mass above the threshold key
  uint32_t ties[SA_W];            // per warp: elements equal to it
  // broadcast within the block
  int bin;
  unsigned long long above, in_bin;
};

__device__ __forceinline__ unsigned long long shfl_up64(unsigned long long v, int o) {
  return __shfl_up_sync(0xffffffffu, v, o);
}

template <class E>
__global__ void __launch_bounds__(SA_T) sample_kernel(const SampleArgs a, int stage_vecs) {
  typedef typename E::raw raw;
  constexpr int PER = 16 / (int)sizeof(raw);  // elements of a 16-byte piece
  extern __shared__ __align__(16) uint8_t sa_smem[];
  __shared__ SampleShared s;
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int row = blockIdx.x / C;
  const int t = threadIdx.x, lane = t & 31, wp = t >> 5;
  pdl_trigger();
  pdl_wait();

  // The row in 16-byte pieces of the address space: piece v holds elements v PER - skew .. + PER. Block `rank` stages
  // pieces [v0, v1); elements outside the row become fillers.
  const raw *x = reinterpret_cast<const raw *>(a.logits) + row * a.stride;
  const int skew = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(raw));
  const int NV = (a.V + skew + PER - 1) / PER;
  const int per_block = (NV + C - 1) / C;
  const int v0 = min(rank * per_block, NV), v1 = min(v0 + per_block, NV), nv = v1 - v0;
  uint4 *stage = reinterpret_cast<uint4 *>(sa_smem);
  float best = -INFINITY;
  int bi = 0x7fffffff;
  constexpr raw FILL = (raw)~(raw)0;
  for (int v = t; v < nv; v += SA_T) {
    const int e0 = (v0 + v) * PER - skew;
    uint4 q;
    raw *qr = reinterpret_cast<raw *>(&q);
    if (e0 >= 0 && e0 + PER <= a.V) {
      q = ld_cg16(x + e0);
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) qr[j] = (e0 + j >= 0 && e0 + j < a.V) ? __ldcg(x + e0 + j) : FILL;
    }
    stage[v] = q;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const float f = E::up(qr[j]);
      if (e0 + j >= 0 && e0 + j < a.V && better(f, e0 + j, best, bi)) {
        best = f;
        bi = e0 + j;
      }
    }
  }
  for (int i = t; i < 2 * SA_BINS; i += SA_T) (&s.cnt[0][0])[i] = (&s.lo[0][0])[i] = (&s.hi[0][0])[i] = 0;
  if (t < 2) {
    s.kmin[t] = 0xffffffffu;
    s.kmax[t] = 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float v2 = __shfl_xor_sync(0xffffffffu, best, o);
    const int i2 = __shfl_xor_sync(0xffffffffu, bi, o);
    if (better(v2, i2, best, bi)) {
      best = v2;
      bi = i2;
    }
  }
  if (lane == 0) {
    s.best_v[wp] = best;
    s.best_i[wp] = bi;
  }
  __syncthreads();
  for (int w = 0; w < SA_W; ++w)
    if (better(s.best_v[w], s.best_i[w], best, bi)) {
      best = s.best_v[w];
      bi = s.best_i[w];
    }
  if (t == 0) {
    s.row_v = best;
    s.row_i = bi;
  }
  cl.sync();
  for (int c = 0; c < C; ++c) {
    const SampleShared *o = cl.map_shared_rank(&s, c);
    const float v2 = o->row_v;
    const int i2 = o->row_i;
    if (better(v2, i2, best, bi)) {
      best = v2;
      bi = i2;
    }
  }

  const float T = a.temperature ? __ldcg(a.temperature + row) : 1.f;
  const float top_p = a.top_p ? __ldcg(a.top_p + row) : 1.f;
  const float min_p = a.min_p ? __ldcg(a.min_p + row) : 0.f;
  const int top_k = a.top_k ? __ldcg(a.top_k + row) : 0;
  const float mx = best;
  auto finish = [&](int token) {
    a.tok[row] = token;
    if (a.pos && row == 0) a.pos[0] = __ldcg(reinterpret_cast<const long long *>(a.pos)) + 1;
  };
  // greedy, a NaN, nothing but -inf, or only one token kept: the first largest
  if (!(T > 0.f) || mx != mx || mx == -INFINITY || top_k == 1) {
    if (rank == 0 && t == 0) finish(bi);
    cl.sync();  // no block leaves while another may still read its shared memory
    return;
  }

  const double dmx = (double)mx, rT = 1.0 / (double)T;
  auto weight = [&](float f) -> double {  // of a non-filler value f <= mx
    return f == mx ? 1.0 : f == -INFINITY ? 0.0 : exp(((double)f - dmx) * rT);
  };
  auto fixed = [&](double w) { return (unsigned long long)__double2ull_rn(w * SA_ONE); };
  const float bin_scale = (float)(1.4426950408889634 * (SA_BINS / 46.0)) / T;
  auto bin_of = [&](float f) {  // level 0: linear in x, monotone; the last bin takes all that is below 2^-46
    const float d = f == mx ? 0.f : (mx - f) * bin_scale;
    return d < (float)(SA_BINS - 1) ? (int)d : SA_BINS - 1;
  };

  // `thr`: keys above it are in; of the keys equal to it the first `thr_ties` in index order.
  uint32_t thr = 0;
  unsigned long long thr_ties = ~0ull;
  int buf = 0;  // histogram buffer of the next level (the other one may still be read by a neighbour)

  // Tightens (thr, thr_ties) to the shortest prefix of the order that reaches `need` of the measure: elements
  // (MASS = false) or fixed-point mass (true; then frac >= 0 asks for need = ceil(frac * total)). Keys at or above
  // thr take part, those equal to it as a lump of thr_ties elements.
  auto select = [&](bool mass, unsigned long long need, double frac) {
    uint32_t klo = thr, khi = 0xffffffffu;  // keys still in question: [klo, khi]
    unsigned long long above = 0;
    int level = 0, shift = 0;
    const uint32_t thr0 = thr;
    const unsigned long long ties0 = thr_ties;
    for (;;) {
      uint32_t *cnt = s.cnt[buf], *lo = s.lo[buf], *hi = s.hi[buf];
      auto add = [&](int bin, unsigned long long m) {
        const uint32_t ml = (uint32_t)m, mh = (uint32_t)(m >> 32);
        if (!mass) {
          atomicAdd(&cnt[bin], ml);
          return;
        }
        uint32_t carry = mh;
        if (ml) {
          const uint32_t old = atomicAdd(&lo[bin], ml);
          carry += (old + ml < old) ? 1u : 0u;
        }
        if (carry) atomicAdd(&hi[bin], carry);
      };
      for (int v = t; v < nv; v += SA_T) {
        const uint4 q = stage[v];
        const raw *qr = reinterpret_cast<const raw *>(&q);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const uint32_t k = key_of<E>(qr[j]);
          if (k == 0 || k < klo || k > khi) continue;
          if (k == thr0 && ties0 != ~0ull) continue;  // the lump below
          const float f = value_of<E>(k);
          const int bin = level == 0 ? bin_of(f) : (int)((khi - k) >> shift);
          add(bin, mass ? fixed(weight(f)) : 1ull);
        }
      }
      if (ties0 != ~0ull && rank == 0 && t == 0 && thr0 >= klo && thr0 <= khi) {
        const float f = value_of<E>(thr0);
        add(level == 0 ? bin_of(f) : (int)((khi - thr0) >> shift), mass ? fixed(weight(f)) * ties0 : ties0);
      }
      cl.sync();
      // totals of this thread's two bins over the cluster, then a block scan to find the crossing
      unsigned long long m[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 2; ++j)
        for (int c = 0; c < C; ++c) {
          const SampleShared *o = cl.map_shared_rank(&s, c);
          m[j] += mass ? ((unsigned long long)o->hi[buf][2 * t + j] << 32) + o->lo[buf][2 * t + j]
                       : o->cnt[buf][2 * t + j];
        }
      unsigned long long run = m[0] + m[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long r2 = shfl_up64(run, o);
        if (lane >= o) run += r2;
      }
      if (lane == 31) s.scan[wp] = run;
      __syncthreads();
      unsigned long long before = 0, total = 0;
      for (int w = 0; w < SA_W; ++w) {
        if (w < wp) before += s.scan[w];
        total += s.scan[w];
      }
      if (level == 0) {
        if (frac >= 0.0) {
          const double want = ceil(frac * (double)total);
          need = want < 1.0 ? 1ull : (unsigned long long)want;
        }
        if (need > total) need = total;
      }
      run += before - (m[0] + m[1]) + above;  // measure above this thread's first bin
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (run < need && need <= run + m[j]) {  // exactly one bin of the block
          s.bin = 2 * t + j;
          s.above = run;
          s.in_bin = m[j];
        }
        run += m[j];
      }
      __syncthreads();
      const int bin = s.bin;
      above = s.above;
      // the other buffer is free again (every block has passed the cluster barrier above): clear it for the next level
      for (int i = t; i < SA_BINS; i += SA_T) s.cnt[buf ^ 1][i] = s.lo[buf ^ 1][i] = s.hi[buf ^ 1][i] = 0;
      if (level > 0 && shift == 0) {  // one key
        const uint32_t k = khi - (uint32_t)bin;
        if (mass) {
          const unsigned long long w = fixed(weight(value_of<E>(k)));
          thr_ties = (need - above + w - 1) / w;
        } else {
          thr_ties = need - above;
        }
        thr = k;
        buf ^= 1;
        __syncthreads();
        return;
      }
      // the keys of the bin: their smallest and largest, over the cluster
      uint32_t mn = 0xffffffffu, mk = 0;
      if (level == 0) {
        for (int v = t; v < nv; v += SA_T) {
          const uint4 q = stage[v];
          const raw *qr = reinterpret_cast<const raw *>(&q);
#pragma unroll
          for (int j = 0; j < PER; ++j) {
            const uint32_t k = key_of<E>(qr[j]);
            if (k == 0 || k < klo) continue;
            if (bin_of(value_of<E>(k)) != bin) continue;
            mn = min(mn, k);
            mk = max(mk, k);
          }
        }
        mn = __reduce_min_sync(0xffffffffu, mn);
        mk = __reduce_max_sync(0xffffffffu, mk);
        if (lane == 0) {
          atomicMin(&s.kmin[mass], mn);
          atomicMax(&s.kmax[mass], mk);
        }
        cl.sync();
        mn = 0xffffffffu;
        mk = 0;
        for (int c = 0; c < C; ++c) {
          const SampleShared *o = cl.map_shared_rank(&s, c);
          mn = min(mn, o->kmin[mass]);
          mk = max(mk, o->kmax[mass]);
        }
        klo = max(klo, mn);
        khi = mk;
      } else {
        const uint32_t top = khi - ((uint32_t)bin << shift);
        const uint32_t span = (1u << shift) - 1;
        klo = max(klo, top >= span ? top - span : 0u);
        khi = top;
      }
      shift = max(0, 32 - __clz(khi - klo) - 10);
      ++level;
      buf ^= 1;
      __syncthreads();
    }
  };

  if (top_k > 0 && top_k < a.V) select(false, (unsigned long long)top_k, -1.0);
  if (top_p < 1.f) select(true, 1ull, fmax(0.0, (double)top_p));
  const double mp = min_p > 0.f ? fmin((double)min_p, 1.0) : 0.0;

  // The draw. Warp w of block r holds a contiguous run of pieces, so warps in (block, warp) order are in index order.
  // Per warp: the mass above the threshold key, and how many equal it (all of one weight: the kept ones among them
  // follow from the number of ties before the warp).
  const float thr_v = value_of<E>(thr);
  const double thr_wd = thr ? weight(thr_v) : 0.0;
  const unsigned long long thr_w = (thr && thr_wd >= mp) ? fixed(thr_wd) : 0ull;
  const int per_warp = (nv + SA_W - 1) / SA_W;
  const int w0 = min(wp * per_warp, nv), w1 = min(w0 + per_warp, nv);
  auto kept = [&](uint32_t k) -> unsigned long long {  // weight of a key above the threshold, else 0
    if (k <= thr) return 0ull;
    const double w = weight(value_of<E>(k));
    return w >= mp ? fixed(w) : 0ull;
  };
  unsigned long long m = 0;
  uint32_t ties = 0;
  for (int v = w0 + lane; v < w1; v += 32) {
    const uint4 q = stage[v];
    const raw *qr = reinterpret_cast<const raw *>(&q);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint32_t k = key_of<E>(qr[j]);
      m += kept(k);
      ties += (k == thr && thr) ? 1u : 0u;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    m += __shfl_xor_sync(0xffffffffu, m, o);
    ties += __shfl_xor_sync(0xffffffffu, ties, o);
  }
  if (lane == 0) {
    s.mass[wp] = m;
    s.ties[wp] = ties;
  }
  cl.sync();
  // every warp walks the cluster's warps in order: 32 at a time
  unsigned long long my_before = 0, tie_before = 0, total = 0, my_mass = 0;
  {
    unsigned long long tie_run = 0;
    for (int c0 = 0; c0 < C * SA_W; c0 += 32) {
      const int id = c0 + lane;
      unsigned long long mm = 0, tt = 0;
      if (id < C * SA_W) {
        const SampleShared *o = cl.map_shared_rank(&s, id / SA_W);
        mm = o->mass[id % SA_W];
        tt = o->ties[id % SA_W];
      }
      unsigned long long ts = tt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long r2 = shfl_up64(ts, o);
        if (lane >= o) ts += r2;
      }
      const unsigned long long tb = tie_run + ts - tt;  // ties before this warp
      const unsigned long long tk = tb >= thr_ties ? 0ull : (tt < thr_ties - tb ? tt : thr_ties - tb);
      mm += tk * thr_w;
      unsigned long long ms = mm;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long r2 = shfl_up64(ms, o);
        if (lane >= o) ms += r2;
      }
      const int mine = rank * SA_W + wp - c0;
      if (mine >= 0 && mine < 32) {
        my_before = total + __shfl_sync(0xffffffffu, ms - mm, mine);
        tie_before = __shfl_sync(0xffffffffu, tb, mine);
        my_mass = __shfl_sync(0xffffffffu, mm, mine);
      }
      tie_run += __shfl_sync(0xffffffffu, ts, 31);
      total += __shfl_sync(0xffffffffu, ms, 31);
    }
  }
  const double du = fmin(fmax((double)__ldcg(a.u + row), 0.0), 1.0);  // a NaN counts as 0
  unsigned long long target = (unsigned long long)(du * (double)total);
  if (target >= total) target = total - 1;  // total >= 1: the largest weight is kept
  if (my_before <= target && target < my_before + my_mass) {  // one warp of the cluster
    unsigned long long run = my_before, tie_run = tie_before;
    bool found = false;
    for (int vb = w0; vb < w1 && !found; vb += 32) {
      const int v = vb + lane;
      uint32_t k[PER];
      unsigned long long tt = 0;
      if (v < w1) {
        const uint4 q = stage[v];
        const raw *qr = reinterpret_cast<const raw *>(&q);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          k[j] = key_of<E>(qr[j]);
          tt += (k[j] == thr && thr) ? 1u : 0u;
        }
      } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) k[j] = 0;
      }
      unsigned long long ts = tt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long r2 = shfl_up64(ts, o);
        if (lane >= o) ts += r2;
      }
      unsigned long long tb = tie_run + ts - tt, mm = 0, w[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        w[j] = kept(k[j]);
        if (k[j] == thr && thr) {
          if (tb < thr_ties) w[j] = thr_w;
          ++tb;
        }
        mm += w[j];
      }
      unsigned long long ms = mm;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long r2 = shfl_up64(ms, o);
        if (lane >= o) ms += r2;
      }
      unsigned long long at = run + ms - mm;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (at <= target && target < at + w[j]) {
          finish((v0 + v) * PER - skew + j);
          found = true;
        }
        at += w[j];
      }
      found = __any_sync(0xffffffffu, found);
      run += __shfl_sync(0xffffffffu, ms, 31);
      tie_run += __shfl_sync(0xffffffffu, ts, 31);
    }
  }
  cl.sync();
}

template <class E>
cudaError_t launch(const SampleArgs &a, int B, bool pdl, cudaStream_t st) {
  constexpr int PER = 16 / (int)sizeof(typename E::raw);
  static std::atomic<int> attr_set[64];  // the shared-memory opt-in, once per device
  int dev = 0;
  if (const cudaError_t e = cudaGetDevice(&dev)) return e;
  if (dev < 64 && !attr_set[dev].load(std::memory_order_acquire)) {
    if (const cudaError_t e =
            cudaFuncSetAttribute(sample_kernel<E>, cudaFuncAttributeMaxDynamicSharedMemorySize, SA_MAX_STAGE))
      return e;
    attr_set[dev].store(1, std::memory_order_release);
  }
  const int NV = (a.V + 2 * PER - 2) / PER;  // pieces of a row at the worst skew
  // Blocks per row: as many as its bytes need, then doubled while the batch leaves SMs idle.
  int C = 1;
  while (C < SA_MAX_C && ((NV + C - 1) / C) * 16 > SA_MAX_STAGE) C *= 2;
  while (C < SA_MAX_C && 2 * C * B <= device_sm_count() && NV > 2 * C * SA_T) C *= 2;
  const int per_block = (NV + C - 1) / C;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = pdl_config(dim3((unsigned)(B * C)), dim3(SA_T), pdl, st, attr);
  attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
  attr[cfg.numAttrs].val.clusterDim.x = C;
  attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
  ++cfg.numAttrs;
  cfg.dynamicSmemBytes = (size_t)per_block * 16;
  return cudaLaunchKernelEx(&cfg, sample_kernel<E>, a, per_block);
}

}  // namespace

cudaError_t launch_sample_next(const void *logits, int dtype, long long stride, const float *temperature,
                               const int *top_k, const float *top_p, const float *min_p, const float *u, int64_t *tok,
                               int64_t *pos, int B, int V, bool pdl, cudaStream_t st) {
  const SampleArgs a{logits, stride, temperature, top_k, top_p, min_p, u, tok, pos, V};
  if (dtype == 0) return launch<B16>(a, B, pdl, st);
  if (dtype == 1) return launch<H16>(a, B, pdl, st);
  return launch<F32>(a, B, pdl, st);
}

}  // namespace lfm2q
