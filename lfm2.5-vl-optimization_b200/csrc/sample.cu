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
// A cluster of C thread blocks holds one row in shared memory, read once. A histogram of counts (1024 bins linear in x,
// so that a peaked row spreads over them) shows where the cut must lie: with top_k its bin, exactly; with top_p alone the
// bin where the counts times the bins' middle weights cross. The elements from there on (top_k: down to the bin) or
// within a few bins of it (top_p) go into a list of at most 2048, one pass sums the weights of the others, and block 0
// sorts the list and finds the cut in it. Where the list would be longer (thousands of equal logits, a larger top_k), or
// the sums show that the cut lies outside it, the row is done again by exact histograms: level by level, 1024 bins of
// the order-preserving integer key inside the chosen bin, until a bin is one key.
//
// What bounds it: instructions, against 2 to 4 bytes to load an element, and the latency of a row's phases (the cluster's
// four barriers and the sort, some microseconds). 256 rows of 65536, in issue slots an element by counter: 132 in fp32 with
// a nucleus alone (loads and maximum, counts, weights; 20 of them fp64), 75 in bf16 unfiltered (no counts), 47 in bf16 with
// a top_k of 50 (no weights). They take 121 us (0.55 TB/s), 65 us and 43 us; two blocks an SM issue 2.3 to 2.4 instructions
// a clock, the fp64 pipe is 18 %, 32 % and 1 % busy. min_p alone weighs every element too, 65 us. One row in bf16 10.7 us.
// The list replaces an exact histogram over the whole row, several passes. Rows that still take them: 16 with a top_k of
// 5000 39 us; 256 with a top_k of 50 at a temperature so low (0.05) that fewer tokens than that lie within 46 binary
// orders of the largest 139 us. The other blocks leave before the list is sorted, so the next row starts on their SMs
// (124 -> 120 us), and the whole block searches the piece that holds the token (120 -> 117; a warp did it before).
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
constexpr int SA_STAGE = 65 * 1024;     // bytes of a row that one block stages (so that two blocks share an SM) ...
constexpr int SA_MAX_STAGE = 160 * 1024;  // ... and at most
constexpr int SA_LIST = 2048;           // elements around the cut
constexpr int SA_FEW = 128;             // a list (with top_k) that is compared pair by pair
constexpr int SA_IDX_BITS = 18;

// Element types: raw storage, an order-preserving key (equal keys <=> equal values: -0 takes +0's) and its inverse.
// Key 0 is a filler, below every value (it would be a negative NaN; rows with a NaN never get here).
// max2: the larger of each element of two words, a NaN if there is one.
struct B16 {
  typedef unsigned short raw;
  static constexpr int KEY_BITS = 16;
  static constexpr uint32_t LOWEST = 0xff80ff80u;
  static __device__ __forceinline__ float up(raw r) { return __uint_as_float((uint32_t)r << 16); }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
};
struct H16 {
  typedef unsigned short raw;
  static constexpr int KEY_BITS = 16;
  static constexpr uint32_t LOWEST = 0xfc00fc00u;
  static __device__ __forceinline__ float up(raw r) { return __half2float(__ushort_as_half(r)); }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
};
struct F32 {
  typedef uint32_t raw;
  static constexpr int KEY_BITS = 32;
  static constexpr uint32_t LOWEST = 0xff800000u;
  static __device__ __forceinline__ float up(raw r) { return __uint_as_float(r); }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.NaN.f32 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
};
template <class E>
__device__ __forceinline__ float top_of(uint32_t m) {  // of a word's elements
  if (sizeof(typename E::raw) == 4) return E::up((typename E::raw)m);
  const float lo = E::up((typename E::raw)(m & 0xffffu)), hi = E::up((typename E::raw)(m >> 16));
  return lo != lo ? lo : hi != hi ? hi : fmaxf(lo, hi);
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
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

struct SampleShared {
  float best[SA_W];
  float row_best;  // this block's maximum, and the first index of the row's in it: read by the cluster
  int row_at;
  unsigned long long scan[2][SA_W];
  float2 bins[SA_W];  // per warp: counts (as bits) and masses of its bins
  unsigned long long mass[SA_W];  // per warp: kept mass above the list (the exact path: above the threshold key)
  uint32_t ties[SA_W];            // exact path, per warp: elements equal to the threshold key
  unsigned long long all, above;  // this block's whole mass, and its mass above the list
  uint32_t kmin[2], kmax[2];      // exact path: [0] the selection by count, [1] by mass
  int n_list, again;              // list elements of this block; do the row by exact histograms
  // broadcast within the block
  int bin, cut;
  unsigned long long before, in_bin;
  union {
    struct {
      uint32_t cnt[SA_BINS];               // this block's counts
      int frac[SA_BINS];                   // and, in 2^-12, the sum of how far from the bins' middles they lie
      uint32_t cum[SA_BINS];               // the cluster's counts, summed up
      unsigned long long key[SA_LIST];     // the list: key, then lowest index first
      unsigned long long pre[SA_LIST];     // running weights of the sorted list
      unsigned long long warps[SA_MAX_C * SA_W];
    } f;
    struct {
      uint32_t cnt[2][SA_BINS], lo[2][SA_BINS], hi[2][SA_BINS];
    } h;
  };
};

// adds v to a word of shared memory, OFF bytes from addr, where `in`; without a branch (64 rows with a top_k of 100: 20.0 us
// with branches, 18.6 so)
template <int OFF>
__device__ __forceinline__ void add_if(bool in, uint32_t addr, uint32_t v) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %0, 0;\n\t@p red.shared.add.u32 [%1 + %3], %2;\n\t}" ::"r"((int)in),
               "r"(addr), "r"(v), "n"(OFF));  // (no clobber: loads may pass it, the barriers do not)
}
__device__ __forceinline__ unsigned long long shfl_up64(unsigned long long v, int o) {
  return __shfl_up_sync(0xffffffffu, v, o);
}

// Weights of a row. 2^z for z in [-50, 0]: z = n + r with r in [-1/2, 1/2] by adding and subtracting 1.5 2^52 (n is in
// the sum's low bits), 2^r = 1 + r q(r), q the Chebyshev interpolant of degree 9 of (2^r - 1) / r on that interval
// (computed in 60 digits; its relative error is below 2^-50), n added to the exponent.
struct Weigher {
  float mx;
  double dmx, c;  // the maximum, log2 e / T
  __device__ __forceinline__ double operator()(float f) const {
    const double z = ((double)f - dmx) * c;
    return f == mx ? 1.0 : z > -50.0 ? power(z) : 0.0;  // (also 0 where an infinite T meets an infinite logit)
  }
  // the same (2^-60 for 0) for a finite maximum and temperature, without a branch: several chains of these interleave
  __device__ __forceinline__ double finite(float f) const { return power(fmax(((double)f - dmx) * c, -60.0)); }
  static __device__ __forceinline__ double power(double z) {
    const double big = 6755399441055744.0, t = z + big, r = z - (t - big);
    double q = 7.070977866508139e-09;
    q = fma(q, r, 1.0205905413765595e-07);
    q = fma(q, r, 1.3215451633221434e-06);
    q = fma(q, r, 1.5252672924850737e-05);
    q = fma(q, r, 0.00015403530424776529);
    q = fma(q, r, 0.0013333558200794592);
    q = fma(q, r, 0.009618129107618665);
    q = fma(q, r, 0.05550410866465167);
    q = fma(q, r, 0.24022650695910075);
    q = fma(q, r, 0.6931471805599462);
    q = fma(q, r, 1.0);
    return __hiloint2double(__double2hiint(q) + (__double2loint(t) << 20), __double2loint(q));
  }
  // in steps of 2^-44, to nearest: the low bits of w + 2^8
  static __device__ __forceinline__ unsigned long long fixed(double w) {
    return (unsigned long long)(__double_as_longlong(w + 256.0) - __double_as_longlong(256.0));
  }
};
// Level 0 bins: linear in x, monotone, bin i around 2^(-46 i / 1024) of the largest weight; the last one takes all that
// weighs less than 2^-45.9. The maximum is finite. The place on that line plus 2^23 rounds to the bin, its low bits. Which
// bin an element falls into, and whether it is one before the last, is decided here alone: the list is sized by the counts
// of one pass and filled by the next, which has to see the same bins.
constexpr float SA_RND = 8388608.f, SA_TO_INT = 12582912.f;
struct Binner {
  float mx, scale;
  // 2^23 + bin. The roundings are spelt out, for the compiler may fuse a * b + c in one place and not in another, which
  // moves an element next to a bin's edge.
  __device__ __forceinline__ float rounded(float f) const { return __fmaf_rn(__fsub_rn(mx, f), scale, SA_RND); }
  // how far f lies from the middle of its bin, in bins
  __device__ __forceinline__ float off(float f, float rnd) const { return fmaf(mx - f, scale, SA_RND - rnd); }
  static __device__ __forceinline__ bool early(float rnd) { return rnd < SA_RND + (float)(SA_BINS - 1); }  // (no NaN)
  __device__ __forceinline__ int operator()(float f) const {
    const float rnd = rounded(f);
    return early(rnd) ? __float_as_int(rnd) - __float_as_int(SA_RND) : SA_BINS - 1;
  }
};
// What a block of the cluster has of the row.
struct RowPart {
  const uint4 *stage;
  int v0, nv, skew, per_block, NV;
};
struct Params {
  float min_p, top_p, u;
  int top_k;
};

// sum over the block's warps before this one, and in all, of per-thread values already scanned within the warp
__device__ __forceinline__ void block_offsets(unsigned long long last, unsigned long long *slots,
                                              unsigned long long &before, unsigned long long &total) {
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  if (lane == 31) slots[wp] = last;
  __syncthreads();
  before = total = 0;
#pragma unroll
  for (int w = 0; w < SA_W; ++w) {
    const unsigned long long v = slots[w];
    if (w < wp) before += v;
    total += v;
  }
}
__device__ __forceinline__ unsigned long long warp_scan(unsigned long long v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long r = shfl_up64(v, o);
    if (lane >= o) v += r;
  }
  return v;
}
// what(block of the cluster) for every block, all in flight together (a load from another block's shared memory takes
// some 700 cycles)
template <class V, class F>
__device__ __forceinline__ void of_cluster(cg::cluster_group &cl, SampleShared *s, V (&v)[SA_MAX_C], V none, F what) {
  const int C = (int)cl.num_blocks();
#pragma unroll
  for (int c = 0; c < SA_MAX_C; ++c) v[c] = c < C ? what(cl.map_shared_rank(s, c)) : none;
}

// Bitonic sort, descending, of N keys (a power of two >= 64) in shared memory by the whole block: strides up to 32 within
// a warp's 64 keys (two a lane), longer ones through shared memory. Ends with a barrier.
__device__ __forceinline__ void sort_chunk(unsigned long long *key, int base, int k0, int k1) {
  const int lane = threadIdx.x & 31;
  unsigned long long x[2] = {key[base + lane], key[base + 32 + lane]};
  for (int k = k0; k <= k1; k *= 2) {
    if (k >= 64) {  // stride 32: the lane's own two
      const bool down = (base & k) == 0;
      if ((x[0] < x[1]) == down) {
        const unsigned long long y = x[0];
        x[0] = x[1];
        x[1] = y;
      }
    }
    for (int j = min(k / 2, 16); j > 0; j /= 2)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned long long y = __shfl_xor_sync(0xffffffffu, x[h], j);
        const bool larger = ((lane & j) == 0) == (((base + 32 * h + lane) & k) == 0);
        x[h] = (x[h] > y) == larger ? x[h] : y;
      }
  }
  key[base + lane] = x[0];
  key[base + 32 + lane] = x[1];
}
__device__ __forceinline__ void sort_keys(unsigned long long *key, int N) {
  const int t = threadIdx.x, wp = t >> 5;
  for (int base = 64 * wp; base < N; base += 64 * SA_W) sort_chunk(key, base, 2, 64);
  __syncthreads();
  for (int k = 128; k <= N; k *= 2) {
    for (int j = k / 2; j >= 64; j /= 2) {
      for (int i = t; i < N / 2; i += SA_T) {
        const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
        const unsigned long long p = key[lo], q = key[hi];
        if ((p < q) == ((lo & k) == 0)) {
          key[lo] = q;
          key[hi] = p;
        }
      }
      __syncthreads();
    }
    for (int base = 64 * wp; base < N; base += 64 * SA_W) sort_chunk(key, base, k, k);
    __syncthreads();
  }
}

__device__ __forceinline__ unsigned long long target_of(float u, unsigned long long total) {
  const double du = fmin(fmax((double)u, 0.0), 1.0);  // a NaN counts as 0
  const unsigned long long t = (unsigned long long)(du * (double)total);
  return t < total ? t : total - 1;  // total >= 1: the largest weight is kept
}
__device__ __forceinline__ unsigned long long mass_needed(float p, unsigned long long total) {
  const double want = ceil(fmax(0.0, (double)p) * (double)total);
  return want < 1.0 ? 1ull : min((unsigned long long)want, total);
}

// The list of a row with a top_k, n <= SA_FEW: all that is kept is in it, so the token is too. Every element is compared
// with every other, by as many threads as there are for one, which gives its place in the order of keys and in that of
// indexes; one warp then sums in both orders. In place of the sort, sums over the block and a second look at the row, each
// of them barriers and chains (one row with a top_k of 50: 13.3 -> 10.5 us, 64 with 100: 23.2 -> 20.0, 256 with 50: 51.9 -> 42.6).
template <class E, class F>
__device__ __forceinline__ void draw_few(SampleShared &s, int n, const Weigher &weigh, double mp, bool use_p,
                                         const Params &par, F finish) {
  constexpr unsigned INDEX = (1 << SA_IDX_BITS) - 1, HIGH = 1u << 31;
  constexpr int EACH = SA_FEW / 32;
  const int t = threadIdx.x, lane = t & 31, lg = min(5, 31 - __clz(SA_T / n)), many = 1 << lg;  // threads an element
  const int i = t >> lg, sub = t & (many - 1);
  const unsigned long long key = i < n ? s.f.key[i] : 0;
  const unsigned low = (unsigned)key & INDEX;
  int rank = 0, place = 0;
#pragma unroll 4
  for (int j = sub; j < n; j += many) {
    const unsigned long long k = s.f.key[j];
    rank += k > key;
    place += ((unsigned)k & INDEX) > low;  // (the low bits fall as the index rises)
  }
  for (int o = 1; o < many; o <<= 1) {
    rank += __shfl_xor_sync(0xffffffffu, rank, o);
    place += __shfl_xor_sync(0xffffffffu, place, o);
  }
  if (i < n && sub == 0) {
    const double w = weigh(value_of<E>((uint32_t)(key >> SA_IDX_BITS)));
    s.f.pre[rank] = rank < par.top_k ? Weigher::fixed(w) : 0;
    s.f.cum[rank] = place | (w >= mp ? HIGH : 0u);
    s.f.cnt[place] = INDEX - low;
  }
  __syncthreads();
  if (t >= 32) return;
  unsigned long long w[EACH], run = 0;
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    w[j] = EACH * lane + j < n ? s.f.pre[EACH * lane + j] : 0;
    run += w[j];
  }
  unsigned long long sum = warp_scan(run);
  run = sum - run;
  const unsigned long long need = use_p ? mass_needed(par.top_p, __shfl_sync(0xffffffffu, sum, 31)) : ~0ull;
#pragma unroll
  for (int j = 0; j < EACH; ++j)
    if (EACH * lane + j < n) {
      const uint32_t at = s.f.cum[EACH * lane + j];
      s.f.key[at & ~HIGH] = run < need && at & HIGH ? w[j] : 0;
      run += w[j];
    }
  __syncwarp();
  run = 0;
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    w[j] = EACH * lane + j < n ? s.f.key[EACH * lane + j] : 0;
    run += w[j];
  }
  sum = warp_scan(run);
  run = sum - run;
  const unsigned long long target = target_of(par.u, __shfl_sync(0xffffffffu, sum, 31));
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    if (run <= target && target < run + w[j]) finish((int)s.f.cnt[EACH * lane + j]);
    run += w[j];
  }
}

// The row by exact histograms: for any number of ties and any top_k. All blocks of the cluster; the token comes out of
// one lane of one block (the others return -1).
template <class E>
__device__ __noinline__ int sample_exact(cg::cluster_group cl, SampleShared &s, const RowPart row, const Weigher weigh,
                                         const Binner bins, const Params par, int V) {
  typedef typename E::raw raw;
  constexpr int PER = 16 / (int)sizeof(raw);
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int t = threadIdx.x, lane = t & 31, wp = t >> 5;
  int token = -1;
  auto finish = [&](int i) { token = i; };
  for (int i = t; i < 2 * SA_BINS; i += SA_T) (&s.h.cnt[0][0])[i] = (&s.h.lo[0][0])[i] = (&s.h.hi[0][0])[i] = 0;
  if (t < 2) {
    s.kmin[t] = 0xffffffffu;
    s.kmax[t] = 0;
  }
  __syncthreads();

  // `thr`: keys above it are in; of the keys equal to it the first `thr_ties` in index order.
  uint32_t thr = 0;
  unsigned long long thr_ties = ~0ull;
  int buf = 0;  // histogram buffer of the next level (the other one may still be read by a neighbour)

  // Tightens (thr, thr_ties) to the shortest prefix of the order that reaches `need` of the measure: elements
  // (MASS = false) or fixed-point mass (true; then frac >= 0 asks for need = ceil(frac * total)). Keys at or above
  // thr take part, those equal to it as a lump of thr_ties elements.
  auto select = [&](bool mass, unsigned long long need, float frac) {
    uint32_t klo = thr, khi = 0xffffffffu;  // keys still in question: [klo, khi]
    unsigned long long above = 0;
    int level = 0, shift = 0;
    const uint32_t thr0 = thr;
    const unsigned long long ties0 = thr_ties;
    for (;;) {
      uint32_t *cnt = s.h.cnt[buf], *lo = s.h.lo[buf], *hi = s.h.hi[buf];
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
      for (int v = t; v < row.nv; v += SA_T) {
        const uint4 q = row.stage[v];
        const raw *qr = reinterpret_cast<const raw *>(&q);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const uint32_t k = key_of<E>(qr[j]);
          if (k == 0 || k < klo || k > khi) continue;
          if (k == thr0 && ties0 != ~0ull) continue;  // the lump below
          const float f = value_of<E>(k);
          const int bin = level == 0 ? bins(f) : (int)((khi - k) >> shift);
          add(bin, mass ? Weigher::fixed(weigh(f)) : 1ull);
        }
      }
      if (ties0 != ~0ull && rank == 0 && t == 0 && thr0 >= klo && thr0 <= khi) {
        const float f = value_of<E>(thr0);
        add(level == 0 ? bins(f) : (int)((khi - thr0) >> shift), mass ? Weigher::fixed(weigh(f)) * ties0 : ties0);
      }
      cl.sync();
      // totals of this thread's two bins over the cluster, then a block scan to find the crossing
      unsigned long long m[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 2; ++j)
        for (int c = 0; c < C; ++c) {
          const SampleShared *o = cl.map_shared_rank(&s, c);
          m[j] += mass ? ((unsigned long long)o->h.hi[buf][2 * t + j] << 32) + o->h.lo[buf][2 * t + j]
                       : o->h.cnt[buf][2 * t + j];
        }
      unsigned long long run = m[0] + m[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long r2 = shfl_up64(run, o);
        if (lane >= o) run += r2;
      }
      if (lane == 31) s.scan[0][wp] = run;
      __syncthreads();
      unsigned long long before = 0, total = 0;
      for (int w = 0; w < SA_W; ++w) {
        if (w < wp) before += s.scan[0][w];
        total += s.scan[0][w];
      }
      if (level == 0) {
        if (frac >= 0.f) {
          need = mass_needed(frac, total);
        }
        if (need > total) need = total;
      }
      run += before - (m[0] + m[1]) + above;  // measure above this thread's first bin
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (run < need && need <= run + m[j]) {  // exactly one bin of the block
          s.bin = 2 * t + j;
          s.before = run;
          s.in_bin = m[j];
        }
        run += m[j];
      }
      __syncthreads();
      const int bin = s.bin;
      above = s.before;
      // the other buffer is free again (every block has passed the cluster barrier above): clear it for the next level
      for (int i = t; i < SA_BINS; i += SA_T) s.h.cnt[buf ^ 1][i] = s.h.lo[buf ^ 1][i] = s.h.hi[buf ^ 1][i] = 0;
      if (level > 0 && shift == 0) {  // one key
        const uint32_t k = khi - (uint32_t)bin;
        if (mass) {
          const unsigned long long w = Weigher::fixed(weigh(value_of<E>(k)));
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
        for (int v = t; v < row.nv; v += SA_T) {
          const uint4 q = row.stage[v];
          const raw *qr = reinterpret_cast<const raw *>(&q);
#pragma unroll
          for (int j = 0; j < PER; ++j) {
            const uint32_t k = key_of<E>(qr[j]);
            if (k == 0 || k < klo) continue;
            if (bins(value_of<E>(k)) != bin) continue;
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

  if (par.top_k > 0 && par.top_k < V) select(false, (unsigned long long)par.top_k, -1.f);
  if (par.top_p < 1.f) select(true, 1ull, fmaxf(0.f, par.top_p));
  const double mp = par.min_p > 0.f ? fmin((double)par.min_p, 1.0) : 0.0;

  // The draw. Warp w of block r holds a contiguous run of pieces, so warps in (block, warp) order are in index order.
  // Per warp: the mass above the threshold key, and how many equal it (all of one weight: the kept ones among them
  // follow from the number of ties before the warp).
  const float thr_v = value_of<E>(thr);
  const double thr_wd = thr ? weigh(thr_v) : 0.0;
  const unsigned long long thr_w = (thr && thr_wd >= mp) ? Weigher::fixed(thr_wd) : 0ull;
  const int per_warp = (row.nv + SA_W - 1) / SA_W;
  const int w0 = min(wp * per_warp, row.nv), w1 = min(w0 + per_warp, row.nv);
  auto kept = [&](uint32_t k) -> unsigned long long {  // weight of a key above the threshold, else 0
    if (k <= thr) return 0ull;
    const double w = weigh(value_of<E>(k));
    return w >= mp ? Weigher::fixed(w) : 0ull;
  };
  unsigned long long m = 0;
  uint32_t ties = 0;
  for (int v = w0 + lane; v < w1; v += 32) {
    const uint4 q = row.stage[v];
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
  const unsigned long long target = target_of(par.u, total);
  if (my_before <= target && target < my_before + my_mass) {  // one warp of the cluster
    unsigned long long run = my_before, tie_run = tie_before;
    bool found = false;
    for (int vb = w0; vb < w1 && !found; vb += 32) {
      const int v = vb + lane;
      uint32_t k[PER];
      unsigned long long tt = 0;
      if (v < w1) {
        const uint4 q = row.stage[v];
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
          finish((row.v0 + v) * PER - row.skew + j);
          found = true;
        }
        at += w[j];
      }
      found = __any_sync(0xffffffffu, found);
      run += __shfl_sync(0xffffffffu, ms, 31);
      tie_run += __shfl_sync(0xffffffffu, ts, 31);
    }
  }
  return token;
}

template <class E>
__global__ void __launch_bounds__(SA_T, 2) sample_kernel(const SampleArgs a) {
  typedef typename E::raw raw;
  constexpr int PER = 16 / (int)sizeof(raw);  // elements of a 16-byte piece
  extern __shared__ __align__(16) uint8_t sa_smem[];
  __shared__ SampleShared s;
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int r = blockIdx.x / C;
  const int t = threadIdx.x, lane = t & 31, wp = t >> 5;
  pdl_trigger();
  for (int i = t; i < SA_BINS; i += SA_T) s.f.cnt[i] = s.f.frac[i] = 0;
  if (t == 0) s.n_list = s.again = 0;
  pdl_wait();

  // The row in 16-byte pieces of the address space: piece v holds elements v PER - skew .. + PER. Block `rank` stages
  // pieces [v0, v1), warp w of it a contiguous run of them; elements outside the row become fillers.
  const raw *x = reinterpret_cast<const raw *>(a.logits) + r * a.stride;
  const int skew = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(raw));
  const int NV = (a.V + skew + PER - 1) / PER;
  const int per_block = (NV + C - 1) / C;
  const int v0 = min(rank * per_block, NV), nv = min(v0 + per_block, NV) - v0;
  const int per_warp = (nv + SA_W - 1) / SA_W;
  const int w0 = min(wp * per_warp, nv), w1 = min(w0 + per_warp, nv);
  uint4 *stage = reinterpret_cast<uint4 *>(sa_smem);
  constexpr raw FILL = (raw)~(raw)0;
  constexpr int UN = 8;  // pieces in flight a thread
  uint32_t mw[4] = {E::LOWEST, E::LOWEST, E::LOWEST, E::LOWEST};
  float best = -INFINITY;
  for (int vb = w0 + lane; vb < w1; vb += 32 * UN) {
    uint4 q[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int v = vb + 32 * u, e0 = (v0 + v) * PER - skew;
      if (v >= w1) break;
      if (e0 >= 0 && e0 + PER <= a.V) {
        q[u] = ld_cg16(x + e0);
        continue;
      }
      raw *qr = reinterpret_cast<raw *>(&q[u]);  // a piece that the row only touches: at most two a row
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const bool in = e0 + j >= 0 && e0 + j < a.V;
        qr[j] = in ? __ldcg(x + e0 + j) : FILL;
        if (in) best = max_nan(best, E::up(qr[j]));
      }
      stage[v] = q[u];
      q[u] = make_uint4(E::LOWEST, E::LOWEST, E::LOWEST, E::LOWEST);
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int v = vb + 32 * u, e0 = (v0 + v) * PER - skew;
      if (v >= w1) break;
      if (e0 >= 0 && e0 + PER <= a.V) stage[v] = q[u];
      mw[0] = E::max2(mw[0], q[u].x);
      mw[1] = E::max2(mw[1], q[u].y);
      mw[2] = E::max2(mw[2], q[u].z);
      mw[3] = E::max2(mw[3], q[u].w);
    }
  }
  best = max_nan(best, top_of<E>(E::max2(E::max2(mw[0], mw[1]), E::max2(mw[2], mw[3]))));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max_nan(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) s.best[wp] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < SA_W; ++w) best = max_nan(best, s.best[w]);
  if (t == 0) {
    s.row_best = best;
    s.row_at = 0x7fffffff;
  }
  cl.sync();
  {
    float v[SA_MAX_C];
    of_cluster(cl, &s, v, -INFINITY, [](const SampleShared *o) { return o->row_best; });
#pragma unroll
    for (int c = 0; c < SA_MAX_C; ++c) best = max_nan(best, v[c]);
  }

  const float T = a.temperature ? __ldcg(a.temperature + r) : 1.f;
  Params par;
  par.top_p = a.top_p ? __ldcg(a.top_p + r) : 1.f;
  par.min_p = a.min_p ? __ldcg(a.min_p + r) : 0.f;
  par.top_k = a.top_k ? __ldcg(a.top_k + r) : 0;
  par.u = __ldcg(a.u + r);
  auto finish = [&](int token) {
    a.tok[r] = token;
    if (a.pos && r == 0) a.pos[0] = __ldcg(reinterpret_cast<const long long *>(a.pos)) + 1;
  };
  // greedy, a NaN, nothing but -inf, or only one token kept: the first largest
  if (!(T > 0.f) || best != best || best == -INFINITY || par.top_k == 1) {
    int at = 0x7fffffff;
    for (int v = w0 + lane; v < w1 && at == 0x7fffffff; v += 32) {
      const uint4 q = stage[v];
      const raw *qr = reinterpret_cast<const raw *>(&q);
#pragma unroll
      for (int j = PER - 1; j >= 0; --j) {
        const int e = (v0 + v) * PER - skew + j;
        const float f = E::up(qr[j]);
        if (e >= 0 && e < a.V && (best != best ? f != f : f == best)) at = e;
      }
    }
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) atomicMin(&s.row_at, at);
    cl.sync();
    if (rank == 0 && t == 0) {
      for (int c = 0; c < C; ++c) at = min(at, cl.map_shared_rank(&s, c)->row_at);
      finish(at);
    }
    cl.sync();  // no block leaves while another may still read its shared memory
    return;
  }
  const Weigher weigh{best, (double)best, 1.4426950408889634 / (double)T};
  const Binner bins{best, (float)(1.4426950408889634 * (SA_BINS / 46.0)) / T};
  const double mp = par.min_p > 0.f ? fmin((double)par.min_p, 1.0) : 0.0;
  const bool use_k = par.top_k > 0 && par.top_k < a.V, use_p = par.top_p < 1.f;
  const RowPart part{stage, v0, nv, skew, per_block, NV};

  // ---------------------------------------------------------------- where the cut lies: bins [b_lo, b_hi]
  int b_lo = SA_BINS, b_hi = -1;  // no cut: everything is "above"
  uint32_t held = 0;              // elements in them
  // the exact histograms where the list would be too long, or where the bins and the branch-free weights would meet 0
  // times infinity: an infinite maximum, a temperature near 0 (every block finds the same)
  bool again = best == INFINITY || !(bins.scale < 1e30f);
  if ((use_k || use_p) && !again) {
    const uint32_t cnt0 = (uint32_t)__cvta_generic_to_shared(s.f.cnt) - 4 * __float_as_uint(SA_RND);
    for (int v = w0 + lane; v < w1; v += 32) {
      const uint4 q = stage[v];
      const raw *qr = reinterpret_cast<const raw *>(&q);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const float f = E::up(qr[j]), rnd = bins.rounded(f);
        const bool in = Binner::early(rnd);  // (a filler is a NaN)
        const uint32_t cnt = cnt0 + 4 * __float_as_uint(rnd);
        add_if<0>(in, cnt, 1);
        // the offset from the middle times 2^12, to an integer by adding 1.5 2^23, whose bits go once the counts are known
        if (!use_k)
          add_if<sizeof(s.f.cnt)>(in, cnt, __float_as_uint(fmaf(bins.off(f, rnd), 4096.f, SA_TO_INT)));
      }
    }
    cl.sync();
    // this thread's two bins over the cluster, summed up: the counts, and the masses to some 10^-5: an element at
    // d from its bin's middle weighs the middle's weight times 1 - h d + h^2 / 24 on average, h = 46 ln 2 / 1024
    uint32_t n[2] = {0, 0};
    int fr[2] = {0, 0};
    {
      uint2 v[SA_MAX_C];
      of_cluster(cl, &s, v, make_uint2(0, 0), [&](const SampleShared *o) {
        return *reinterpret_cast<const uint2 *>(&o->f.cnt[2 * t]);
      });
      int2 w[SA_MAX_C];
      of_cluster(cl, &s, w, make_int2(0, 0), [&](const SampleShared *o) {
        return use_k ? make_int2(0, 0) : *reinterpret_cast<const int2 *>(&o->f.frac[2 * t]);
      });
#pragma unroll
      for (int c = 0; c < SA_MAX_C; ++c) {
        n[0] += v[c].x;
        n[1] += v[c].y;
        fr[0] += w[c].x;
        fr[1] += w[c].y;
      }
      fr[0] -= n[0] * __float_as_uint(SA_TO_INT);  // (modulo 2^32; the sums themselves fit)
      fr[1] -= n[1] * __float_as_uint(SA_TO_INT);
    }
    constexpr float H = 0.69314718f * 46.f / SA_BINS;
    float m[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
      m[j] = fmaxf(0.f, exp2f(-(2 * t + j) * (46.f / SA_BINS)) * (n[j] * (1.f + H * H / 24) - fr[j] * (H / 4096)));
    uint32_t c1 = n[0] + n[1];
    float e1 = m[0] + m[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t c = __shfl_up_sync(0xffffffffu, c1, o);
      const float e = __shfl_up_sync(0xffffffffu, e1, o);
      if (lane >= o) {
        c1 += c;
        e1 += e;
      }
    }
    if (lane == 31) s.bins[wp] = make_float2(__uint_as_float(c1), e1);
    if (t == 0) s.bin = SA_BINS - 1;
    __syncthreads();
    float mass = 0.f;
#pragma unroll
    for (int w = 0; w < SA_W; ++w) {
      const float2 v = s.bins[w];
      if (w < wp) {
        c1 += __float_as_uint(v.x);
        e1 += v.y;
      }
      mass += v.y;
    }
    const uint32_t c0 = c1 - n[1];
    const float e0 = e1 - m[1];
    s.f.cum[2 * t] = c0;
    s.f.cum[2 * t + 1] = c1;
    if (use_k) {
      const uint32_t k = par.top_k;
      if (c0 - n[0] < k && k <= c0) s.bin = 2 * t;
      if (c0 < k && k <= c1) s.bin = 2 * t + 1;
    } else {
      // the bin that the wanted mass falls into, and its neighbour where it comes near the edge (rounding may leave the
      // mass to two bins or to none: any of them will do, the sums decide whether the cut is in the list)
      const float want = fmaxf(0.f, par.top_p) * mass, slack = 4e-5f * mass;
      const float lo[2] = {e0 - m[0], e0}, hi[2] = {e0, e1};
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (lo[j] <= want && want <= hi[j] && n[j])
          s.bin = (2 * t + j) | (want - lo[j] < slack ? 1 << 16 : 0) | (hi[j] - want < slack ? 1 << 17 : 0);
    }
    __syncthreads();
    const int at = s.bin & 0xffff;
    if (use_k) {
      b_lo = 0;
      b_hi = at;
      held = s.f.cum[at];
      again = at == SA_BINS - 1 || held > SA_LIST;
    } else {
      b_lo = max(0, at - (s.bin >> 16 & 1));
      b_hi = min(SA_BINS - 2, at + (s.bin >> 17 & 1));
      // (an empty neighbour holds nothing that could be cut: the next one with elements does)
      while (s.bin >> 16 & 1 && b_lo > 0 && s.f.cum[b_lo] == s.f.cum[b_lo - 1]) --b_lo;
      while (s.bin >> 17 & 1 && b_hi < SA_BINS - 2 && s.f.cum[b_hi] == s.f.cum[b_hi - 1]) ++b_hi;
      held = s.f.cum[b_hi] - (b_lo ? s.f.cum[b_lo - 1] : 0u);
      again = b_hi < b_lo || held > SA_LIST;
    }
  }

  if (!again) {
    // -------------------------------------------------------------- weights above the list, and the list
    unsigned long long all = 0, above = 0, kept = 0;
    const bool no_cut = !(use_k || use_p);
    const float r_lo = SA_RND + (float)b_lo, r_hi = SA_RND + (float)b_hi;
    constexpr int UN2 = 8 / PER;  // eight elements a step
    for (int vb = w0 + lane; vb < w1; vb += 32 * UN2) {
      float f[8];
      uint32_t listed = 0;
#pragma unroll
      for (int u = 0; u < UN2; ++u) {
        const bool in = vb + 32 * u < w1;
        const uint4 q = stage[in ? vb + 32 * u : vb];
        const raw *qr = reinterpret_cast<const raw *>(&q);
#pragma unroll
        for (int j = 0; j < PER; ++j) f[u * PER + j] = in ? E::up(qr[j]) : __int_as_float(0x7fffffff);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {  // (a filler is a NaN: it weighs nothing and lies in no bin)
        const float rnd = bins.rounded(f[j]);
        if (rnd >= r_lo && rnd <= r_hi) listed |= 1u << j;
      }
      if (!use_k) {
        double w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = weigh.finite(f[j]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const unsigned long long wf = Weigher::fixed(w[j]);
          all += wf;
          // (without a cut no bin is asked: a difference beyond the largest float has none, and may weigh something)
          if (no_cut || bins.rounded(f[j]) < r_lo) {
            above += wf;
            if (mp > 0.0 && w[j] >= mp) kept += wf;
          }
        }
      }
      for (; listed; listed &= listed - 1) {
        const int j = __ffs(listed) - 1, v = vb + 32 * (j / PER), k = j % PER;
        const raw x0 = reinterpret_cast<const raw *>(&stage[v])[k];
        const int slot = atomicAdd(&s.n_list, 1);
        if (slot < SA_LIST)  // (the counts say so too)
          s.f.key[slot] = (unsigned long long)key_of<E>(x0) << SA_IDX_BITS |
                          (unsigned)((1 << SA_IDX_BITS) - 1 - ((v0 + v) * PER - skew + k));
      }
    }
    if (mp == 0.0) kept = above;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      all += __shfl_xor_sync(0xffffffffu, all, o);
      above += __shfl_xor_sync(0xffffffffu, above, o);
      kept += __shfl_xor_sync(0xffffffffu, kept, o);
    }
    if (lane == 0) {
      s.mass[wp] = kept;
      s.scan[0][wp] = all;
      s.scan[1][wp] = above;
    }
    __syncthreads();
    if (t == 0) {
      unsigned long long x0 = 0, x1 = 0;
      for (int w = 0; w < SA_W; ++w) {
        x0 += s.scan[0][w];
        x1 += s.scan[1][w];
      }
      s.all = x0;
      s.above = x1;
    }
    cl.sync();
    // -------------------------------------------------------------- block 0 brings it together; the others are done
    int n = 0;
    unsigned long long M = 0, A = 0;
    if (rank == 0) {
      int from[SA_MAX_C];
      {
        of_cluster(cl, &s, from, 0, [](const SampleShared *o) { return o->n_list; });
        ulonglong2 v[SA_MAX_C];
        of_cluster(cl, &s, v, make_ulonglong2(0, 0),
                   [](const SampleShared *o) { return make_ulonglong2(o->all, o->above); });
        if (t < C * SA_W) s.f.warps[t] = cl.map_shared_rank(&s, t / SA_W)->mass[t % SA_W];
#pragma unroll
        for (int c = 0; c < SA_MAX_C; ++c) {
          M += v[c].x;
          A += v[c].y;
          const int nc = from[c];
          from[c] = n;  // where block c's part of the list goes; block 0's is there
          n += nc;
        }
      }
      const bool whole = n == (int)held;  // the list holds what was counted
      if (!whole) {
        n = 0;
        if (t < C) cl.map_shared_rank(&s, t)->again = 1;
      }
      for (int i = t; i < n; i += SA_T) {
        int c = 0;
#pragma unroll
        for (int k = 1; k < SA_MAX_C; ++k)
          if (k < C && i >= from[k]) c = k;
        int at = 0;
#pragma unroll
        for (int k = 0; k < SA_MAX_C; ++k)
          if (c == k) at = i - from[k];
        if (c > 0) s.f.key[i] = cl.map_shared_rank(&s, c)->f.key[at];
      }
      if (t == 0) s.cut = 0;
      __syncthreads();
      if (whole && use_p && !use_k) {  // does the cut lie in the list?
        unsigned long long sum = 0, before, total;
        for (int i = t; i < n; i += SA_T)
          sum += Weigher::fixed(weigh(value_of<E>((uint32_t)(s.f.key[i] >> SA_IDX_BITS))));
        block_offsets(warp_scan(sum), s.scan[0], before, total);
        const unsigned long long need = mass_needed(par.top_p, M);
        if (!(A < need && need <= A + total) && t < C) cl.map_shared_rank(&s, t)->again = 1;
      }
    }
    cl.sync();
    again = s.again != 0;
    if (!again) {
      if (rank != 0) return;
      if (use_k && n <= SA_FEW) {
        draw_few<E>(s, n, weigh, mp, use_p, par, finish);
        return;
      }
      // ------------------------------------------------------------ sort the list, find the cut, draw
      int N2 = 64;
      while (N2 < n) N2 *= 2;
      for (int i = n + t; i < N2; i += SA_T) s.f.key[i] = 0;
      __syncthreads();
      sort_keys(s.f.key, N2);  // (no two keys are equal: their indexes differ)
      constexpr int EACH = SA_LIST / SA_T;  // consecutive list elements a thread
      const int each = (n + SA_T - 1) / SA_T;
      unsigned long long wl[EACH], run = 0;
      bool high[EACH];
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        const int i = t * each + j;
        wl[j] = 0;
        high[j] = false;
        if (j < each && i < n) {
          const double w = weigh(value_of<E>((uint32_t)(s.f.key[i] >> SA_IDX_BITS)));
          wl[j] = Weigher::fixed(w);
          high[j] = w >= mp;
        }
        run += wl[j];
      }
      unsigned long long before, total;
      const unsigned long long scanned = warp_scan(run);
      block_offsets(scanned, s.scan[0], before, total);
      run = before + scanned - run;
#pragma unroll
      for (int j = 0; j < EACH; ++j)
        if (j < each && t * each + j < n) {
          run += wl[j];
          s.f.pre[t * each + j] = run;
        }
      __syncthreads();
      // the list's first `cut` elements are kept
      int limit = n;
      if (use_k) {
        limit = par.top_k;  // <= n
        M = s.f.pre[limit - 1];
      }
      const unsigned long long need = use_p ? mass_needed(par.top_p, M) : 0;
      if (use_p) {
        for (int i = t; i < limit; i += SA_T)
          if (A + (i ? s.f.pre[i - 1] : 0) < need && need <= A + s.f.pre[i]) s.cut = i + 1;
      } else if (t == 0) {
        s.cut = use_k ? limit : 0;
      }
      __syncthreads();
      const int cut = s.cut;
      const unsigned long long last = cut ? s.f.key[cut - 1] : 0;  // kept: this key or a higher one (0: all)
      // the kept list elements' weights to the warps that hold them
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        const int i = t * each + j;
        if (j < each && i < cut && high[j]) {
          const int e = (1 << SA_IDX_BITS) - 1 - (int)(s.f.key[i] & ((1 << SA_IDX_BITS) - 1));
          const int v = (e + skew) / PER, b = v / per_block, bv = min(per_block, NV - b * per_block);
          atomicAdd(&s.f.warps[b * SA_W + (v - b * per_block) / ((bv + SA_W - 1) / SA_W)], wl[j]);
        }
      }
      __syncthreads();
      if (wp == 0) {
        // the warp segment in which the running mass passes the target
        unsigned long long m[SA_MAX_C * SA_W / 32], mine = 0;
#pragma unroll
        for (int j = 0; j < SA_MAX_C * SA_W / 32; ++j) {
          const int i = lane * (SA_MAX_C * SA_W / 32) + j;
          m[j] = i < C * SA_W ? s.f.warps[i] : 0;
          mine += m[j];
        }
        const unsigned long long inc = warp_scan(mine);
        const unsigned long long target = target_of(par.u, __shfl_sync(0xffffffffu, inc, 31));
        int seg = -1;
        unsigned long long at = inc - mine, seg_before = 0;
#pragma unroll
        for (int j = 0; j < SA_MAX_C * SA_W / 32; ++j) {
          if (at <= target && target < at + m[j]) {
            seg = lane * (SA_MAX_C * SA_W / 32) + j;
            seg_before = at;
          }
          at += m[j];
        }
        if (seg >= 0) {  // one lane
          s.bin = seg;
          s.before = seg_before;
          s.in_bin = target;
        }
      }
      __syncthreads();
      // its pieces again, one a thread, in index order
      const int seg = s.bin;
      unsigned long long at = s.before;
      const unsigned long long target = s.in_bin;
      const int b = seg / SA_W, bv0 = b * per_block, bv = min(per_block, NV - bv0), pw = (bv + SA_W - 1) / SA_W;
      const int s0 = min(seg % SA_W * pw, bv), s1 = min(s0 + pw, bv);
      for (int vb = s0; vb < s1 && at <= target; vb += SA_T) {
        const int v = vb + t, e0 = (bv0 + v) * PER - skew;
        unsigned long long w[PER], mm = 0;
        if (v < s1) {
          uint4 q;
          raw *qr = reinterpret_cast<raw *>(&q);
          if (e0 >= 0 && e0 + PER <= a.V) {
            q = ld_cg16(x + e0);
          } else {
#pragma unroll
            for (int j = 0; j < PER; ++j) qr[j] = e0 + j >= 0 && e0 + j < a.V ? __ldcg(x + e0 + j) : FILL;
          }
#pragma unroll
          for (int j = 0; j < PER; ++j) {
            const float f = E::up(qr[j]);
            const unsigned long long key =
                (unsigned long long)key_of<E>(qr[j]) << SA_IDX_BITS | (unsigned)((1 << SA_IDX_BITS) - 1 - (e0 + j));
            const double wd = weigh.finite(f);
            w[j] = f == f && key >= last && wd >= mp ? Weigher::fixed(wd) : 0;
            mm += w[j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < PER; ++j) w[j] = 0;
        }
        const unsigned long long ms = warp_scan(mm);
        unsigned long long before, total;
        __syncthreads();  // (the slots of the round before have been read)
        block_offsets(ms, s.scan[1], before, total);
        unsigned long long run2 = at + before + ms - mm;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          if (run2 <= target && target < run2 + w[j]) finish(e0 + j);
          run2 += w[j];
        }
        at += total;
      }
      return;
    }
  }
  cl.sync();  // the counts have been read by every block
  const int token = sample_exact<E>(cl, s, part, weigh, bins, par, a.V);
  if (token >= 0) finish(token);
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
  while (C < SA_MAX_C && ((NV + C - 1) / C) * 16 > SA_STAGE) C *= 2;
  while (C < SA_MAX_C && C * B <= device_sm_count() && NV > 2 * C * SA_T) C *= 2;  // two blocks an SM
  const int per_block = (NV + C - 1) / C;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = pdl_config(dim3((unsigned)(B * C)), dim3(SA_T), pdl, st, attr);
  attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
  attr[cfg.numAttrs].val.clusterDim.x = C;
  attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
  ++cfg.numAttrs;
  cfg.dynamicSmemBytes = (size_t)per_block * 16;
  return cudaLaunchKernelEx(&cfg, sample_kernel<E>, a);
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
