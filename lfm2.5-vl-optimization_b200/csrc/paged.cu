// The paged KV cache of a batch of requests: block tables and slot maps from request lengths (kv_slots), and the q/k
// norm + rotary positions + cache write of a batch of tokens (qk_norm_rope_kv_paged).
//
// Cache: kc / vc [num_pages, NKV, page, D]; position t of request b lives on page table[b][t / page], row t % page;
// its slot is table[b][t / page] * page + t % page. With page = max_len and table[b] = {b} this is the dense cache of
// decode_attention_split, so both kinds of decode step share one layout.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "common.cuh"
#include "launch.h"

namespace lfm2q {
namespace {

// ------------------------------------------------------------------ kv_slots
// need_b pages and tok_b tokens of a valid request; granted while the running sums (over all valid requests, in
// order) stay within the free pages and the token capacity. One block: the scans run over a block's worth of requests at
// a time, the page moves one warp a request. The kernel is latency, a chain of dependent loads (lengths, free pages,
// table) and barriers, so: the second scan (offsets without the refused requests) and the one of returned pages run only
// where there are such, the search for a token's request runs in shared memory, and a small batch takes a small block.
// Sums saturate at 2^31 - 1, past every limit (2^30 at most), and two of them add up within 32 bits. 37 requests x 16 tokens
// and the removal of those that were not accepted (two calls, 11 KB): 9.9 us; 64 requests x 1024 tokens (1.1 MB; a second
// kernel over the whole device writes the rows where there may be more than SL_FILL): 14.8 us for the two calls.
constexpr uint32_t SL_MAX = 0x7fffffffu;
constexpr int SL_BIG = 1024;     // threads for batches of more than 256 requests
constexpr int SL_FILL = 4096;    // token rows that the block fills itself

struct SlotArgs {
  const int *lens, *want;
  int *table, *freelist, *n_free;
  int *got, *cu;
  int64_t *positions, *slots;
  int B, width, pool, page;
  int capacity;
};

__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, SL_MAX); }
// inclusive saturating scans of two values over a block of SL_T threads, and their totals; part: [SL_T / 32]
template <int SL_T>
__device__ __forceinline__ void block_scan2(uint32_t &a, uint32_t &b, uint2 &total, uint2 *part) {
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t a2 = __shfl_up_sync(0xffffffffu, a, o), b2 = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) {
      a = sat_add(a, a2);
      b = sat_add(b, b2);
    }
  }
  __syncthreads();  // part's last readers
  if (lane == 31) part[wp] = make_uint2(a, b);
  __syncthreads();
  uint32_t ta = 0, tb = 0;
#pragma unroll
  for (int w = 0; w < SL_T / 32; ++w) {
    if (w == wp) {
      a = sat_add(a, ta);
      b = sat_add(b, tb);
    }
    ta = sat_add(ta, part[w].x);
    tb = sat_add(tb, part[w].y);
  }
  total = make_uint2(ta, tb);
}

__device__ __forceinline__ int pages_of(int len, int page) { return (int)(((unsigned)len + page - 1) / (unsigned)page); }

// Token i of the batch: its request is the last b with cu[b] <= i (requests without tokens share an offset with the next
// one, and the last of them is the one that holds i). SHARED: cu and lens are copies in shared memory.
template <bool SHARED>
__device__ __forceinline__ void fill_slot(const SlotArgs &a, const int *cu, const int *lens, int i) {
  int lo = 0, hi = a.B;  // cu[lo] <= i < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((SHARED ? cu[mid] : __ldcg(cu + mid)) <= i) lo = mid;
    else hi = mid;
  }
  const unsigned pos = SHARED ? lens[lo] + (i - cu[lo]) : __ldcg(lens + lo) + (i - __ldcg(cu + lo));
  const unsigned pg = pos / (unsigned)a.page;
  a.positions[i] = pos;
  a.slots[i] = (long long)__ldcg(a.table + (size_t)lo * a.width + pg) * a.page + (pos - pg * a.page);
}

template <int SL_T>
__global__ void __launch_bounds__(SL_T) kv_slots_kernel(const SlotArgs a) {
  __shared__ uint2 part[SL_T / 32];
  __shared__ int s_old[SL_T], s_need[SL_T], s_ret[SL_T];  // old page count, pages taken / returned
  __shared__ int s_need_off[SL_T], s_ret_off[SL_T], s_cu[SL_T], s_len[SL_T];
  pdl_trigger();
  pdl_wait();
  const int t = threadIdx.x, lane = t & 31, wp = t >> 5;
  const int room = a.width * a.page;  // <= 2^30
  const bool one = a.B <= SL_T;       // one chunk: everything stays in shared memory
  uint32_t need_run = 0, tok_run = 0, tok_off = 0, P = 0, R = 0, n0 = 0;
  // pass 1: what is granted, and the offsets of the granted
  for (int b0 = 0; b0 == 0 || b0 < a.B; b0 += SL_T) {
    const int b = b0 + t;
    int len = 0, want = 0;
    if (b < a.B) {
      len = __ldcg(a.lens + b);
      want = __ldcg(a.want + b);
    }
    if (b0 == 0) n0 = min(max(__ldcg(a.n_free), 0), a.pool);
    bool ok = b < a.B && len >= 0 && want >= 0 && len <= room && want <= room;
    const int old = ok ? pages_of(len, a.page) : 0, now = ok ? pages_of(want, a.page) : 0;
    uint32_t need = ok ? max(0, now - old) : 0, tok = ok ? max(0, want - len) : 0;
    uint32_t ns = need, ts = tok;
    uint2 total;
    block_scan2<SL_T>(ns, ts, total, part);
    const bool fits = (need == 0 || sat_add(need_run, ns) <= n0) && (tok == 0 || sat_add(tok_run, ts) <= (uint32_t)a.capacity);
    need_run = sat_add(need_run, total.x);
    tok_run = sat_add(tok_run, total.y);
    if (__syncthreads_or(ok && !fits)) {  // without the refused
      ok = ok && fits;
      if (!ok) need = tok = 0;
      ns = need;
      ts = tok;
      block_scan2<SL_T>(ns, ts, total, part);
    }
    uint32_t ret = ok ? max(0, old - now) : 0, rs = ret, zero = 0;
    uint2 rtotal = make_uint2(0, 0);
    if (__syncthreads_or(ret)) block_scan2<SL_T>(rs, zero, rtotal, part);
    const int at = (int)(tok_off + ts - tok);
    if (b < a.B) {
      a.got[b] = ok ? want : len;
      a.cu[b] = at;
    }
    if (one) {
      s_old[t] = old;
      s_need[t] = (int)need;
      s_ret[t] = (int)ret;
      s_need_off[t] = (int)(ns - need);
      s_ret_off[t] = (int)(rs - ret);
      s_cu[t] = at;
      s_len[t] = len;
    }
    P += total.x;
    tok_off += total.y;
    R += rtotal.x;
  }
  if (t == 0) a.cu[a.B] = (int)tok_off;
  __syncthreads();

  // passes 2 and 3: taken pages, then (a barrier later: the returned ones overwrite the stack entries that the taken
  // ones were read from) returned pages
  for (int take = 1; take >= 0; --take) {
    if ((take ? P : R) == 0) continue;
    uint32_t off_run = 0;
    for (int b0 = 0; b0 < a.B; b0 += SL_T) {
      if (!one) {  // several chunks: a request's moves follow from lens and got
        const int b = b0 + t;
        int old = 0, moves = 0;
        if (b < a.B) {
          const int got = __ldcg(a.got + b), len = __ldcg(a.lens + b);
          if (got != len) {  // granted, so both are valid
            old = pages_of(len, a.page);
            moves = max(0, take ? pages_of(got, a.page) - old : old - pages_of(got, a.page));
          }
        }
        uint32_t m = moves, z = 0;
        uint2 total;
        block_scan2<SL_T>(m, z, total, part);
        s_old[t] = old;
        (take ? s_need : s_ret)[t] = moves;
        (take ? s_need_off : s_ret_off)[t] = (int)(off_run + m - moves);
        off_run += total.x;
        __syncthreads();
      }
      const int nb = min(SL_T, a.B - b0);
      for (int r = wp; r < nb; r += SL_T / 32) {
        int *row = a.table + (size_t)(b0 + r) * a.width;
        if (take) {
          for (int j = lane; j < s_need[r]; j += 32)
            row[s_old[r] + j] = __ldcg(a.freelist + ((int)n0 - 1 - (s_need_off[r] + j)));
        } else {
          const int keep = s_old[r] - s_ret[r];
          for (int j = lane; j < s_ret[r]; j += 32) {
            const long long at = (long long)n0 - P + R - 1 - (s_ret_off[r] + j);
            if (at >= 0 && at < a.pool) a.freelist[at] = __ldcg(row + keep + j);
            row[keep + j] = -1;
          }
        }
      }
      __syncthreads();
    }
  }
  if (t == 0) a.n_free[0] = (int)min((long long)a.pool, (long long)n0 - P + R);
  if (a.capacity <= SL_FILL)
    for (int i = t; i < (int)tok_off; i += SL_T) {
      if (one) fill_slot<true>(a, s_cu, s_len, i);
      else fill_slot<false>(a, a.cu, a.lens, i);
    }
}

// Larger token capacities: a launch of its own. The offsets come into shared memory where they fit.
constexpr int SF_T = 256, SF_MAX_B = 2048;
__global__ void __launch_bounds__(SF_T) kv_slots_fill_kernel(const SlotArgs a) {
  __shared__ int s_cu[SF_MAX_B], s_len[SF_MAX_B];
  pdl_trigger();
  pdl_wait();
  const int n = __ldcg(a.cu + a.B);
  if ((long long)blockIdx.x * SF_T >= n) return;
  const bool small = a.B <= SF_MAX_B;
  if (small) {
    for (int b = threadIdx.x; b < a.B; b += SF_T) {
      s_cu[b] = __ldcg(a.cu + b);
      s_len[b] = __ldcg(a.lens + b);
    }
    __syncthreads();
  }
  for (long long i = (long long)blockIdx.x * SF_T + threadIdx.x; i < n; i += (long long)gridDim.x * SF_T) {
    if (small) fill_slot<true>(a, s_cu, s_len, (int)i);
    else fill_slot<false>(a, a.cu, a.lens, (int)i);
  }
}

// ------------------------------------------------------------------ qk_norm_rope_kv_paged
template <class T>
struct Half2;
template <>
struct Half2<bf16> {
  static __device__ __forceinline__ float2 up(uint32_t u) { return make_float2(bf_lo(u), bf_hi(u)); }
  static __device__ __forceinline__ uint32_t down(float a, float b) { return pack_bf16x2(a, b); }
};
template <>
struct Half2<__half> {
  static __device__ __forceinline__ float2 up(uint32_t u) { return __half22float2(*reinterpret_cast<__half2 *>(&u)); }
  static __device__ __forceinline__ uint32_t down(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
};

struct RopeArgs {
  const void *qkv, *qw, *kw;
  const float *inv_freq;
  const int64_t *positions, *slots;
  void *q_out, *kc, *vc;
  long long row_stride, cache_slots;
  int N, NQ, NKV, page, rot;
  float scaling, eps;
};

// One block a token: its cosines and sines once, in shared memory, then every head in 16-byte pieces (8 or 16 lanes a
// head). The half layout's partner value is rot / 16 lanes away (rot is a multiple of 16), the interleaved one's is
// in the same lane. Everything in fp32 and rounded once; the angle positions[n] * inv_freq[i] is formed and reduced
// in fp64 (exact product, then off by about n_turns * 2^-52): in fp32 a position of 10^6 would lose the angle's
// fourth digit.
// Two shapes of block, either for any number of heads (a block goes round its token's pieces until they are done): 128
// threads with 6 pieces each in flight and 8 blocks an SM for many tokens, 384 threads with 2 for few, up to two tokens an
// SM, where a token's latency counts. Both sides, many | few, half layout with norm, bf16, us:
//            48 heads of 128   48 heads of 64   8 heads of 64   80 heads of 128
//   1 token        4.9 | 3.1        3.4 | 2.3       2.2 | 2.2         8.0 | 4.3
//   150            5.3 | 4.2        3.6 | 2.8       2.3 | 2.4         8.7 | 6.0
//   300            6.5 | 5.8        3.9 | 3.5       2.3 | 2.5        11.9 | 9.7
//   2000          20.0 | 19.0      10.6 | 11.4      4.3 | 7.0        33.1 | 30.9
//   16384        113.9 | 118.7     56.3 | 71.2     25.6 | 48.6      204.5 | 207.2
// The shapes were found on 16384 tokens with 48 heads of 128 in the interleaved layout (256 x 4: 78 us, 128 x 3: 75 us,
// 128 x 6: 67 us, 6.0 TB/s, 91 % of the measured copy rate), where HBM bounds. The half layout, whose pairs lie in
// two lanes, takes 114 us there (3.5 TB/s; 105 without the norm, as the interleaved one takes 60 in place of 68): eight
// exchanges a piece. Few heads are bounded by a block's beginning: 8 heads of 64 leave half of the 128 threads without a
// piece (26 us, 1.3 TB/s).
struct RopeMany {
  static constexpr int T = 128, UN = 6, BLOCKS = 8;
};
struct RopeFew {
  static constexpr int T = 384, UN = 2, BLOCKS = 4;
};
template <class T, int D, bool INTER, class SHAPE>
__global__ void __launch_bounds__(SHAPE::T, SHAPE::BLOCKS) rope_paged_kernel(const RopeArgs a) {
  constexpr int RP_T = SHAPE::T, RP_UN = SHAPE::UN;  // pieces a thread keeps in flight
  constexpr int LPH = D / 8;                         // lanes per head
  __shared__ float2 cs[D / 2];
  pdl_trigger();
  pdl_wait();
  const int n = blockIdx.x, t = threadIdx.x;
  const int NH = a.NQ + 2 * a.NKV, pieces = NH * LPH;
  const int padded = (pieces + 31) & ~31;  // whole warps take part in the shuffles
  const uint4 *src = reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(a.qkv) + n * a.row_stride);
  uint4 raw[RP_UN];
#pragma unroll
  for (int u = 0; u < RP_UN; ++u)
    if (t + u * RP_T < pieces) raw[u] = ld_cg16(src + t + u * RP_T);
  const long long slot = __ldcg(reinterpret_cast<const long long *>(a.slots) + n);
  if (t < a.rot / 2) {
    // in turns: the fraction keeps 2^-25 of one after its rounding to fp32
    const double turns = (double)__ldcg(reinterpret_cast<const long long *>(a.positions) + n) * (double)__ldg(a.inv_freq + t) *
                         0.15915494309189533577;
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    cs[t] = make_float2(c * a.scaling, s * a.scaling);
  }
  __syncthreads();
  const bool cached = slot >= 0 && slot < a.cache_slots;
  T *krow = nullptr, *vrow = nullptr;
  if (cached) {
    const unsigned pg = (unsigned)slot / (unsigned)a.page;  // (fewer than 2^32 slots: a cache of 2^38 elements)
    const size_t at = ((size_t)pg * a.NKV * a.page + ((unsigned)slot - pg * a.page)) * D;
    krow = reinterpret_cast<T *>(a.kc) + at;
    vrow = reinterpret_cast<T *>(a.vc) + at;
  }
  const size_t head_step = (size_t)a.page * D;  // cache: from one KV head's row to the next
  T *qrow = reinterpret_cast<T *>(a.q_out) + (size_t)n * a.NQ * D;
  for (int p0 = t; p0 < padded; p0 += RP_UN * RP_T) {
#pragma unroll
    for (int u = 0; u < RP_UN; ++u) {
      const int p = p0 + u * RP_T;
      if (p >= padded) break;  // whole warps: padded and the strides are multiples of 32
      const bool live = p < pieces;
      if (p0 != t && live) raw[u] = ld_cg16(src + p);
      const int head = p / LPH, sub = p % LPH;
      const uint4 rv = live ? raw[u] : make_uint4(0, 0, 0, 0);
      if (head >= a.NQ + a.NKV && live && cached)  // values pass unchanged
        *reinterpret_cast<uint4 *>(vrow + (head - a.NQ - a.NKV) * head_step + 8 * sub) = rv;
      if (__all_sync(0xffffffffu, head >= a.NQ + a.NKV)) continue;  // (the shuffles below need every lane otherwise)
      float x[8];
      {
        const uint32_t w[4] = {rv.x, rv.y, rv.z, rv.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = Half2<T>::up(w[j]);
          x[2 * j] = f.x;
          x[2 * j + 1] = f.y;
        }
      }
      const bool is_q = head < a.NQ;
      const T *nw = reinterpret_cast<const T *>(is_q ? a.qw : a.kw);
      if (a.qw) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float rs = rsqrtf(ss / D + a.eps);
        const uint4 wv = __ldg(reinterpret_cast<const uint4 *>(nw) + sub);
        const uint32_t w[4] = {wv.x, wv.y, wv.z, wv.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = Half2<T>::up(w[j]);
          x[2 * j] *= rs * f.x;
          x[2 * j + 1] *= rs * f.y;
        }
      }
      if (INTER) {
        if (8 * sub < a.rot) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 e = cs[4 * sub + j];
            const float lo = x[2 * j], hi = x[2 * j + 1];
            x[2 * j] = lo * e.x - hi * e.y;
            x[2 * j + 1] = hi * e.x + lo * e.y;
          }
        }
      } else {
        const int hl = a.rot / 16;  // lanes between the halves
        const bool first = sub < hl, in = sub < 2 * hl;
        const int lane = t & 31, other = in ? (first ? lane + hl : lane - hl) : lane;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float y = __shfl_sync(0xffffffffu, x[j], other);
          if (in) {
            const float2 e = cs[8 * (first ? sub : sub - hl) + j];
            x[j] = first ? x[j] * e.x - y * e.y : x[j] * e.x + y * e.y;
          }
        }
      }
      if (!live || head >= a.NQ + a.NKV) continue;
      const uint4 o = make_uint4(Half2<T>::down(x[0], x[1]), Half2<T>::down(x[2], x[3]), Half2<T>::down(x[4], x[5]),
                                 Half2<T>::down(x[6], x[7]));
      if (is_q)
        *reinterpret_cast<uint4 *>(qrow + (size_t)head * D + 8 * sub) = o;
      else if (cached)
        *reinterpret_cast<uint4 *>(krow + (head - a.NQ) * head_step + 8 * sub) = o;
    }
  }
}

}  // namespace

cudaError_t launch_kv_slots(const int *lens, const int *want, int *table, int *freelist, int *n_free, int *got, int *cu,
                            int64_t *positions, int64_t *slots, int B, int width, int pool, int page,
                            long long capacity, bool pdl, cudaStream_t st) {
  const SlotArgs a{lens, want, table, freelist, n_free, got, cu, positions, slots, B, width, pool, page, (int)capacity};
  cudaLaunchAttribute attr;
  cudaLaunchConfig_t cfg = pdl_config(dim3(1), dim3(B <= 256 ? 256 : SL_BIG), pdl, st, &attr);
  if (const cudaError_t e = B <= 256 ? cudaLaunchKernelEx(&cfg, kv_slots_kernel<256>, a)
                                     : cudaLaunchKernelEx(&cfg, kv_slots_kernel<SL_BIG>, a))
    return e;
  if (capacity <= SL_FILL) return cudaSuccess;
  cfg.gridDim = dim3((unsigned)std::min<long long>((capacity + SF_T - 1) / SF_T, 4LL * device_sm_count()));
  cfg.blockDim = dim3(SF_T);
  return cudaLaunchKernelEx(&cfg, kv_slots_fill_kernel, a);
}

cudaError_t launch_qk_norm_rope_kv_paged(const void *qkv, long long row_stride, const void *qw, const void *kw,
                                         const float *inv_freq, int rot, float scaling, const int64_t *positions,
                                         const int64_t *slots, void *q_out, void *kc, void *vc, int N, int NQ, int NKV,
                                         int D, long long num_pages, int page, float eps, bool interleaved, bool half,
                                         bool pdl, cudaStream_t st) {
  const RopeArgs a{qkv, qw, kw, inv_freq, positions, slots, q_out, kc, vc, row_stride, num_pages * page,
                   N, NQ, NKV, page, rot, scaling, eps};
  auto go = [&](auto many, auto few) {
    const bool is_few = N <= 2 * device_sm_count();
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = pdl_config(dim3(N), dim3(is_few ? RopeFew::T : RopeMany::T), pdl, st, &attr);
    return cudaLaunchKernelEx(&cfg, is_few ? few : many, a);
  };
#define LFM2Q_ROPE(T, D, I) go(rope_paged_kernel<T, D, I, RopeMany>, rope_paged_kernel<T, D, I, RopeFew>)
  if (half) {
    if (D == 64) return interleaved ? LFM2Q_ROPE(__half, 64, true) : LFM2Q_ROPE(__half, 64, false);
    return interleaved ? LFM2Q_ROPE(__half, 128, true) : LFM2Q_ROPE(__half, 128, false);
  }
  if (D == 64) return interleaved ? LFM2Q_ROPE(bf16, 64, true) : LFM2Q_ROPE(bf16, 64, false);
  return interleaved ? LFM2Q_ROPE(bf16, 128, true) : LFM2Q_ROPE(bf16, 128, false);
#undef LFM2Q_ROPE
}

}  // namespace lfm2q
