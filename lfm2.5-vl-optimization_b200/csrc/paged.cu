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
// order) stay within the free pages and the token capacity. One block: the scans run over 1024 requests at a time,
// the page moves one warp a request. The kernel is latency: a few dependent loads and three block scans.
constexpr int SL_T = 1024;

struct SlotArgs {
  const int *lens, *want;
  int *table, *freelist, *n_free;
  int *got, *cu;
  int64_t *positions, *slots;
  int B, width, pool, page;
  long long capacity;
};

// inclusive scans of a, b and c over the block's 1024 threads (64-bit: sums of wild requests do not wrap)
__device__ __forceinline__ void block_scan3(long long &a, long long &b, long long &c, long long (*part)[3]) {
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a2 = __shfl_up_sync(0xffffffffu, a, o), b2 = __shfl_up_sync(0xffffffffu, b, o),
                    c2 = __shfl_up_sync(0xffffffffu, c, o);
    if (lane >= o) {
      a += a2;
      b += b2;
      c += c2;
    }
  }
  __syncthreads();  // part's last readers
  if (lane == 31) {
    part[wp][0] = a;
    part[wp][1] = b;
    part[wp][2] = c;
  }
  __syncthreads();
  if (wp == 0) {
    long long x = part[lane][0], y = part[lane][1], z = part[lane][2];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x2 = __shfl_up_sync(0xffffffffu, x, o), y2 = __shfl_up_sync(0xffffffffu, y, o),
                      z2 = __shfl_up_sync(0xffffffffu, z, o);
      if (lane >= o) {
        x += x2;
        y += y2;
        z += z2;
      }
    }
    part[lane][0] = x;
    part[lane][1] = y;
    part[lane][2] = z;
  }
  __syncthreads();
  if (wp > 0) {
    a += part[wp - 1][0];
    b += part[wp - 1][1];
    c += part[wp - 1][2];
  }
}

__device__ __forceinline__ int pages_of(long long len, int page) { return (int)((len + page - 1) / page); }

// token i of the batch: its request is the last b with cu[b] <= i (requests without tokens share an offset with the
// next one, and the last of them is the one that holds i)
__device__ __forceinline__ void fill_slot(const SlotArgs &a, long long i) {
  int lo = 0, hi = a.B;  // cu[lo] <= i < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldcg(a.cu + mid) <= i) lo = mid;
    else hi = mid;
  }
  const long long pos = __ldcg(a.lens + lo) + (i - __ldcg(a.cu + lo));
  a.positions[i] = pos;
  a.slots[i] = (long long)__ldcg(a.table + (size_t)lo * a.width + pos / a.page) * a.page + pos % a.page;
}

template <bool FILL>
__global__ void __launch_bounds__(SL_T) kv_slots_kernel(const SlotArgs a) {
  __shared__ long long part[32][3];
  __shared__ int s_old[SL_T], s_need[SL_T], s_ret[SL_T];  // old page count, pages taken / returned
  __shared__ int s_need_off[SL_T], s_ret_off[SL_T];
  pdl_trigger();
  pdl_wait();
  const int t = threadIdx.x, lane = t & 31, wp = t >> 5;
  const long long room = (long long)a.width * a.page;
  const int n0 = min(max(__ldcg(a.n_free), 0), a.pool);
  // pass 1: what is granted. Offsets of the granted requests come out of a second scan, since a refused one takes
  // nothing.
  long long need_run = 0, tok_run = 0, tok_off = 0, P = 0, R = 0;
  for (int b0 = 0; b0 < a.B; b0 += SL_T) {
    const int b = b0 + t;
    long long len = 0, want = 0, need = 0, tok = 0, zero = 0;
    bool ok = false;
    if (b < a.B) {
      len = __ldcg(a.lens + b);
      want = __ldcg(a.want + b);
      ok = len >= 0 && want >= 0 && len <= room && want <= room;
      if (ok) {
        need = max(0, pages_of(want, a.page) - pages_of(len, a.page));
        tok = max(0ll, want - len);
      }
    }
    long long ns = need, ts = tok;
    block_scan3(ns, ts, zero, part);
    ok = ok && (need == 0 || need_run + ns <= n0) && (tok == 0 || tok_run + ts <= a.capacity);
    need_run += part[31][0];
    tok_run += part[31][1];
    if (!ok) need = tok = 0;
    long long ret = ok ? max(0, pages_of(len, a.page) - pages_of(want, a.page)) : 0;
    long long gn = need, gt = tok, gr = ret;
    block_scan3(gn, gt, gr, part);
    if (b < a.B) {
      a.got[b] = (int)(ok ? want : len);
      a.cu[b] = (int)(tok_off + gt - tok);
    }
    if (a.B <= SL_T) {  // one chunk: the offsets stay where the page moves read them
      s_old[t] = ok ? pages_of(len, a.page) : 0;
      s_need[t] = (int)need;
      s_ret[t] = (int)ret;
      s_need_off[t] = (int)(gn - need);
      s_ret_off[t] = (int)(gr - ret);
    }
    P += part[31][0];
    tok_off += part[31][1];
    R += part[31][2];
  }
  if (t == 0) a.cu[a.B] = (int)tok_off;
  __syncthreads();

  // passes 2 and 3: taken pages, then (a barrier later: the returned ones overwrite the stack entries that the taken
  // ones were read from) returned pages
  for (int take = 1; take >= 0; --take) {
    if ((take ? P : R) == 0) continue;
    long long off_run = 0;
    for (int b0 = 0; b0 < a.B; b0 += SL_T) {
      if (a.B > SL_T) {  // several chunks: a request's moves follow from lens and got
        const int b = b0 + t;
        int old = 0, moves = 0;
        if (b < a.B) {
          const int got = __ldcg(a.got + b), len = __ldcg(a.lens + b);
          if (got != len) {  // granted, so both are valid
            old = pages_of(len, a.page);
            moves = max(0, take ? pages_of(got, a.page) - old : old - pages_of(got, a.page));
          }
        }
        long long m = moves, z0 = 0, z1 = 0;
        block_scan3(m, z0, z1, part);
        s_old[t] = old;
        (take ? s_need : s_ret)[t] = moves;
        (take ? s_need_off : s_ret_off)[t] = (int)(off_run + m - moves);
        off_run += part[31][0];
        __syncthreads();
      }
      const int nb = min(SL_T, a.B - b0);
      for (int r = wp; r < nb; r += SL_T / 32) {
        int *row = a.table + (size_t)(b0 + r) * a.width;
        if (take) {
          for (int j = lane; j < s_need[r]; j += 32)
            row[s_old[r] + j] = __ldcg(a.freelist + (n0 - 1 - (s_need_off[r] + j)));
        } else {
          const int keep = s_old[r] - s_ret[r];
          for (int j = lane; j < s_ret[r]; j += 32) {
            const long long at = n0 - P + R - 1 - (s_ret_off[r] + j);
            if (at >= 0 && at < a.pool) a.freelist[at] = __ldcg(row + keep + j);
            row[keep + j] = -1;
          }
        }
      }
      __syncthreads();
    }
  }
  if (t == 0) a.n_free[0] = (int)min((long long)a.pool, n0 - P + R);
  if (FILL) {
    __syncthreads();
    const long long n = tok_off;
    for (long long i = t; i < n; i += SL_T) fill_slot(a, i);
  }
}

__global__ void __launch_bounds__(256) kv_slots_fill_kernel(const SlotArgs a) {
  pdl_trigger();
  pdl_wait();
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i < __ldcg(a.cu + a.B)) fill_slot(a, i);
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
constexpr int RP_T = 256;
constexpr int RP_UN = 4;  // pieces a thread keeps in flight
template <class T, int D, bool INTER>
__global__ void __launch_bounds__(RP_T) rope_paged_kernel(const RopeArgs a) {
  constexpr int LPH = D / 8;  // lanes per head
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
    const double turn = 6.283185307179586476925;
    const double ang = (double)__ldcg(reinterpret_cast<const long long *>(a.positions) + n) * (double)__ldg(a.inv_freq + t);
    const float r = (float)fma(-rint(ang * (1.0 / turn)), turn, ang);
    float s, c;
    sincosf(r, &s, &c);
    cs[t] = make_float2(c * a.scaling, s * a.scaling);
  }
  __syncthreads();
  const bool cached = slot >= 0 && slot < a.cache_slots;
  T *krow = nullptr, *vrow = nullptr;
  if (cached) {
    const size_t at = ((size_t)(slot / a.page) * a.NKV * a.page + (size_t)(slot % a.page)) * D;
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
      if (head >= a.NQ + a.NKV || !live) {
        // values pass unchanged; the shuffles below need every lane of a warp that still holds q or k pieces
        if (live && cached) *reinterpret_cast<uint4 *>(vrow + (head - a.NQ - a.NKV) * head_step + 8 * sub) = rv;
      }
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
  const SlotArgs a{lens, want, table, freelist, n_free, got, cu, positions, slots, B, width, pool, page, capacity};
  cudaLaunchAttribute attr;
  // Up to 4096 token slots the one block fills them itself; more get a launch of their own with a block per 256.
  if (capacity <= 4 * SL_T) {
    const cudaLaunchConfig_t cfg = pdl_config(dim3(1), dim3(SL_T), pdl, st, &attr);
    return cudaLaunchKernelEx(&cfg, kv_slots_kernel<true>, a);
  }
  cudaLaunchConfig_t cfg = pdl_config(dim3(1), dim3(SL_T), pdl, st, &attr);
  if (const cudaError_t e = cudaLaunchKernelEx(&cfg, kv_slots_kernel<false>, a)) return e;
  cfg.gridDim = dim3((unsigned)((capacity + 255) / 256));
  cfg.blockDim = dim3(256);
  return cudaLaunchKernelEx(&cfg, kv_slots_fill_kernel, a);
}

cudaError_t launch_qk_norm_rope_kv_paged(const void *qkv, long long row_stride, const void *qw, const void *kw,
                                         const float *inv_freq, int rot, float scaling, const int64_t *positions,
                                         const int64_t *slots, void *q_out, void *kc, void *vc, int N, int NQ, int NKV,
                                         int D, long long num_pages, int page, float eps, bool interleaved, bool half,
                                         bool pdl, cudaStream_t st) {
  const RopeArgs a{qkv, qw, kw, inv_freq, positions, slots, q_out, kc, vc, row_stride, num_pages * page,
                   N, NQ, NKV, page, rot, scaling, eps};
  cudaLaunchAttribute attr;
  const cudaLaunchConfig_t cfg = pdl_config(dim3(N), dim3(RP_T), pdl, st, &attr);
  auto go = [&](auto kernel) { return cudaLaunchKernelEx(&cfg, kernel, a); };
  if (half) {
    if (D == 64) return interleaved ? go(rope_paged_kernel<__half, 64, true>) : go(rope_paged_kernel<__half, 64, false>);
    return interleaved ? go(rope_paged_kernel<__half, 128, true>) : go(rope_paged_kernel<__half, 128, false>);
  }
  if (D == 64) return interleaved ? go(rope_paged_kernel<bf16, 64, true>) : go(rope_paged_kernel<bf16, 64, false>);
  return interleaved ? go(rope_paged_kernel<bf16, 128, true>) : go(rope_paged_kernel<bf16, 128, false>);
}

}  // namespace lfm2q
