// Attention of drafted tokens over a paged KV cache on the fifth-generation tensor cores: the kernel for caches whose
// pages are multiples of 8 positions (tree_attention.cu has the mathematics, the form for other pages, and the join of
// the splits).
//
// A block takes 128 rows (queries times heads of one KV head) of one request and one split of its positions. Warp 4
// streams K and V tiles of 64 positions by TMA into 128-byte-swizzled stages (boxes of up to 64 rows that never cross
// a page; one lane a box); warp 5 issues tcgen05.mma: S = Q K^T into one of two 64-column TMEM buffers, then
// O += P V with P read back from TMEM (it lies over its S) and V as it is in the cache (an MN-major operand); warps 0-3
// do the softmax, one thread a row, so that a row's maximum and sum need no exchange between lanes. While tile n is in
// the softmax, S of tile n + 1 is computed and O of tile n - 1 accumulated. O stays in TMEM; it is rescaled only when a
// row's maximum has grown by more than 2^8 since the last time (the probabilities then reach at most 2^8, exact as far
// as floating point goes), which after the first tiles is rare.
//
// Per tile and row: 64 exponentials and about 4 times as many fp32 operations against 16 KB of K and V (head dim 64) a
// block. 128 rows: bounded by the exponentials (16 a cycle and SM: 512 cycles a tile; 16 KB take 700 cycles of one SM's
// share of the HBM rate), so two blocks an SM (96 KB of shared memory and 256 TMEM columns each) keep both busy.
//
// Every wait is bounded (about a second of SM clocks); a wait that gives up sets the device error word that
// lfm2q_check_device reports, and the block ends without writing its rows.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <mutex>
#include <type_traits>

#include "launch.h"
#include "tree_attention.cuh"

namespace lfm2q {

__device__ int g_tree_err = 0;  // sticky: 1 = a pipeline wait gave up

namespace {

constexpr int TT_ROWS = 128;
constexpr int TT_THREADS = 192;
constexpr int TT_ATOM = TT_ROWS * 128;         // 64 dims of the query tile
constexpr int TT_HALF = TA_KEYS * 128;         // 64 dims of a K (or V) tile
constexpr int TT_TMEM = 256;                   // columns: S0 | S1 | O
constexpr long long TT_WAIT_LIMIT = 1ll << 31;
constexpr float TT_SLACK = 8.f;                // log2 of what a row's maximum may grow before O is rescaled

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait for the phase with the given parity. False: this or another role gave up.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int *stop) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (*stop) return false;
    if (clock64() - t0 > TT_WAIT_LIMIT) {
      *stop = 1;
      atomicCAS(&g_tree_err, 0, 1);
      return false;
    }
  }
  return true;
}
// one lane waits, the warp follows its verdict (the .sync.aligned TMEM accesses need a convergent warp)
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *stop) {
  bool ok = true;
  if ((threadIdx.x & 31) == 0) ok = mbar_wait(bar, parity, stop);
  return __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// Operand in rows of 128 bytes, 128-byte swizzle, 8-row atoms 1024 bytes apart. lbo: MN-major operands wider than 64,
// from one 64-wide block to the next (bytes).
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// kind::f16 instruction descriptor, fp32 accumulation, M = 128
__host__ __device__ constexpr uint32_t idesc_f16(int n, bool bf, bool b_mn_major) {
  return (1u << 4) | (bf ? (1u << 7) | (1u << 10) : 0u) | (b_mn_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(TT_ROWS >> 4) << 24);
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

#define TT_REGS32(r, c)                                                                                                \
  c(r[0]), c(r[1]), c(r[2]), c(r[3]), c(r[4]), c(r[5]), c(r[6]), c(r[7]), c(r[8]), c(r[9]), c(r[10]), c(r[11]),       \
      c(r[12]), c(r[13]), c(r[14]), c(r[15]), c(r[16]), c(r[17]), c(r[18]), c(r[19]), c(r[20]), c(r[21]), c(r[22]),   \
      c(r[23]), c(r[24]), c(r[25]), c(r[26]), c(r[27]), c(r[28]), c(r[29]), c(r[30]), c(r[31])
#define TT_OUT(x) "=r"(x)
#define TT_IN(x) "r"(x)
#define TT_TIE(x) "+r"(x)
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : TT_REGS32(r, TT_OUT)
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::TT_REGS32(r, TT_IN),
      "r"(taddr)
      : "memory");
}
// wait for this thread's TMEM loads, the registers tied to the wait so that no use of them moves before it
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : TT_REGS32(r, TT_TIE) : : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int D>
struct TcShape {
  static constexpr int HALVES = D / 64;
  static constexpr int STAGES = D == 64 ? 5 : 2;
  static constexpr int Q_BYTES = HALVES * TT_ATOM;
  static constexpr int KV_BYTES = HALVES * TT_HALF;  // a K (or V) tile
  static constexpr int SMEM = Q_BYTES + 2 * STAGES * KV_BYTES + 1024;  // room to align the base to 1024
};

template <class T, int D>
__global__ void __launch_bounds__(TT_THREADS, 2)
    tree_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const TreeArgs a,
                   int row_tiles, int box) {
  using L = TcShape<D>;
  constexpr int STAGES = L::STAGES, HALVES = L::HALVES;
  constexpr bool BF = std::is_same<T, bf16>::value;
  extern __shared__ uint8_t tt_smem[];
  __shared__ __align__(8) uint64_t full_k[STAGES], full_v[STAGES], empty[STAGES], s_full[2], p_full[2], pv_done, o_full;
  __shared__ unsigned long long live[STAGES];  // keys of the stage's tile that exist
  __shared__ unsigned long long apart;         // drafts that were taken out of the second product
  __shared__ uint32_t tmem_slot;
  __shared__ int stop, red;
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(tt_smem) + 1023) & ~uintptr_t(1023));
  const uint32_t sq = smem_addr(smem), sk = sq + L::Q_BYTES, sv = sk + STAGES * L::KV_BYTES;
  uint8_t *gv = smem + L::Q_BYTES + STAGES * L::KV_BYTES;  // the V stages, generic address
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_trigger();
  pdl_wait();

  const int rt = blockIdx.x % row_tiles, bk = blockIdx.x / row_tiles, kvh = bk % a.NKV, b = bk / a.NKV;
  const int split = blockIdx.y, r_base = rt * TT_ROWS;
  const Request rq(a, b);
  const int rows = min(rq.T * a.G - r_base, TT_ROWS);
  if (rows <= 0) return;
  const int chunk = a.S == 1 ? (rq.len + TA_KEYS - 1) / TA_KEYS * TA_KEYS : split_chunk(a, &red);
  const int t0 = (int)min((long long)split * chunk, (long long)rq.len), t1 = t0 + min(rq.len - t0, chunk);
  const int tiles = (t1 - t0 + TA_KEYS - 1) / TA_KEYS;
  const int row = threadIdx.x;  // warps 0-3: the thread's row of the tile
  const int tok = (r_base + row) / a.G, head = kvh * a.G + (r_base + row) % a.G;
  const size_t out_row = (size_t)(rq.n0 + tok) * a.NQ + head;
  if (tiles == 0) {  // nothing to see here
    if (row < rows) {
      if (a.S == 1) {
        uint4 *dst = reinterpret_cast<uint4 *>(reinterpret_cast<T *>(a.out) + out_row * D);
        for (int j = 0; j < D / 8; ++j) dst[j] = make_uint4(0, 0, 0, 0);
      } else {
        *reinterpret_cast<float2 *>(a.ws + (out_row * a.S + split) * (D + 2)) = make_float2(-INFINITY, 0.f);
      }
    }
    return;
  }
  const int active = (rows + 31) / 32;  // softmax warps with rows
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(smem_addr(&full_k[i]), 1);
      mbar_init(smem_addr(&full_v[i]), 1);
      mbar_init(smem_addr(&empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_addr(&s_full[i]), 1);
      mbar_init(smem_addr(&p_full[i]), active);
    }
    mbar_init(smem_addr(&pv_done), 1);
    mbar_init(smem_addr(&o_full), 1);
    stop = 0;
    apart = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)),
                 "r"(TT_TMEM)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // queries, in the swizzled layout of the first product's A operand; rows behind the last are zeros
  for (int i = threadIdx.x; i < TT_ROWS * (D / 8); i += TT_THREADS) {
    const int r = i / (D / 8), c = i % (D / 8), gr = r_base + r;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < rows)
      v = ld_cg16(reinterpret_cast<const T *>(a.q) +
                  ((size_t)(rq.n0 + gr / a.G) * a.NQ + kvh * a.G + gr % a.G) * D + 8 * c);
    *reinterpret_cast<uint4 *>(smem + (c >> 3) * TT_ATOM + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v;
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the generic writes, before the MMAs read them
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int *table = a.table + (size_t)b * a.width;

  if (warp == 4) {
    // ---------------------------------------------------------------- K and V tiles
    const int boxes = TA_KEYS / box;
    int issued = 0;
    for (int n = 0; n < tiles; ++n, ++issued) {
      const int st = n % STAGES, base = t0 + n * TA_KEYS;
      int pg[2], y[2];
      uint32_t mine = 0;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int i = lane + 32 * u, t = base + i * box;
        pg[u] = -1;
        if (i < boxes && t < t1) {
          pg[u] = __ldcg(table + t / a.page);
          y[u] = t % a.page;
        }
        if (pg[u] < 0 || pg[u] >= a.num_pages) pg[u] = -1;
        else ++mine;
      }
      const uint32_t loads = __reduce_add_sync(0xffffffffu, mine);
      unsigned long long keys = 0;  // of this lane's boxes
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (pg[u] >= 0) {
          const int i = lane + 32 * u, n_live = min(box, t1 - (base + i * box));
          keys |= (n_live >= 64 ? ~0ull : (1ull << n_live) - 1) << (i * box);
        }
      const uint32_t klo = __reduce_or_sync(0xffffffffu, (uint32_t)keys),
                     khi = __reduce_or_sync(0xffffffffu, (uint32_t)(keys >> 32));
      if (n >= STAGES && !warp_wait(smem_addr(&empty[st]), (uint32_t)((n / STAGES - 1) & 1), &stop)) break;
      const uint32_t fk = smem_addr(&full_k[st]), fv = smem_addr(&full_v[st]);
      if (lane == 0) {
        live[st] = (unsigned long long)khi << 32 | klo;
        mbar_expect_tx(fk, loads * box * 128 * HALVES);
        mbar_expect_tx(fv, loads * box * 128 * HALVES);
      }
      __syncwarp();
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (pg[u] >= 0)
#pragma unroll
          for (int h = 0; h < HALVES; ++h)
            tma_load_3d(sk + st * L::KV_BYTES + h * TT_HALF + (lane + 32 * u) * box * 128, &tmK, fk, 64 * h, y[u],
                        pg[u] * a.NKV + kvh);
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (pg[u] >= 0)
#pragma unroll
          for (int h = 0; h < HALVES; ++h)
            tma_load_3d(sv + st * L::KV_BYTES + h * TT_HALF + (lane + 32 * u) * box * 128, &tmV, fv, 64 * h, y[u],
                        pg[u] * a.NKV + kvh);
    }
    if (issued < tiles && lane == 0) {  // gave up: no copy may land after the block has left
      int late = 0;
      for (int n = max(0, issued - STAGES); n < issued; ++n) {
        mbar_wait(smem_addr(&full_k[n % STAGES]), (uint32_t)((n / STAGES) & 1), &late);
        mbar_wait(smem_addr(&full_v[n % STAGES]), (uint32_t)((n / STAGES) & 1), &late);
      }
    }
  } else if (warp == 5) {
    // ---------------------------------------------------------------- MMAs
    if (lane == 0) {
      constexpr uint32_t ID_S = idesc_f16(TA_KEYS, BF, false), ID_O = idesc_f16(D, BF, true);
      auto scores = [&](int n) {
        const int st = n % STAGES;
        // P of tile n - 2 lies in this buffer until its product is done
        if (n >= 2 && !mbar_wait(smem_addr(&pv_done), (uint32_t)(n & 1), &stop)) return false;
        if (!mbar_wait(smem_addr(&full_k[st]), (uint32_t)((n / STAGES) & 1), &stop)) return false;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_ss(tmem + (n & 1) * TA_KEYS, sw128_desc(sq + (k >> 2) * TT_ATOM, 16) + 2 * (k & 3),
                  sw128_desc(sk + st * L::KV_BYTES + (k >> 2) * TT_HALF, 16) + 2 * (k & 3), ID_S, k != 0);
        umma_commit(smem_addr(&s_full[n & 1]));
        return true;
      };
      bool ok = scores(0);
      for (int n = 0; n < tiles && ok; ++n) {
        const int st = n % STAGES;
        ok = (n + 1 >= tiles || scores(n + 1)) &&
             mbar_wait(smem_addr(&p_full[n & 1]), (uint32_t)((n >> 1) & 1), &stop) &&
             mbar_wait(smem_addr(&full_v[st]), (uint32_t)((n / STAGES) & 1), &stop);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < TA_KEYS / 16; ++k)
          umma_ts(tmem + 2 * TA_KEYS, tmem + (n & 1) * TA_KEYS + 8 * k,
                  sw128_desc(sv + st * L::KV_BYTES + k * 2048, TT_HALF), ID_O, (n | k) != 0);
        umma_commit(smem_addr(&empty[st]));
        umma_commit(smem_addr(&pv_done));
      }
      umma_commit(smem_addr(&o_full));
      int late = 0;
      if (!ok) mbar_wait(smem_addr(&o_full), 0, &late);  // gave up: the MMAs in flight finish first
    }
  } else if (warp < active) {
    // ---------------------------------------------------------------- softmax, one thread a row
    const uint32_t lane_at = (uint32_t)(warp * 32) << 16;
    unsigned long long see = 0;
    if (row < rows) see = a.mask ? __ldcg(a.mask + rq.n0 + tok) : (tok >= 63 ? ~0ull : (2ull << tok) - 1);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int n = 0; n < tiles; ++n) {
      const int st = n % STAGES, base = t0 + n * TA_KEYS;
      const uint32_t sbuf = tmem + lane_at + (n & 1) * TA_KEYS;
      ok = warp_wait(smem_addr(&s_full[n & 1]), (uint32_t)((n >> 1) & 1), &stop);
      if (!ok) break;
      tc_fence_after();
      uint32_t s0[32], s1[32];
      tmem_ld32(sbuf, s0);
      tmem_ld32(sbuf + 32, s1);
      // keys of the tile that this row sees
      unsigned long long vis = *(volatile unsigned long long *)&live[st];
      const unsigned long long exists = vis;
      const int d0 = base - rq.ctx;  // draft of the tile's first key
      if (d0 > -TA_KEYS) vis &= d0 >= 0 ? (d0 < 64 ? see >> d0 : 0ull) : (1ull << -d0) - 1 | see << -d0;
      tmem_ld_wait(s0);
      tmem_ld_wait(s1);
      if (__any_sync(0xffffffffu, vis != ~0ull)) {
        const uint32_t v0 = (uint32_t)vis, v1 = (uint32_t)(vis >> 32);
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          if (!((v0 >> j) & 1)) s0[j] = 0xff800000u;
          if (!((v1 >> j) & 1)) s1[j] = 0xff800000u;
        }
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < 32; ++j) mx[j & 3] = fmaxf(mx[j & 3], fmaxf(__uint_as_float(s0[j]), __uint_as_float(s1[j])));
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2;
      const bool grow = top > m + TT_SLACK || (m == -INFINITY && top > -INFINITY);
      if (__any_sync(0xffffffffu, grow)) {
        const float corr = grow ? ex2(m - top) : 1.f;  // 0 while the row has seen nothing
        if (grow) m = top;
        l *= corr;
        if (n > 0) {
          ok = warp_wait(smem_addr(&pv_done), (uint32_t)((n - 1) & 1), &stop);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(tmem + lane_at + 2 * TA_KEYS + 32 * c, o);
            tmem_ld_wait(o);
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * corr);
            tmem_st32(tmem + lane_at + 2 * TA_KEYS + 32 * c, o);
          }
        }
      }
      const float ms = m == -INFINITY ? 0.f : m;
      uint32_t p[32];
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float e0 = ex2(fmaf(__uint_as_float(s0[2 * j]), a.scale_log2, -ms));
        const float e1 = ex2(fmaf(__uint_as_float(s0[2 * j + 1]), a.scale_log2, -ms));
        const float f0 = ex2(fmaf(__uint_as_float(s1[2 * j]), a.scale_log2, -ms));
        const float f1 = ex2(fmaf(__uint_as_float(s1[2 * j + 1]), a.scale_log2, -ms));
        p[j] = Pair<T>::pack(e0, e1);
        p[16 + j] = Pair<T>::pack(f0, f1);
        sum[0] += e0;
        sum[1] += e1;
        sum[2] += f0;
        sum[3] += f1;
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_st32(sbuf, p);
      // A key that a row does not see has p = 0, but 0 times an infinity or a NaN is a NaN: value rows that hold one
      // are zeroed in shared memory (stale ones of keys that do not exist, too), and drafts among them are added at
      // the end to the rows that see them.
      if (warp == 0 && (d0 > -TA_KEYS || exists != ~0ull)) {
        ok = warp_wait(smem_addr(&full_v[st]), (uint32_t)((n / STAGES) & 1), &stop);
        if (!ok) break;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const int r = g * 32 + lane;
          uint4 *vr = reinterpret_cast<uint4 *>(gv + st * L::KV_BYTES + r * 128);
          bool bad = false;
          if (base + r >= rq.ctx || !((exists >> r) & 1)) {
            for (int h = 0; h < HALVES; ++h)
              for (int c = 0; c < 8; ++c) {
                const uint4 u = vr[h * (TT_HALF / 16) + c];
                bad = bad || !(Pair<T>::finite(u.x) && Pair<T>::finite(u.y) && Pair<T>::finite(u.z) && Pair<T>::finite(u.w));
              }
            if (bad)
              for (int h = 0; h < HALVES; ++h)
                for (int c = 0; c < 8; ++c) vr[h * (TT_HALF / 16) + c] = make_uint4(0, 0, 0, 0);
          }
          if (bad && ((exists >> r) & 1)) atomicOr(&apart, 1ull << (base + r - rq.ctx));
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&p_full[n & 1]));
    }
    // ---------------------------------------------------------------- out, or this split's partial
    ok = ok && warp_wait(smem_addr(&o_full), 0, &stop) && *(volatile int *)&stop == 0;
    ok = __all_sync(0xffffffffu, ok);
    if (ok) {
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const unsigned long long extra = *(volatile unsigned long long *)&apart & see;
      float *part = a.ws + (out_row * a.S + split) * (D + 2);
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(tmem + lane_at + 2 * TA_KEYS + 32 * c, o);
        tmem_ld_wait(o);
        if (extra && row < rows) {  // rare: the score again from global memory, and p v added
          const uint32_t *qr = reinterpret_cast<const uint32_t *>(reinterpret_cast<const T *>(a.q) + out_row * D);
          for (unsigned long long left = extra; left; left &= left - 1) {
            const int t = rq.ctx + __ffsll(left) - 1;
            const size_t at = (((size_t)__ldcg(table + t / a.page) * a.NKV + kvh) * a.page + t % a.page) * D;
            const uint32_t *kr = reinterpret_cast<const uint32_t *>(reinterpret_cast<const T *>(a.kc) + at);
            const uint32_t *vr = reinterpret_cast<const uint32_t *>(reinterpret_cast<const T *>(a.vc) + at) + 16 * c;
            float dot = 0.f;
            for (int j = 0; j < D / 2; ++j) {
              const float2 x = Pair<T>::up(__ldcg(qr + j)), y = Pair<T>::up(__ldcg(kr + j));
              dot += x.x * y.x + x.y * y.y;
            }
            const float pr = ex2(fmaf(dot, a.scale_log2, m == -INFINITY ? 0.f : -m));
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float2 v = Pair<T>::up(__ldcg(vr + j));
              o[2 * j] = __float_as_uint(__uint_as_float(o[2 * j]) + pr * v.x);
              o[2 * j + 1] = __float_as_uint(__uint_as_float(o[2 * j + 1]) + pr * v.y);
            }
          }
        }
        if (row < rows) {
          if (a.S == 1) {
            uint4 *dst = reinterpret_cast<uint4 *>(reinterpret_cast<T *>(a.out) + out_row * D + 32 * c);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = Pair<T>::pack(__uint_as_float(o[8 * j + 2 * e]) * inv, __uint_as_float(o[8 * j + 2 * e + 1]) * inv);
              dst[j] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              *reinterpret_cast<float2 *>(part + 2 + 32 * c + 2 * j) =
                  make_float2(__uint_as_float(o[2 * j]), __uint_as_float(o[2 * j + 1]));
          }
        }
      }
      if (a.S > 1 && row < rows) *reinterpret_cast<float2 *>(part) = make_float2(m, l);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TT_TMEM) : "memory");
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// cache [heads, page, D] (heads = num_pages * NKV), box = 64 dims x box rows of one page, 128-byte swizzle
bool make_map(CUtensorMap *map, const void *ptr, int D, int page, long long heads, int box, bool half) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)page, (cuuint64_t)heads};
  const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)D * 2 * page};
  const cuuint32_t boxes[3] = {64, (cuuint32_t)box, 1}, es[3] = {1, 1, 1};
  return fn(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(ptr),
            dims, strides, boxes, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int D>
cudaError_t launch(const TreeArgs &a, bool pdl, cudaStream_t st) {
  auto kernel = tree_tc_kernel<T, D>;
  static std::atomic<int> attr_set[64];  // the shared-memory opt-in, once per device
  int dev = 0;
  if (const cudaError_t e = cudaGetDevice(&dev)) return e;
  if (dev < 64 && !attr_set[dev].load(std::memory_order_acquire)) {
    if (const cudaError_t e =
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TcShape<D>::SMEM))
      return e;
    attr_set[dev].store(1, std::memory_order_release);
  }
  int box = TA_KEYS;  // rows of a TMA box: the largest power of two up to a tile that divides the page
  while (a.page % box) box /= 2;
  CUtensorMap mk, mv;
  const bool half = !std::is_same<T, bf16>::value;
  const long long heads = (long long)a.num_pages * a.NKV;
  if (!make_map(&mk, a.kc, D, a.page, heads, box, half) || !make_map(&mv, a.vc, D, a.page, heads, box, half))
    return cudaErrorNotSupported;
  const int row_tiles = (a.max_q * a.G + TT_ROWS - 1) / TT_ROWS;
  cudaLaunchAttribute attr;
  cudaLaunchConfig_t cfg = pdl_config(dim3(row_tiles * a.NKV * a.B, a.S), dim3(TT_THREADS), pdl, st, &attr);
  cfg.dynamicSmemBytes = TcShape<D>::SMEM;
  return cudaLaunchKernelEx(&cfg, kernel, mk, mv, a, row_tiles, box);
}

}  // namespace

cudaError_t launch_tree_tc(const TreeArgs &a, int D, bool half, bool pdl, cudaStream_t st) {
  if (half) return D == 64 ? launch<__half, 64>(a, pdl, st) : launch<__half, 128>(a, pdl, st);
  return D == 64 ? launch<bf16, 64>(a, pdl, st) : launch<bf16, 128>(a, pdl, st);
}

int tree_device_error(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_tree_err, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v) {
    const int z = 0;
    cudaMemcpyToSymbol(g_tree_err, &z, sizeof(int));
  }
  return v;
}

}  // namespace lfm2q
