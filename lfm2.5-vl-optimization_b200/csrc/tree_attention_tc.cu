// Attention of drafted tokens over a paged KV cache on the fifth-generation tensor cores: the kernel for caches whose
// pages are multiples of 8 positions (tree_attention.cu has the mathematics, the form for other pages, and the join of
// the splits).
//
// A unit is a row tile (128 rows: queries times heads of one KV head) of one request, or two of them that share the K and
// V tiles; the tiles of all units are one line that is cut into equal stretches, one a block (TreePlan). One warp works
// out the block's stretches and streams them: the queries and K and V tiles of 64 positions by TMA into 128-byte-swizzled
// stages (boxes of up to 64 rows that never cross a page; one lane a box). Per row tile one warp issues tcgen05.mma:
// S = Q K^T into one of two 64-column TMEM buffers, then O += P V with P read from TMEM and V as it is in the cache (an
// MN-major operand); four warps do the softmax, one thread a row, so that a row's maximum and sum need no exchange
// between lanes. While tile n is in the softmax, S of tile n + 1 is ready, S of tile n + 2 follows as soon as tile n is
// read, and O of tile n - 1 is accumulated. O stays in TMEM; it is rescaled only when a row's maximum has grown by more
// than 2^8 since the last time (2^4 for fp16; the probabilities then reach at most 2^8, or 2^15 as fp16's are raised by
// 2^11, as exact as below 1), rarely after the first tiles.
//
// What bounds it, by the rows a KV head has (bf16, 32 heads over 8 KV heads of 64, pages of 64). Few rows: the cache's
// bytes. 64 requests x 1 token x 8000 positions: 188 to 214 us from one allocation of the cache to the next, 4.9 to 5.6
// TB/s, 75 to 85 % of the measured copy rate; 32 requests x 16
// drafts x 500 to 4000 positions: 44 us, of which 30 at 5.0 TB/s, 4 until the first tile, 5 in the join. Many rows: the
// softmax. 16 requests x 64 drafts x 8000 to 32000 positions: 305 us, 2.2 TB/s and 0.39 PFLOP/s; without its exponentials
// the same loop took 243 us of 319, without the softmax 201 us. Two row tiles a block
// halve the reads of the cache there; with one row tile (at most 128 rows a request) and heads of 64 two blocks share an SM
// and one loads while the other is in its softmax. Heads of 128: 100 requests x 1 token x 100 to 3000 positions 144 us,
// 4.4 TB/s.
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
constexpr int TT_ATOM = TT_ROWS * 128;         // 64 dims of the query tile
constexpr int TT_HALF = TA_KEYS * 128;         // 64 dims of a K (or V) tile
constexpr long long TT_WAIT_LIMIT = 1ll << 31;
// What a row's maximum may grow before O is rescaled, and how far the probabilities are raised, both in log2. fp16 ends at
// 2^16 and has fixed steps below 2^-14: raised by 11, a probability keeps its 11 bits down to 2^-25 of the largest, and is
// off by at most 2^-36 below that (unraised 2^-25: 32000 keys of 2^-25 each under one of 1 came out as none, 9e-4 of the
// result). bf16 has fp32's exponents.
template <class T>
struct Range {
  static constexpr float SLACK = 8.f, RAISE = 0.f;
};
template <>
struct Range<__half> {
  static constexpr float SLACK = 4.f, RAISE = 11.f;
};

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
// from one 64-wide block to the next (bytes). A descriptor is its low word (the address in 16-byte units and lbo), kept
// in a register and stepped by additions, and one constant high word: the issuing thread's instructions are on the
// pipeline's critical path (descriptors built anew for every MMA took 1000 of the 1900 cycles of a tile).
__device__ __forceinline__ uint32_t sw128_lo(uint32_t saddr, uint32_t lbo) {
  return ((saddr & 0x3FFFFu) >> 4) | (lbo >> 4) << 16;
}
constexpr uint32_t SW128_HI = (1024u >> 4) | 1u << 14 | 2u << 29;
// kind::f16 instruction descriptor, fp32 accumulation, M = 128
__host__ __device__ constexpr uint32_t idesc_f16(int n, bool bf, bool b_mn_major) {
  return (1u << 4) | (bf ? (1u << 7) | (1u << 10) : 0u) | (b_mn_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(TT_ROWS >> 4) << 24);
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "n"(SW128_HI), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_lo), "n"(SW128_HI), "r"(idesc), "r"(accumulate)
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
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {  // and waits
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// wait for this thread's TMEM loads, the registers tied to the wait so that no use of them moves before it
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : TT_REGS32(r, TT_TIE) : : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// every lane of a warp waits
__device__ __forceinline__ bool lanes_wait(uint32_t bar, uint32_t parity, volatile int *stop) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, stop));
}

template <int D, int PIPE>
struct TcShape {
  static constexpr int HALVES = D / 64;
  static constexpr int THREADS = 32 * (5 * PIPE + 1);  // per row tile four softmax warps and one that issues MMAs
  // One row tile: two blocks share an SM at D = 64; at D = 128 they would have room for two stages each, and one block with
  // five is faster (32 requests x 16 drafts 89 -> 84 us, 100 requests x 1 token 158 -> 147).
  // TMEM columns of a row tile: S0 | S1 | O (| P0 | P1 where there is room, 84 -> 82 us; else P lies over its S)
  static constexpr bool OWN_P = D == 64 || PIPE == 1;
  static constexpr int O_COL = 2 * TA_KEYS, P_COL = O_COL + D;
  static constexpr int TMEM_COLS = PIPE == 1 && D == 64 ? 256 : 512;
  static constexpr int BLOCKS = PIPE == 1 && D == 64 ? 2 : 1;  // an SM
  static constexpr int STAGES = PIPE == 1 ? 5 : (D == 64 ? 8 : 4);
  static constexpr int Q_BYTES = HALVES * TT_ATOM;   // per row tile
  static constexpr int KV_BYTES = HALVES * TT_HALF;  // a K (or V) tile
  static constexpr int OUT_BYTES = 2048;             // per softmax warp: 64 bytes of its 32 rows on their way out
  static constexpr int SMEM = PIPE * (Q_BYTES + 4 * OUT_BYTES) + 2 * STAGES * KV_BYTES + 1024;  // 1024: to align the base
};

// A stretch of one unit's tiles. The loading warp works out the block's segments and hands each to the other warps in
// shared memory together with its queries; tiles = 0 ends the block.
struct Segment {
  int b, kvh, tok0, n0;       // request, KV head, first query of the unit, the request's first row of q
  int T, ctx, t0, tiles;      // queries and cached positions of the request; the stretch
  int part, parts;            // which part of the unit this is, of how many
};

// A warp's rows of O times inv, to base + rel D: in the output's type, or fp32. 16 dims at a time go through shared memory
// (`stage`, 2 KB), so that two or four lanes write one row's bytes: stores of 16 bytes to 32 rows at once take 32 turns of
// the memory pipe each (5 requests x 13 drafts, 104 rows of 128: 19.3 us so, 18.0 us through shared memory). Out of line:
// the registers of the loop over the tiles are full.
template <class T, int D, bool OUT>
__device__ __noinline__ void rows_out(uint32_t t_o, float inv, uint4 *stage, void *base, int rel, int rows) {
  constexpr int PIECES = OUT ? 2 : 4, LG = OUT ? 1 : 2, BYTES = D * (OUT ? 2 : 4);  // pieces of 16 bytes a row
  const int lane = threadIdx.x & 31, x = lane & (PIECES - 1);
  uint8_t *dst[PIECES];
  const uint4 *src[PIECES];
#pragma unroll
  for (int k = 0; k < PIECES; ++k) {
    const int r = (32 * k + lane) >> LG;
    dst[k] = static_cast<uint8_t *>(base) + (size_t)__shfl_sync(0xffffffffu, rel, r) * BYTES + 16 * x;
    src[k] = stage + (r << LG) + (x ^ (r >> LG & (PIECES - 1)));
  }
#pragma unroll 1
  for (int c = 0; c < D / 16; ++c) {
    uint32_t o[16];
    tmem_ld16(t_o + 16 * c, o);
#pragma unroll
    for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * inv);
    if (OUT) {
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = Pair<T>::pack(__uint_as_float(o[2 * j]), __uint_as_float(o[2 * j + 1]));
    }
#pragma unroll
    for (int k = 0; k < PIECES; ++k)
      stage[(lane << LG) + (k ^ (lane >> LG & (PIECES - 1)))] =
          make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
    __syncwarp();
    uint4 w[PIECES];
#pragma unroll
    for (int k = 0; k < PIECES; ++k) w[k] = *src[k];
    __syncwarp();
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      if ((32 * k + lane) >> LG < rows) *reinterpret_cast<uint4 *>(dst[k]) = w[k];
      dst[k] += 16 * PIECES;
    }
  }
}

// The drafts of `extra`, left out of the second product, added to a row of O: the score again from global memory, and
// p v. Rare, so out of line. For a whole warp.
template <class T, int D>
__device__ __noinline__ void add_apart(const TreeArgs &a, unsigned long long extra, uint32_t t_o, size_t row, int kvh,
                                       int ctx, const int *table, float m) {
  const uint32_t *qr = reinterpret_cast<const uint32_t *>(reinterpret_cast<const T *>(a.q) + row * D);
  for (int c = 0; c < D / 32; ++c) {
    uint32_t o[32];
    tmem_ld32(t_o + 32 * c, o);
    tmem_ld_wait(o);
    for (unsigned long long rest = extra; rest; rest &= rest - 1) {
      const int t = ctx + __ffsll(rest) - 1;
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
    __syncwarp();
    tmem_st32(t_o + 32 * c, o);
  }
  tmem_st_wait();
}

template <class T, int D, int PIPE>
__global__ void __launch_bounds__(TcShape<D, PIPE>::THREADS, TcShape<D, PIPE>::BLOCKS)
    tree_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                   const __grid_constant__ CUtensorMap tmV, const __grid_constant__ TreeArgs a, int box, int tpt) {
  using L = TcShape<D, PIPE>;
  constexpr int STAGES = L::STAGES, HALVES = L::HALVES;
  constexpr bool BF = std::is_same<T, bf16>::value;
  constexpr int W_TMA = 4 * PIPE, W_MMA = W_TMA + 1;
  constexpr int TMEM_COLS = L::TMEM_COLS;
  extern __shared__ uint8_t tt_smem[];
  __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES], q_full, q_empty, s_full[PIPE][2], p_full[PIPE][2],
      pv_done[PIPE], o_full[PIPE], drained[PIPE];
  __shared__ unsigned long long live[STAGES];  // keys of the stage's tile that exist
  __shared__ unsigned long long apart[4];      // drafts that were taken out of the second product, by segment
  __shared__ Segment segs[4];
  __shared__ uint32_t tmem_slot;
  __shared__ int stop;
  __shared__ int cleaned;  // tiles whose value rows the first warp has looked through
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(tt_smem) + 1023) & ~uintptr_t(1023));
  const uint32_t sq = smem_addr(smem), sk = sq + PIPE * L::Q_BYTES, sv = sk + STAGES * L::KV_BYTES;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(smem_addr(&full[i]), 1);
      mbar_init(smem_addr(&empty[i]), PIPE);
    }
    for (int p = 0; p < PIPE; ++p) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(smem_addr(&s_full[p][i]), 1);
        mbar_init(smem_addr(&p_full[p][i]), 4);
      }
      mbar_init(smem_addr(&pv_done[p]), 1);
      mbar_init(smem_addr(&o_full[p]), 1);
      mbar_init(smem_addr(&drained[p]), 1);
    }
    mbar_init(smem_addr(&q_full), 1);
    mbar_init(smem_addr(&q_empty), PIPE);
    stop = cleaned = 0;
    apart[0] = apart[1] = apart[2] = apart[3] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == W_TMA && lane < 3)
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(lane == 0 ? &tmQ : lane == 1 ? &tmK : &tmV))
                 : "memory");
  if (warp == W_MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)),
                 "r"(TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // The next kernel may start only now that this block has its tensor memory: one that took the SM's first would hold
  // it until this grid ends.
  pdl_trigger();
  pdl_wait();

  if (warp == W_TMA) {
    // ---------------------------------------------------------------- segments, queries, K and V tiles
    const TreePlan plan(a, PIPE * tpt * a.G, gridDim.x, blockIdx.x);
    const int boxes = TA_KEYS / box, page_step = TA_KEYS / a.page, row_step = TA_KEYS % a.page;
    int left = plan.count, b = plan.b, base = plan.base, st = 0, ph = 1;  // a fresh barrier passes a wait for phase 1
    // of request b: tiles of a unit, its span on the line, units of a head and in all; the next unit, tile within it
    Request rq;
    int tiles = 0, span = 0, per_head = 1, units = 0, unit = 0, j0 = 0;
    bool next = true, begun = false;
    uint32_t issued = 0, seg = 0;
    bool ok = true, more = true;
    for (; ok && more; ++seg) {
      more = false;
      Segment g = {};
      int t1 = 0;
      while (left > 0 && b < a.B) {
        if (next) {
          rq = plan.request(a, b);
          tiles = plan.tiles(rq);
          span = plan.span(a, tiles);
          per_head = plan.per_head(a, rq);
          units = rq.T > 0 ? a.NKV * per_head : 0;
          unit = begun ? 0 : (plan.x0 - base) / span;
          j0 = begun ? 0 : plan.x0 - base - unit * span;
          next = false;
          begun = true;
        }
        if (unit == units) {
          base += units * span;
          ++b;
          next = true;
          continue;
        }
        const int step = min(span - j0, left), from = j0, u = unit, first = base + unit * span;
        left -= step;
        j0 += step;
        if (j0 == span) {
          ++unit;
          j0 = 0;
        }
        const int take = a.S == 1 ? tiles : min(tiles - from, step);
        if (take <= 0) continue;  // the end of a unit's span holds no tiles
        // the stretches that hold the unit's first tile and its last, of which this is number blockIdx.x
        int part0 = blockIdx.x, part1 = part0;
        if (a.S > 1) {
          const int end = first + tiles - 1;
          if (first < plan.x0) part0 = first / plan.quota;
          if (end - plan.x0 >= plan.quota) part1 = end / plan.quota;
        }
        const int kvh = per_head == 1 ? u : u / per_head;
        g = {b, kvh, (u - kvh * per_head) * PIPE * tpt, rq.n0, rq.T, rq.ctx, from * TA_KEYS, take,
             (int)blockIdx.x - part0, part1 - part0 + 1};
        t1 = min(rq.len, (from + take) * TA_KEYS);
        more = true;
        break;
      }
      // Page numbers come a tile ahead, one lane a box: their load takes as long as a tile (loaded where they were used,
      // the loading warp bounded the kernel, 217 us where it is 185 now).
      const int *table = a.table + (size_t)g.b * a.width;
      const int at0 = g.t0 + lane * box;
      int idx = at0 / a.page, y = at0 - idx * a.page;
      int ahead = lane < boxes && at0 < t1 ? __ldcg(table + idx) : -1;
      // the queries' place is free when the last scores of the segment before are done
      ok = warp_wait(smem_addr(&q_empty), (seg & 1) ^ 1, &stop);
      if (!ok) break;
      if (lane == 0) {
        segs[seg & 3] = g;
        const int tiles_q = !more ? 0 : PIPE > 1 && g.T - g.tok0 > tpt ? 2 : 1;
        mbar_expect_tx(smem_addr(&q_full), tiles_q * HALVES * tpt * a.G * 128);
        for (int p = 0; p < tiles_q; ++p)
          for (int h = 0; h < HALVES; ++h)
            tma_load_3d(sq + p * L::Q_BYTES + h * TT_ATOM, &tmQ, smem_addr(&q_full), 64 * h, g.kvh * a.G,
                        g.n0 + g.tok0 + p * tpt);
      }
      for (int n = 0; n < g.tiles; ++n, ++issued) {
        const int t = at0 + n * TA_KEYS, pg = ahead, row = y;
        idx += page_step;
        y += row_step;
        if (y >= a.page) {
          y -= a.page;
          ++idx;
        }
        ahead = n + 1 < g.tiles && lane < boxes && t + TA_KEYS < t1 ? __ldcg(table + idx) : -1;
        const bool there = pg >= 0 && pg < a.num_pages;
        unsigned long long keys = 0;  // of this lane's box
        if (there) {
          const int n_live = min(box, t1 - t);
          keys = (n_live >= 64 ? ~0ull : (1ull << n_live) - 1) << (lane * box);
        }
        const uint32_t loads = __popc(__ballot_sync(0xffffffffu, there));
        const uint32_t klo = __reduce_or_sync(0xffffffffu, (uint32_t)keys),
                       khi = __reduce_or_sync(0xffffffffu, (uint32_t)(keys >> 32));
        ok = warp_wait(smem_addr(&empty[st]), (uint32_t)ph, &stop);
        if (!ok) break;
        const uint32_t bar = smem_addr(&full[st]);
        if (lane == 0) {
          live[st] = (unsigned long long)khi << 32 | klo;
          mbar_expect_tx(bar, 2 * loads * box * 128 * HALVES);
        }
        __syncwarp();
        if (there) {
          const uint32_t to = st * L::KV_BYTES + lane * box * 128;
          const int z = pg * a.NKV + g.kvh;
#pragma unroll
          for (int h = 0; h < HALVES; ++h) tma_load_3d(sk + to + h * TT_HALF, &tmK, bar, 64 * h, row, z);
#pragma unroll
          for (int h = 0; h < HALVES; ++h) tma_load_3d(sv + to + h * TT_HALF, &tmV, bar, 64 * h, row, z);
        }
        if (++st == STAGES) {
          st = 0;
          ph ^= 1;
        }
      }
    }
    if (!ok && lane == 0) {  // gave up: no copy may land after the block has left
      int late = 0;
      for (uint32_t n = issued > STAGES ? issued - STAGES : 0; n < issued; ++n) {
        mbar_wait(smem_addr(&full[n % STAGES]), (n / STAGES) & 1, &late);
      }
      if (seg > 0) mbar_wait(smem_addr(&q_full), (seg - 1) & 1, &late);
    }
  } else if (warp >= W_MMA) {
    // ---------------------------------------------------------------- MMAs of row tile p
    // One thread issues them, and what it does a tile (waits of 100 cycles, MMAs of 60, commits of 80) bounds the tile
    // when it is much: so a warp of its own for every row tile, one barrier for K and V, and no wait that the order of
    // the MMAs makes needless.
    if (lane == 0) {
      constexpr uint32_t ID_S = idesc_f16(TA_KEYS, BF, false), ID_O = idesc_f16(D, BF, true);
      const int p = warp - W_MMA;
      const uint32_t q_lo = sw128_lo(sq + p * L::Q_BYTES, 16), k_lo = sw128_lo(sk, 16), v_lo = sw128_lo(sv, TT_HALF);
      const uint32_t t_s = tmem + 256 * p, t_o = t_s + L::O_COL, t_p = L::OWN_P ? t_s + L::P_COL : t_s;
      constexpr uint32_t P_STEP = L::OWN_P ? TA_KEYS / 2 : TA_KEYS;
      int kst = 0, kph = 0, st = 0;  // stage and phase of the next scores' tile, stage of the next product's
      uint32_t cnt = 0, seg = 0;     // tiles and segments so far
      bool ok = true;
      auto scores = [&](uint32_t i) {
        ok = mbar_wait(smem_addr(&full[kst]), (uint32_t)kph, &stop);
        if (!ok) return;
        tc_fence_after();
        const uint32_t kt = k_lo + kst * (L::KV_BYTES / 16);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_ss(t_s + i * TA_KEYS, q_lo + (k >> 2) * (TT_ATOM / 16) + 2 * (k & 3),
                  kt + (k >> 2) * (TT_HALF / 16) + 2 * (k & 3), ID_S, k != 0);
        umma_commit(smem_addr(&s_full[p][i]));
        if (++kst == STAGES) {
          kst = 0;
          kph ^= 1;
        }
      };
      for (;; ++seg) {
        ok = mbar_wait(smem_addr(&q_full), seg & 1, &stop);
        if (!ok) break;
        const int tiles = *(volatile int *)&segs[seg & 3].tiles;
        if (tiles == 0) break;
        // Scores run two tiles ahead of the softmax's end, so that it always finds the next tile ready.
        scores(cnt & 1);
        if (ok && tiles > 1) scores((cnt + 1) & 1);
        for (int n = 0; n < tiles && ok; ++n, ++cnt) {
          const uint32_t i = cnt & 1;
          ok = mbar_wait(smem_addr(&p_full[p][i]), (cnt >> 1) & 1, &stop);
          if (!ok) break;
          tc_fence_after();
          const uint32_t vt = v_lo + st * (L::KV_BYTES / 16), pt = t_p + i * P_STEP;
#pragma unroll
          for (int k = 0; k < TA_KEYS / 16; ++k) umma_ts(t_o, pt + 8 * k, vt + k * (2048 / 16), ID_O, (n | k) != 0);
          umma_commit(smem_addr(&empty[st]));
          if (n == tiles - 1) umma_commit(smem_addr(&o_full[p]));
          if (!L::OWN_P || n == tiles - 2) umma_commit(smem_addr(&pv_done[p]));
          if (n + 2 < tiles) {
            // S of tile n + 2 goes where tile n's was: read by the softmax (p_full), and where P lies over it multiplied
            if (!L::OWN_P) ok = mbar_wait(smem_addr(&pv_done[p]), i, &stop);
            if (ok) scores(i);
          } else if (!L::OWN_P) {
            ok = mbar_wait(smem_addr(&pv_done[p]), i, &stop);
          }
          // the queries have been read; not before the softmax has taken this segment up (its barrier then is at most
          // one phase ahead of any waiter)
          if (ok && n == max(tiles - 3, 0)) umma_commit(smem_addr(&q_empty));
          if (++st == STAGES) st = 0;
        }
        if (!ok) break;
      }
      if (!ok) {  // gave up: the MMAs in flight finish first
        int late = 0;
        umma_commit(smem_addr(&drained[p]));
        mbar_wait(smem_addr(&drained[p]), 0, &late);
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax, one thread a row
    const int pipe = warp >> 2, quarter = warp & 3, row = threadIdx.x & (TT_ROWS - 1);
    const uint32_t tbase = tmem + 256 * pipe + ((uint32_t)(quarter * 32) << 16);
    const uint32_t t_o = tbase + L::O_COL;
    const int my_tok = row / a.G, my_head = row - my_tok * a.G;
    uint4 *out_stage = reinterpret_cast<uint4 *>(smem + PIPE * L::Q_BYTES + 2 * STAGES * L::KV_BYTES + warp * L::OUT_BYTES);
    uint32_t cnt = 0, seg = 0, pairs = 0;  // tiles, segments, segments of two tiles or more
    int st = 0, ph = 0, edges = 0;
    bool ok = true;
    for (;; ++seg) {
      ok = lanes_wait(smem_addr(&q_full), seg & 1, &stop);
      if (!ok) break;
      const volatile Segment *g = &segs[seg & 3];
      const int tiles = g->tiles, ctx = g->ctx, t0 = g->t0;
      if (tiles == 0) break;
      const int tok0 = g->tok0 + pipe * tpt, toks = min(g->T - tok0, tpt);  // this row tile's queries (none: <= 0)
      const bool active = quarter * 32 < toks * a.G, has = row < toks * a.G;
      unsigned long long see = 0;
      if (has) {
        const int tok = tok0 + my_tok;
        see = a.mask ? __ldcg(a.mask + g->n0 + tok) : (tok >= 63 ? ~0ull : (2ull << tok) - 1);
      }
      float m = -INFINITY, l = 0.f;  // m: the maximum less what the probabilities are raised by
      for (int n = 0; n < tiles; ++n, ++cnt) {
        const uint32_t sbuf = tbase + (cnt & 1) * TA_KEYS;
        const uint32_t pbuf = L::OWN_P ? tbase + L::P_COL + (cnt & 1) * (TA_KEYS / 2) : sbuf;
        const uint32_t pbar = smem_addr(&p_full[pipe][cnt & 1]);
        ok = lanes_wait(smem_addr(&s_full[pipe][cnt & 1]), (cnt >> 1) & 1, &stop);
        if (!ok) break;
        const unsigned long long exists = *(volatile unsigned long long *)&live[st];
        const int d0 = t0 + n * TA_KEYS - ctx;  // draft of the tile's first key
        const bool edge = d0 > -TA_KEYS || exists != ~0ull;
        edges += edge;
        if (!active) {
          if (lane == 0) mbar_arrive(pbar);  // keeps step: a row tile's barriers count all four warps
        } else {
          tc_fence_after();
          uint32_t s0[32], s1[32];
          tmem_ld32(sbuf, s0);
          tmem_ld32(sbuf + 32, s1);
          unsigned long long vis = exists;  // keys of the tile that this row sees
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
          // The probabilities with the maximum so far, while the tile's own is found (the exponentials and the
          // comparisons run on different units); again where that has grown too much, which is rare.
          const float2 c2 = make_float2(a.scale_log2, a.scale_log2);
          uint32_t p[32];
          float sum;
          auto probabilities = [&]() {
            const float ms = m == -INFINITY ? 0.f : m;
            const float2 m2 = make_float2(-ms, -ms);
            float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float2 x = ffma2(make_float2(__uint_as_float(s0[2 * j]), __uint_as_float(s0[2 * j + 1])), c2, m2);
              const float2 y = ffma2(make_float2(__uint_as_float(s1[2 * j]), __uint_as_float(s1[2 * j + 1])), c2, m2);
              const float2 e = make_float2(ex2(x.x), ex2(x.y)), f = make_float2(ex2(y.x), ex2(y.y));
              p[j] = Pair<T>::pack(e.x, e.y);
              p[16 + j] = Pair<T>::pack(f.x, f.y);
              sum0 = fadd2(sum0, e);
              sum1 = fadd2(sum1, f);
            }
            sum = (sum0.x + sum0.y) + (sum1.x + sum1.y);
          };
          auto largest = [&]() {
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 32; ++j) mx[j & 3] = max3(mx[j & 3], __uint_as_float(s0[j]), __uint_as_float(s1[j]));
            return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2;
          };
          // (a unit's first tile starts with its own: 0.4 us of 11.5 for one token; of no use to the long units of PIPE 2)
          if (PIPE == 1 && n == 0) m = largest() - Range<T>::RAISE;
          probabilities();
          const float top = largest();
          const bool grow = top > m + (Range<T>::RAISE + Range<T>::SLACK) || (m == -INFINITY && top > -INFINITY);
          if (__any_sync(0xffffffffu, grow)) {
            const float corr = grow ? ex2(m - (top - Range<T>::RAISE)) : 1.f;  // 0 while the row has seen nothing
            if (grow) m = top - Range<T>::RAISE;
            l *= corr;
            if (n > 0) {
              // the product of tile n - 1: done when S of tile n + 1 is, which was issued after it
              ok = !L::OWN_P ? lanes_wait(smem_addr(&pv_done[pipe]), (cnt - 1) & 1, &stop)
                   : n + 1 < tiles
                       ? lanes_wait(smem_addr(&s_full[pipe][(cnt + 1) & 1]), ((cnt + 1) >> 1) & 1, &stop)
                       : lanes_wait(smem_addr(&pv_done[pipe]), pairs & 1, &stop);
              if (!ok) break;
              tc_fence_after();
#pragma unroll
              for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tmem_ld32(t_o + 32 * c, o);
                tmem_ld_wait(o);
#pragma unroll
                for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * corr);
                tmem_st32(t_o + 32 * c, o);
              }
            }
            probabilities();
          }
          l += sum;
          tmem_st32(pbuf, p);
          // A key that a row does not see has p = 0, but 0 times an infinity or a NaN is a NaN: value rows that hold
          // one are zeroed in shared memory (stale ones of keys that do not exist, too), and drafts among them are
          // added at the end to the rows that see them. The first warp does it, and the other row tile's first warp
          // waits for it, before they let the product go ahead.
          if (edge && warp == 0) {
            ok = lanes_wait(smem_addr(&full[st]), (uint32_t)ph, &stop);  // it has landed: S came of it
            if (!ok) break;
#pragma unroll
            for (int h2 = 0; h2 < 2; ++h2) {
              const int r = h2 * 32 + lane;
              const bool there = (exists >> r) & 1;
              const bool look = d0 + r >= 0 || !there;
              if (!__any_sync(0xffffffffu, look)) continue;
              uint4 *vr = reinterpret_cast<uint4 *>(smem + PIPE * L::Q_BYTES + STAGES * L::KV_BYTES + st * L::KV_BYTES +
                                                    r * 128);
              bool bad = false;
              for (int h = 0; h < HALVES; ++h)
#pragma unroll
                for (int c = 0; c < 8; ++c) {  // every lane at another 16 bytes of its row: no bank twice
                  const uint4 u = vr[h * (TT_HALF / 16) + ((c + lane) & 7)];
                  bad = bad ||
                        !(Pair<T>::finite(u.x) && Pair<T>::finite(u.y) && Pair<T>::finite(u.z) && Pair<T>::finite(u.w));
                }
              if (bad && look) {
                for (int h = 0; h < HALVES; ++h)
                  for (int c = 0; c < 8; ++c) vr[h * (TT_HALF / 16) + c] = make_uint4(0, 0, 0, 0);
                if (there) atomicOr(&apart[seg & 3], 1ull << (d0 + r));
              }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (PIPE > 1 && lane == 0) {
              __threadfence_block();
              *(volatile int *)&cleaned = edges;
            }
          } else if (PIPE > 1 && edge && warp == 4) {
            const long long since = clock64();
            while (ok && *(volatile int *)&cleaned < edges)
              ok = *(volatile int *)&stop == 0 && clock64() - since < TT_WAIT_LIMIT;
            ok = __all_sync(0xffffffffu, ok);
            __threadfence_block();
            if (!ok) {
              stop = 1;
              atomicCAS(&g_tree_err, 0, 1);
              break;
            }
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(pbar);
        }
        if (++st == STAGES) {
          st = 0;
          ph ^= 1;
        }
      }
      pairs += tiles > 1;
      // ---------------------------------------------------------------- out, or this split's partial
      ok = ok && lanes_wait(smem_addr(&o_full[pipe]), seg & 1, &stop) && *(volatile int *)&stop == 0;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      // The word of two segments on: every row tile has left the segment two back, whose word that was (this one's
      // last product came after all of the last one's, whose P came after that).
      if (warp == 0 && lane == 0) apart[(seg + 2) & 3] = 0;
      if (!active) continue;
      tc_fence_after();
      const int parts = g->parts;
      const int rel = (tok0 + my_tok) * a.NQ + my_head, rows = toks * a.G - quarter * 32;
      const size_t first_row = (size_t)g->n0 * a.NQ + g->kvh * a.G;
      const float inv = l == 0.f ? 0.f : __fdividef(1.f, l);
      const unsigned long long extra = *(volatile unsigned long long *)&apart[seg & 3] & see;
      if (__any_sync(0xffffffffu, extra != 0))
        add_apart<T, D>(a, extra, t_o, first_row + rel, g->kvh, ctx, a.table + (size_t)g->b * a.width, m);
      if (parts == 1)
        rows_out<T, D, true>(t_o, inv, out_stage, reinterpret_cast<T *>(a.out) + first_row * D, rel, rows);
      else
        rows_out<T, D, false>(t_o, inv, out_stage, ws_acc(a, D, g->part, first_row), rel, rows);
      if (a.S > 1 && has) {
        float *info = ws_row(a, D, first_row + rel);
        if (parts > 1) info[1 + g->part] = l == 0.f ? -INFINITY : m + __log2f(l);
        if (g->part == 0) reinterpret_cast<int *>(info)[0] = parts;
      }
      tc_fence_before();  // O has been read, before the next segment's first product (ordered by its P)
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == W_MMA) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
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

// [z, y, D] with 64 dims x rows of y x depth of z a box, 128-byte swizzle; boxes past the end read zeros
bool make_map(CUtensorMap *map, const void *ptr, int D, long long y, long long z, int rows, int depth, bool half) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)y, (cuuint64_t)z};
  const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)D * 2 * y};
  const cuuint32_t boxes[3] = {64, (cuuint32_t)rows, (cuuint32_t)depth}, es[3] = {1, 1, 1};
  return fn(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(ptr),
            dims, strides, boxes, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int D, int PIPE>
cudaError_t launch(const TreeArgs &a, bool pdl, cudaStream_t st) {
  using L = TcShape<D, PIPE>;
  auto kernel = tree_tc_kernel<T, D, PIPE>;
  static std::atomic<int> attr_set[64];  // the shared-memory opt-in, once per device
  int dev = 0;
  if (const cudaError_t e = cudaGetDevice(&dev)) return e;
  if (dev < 64 && !attr_set[dev].load(std::memory_order_acquire)) {
    if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM))
      return e;
    attr_set[dev].store(1, std::memory_order_release);
  }
  int box = TA_KEYS;  // rows of a TMA box: the largest power of two up to a tile that divides the page
  while (a.page % box) box /= 2;
  const int tpt = TT_ROWS / a.G;  // queries per row tile: whole ones, so that a box of the query map is a row tile
  CUtensorMap mq, mk, mv;
  const bool half = !std::is_same<T, bf16>::value;
  const long long heads = (long long)a.num_pages * a.NKV;
  if (!make_map(&mq, a.q, D, a.NQ, a.N, a.G, tpt, half) || !make_map(&mk, a.kc, D, a.page, heads, box, 1, half) ||
      !make_map(&mv, a.vc, D, a.page, heads, box, 1, half))
    return cudaErrorNotSupported;
  cudaLaunchAttribute attr;
  cudaLaunchConfig_t cfg = pdl_config(dim3(L::BLOCKS * device_sm_count()), dim3(L::THREADS), pdl, st, &attr);
  cfg.dynamicSmemBytes = L::SMEM;
  return cudaLaunchKernelEx(&cfg, kernel, mq, mk, mv, a, box, tpt);
}
template <class T, int D>
cudaError_t launch_form(const TreeArgs &a, bool pdl, cudaStream_t st) {
  // Up to 128 rows a request: one row tile a block. More: two row tiles a block, which share the K and V tiles.
  if (a.max_q <= TT_ROWS / a.G) return launch<T, D, 1>(a, pdl, st);
  return launch<T, D, 2>(a, pdl, st);
}

}  // namespace

cudaError_t launch_tree_tc(const TreeArgs &a, int D, bool half, bool pdl, cudaStream_t st) {
  if (half) return D == 64 ? launch_form<__half, 64>(a, pdl, st) : launch_form<__half, 128>(a, pdl, st);
  return D == 64 ? launch_form<bf16, 64>(a, pdl, st) : launch_form<bf16, 128>(a, pdl, st);
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
