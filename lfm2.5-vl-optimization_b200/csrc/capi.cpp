// C ABI of liblfm2q (include/lfm2q.h): host-side argument checks, device check, dispatch to the launchers.
//
// The checks restate the reference bindings' TORCH_CHECKs (kernels/int8_gemm.cpp:20-141,
// kernels/lfm2_decode.cpp:73-150) with the limits of this build, and run before anything touches the device,
// so a bad call returns LFM2Q_EINVAL (and a message) on any machine, with or without a GPU.
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <cstdio>
#include <mutex>
#include <cstring>
#include <string>
#include <vector>

#include "../../include/lfm2q.h"
#include "launch.h"

namespace lfm2q {

static thread_local std::string g_last_error;
static std::atomic<bool> g_pdl{true};

static int fail(int code, const std::string &msg) {
  g_last_error = msg;
  return code;
}

static bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Device facts, filled once per device (std::call_once: concurrent first calls from several threads see the
// complete record).
struct DevInfo {
  int sms = 0;
  int supported = 0;
};
static DevInfo g_dev[64];
static std::once_flag g_dev_once[64];

static const DevInfo &dev_info() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    static const DevInfo none;
    return none;
  }
  std::call_once(g_dev_once[dev], [dev] {
    int major = 0, minor = 0, sms = 0;
    cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
    cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    g_dev[dev].sms = sms;
    g_dev[dev].supported = (major == 10 && minor == 0) ? 1 : 0;
  });
  return g_dev[dev];
}

int device_sm_count() {
  const int s = dev_info().sms;
  return s > 0 ? s : 148;
}
bool device_is_sm100() { return dev_info().supported == 1; }

static int device_gate() {
  if (!device_is_sm100())
    return fail(LFM2Q_ENOTSUP, "lfm2q: the current CUDA device is not an sm_100 (B200) GPU, or no device is visible");
  return LFM2Q_OK;
}

static int launched(cudaError_t e, const char *what) {
  if (e == cudaSuccess) return LFM2Q_OK;
  return fail(LFM2Q_ECUDA, std::string("lfm2q: ") + what + ": " + cudaGetErrorString(e));
}

#define REQUIRE(cond, msg) \
  do {                     \
    if (!(cond)) return fail(LFM2Q_EINVAL, std::string("lfm2q: ") + (msg)); \
  } while (0)

}  // namespace lfm2q

using namespace lfm2q;

extern "C" {

const char *lfm2q_last_error(void) { return g_last_error.c_str(); }

const char *lfm2q_version(void) { return "lfm2q 0.1.0 (sm_100a)"; }

int lfm2q_device_supported(void) { return device_is_sm100() ? 1 : 0; }

int lfm2q_check_device(int clear) {
  if (int e = device_gate()) return e;
  const int v = gemm_device_error(clear != 0);
  const int a = attn_device_error(clear != 0);
  const int t = tree_device_error(clear != 0);
  if (v) return fail(LFM2Q_ETIMEOUT, "lfm2q: a GEMM pipeline wait timed out on the device");
  if (a) return fail(LFM2Q_ETIMEOUT, "lfm2q: a decode-attention stage wait timed out on the device");
  if (t) return fail(LFM2Q_ETIMEOUT, "lfm2q: a tree-attention pipeline wait timed out on the device");
  return LFM2Q_OK;
}

int lfm2q_selftest_wait_timeout(int limit_log2, void *stream) {
  REQUIRE(limit_log2 >= 10 && limit_log2 <= 31, "limit_log2 must be in [10, 31] (clock cycles = 2^limit_log2)");
  if (int e = device_gate()) return e;
  return launched(launch_wait_timeout_selftest(limit_log2, (cudaStream_t)stream), "selftest_wait_timeout");
}

void lfm2q_set_pdl(int on) {
  g_pdl.store(on != 0);
  gemm_set_pdl(on != 0);
}
void lfm2q_set_gemv_trigger(int early) { gemv_set_early_trigger(early != 0); }
void lfm2q_set_gemv_impl(int) {}
void lfm2q_set_gemv_path(int path) { gemv_set_impl(path >= 1 && path <= 4 ? path : 0); }
void lfm2q_set_gemm_tile(int bn) { gemm_set_tile_override(bn); }

// ------------------------------------------------------------------ quantizers
int lfm2q_quant_rows(const uint16_t *x, int8_t *q, float *s, int rows, int K, void *stream) {
  REQUIRE(rows >= 0 && K > 0, "rows must be >= 0 and K > 0");
  REQUIRE(K % 8 == 0 && K <= 16384, "K must be a multiple of 8, <= 16384");
  REQUIRE(rows == 0 || (x && q && s), "x, q and s must be non-null");
  REQUIRE(aligned16(x) && aligned16(q), "x and q must be 16-byte aligned");
  if (rows == 0) return LFM2Q_OK;
  if (int e = device_gate()) return e;
  // programmatic dependent launch at every size: the quantizer's launch overlaps the previous kernel's tail and the
  // GEMM after it starts its weight loads early (config-5 job at 8192 rows per GPU: 13.6 -> 13.2 ms per step; no
  // change at 65536 rows)
  return launched(launch_quant_rows(x, q, s, rows, K, g_pdl.load(), (cudaStream_t)stream), "quant_rows");
}

int lfm2q_quant_groups(const uint16_t *x, int8_t *q, float *sT, int rows, int K, void *stream) {
  REQUIRE(rows >= 0 && K > 0, "rows must be >= 0 and K > 0");
  REQUIRE(K % 64 == 0 && K <= 16384, "grouped shapes: K must be a multiple of 64, <= 16384");
  REQUIRE(rows == 0 || (x && q && sT), "x, q and s must be non-null");
  REQUIRE(aligned16(x) && aligned16(q), "x and q must be 16-byte aligned");
  if (rows == 0) return LFM2Q_OK;
  if (int e = device_gate()) return e;
  return launched(launch_quant_groups(x, q, sT, rows, K, g_pdl.load(), (cudaStream_t)stream),
                  "quant_groups");
}

// ------------------------------------------------------------------ GEMMs
static int check_gemm_common(const void *w, const float *sw, const uint16_t *bias, const void *y, int M, int N,
                             int K) {
  REQUIRE(M >= 0 && N > 0 && K > 0, "need M >= 0, N > 0, K > 0");
  REQUIRE(K % 16 == 0 && N % 8 == 0, "need K % 16 == 0 and N % 8 == 0");
  REQUIRE(w && sw && y, "w, sw and y must be non-null");
  REQUIRE(aligned16(w) && aligned16(sw) && aligned16(y) && aligned16(bias), "w, sw, bias and y must be 16-byte aligned");
  return LFM2Q_OK;
}

int lfm2q_gemm_i8(const int8_t *xq, const float *sx, int grouped, const int8_t *w, const float *sw,
                  const uint16_t *bias, uint16_t *y, int M, int N, int K, int gelu, void *stream) {
  if (int e = check_gemm_common(w, sw, bias, y, M, N, K)) return e;
  REQUIRE(M == 0 || (xq && sx), "xq and sx must be non-null");
  REQUIRE(aligned16(xq), "xq must be 16-byte aligned");
  if (grouped) REQUIRE(K % 64 == 0, "sx shape: grouped scales need K % 64 == 0");
  if (M == 0) return LFM2Q_OK;
  if (int e = device_gate()) return e;
  return launched(launch_gemm_i8(xq, sx, w, sw, bias, y, M, N, K, gelu != 0, grouped != 0, (cudaStream_t)stream),
                  "gemm_i8");
}

int lfm2q_gemm_i8_q(const int8_t *xq, const float *sxT, const int8_t *w, const float *sw, const uint16_t *bias,
                    int8_t *yq, float *ysT, int M, int N, int K, int gelu, void *stream) {
  REQUIRE(M >= 0 && N > 0 && K > 0, "need M >= 0, N > 0, K > 0");
  REQUIRE(K % 64 == 0, "sxT shape: K must be a multiple of 64");
  REQUIRE(N % 128 == 0, "w [N, K] with N % 128 == 0");
  REQUIRE(w && sw && yq && ysT && (M == 0 || (xq && sxT)), "pointers must be non-null");
  REQUIRE(aligned16(xq) && aligned16(w) && aligned16(sw) && aligned16(bias) && aligned16(yq),
          "xq, w, sw, bias and yq must be 16-byte aligned");
  if (M == 0) return LFM2Q_OK;
  if (int e = device_gate()) return e;
  return launched(launch_gemm_i8_q(xq, sxT, w, sw, bias, yq, ysT, M, N, K, gelu != 0, (cudaStream_t)stream),
                  "gemm_i8_q");
}

int lfm2q_gemm_i8_silu(const int8_t *xq, const float *sx, const int8_t *w, const float *sw, const uint16_t *bias,
                       uint16_t *y, int M, int I, int K, void *stream) {
  REQUIRE(M >= 0 && I > 0 && K > 0, "need M >= 0, I > 0, K > 0");
  REQUIRE(K % 16 == 0 && I % 8 == 0, "need K % 16 == 0 and I % 8 == 0");
  REQUIRE(w && sw && y && (M == 0 || (xq && sx)), "pointers must be non-null");
  REQUIRE(aligned16(xq) && aligned16(w) && aligned16(sw) && aligned16(bias) && aligned16(y),
          "xq, w, sw, bias and y must be 16-byte aligned");
  REQUIRE(aligned16(sw + I) && aligned16(bias ? bias + I : nullptr), "I must keep the up-half scales 16-byte aligned");
  if (M == 0) return LFM2Q_OK;
  if (int e = device_gate()) return e;
  return launched(launch_gemm_i8_silu(xq, sx, w, sw, bias, y, M, I, K, (cudaStream_t)stream), "gemm_i8_silu");
}

int lfm2q_gemm_w8(const uint16_t *x, const int8_t *w, const float *sw, const uint16_t *bias, uint16_t *y, int M,
                  int N, int K, int gelu, void *stream) {
  if (int e = check_gemm_common(w, sw, bias, y, M, N, K)) return e;
  REQUIRE(M == 0 || x, "x must be non-null");
  REQUIRE(aligned16(x), "x must be 16-byte aligned");
  if (M == 0) return LFM2Q_OK;
  if (int e = device_gate()) return e;
  return launched(launch_gemm_w8(x, w, sw, bias, y, M, N, K, gelu != 0, (cudaStream_t)stream), "gemm_w8");
}

// ------------------------------------------------------------------ producers
int lfm2q_add_layernorm_q(uint16_t *h, const uint16_t *y, const uint16_t *w, const uint16_t *b, int8_t *q, float *s,
                          int rows, int D, float eps, int grouped, void *stream) {
  REQUIRE(rows >= 0 && D > 0, "rows must be >= 0 and D > 0");
  REQUIRE(D % 8 == 0 && D <= 16384, "D must be a multiple of 8, <= 16384");
  if (grouped) REQUIRE(D % 64 == 0, "s shape: grouped scales need D % 64 == 0");
  REQUIRE(h && w && b && q && s, "h, w, b, q and s must be non-null");
  REQUIRE(aligned16(h) && aligned16(y) && aligned16(w) && aligned16(b) && aligned16(q),
          "h, y, w, b and q must be 16-byte aligned");
  if (rows == 0) return LFM2Q_OK;
  if (int e = device_gate()) return e;
  return launched(launch_add_layernorm_q(h, y, w, b, q, s, rows, D, eps, grouped != 0, (cudaStream_t)stream),
                  "add_layernorm_q");
}

int lfm2q_add_rmsnorm_q(uint16_t *h, const uint16_t *y, const uint16_t *w, int8_t *q, float *s, int rows, int H,
                        float eps, int grouped, void *stream) {
  REQUIRE(rows >= 0 && H > 0, "rows must be >= 0 and H > 0");
  REQUIRE(H % 8 == 0 && H <= 16384, "w shape: H must be a multiple of 8, <= 16384");
  if (grouped) REQUIRE(H % 64 == 0, "s shape: grouped scales need H % 64 == 0");
  REQUIRE(h && w && q && s, "h, w, q and s must be non-null");
  REQUIRE(aligned16(h) && aligned16(y), "h and y must be 16-byte aligned");
  if (rows == 0) return LFM2Q_OK;
  if (int e = device_gate()) return e;
  return launched(launch_add_rmsnorm_q(h, y, w, q, s, rows, H, eps, grouped != 0, (cudaStream_t)stream),
                  "add_rmsnorm_q");
}

int lfm2q_silu_mul_q(const uint16_t *g, int8_t *q, float *s, int rows, int I, int grouped, void *stream) {
  REQUIRE(rows >= 0 && I > 0, "rows must be >= 0 and I > 0");
  REQUIRE(I % 8 == 0 && I <= 16384, "I shape: I must be a multiple of 8, <= 16384");
  if (grouped) REQUIRE(I % 64 == 0, "s shape: grouped scales need I % 64 == 0");
  REQUIRE(g && q && s, "g, q and s must be non-null");
  REQUIRE(aligned16(g), "g must be 16-byte aligned");
  if (rows == 0) return LFM2Q_OK;
  if (int e = device_gate()) return e;
  return launched(launch_silu_mul_q(g, q, s, rows, I, grouped != 0, (cudaStream_t)stream), "silu_mul_q");
}

// ------------------------------------------------------------------ GEMV
int lfm2q_gemv(const void *W, int w_is_int8, const float *scale, const uint16_t *x, uint16_t *y, int N, int K,
               int rows, int B, void *stream) {
  REQUIRE(N > 0 && K > 0 && B >= 1, "x [B, K], y [B, N]: need N > 0, K > 0, B >= 1");
  REQUIRE(K % (w_is_int8 ? 512 : 256) == 0, "K must be a multiple of 256 (bf16) / 512 (int8)");
  REQUIRE(W && x && y, "W, x and y must be non-null");
  REQUIRE(!w_is_int8 || scale, "int8 W needs fp32 scale");
  REQUIRE(aligned16(W) && aligned16(x), "W and x must be 16-byte aligned");
  if (int e = device_gate()) return e;
  return launched(launch_gemv(W, w_is_int8 != 0, scale, x, y, N, K, rows, B, g_pdl.load(), (cudaStream_t)stream),
                  "gemv");
}

int lfm2q_gemv_a8(const int8_t *W, const float *sw, const int8_t *xq, const float *sx, const uint16_t *bias,
                  uint16_t *y, int N, int K, int B, int gelu, void *stream) {
  REQUIRE(N > 0 && K > 0 && B >= 1, "xq [B, K], y [B, N]: need N > 0, K > 0, B >= 1");
  REQUIRE(K % 64 == 0, "K must be a multiple of 64");
  REQUIRE(W && sw && xq && sx && y, "W, sw, xq, sx and y must be non-null");
  REQUIRE(aligned16(W) && aligned16(xq) && aligned16(y) && aligned16(bias), "W, xq, bias and y must be 16-byte aligned");
  if (int e = device_gate()) return e;
  return launched(launch_gemv_a8(W, sw, xq, sx, bias, y, N, K, B, gelu != 0, g_pdl.load(), (cudaStream_t)stream),
                  "gemv_a8");
}

int lfm2q_linear_a8(const uint16_t *x, const int8_t *W, const float *sw, const uint16_t *bias, uint16_t *y, int N,
                    int K, int B, int gelu, void *stream) {
  REQUIRE(N > 0 && K > 0 && B >= 1, "x [B, K], y [B, N]: need N > 0, K > 0, B >= 1");
  REQUIRE(K % 64 == 0 && K <= 16384, "K must be a multiple of 64, <= 16384");
  REQUIRE(W && sw && x && y, "W, sw, x and y must be non-null");
  REQUIRE(aligned16(W) && aligned16(x) && aligned16(y) && aligned16(bias), "W, x, bias and y must be 16-byte aligned");
  if (int e = device_gate()) return e;
  return launched(launch_linear_a8(x, W, sw, bias, y, N, K, B, gelu != 0, g_pdl.load(), (cudaStream_t)stream),
                  "linear_a8");
}

int lfm2q_gemv_chain(const lfm2q_gemv_layer *layers, int n_layers, int B, void *stream) {
  REQUIRE(n_layers >= 1 && n_layers <= LFM2Q_CHAIN_MAX_LAYERS, "n_layers must be in [1, 96]");
  REQUIRE(B >= 1 && B <= LFM2Q_CHAIN_MAX_TOKENS, "x [B, K]: the chained GEMV takes 1 <= B <= 4 tokens");
  REQUIRE(layers != nullptr, "layers must be non-null");
  std::vector<ChainLayer> L((size_t)n_layers);
  for (int l = 0; l < n_layers; ++l) {
    const lfm2q_gemv_layer &g = layers[l];
    const std::string at = "layer " + std::to_string(l) + ": ";
    REQUIRE(g.W && g.scale && g.x && g.y, at + "W, scale, x and y must be non-null");
    REQUIRE(aligned16(g.W) && aligned16(g.x), at + "W and x must be 16-byte aligned");
    REQUIRE(g.N > 0 && g.K >= 512 && g.K % 512 == 0, at + "need N > 0 and K a positive multiple of 512");
    const uintptr_t x0 = reinterpret_cast<uintptr_t>(g.x), x1 = x0 + (size_t)B * g.K * 2;
    const uintptr_t y0 = reinterpret_cast<uintptr_t>(g.y), y1 = y0 + (size_t)B * g.N * 2;
    REQUIRE(x1 <= y0 || y1 <= x0, at + "y must not overlap x");
    L[(size_t)l] = ChainLayer{g.W, g.scale, g.x, g.y, g.N, g.K};
  }
  if (int e = device_gate()) return e;
  return launched(launch_gemv_chain(L.data(), n_layers, B, g_pdl.load(), (cudaStream_t)stream), "gemv_chain");
}

int lfm2q_gemv_w4(const uint8_t *Wp, const float *S, const uint16_t *x, uint16_t *y, int N, int K, int group, int B,
                  void *stream) {
  REQUIRE(N > 0 && K > 0 && B >= 1 && B <= 4, "Wp [N, K/2], x [B, K]: need N > 0, K > 0, 1 <= B <= 4");
  REQUIRE(group > 0 && group % 128 == 0 && K % group == 0, "group size must be a multiple of 128 dividing K");
  REQUIRE(Wp && S && x && y, "Wp, S, x and y must be non-null");
  REQUIRE(aligned16(Wp) && aligned16(x), "Wp and x must be 16-byte aligned");
  REQUIRE(gemv_w4_slices(K, B) != 0, "K too large for this batch (B * K <= 16384 and the token slices in 160 KB)");
  if (int e = device_gate()) return e;
  return launched(launch_gemv_w4(Wp, S, x, y, N, K, group, B, g_pdl.load(), gemv_trigger_mode(), (cudaStream_t)stream),
                  "gemv_w4");
}

int lfm2q_gemv_epi(int epi, const void *W, int w_is_int8, const float *scale, const uint16_t *x, uint16_t *y, int S,
                   int K, uint16_t *state, const uint16_t *cw, const uint16_t *cbias, void *stream) {
  REQUIRE(epi == 0 || epi == 1, "epi 0 (swiglu) or 1 (shortconv)");
  REQUIRE(S > 0 && K > 0, "batch 1: x [1, K], y [1, S]");
  REQUIRE(K % (w_is_int8 ? 512 : 256) == 0, "K must be a multiple of 256 (bf16) / 512 (int8)");
  REQUIRE(W && x && y, "W, x and y must be non-null");
  REQUIRE(!w_is_int8 || scale, "int8 W needs fp32 scale");
  REQUIRE(epi == 0 || (state && cw), "shortconv epilogue needs state and conv weight");
  REQUIRE(aligned16(W) && aligned16(x), "W and x must be 16-byte aligned");
  if (int e = device_gate()) return e;
  return launched(launch_gemv_epi(epi, W, w_is_int8 != 0, scale, x, y, S, K, state, cw, cbias, g_pdl.load(),
                                  (cudaStream_t)stream),
                  "gemv_epi");
}

// ------------------------------------------------------------------ decode step kernels
int lfm2q_add_rmsnorm(uint16_t *h, const uint16_t *y, const uint16_t *w, uint16_t *x, int rows, int H, float eps,
                      void *stream) {
  REQUIRE(rows >= 0 && H > 0 && H <= 8192, "h [rows, H]: need rows >= 0 and 0 < H <= 8192");
  if (rows == 0) return LFM2Q_OK;
  REQUIRE(h && w && x, "h, w and x must be non-null");
  if (int e = device_gate()) return e;
  return launched(launch_add_rmsnorm(h, y, w, x, rows, H, eps, g_pdl.load(), (cudaStream_t)stream), "add_rmsnorm");
}

int lfm2q_embed_rmsnorm(const int64_t *tok, const uint16_t *embed, const uint16_t *w, uint16_t *h, uint16_t *x,
                        int rows, int H, float eps, void *stream) {
  REQUIRE(rows >= 0 && H > 0 && H <= 8192, "embed [V, H], h / x [rows, H]: need rows >= 0 and 0 < H <= 8192");
  if (rows == 0) return LFM2Q_OK;
  REQUIRE(tok && embed && w && h && x, "tok, embed, w, h and x must be non-null");
  if (int e = device_gate()) return e;
  return launched(launch_embed_rmsnorm(tok, embed, w, h, x, rows, H, eps, g_pdl.load(), (cudaStream_t)stream),
                  "embed_rmsnorm");
}

int lfm2q_argmax_next(const uint16_t *logits, int64_t *tok, int64_t *pos, int B, int V, void *stream) {
  REQUIRE(B >= 0 && B <= 65535 && V > 0, "logits [B, V]: need 0 <= B <= 65535 and V > 0");
  if (B == 0) return LFM2Q_OK;
  REQUIRE(logits && tok, "logits and tok must be non-null");
  REQUIRE(aligned16(logits) && (V % 8 == 0 || B == 1),
          "logits must be 16-byte aligned, and V a multiple of 8 when B > 1 (every row 16-byte aligned)");
  if (int e = device_gate()) return e;
  return launched(launch_argmax_next(logits, tok, pos, B, V, g_pdl.load(), (cudaStream_t)stream), "argmax_next");
}

int lfm2q_shortconv_step(const uint16_t *bcx, uint16_t *state, const uint16_t *w, const uint16_t *bias, uint16_t *y,
                         int B, int H, void *stream) {
  REQUIRE(B >= 0 && H > 0, "bcx [B, 3H], state [B, H, 3], w [H, 3], y [B, H]: need B >= 0, H > 0");
  REQUIRE(B <= 65535, "B <= 65535");
  if (B == 0) return LFM2Q_OK;
  REQUIRE(bcx && state && w && y, "bcx, state, w and y must be non-null");
  if (int e = device_gate()) return e;
  return launched(launch_shortconv_step(bcx, state, w, bias, y, B, H, g_pdl.load(), (cudaStream_t)stream),
                  "shortconv_step");
}

int lfm2q_qk_norm_rope_kv(const uint16_t *qkv, const uint16_t *qw, const uint16_t *kw, const float *inv_freq,
                          float scaling, const int64_t *pos, uint16_t *q_out, uint16_t *kc, uint16_t *vc, int B,
                          int NQ, int NKV, int max_len, float eps, void *stream) {
  REQUIRE(B >= 0 && NQ > 0 && NKV > 0 && max_len > 0, "qkv [B, (NQ + 2 NKV) * 64]: need B >= 0, NQ, NKV, max_len > 0");
  REQUIRE((long long)B * (NQ + 2 * NKV) <= 0x7fffffffLL, "B * (NQ + 2 NKV) too large");
  if (B == 0) return LFM2Q_OK;
  REQUIRE(qkv && qw && kw && inv_freq && pos && q_out && kc && vc, "every pointer must be non-null");
  REQUIRE(aligned16(qkv) && aligned16(vc), "qkv and vc must be 16-byte aligned");
  if (int e = device_gate()) return e;
  return launched(launch_qk_norm_rope_kv(qkv, qw, kw, inv_freq, scaling, pos, q_out, kc, vc, B, NQ, NKV, max_len, eps,
                                         g_pdl.load(), (cudaStream_t)stream),
                  "qk_norm_rope_kv");
}

// ------------------------------------------------------------------ decode attention
int lfm2q_decode_attention_split(const uint16_t *q, const uint16_t *kc, const uint16_t *vc, const int64_t *pos,
                                 uint16_t *out, float *ws, int B, int NQ, int NKV, int max_len, int S, float scale,
                                 void *stream) {
  REQUIRE(B >= 0 && NKV > 0 && max_len > 0, "q [B, NQ, 64], kc / vc [B, NKV, max_len, 64]: need B >= 0, NKV > 0, "
                                            "max_len > 0");
  REQUIRE(NQ == 4 * NKV, "head_dim 64 and 4 query heads per KV head only");
  REQUIRE(S >= 1 && S <= 65535, "ws [B, NQ, S, 66]: need 1 <= S <= 65535");
  REQUIRE((long long)B * NKV <= 0x7fffffffLL, "B * NKV too large");
  if (B == 0) return LFM2Q_OK;
  REQUIRE(q && kc && vc && pos && out && ws, "q, kc, vc, pos, out and ws must be non-null");
  REQUIRE(aligned16(q) && aligned16(kc) && aligned16(vc), "q, kc and vc must be 16-byte aligned");
  if (int e = device_gate()) return e;
  return launched(launch_decode_attention_split(q, kc, vc, pos, out, ws, B, NQ, NKV, max_len, S, scale, g_pdl.load(),
                                                (cudaStream_t)stream),
                  "decode_attention_split");
}

// Allocation-free variant: the partials live in the library's static device workspace (ATTN_STATIC_WS_FLOATS).
int lfm2q_decode_attention_split_noalloc(const uint16_t *q, const uint16_t *kc, const uint16_t *vc,
                                         const int64_t *pos, uint16_t *out, int B, int NQ, int NKV, int max_len, int S,
                                         float scale, void *stream) {
  static_assert(ATTN_STATIC_WS_FLOATS == LFM2Q_ATTN_NOALLOC_MAX_WS_FLOATS, "header and library disagree");
  REQUIRE(B >= 0 && NKV > 0 && max_len > 0, "q [B, NQ, 64], kc / vc [B, NKV, max_len, 64]: need B >= 0, NKV > 0, "
                                            "max_len > 0");
  REQUIRE(NQ == 4 * NKV, "head_dim 64 and 4 query heads per KV head only");
  REQUIRE(S >= 1 && S <= 65535, "need 1 <= S <= 65535");
  REQUIRE((long long)B * NQ * S * 66 <= ATTN_STATIC_WS_FLOATS,
          "B * NQ * S * 66 exceeds the static workspace of decode_attention_split_noalloc (" +
              std::to_string(ATTN_STATIC_WS_FLOATS) + " floats, 8 MiB): use lfm2q_decode_attention_split with a "
              "caller-allocated ws, or fewer splits");
  if (B == 0) return LFM2Q_OK;
  REQUIRE(q && kc && vc && pos && out, "q, kc, vc, pos and out must be non-null");
  REQUIRE(aligned16(q) && aligned16(kc) && aligned16(vc), "q, kc and vc must be 16-byte aligned");
  if (int e = device_gate()) return e;
  return launched(launch_decode_attention_split_static(q, kc, vc, pos, out, B, NQ, NKV, max_len, S, scale,
                                                       g_pdl.load(), (cudaStream_t)stream),
                  "decode_attention_split_noalloc");
}

// ------------------------------------------------------------------ batches of requests over a paged cache
int lfm2q_kv_slots(const int32_t *lens, const int32_t *new_lens, int32_t *table, int32_t *free_pages, int32_t *n_free,
                   int32_t *got, int32_t *cu, int64_t *positions, int64_t *slots, int B, int max_pages, int num_pages,
                   int page, int64_t capacity, void *stream) {
  REQUIRE(B >= 0 && max_pages > 0 && num_pages > 0 && page > 0,
          "table [B, max_pages], free_pages [num_pages]: need B >= 0, max_pages, num_pages, page > 0");
  REQUIRE((long long)max_pages * page <= (1ll << 30) && (long long)num_pages <= (1ll << 30),
          "max_pages * page and num_pages must be <= 2^30");
  REQUIRE(B <= (1 << 24), "B must be <= 2^24");
  REQUIRE(capacity >= 0 && capacity <= (1ll << 30), "positions / slots [capacity]: need 0 <= capacity <= 2^30");
  REQUIRE(free_pages && n_free && cu && (B == 0 || (lens && new_lens && table && got)) &&
              (capacity == 0 || (positions && slots)),
          "every pointer must be non-null");
  REQUIRE(B == 0 || (got != new_lens && got != lens), "got must be neither lens nor new_lens");
  if (int e = device_gate()) return e;
  return launched(launch_kv_slots(lens, new_lens, table, free_pages, n_free, got, cu, positions, slots, B, max_pages,
                                  num_pages, page, capacity, g_pdl.load(), (cudaStream_t)stream),
                  "kv_slots");
}

static int check_half(int dtype, int D) {
  REQUIRE(dtype == LFM2Q_BF16 || dtype == LFM2Q_FP16, "dtype must be LFM2Q_BF16 or LFM2Q_FP16");
  REQUIRE(D == 64 || D == 128, "head_dim 64 or 128 only");
  return LFM2Q_OK;
}

int lfm2q_qk_norm_rope_kv_paged(const uint16_t *qkv, int64_t row_stride, const uint16_t *qw, const uint16_t *kw,
                                const float *inv_freq, int rot_dim, float scaling, const int64_t *positions,
                                const int64_t *slots, uint16_t *q_out, uint16_t *kc, uint16_t *vc, int dtype, int N,
                                int NQ, int NKV, int D, int num_pages, int page, float eps, int interleaved,
                                void *stream) {
  if (int e = check_half(dtype, D)) return e;
  REQUIRE(N >= 0 && NQ > 0 && NKV > 0 && num_pages > 0 && page > 0,
          "qkv [N, (NQ + 2 NKV) * D], kc / vc [num_pages, NKV, page, D]: need N >= 0 and the others > 0");
  REQUIRE((long long)NQ + 2ll * NKV <= 65536, "NQ + 2 NKV must be <= 65536");
  REQUIRE((long long)num_pages * page <= 0xffffffffll, "num_pages * page must be < 2^32");
  REQUIRE(rot_dim > 0 && rot_dim <= D && rot_dim % 16 == 0, "rot_dim must be a multiple of 16 in [16, D]");
  REQUIRE(row_stride >= ((long long)NQ + 2ll * NKV) * D && row_stride % 8 == 0,
          "qkv rows: the stride must be a multiple of 8 and hold (NQ + 2 NKV) * D");
  if (N == 0) return LFM2Q_OK;
  REQUIRE(qkv && inv_freq && positions && slots && q_out && kc && vc, "every pointer but qw and kw must be non-null");
  REQUIRE((qw == nullptr) == (kw == nullptr), "qw and kw: both or neither");
  REQUIRE(aligned16(qkv) && aligned16(qw) && aligned16(kw) && aligned16(q_out) && aligned16(kc) && aligned16(vc),
          "qkv, qw, kw, q_out, kc and vc must be 16-byte aligned");
  if (int e = device_gate()) return e;
  return launched(launch_qk_norm_rope_kv_paged(qkv, row_stride, qw, kw, inv_freq, rot_dim, scaling, positions, slots,
                                               q_out, kc, vc, N, NQ, NKV, D, num_pages, page, eps, interleaved != 0,
                                               dtype == LFM2Q_FP16, g_pdl.load(), (cudaStream_t)stream),
                  "qk_norm_rope_kv_paged");
}

int lfm2q_tree_attention_splits(int B, int NQ, int NKV, int D, int max_q, int max_len) {
  if (B <= 0 || NKV <= 0 || NQ < NKV || max_q <= 0 || max_len <= 0) return 1;
  return tree_attention_splits(B, NQ, NKV, D, max_q, max_len);
}

int lfm2q_tree_attention(const uint16_t *q, const uint16_t *kc, const uint16_t *vc, const int32_t *table,
                         const int32_t *ctx, const int32_t *cu, const int64_t *mask, uint16_t *out, float *ws,
                         int dtype, int N, int B, int NQ, int NKV, int D, int num_pages, int page, int max_pages, int S,
                         int max_q, float scale, void *stream) {
  if (int e = check_half(dtype, D)) return e;
  REQUIRE(N >= 0 && B >= 0 && NKV > 0 && num_pages > 0 && page > 0 && max_pages > 0,
          "q [N, NQ, D], kc / vc [num_pages, NKV, page, D], table [B, max_pages]: need N, B >= 0 and the others > 0");
  REQUIRE(NQ > 0 && NQ % NKV == 0 && NQ / NKV <= 64, "NQ must be a multiple of NKV, at most 64 times it");
  REQUIRE(max_q >= 1 && max_q <= 64, "max_q (drafted tokens of a request) must be in [1, 64]");
  REQUIRE((long long)max_pages * page <= (1ll << 30), "max_pages * page must be <= 2^30");
  REQUIRE(B <= 65535 && (long long)B * NKV * max_q <= 0x7fffffffLL, "B must be <= 65535 and B * NKV * max_q < 2^31");
  REQUIRE((long long)num_pages * NKV <= 0x7fffffffLL, "num_pages * NKV must be < 2^31");
  // (a request's rows in tiles of 128, its positions in tiles of 64 and 8 for a beginning and an end)
  const long long row_tiles = (max_q * (NQ / NKV) + 127) / (128 / (NQ / NKV) * (NQ / NKV));
  REQUIRE((double)B * NKV * row_tiles * ((double)max_pages * page / 64 + 8) < 2147483648.0 - 65536,
          "B * NKV * (tiles of 128 rows a request) * (max_pages * page / 64) must be < 2^31");
  REQUIRE(S >= 1 && S <= 65535, "ws [N, NQ, S, D + 2]: need 1 <= S <= 65535");
  REQUIRE(scale > 0.f && scale < 1e30f, "scale must be positive and finite");
  if (N == 0 || B == 0) return LFM2Q_OK;
  REQUIRE(q && kc && vc && table && ctx && cu && out, "q, kc, vc, table, ctx, cu and out must be non-null");
  REQUIRE(S == 1 || ws, "ws must be non-null when S > 1");
  REQUIRE(aligned16(q) && aligned16(kc) && aligned16(vc) && aligned16(out) && aligned16(ws),
          "q, kc, vc, out and ws must be 16-byte aligned");
  if (int e = device_gate()) return e;
  return launched(launch_tree_attention(q, kc, vc, table, ctx, cu, mask, out, ws, N, B, NQ, NKV, D, num_pages, page,
                                        max_pages, S, max_q, scale, dtype == LFM2Q_FP16, g_pdl.load(),
                                        (cudaStream_t)stream),
                  "tree_attention");
}

int lfm2q_sample_next(const void *logits, int dtype, int64_t row_stride, const float *temperature, const int32_t *top_k,
                      const float *top_p, const float *min_p, const float *u, int64_t *tok, int64_t *pos, int B, int V,
                      void *stream) {
  REQUIRE(dtype == LFM2Q_BF16 || dtype == LFM2Q_FP16 || dtype == LFM2Q_FP32,
          "dtype must be LFM2Q_BF16, LFM2Q_FP16 or LFM2Q_FP32");
  REQUIRE(B >= 0 && B <= 65535 && V > 0 && V <= (1 << 18), "logits [B, V]: need 0 <= B <= 65535 and 0 < V <= 262144");
  REQUIRE(row_stride >= V, "logits rows: the stride must be >= V");
  if (B == 0) return LFM2Q_OK;
  REQUIRE(logits && u && tok, "logits, u and tok must be non-null");
  REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == LFM2Q_FP32 ? 4 : 2) == 0,
          "logits must be aligned to their elements");
  if (int e = device_gate()) return e;
  return launched(launch_sample_next(logits, dtype, row_stride, temperature, top_k, top_p, min_p, u, tok, pos, B, V,
                                     g_pdl.load(), (cudaStream_t)stream),
                  "sample_next");
}

int lfm2q_call_words(int op, const void *words, int count) {
  // arguments of each entry point, and which of them are int (a bit each)
  static const struct {
    int count;
    uint32_t ints;
  } ops[] = {{15, 0xfu << 9}, {22, 1u << 5 | 0x7fu << 12 | 1u << 20}, {22, 0x7ffu << 9}, {13, 1u << 1 | 3u << 10}};
  REQUIRE(op >= 0 && op < (int)(sizeof(ops) / sizeof(ops[0])), "call_words: no such operator");
  REQUIRE(words && count == ops[op].count, "call_words: the operator has another number of arguments");
  int64_t w[24];
  std::memcpy(w, words, (size_t)count * 8);
  for (int k = 0; k < count; ++k)
    REQUIRE(!(ops[op].ints >> k & 1) || w[k] == (int32_t)w[k], "call_words: an argument does not fit its 32 bits");
  const auto p = [&](int k) { return reinterpret_cast<void *>(w[k]); };
  const auto i = [&](int k) { return (int)w[k]; };
  const auto f = [&](int k) {
    double d;
    std::memcpy(&d, &w[k], 8);
    return (float)d;
  };
  typedef uint16_t u16;
  typedef int32_t i32;
  switch (op) {
    case LFM2Q_KV_SLOTS:
      return lfm2q_kv_slots((i32 *)p(0), (i32 *)p(1), (i32 *)p(2), (i32 *)p(3), (i32 *)p(4), (i32 *)p(5), (i32 *)p(6),
                            (int64_t *)p(7), (int64_t *)p(8), i(9), i(10), i(11), i(12), w[13], p(14));
    case LFM2Q_QK_NORM_ROPE_KV_PAGED:
      return lfm2q_qk_norm_rope_kv_paged((u16 *)p(0), w[1], (u16 *)p(2), (u16 *)p(3), (float *)p(4), i(5), f(6),
                                         (int64_t *)p(7), (int64_t *)p(8), (u16 *)p(9), (u16 *)p(10), (u16 *)p(11),
                                         i(12), i(13), i(14), i(15), i(16), i(17), i(18), f(19), i(20), p(21));
    case LFM2Q_TREE_ATTENTION:
      return lfm2q_tree_attention((u16 *)p(0), (u16 *)p(1), (u16 *)p(2), (i32 *)p(3), (i32 *)p(4), (i32 *)p(5),
                                  (int64_t *)p(6), (u16 *)p(7), (float *)p(8), i(9), i(10), i(11), i(12), i(13), i(14),
                                  i(15), i(16), i(17), i(18), i(19), f(20), p(21));
    default:
      return lfm2q_sample_next(p(0), i(1), w[2], (float *)p(3), (i32 *)p(4), (float *)p(5), (float *)p(6),
                               (float *)p(7), (int64_t *)p(8), (int64_t *)p(9), i(10), i(11), p(12));
  }
}

}  // extern "C"
