// A layer's pass in 8-bit integers as one call: the training forward and backward of a linear and of the gated
// MLP, as the quantizer's, the products' and the gated GELU's own entries in turn on one workspace (from
// Python each of those is 10 us of host time, in the autograd engine's thread up to twice that: 500 x 2048 x 2560
// trained 171 us as six calls, 118-129 as two, by machine).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "gemm_kernel.hpp"
#include "int8.hpp"

namespace bf8 {
namespace {

int64_t pad16(int64_t rows) { return (rows + 15) / 16 * 16; }

// Parts of a workspace, 256-byte aligned one after another.
struct Parts {
  size_t at = 0;
  size_t take(size_t bytes) {
    const size_t o = at;
    at += (bytes + 255) / 256 * 256;
    return o;
  }
};

// The row copies of x and W, then what the quantizations or the product need. (least: without the product's, which runs
// a plan that needs less where less is there.)
struct ForwardWs {
  size_t x, x_scale, w, w_scale, rest, least, bytes;
};
ForwardWs forward_ws(int64_t M, int64_t N, int64_t K, bool keep_x, bool keep_w) {
  ForwardWs f{};
  Parts p;
  f.x = p.take((size_t)M * K);
  f.x_scale = p.take((size_t)M * 4);
  f.w = p.take((size_t)N * K);
  f.w_scale = p.take((size_t)N * 4);
  f.rest = p.at;
  size_t rest = 0;
  if (keep_x) rest = std::max(rest, bf8_quantize_int8_workspace(M, K, 1));
  if (keep_w) rest = std::max(rest, bf8_quantize_int8_workspace(N, K, 1));
  f.least = f.rest + rest;
  f.bytes = f.rest + std::max(rest, bf8_gemm_int8_workspace(M, N, K));
  return f;
}

// dy's codes and scales by row and by column, then what the quantization or a product needs.
struct BackwardWs {
  size_t rows, row_scale, cols, col_scale, rest, least, bytes;
};
BackwardWs backward_ws(int64_t M, int64_t N, int64_t K, bool dx, bool dw) {
  const int64_t Mp = pad16(M);
  BackwardWs w{};
  Parts p;
  if (dx) {
    w.rows = p.take((size_t)M * N);
    w.row_scale = p.take((size_t)M * 4);
  }
  if (dw) {
    w.cols = p.take((size_t)N * Mp);
    w.col_scale = p.take((size_t)N * 4);
  }
  w.rest = p.at;
  size_t rest = dw ? bf8_quantize_int8_workspace(M, N, dx) : 0;
  w.least = w.rest + rest;
  if (dx) rest = std::max(rest, bf8_gemm_int8_workspace(M, K, N));
  if (dw) rest = std::max(rest, bf8_gemm_int8_workspace(N, K, Mp));
  w.bytes = w.rest + rest;
  return w;
}

// x's and H's row copies, H (bf16), and what the quantizations or the down product need.
struct MlpForwardWs {
  size_t x, x_scale, h, h8, h_scale, rest, least, bytes;
};
MlpForwardWs mlp_forward_ws(int64_t M, int64_t K, int64_t I, int64_t N, bool keep_x, bool keep_h) {
  MlpForwardWs w{};
  Parts p;
  w.x = p.take((size_t)M * K);
  w.x_scale = p.take((size_t)M * 4);
  w.h = p.take((size_t)M * I * 2);
  w.h8 = p.take((size_t)M * I);
  w.h_scale = p.take((size_t)M * 4);
  w.rest = p.at;
  size_t rest = 0;
  if (keep_x) rest = std::max(rest, bf8_quantize_int8_workspace(M, K, 1));
  if (keep_h) rest = std::max({rest, bf8_quantize_int8_workspace(M, I, 1), int8_tile_maxima_bytes(M, I)});
  w.least = w.rest + rest;
  w.bytes = w.rest + std::max(rest, bf8_gemm_int8_workspace(M, N, I));
  return w;
}

// dH, then either the linear backward's workspace or dGU (bf16), its codes and scales by row and by column and what
// their maxima and the products need.
constexpr int64_t kMaximaRows = 1024;  // (as the gated backward's codes alone: from here on by the maxima it leaves)
struct MlpWs {
  size_t dh, linear, dgu, rows, row_scale, cols, col_scale, rest, least, bytes;
};
MlpWs mlp_ws(int64_t M, int64_t K, int64_t I, int64_t N, bool dx, bool dgu, bool dd) {
  MlpWs w{};
  Parts p;
  const bool dh = dx || dgu;
  if (dh) w.dh = p.take((size_t)M * I * 2);
  w.linear = p.at;
  const BackwardWs linear = backward_ws(M, N, I, dh, dd);
  w.least = w.linear + linear.least;
  w.bytes = w.linear + linear.bytes;
  if (!dh) return w;
  w.dgu = p.take((size_t)M * 2 * I * 2);
  if (dx) {
    w.rows = p.take((size_t)M * 2 * I);
    w.row_scale = p.take((size_t)M * 4);
  }
  if (dgu) {
    w.cols = p.take((size_t)2 * I * pad16(M));
    w.col_scale = p.take((size_t)2 * I * 4);
  }
  w.rest = p.at;
  size_t rest = M >= kMaximaRows ? bf8_geglu_bwd_mxint8_maxima(M, I) : dgu ? bf8_quantize_int8_workspace(M, 2 * I, dx) : 0;
  w.least = std::max(w.least, w.rest + rest);
  if (dx) rest = std::max(rest, bf8_gemm_int8_workspace(M, K, 2 * I));
  if (dgu) rest = std::max(rest, bf8_gemm_int8_workspace(2 * I, K, pad16(M)));
  w.bytes = std::max(w.bytes, w.rest + rest);
  return w;
}

}  // namespace
}  // namespace bf8

using namespace bf8;

extern "C" {

size_t bf8_linear_int8_forward_workspace(int64_t M, int64_t N, int64_t K, int keep_x, int keep_w) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return forward_ws(M, N, K, keep_x != 0, keep_w != 0).bytes;
}

int bf8_linear_int8_forward(const void* x, const void* W, int64_t M, int64_t N, int64_t K, const void* bias,
                            void* C, int8_t* Xt, float* xt_scale, int8_t* Wt, float* wt_scale, void* ws,
                            size_t ws_bytes, void* stream) {
  const char* who = "bf8_linear_int8_forward";
  BF8_CHECK(M > 0 && N > 0 && K > 0, "%s: empty or negative shape", who);
  BF8_CHECK(K % 16 == 0 && K <= 32768 && N % 8 == 0, "%s: need K %% 16 == 0, K <= 32768 and N %% 8 == 0", who);
  BF8_CHECK(x && W && C && (Xt == nullptr) == (xt_scale == nullptr) && (Wt == nullptr) == (wt_scale == nullptr),
            "%s: NULL pointer", who);
  BF8_CHECK((((uintptr_t)x | (uintptr_t)W | (uintptr_t)C | (uintptr_t)Xt | (uintptr_t)xt_scale | (uintptr_t)Wt |
              (uintptr_t)wt_scale) & 15) == 0 && ((uintptr_t)bias & 7) == 0,
            "%s: every tensor must be 16-byte (bias 8-byte) aligned", who);
  BF8_CHECK(M < (1LL << 31) && N < (1LL << 31) && std::max(M, N) * K < (1LL << 31),
            "%s: operands of 2 GiB and more", who);
  const ForwardWs f = forward_ws(M, N, K, Xt, Wt);
  BF8_CHECK(ws && ((uintptr_t)ws & 255) == 0 && ws_bytes >= f.least,
            "%s: workspace needs %zu bytes, 256-byte aligned (got %zu)", who, f.least, ws_bytes);
  int8_t* const base = (int8_t*)ws;
  float *const xs = (float*)(base + f.x_scale), *const wsc = (float*)(base + f.w_scale);
  void* const rest = base + f.rest;
  const size_t rest_bytes = ws_bytes - f.rest;
  if (const int rc = bf8_quantize_int8_bf16(x, M, K, base, xs, Xt, xt_scale, rest, rest_bytes, stream)) return rc;
  if (const int rc = bf8_quantize_int8_bf16(W, N, K, base + f.w, wsc, Wt, wt_scale, rest, rest_bytes, stream)) return rc;
  return bf8_gemm_int8(base, K, xs, base + f.w, K, wsc, M, N, K, bias, C, BF8_OUT_BF16, N, rest, rest_bytes, stream);
}

size_t bf8_linear_int8_backward_workspace(int64_t M, int64_t N, int64_t K, int dx, int dw) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return backward_ws(M, N, K, dx != 0, dw != 0).bytes;
}

int bf8_linear_int8_backward(const void* dy, int64_t M, int64_t N, int64_t K, const int8_t* Wt,
                             const float* wt_scale, const int8_t* Xt, const float* xt_scale, void* dx, void* dw,
                             void* ws, size_t ws_bytes, void* stream) {
  const char* who = "bf8_linear_int8_backward";
  BF8_CHECK(M > 0 && N > 0 && K > 0, "%s: empty or negative shape", who);
  BF8_CHECK(N % 16 == 0 && N <= 32768 && K % 8 == 0 && (!dw || M <= kInt8MaxK),
            "%s: need N %% 16 == 0, N <= 32768, K %% 8 == 0 and for dw M <= %lld", who, (long long)kInt8MaxK);
  BF8_CHECK(dx || dw, "%s: nothing requested", who);
  BF8_CHECK(dy && (!dx || (Wt && wt_scale)) && (!dw || (Xt && xt_scale)), "%s: NULL pointer", who);
  BF8_CHECK((((uintptr_t)dy | (uintptr_t)Wt | (uintptr_t)wt_scale | (uintptr_t)Xt | (uintptr_t)xt_scale |
              (uintptr_t)dx | (uintptr_t)dw) & 15) == 0,
            "%s: every tensor must be 16-byte aligned", who);
  const int64_t most = std::max(dx ? std::max(M, K) * N : 0, dw ? std::max(N, K) * pad16(M) : 0);
  BF8_CHECK(M < (1LL << 31) && K < (1LL << 31) && most < (1LL << 31), "%s: operands of 2 GiB and more", who);
  const BackwardWs w = backward_ws(M, N, K, dx, dw);
  BF8_CHECK(ws && ((uintptr_t)ws & 255) == 0 && ws_bytes >= w.least,
            "%s: workspace needs %zu bytes, 256-byte aligned (got %zu)", who, w.least, ws_bytes);
  int8_t* const base = (int8_t*)ws;
  int8_t *const rows = dx ? base + w.rows : nullptr, *const cols = dw ? base + w.cols : nullptr;
  float* const rs = dx ? (float*)(base + w.row_scale) : nullptr;
  float* const cs = dw ? (float*)(base + w.col_scale) : nullptr;
  void* const rest = base + w.rest;
  const size_t rest_bytes = ws_bytes - w.rest;
  if (const int rc = bf8_quantize_int8_bf16(dy, M, N, rows, rs, cols, cs, rest, rest_bytes, stream)) return rc;
  const int64_t Mp = pad16(M);
  if (dw)
    if (const int rc = bf8_gemm_int8(cols, Mp, cs, Xt, Mp, xt_scale, N, K, Mp, nullptr, dw, BF8_OUT_BF16, K, rest,
                                     rest_bytes, stream))
      return rc;
  // (dx last: what reads it next finds it in the caches)
  return dx ? bf8_gemm_int8(rows, N, rs, Wt, N, wt_scale, M, K, N, nullptr, dx, BF8_OUT_BF16, K, rest, rest_bytes,
                            stream)
            : BF8_OK;
}

size_t bf8_geglu_mlp_int8_forward_workspace(int64_t M, int64_t K, int64_t I, int64_t N, int keep_x, int keep_h) {
  if (M <= 0 || K <= 0 || I <= 0 || N <= 0) return 0;
  return mlp_forward_ws(M, K, I, N, keep_x != 0, keep_h != 0).bytes;
}

int bf8_geglu_mlp_int8_forward(const void* x, int64_t M, int64_t K, int64_t I, int64_t N, const int8_t* W_gu,
                               const float* w_gu_scale, const int8_t* W_down, const float* w_down_scale, void* Y,
                               int8_t* GU8, uint8_t* GU8_exp, int8_t* Xt, float* xt_scale, int8_t* Ht,
                               float* ht_scale, void* ws, size_t ws_bytes, void* stream) {
  const char* who = "bf8_geglu_mlp_int8_forward";
  BF8_CHECK(M > 0 && K > 0 && I > 0 && N > 0, "%s: empty or negative shape", who);
  BF8_CHECK(K % 16 == 0 && K <= 32768 && I % 128 == 0 && I <= 32768 && N % 8 == 0 && M < (1LL << 31),
            "%s: need K %% 16 == 0, I %% 128 == 0, both 32768 at most, and N %% 8 == 0", who);
  BF8_CHECK(x && W_gu && w_gu_scale && W_down && w_down_scale && Y && (GU8 == nullptr) == (GU8_exp == nullptr) &&
                (Xt == nullptr) == (xt_scale == nullptr) && (Ht == nullptr) == (ht_scale == nullptr),
            "%s: NULL pointer", who);
  // (here, and not by what reads them: H's copies are written by one of two quantizations, and most of the work is done
  // before the down product)
  BF8_CHECK((((uintptr_t)x | (uintptr_t)W_gu | (uintptr_t)w_gu_scale | (uintptr_t)W_down | (uintptr_t)w_down_scale |
              (uintptr_t)Y | (uintptr_t)Xt | (uintptr_t)xt_scale | (uintptr_t)Ht | (uintptr_t)ht_scale) & 15) == 0 &&
                ((uintptr_t)GU8 & 7) == 0,
            "%s: every tensor must be 16-byte (GU8 8-byte) aligned", who);
  BF8_CHECK(N < (1LL << 31) && std::max(M, 2 * I) * K < (1LL << 31) && std::max(M, N) * I < (1LL << 31),
            "%s: operands of 2 GiB and more", who);
  const MlpForwardWs w = mlp_forward_ws(M, K, I, N, Xt, Ht);
  BF8_CHECK(ws && ((uintptr_t)ws & 255) == 0 && ws_bytes >= w.least,
            "%s: workspace needs %zu bytes, 256-byte aligned (got %zu)", who, w.least, ws_bytes);
  uint8_t* const base = (uint8_t*)ws;
  int8_t *const x8 = (int8_t*)base + w.x, *const h8 = (int8_t*)base + w.h8;
  float *const xs = (float*)(base + w.x_scale), *const hs = (float*)(base + w.h_scale);
  void *const H = base + w.h, *const rest = base + w.rest;
  const size_t rest_bytes = ws_bytes - w.rest;
  if (const int rc = bf8_quantize_int8_bf16(x, M, K, x8, xs, Xt, xt_scale, rest, rest_bytes, stream)) return rc;
  // both copies of H by the maxima that the product leaves, where it does
  const bool maxima = Ht && geglu_int8_leaves_maxima(M, I, K);
  const Int8Maxima hm = int8_tile_maxima(rest, M, I);
  if (const int rc = gemm_geglu_int8(who, x8, K, xs, W_gu, K, w_gu_scale, M, I, K, H, GU8, GU8_exp,
                                     maxima ? &hm : nullptr, stream))
    return rc;
  if (const int rc = maxima ? int8_codes_of_maxima((const uint16_t*)H, hm, h8, hs, Ht, ht_scale, as_stream(stream))
                            : bf8_quantize_int8_bf16(H, M, I, h8, hs, Ht, ht_scale, rest, rest_bytes, stream))
    return rc;
  return bf8_gemm_int8(h8, I, hs, W_down, I, w_down_scale, M, N, I, nullptr, Y, BF8_OUT_BF16, N, rest, rest_bytes,
                       stream);
}

size_t bf8_geglu_mlp_int8_backward_workspace(int64_t M, int64_t K, int64_t I, int64_t N, int dx, int dgu, int dd) {
  if (M <= 0 || K <= 0 || I <= 0 || N <= 0) return 0;
  return mlp_ws(M, K, I, N, dx != 0, dgu != 0, dd != 0).bytes;
}

int bf8_geglu_mlp_int8_backward(const void* dy, int64_t M, int64_t K, int64_t I, int64_t N, const int8_t* GU8,
                                const uint8_t* GU8_exp, const int8_t* Xt, const float* xt_scale, const int8_t* Ht,
                                const float* ht_scale, const int8_t* Wt_gu, const float* wt_gu_scale,
                                const int8_t* Wt_down, const float* wt_down_scale, void* dx, void* dW_gu,
                                void* dW_down, void* ws, size_t ws_bytes, void* stream) {
  const char* who = "bf8_geglu_mlp_int8_backward";
  BF8_CHECK(M > 0 && K > 0 && I > 0 && N > 0, "%s: empty or negative shape", who);
  BF8_CHECK(I % 32 == 0 && 2 * I <= 32768 && N % 16 == 0 && N <= 32768 && K % 8 == 0 && M < (1LL << 31),
            "%s: need I %% 32 == 0, I <= 16384, N %% 16 == 0, N <= 32768 and K %% 8 == 0", who);
  BF8_CHECK(dx || dW_gu || dW_down, "%s: nothing requested", who);
  const bool dh = dx || dW_gu;
  BF8_CHECK(dy && (!dh || (GU8 && GU8_exp && Wt_down && wt_down_scale)) && (!dx || (Wt_gu && wt_gu_scale)) &&
                (!dW_gu || (Xt && xt_scale)) && (!dW_down || (Ht && ht_scale)),
            "%s: NULL pointer", who);
  BF8_CHECK(!(dW_gu || dW_down) || M <= kInt8MaxK, "%s: for a weight's gradient M is %lld at most", who,
            (long long)kInt8MaxK);
  // (here, and not by the products that read them, before which most of the work is done)
  BF8_CHECK((((uintptr_t)dy | (uintptr_t)Xt | (uintptr_t)xt_scale | (uintptr_t)Ht | (uintptr_t)ht_scale |
              (uintptr_t)Wt_gu | (uintptr_t)wt_gu_scale | (uintptr_t)Wt_down | (uintptr_t)wt_down_scale |
              (uintptr_t)dx | (uintptr_t)dW_gu | (uintptr_t)dW_down) & 15) == 0 && ((uintptr_t)GU8 & 7) == 0,
            "%s: every tensor must be 16-byte (GU8 8-byte) aligned", who);
  const int64_t Mp = pad16(M);
  const int64_t most = std::max({dh ? std::max(M, I) * N : 0, dW_down ? std::max(N, I) * Mp : 0,
                                 dx ? std::max(M, K) * 2 * I : 0, dW_gu ? std::max(2 * I, K) * Mp : 0});
  BF8_CHECK(K < (1LL << 31) && most < (1LL << 31), "%s: operands of 2 GiB and more", who);
  const MlpWs w = mlp_ws(M, K, I, N, dx, dW_gu, dW_down);
  BF8_CHECK(ws && ((uintptr_t)ws & 255) == 0 && ws_bytes >= w.least,
            "%s: workspace needs %zu bytes, 256-byte aligned (got %zu)", who, w.least, ws_bytes);
  uint8_t* const base = (uint8_t*)ws;
  void* const dH = dh ? base + w.dh : nullptr;
  if (const int rc = bf8_linear_int8_backward(dy, M, N, I, Wt_down, wt_down_scale, Ht, ht_scale, dH, dW_down,
                                              base + w.linear, ws_bytes - w.linear, stream))
    return rc;
  if (!dh) return BF8_OK;
  int8_t *const rows = dx ? (int8_t*)base + w.rows : nullptr, *const cols = dW_gu ? (int8_t*)base + w.cols : nullptr;
  float* const rs = dx ? (float*)(base + w.row_scale) : nullptr;
  float* const cs = dW_gu ? (float*)(base + w.col_scale) : nullptr;
  void *const dGU = base + w.dgu, *const rest = base + w.rest;
  const size_t rest_bytes = ws_bytes - w.rest;
  const bool maxima = M >= kMaximaRows;
  if (const int rc = bf8_geglu_bwd_mxint8(dH, GU8, GU8_exp, M, I, dGU, maxima ? rest : nullptr,
                                          maxima ? rest_bytes : 0, stream))
    return rc;
  if (const int rc = maxima ? bf8_quantize_int8_maxima_bf16(dGU, M, 2 * I, 2, rows, rs, cols, cs, rest, rest_bytes,
                                                            stream)
                            : bf8_quantize_int8_bf16(dGU, M, 2 * I, rows, rs, cols, cs, rest, rest_bytes, stream))
    return rc;
  if (dW_gu)
    if (const int rc = bf8_gemm_int8(cols, Mp, cs, Xt, Mp, xt_scale, 2 * I, K, Mp, nullptr, dW_gu, BF8_OUT_BF16, K,
                                     rest, rest_bytes, stream))
      return rc;
  return dx ? bf8_gemm_int8(rows, 2 * I, rs, Wt_gu, 2 * I, wt_gu_scale, M, K, 2 * I, nullptr, dx, BF8_OUT_BF16, K,
                            rest, rest_bytes, stream)
            : BF8_OK;
}

}  // extern "C"
