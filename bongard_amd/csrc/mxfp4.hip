// MXFP4 for gfx950: the quantizer of bf16 tensors into blocks of 32 e2m1 codes under one power of
// two (OCP Microscaling Formats v1.0, section 5), their exact read-back, and the product of two
// such operands on the block-scaled FP4 MFMA.
//
// The scale of a block is the smallest power of two 2^k with max |x| <= 6 * 2^k (e = k + 127), so no
// value is clipped: the specification's own floor(log2(max)) - 2 would clip the magnitudes between
// 6 and 8 steps of the grid, a bias that the gradients of a training step carry on. It is the rule of the MXFP8 quantizer (mx.hip) for a
// largest value of 6. Codes round to nearest, ties to the even code; x ~ e2m1(q) * 2^(e - 127), which
// bf16 holds exactly (but for what overflows in a block that holds inf: bf16 rounds it to inf).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "mxfp4.hpp"

namespace bf8 {
namespace {

constexpr int64_t kMaxMx4Blocks = 1 << 20;

template <int LPR, int W>
__global__ __launch_bounds__(64 * W) void mx4_tile_kernel(const uint16_t* __restrict__ x,
                                                          Mx4Out p) {
  using T = Mx4Tile<LPR, W>;
  __shared__ typename T::Shared sh;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int64_t tiles_c = (p.cols + T::kCols - 1) / T::kCols;
  const int64_t tiles_r = (p.rows + T::kRows - 1) / T::kRows;
  for (int64_t t = blockIdx.x; t < tiles_c * tiles_r; t += gridDim.x) {
    const int64_t r0 = (t / tiles_c) * T::kRows, c0 = (t % tiles_c) * T::kCols;
    const int64_t c = c0 + 8 * (lane % LPR), r = r0 + 32 * wid + T::RL * (lane / LPR);
    uint4 v[T::RL];
#pragma unroll
    for (int k = 0; k < T::RL; ++k) {
      v[k] = make_uint4(0u, 0u, 0u, 0u);
      if (r + k < p.rows && c < p.cols)
        v[k] = *reinterpret_cast<const uint4*>(x + (r + k) * p.cols + c);
    }
    mx4_tile_finish<LPR, W>(p, r0, c0, v, sh, wid, lane);
  }
}

// bf16 [rows, cols] of codes and planes: a thread reads 4 code bytes and writes 8 values.
__global__ __launch_bounds__(256) void mx4_dequant_kernel(const uint8_t* __restrict__ q,
                                                          const uint32_t* __restrict__ planes,
                                                          int64_t rows, int64_t cols,
                                                          uint16_t* __restrict__ out) {
  const int64_t per_row = cols >> 3, n = rows * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / per_row, c = (i % per_row) * 8;
    const uint32_t code = *reinterpret_cast<const uint32_t*>(q + ((row * cols + c) >> 1));
    const uint32_t e = (planes[(c >> 7) * rows + row] >> (8 * ((c >> 5) & 3))) & 0xFFu;
    const float s = e == 0xFFu ? __uint_as_float(0x7FC00000u)
                               : e == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(e << 23);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t b = (code >> (8 * j)) & 0xFFu;
      const auto v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(b, 1.0f, 0);
      w[j] = pack_bf16x2(v[0] * s, v[1] * s);
    }
    *reinterpret_cast<uint4*>(out + row * cols + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));

// C [M, N] = A . B^T of MXFP4 operands, one 32 x 32 tile a wave straight from memory: lane l of the
// FP4 MFMA supplies the 32 K-values (16 bytes) of row l & 31, block l >> 5 of the step of 64, with
// that block's scale.
template <int OUT>
__global__ __launch_bounds__(64) void mx4_gemm_kernel(
    const uint8_t* __restrict__ A, int64_t lda, const uint32_t* __restrict__ pa,
    const uint8_t* __restrict__ B, int64_t ldb, const uint32_t* __restrict__ pb, int64_t M,
    int64_t N, int64_t K, const uint16_t* __restrict__ bias, void* __restrict__ C, int64_t ldc) {
  const int lane = threadIdx.x, half = lane >> 5;
  const int64_t tiles_n = (N + 31) / 32;
  const int64_t m = blockIdx.x / tiles_n * 32 + (lane & 31), n = blockIdx.x % tiles_n * 32 + (lane & 31);
  v16f acc;
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
  auto load = [&](const uint8_t* q, int64_t ld, const uint32_t* p, int64_t rows, int64_t row,
                  int64_t blk, v8i& f, int& s) {
    const bool in = row < rows && 32 * blk < K;
    const uint4 d = in ? *reinterpret_cast<const uint4*>(q + row * ld + 16 * blk)
                       : make_uint4(0u, 0u, 0u, 0u);
    s = in ? (int)((p[(blk >> 2) * rows + row] >> (8 * (blk & 3))) & 0xFFu) : (int)kMxPadScale;
    f[0] = (int)d.x; f[1] = (int)d.y; f[2] = (int)d.z; f[3] = (int)d.w;
    f[4] = f[5] = f[6] = f[7] = 0;
  };
  for (int64_t k = 0; k < K; k += 64) {
    v8i a, b;
    int sa, sb;
    load(A, lda, pa, M, m, (k >> 5) + half, a, sa);
    load(B, ldb, pb, N, n, (k >> 5) + half, b, sb);
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b, a, acc, 4, 4, 0, sb, 0, sa);
  }
  if (m >= M) return;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int64_t col = n - (lane & 31) + 8 * (i >> 2) + 4 * half + (i & 3);
    if (col >= N) continue;
    const float v = acc[i] + (bias ? bf16_lo(bias[col]) : 0.0f);
    if (OUT == BF8_OUT_BF16)
      reinterpret_cast<uint16_t*>(C)[m * ldc + col] = (uint16_t)f32_to_bf16_bits(v);
    else
      reinterpret_cast<float*>(C)[m * ldc + col] = v;
  }
}

template <int LPR, int W>
int mx4_launch(const uint16_t* x, const Mx4Out& p, hipStream_t s) {
  using T = Mx4Tile<LPR, W>;
  const int64_t tiles =
      (p.rows + T::kRows - 1) / T::kRows * ((p.cols + T::kCols - 1) / T::kCols);
  hipLaunchKernelGGL((mx4_tile_kernel<LPR, W>), dim3((unsigned)std::min(tiles, kMaxMx4Blocks)),
                     dim3(64 * W), 0, s, x, p);
  return launch_status("mx4_tile_kernel");
}

}  // namespace
}  // namespace bf8

using namespace bf8;

extern "C" {

// The outputs of a quantizer of [rows, cols].
static int check_mx4_out(const char* who, const Mx4Out& p) {
  BF8_CHECK(p.rows >= 0 && p.cols >= 0, "%s: negative shape", who);
  BF8_CHECK((p.out == nullptr) == (p.planes == nullptr) &&
                (p.out_t == nullptr) == (p.planes_t == nullptr) && (p.out || p.out_t),
            "%s: give out and / or out_t, each with its scale planes", who);
  BF8_CHECK(!p.out || p.cols % 32 == 0, "%s: blocks along rows need cols %% 32 == 0 (got %lld)",
            who, (long long)p.cols);
  BF8_CHECK(p.cols % 8 == 0, "%s: need cols %% 8 == 0 (got %lld)", who, (long long)p.cols);
  BF8_CHECK(((uintptr_t)p.out & 3) == 0 && ((uintptr_t)p.out_t & 15) == 0 &&
                (((uintptr_t)p.planes | (uintptr_t)p.planes_t) & 3) == 0,
            "%s: out_t 16-byte, out and scale planes 4-byte aligned", who);
  return BF8_OK;
}

int bf8_quantize_mxfp4_bf16(const void* x, int64_t rows, int64_t cols, uint8_t* out,
                            uint32_t* out_planes, uint8_t* out_t, uint32_t* out_t_planes,
                            void* stream) {
  const char* who = "bf8_quantize_mxfp4_bf16";
  const Mx4Out p{rows, cols, out, out_planes, out_t, out_t_planes};
  if (const int rc = check_mx4_out(who, p)) return rc;
  if (rows == 0 || cols == 0) return BF8_OK;
  BF8_CHECK(x && ((uintptr_t)x & 15) == 0, "%s: x must be given, 16-byte aligned", who);
  return mx4_launch<8, 1>((const uint16_t*)x, p, as_stream(stream));
}

int bf8_dequant_mxfp4(const uint8_t* codes, const uint32_t* planes, int64_t rows, int64_t cols,
                      void* out, void* stream) {
  const char* who = "bf8_dequant_mxfp4";
  BF8_CHECK(rows >= 0 && cols >= 0 && cols % 32 == 0,
            "%s: need cols %% 32 == 0 (rows %lld, cols %lld)", who, (long long)rows, (long long)cols);
  if (rows == 0 || cols == 0) return BF8_OK;
  BF8_CHECK(codes && planes && out, "%s: NULL pointer", who);
  BF8_CHECK((((uintptr_t)codes | (uintptr_t)planes) & 3) == 0 && ((uintptr_t)out & 15) == 0,
            "%s: out 16-byte, codes and planes 4-byte aligned", who);
  const int64_t n = rows * (cols / 8);
  hipLaunchKernelGGL(mx4_dequant_kernel, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 1 << 20)),
                     dim3(256), 0, as_stream(stream), codes, planes, rows, cols, (uint16_t*)out);
  return launch_status("mx4_dequant_kernel");
}

size_t bf8_gemm_mxfp4_workspace(int64_t M, int64_t N, int64_t K) { return 0; }

int bf8_gemm_mxfp4(const uint8_t* A, int64_t lda, const uint32_t* A_planes, const uint8_t* B,
                   int64_t ldb, const uint32_t* B_planes, int64_t M, int64_t N, int64_t K,
                   const void* bias, void* C, int out_dtype, int64_t ldc, void* ws,
                   size_t ws_bytes, void* stream) {
  const char* who = "bf8_gemm_mxfp4";
  BF8_CHECK(out_dtype == BF8_OUT_BF16 || out_dtype == BF8_OUT_F32, "%s: bad out_dtype", who);
  BF8_CHECK(M >= 0 && N >= 0 && K >= 0, "%s: negative shape", who);
  BF8_CHECK(K % 32 == 0, "%s: K must be a multiple of the 32-element block (got %lld)", who,
            (long long)K);
  BF8_CHECK(N % 8 == 0 && ldc >= N && ldc % 4 == 0, "%s: need N %% 8 == 0, ldc >= N, ldc %% 4 == 0",
            who);
  BF8_CHECK(((uintptr_t)C & 15) == 0 && ((uintptr_t)bias & 7) == 0,
            "%s: C must be 16-byte, bias 8-byte aligned", who);
  BF8_CHECK(ws_bytes == 0 || (ws && ((uintptr_t)ws & 255) == 0),
            "%s: workspace must be 256-byte aligned", who);
  if (M == 0 || N == 0) return BF8_OK;
  BF8_CHECK(K > 0, "%s: K == 0 is not supported", who);
  BF8_CHECK(A && A_planes && B && B_planes && C, "%s: NULL pointer", who);
  BF8_CHECK(lda % 16 == 0 && ldb % 16 == 0 && 2 * lda >= K && 2 * ldb >= K &&
                (((uintptr_t)A | (uintptr_t)B) & 15) == 0,
            "%s: A and B need 16-byte aligned bases and row strides >= K / 2 bytes", who);
  BF8_CHECK((((uintptr_t)A_planes | (uintptr_t)B_planes) & 3) == 0,
            "%s: scale planes need 4-byte alignment", who);
  BF8_CHECK(M * lda < (1LL << 31) && N * ldb < (1LL << 31), "%s: operand larger than 2 GiB", who);
  const int64_t tiles = ((M + 31) / 32) * ((N + 31) / 32);
  BF8_CHECK(tiles < (1LL << 31), "%s: output too large", who);
  hipStream_t s = as_stream(stream);
  if (out_dtype == BF8_OUT_BF16)
    hipLaunchKernelGGL(mx4_gemm_kernel<BF8_OUT_BF16>, dim3((unsigned)tiles), dim3(64), 0, s, A, lda,
                       A_planes, B, ldb, B_planes, M, N, K, (const uint16_t*)bias, C, ldc);
  else
    hipLaunchKernelGGL(mx4_gemm_kernel<BF8_OUT_F32>, dim3((unsigned)tiles), dim3(64), 0, s, A, lda,
                       A_planes, B, ldb, B_planes, M, N, K, (const uint16_t*)bias, C, ldc);
  return launch_status("mx4_gemm_kernel");
}

}  // extern "C"
