// MXFP4 for gfx950: the quantizer of bf16 tensors into blocks of 32 e2m1 codes under one power of
// two (OCP Microscaling Formats v1.0, section 5) and their exact read-back. The products are
// gemm.hip's.
//
// The scale of a block is the smallest power of two 2^k with max |x| <= 6 * 2^k (e = k + 127), so no
// value is clipped: the specification's own floor(log2(max)) - 2 would clip the magnitudes between
// 6 and 8 steps of the grid, a bias that the gradients of a training step carry on. It is the rule of the MXFP8 quantizer (mx.hip) for a
// largest value of 6. Codes round to nearest, ties to the even code; x ~ e2m1(q) * 2^(e - 127), which
// bf16 holds exactly (but for what overflows in a block that holds inf: bf16 rounds it to inf).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "gelu.hpp"
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

// d_g (G) or d_u of the lane's RL rows of a tile, four rows' loads at a time.
template <bool G, int RL>
__device__ __forceinline__ void geglu_bwd_rows(const uint16_t* dp, const uint16_t* gp, int64_t I,
                                               int64_t rows_left, const uint16_t* ta,
                                               const uint32_t* tf, uint4 (&v)[RL]) {
#pragma unroll
  for (int q = 0; q < RL / 4; ++q) {
    uint4 d[4], g[4], u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int row = 4 * q + k;
      d[k] = g[k] = u[k] = make_uint4(0u, 0u, 0u, 0u);
      if (row < rows_left) {
        d[k] = *reinterpret_cast<const uint4*>(dp + row * I);
        g[k] = *reinterpret_cast<const uint4*>(gp + row * 2 * I);
        if (G) u[k] = *reinterpret_cast<const uint4*>(gp + row * 2 * I + I);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) v[4 * q + k] = geglu_bwd8_half<G>(d[k], g[k], u[k], ta, tf);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The gated-GELU backward and the quantization of its dGU [M, 2I] (p: rows M, cols 2I) from
// dH [M, I] and GU [M, 2I], I % 128 == 0: dGU goes from registers to its copies. The first half of
// a block's waves take the d_g tile of 32 W x 8 LPR elements of H, the others its d_u tile.
template <int LPR, int W>
__global__ __launch_bounds__(128 * W) void geglu_bwd_mx4_kernel(const uint16_t* __restrict__ dH,
                                                                const uint16_t* __restrict__ GU,
                                                                int64_t I, Mx4Out p) {
  using T = Mx4Tile<LPR, W>;
  __shared__ __attribute__((aligned(16))) uint16_t ta[kGeluABytes / 2];
  __shared__ __attribute__((aligned(16))) uint32_t tf[kGeluFBytes / 4];
  __shared__ typename T::Shared sh[2];
  load_gelu_tables<128 * W>(ta, tf);
  __syncthreads();
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wid = w % W, half = w / W;
  const int64_t tiles_c = I / T::kCols, tiles_r = (p.rows + T::kRows - 1) / T::kRows;
  for (int64_t t = blockIdx.x; t < tiles_c * tiles_r; t += gridDim.x) {
    const int64_t r0 = (t / tiles_c) * T::kRows, c0 = (t % tiles_c) * T::kCols;
    const int64_t r = r0 + 32 * wid + T::RL * (lane / LPR);
    const uint16_t* dp = dH + r * I + c0 + 8 * (lane % LPR);
    const uint16_t* gp = GU + r * 2 * I + c0 + 8 * (lane % LPR);
    uint4 v[T::RL];
    if (half == 0)
      geglu_bwd_rows<true, T::RL>(dp, gp, I, p.rows - r, ta, tf, v);
    else
      geglu_bwd_rows<false, T::RL>(dp, gp, I, p.rows - r, ta, tf, v);
    mx4_tile_finish<LPR, W>(p, r0, half * I + c0, v, sh[half], wid, lane);
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

int bf8_geglu_bwd_mxfp4(const void* dH, const void* GU, int64_t M, int64_t I, uint8_t* out,
                        uint32_t* out_planes, uint8_t* out_t, uint32_t* out_t_planes,
                        void* stream) {
  const char* who = "bf8_geglu_bwd_mxfp4";
  BF8_CHECK(I % 128 == 0, "%s: need I %% 128 == 0 (got %lld)", who, (long long)I);
  const Mx4Out p{M, 2 * I, out, out_planes, out_t, out_t_planes};
  if (const int rc = check_mx4_out(who, p)) return rc;
  if (M == 0 || I == 0) return BF8_OK;
  BF8_CHECK(dH && GU && (((uintptr_t)dH | (uintptr_t)GU) & 15) == 0,
            "%s: dH and GU must be given, 16-byte aligned", who);
  const auto* d = (const uint16_t*)dH;
  const auto* g = (const uint16_t*)GU;
  const int64_t tiles = ((M + 127) / 128) * (I / 128);
  hipLaunchKernelGGL((geglu_bwd_mx4_kernel<16, 4>), dim3((unsigned)std::min<int64_t>(tiles, 512)),
                     dim3(512), 0, as_stream(stream), d, g, I, p);
  return launch_status("geglu_bwd_mx4_kernel");
}

}  // extern "C"
