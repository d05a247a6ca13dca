// MXFP4 for gfx950: the quantizer of bf16 tensors into blocks of 32 e2m1 codes under one power of
// two (OCP Microscaling Formats v1.0, section 5) and their exact read-back. The products are
// gemm.hip's.
//
// The scale of a block is the smallest power of two 2^k with max |x| <= 6 * 2^k (e = k + 127), so
// no value is clipped: the specification's own floor(log2(max)) - 2 would clip the magnitudes
// between 6 and 8 steps of the grid, a bias that the gradients of a training step carry on. It is
// the rule of the MXFP8 quantizer (mx.hip) for a largest value of 6. Codes round to nearest, ties
// to the even code; x ~ e2m1(q) * 2^(e - 127), which bf16 holds exactly (but for what overflows in
// a block that holds inf: bf16 rounds it to inf).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "gelu.hpp"
#include "mxfp4.hpp"

namespace bf8 {
namespace {

// A block of W waves takes W tiles one below the other. Memory-bound: 2 B read, 17 / 32 B written
// an element and copy; one pass for both copies. Inputs rotated past the MALL, W = 1 / 4 / 8, us (a
// copy of as many bytes at the 5.1 TB/s of large ones): along rows [512, 10240] 5.4 / 5.5 / 5.4
// (2.6), [4096, 10240] 24.6 / 24.7 / 24.8 (20.8), [4096, 20480] 45.7 / 46.1 / 47.0 (41.6); both
// copies [500, 2048] 3.8 / 4.2 / 5.2, [2001, 4096] 8.9 / 9.1 / 9.1 (4.9), [4096, 2560] 12.1 / 10.7
// / 11.8 (6.3), [2560, 10240] 23.0 / 21.5 / 22.6 (15.7), [4096, 10240] 35.6 / 31.4 / 30.1 (25.2),
// [20480, 2560] 48.9 / 40.7 / 38.3 (31.5): columnwise codes in pieces of 16 bytes cost the large
// tensors a quarter, waiting for the block's other waves the small ones as much. Loads behind a
// branch each (a wait each) took 24% more at [4096, 2560].
template <int W>
__global__ __launch_bounds__(64 * W) void mx4_kernel(const uint16_t* __restrict__ x, Mx4Out p) {
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t tiles_c = (uint32_t)((p.cols + kMx4Cols - 1) / kMx4Cols);
  const int64_t r0 = ((int64_t)(blockIdx.x / tiles_c) * W + wid) * kMx4Rows;
  const int64_t c0 = (int64_t)(blockIdx.x % tiles_c) * kMx4Cols;
  __shared__ Mx4Stage<W> sh;
  const int64_t c = c0 + 8 * (lane & 15);
  const uint32_t ld = 2 * (uint32_t)p.cols;
  const uint32_t left = (uint32_t)max((int64_t)0, min(p.rows - r0, (int64_t)kMx4Rows));
  const Window w = window(x + r0 * p.cols, left * ld);
  const uint32_t o = c < p.cols ? 8 * (lane >> 4) * ld + 2 * (uint32_t)c : kPastEnd;
  uint4 v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = window_load(w, o + k * ld);
  mx4_wave_tile<W>(p, r0, c0, v, &sh, wid, lane);
}

// geglu_bwd8_half out of line, for rows with a gate outside the gelu tables (0, below 2^-16, 8 and
// above): inlined for eight rows of both halves its rules made a loop of 17,000 instructions, most of
// the time of which went into fetching them.
template <bool G>
__device__ __noinline__ uint4 geglu_bwd8_outside(uint4 dh, uint4 g, uint4 u, const uint16_t* ta,
                                                 const uint32_t* tf) {
  return geglu_bwd8_half<G>(dh, g, u, ta, tf);
}

// The same for gates inside the tables; `outside` is not 0 where one is not. (A NaN keeps what bits
// it has: the quantizer takes every NaN alike.)
template <bool G>
__device__ __forceinline__ uint4 geglu_bwd8_inside(uint4 dh, uint4 g, uint4 u, const uint16_t* ta,
                                                   const uint32_t* tf, uint32_t& outside) {
  const uint32_t dw[4] = {dh.x, dh.y, dh.z, dh.w}, gw[4] = {g.x, g.y, g.z, g.w};
  const uint32_t uw[4] = {u.x, u.y, u.z, u.w};
  uint32_t ix[4], t[8], o[4];
#pragma unroll
  for (int w = 0; w < 4; ++w)
    ix[w] = G ? gelu_factor_index2(gw[w], outside) : gelu_index2(gw[w], outside);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    t[2 * w] = G ? tf[ix[w] & 0xFFFFu] : ta[ix[w] & 0xFFFFu];
    t[2 * w + 1] = G ? tf[ix[w] >> 16] : ta[ix[w] >> 16];
  }
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float d0 = bf16_lo(dw[w]), d1 = bf16_hi(dw[w]);
    if constexpr (G) {
      const uint32_t da = pack_bf16x2(d0 * bf16_lo(uw[w]), d1 * bf16_hi(uw[w]));
      o[w] = pack_bf16x2(bf16_lo(da) * __uint_as_float(t[2 * w]),
                         bf16_hi(da) * __uint_as_float(t[2 * w + 1]));
    } else {
      o[w] = pack_bf16x2(d0 * __uint_as_float(t[2 * w] << 16), d1 * __uint_as_float(t[2 * w + 1] << 16));
    }
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// d_g (G) or d_u of the lane's eight rows of a tile, four rows' loads at a time. wd, wg: windows of dH and GU
// from the tile's first row on, od, og: the lane's offsets in them; ld: bytes of a row of dH.
template <bool G>
__device__ __forceinline__ void geglu_bwd_rows(Window wd, Window wg, uint32_t od, uint32_t og,
                                               uint32_t ld, const uint16_t* ta, const uint32_t* tf,
                                               uint4 (&v)[8]) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    uint4 d[4], g[4], u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t row = 4 * q + k;
      d[k] = window_load(wd, od + row * ld);
      g[k] = window_load(wg, og + 2 * row * ld);
      u[k] = G ? window_load(wg, og + (2 * row + 1) * ld) : make_uint4(0u, 0u, 0u, 0u);
    }
    uint32_t outside[4] = {};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[4 * q + k] = geglu_bwd8_inside<G>(d[k], g[k], u[k], ta, tf, outside[k]);
      __builtin_amdgcn_sched_barrier(0);  // row by row: interleaved, the rows' values spill
    }
    if (__builtin_expect(__any((outside[0] | outside[1] | outside[2] | outside[3]) != 0), 0)) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (__any(outside[k] != 0)) v[4 * q + k] = geglu_bwd8_outside<G>(d[k], g[k], u[k], ta, tf);
    }
  }
}

// The gated-GELU backward and the quantization of its dGU [M, 2I] (p: rows M, cols 2I) from dH [M,
// I] and GU [M, 2I], I % 128 == 0: dGU goes from registers to its copies. A block takes W / 2 tiles
// of H one below the other, of each the d_g tile by one wave and the d_u tile by another. 6 B read (10 B
// of loads: dH and the gate by both waves), 17 / 16 B a copy written per element of H; the lookups and conversions, 22 instructions an
// element of dGU, take about as long as the bytes and overlap them by half. W = 8 keeps 64 bytes a lane
// in scratch (13 registers), to fit four waves a SIMD. Both copies, W = 2 / 8,
// us (a copy of as many bytes): [64, 10240] 9.0 / 17.4, [512, 10240] 20.3 / 23.8 (8.4), [2001,
// 10240] 63.8 / 58.1 (32.6), [4096, 10240] 115 / 104 (66.8), [8192, 10240] 236 / 200 (134); in two
// passes 73 + 66 at [4096, 10240].
template <int W>
__global__ __launch_bounds__(64 * W, 4) void geglu_bwd_mx4_kernel(const uint16_t* __restrict__ dH,
                                                               const uint16_t* __restrict__ GU,
                                                               int64_t I, Mx4Out p) {
  __shared__ __attribute__((aligned(16))) uint16_t ta[kGeluABytes / 2];
  __shared__ __attribute__((aligned(16))) uint32_t tf[kGeluFBytes / 4];
  __shared__ Mx4Stage<W / 2> sh[2];
  load_gelu_tables<64 * W>(ta, tf);
  __syncthreads();
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wid = w >> 1, half = w & 1;
  const uint32_t tiles_c = (uint32_t)(I / kMx4Cols);
  const uint32_t tiles = tiles_c * (uint32_t)((p.rows + 16 * W - 1) / (16 * W));
  for (uint32_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t r0 = ((int64_t)(t / tiles_c) * (W / 2) + wid) * kMx4Rows;
    const int64_t c0 = (int64_t)(t % tiles_c) * kMx4Cols;
    const uint32_t ld = 2 * (uint32_t)I;
    const uint32_t left = (uint32_t)max((int64_t)0, min(p.rows - r0, (int64_t)kMx4Rows));
    const Window wd = window(dH + r0 * I, left * ld), wg = window(GU + r0 * 2 * I, left * 2 * ld);
    const uint32_t oc = 2 * (uint32_t)c0 + 16 * (lane & 15), rg = 8 * (lane >> 4);
    uint4 v[8];
    if (half == 0)
      geglu_bwd_rows<true>(wd, wg, oc + rg * ld, oc + 2 * rg * ld, ld, ta, tf, v);
    else
      geglu_bwd_rows<false>(wd, wg, oc + rg * ld, oc + 2 * rg * ld, ld, ta, tf, v);
    if (p.out_t) __syncthreads();  // the tile before has left the stage
    mx4_wave_tile<W / 2>(p, r0, half * I + c0, v, &sh[half], wid, lane);
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

// Elements up to which a tensor's columnwise codes leave each wave by themselves, and in 64-byte pieces
// (mx4_kernel's figures).
constexpr int64_t kMx4Alone = 8 << 20, kMx4Four = 32 << 20;
// Elements of H up to which the gated backward's blocks are of two waves (its kernel's figures).
constexpr int64_t kBwdTwo = 8 << 20;

template <int W>
int mx4_launch(const uint16_t* x, const Mx4Out& p, hipStream_t s) {
  const int64_t tiles = (p.rows + kMx4Rows * W - 1) / (kMx4Rows * W) * ((p.cols + kMx4Cols - 1) / kMx4Cols);
  hipLaunchKernelGGL(mx4_kernel<W>, dim3((unsigned)tiles), dim3(64 * W), 0, s, x, p);
  return launch_status("mx4_kernel");
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
  BF8_CHECK(p.cols % 8 == 0 && p.cols < (1 << 24), "%s: need cols %% 8 == 0 and cols < 2^24 (got %lld)",
            who, (long long)p.cols);
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
  const auto* xs = (const uint16_t*)x;
  hipStream_t s = as_stream(stream);
  if (!out_t || rows * cols <= kMx4Alone) return mx4_launch<1>(xs, p, s);
  return rows * cols <= kMx4Four ? mx4_launch<4>(xs, p, s) : mx4_launch<8>(xs, p, s);
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
  // (the kernel's figures; several tiles a block keep the tables' load small beside them)
  if (M * I <= kBwdTwo) {
    const int64_t tiles = (M + 31) / 32 * (I / 128);
    hipLaunchKernelGGL(geglu_bwd_mx4_kernel<2>, dim3((unsigned)std::min<int64_t>(tiles, 1024)),
                       dim3(128), 0, as_stream(stream), d, g, I, p);
  } else {
    const int64_t tiles = (M + 127) / 128 * (I / 128);
    hipLaunchKernelGGL(geglu_bwd_mx4_kernel<8>, dim3((unsigned)std::min<int64_t>(tiles, 512)),
                       dim3(512), 0, as_stream(stream), d, g, I, p);
  }
  return launch_status("geglu_bwd_mx4_kernel");
}

}  // extern "C"
