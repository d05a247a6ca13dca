// 8-bit integer operands for gfx950: the quantizer of bf16 tensors with one scale for each row (token,
// output channel) and / or one for each column (for the backward's products, which sum over the other
// dimension), and the read-back. The products are gemm.hip's.
//
// Per row: scale = max(max |x|, 2^-40) / 127, code = 127 x / max(max |x|, 2^-40) rounded to nearest, ties
// to even (int8.hpp); x ~ code * scale. The columnwise copy is stored transposed, [cols, R] with R the
// rows rounded up to 16 and zeros past the rows, so that any number of rows is an operand.
//
// Kernels (x is read at most twice):
//   int8_row_kernel        one pass: each row's maximum, scale and codes; per-block column maxima
//   int8_col_scale_kernel  the blocks' column maxima -> scale and multiplier of each column
//   int8_col_kernel        second pass: the columns' codes, turned in LDS
#include <hip/hip_runtime.h>

#include <algorithm>

#include "int8.hpp"

namespace bf8 {
namespace {

constexpr int kNT = 512;                 // threads of the row kernel (8 waves)
constexpr int64_t kMaxCols = 32768;      // widest row that the row kernel holds in registers
constexpr int64_t kBlocksColumns = 512;  // row-kernel blocks where it writes column maxima
constexpr int64_t kBlocksRows = 2048;    // ... where it does not
constexpr int kScaleNT = 1024;
constexpr int kColNT = 256;
constexpr int kTile = 128;               // column kernel's tile (rows x cols)
constexpr int kPitch = kTile / 4 + 1;    // dwords per staged row (odd)
constexpr int64_t kMaxColBlocks = 2048;

// Max of m over the TPR threads of a row; every thread of the block must call it (TPR > 64: through LDS).
template <int TPR>
__device__ __forceinline__ uint32_t group_max(uint32_t m) {
  m = wave_max_u32(m);
  if constexpr (TPR == 64) {
    return m;
  } else {
    constexpr int W = TPR / 64;
    __shared__ uint32_t red[kNT / 64];
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) red[w] = m;
    __syncthreads();
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) r = max(r, red[w / W * W + i]);
    __syncthreads();
    return r;
  }
}

// Rows [blockIdx.x * strip, + strip) of x, one row per TPR threads at a time (strip is a multiple of the
// kNT / TPR rows taken at once, so every group runs the same number of steps). Thread tl of a group holds
// the row's 16-byte vectors tl, tl + TPR, ... (V of them); the next row's are loaded before this
// row's maximum is known. out / row_scale, colpart ([gridDim.x][cols] bf16 keys): each may be NULL.
template <int TPR, int V>
__global__ __launch_bounds__(kNT) void int8_row_kernel(const uint16_t* __restrict__ x, int64_t rows,
                                                       int cols, int64_t strip,
                                                       int8_t* __restrict__ out,
                                                       float* __restrict__ row_scale,
                                                       uint16_t* __restrict__ colpart) {
  constexpr int G = kNT / TPR;
  extern __shared__ uint4 cbuf[];  // [G - 1][cols / 8] column keys of groups 1.. (colpart)
  const int g = threadIdx.x / TPR, tl = threadIdx.x % TPR;
  const int nvec = cols >> 3;
  uint4 ck[V];
#pragma unroll
  for (int j = 0; j < V; ++j) ck[j] = make_uint4(0u, 0u, 0u, 0u);
  const int64_t r0 = blockIdx.x * strip;
  constexpr bool kAhead = V < 8;  // (eight vectors of two rows leave too few waves)
  uint4 next[V];
  auto load = [&](int64_t r) {
    const uint4* xr = reinterpret_cast<const uint4*>(x + r * cols);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int v = tl + TPR * j;
      next[j] = (r < rows && v < nvec) ? xr[v] : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  if (kAhead) load(r0 + g);
  for (int64_t rr = g; rr < strip; rr += G) {
    const int64_t r = r0 + rr;
    if (!kAhead) load(r);
    uint4 xv[V];
#pragma unroll
    for (int j = 0; j < V; ++j) xv[j] = next[j];
    if (kAhead && rr + G < strip) load(r + G);
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      m = max(m, absmax16(xv[j]));
      if (colpart)
        ck[j] = make_uint4(pk_max_u16(ck[j].x, xv[j].x & 0x7FFF7FFFu),
                           pk_max_u16(ck[j].y, xv[j].y & 0x7FFF7FFFu),
                           pk_max_u16(ck[j].z, xv[j].z & 0x7FFF7FFFu),
                           pk_max_u16(ck[j].w, xv[j].w & 0x7FFF7FFFu));
    }
    if (!out) continue;
    m = group_max<TPR>(m);
    if (r >= rows) continue;
    const Int8Scale s = int8_scale(m << 16);
    if (tl == 0) row_scale[r] = s.scale;
    uint2* orow = reinterpret_cast<uint2*>(out + r * cols);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int v = tl + TPR * j;
      if (v < nvec) orow[v] = int8_codes8(xv[j], s.mult);
    }
  }
  if (!colpart) return;
  uint4* dst = reinterpret_cast<uint4*>(colpart + (int64_t)blockIdx.x * cols);
  if constexpr (G == 1) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int v = tl + TPR * j;
      if (v < nvec) dst[v] = ck[j];
    }
  } else {
    // groups 1.. hand their keys to group 0, whose threads hold the same columns
    if (g > 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int v = tl + TPR * j;
        if (v < nvec) cbuf[(g - 1) * nvec + v] = ck[j];
      }
    }
    __syncthreads();
    if (g == 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int v = tl + TPR * j;
        if (v >= nvec) continue;
        uint4 k = ck[j];
#pragma unroll
        for (int gg = 1; gg < G; ++gg) {
          const uint4 o = cbuf[(gg - 1) * nvec + v];
          k = make_uint4(pk_max_u16(k.x, o.x), pk_max_u16(k.y, o.y), pk_max_u16(k.z, o.z),
                         pk_max_u16(k.w, o.w));
        }
        dst[v] = k;
      }
    }
  }
}

// Scale and multiplier of each column from the row kernel's maxima [nblk][cols]: a block takes 64 columns
// (8 threads of 8) and spreads the nblk rows over 128 thread rows.
__global__ __launch_bounds__(kScaleNT) void int8_col_scale_kernel(
    const uint16_t* __restrict__ colpart, int nblk, int cols, float* __restrict__ col_mult,
    float* __restrict__ col_scale) {
  constexpr int kTR = kScaleNT / 8, kW = kScaleNT / 64;
  __shared__ uint4 red[kW][8];
  const int cg = threadIdx.x & 7, rg = threadIdx.x >> 3;
  const int nvec = cols >> 3;
  const int v = blockIdx.x * 8 + cg;
  uint32_t k[4] = {0u, 0u, 0u, 0u};
  if (v < nvec) {
    const uint4* src = reinterpret_cast<const uint4*>(colpart);
#pragma unroll 4
    for (int b = rg; b < nblk; b += kTR) {
      const uint4 o = src[(int64_t)b * nvec + v];
      k[0] = pk_max_u16(k[0], o.x);
      k[1] = pk_max_u16(k[1], o.y);
      k[2] = pk_max_u16(k[2], o.z);
      k[3] = pk_max_u16(k[3], o.w);
    }
  }
#pragma unroll
  for (int off = 8; off < 64; off <<= 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) k[i] = pk_max_u16(k[i], (uint32_t)__shfl_xor((int)k[i], off, 64));
  }
  if ((threadIdx.x & 63) < 8) red[threadIdx.x >> 6][cg] = make_uint4(k[0], k[1], k[2], k[3]);
  __syncthreads();
  const int c = blockIdx.x * 64 + threadIdx.x;
  if (threadIdx.x >= 64 || c >= cols) return;
  uint32_t m = 0;
#pragma unroll
  for (int w = 0; w < kW; ++w)
    m = max(m, (uint32_t)reinterpret_cast<const uint16_t*>(red[w])[threadIdx.x]);
  const Int8Scale s = int8_scale(m << 16);
  col_mult[c] = s.mult;
  col_scale[c] = s.scale;
}

// out_t [cols, ld] = the columns' codes. A block takes 128 x 128 tiles, each wave 32 rows of all 128
// columns: lane l holds columns 8 (l & 15) .. +7 of the rows 4 k + l / 16, k < 8; the codes meet in LDS and
// each wave turns 32 columns of all 128 rows, so that every store instruction writes whole 128-byte
// lines. Rows past the tensor's are zeros.
__global__ __launch_bounds__(kColNT) void int8_col_kernel(const uint16_t* __restrict__ x,
                                                          int64_t rows, int64_t cols, int64_t ld,
                                                          const float* __restrict__ col_mult,
                                                          int8_t* __restrict__ out_t) {
  __shared__ uint32_t stage[kTile * kPitch];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int64_t tiles_c = (cols + kTile - 1) / kTile;
  const int64_t ntiles = tiles_c * ((rows + kTile - 1) / kTile);
  const int cl = lane & 15, lr = lane >> 4;
  for (int64_t t = blockIdx.x; t < ntiles; t += gridDim.x) {
    const int64_t r0 = (t / tiles_c) * kTile, c0 = (t % tiles_c) * kTile;
    const int64_t c = c0 + 8 * cl;
    uint4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int64_t r = r0 + 32 * wid + 4 * k + lr;
      v[k] = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows && c < cols) v[k] = *reinterpret_cast<const uint4*>(x + r * cols + c);
    }
    float m[8] = {};
    if (c < cols) {
      const float4 s0 = reinterpret_cast<const float4*>(col_mult + c)[0];
      const float4 s1 = reinterpret_cast<const float4*>(col_mult + c)[1];
      m[0] = s0.x; m[1] = s0.y; m[2] = s0.z; m[3] = s0.w;
      m[4] = s1.x; m[5] = s1.y; m[6] = s1.z; m[7] = s1.w;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint2 q = int8_codes8(v[k], m);
      uint32_t* d = stage + (32 * wid + 4 * k + lr) * kPitch + 2 * cl;
      d[0] = q.x;
      d[1] = q.y;
    }
    __syncthreads();
    // lane: 16 rows (lane & 7) x 4 columns (lane >> 3) of the wave's 32 columns
    const int rg = (lane & 7) * 16, cg = 8 * wid + (lane >> 3);
    uint32_t d[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) d[i] = stage[(rg + i) * kPitch + cg];
    uint4 tq[4];
    transpose_4x16(d, tq);
    if (r0 + rg < rows) {  // ld holds whole pieces of 16 rows
#pragma unroll
      for (int cc = 0; cc < 4; ++cc) {
        const int64_t tr = c0 + 4 * cg + cc;  // row of out_t (a column of x)
        if (tr < cols) *reinterpret_cast<uint4*>(out_t + tr * ld + r0 + rg) = tq[cc];
      }
    }
    __syncthreads();
  }
}

// bf16 [rows, cols] of codes [rows, cols] and a scale a row, 8 values a thread.
__global__ __launch_bounds__(256) void int8_dequant_kernel(const int8_t* __restrict__ q,
                                                           const float* __restrict__ scale,
                                                           int64_t rows, int64_t cols,
                                                           uint16_t* __restrict__ out) {
  const int64_t per_row = cols >> 3, n = rows * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const float s = scale[i / per_row];
    const uint2 c = reinterpret_cast<const uint2*>(q)[i];
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t d = j < 2 ? c.x : c.y;
      w[j] = pack_bf16x2(code_f32(d, 2 * (j & 1)) * s, code_f32(d, 2 * (j & 1) + 1) * s);
    }
    reinterpret_cast<uint4*>(out)[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Checkpoint blocks of 32 along the rows of x: four lanes of 8 values a block (per_row of them a row, a
// multiple of four; past the row they hold zeros).
__global__ __launch_bounds__(256) void mxi8_kernel(const uint16_t* __restrict__ x, int64_t rows,
                                                   int64_t cols, int64_t per_row,
                                                   int8_t* __restrict__ out,
                                                   uint8_t* __restrict__ exps) {
  const int64_t n = rows * per_row, stride = (int64_t)gridDim.x * 256;  // whole blocks in any stride
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += stride) {
    const int64_t row = i / per_row, c = (i - row * per_row) * 8;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (c < cols) v = *reinterpret_cast<const uint4*>(x + row * cols + c);
    const uint32_t e = mxi8_exponent(quad_max(absmax16(v)));
    if (c < cols) *reinterpret_cast<uint2*>(out + row * cols + c) = mxi8_codes8(v, e);
    if ((i & 3) == 0) exps[row * (per_row >> 2) + (c >> 5)] = (uint8_t)e;
  }
}

__global__ __launch_bounds__(256) void mxi8_dequant_kernel(const int8_t* __restrict__ q,
                                                           const uint8_t* __restrict__ exps,
                                                           int64_t rows, int64_t cols,
                                                           uint16_t* __restrict__ out) {
  const int64_t per_row = cols >> 3, blocks = (cols + 31) >> 5, n = rows * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / per_row, v = i - row * per_row;
    const float step = mxi8_step(exps[row * blocks + (v >> 2)]);
    reinterpret_cast<uint4*>(out)[i] = mxi8_values8(reinterpret_cast<const uint2*>(q)[i], step);
  }
}

// Sums of columns: block (x, y) adds rows y, y + gridDim.y, .. (eight of them a step, of 256 columns) in
// fp32 into part[y][cols]; column_finish_kernel adds the parts in order.
constexpr int kSumCols = 256;
constexpr int64_t kSumStrips = 64;
int64_t sum_strips(int64_t rows) { return std::min<int64_t>((rows + 7) / 8, kSumStrips); }

__global__ __launch_bounds__(256) void column_sums_kernel(const uint16_t* __restrict__ x, int64_t rows,
                                                          int64_t cols, float* __restrict__ part) {
  __shared__ float red[8][kSumCols + 1];
  const int l = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * kSumCols + 8 * l;
  float a[8] = {};
  if (c < cols)
    for (int64_t r = (int64_t)blockIdx.y * 8 + g; r < rows; r += (int64_t)gridDim.y * 8) {
      const uint4 v = *reinterpret_cast<const uint4*>(x + r * cols + c);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[2 * e] += bf16_lo(w[e]);
        a[2 * e + 1] += bf16_hi(w[e]);
      }
    }
#pragma unroll
  for (int e = 0; e < 8; ++e) red[g][8 * l + e] = a[e];
  __syncthreads();
  const int64_t col = (int64_t)blockIdx.x * kSumCols + threadIdx.x;
  if (col >= cols) return;
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s += red[i][threadIdx.x];
  part[blockIdx.y * cols + col] = s;
}

__global__ __launch_bounds__(256) void column_finish_kernel(const float* __restrict__ part, int strips,
                                                            int64_t cols, uint16_t* __restrict__ out) {
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col >= cols) return;
  float s = 0.0f;
#pragma unroll 8
  for (int i = 0; i < strips; ++i) s += part[i * cols + col];
  out[col] = (uint16_t)f32_to_bf16_bits(s);
}

struct RowPlan {
  int tpr, v;
  int64_t strip, blocks;
  size_t part_bytes;  // column maxima, 256-byte aligned
};

RowPlan row_plan(int64_t rows, int64_t cols, bool colwise) {
  RowPlan p{};
  p.tpr = cols <= 4096 ? 64 : cols <= 16384 ? 256 : 512;
  p.v = (int)((cols / 8 + p.tpr - 1) / p.tpr);  // <= 8
  const int64_t groups = kNT / p.tpr, cap = colwise ? kBlocksColumns : kBlocksRows;
  p.strip = ((rows + cap - 1) / cap + groups - 1) / groups * groups;
  p.blocks = (rows + p.strip - 1) / p.strip;
  p.part_bytes = colwise ? ((size_t)p.blocks * (size_t)cols * 2 + 255) / 256 * 256 : 0;
  return p;
}

template <int TPR>
void launch_rows(const RowPlan& p, const uint16_t* x, int64_t rows, int cols, int8_t* out,
                 float* row_scale, uint16_t* colpart, hipStream_t s) {
  const size_t lds = colpart ? (size_t)(kNT / TPR - 1) * cols * 2 : 0;
#define BF8_INT8_ROW(VV)                                                                        \
  case VV:                                                                                      \
    hipLaunchKernelGGL((int8_row_kernel<TPR, VV>), dim3((unsigned)p.blocks), dim3(kNT), lds, s, \
                       x, rows, cols, p.strip, out, row_scale, colpart);                        \
    break
  switch (p.v) {
    BF8_INT8_ROW(1);
    BF8_INT8_ROW(2);
    BF8_INT8_ROW(3);
    BF8_INT8_ROW(4);
    BF8_INT8_ROW(5);
    BF8_INT8_ROW(6);
    BF8_INT8_ROW(7);
    BF8_INT8_ROW(8);
  }
#undef BF8_INT8_ROW
}

}  // namespace
}  // namespace bf8

using namespace bf8;

extern "C" {

size_t bf8_quantize_int8_workspace(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0 || cols > kMaxCols) return 0;
  return row_plan(rows, cols, true).part_bytes + (size_t)cols * 4;
}

int bf8_quantize_int8_bf16(const void* x, int64_t rows, int64_t cols, int8_t* out, float* row_scale,
                           int8_t* out_t, float* col_scale, void* ws, size_t ws_bytes,
                           void* stream) {
  const char* who = "bf8_quantize_int8_bf16";
  BF8_CHECK(rows >= 0 && cols >= 0 && rows < (1LL << 31), "%s: bad shape", who);
  BF8_CHECK(cols % 8 == 0 && cols <= kMaxCols, "%s: need cols %% 8 == 0 and cols <= %lld (got %lld)",
            who, (long long)kMaxCols, (long long)cols);
  BF8_CHECK((out == nullptr) == (row_scale == nullptr) && (out_t == nullptr) == (col_scale == nullptr) &&
                (out || out_t),
            "%s: give out with row_scale and / or out_t with col_scale", who);
  if (rows == 0 || cols == 0) return BF8_OK;
  BF8_CHECK(x != nullptr, "%s: x is NULL", who);
  BF8_CHECK((((uintptr_t)x | (uintptr_t)out_t) & 15) == 0 && ((uintptr_t)out & 7) == 0,
            "%s: x and out_t must be 16-byte, out 8-byte aligned", who);
  if (out_t)
    BF8_CHECK(ws && ws_bytes >= bf8_quantize_int8_workspace(rows, cols) && ((uintptr_t)ws & 255) == 0,
              "%s: workspace needs %zu bytes, 256-byte aligned (got %zu)", who,
              bf8_quantize_int8_workspace(rows, cols), ws_bytes);
  const auto* xs = (const uint16_t*)x;
  hipStream_t s = as_stream(stream);
  const RowPlan p = row_plan(rows, cols, out_t != nullptr);
  uint16_t* colpart = out_t ? (uint16_t*)ws : nullptr;
  if (p.tpr == 64)
    launch_rows<64>(p, xs, rows, (int)cols, out, row_scale, colpart, s);
  else if (p.tpr == 256)
    launch_rows<256>(p, xs, rows, (int)cols, out, row_scale, colpart, s);
  else
    launch_rows<512>(p, xs, rows, (int)cols, out, row_scale, colpart, s);
  int rc = launch_status("int8_row_kernel");
  if (rc != BF8_OK || !out_t) return rc;
  float* col_mult = (float*)((uint8_t*)ws + p.part_bytes);
  hipLaunchKernelGGL(int8_col_scale_kernel, dim3((unsigned)((cols / 8 + 7) / 8)), dim3(kScaleNT), 0, s,
                     colpart, (int)p.blocks, (int)cols, col_mult, col_scale);
  if ((rc = launch_status("int8_col_scale_kernel")) != BF8_OK) return rc;
  const int64_t tiles = ((rows + kTile - 1) / kTile) * ((cols + kTile - 1) / kTile);
  hipLaunchKernelGGL(int8_col_kernel, dim3((unsigned)std::min(tiles, kMaxColBlocks)), dim3(kColNT), 0, s,
                     xs, rows, cols, (rows + 15) / 16 * 16, col_mult, out_t);
  return launch_status("int8_col_kernel");
}

int bf8_dequant_int8(const int8_t* codes, const float* scale, int64_t rows, int64_t cols, void* out,
                     void* stream) {
  const char* who = "bf8_dequant_int8";
  BF8_CHECK(rows >= 0 && cols >= 0 && cols % 8 == 0, "%s: need cols %% 8 == 0 (rows %lld, cols %lld)",
            who, (long long)rows, (long long)cols);
  if (rows == 0 || cols == 0) return BF8_OK;
  BF8_CHECK(codes && scale && out, "%s: NULL pointer", who);
  BF8_CHECK(((uintptr_t)codes & 7) == 0 && ((uintptr_t)out & 15) == 0,
            "%s: out must be 16-byte, codes 8-byte aligned", who);
  const int64_t n = rows * (cols / 8);
  hipLaunchKernelGGL(int8_dequant_kernel, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 1 << 20)),
                     dim3(256), 0, as_stream(stream), codes, scale, rows, cols, (uint16_t*)out);
  return launch_status("int8_dequant_kernel");
}

static int check_mxi8(const char* who, int64_t rows, int64_t cols, const void* bf16, const void* codes,
                      const void* exps) {
  BF8_CHECK(rows >= 0 && cols >= 0 && cols % 8 == 0, "%s: need cols %% 8 == 0 (rows %lld, cols %lld)",
            who, (long long)rows, (long long)cols);
  if (rows == 0 || cols == 0) return BF8_OK;
  BF8_CHECK(bf16 && codes && exps, "%s: NULL pointer", who);
  BF8_CHECK(((uintptr_t)bf16 & 15) == 0 && ((uintptr_t)codes & 7) == 0,
            "%s: the bf16 tensor must be 16-byte, codes 8-byte aligned", who);
  return BF8_OK;
}

int bf8_quantize_mxint8_bf16(const void* x, int64_t rows, int64_t cols, int8_t* codes, uint8_t* exps,
                             void* stream) {
  if (const int rc = check_mxi8("bf8_quantize_mxint8_bf16", rows, cols, x, codes, exps)) return rc;
  if (rows == 0 || cols == 0) return BF8_OK;
  const int64_t per_row = (cols + 31) / 32 * 4, n = rows * per_row;
  hipLaunchKernelGGL(mxi8_kernel, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 1 << 20)), dim3(256),
                     0, as_stream(stream), (const uint16_t*)x, rows, cols, per_row, codes, exps);
  return launch_status("mxi8_kernel");
}

int bf8_dequant_mxint8(const int8_t* codes, const uint8_t* exps, int64_t rows, int64_t cols, void* out,
                       void* stream) {
  if (const int rc = check_mxi8("bf8_dequant_mxint8", rows, cols, out, codes, exps)) return rc;
  if (rows == 0 || cols == 0) return BF8_OK;
  const int64_t n = rows * (cols / 8);
  hipLaunchKernelGGL(mxi8_dequant_kernel, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 1 << 20)),
                     dim3(256), 0, as_stream(stream), codes, exps, rows, cols, (uint16_t*)out);
  return launch_status("mxi8_dequant_kernel");
}

size_t bf8_column_sums_workspace(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return (size_t)sum_strips(rows) * (size_t)cols * sizeof(float);
}

int bf8_column_sums_bf16(const void* x, int64_t rows, int64_t cols, void* out, void* ws, size_t ws_bytes,
                         void* stream) {
  const char* who = "bf8_column_sums_bf16";
  BF8_CHECK(rows > 0 && cols >= 0 && cols % 8 == 0 && cols < (1LL << 31),
            "%s: need rows > 0 and cols %% 8 == 0 (rows %lld, cols %lld)", who, (long long)rows,
            (long long)cols);
  if (cols == 0) return BF8_OK;
  BF8_CHECK(x && out && ((uintptr_t)x & 15) == 0, "%s: x (16-byte aligned) and out must be given", who);
  BF8_CHECK(ws && ws_bytes >= bf8_column_sums_workspace(rows, cols) && ((uintptr_t)ws & 15) == 0,
            "%s: workspace of %zu bytes, need %zu, 16-byte aligned", who, ws_bytes,
            bf8_column_sums_workspace(rows, cols));
  hipStream_t s = as_stream(stream);
  const int64_t strips = sum_strips(rows);
  hipLaunchKernelGGL(column_sums_kernel,
                     dim3((unsigned)((cols + kSumCols - 1) / kSumCols), (unsigned)strips), dim3(256), 0, s,
                     (const uint16_t*)x, rows, cols, (float*)ws);
  if (const int rc = launch_status("column_sums_kernel")) return rc;
  hipLaunchKernelGGL(column_finish_kernel, dim3((unsigned)((cols + 255) / 256)), dim3(256), 0, s,
                     (const float*)ws, (int)strips, cols, (uint16_t*)out);
  return launch_status("column_finish_kernel");
}

}  // extern "C"
