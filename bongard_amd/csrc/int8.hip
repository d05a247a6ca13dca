// 8-bit integer operands for gfx950: the quantizer of bf16 tensors with one scale for each row (token,
// output channel) and / or one for each column (for the backward's products, which sum over the other
// dimension), and the read-back. The products are gemm.hip's.
//
// Per row: scale = max(max |x|, 2^-40) / 127, code = 127 x / max(max |x|, 2^-40) rounded to nearest, ties
// to even (int8.hpp); x ~ code * scale. The columnwise copy is stored transposed, [cols, R] with R the
// rows rounded up to 16 and zeros past the rows, so that any number of rows is an operand.
//
// Kernels (x is read once for rows alone, else twice):
//   int8_row_kernel     rows alone: each row's maximum, scale and codes in one pass
//   int8_maxima_kernel  else one pass for the maxima: of each row in tiles of 512 columns, of each column in
//                       strips of rows (the gated-GELU backward writes its output's itself, mlp.hip)
//   int8_tile_kernel    and one for the codes: a tile's scales from those maxima, either copy or both
//   int8_pair_kernel    both copies of few rows in one launch: some blocks take rows, the others all rows of
//                       32 columns
#include <hip/hip_runtime.h>

#include <algorithm>

#include "int8.hpp"

namespace bf8 {
namespace {

constexpr int kNT = 512;               // threads of the row kernel (8 waves)
constexpr int64_t kMaxCols = 32768;    // widest row that the row kernel holds in registers
constexpr int64_t kRowBlocks = 2048;   // its most blocks
constexpr int kTileNT = 256;
constexpr int kTile = 128;             // the tile kernel's tile (rows x cols)
constexpr int kPitch = kTile / 4 + 1;  // dwords per staged row (odd)
constexpr int64_t kTileBlocks = 1024;

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
// row's maximum is known. Bound by memory (2 B read, 1 written an element): [4096, 10240] 22.0 us, [20480, 2560]
// 27.2 (5.7-5.8 TB/s), [64, 2560] 3.2.
template <int TPR, int V>
__global__ __launch_bounds__(kNT) void int8_row_kernel(const uint16_t* __restrict__ x, int64_t rows,
                                                       int cols, int64_t strip,
                                                       int8_t* __restrict__ out,
                                                       float* __restrict__ row_scale) {
  constexpr int G = kNT / TPR;
  const int g = threadIdx.x / TPR, tl = threadIdx.x % TPR;
  const int nvec = cols >> 3;
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
    for (int j = 0; j < V; ++j) m = max(m, absmax16(xv[j]));
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
}

// The maxima of strips of rows (a multiple of 32) by 512 columns, a block each: lane l of a wave holds
// columns 8 l .. +7 of the tile, the waves take eight rows at a time by turns. Bound by memory (2 B an element):
// [20480, 2560] 22.8 us, [4096, 10240] 21.8 (4.6 and 3.8 TB/s).
__global__ __launch_bounds__(kTileNT) void int8_maxima_kernel(const uint16_t* __restrict__ x,
                                                              Int8Maxima p) {
  __shared__ uint4 red[kTileNT / 64][64];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int tc = blockIdx.x % p.row_tiles;
  const int64_t ts = blockIdx.x / p.row_tiles;
  const int64_t r0 = ts * p.strip, c = 512 * tc + 8 * lane;
  const int64_t left = min((int64_t)p.strip, p.rows - r0);
  uint4 k = make_uint4(0u, 0u, 0u, 0u);
  for (int r = 8 * wid; r < left; r += 8 * (kTileNT / 64)) {
    const Window w = window(x + (r0 + r) * p.cols, (uint32_t)(min((int64_t)8, left - r) * p.cols * 2));
    uint4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = window_load(w, c < p.cols ? 2u * (uint32_t)(i * p.cols + c) : kPastEnd);
    Int8Rows m;
#pragma unroll
    for (int i = 0; i < 8; ++i) m.add(i, v[i], k);
    m.store(p, r0 + r, tc, lane);
  }
  int8_column_maxima<kTileNT / 64>(p, red, k, ts, c, wid, lane);
}

// The codes of 128 x 128 tiles. The tile's row and column maxima first: 16 threads hold 128 of either, 16 groups
// of them take the tiles (strips) by turns. Each wave casts 32 rows of all 128 columns: lane l holds columns
// 8 (l & 15) .. +7 of the rows 4 k + l / 16, k < 8; the columnwise codes meet in LDS and each wave turns 32
// columns of all 128 rows, so that every store instruction writes whole 128-byte lines. Rows past the
// tensor's are zeros in out_t [cols, ld]. Bound by memory (2 B read, 1 written an element and copy, x in part from
// the memory-side cache): both copies of [4096, 20480] 70 us, [20480, 2560] 43, [4096, 10240] 33 (4.8-5.1 TB/s). Tiles
// of 256 rows measured level. Both copies keep 12 bytes a lane in scratch under the bound of four waves a SIMD.
template <bool ROWS, bool COLS>
__global__ __launch_bounds__(kTileNT, 4) void int8_tile_kernel(const uint16_t* __restrict__ x, Int8Maxima p,
                                                            int64_t ld,
                                                            int8_t* __restrict__ out,
                                                            float* __restrict__ row_scale,
                                                            int8_t* __restrict__ out_t,
                                                            float* __restrict__ col_scale) {
  __shared__ uint32_t stage[kTile * kPitch];
  __shared__ float mults[2][kTile];
  uint4(*red)[2][16] = reinterpret_cast<uint4(*)[2][16]>(stage);  // [group][rows, columns][8 each]
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int64_t rows = p.rows, cols = p.cols;
  const int64_t tiles_c = (cols + kTile - 1) / kTile;
  const int64_t ntiles = tiles_c * ((rows + kTile - 1) / kTile);
  const int cl = lane & 15, lr = lane >> 4;
  for (int64_t t = blockIdx.x; t < ntiles; t += gridDim.x) {
    const int64_t r0 = (t / tiles_c) * kTile, c0 = (t % tiles_c) * kTile;
    const int64_t c = c0 + 8 * cl;
    const int left = (int)min((int64_t)kTile, rows - r0);
    const Window w = window(x + r0 * cols, (uint32_t)(left * cols * 2));
    uint4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      v[k] = window_load(w, c < cols ? 2u * (uint32_t)((32 * wid + 4 * k + lr) * cols + c) : kPastEnd);
    {
      const int g = threadIdx.x >> 4, e = 8 * (threadIdx.x & 15);
      auto more = [](uint4 a, uint4 b) __attribute__((always_inline)) {
        return make_uint4(pk_max_u16(a.x, b.x), pk_max_u16(a.y, b.y), pk_max_u16(a.z, b.z),
                          pk_max_u16(a.w, b.w));
      };
      uint4 a = make_uint4(0u, 0u, 0u, 0u), b = a;
      if (ROWS && e < left)
#pragma unroll 4
        for (int i = g; i < p.row_tiles; i += 16)
          a = more(a, *reinterpret_cast<const uint4*>(p.rowpart + i * int8_row_pad(rows) + r0 + e));
      if (COLS && c0 + e < cols)
#pragma unroll 4
        for (int i = g; i < p.strips; i += 16)
          b = more(b, *reinterpret_cast<const uint4*>(p.colpart + (int64_t)i * cols + c0 + e));
      if (ROWS) red[g][0][threadIdx.x & 15] = a;
      if (COLS) red[g][1][threadIdx.x & 15] = b;
      __syncthreads();
      const int which = threadIdx.x >> 7, i = threadIdx.x & 127;  // threads 0 .. 127: rows, the others: columns
      if (which ? COLS : ROWS) {
        uint32_t m = 0;
#pragma unroll
        for (int gg = 0; gg < 16; ++gg) m = max(m, (uint32_t)reinterpret_cast<const uint16_t*>(red[gg][which])[i]);
        const Int8Scale s = int8_scale(m << 16);
        mults[which][i] = s.mult;
        if (!which && c0 == 0 && i < left) row_scale[r0 + i] = s.scale;
        if (which && r0 == 0 && c0 + i < cols) col_scale[c0 + i] = s.scale;
      }
      __syncthreads();
    }
    if constexpr (ROWS) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int r = 32 * wid + 4 * k + lr;
        if (r < left && c < cols)
          *reinterpret_cast<uint2*>(out + (r0 + r) * cols + c) = int8_codes8(v[k], mults[0][r]);
      }
    }
    if constexpr (!COLS) continue;
    float m[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) m[e] = mults[1][8 * cl + e];
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
    if (rg < left) {  // ld holds whole pieces of 16 rows
#pragma unroll
      for (int cc = 0; cc < 4; ++cc) {
        const int64_t tr = c0 + 4 * cg + cc;  // row of out_t (a column of x)
        if (tr < cols) *reinterpret_cast<uint4*>(out_t + tr * ld + r0 + rg) = tq[cc];
      }
    }
    __syncthreads();
  }
}

// Both copies of up to 128 R rows. Blocks [0, row_blocks) are int8_row_kernel's of eight rows each (TPR 64, V
// vectors a lane). Of the others each takes 32 columns of all rows: four lanes a row (8 columns each), 128 rows
// a step, R steps held in registers; the columns' maxima by packed 16-bit maxima over lanes and waves, the
// codes turned in LDS. Bound by latency: [64, 2560] 4.1 us, [500, 2560] 6.7 (two passes over
// tiles, as below it 1,024 rows, 11.3).
constexpr int kPairCols = 32, kPairPitch = kPairCols / 4 + 1;
template <int V, int R>
__global__ __launch_bounds__(kNT) void int8_pair_kernel(const uint16_t* __restrict__ x, int rows, int cols,
                                                        int row_blocks, int8_t* __restrict__ out,
                                                        float* __restrict__ row_scale,
                                                        int8_t* __restrict__ out_t,
                                                        float* __restrict__ col_scale) {
  __shared__ uint32_t stage[R * 128 * kPairPitch];
  __shared__ uint4 top[kNT / 64][4];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  if ((int)blockIdx.x < row_blocks) {
    const int r = blockIdx.x * 8 + wid, nvec = cols >> 3;
    if (r >= rows) return;
    const Window w = window(x + (int64_t)r * cols, 2u * cols);
    uint4 v[V];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = window_load(w, 16u * (lane + 64 * j));
#pragma unroll
    for (int j = 0; j < V; ++j) m = max(m, absmax16(v[j]));
    const Int8Scale s = int8_scale(wave_max_u32(m) << 16);
    if (lane == 0) row_scale[r] = s.scale;
    uint2* orow = reinterpret_cast<uint2*>(out + (int64_t)r * cols);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (lane + 64 * j < nvec) orow[lane + 64 * j] = int8_codes8(v[j], s.mult);
    return;
  }
  const int c0 = (blockIdx.x - row_blocks) * kPairCols, cg = threadIdx.x & 3, rl = threadIdx.x >> 2;
  const int c = c0 + 8 * cg, ld = (rows + 15) / 16 * 16;
  const Window w = window(x, (uint32_t)(2 * rows * cols));
  uint4 v[R];
#pragma unroll
  for (int i = 0; i < R; ++i)
    v[i] = window_load(w, c < cols && 128 * i + rl < rows ? 2u * ((128 * i + rl) * cols + c) : kPastEnd);
  uint4 k = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
  for (int i = 0; i < R; ++i)
    k = make_uint4(pk_max_u16(k.x, v[i].x & 0x7FFF7FFFu), pk_max_u16(k.y, v[i].y & 0x7FFF7FFFu),
                   pk_max_u16(k.z, v[i].z & 0x7FFF7FFFu), pk_max_u16(k.w, v[i].w & 0x7FFF7FFFu));
#pragma unroll
  for (int off = 4; off < 64; off <<= 1)
    k = make_uint4(pk_max_u16(k.x, (uint32_t)__shfl_xor((int)k.x, off, 64)),
                   pk_max_u16(k.y, (uint32_t)__shfl_xor((int)k.y, off, 64)),
                   pk_max_u16(k.z, (uint32_t)__shfl_xor((int)k.z, off, 64)),
                   pk_max_u16(k.w, (uint32_t)__shfl_xor((int)k.w, off, 64)));
  if (lane < 4) top[wid][lane] = k;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kNT / 64; ++i) {
    const uint4 o = top[i][cg];
    k = make_uint4(pk_max_u16(k.x, o.x), pk_max_u16(k.y, o.y), pk_max_u16(k.z, o.z), pk_max_u16(k.w, o.w));
  }
  float mult[8], scale[8];
  const uint32_t kw[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const Int8Scale s = int8_scale(e & 1 ? kw[e >> 1] & 0xFFFF0000u : kw[e >> 1] << 16);
    mult[e] = s.mult;
    scale[e] = s.scale;
  }
  if (rl == 0 && c < cols) {
    reinterpret_cast<float4*>(col_scale + c)[0] = make_float4(scale[0], scale[1], scale[2], scale[3]);
    reinterpret_cast<float4*>(col_scale + c)[1] = make_float4(scale[4], scale[5], scale[6], scale[7]);
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const uint2 q = int8_codes8(v[i], mult);
    uint32_t* d = stage + (128 * i + rl) * kPairPitch + 2 * cg;
    d[0] = q.x;
    d[1] = q.y;
  }
  __syncthreads();
  // a thread turns 16 rows of 4 columns: 8 pieces of rows a step of 128, 8 groups of columns
  for (int it = threadIdx.x; it < R * 64; it += kNT) {
    const int r = (it & (8 * R - 1)) * 16, g = it / (8 * R);
    if (r >= rows || c0 + 4 * g >= cols) continue;
    uint32_t d[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) d[i] = stage[(r + i) * kPairPitch + g];
    uint4 tq[4];
    transpose_4x16(d, tq);
#pragma unroll
    for (int cc = 0; cc < 4; ++cc)
      *reinterpret_cast<uint4*>(out_t + (int64_t)(c0 + 4 * g + cc) * ld + r) = tq[cc];
  }
}

// bf16 [rows, cols] of codes [rows, cols] and a scale a row, 8 values a thread. Bound by memory: [20480, 2560] 24.9 us
// (6.3 TB/s), [64, 2560] 2.3.
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
// multiple of four; past the row they hold zeros). Bound by memory: [20480, 2560] 31.1 us (5.1 TB/s), its read-back
// 25.9 (6.2).
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
// fp32 into part[y][cols]; column_finish_kernel adds the parts in order. Bound by memory, of few rows by the two
// launches: [20480, 2560] 29.4 us (3.6 TB/s), [500, 2560] 8.8.
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

template <int TPR>
void launch_rows(const uint16_t* x, int64_t rows, int cols, int8_t* out, float* row_scale,
                 hipStream_t s) {
  const int64_t groups = kNT / TPR;
  const int64_t strip = ((rows + kRowBlocks - 1) / kRowBlocks + groups - 1) / groups * groups;
  const dim3 grid((unsigned)((rows + strip - 1) / strip));
#define BF8_INT8_ROW(VV)                                                                          \
  case VV:                                                                                        \
    hipLaunchKernelGGL((int8_row_kernel<TPR, VV>), grid, dim3(kNT), 0, s, x, rows, cols, strip,   \
                       out, row_scale);                                                           \
    break
  switch ((cols / 8 + TPR - 1) / TPR) {
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

// Tensors whose both copies int8_pair_kernel makes.
bool pair_fits(int64_t rows, int64_t cols) { return rows <= 1024 && cols <= 4096; }

int launch_tiles(const uint16_t* x, const Int8Maxima& p, int8_t* out, float* row_scale, int8_t* out_t,
                 float* col_scale, hipStream_t s) {
  const int64_t tiles = ((p.rows + kTile - 1) / kTile) * ((p.cols + kTile - 1) / kTile);
  const auto kernel = !out_t ? int8_tile_kernel<true, false>
                      : out  ? int8_tile_kernel<true, true>
                             : int8_tile_kernel<false, true>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(tiles, kTileBlocks)), dim3(kTileNT), 0, s, x, p,
                     (p.rows + 15) / 16 * 16, out, row_scale, out_t, col_scale);
  return launch_status("int8_tile_kernel");
}

int launch_pair(const uint16_t* x, int rows, int cols, int8_t* out, float* row_scale, int8_t* out_t,
                float* col_scale, hipStream_t s) {
  const int row_blocks = out ? (rows + 7) / 8 : 0, v = (cols / 8 + 63) / 64;
  const dim3 grid((unsigned)(row_blocks + (cols + kPairCols - 1) / kPairCols));
  const auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kNT), 0, s, x, rows, cols, row_blocks, out, row_scale, out_t,
                       col_scale);
  };
#define BF8_INT8_PAIR(R)                                             \
  if (v <= 2)                                                        \
    run(int8_pair_kernel<2, R>);                                     \
  else if (v <= 5)                                                   \
    run(int8_pair_kernel<5, R>);                                     \
  else                                                               \
    run(int8_pair_kernel<8, R>)
  if (rows <= 128) {
    BF8_INT8_PAIR(1);
  } else if (rows <= 512) {
    BF8_INT8_PAIR(4);
  } else {
    BF8_INT8_PAIR(8);
  }
#undef BF8_INT8_PAIR
  return launch_status("int8_pair_kernel");
}

}  // namespace

int int8_codes_of_maxima(const uint16_t* x, const Int8Maxima& p, int8_t* out, float* row_scale, int8_t* out_t,
                         float* col_scale, hipStream_t s) {
  return launch_tiles(x, p, out, row_scale, out_t, col_scale, s);
}
}  // namespace bf8

using namespace bf8;

extern "C" {

size_t bf8_quantize_int8_workspace(int64_t rows, int64_t cols, int both) {
  if (rows <= 0 || cols <= 0 || cols > kMaxCols || (both && pair_fits(rows, cols))) return 0;
  return int8_maxima_bytes(rows, cols);
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
  BF8_CHECK(!out_t || ((uintptr_t)col_scale & 15) == 0, "%s: col_scale must be 16-byte aligned", who);
  hipStream_t s = as_stream(stream);
  const auto* xs = (const uint16_t*)x;
  if (out && out_t && pair_fits(rows, cols))
    return launch_pair(xs, (int)rows, (int)cols, out, row_scale, out_t, col_scale, s);
  if (out_t)
    BF8_CHECK(ws && ws_bytes >= bf8_quantize_int8_workspace(rows, cols, 0) && ((uintptr_t)ws & 255) == 0,
              "%s: workspace needs %zu bytes, 256-byte aligned (got %zu)", who,
              bf8_quantize_int8_workspace(rows, cols, 0), ws_bytes);
  if (out_t && pair_fits(rows, cols))  // (the columnwise copy alone: 64 x 2560 4.1 us, in two launches 6.4)
    return launch_pair(xs, (int)rows, (int)cols, nullptr, nullptr, out_t, col_scale, s);
  if (!out_t) {
    if (cols <= 4096)
      launch_rows<64>(xs, rows, (int)cols, out, row_scale, s);
    else if (cols <= 16384)
      launch_rows<256>(xs, rows, (int)cols, out, row_scale, s);
    else
      launch_rows<512>(xs, rows, (int)cols, out, row_scale, s);
    return launch_status("int8_row_kernel");
  }
  const Int8Maxima p = int8_maxima(ws, rows, cols);
  hipLaunchKernelGGL(int8_maxima_kernel, dim3((unsigned)p.strips * p.row_tiles), dim3(kTileNT), 0, s, xs, p);
  if (const int rc = launch_status("int8_maxima_kernel")) return rc;
  return launch_tiles(xs, p, out, row_scale, out_t, col_scale, s);
}

int bf8_quantize_int8_maxima_bf16(const void* x, int64_t rows, int64_t cols, int halves, int8_t* out,
                                  float* row_scale, int8_t* out_t, float* col_scale, const void* maxima,
                                  size_t maxima_bytes, void* stream) {
  const char* who = "bf8_quantize_int8_maxima_bf16";
  BF8_CHECK(rows >= 0 && cols >= 0 && rows < (1LL << 31) && cols < (1 << 24), "%s: bad shape", who);
  BF8_CHECK((halves == 1 || halves == 2) && cols % (8 * halves) == 0,
            "%s: need cols %% 8 == 0 of each of 1 or 2 parts (got %lld of %d)", who, (long long)cols, halves);
  BF8_CHECK((out == nullptr) == (row_scale == nullptr) && (out_t == nullptr) == (col_scale == nullptr) &&
                (out || out_t),
            "%s: give out with row_scale and / or out_t with col_scale", who);
  if (rows == 0 || cols == 0) return BF8_OK;
  BF8_CHECK((((uintptr_t)x | (uintptr_t)out_t | (uintptr_t)col_scale) & 15) == 0 && ((uintptr_t)out & 7) == 0,
            "%s: x, out_t and col_scale must be 16-byte, out 8-byte aligned", who);
  BF8_CHECK(x && maxima && ((uintptr_t)maxima & 255) == 0 &&
                maxima_bytes >= int8_maxima_bytes(rows, cols, halves),
            "%s: x and %zu bytes of maxima, 256-byte aligned, must be given (got %zu)", who,
            int8_maxima_bytes(rows, cols, halves), maxima_bytes);
  return launch_tiles((const uint16_t*)x, int8_maxima(const_cast<void*>(maxima), rows, cols, halves), out,
                      row_scale, out_t, col_scale, as_stream(stream));
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
