// Layer norm of the rows of a bf16 tensor and its backward, for gfx950. Per row, in fp32:
//   mean = sum(x) / cols,  r = 1 / sqrt(sum((x - mean)^2) / cols + eps),  n = (x - mean) r
//   y    = bf16(n w + b)
// The backward of dy, from x, mean and r:
//   c  = dy w,  dx = bf16(r (c - mean(c) - n mean(c n)))
//   dw = bf16(sum over rows of dy n),  db = bf16(sum over rows of dy)
// The forward can write x's checkpoint (blocks of 32 codes under a power of two, int8.hpp) in the same
// pass; the backward then reads that instead of x: n of the values it holds, with the mean and r of x
// itself. Sums over rows go through per-block partials added in a fixed order (deterministic).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "int8.hpp"

namespace bf8 {
namespace {

constexpr int kMaxCols = 16384;
constexpr int64_t kMaxFwdBlocks = 2048, kFewRows = 512;
struct LayerNorm {
  const uint16_t *x, *w, *b;
  int64_t rows;
  int cols;
  float eps;
  uint16_t* y;
  float *mean, *rstd;
  int8_t* x8;
  uint8_t* x8_e;
  const uint16_t* dy;
  uint16_t* dx;
  float* part;  // [blocks][2][cols]: sums of dy n, of dy
};

// Threads of a block whose rows take WPR waves each: four rows of one wave, or one row of more.
constexpr int block_threads(int wpr) { return wpr == 1 ? 256 : 64 * wpr; }

// Sums of N values over the row's threads: a wave, or the block's waves through LDS, added in order.
template <int N, int WPR>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*red)[WPR]) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], off, 64);
  if constexpr (WPR > 1) {
    const int wid = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) red[i][wid] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = red[i][0];
#pragma unroll
      for (int w = 1; w < WPR; ++w) v[i] += red[i][w];
    }
  }
}

// Row `row` of a [rows, cols] tensor of `bytes` an element: past its end, and anywhere in one that is NULL,
// it reads as zeros and is not written.
__device__ __forceinline__ Window row_of(const void* p, int64_t row, int cols, int bytes = 2) {
  return window((const uint8_t*)p + row * cols * bytes, p ? (uint32_t)(bytes * cols) : 0u);
}

template <int V, int WPR>
__device__ __forceinline__ void load_row(Window w, int t, uint4 (&v)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = window_load(w, 16u * (t + 64 * WPR * j));
}

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = bf16_lo(w[e]);
    f[2 * e + 1] = bf16_hi(w[e]);
  }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                    pack_bf16x2(f[6], f[7]));
}

// From here on the compiler knows nothing of v, so that it unpacks it again where it is used next
// and does not hold two floats for each of its dwords.
__device__ __forceinline__ void keep_packed(uint4& v) {
  asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w));
}

// A row takes WPR waves, a thread V pieces of 8 columns of it. Bound by memory (4 bytes an element, 5.03 with the
// checkpoint): [18494, 2560] 32 us as a wave a row (35 at a copy's rate; from the memory-side cache in part), with the
// checkpoint 41 (three waves 33 and 43: a barrier between two sums); [3001, 4104] as three waves 11.3 and 16.1 us
// (five 13.1, nine 14.9, sixteen 20.7: idle lanes, and fewer rows in flight on a CU); [4096, 8192] as four waves of
// four pieces 22.9 and 30.5 (eight of two 23.6 and 32.1, sixteen of one 28.8 and 40.1). Few rows take more waves:
// [64, 2560] as five 3.2 us, as one 3.7.
template <int V, int WPR, bool CKPT>
__global__ __launch_bounds__(block_threads(WPR)) void layer_norm_kernel(LayerNorm p) {
  __shared__ float red[2][1][WPR];
  const int t = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t first = WPR == 1 ? (int64_t)blockIdx.x * 4 + wid : blockIdx.x;
  const int64_t stride = WPR == 1 ? (int64_t)gridDim.x * 4 : gridDim.x;
  const int nvec = p.cols >> 3, blocks = (p.cols + 31) >> 5;
  uint4 w[V], b[V];
  load_row<V, WPR>(row_of(p.w, 0, p.cols), t, w);
  load_row<V, WPR>(row_of(p.b, 0, p.cols), t, b);
  for (int64_t row = first; row < p.rows; row += stride) {
    uint4 x[V];
    load_row<V, WPR>(row_of(p.x, row, p.cols), t, x);
    float s[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float f[8];
      unpack8(x[j], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[0] += f[e];
    }
    row_sum<1, WPR>(s, red[0]);
    const float mean = __fdiv_rn(s[0], (float)p.cols);
    s[0] = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float in = t + 64 * WPR * j < nvec ? 1.0f : 0.0f;  // pieces past the row count nothing
      float f[8];
      keep_packed(x[j]);
      unpack8(x[j], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = (f[e] - mean) * in;
        s[0] = fmaf(d, d, s[0]);
      }
    }
    row_sum<1, WPR>(s, red[1]);
    const float r = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(s[0], (float)p.cols) + p.eps));
    if (t == 0 && p.mean) {
      p.mean[row] = mean;
      p.rstd[row] = r;
    }
    const Window y = row_of(p.y, row, p.cols);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = t + 64 * WPR * j;
      if constexpr (CKPT) {  // (four lanes hold a block: all of them take part)
        const uint32_t e = mxi8_exponent(quad_max(absmax16(x[j])));
        if (i < nvec) {
          reinterpret_cast<uint2*>(p.x8 + row * p.cols)[i] = mxi8_codes8(x[j], e);
          if ((i & 3) == 0) p.x8_e[row * blocks + (i >> 2)] = (uint8_t)e;
        }
      }
      float f[8], g[8], h[8];
      keep_packed(x[j]);
      keep_packed(w[j]);
      keep_packed(b[j]);
      unpack8(x[j], f);
      unpack8(w[j], g);
      unpack8(b[j], h);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = fmaf((f[e] - mean) * r, g[e], h[e]);
      window_store(y, 16u * i, pack8(f));
    }
  }
}

// The n of piece i of a row, from x or from its checkpoint.
template <bool CKPT>
struct Piece {
  uint4 x;
};
template <>
struct Piece<true> {
  uint2 q;
  uint32_t e;
};

// A thread's sums of dy n and dy into the block's partial row: t of `threads` of a row.
template <int V>
__device__ __forceinline__ void write_sums(const LayerNorm& p, int t, int threads, const float (&aw)[V][8],
                                           const float (&ab)[V][8]) {
  float* dst = p.part + (int64_t)blockIdx.x * 2 * p.cols;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = t + threads * j;
    if (i >= p.cols >> 3) continue;
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const float(&a)[8] = h < 2 ? aw[j] : ab[j];
      *reinterpret_cast<float4*>(dst + (h < 2 ? 0 : p.cols) + 8 * i + 4 * (h & 1)) =
          make_float4(a[4 * (h & 1)], a[4 * (h & 1) + 1], a[4 * (h & 1) + 2], a[4 * (h & 1) + 3]);
    }
  }
}

// Rows of up to 1,536 columns, a wave each: their column sums stay in the wave's registers and the block's four
// waves add theirs at the end. [20000, 640] 25.5 us with the kernel that adds the partials, [8000, 1536] 21.2 (the
// kernel below 29.0 and 24.2); from 2,048 columns on a wave's sums and rows leave one wave a SIMD ([18494, 2560] 66,
// the kernel below 57).
template <int V, bool CKPT>
__global__ __launch_bounds__(256) void layer_norm_bwd_kernel(LayerNorm p) {
  __shared__ float4 sums[2 * V * 4 * 64];  // two waves' column sums
  const int t = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t first = (int64_t)blockIdx.x * 4 + wid;
  const int64_t stride = (int64_t)gridDim.x * 4;
  const int nvec = p.cols >> 3, blocks = (p.cols + 31) >> 5;
  const float inv = 1.0f / (float)p.cols;
  uint4 w[V];
  load_row<V, 1>(row_of(p.w, 0, p.cols), t, w);
  float aw[V][8], ab[V][8];
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) aw[j][e] = ab[j][e] = 0.0f;
  for (int64_t row = first; row < p.rows; row += stride) {
    uint4 dy[V];
    Piece<CKPT> x[V];
    load_row<V, 1>(row_of(p.dy, row, p.cols), t, dy);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = t + 64 * j;
      if constexpr (CKPT) {
        x[j].q = make_uint2(0u, 0u);
        x[j].e = 133u;
        if (i < nvec) {
          x[j].q = reinterpret_cast<const uint2*>(p.x8 + row * p.cols)[i];
          x[j].e = p.x8_e[row * blocks + (i >> 2)];
        }
      } else {
        x[j].x = window_load(row_of(p.x, row, p.cols), 16u * i);
      }
    }
    const float mean = p.mean[row], r = p.rstd[row];
    auto norm = [&](int j, float (&n)[8]) __attribute__((always_inline)) {
      if constexpr (CKPT) {
        const float step = mxi8_step(x[j].e);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          n[e] = (code_f32(e < 4 ? x[j].q.x : x[j].q.y, e & 3) * step - mean) * r;
      } else {
        keep_packed(x[j].x);
        unpack8(x[j].x, n);
#pragma unroll
        for (int e = 0; e < 8; ++e) n[e] = (n[e] - mean) * r;
      }
    };
    float s[2] = {0.0f, 0.0f};  // sums of c, c n (dy reads as zeros past the row)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float n[8], d[8], g[8];
      norm(j, n);
      unpack8(dy[j], d);
      keep_packed(w[j]);
      unpack8(w[j], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        aw[j][e] = fmaf(d[e], n[e], aw[j][e]);
        ab[j][e] += d[e];
        const float c = d[e] * g[e];
        s[0] += c;
        s[1] = fmaf(c, n[e], s[1]);
      }
    }
    if (!p.dx) continue;
    row_sum<2, 1>(s, nullptr);
    const float m0 = s[0] * inv, m1 = s[1] * inv;
    const Window dx = row_of(p.dx, row, p.cols);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float n[8], d[8], g[8];
      norm(j, n);
      keep_packed(dy[j]);
      unpack8(dy[j], d);
      keep_packed(w[j]);
      unpack8(w[j], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = r * (fmaf(d[e], g[e], -m0) - n[e] * m1);
      window_store(dx, 16u * (t + 64 * j), pack8(d));
    }
  }
  if (!p.part) return;
  // the block's four waves add their sums: 2 to 0 and 3 to 1, then 1 to 0
  auto give = [&](int to) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const float(&a)[8] = h < 2 ? aw[j] : ab[j];
        sums[(to * 4 * V + 4 * j + h) * 64 + t] =
            make_float4(a[4 * (h & 1)], a[4 * (h & 1) + 1], a[4 * (h & 1) + 2], a[4 * (h & 1) + 3]);
      }
  };
  auto take = [&](int from) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        float(&a)[8] = h < 2 ? aw[j] : ab[j];
        const float4 b = sums[(from * 4 * V + 4 * j + h) * 64 + t];
        a[4 * (h & 1)] += b.x;
        a[4 * (h & 1) + 1] += b.y;
        a[4 * (h & 1) + 2] += b.z;
        a[4 * (h & 1) + 3] += b.w;
      }
  };
  if (wid >= 2) give(wid - 2);
  __syncthreads();
  if (wid < 2) take(wid);
  __syncthreads();
  if (wid == 1) give(0);
  __syncthreads();
  if (wid == 0) {
    take(0);
    write_sums<V>(p, t, 64, aw, ab);
  }
}

// Sums over the block of N values a thread (2 or 4): a wave's lanes halve them by exchanges until a lane holds
// one of them, red[wave][N] joins the waves, which are added in order. One barrier: the caller gives a call
// other LDS than the one before.
template <int N>
__device__ __forceinline__ void block_sums(float (&v)[N], float* red) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, waves = blockDim.x >> 6;
  int n = N, off = 32;
#pragma unroll
  for (; n > 1; n /= 2, off /= 2) {
    const bool up = lane & off;
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float give = up ? v[i] : v[i + n / 2], keep = up ? v[i + n / 2] : v[i];
      v[i] = keep + __shfl_xor(give, off, 64);
    }
  }
#pragma unroll
  for (; off >= 1; off /= 2) v[0] += __shfl_xor(v[0], off, 64);
  constexpr int kLanes = 64 / N;  // that hold the same sum
  if ((lane & (kLanes - 1)) == 0) red[wid * N + lane / kLanes] = v[0];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = red[i];
  for (int w = 1; w < waves; ++w)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += red[w * N + i];
}

// A row of the block: thread t's pieces t, t + blockDim.x.
template <int V>
__device__ __forceinline__ void load_block_row(Window w, uint4 (&v)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = window_load(w, 16u * (threadIdx.x + blockDim.x * j));
}

// R rows of the backward's inputs, x or its checkpoint.
template <int V, int R, bool CKPT>
struct BwdRows {
  uint4 dy[R][V], x[CKPT ? 1 : R][V];
  uint2 q[CKPT ? R : 1][V];
  uint32_t e[CKPT ? R : 1][V];
  float mean[R], rstd[R];

  // rows past the tensor's read as zeros
  __device__ __forceinline__ void load(const LayerNorm& p, int64_t r0) {
    const int blocks = (p.cols + 31) >> 5;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t row = r0 + i;
      const bool in = row < p.rows;
      load_block_row<V>(row_of(in ? p.dy : nullptr, row, p.cols), dy[i]);
      if constexpr (CKPT) {
        const Window wq = row_of(in ? p.x8 : nullptr, row, p.cols, 1);
        const Window we = row_of(in ? p.x8_e : nullptr, row, blocks, 1);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const uint32_t k = threadIdx.x + blockDim.x * j;
          q[i][j] = window_load8(wq, 8 * k);
          e[i][j] = window_load1(we, k >> 2);
        }
      } else {
        load_block_row<V>(row_of(in ? p.x : nullptr, row, p.cols), x[i]);
      }
      mean[i] = in ? p.mean[row] : 0.0f;
      rstd[i] = in ? p.rstd[row] : 0.0f;
    }
  }

  __device__ __forceinline__ void norm(int i, int j, float (&n)[8]) {
    if constexpr (CKPT) {
      const float step = mxi8_step(e[i][j]);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        n[k] = (code_f32(k < 4 ? q[i][j].x : q[i][j].y, k & 3) * step - mean[i]) * rstd[i];
    } else {
      keep_packed(x[i][j]);
      unpack8(x[i][j], n);
#pragma unroll
      for (int k = 0; k < 8; ++k) n[k] = (n[k] - mean[i]) * rstd[i];
    }
  }
};

// Wider rows: a block of ceil(cols / 512) waves a row (V 1; V 2 from 8,200 columns on), so that a thread keeps 16 sums
// a piece and the card 10 or 16 waves a CU. Either R 2 rows between two barriers, or (AHEAD, more than 2,560
// columns, where one block has a CU) a row, with the next one's loads under its reductions. Bound by memory (6
// bytes an element, 5.03 from a checkpoint, and 8 bytes a column and block of partials): with the kernel that
// adds those [18494, 2560] 56.8 us, from a checkpoint 55.7 (AHEAD 61 and 68), [3001, 4104] 26.5 (two rows 29.2),
// [4096, 8192] 48 (two rows 52), [3000, 16384] 77 (72 from a checkpoint).
template <int V, int R, bool AHEAD, bool CKPT>
__global__ __launch_bounds__(1024) void layer_norm_bwd_block_kernel(LayerNorm p) {
  __shared__ float red[2][16 * 2 * R];
  const int t = threadIdx.x;
  const float inv = 1.0f / (float)p.cols;
  uint4 w[V];
  load_block_row<V>(row_of(p.w, 0, p.cols), w);
  float aw[V][8], ab[V][8];
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) aw[j][e] = ab[j][e] = 0.0f;
  const int64_t stride = (int64_t)gridDim.x * R;
  BwdRows<V, R, CKPT> in;
  if (AHEAD) in.load(p, (int64_t)blockIdx.x * R);
  int odd = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * R; r0 < p.rows; r0 += stride) {
    if (!AHEAD) in.load(p, r0);
    float s[2 * R], n[R][V][8], c[R][V][8];  // sums of c, c n (dy reads as zeros past the row)
    float r[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      r[i] = in.rstd[i];
      s[2 * i] = s[2 * i + 1] = 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float g[8];
        in.norm(i, j, n[i][j]);
        unpack8(in.dy[i][j], c[i][j]);
        keep_packed(w[j]);
        unpack8(w[j], g);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          aw[j][e] = fmaf(c[i][j][e], n[i][j][e], aw[j][e]);
          ab[j][e] += c[i][j][e];
          c[i][j][e] *= g[e];
          s[2 * i] += c[i][j][e];
          s[2 * i + 1] = fmaf(c[i][j][e], n[i][j][e], s[2 * i + 1]);
        }
      }
    }
    if (AHEAD) in.load(p, r0 + stride);
    if (!p.dx) continue;
    block_sums<2 * R>(s, red[odd]);
    odd ^= 1;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float m0 = s[2 * i] * inv, m1 = s[2 * i + 1] * inv;
      const Window dx = row_of(r0 + i < p.rows ? p.dx : nullptr, r0 + i, p.cols);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float d[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = r[i] * (fmaf(n[i][j][e], -m1, c[i][j][e]) - m0);
        window_store(dx, 16u * (t + blockDim.x * j), pack8(d));
      }
    }
  }
  if (!p.part) return;
  write_sums<V>(p, t, blockDim.x, aw, ab);
}

// The weight's and the bias' gradients from the blocks' partials: blockIdx.y 0 and 1. A block takes 16
// columns (a 64-byte segment of each partial row), its 64 thread groups every 64th row.
constexpr int kRedNT = 1024, kRedCols = 16, kRedGroups = kRedNT / kRedCols;
__global__ __launch_bounds__(kRedNT) void layer_norm_wgrad_kernel(const float* __restrict__ part,
                                                                  int nblocks, int cols,
                                                                  uint16_t* __restrict__ dw,
                                                                  uint16_t* __restrict__ db) {
  __shared__ float red[kRedGroups][kRedCols + 1];
  uint16_t* out = blockIdx.y == 0 ? dw : db;
  if (!out) return;
  const int lc = threadIdx.x % kRedCols, g = threadIdx.x / kRedCols;
  const int col = blockIdx.x * kRedCols + lc;
  float a = 0.0f;
  if (col < cols)
    for (int b = g; b < nblocks; b += kRedGroups)
      a += part[((int64_t)b * 2 + blockIdx.y) * cols + col];
  red[g][lc] = a;
  __syncthreads();
#pragma unroll
  for (int s = kRedGroups / 2; s >= 1; s >>= 1) {
    if (g < s) red[g][lc] += red[g + s][lc];
    __syncthreads();
  }
  if (g == 0 && col < cols) out[col] = (uint16_t)f32_to_bf16_bits(red[0][lc]);
}

int64_t row_blocks(int64_t rows, int per, int64_t most) {
  return std::max<int64_t>(1, std::min((rows + per - 1) / per, most));
}

// The backward's rows and blocks: as many as are resident at once, as each adds a partial row.
constexpr int kWaveCols = 1536, kTwoRowCols = 2560, kOnePieceCols = 8192;
int bwd_threads(int64_t cols) {
  if (cols <= kWaveCols) return 256;
  const int64_t per_wave = cols <= kOnePieceCols ? 512 : 1024;
  return 64 * (int)((cols + per_wave - 1) / per_wave);
}
int64_t bwd_blocks(int64_t rows, int64_t cols) {
  if (cols <= kWaveCols) return row_blocks(rows, 4, 512);
  return cols <= kTwoRowCols ? row_blocks(rows, 2, 512) : row_blocks(rows, 1, 256);
}

int check_common(const char* who, int64_t rows, int64_t cols, const void* x8, const void* x8_e) {
  BF8_CHECK(rows >= 0 && cols > 0, "%s: bad shape", who);
  BF8_CHECK(cols % 8 == 0 && cols <= kMaxCols, "%s: need cols %% 8 == 0 and cols <= %d (got %lld)",
            who, kMaxCols, (long long)cols);
  BF8_CHECK((x8 == nullptr) == (x8_e == nullptr) && ((uintptr_t)x8 & 7) == 0,
            "%s: x8 (8-byte aligned) and its block exponents go together", who);
  return BF8_OK;
}

}  // namespace
}  // namespace bf8

using namespace bf8;

extern "C" {

int bf8_layernorm_bf16(const void* x, int64_t rows, int64_t cols, const void* weight, const void* bias,
                       float eps, void* y, float* mean, float* rstd, int8_t* x8, uint8_t* x8_exp,
                       void* stream) {
  const char* who = "bf8_layernorm_bf16";
  if (const int rc = check_common(who, rows, cols, x8, x8_exp)) return rc;
  if (rows == 0) return BF8_OK;
  BF8_CHECK(x && weight && y, "%s: NULL pointer", who);
  BF8_CHECK((mean == nullptr) == (rstd == nullptr), "%s: mean and rstd go together", who);
  BF8_CHECK((((uintptr_t)x | (uintptr_t)weight | (uintptr_t)bias | (uintptr_t)y) & 15) == 0,
            "%s: every tensor must be 16-byte aligned", who);
  LayerNorm p{};
  p.x = (const uint16_t*)x; p.w = (const uint16_t*)weight; p.b = (const uint16_t*)bias;
  p.rows = rows; p.cols = (int)cols; p.eps = eps;
  p.y = (uint16_t*)y; p.mean = mean; p.rstd = rstd; p.x8 = x8; p.x8_e = x8_exp;
  const int pieces = (int)cols / 8;
#define BF8_LN_FWD(V, W)                                                                               \
  {                                                                                                    \
    const dim3 grid((unsigned)row_blocks(rows, W == 1 ? 4 : 1, kMaxFwdBlocks));                        \
    if (x8)                                                                                            \
      hipLaunchKernelGGL((layer_norm_kernel<V, W, true>), grid, dim3(block_threads(W)), 0,             \
                         as_stream(stream), p);                                                        \
    else                                                                                               \
      hipLaunchKernelGGL((layer_norm_kernel<V, W, false>), grid, dim3(block_threads(W)), 0,            \
                         as_stream(stream), p);                                                        \
  }
  // (each is run by the rows it is the narrowest for; few rows of 1,544 .. 2,560 columns: five waves each)
  if (pieces <= 64) BF8_LN_FWD(1, 1)
  else if (pieces <= 128) BF8_LN_FWD(2, 1)
  else if (pieces <= 192) BF8_LN_FWD(3, 1)
  else if (pieces <= 320 && rows <= kFewRows) BF8_LN_FWD(1, 5)
  else if (pieces <= 256) BF8_LN_FWD(4, 1)
  else if (pieces <= 320) BF8_LN_FWD(5, 1)
  else if (pieces <= 384) BF8_LN_FWD(2, 3)
  else if (pieces <= 576) BF8_LN_FWD(3, 3)
  else if (pieces <= 768) BF8_LN_FWD(3, 4)
  else if (pieces <= 1024) BF8_LN_FWD(4, 4)
  else if (pieces <= 1536) BF8_LN_FWD(3, 8)
  else BF8_LN_FWD(4, 8)
#undef BF8_LN_FWD
  return launch_status("layer_norm_kernel");
}

size_t bf8_layernorm_bwd_workspace(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0 || cols > kMaxCols) return 0;
  return (size_t)bwd_blocks(rows, cols) * 2 * (size_t)cols * sizeof(float);
}

int bf8_layernorm_bwd_bf16(const void* x, const int8_t* x8, const uint8_t* x8_exp, const void* dy,
                           int64_t rows, int64_t cols, const void* weight, const float* mean,
                           const float* rstd, void* dx, void* dweight, void* dbias, void* ws,
                           size_t ws_bytes, void* stream) {
  const char* who = "bf8_layernorm_bwd_bf16";
  if (const int rc = check_common(who, rows, cols, x8, x8_exp)) return rc;
  BF8_CHECK(rows > 0, "%s: no rows", who);
  BF8_CHECK((x == nullptr) != (x8 == nullptr), "%s: give x or its checkpoint x8", who);
  BF8_CHECK(dy && weight && mean && rstd, "%s: NULL pointer", who);
  BF8_CHECK(dx || dweight || dbias, "%s: nothing requested", who);
  BF8_CHECK((((uintptr_t)x | (uintptr_t)dy | (uintptr_t)weight | (uintptr_t)dx) & 15) == 0,
            "%s: every tensor must be 16-byte aligned", who);
  const bool wgrad = dweight || dbias;
  BF8_CHECK(!wgrad || (ws && ((uintptr_t)ws & 15) == 0 &&
                       ws_bytes >= bf8_layernorm_bwd_workspace(rows, cols)),
            "%s: workspace of %zu bytes, need %zu, 16-byte aligned", who, ws_bytes,
            bf8_layernorm_bwd_workspace(rows, cols));
  LayerNorm p{};
  p.x = (const uint16_t*)x; p.w = (const uint16_t*)weight;
  p.rows = rows; p.cols = (int)cols;
  p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd);
  p.x8 = const_cast<int8_t*>(x8); p.x8_e = const_cast<uint8_t*>(x8_exp);
  p.dy = (const uint16_t*)dy; p.dx = (uint16_t*)dx;
  p.part = wgrad ? (float*)ws : nullptr;
  const int64_t nb = bwd_blocks(rows, cols);
  const dim3 grid((unsigned)nb), block(bwd_threads(cols));
  const hipStream_t st = as_stream(stream);
#define BF8_LN_BWD(KERNEL, ...)                                                   \
  {                                                                               \
    if (x8)                                                                       \
      hipLaunchKernelGGL((KERNEL<__VA_ARGS__, true>), grid, block, 0, st, p);     \
    else                                                                          \
      hipLaunchKernelGGL((KERNEL<__VA_ARGS__, false>), grid, block, 0, st, p);    \
  }
  if (cols <= 512) BF8_LN_BWD(layer_norm_bwd_kernel, 1)
  else if (cols <= 1024) BF8_LN_BWD(layer_norm_bwd_kernel, 2)
  else if (cols <= kWaveCols) BF8_LN_BWD(layer_norm_bwd_kernel, 3)
  else if (cols <= kTwoRowCols) BF8_LN_BWD(layer_norm_bwd_block_kernel, 1, 2, false)
  else if (cols <= kOnePieceCols) BF8_LN_BWD(layer_norm_bwd_block_kernel, 1, 1, true)
  else BF8_LN_BWD(layer_norm_bwd_block_kernel, 2, 1, true)
#undef BF8_LN_BWD
  const int rc = launch_status("layer_norm_bwd_kernel");
  if (rc != BF8_OK || !wgrad) return rc;
  hipLaunchKernelGGL(layer_norm_wgrad_kernel, dim3((unsigned)((cols + kRedCols - 1) / kRedCols), 2),
                     dim3(kRedNT), 0, as_stream(stream), (const float*)ws, (int)nb, (int)cols,
                     (uint16_t*)dweight, (uint16_t*)dbias);
  return launch_status("layer_norm_wgrad_kernel");
}

}  // extern "C"
