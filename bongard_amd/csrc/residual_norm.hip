// The norms on either side of a residual connection as one kernel for gfx950, and its backward.
//
// A T5Gemma2 layer norms a block's output, adds it to the residual stream and norms the sum for
// the next block (HF modeling_t5gemma2.py:468-495: post_self_attn_layernorm, the addition,
// pre_feedforward_layernorm; again around the MLP). Per row, in fp32 from bf16 inputs:
//   r1  = 1 / sqrt(mean(h^2) + eps),        n1 = h r1
//   out = bf16(a res + g n1 (z + post))     a: residual scale, g: gate (1 without one), z: 1 where
//   r2  = 1 / sqrt(mean(out^2) + eps),      the weights are zero-centred, else 0
//   y   = bf16(n2 (z + pre)),               n2 = out r2
// out is rounded once (the unfused chain rounds the normed h as well) and y is the norm of the
// rounded out: the stream as it is stored, which the backward reads. Backward of dout and dy:
//   d    = dout + r2 (c - n2 mean(c n2)),   c = dy (z + pre)
//   dres = bf16(a d)
//   dh   = bf16(r1 (e - n1 mean(e n1))),    e = g d (z + post)
//   dpre = bf16(P), P = sum over rows of dy n2;   dpost = bf16(g S), dgate = bf16((z + post) S),
//   S = sum over rows of d n1
// Sums over rows go through per-block partials added in a fixed order (deterministic).
//
// Both are bound by memory: 8 bytes an element forward and 12 backward, one read and one write of
// each tensor. A row is held in registers across its two sums, up to 2,560 columns by one wave (no
// barrier), wider ones by a block. Accesses go through a buffer descriptor of the row, which
// drops what lies past its end without a branch: behind a branch each load was waited for before
// the next. The backward also holds the column sums of its block (16 registers per 8 columns); with the
// weights read from LDS where they are used and bf16 pairs unpacked anew in each pass it takes 251
// registers at 2,560 columns, two waves a SIMD (held as floats: 471, one wave). Rows past 8,192 columns
// spill: the backward's block of 16 waves has 128 registers a lane and keeps 35 more in scratch.
// Measured, 18,494 x 2,560: forward 74 us, 5.1 TB/s; backward with the weights' gradients 122 us,
// 4.7 TB/s (140 with the weights in registers). 3,001 x 2,560: 12.3 and 27 us (13.7 and 42).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.hpp"

namespace bf8 {
namespace {

constexpr int kMaxCols = 16384;
constexpr int64_t kMaxFwdBlocks = 2048;  // (1,024 blocks are level with them)
// The backward's blocks: those resident at once (two a CU, or one of 16 waves), as each adds a
// partial row to the weights' sums. 768 instead of 512: 135 us for 124 at 18,494 x 2,560; 256: 118
// for 122 there but 58 for 48 at 4,096 x 4,096. 512 instead of 256 of the wide ones: 120 us for 107
// (4,096 x 8,192).
constexpr int64_t max_bwd_blocks(int64_t cols) { return cols <= 4096 ? 512 : 256; }

struct ResNorm {
  const uint16_t *h, *res, *post, *pre, *gate;  // backward: res is the forward's out
  int64_t rows;
  int cols;
  float scale, eps, z;
  uint16_t *out, *y;
  const uint16_t *dout, *dy;
  uint16_t *dh, *dres;
  float* part;  // [blocks][2][cols]: P, S
};

// Threads of a block whose rows take WPR waves each: four rows of one wave, or one row of more.
constexpr int block_threads(int wpr) { return 64 * (wpr < 4 ? 4 : wpr); }

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

// Row `row` of a [rows, cols] tensor: past its end, and anywhere in one that is NULL, it reads as zeros.
__device__ __forceinline__ Window row_of(const uint16_t* p, int64_t row, int cols) {
  return window(p + row * cols, p ? 2u * cols : 0u);
}

// The thread's V pieces of a row lie 64 WPR pieces of 16 bytes apart.
template <int V, int WPR>
__device__ __forceinline__ void load_row(Window w, int t, uint4 (&v)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = window_load(w, 16u * (t + 64 * WPR * j));
}

// From here on the compiler knows nothing of v, so that it unpacks it again where it is used next
// and does not hold two floats for each of its dwords.
__device__ __forceinline__ void keep_packed(uint4& v) {
  asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w));
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

__device__ __forceinline__ float rstd_of(float ss, int cols, float eps) {
  return __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, (float)cols) + eps));
}

template <int V, int WPR>
__global__ __launch_bounds__(block_threads(WPR)) void residual_norm_kernel(ResNorm p) {
  __shared__ float red[2][1][WPR];
  const int t = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t first = WPR == 1 ? (int64_t)blockIdx.x * 4 + wid : blockIdx.x;
  const int64_t stride = WPR == 1 ? (int64_t)gridDim.x * 4 : gridDim.x;
  const float one = p.gate ? 0.0f : 1.0f;  // the gate that is not there
  uint4 post[V], pre[V], gate[V];
  load_row<V, WPR>(row_of(p.post, 0, p.cols), t, post);
  load_row<V, WPR>(row_of(p.pre, 0, p.cols), t, pre);
  load_row<V, WPR>(row_of(p.gate, 0, p.cols), t, gate);
  for (int64_t row = first; row < p.rows; row += stride) {
    uint4 h[V], r[V];
    load_row<V, WPR>(row_of(p.h, row, p.cols), t, h);
    load_row<V, WPR>(row_of(p.res, row, p.cols), t, r);
    const Window out = row_of(p.out, row, p.cols), y = row_of(p.y, row, p.cols);
    float ss[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float x[8];
      unpack8(h[j], x);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss[0] = fmaf(x[e], x[e], ss[0]);
    }
    row_sum<1, WPR>(ss, red[0]);
    const float r1 = rstd_of(ss[0], p.cols, p.eps);
    ss[0] = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float x[8], w[8], s[8], o[8], g[8];
      keep_packed(h[j]);
      keep_packed(post[j]);
      keep_packed(gate[j]);
      unpack8(h[j], x);
      unpack8(post[j], w);
      unpack8(r[j], s);
      unpack8(gate[j], g);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        o[e] = fmaf(p.scale, s[e], ((x[e] * r1) * (p.z + w[e])) * (one + g[e]));
      h[j] = pack8(o);
      unpack8(h[j], o);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss[0] = fmaf(o[e], o[e], ss[0]);
      window_store(out, 16u * (t + 64 * WPR * j), h[j]);
    }
    row_sum<1, WPR>(ss, red[1]);
    const float r2 = rstd_of(ss[0], p.cols, p.eps);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float o[8], w[8];
      keep_packed(h[j]);
      keep_packed(pre[j]);
      unpack8(h[j], o);
      unpack8(pre[j], w);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = (o[e] * r2) * (p.z + w[e]);
      window_store(y, 16u * (t + 64 * WPR * j), pack8(o));
    }
  }
}

// Whether the backward keeps the weights in LDS (6 bytes a column, 48 KB at most).
constexpr bool weights_in_lds(int v, int wpr) { return v * wpr <= 16; }
constexpr size_t bwd_lds(int v, int wpr, int64_t cols) {
  const size_t w = weights_in_lds(v, wpr) ? (size_t)cols * 3 * sizeof(uint16_t) : 0;
  const size_t sums = wpr == 1 ? (size_t)2 * v * 64 * 16 * sizeof(float) : 0;
  return w > sums ? w : sums;
}

template <int V, int WPR>
__global__ __launch_bounds__(block_threads(WPR)) void residual_norm_bwd_kernel(ResNorm p) {
  __shared__ float red[2][3][WPR];
  constexpr bool kLds = weights_in_lds(V, WPR);
  extern __shared__ uint4 dyn[];  // (kLds) post, pre and gate; then (WPR 1) two waves' column sums
  const int t = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nvec = p.cols >> 3;
  const int64_t first = WPR == 1 ? (int64_t)blockIdx.x * 4 + wid : blockIdx.x;
  const int64_t stride = WPR == 1 ? (int64_t)gridDim.x * 4 : gridDim.x;
  const float inv = 1.0f / (float)p.cols;
  const float one = p.gate ? 0.0f : 1.0f;  // the gate that is not there
  const Window weights[3] = {row_of(p.post, 0, p.cols), row_of(p.pre, 0, p.cols),
                             row_of(p.gate, 0, p.cols)};
  if constexpr (kLds) {
#pragma unroll
    for (int k = 0; k < 3; ++k)
      for (int i = threadIdx.x; i < nvec; i += block_threads(WPR))
        dyn[k * nvec + i] = window_load(weights[k], 16u * i);
    __syncthreads();
  }
  // piece j of weight k, read where it is used: its floats, or all the pieces of a wide row, would
  // not fit beside the sums
  auto weight = [&](int k, int j, float (&f)[8]) __attribute__((always_inline)) {
    const int i = t + 64 * WPR * j;
    if constexpr (kLds)
      unpack8(dyn[k * nvec + (i < nvec ? i : 0)], f);
    else
      unpack8(window_load(weights[k], 16u * i), f);
  };
  float accp[V][8], accs[V][8];
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) accp[j][e] = accs[j][e] = 0.0f;
  for (int64_t row = first; row < p.rows; row += stride) {
    uint4 h[V], o[V], dy[V], dout[V];
    load_row<V, WPR>(row_of(p.h, row, p.cols), t, h);
    load_row<V, WPR>(row_of(p.res, row, p.cols), t, o);
    load_row<V, WPR>(row_of(p.dy, row, p.cols), t, dy);
    load_row<V, WPR>(row_of(p.dout, row, p.cols), t, dout);
    const Window dres = row_of(p.dres, row, p.cols), dh = row_of(p.dh, row, p.cols);
    float s[3] = {0.0f, 0.0f, 0.0f};  // sums of h^2, out^2, dy (z + pre) out
#pragma unroll
    for (int j = 0; j < V; ++j) {
      asm volatile("" ::: "memory");
      float x[8], n[8], g[8], w[8];
      unpack8(h[j], x);
      unpack8(o[j], n);
      unpack8(dy[j], g);
      weight(1, j, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[0] = fmaf(x[e], x[e], s[0]);
        s[1] = fmaf(n[e], n[e], s[1]);
        s[2] = fmaf(g[e] * (p.z + w[e]), n[e], s[2]);
      }
    }
    row_sum<3, WPR>(s, red[0]);
    const float r1 = rstd_of(s[0], p.cols, p.eps), r2 = rstd_of(s[1], p.cols, p.eps);
    const float m2 = s[2] * r2 * inv;  // mean(c n2)
    float q[1] = {0.0f};               // sum of e h
    float dd[V][8];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      asm volatile("" ::: "memory");
      keep_packed(h[j]);
      keep_packed(o[j]);
      keep_packed(dy[j]);
      float x[8], n[8], g[8], w[8], u[8], b[8], ga[8];
      unpack8(h[j], x);
      unpack8(o[j], n);
      unpack8(dy[j], g);
      unpack8(dout[j], u);
      weight(0, j, b);
      weight(1, j, w);
      weight(2, j, ga);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float n2 = n[e] * r2;
        accp[j][e] = fmaf(g[e], n2, accp[j][e]);
        const float d = u[e] + r2 * (g[e] * (p.z + w[e]) - n2 * m2);
        accs[j][e] = fmaf(d, x[e] * r1, accs[j][e]);
        u[e] = p.scale * d;
        dd[j][e] = (d * (p.z + b[e])) * (one + ga[e]);
        q[0] = fmaf(dd[j][e], x[e], q[0]);
      }
      window_store(dres, 16u * (t + 64 * WPR * j), pack8(u));
    }
    row_sum<1, WPR>(q, red[1]);
    const float m1 = q[0] * r1 * inv;  // mean(e n1)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      keep_packed(h[j]);
      float x[8];
      unpack8(h[j], x);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = r1 * (dd[j][e] - (x[e] * r1) * m1);
      window_store(dh, 16u * (t + 64 * WPR * j), pack8(x));
    }
  }
  if (!p.part) return;
  auto write_sums = [&]() __attribute__((always_inline)) {
    float* dst = p.part + (int64_t)blockIdx.x * 2 * p.cols;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = t + 64 * WPR * j;
      if (i >= nvec) continue;
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const float(&a)[8] = h < 2 ? accp[j] : accs[j];
        *reinterpret_cast<float4*>(dst + (h < 2 ? 0 : p.cols) + 8 * i + 4 * (h & 1)) =
            make_float4(a[4 * (h & 1)], a[4 * (h & 1) + 1], a[4 * (h & 1) + 2], a[4 * (h & 1) + 3]);
      }
    }
  };
  if constexpr (WPR > 1) {
    write_sums();
  } else {
    // the block's four waves, done with the weights, add their sums: 2 to 0 and 3 to 1, then 1 to 0
    float4* sums = reinterpret_cast<float4*>(dyn);
    auto give = [&](int to) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const float(&a)[8] = h < 2 ? accp[j] : accs[j];
          sums[(to * 4 * V + 4 * j + h) * 64 + t] =
              make_float4(a[4 * (h & 1)], a[4 * (h & 1) + 1], a[4 * (h & 1) + 2], a[4 * (h & 1) + 3]);
        }
    };
    auto take = [&](int from) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          float(&a)[8] = h < 2 ? accp[j] : accs[j];
          const float4 b = sums[(from * 4 * V + 4 * j + h) * 64 + t];
          a[4 * (h & 1)] += b.x;
          a[4 * (h & 1) + 1] += b.y;
          a[4 * (h & 1) + 2] += b.z;
          a[4 * (h & 1) + 3] += b.w;
        }
    };
    __syncthreads();
    if (wid >= 2) give(wid - 2);
    __syncthreads();
    if (wid < 2) take(wid);
    __syncthreads();
    if (wid == 1) give(0);
    __syncthreads();
    if (wid == 0) {
      take(0);
      write_sums();
    }
  }
}

// The weights' gradients from the blocks' partials: blockIdx.y 0 for P, 1 for S. A block takes 16
// columns (a 64-byte segment of each partial row), its 64 thread groups every 64th row.
constexpr int kRedNT = 1024, kRedCols = 16, kRedGroups = kRedNT / kRedCols;
__global__ __launch_bounds__(kRedNT) void residual_norm_wgrad_kernel(
    const float* __restrict__ part, int nblocks, int cols, const uint16_t* __restrict__ post,
    const uint16_t* __restrict__ gate, float z, uint16_t* __restrict__ dpost,
    uint16_t* __restrict__ dpre, uint16_t* __restrict__ dgate) {
  __shared__ float red[kRedGroups][kRedCols + 1];
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
  if (g != 0 || col >= cols) return;
  const float v = red[0][lc];
  if (blockIdx.y == 0) {
    if (dpre) dpre[col] = (uint16_t)f32_to_bf16_bits(v);
  } else {
    if (dpost) dpost[col] = (uint16_t)f32_to_bf16_bits(gate ? v * bf16_lo(gate[col]) : v);
    if (dgate) dgate[col] = (uint16_t)f32_to_bf16_bits(v * (z + bf16_lo(post[col])));
  }
}

// Rows up to 2,560 wide take a wave each, wider ones a block of four waves or sixteen.
constexpr int kWaveCols = 2560;
int64_t row_blocks(int64_t rows, int cols, int64_t most) {
  const int64_t b = cols <= kWaveCols ? (rows + 3) / 4 : rows;
  return std::max<int64_t>(1, std::min(b, most));
}

int check_common(const char* who, int64_t rows, int64_t cols) {
  BF8_CHECK(rows >= 0 && cols > 0, "%s: bad shape", who);
  BF8_CHECK(cols % 8 == 0 && cols <= kMaxCols, "%s: need cols %% 8 == 0 and cols <= %d (got %lld)",
            who, kMaxCols, (long long)cols);
  return BF8_OK;
}

#define BF8_BY_WIDTH(LAUNCH)                                 \
  if (cols <= kWaveCols) {                                   \
    switch ((int)((cols / 8 + 63) / 64)) {                   \
      case 1: LAUNCH(1, 1); break;                           \
      case 2: LAUNCH(2, 1); break;                           \
      case 3: LAUNCH(3, 1); break;                           \
      case 4: LAUNCH(4, 1); break;                           \
      default: LAUNCH(5, 1); break;                          \
    }                                                        \
  } else {                                                   \
    if (cols <= 4096) {                                      \
      LAUNCH(2, 4);                                          \
    } else if (cols <= 8192) {                               \
      LAUNCH(1, 16);                                         \
    } else {                                                 \
      LAUNCH(2, 16);                                         \
    }                                                        \
  }

}  // namespace
}  // namespace bf8

using namespace bf8;

extern "C" {

int bf8_rmsnorm_residual_bf16(const void* h, const void* residual, int64_t rows, int64_t cols,
                              const void* post, const void* pre, const void* gate,
                              float residual_scale, float eps, int zero_centered, void* out,
                              void* y, void* stream) {
  const char* who = "bf8_rmsnorm_residual_bf16";
  if (const int rc = check_common(who, rows, cols)) return rc;
  if (rows == 0) return BF8_OK;
  BF8_CHECK(h && residual && post && pre && out && y, "%s: NULL pointer", who);
  BF8_CHECK((((uintptr_t)h | (uintptr_t)residual | (uintptr_t)post | (uintptr_t)pre |
              (uintptr_t)gate | (uintptr_t)out | (uintptr_t)y) & 15) == 0,
            "%s: every tensor must be 16-byte aligned", who);
  ResNorm p{};
  p.h = (const uint16_t*)h; p.res = (const uint16_t*)residual;
  p.post = (const uint16_t*)post; p.pre = (const uint16_t*)pre; p.gate = (const uint16_t*)gate;
  p.rows = rows; p.cols = (int)cols;
  p.scale = residual_scale; p.eps = eps; p.z = zero_centered ? 1.0f : 0.0f;
  p.out = (uint16_t*)out; p.y = (uint16_t*)y;
  const dim3 grid((unsigned)row_blocks(rows, (int)cols, kMaxFwdBlocks));
#define BF8_RN_FWD(V, W) \
  hipLaunchKernelGGL((residual_norm_kernel<V, W>), grid, dim3(block_threads(W)), 0,     \
                     as_stream(stream), p)
  BF8_BY_WIDTH(BF8_RN_FWD)
#undef BF8_RN_FWD
  return launch_status("residual_norm_kernel");
}

size_t bf8_rmsnorm_residual_bwd_workspace(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0 || cols > kMaxCols) return 0;
  return (size_t)row_blocks(rows, (int)cols, max_bwd_blocks(cols)) * 2 * (size_t)cols * sizeof(float);
}

int bf8_rmsnorm_residual_bwd_bf16(const void* h, const void* out, const void* dout, const void* dy,
                                  int64_t rows, int64_t cols, const void* post, const void* pre,
                                  const void* gate, float residual_scale, float eps,
                                  int zero_centered, void* dh, void* dresidual, void* dpost,
                                  void* dpre, void* dgate, void* ws, size_t ws_bytes,
                                  void* stream) {
  const char* who = "bf8_rmsnorm_residual_bwd_bf16";
  if (const int rc = check_common(who, rows, cols)) return rc;
  BF8_CHECK(rows > 0, "%s: no rows", who);
  BF8_CHECK(h && out && post && pre && (dout || dy), "%s: NULL pointer", who);
  BF8_CHECK(dh || dresidual || dpost || dpre || dgate, "%s: nothing requested", who);
  BF8_CHECK(!dgate || gate, "%s: dgate without a gate", who);
  BF8_CHECK((((uintptr_t)h | (uintptr_t)out | (uintptr_t)dout | (uintptr_t)dy | (uintptr_t)post |
              (uintptr_t)pre | (uintptr_t)gate | (uintptr_t)dh | (uintptr_t)dresidual) & 15) == 0,
            "%s: every tensor must be 16-byte aligned", who);
  const bool wgrad = dpost || dpre || dgate;
  BF8_CHECK(!wgrad || (ws && ((uintptr_t)ws & 15) == 0 &&
                       ws_bytes >= bf8_rmsnorm_residual_bwd_workspace(rows, cols)),
            "%s: workspace of %zu bytes, need %zu, 16-byte aligned", who, ws_bytes,
            bf8_rmsnorm_residual_bwd_workspace(rows, cols));
  ResNorm p{};
  p.h = (const uint16_t*)h; p.res = (const uint16_t*)out;
  p.dout = (const uint16_t*)dout; p.dy = (const uint16_t*)dy;
  p.post = (const uint16_t*)post; p.pre = (const uint16_t*)pre; p.gate = (const uint16_t*)gate;
  p.rows = rows; p.cols = (int)cols;
  p.scale = residual_scale; p.eps = eps; p.z = zero_centered ? 1.0f : 0.0f;
  p.dh = (uint16_t*)dh; p.dres = (uint16_t*)dresidual;
  p.part = wgrad ? (float*)ws : nullptr;
  const int64_t nb = row_blocks(rows, (int)cols, max_bwd_blocks(cols));
  const dim3 grid((unsigned)nb);
#define BF8_RN_BWD(V, W)                                                                      \
  hipLaunchKernelGGL((residual_norm_bwd_kernel<V, W>), grid, dim3(block_threads(W)), bwd_lds(V, W, cols), \
                     as_stream(stream), p)
  BF8_BY_WIDTH(BF8_RN_BWD)
#undef BF8_RN_BWD
  const int rc = launch_status("residual_norm_bwd_kernel");
  if (rc != BF8_OK || !wgrad) return rc;
  hipLaunchKernelGGL(residual_norm_wgrad_kernel,
                     dim3((unsigned)((cols + kRedCols - 1) / kRedCols), 2), dim3(kRedNT), 0,
                     as_stream(stream), (const float*)ws, (int)nb, (int)cols, p.post, p.gate, p.z,
                     (uint16_t*)dpost, (uint16_t*)dpre, (uint16_t*)dgate);
  return launch_status("residual_norm_wgrad_kernel");
}

}  // extern "C"
