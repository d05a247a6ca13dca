// A linear layer of int8 weights on a few tokens (decoding), for gfx950: each token's quantization and the
// product as one kernel where the tokens' codes fit the LDS, else the quantizer and the GEMM.
//
//   s_t = max(max |x_t|, 2^-40) / 127, q_t the codes of x_t (int8.hpp)
//   y[t, n] = s_t w_scale[n] sum_k q_t[k] W[n, k] + bias[n],  the sum exact in int32
// and the gate/up projection with the gated GELU (gelu.hpp): W's rows n and I + n give g and u of
//   h[t, n] = bf16(bf16(gelu(bf16 g)) bf16 u)
#include <hip/hip_runtime.h>

#include <algorithm>

#include "gelu.hpp"
#include "gemm_kernel.hpp"
#include "int8.hpp"

namespace bf8 {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int kWaves = 8, kNT = 64 * kWaves;
constexpr int kStep = 64;        // K bytes of an MFMA
// Steps of weights a wave has in flight (gated: of gate and up rows each; with five of them the registers leave one
// workgroup a CU, 20 us at I 10240, K 2560 instead of 15).
constexpr int kAheadLinear = 5, kAheadGated = 3;
constexpr int kMaxTokens = 32;
// LDS bytes of the tokens' codes up to which one kernel is the faster: linear 32 x 2560 x 2560 10.1 us (quantizer and
// GEMM 13.8), 8 x 2560 x 10240 16.0 (20.5), but 16 x 10240 x 6144 27.3 (23.1); gated 12 x 10240 x 10240 40 (52), but
// 32 x 20480 x 4096 37 (31).
constexpr int64_t kMaxCodes = 81920, kMaxCodesGated = 122880;

struct Tokens {
  const uint16_t* x;  // [M, K]
  const int8_t* W;
  int64_t ldw;
  const float* w_scale;
  int M, N, K, steps;  // N: output channels (gated: I)
  int split;   // waves that share a group of 16 output channels, each a range of K (a power of two)
  int groups;
  const uint16_t* bias;
  void* C;
  int64_t ldc;
};

// Bound by the weights' bytes; for few of them by latency. A wave takes 16 output channels (rows of W) and a
// range of K: its lanes load W in the MFMA's operand layout straight from memory (lane l: row l mod 16,
// bytes 16 (l / 16) .. +15 of each 64), kAhead steps in flight, the first of them while the tokens are
// quantized. The codes lie in LDS as [step][quarter of 64 bytes][token][16 bytes], so that the 64 lanes of
// an operand read 1 KB side by side (lanes of absent tokens read the last one's, and are not stored).
// Bytes past K of a row are whatever follows it: the codes there are zeros. One token of 20480 x 2560 12.5 us (4.2
// TB/s of weights), sixteen 15.4, of 2048 x 2560 5.3 and 7.1, of 2560 x 10240 10.3 (quantizer and GEMM: 20.0, 21.7,
// 12.6, 14.0, 19.4); gated 20480 x 2560 15.4 and 20.5 (26.0, 27.0). Codes written by a kernel of their own and read
// from the L2 beside the weights took 19 us for 16 x 2560 x 10240 and 23 for 16 x 20480 x 2560.
template <int TG, bool F32, bool GATED = false>
__global__ __launch_bounds__(kNT, 4) void int8_tokens_kernel(Tokens p) {
  constexpr int kAhead = GATED ? kAheadGated : kAheadLinear;
  extern __shared__ uint8_t codes[];
  __shared__ float scales[kMaxTokens];
  __shared__ uint32_t top[kWaves];
  __shared__ v4i parts[kWaves][TG][64];
  constexpr int NH = GATED ? 2 : 1;  // rows of W an output channel takes
  __shared__ __attribute__((aligned(16))) uint16_t gelu[GATED ? kGeluABytes / 2 : 8];
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per_block = kWaves / p.split, sub = wid & (p.split - 1), slot = wid / p.split;
  const int s0 = p.steps * sub / p.split, s1 = p.steps * (sub + 1) / p.split;

  auto load = [&](int group, int step, v4i (&w)[NH][kAhead]) __attribute__((always_inline)) {
    const int r0 = group * 16;
    const int rows = min(16, p.N - r0);  // (a group past the last: no bytes)
    const uint32_t o = (uint32_t)((lane & 15) * p.ldw) + 16 * (lane >> 4);
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      const Window win = window(p.W + (int64_t)(h * p.N + r0) * p.ldw,
                                rows > 0 ? (uint32_t)((rows - 1) * p.ldw + p.K) : 0u);
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        w[h][i] = __builtin_bit_cast(v4i, window_load(win, step + i < s1 ? o + kStep * (step + i) : kPastEnd));
    }
  };
  // the group's output channels of this lane: 4 (lane / 16) .. +3; their scales and biases come with the
  // group's first weights
  const int stride = gridDim.x * per_block;
  float4 ws[NH];
#pragma unroll
  for (int h = 0; h < NH; ++h) ws[h] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  uint2 wb = make_uint2(0u, 0u);
  auto load_channels = [&](int group) __attribute__((always_inline)) {
    const int n = group * 16 + 4 * (lane >> 4);
    if (sub != 0 || n >= p.N) return;
#pragma unroll
    for (int h = 0; h < NH; ++h) ws[h] = *reinterpret_cast<const float4*>(p.w_scale + h * p.N + n);
    if (!GATED && p.bias) wb = *reinterpret_cast<const uint2*>(p.bias + n);
  };
  // the tokens' codes: `share` waves a token, the row's 16-byte vectors spread over their lanes; the next
  // token's first kHold of a lane are loaded before this one's maximum is known. More waves share a long row: one
  // each takes 8 x 2560 x 10240 from 16 to 19 us
  constexpr int kHold = 5;
  const int nvec = p.K >> 3;
  int share = p.M >= 5 ? 1 : p.M >= 3 ? 2 : p.M == 2 ? 4 : 8;
  while (share < kWaves && nvec > 64 * kHold * share) share *= 2;
  const int first = 64 * (wid & (share - 1)) + lane;
  auto row = [&](int t) __attribute__((always_inline)) {
    return window(p.x + (int64_t)t * p.K, t < p.M ? 2u * p.K : 0u);
  };
  uint4 next_x[kHold];
#pragma unroll
  for (int j = 0; j < kHold; ++j) next_x[j] = window_load(row(wid / share), 16u * (first + 64 * share * j));
  v4i w[NH][kAhead];
  int base = blockIdx.x * per_block;
  load(base + slot, s0, w);
  load_channels(base + slot);
  if constexpr (GATED) load_gelu_tables<kNT>(gelu, nullptr);
  for (int t0 = 0; t0 < p.M; t0 += kWaves / share) {
    const int t = t0 + wid / share;
    const Window xr = row(t);
    uint4 held[kHold];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < kHold; ++j) {
      held[j] = next_x[j];
      if (t0 + kWaves / share < p.M)
        next_x[j] = window_load(row(t + kWaves / share), 16u * (first + 64 * share * j));
    }
#pragma unroll
    for (int j = 0; j < kHold; ++j) m = max(m, absmax16(held[j]));
    for (int v = first + 64 * share * kHold; v < nvec; v += 64 * share)
      m = max(m, absmax16(window_load(xr, 16u * v)));
    m = wave_max_u32(m);
    if (share > 1) {
      if (lane == 0) top[wid] = m;
      __syncthreads();
      for (int i = 0; i < share; ++i) m = max(m, top[wid / share * share + i]);
      __syncthreads();
    }
    if (t >= p.M) continue;
    const Int8Scale s = int8_scale(m << 16);
    if (first == 0) scales[t] = s.scale;
    auto put = [&](int v, uint4 x) __attribute__((always_inline)) {
      *reinterpret_cast<uint2*>(codes + ((v >> 1) * p.M + t) * 16 + 8 * (v & 1)) = int8_codes8(x, s.mult);
    };
#pragma unroll
    for (int j = 0; j < kHold; ++j) {
      const int v = first + 64 * share * j;
      if (v < nvec) put(v, held[j]);
    }
    for (int v = first + 64 * share * kHold; v < nvec; v += 64 * share) put(v, window_load(xr, 16u * v));
  }
  // the last step's chunks past K
  for (int i = threadIdx.x; i < (p.steps * 4 - p.K / 16) * p.M; i += kNT)
    reinterpret_cast<uint4*>(codes)[p.K / 16 * p.M + i] = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();

  const int tok = lane & 15;
  uint32_t at[TG];
#pragma unroll
  for (int g = 0; g < TG; ++g) at[g] = 16 * ((lane >> 4) * p.M + min(16 * g + tok, p.M - 1));
  const uint32_t per_step = 64 * p.M;
  for (; base < p.groups; base += stride) {
    v4i acc[NH][TG];
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int g = 0; g < TG; ++g) acc[h][g] = v4i{0, 0, 0, 0};
    for (int step = s0; step < s1; step += kAhead) {
      v4i next[NH][kAhead];
      if (step + kAhead < s1)
        load(base + slot, step + kAhead, next);
      else
        load(base + stride + slot, s0, next);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int st = min(step + i, p.steps - 1);  // (steps past the range: weights of zeros)
#pragma unroll
        for (int g = 0; g < TG; ++g) {
          const v4i b = *reinterpret_cast<const v4i*>(codes + st * per_step + at[g]);
#pragma unroll
          for (int h = 0; h < NH; ++h)
            acc[h][g] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[h][i], b, acc[h][g], 0, 0, 0);
        }
      }
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int i = 0; i < kAhead; ++i) w[h][i] = next[h][i];
    }
    float4 f[NH];
#pragma unroll
    for (int h = 0; h < NH; ++h) f[h] = ws[h];
    const uint2 bb = wb;
    load_channels(base + stride + slot);
    if (p.split > 1) {
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        __syncthreads();  // what was there has been read
#pragma unroll
        for (int g = 0; g < TG; ++g) parts[wid][g][lane] = acc[h][g];
        __syncthreads();
        if (sub == 0)
          for (int i = 1; i < p.split; ++i)
#pragma unroll
            for (int g = 0; g < TG; ++g) acc[h][g] += parts[wid + i][g][lane];
      }
      if (sub != 0) continue;
    }
    // acc[g][r]: token 16 g + lane mod 16, channel 4 (lane / 16) + r of the group
    const int n = (base + slot) * 16 + 4 * (lane >> 4);
    if (n >= p.N) continue;
    const float b[4] = {bf16_lo(bb.x), bf16_hi(bb.x), bf16_lo(bb.y), bf16_hi(bb.y)};
#pragma unroll
    for (int g = 0; g < TG; ++g) {
      const int t = 16 * g + tok;
      if (t >= p.M) continue;
      const float s = scales[t];
      float y[NH][4];
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        y[h][0] = __builtin_fmaf((float)acc[h][g][0], s * f[h].x, b[0]);
        y[h][1] = __builtin_fmaf((float)acc[h][g][1], s * f[h].y, b[1]);
        y[h][2] = __builtin_fmaf((float)acc[h][g][2], s * f[h].z, b[2]);
        y[h][3] = __builtin_fmaf((float)acc[h][g][3], s * f[h].w, b[3]);
      }
      if constexpr (F32) {
        *reinterpret_cast<float4*>((float*)p.C + t * p.ldc + n) = make_float4(y[0][0], y[0][1], y[0][2], y[0][3]);
        continue;
      }
      uint2 o = make_uint2(pack_bf16x2(y[0][0], y[0][1]), pack_bf16x2(y[0][2], y[0][3]));
      if constexpr (GATED) {
        uint32_t outside = 0;
        const uint32_t i0 = gelu_index2(o.x, outside), i1 = gelu_index2(o.y, outside);
        uint32_t a[4] = {gelu[i0 & 0xFFFFu], gelu[i0 >> 16], gelu[i1 & 0xFFFFu], gelu[i1 >> 16]};
        if (outside) {
          a[0] = gelu_finish(o.x, a[0]);
          a[1] = gelu_finish(o.x >> 16, a[1]);
          a[2] = gelu_finish(o.y, a[2]);
          a[3] = gelu_finish(o.y >> 16, a[3]);
        }
        o.x = geglu_mul_bf16x2(a[0] | a[1] << 16, pack_bf16x2(y[1][0], y[1][1]));
        o.y = geglu_mul_bf16x2(a[2] | a[3] << 16, pack_bf16x2(y[1][2], y[1][3]));
      }
      *reinterpret_cast<uint2*>((uint16_t*)p.C + t * p.ldc + n) = o;
    }
  }
}

int64_t token_steps(int64_t K) { return (K + kStep - 1) / kStep; }
int64_t code_bytes(int64_t M, int64_t K) { return M * token_steps(K) * kStep; }
bool one_kernel(int64_t M, int64_t K, bool gated) {
  return M <= kMaxTokens && code_bytes(M, K) <= (gated ? kMaxCodesGated : kMaxCodes);
}
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// LDS bytes of a workgroup: the codes, the waves' sums, the table.
int64_t lds_bytes(const Tokens& p, bool gated) {
  return code_bytes(p.M, p.K) + (p.M <= 16 ? 8352 : 16544) + (gated ? kGeluABytes : 0);
}
// Two workgroups a CU; one where the LDS holds no second and a long row's quantization takes more than the evener
// share of the groups gives back (8 x 10240 x 10240 30.9 us, by twice the workgroups 37.6; 32 x 10240 x 2560 17.0
// and 15.4).
int64_t max_blocks(const Tokens& p, bool gated) {
  return 2 * lds_bytes(p, gated) > 160 * 1024 && p.K >= 4096 ? kNumCus : 2 * kNumCus;
}

// What a split of K over `split` waves costs beside what all of them do (us): on the busiest CU its one or two
// workgroups, which quantize the tokens each, and the sets of groups that they take one after another, by their
// weights' bytes and by the batches of loads a wave waits for. Least squares over 218 shapes (M 1 .. 32, N 512 ..
// 32768, I 1024 .. 14336, K 320 .. 3584) at every split: its picks lose 0.8% on average and 8% at worst; with as many
// waves as there are steps for, 10% and 62% (1 x 8192 x 1024: 6.2 us, in four 5.3; 16 x 20480 x 2560: 14.9, in four
// 15.1, in two 17.5).
double split_cost(const Tokens& p, int split, bool gated) {
  const int64_t sets = cdiv(p.groups, kWaves / split), blocks = std::min(sets, max_blocks(p, gated));
  const bool two = blocks > kNumCus;
  const int64_t on_cu = cdiv(sets, blocks) + (two ? cdiv(sets - kNumCus, blocks) : 0);
  const int64_t batches = cdiv(cdiv(p.steps, split), gated ? kAheadGated : kAheadLinear);
  const double rows = 16.0 * (kWaves / split) * (gated ? 2 : 1);
  return (two ? 2 : 1) * (0.78 + 6.12e-5 * p.M * p.K) + on_cu * (1.385e-5 * rows * p.K + (two ? 0.257 : 0.514) * batches);
}

Tokens tokens(const void* x, const int8_t* W, int64_t ldw, const float* w_scale, int64_t M, int64_t N, int64_t K,
              const void* bias, void* C, int64_t ldc, bool gated) {
  Tokens p{};
  p.x = (const uint16_t*)x; p.W = W; p.ldw = ldw; p.w_scale = w_scale;
  p.M = (int)M; p.N = (int)N; p.K = (int)K; p.steps = (int)token_steps(K);
  p.bias = (const uint16_t*)bias; p.C = C; p.ldc = ldc;
  p.groups = (int)((N + 15) / 16);
  p.split = 1;
  double best = 0;
  for (int split = 1; split <= kWaves && split <= p.steps; split *= 2) {
    const double c = split_cost(p, split, gated);
    if (split == 1 || c < best) {
      best = c;
      p.split = split;
    }
  }
  return p;
}
dim3 token_grid(const Tokens& p, bool gated) {
  return dim3((unsigned)std::min<int64_t>(cdiv(p.groups, kWaves / p.split), max_blocks(p, gated)));
}
size_t align256(size_t b) { return (b + 255) / 256 * 256; }

}  // namespace
}  // namespace bf8

using namespace bf8;

extern "C" {

size_t bf8_linear_int8_workspace(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || one_kernel(M, K, false)) return 0;
  return align256((size_t)M * K) + align256((size_t)M * 4) + bf8_gemm_int8_workspace(M, N, K);
}

int bf8_linear_int8(const void* x, const int8_t* W, int64_t ldw, const float* w_scale, int64_t M,
                    int64_t N, int64_t K, const void* bias, void* C, int out_dtype, int64_t ldc,
                    void* ws, size_t ws_bytes, void* stream) {
  const char* who = "bf8_linear_int8";
  BF8_CHECK(out_dtype == BF8_OUT_BF16 || out_dtype == BF8_OUT_F32, "%s: bad out_dtype", who);
  BF8_CHECK(M >= 0 && N >= 0 && K >= 0, "%s: negative shape", who);
  BF8_CHECK(K % 16 == 0 && K <= 32768, "%s: need K %% 16 == 0 and K <= 32768 (got %lld)", who,
            (long long)K);
  BF8_CHECK(N % 8 == 0 && ldc >= N && ldc % 4 == 0, "%s: need N %% 8 == 0, ldc >= N, ldc %% 4 == 0",
            who);
  BF8_CHECK((((uintptr_t)x | (uintptr_t)W | (uintptr_t)w_scale | (uintptr_t)C) & 15) == 0 &&
                ((uintptr_t)bias & 7) == 0,
            "%s: x, W, w_scale and C must be 16-byte, bias 8-byte aligned", who);
  BF8_CHECK(ldw % 16 == 0 && ldw >= K && N * ldw < (1LL << 31) && M * K < (1LL << 31),
            "%s: need a row stride >= K in multiples of 16, operands below 2 GiB", who);
  if (M == 0 || N == 0) return BF8_OK;
  BF8_CHECK(K > 0, "%s: K == 0 is not supported", who);
  BF8_CHECK(x && W && w_scale && C, "%s: NULL pointer", who);
  if (!one_kernel(M, K, false)) {
    const size_t head = align256((size_t)M * K) + align256((size_t)M * 4);
    BF8_CHECK(ws && ((uintptr_t)ws & 255) == 0 && ws_bytes >= head,
              "%s: workspace needs %zu bytes, 256-byte aligned (got %zu)", who,
              bf8_linear_int8_workspace(M, N, K), ws_bytes);
    int8_t* q = (int8_t*)ws;
    float* s = (float*)(q + align256((size_t)M * K));
    const int rc = bf8_quantize_int8_bf16(x, M, K, q, s, nullptr, nullptr, nullptr, 0, stream);
    if (rc != BF8_OK) return rc;
    return bf8_gemm_int8(q, K, s, W, ldw, w_scale, M, N, K, bias, C, out_dtype, ldc,
                         ws_bytes > head ? q + head : nullptr, ws_bytes - head, stream);
  }
  const Tokens p = tokens(x, W, ldw, w_scale, M, N, K, bias, C, ldc, false);
  const bool f32 = out_dtype == BF8_OUT_F32;
  const auto kernel = M <= 16 ? (f32 ? int8_tokens_kernel<1, true> : int8_tokens_kernel<1, false>)
                              : (f32 ? int8_tokens_kernel<2, true> : int8_tokens_kernel<2, false>);
  hipLaunchKernelGGL(kernel, token_grid(p, false), dim3(kNT), (size_t)p.M * p.steps * kStep, as_stream(stream), p);
  return launch_status("int8_tokens_kernel");
}

size_t bf8_linear_geglu_int8_workspace(int64_t M, int64_t I, int64_t K) {
  if (M <= 0 || I <= 0 || K <= 0 || one_kernel(M, K, true)) return 0;
  return align256((size_t)M * K) + align256((size_t)M * 4);
}

int bf8_linear_geglu_int8(const void* x, const int8_t* W, int64_t ldw, const float* w_scale, int64_t M, int64_t I,
                          int64_t K, void* H, void* ws, size_t ws_bytes, void* stream) {
  const char* who = "bf8_linear_geglu_int8";
  BF8_CHECK(M >= 0 && I >= 0 && K >= 0, "%s: negative shape", who);
  BF8_CHECK(I % 128 == 0 && K % 16 == 0 && K <= 32768,
            "%s: need I %% 128 == 0, K %% 16 == 0 and K <= 32768 (got %lld, %lld)", who, (long long)I,
            (long long)K);
  BF8_CHECK((((uintptr_t)x | (uintptr_t)W | (uintptr_t)w_scale | (uintptr_t)H) & 15) == 0,
            "%s: x, W, w_scale and H must be 16-byte aligned", who);
  BF8_CHECK(ldw % 16 == 0 && ldw >= K && 2 * I * ldw < (1LL << 31) && M * K < (1LL << 31),
            "%s: need a row stride >= K in multiples of 16, operands below 2 GiB", who);
  if (M == 0 || I == 0) return BF8_OK;
  BF8_CHECK(K > 0, "%s: K == 0 is not supported", who);
  BF8_CHECK(x && W && w_scale && H, "%s: NULL pointer", who);
  if (!one_kernel(M, K, true)) {
    const size_t need = bf8_linear_geglu_int8_workspace(M, I, K);
    BF8_CHECK(ws && ((uintptr_t)ws & 255) == 0 && ws_bytes >= need,
              "%s: workspace needs %zu bytes, 256-byte aligned (got %zu)", who, need, ws_bytes);
    int8_t* q = (int8_t*)ws;
    float* s = (float*)(q + align256((size_t)M * K));
    if (const int rc = bf8_quantize_int8_bf16(x, M, K, q, s, nullptr, nullptr, nullptr, 0, stream)) return rc;
    return bf8_gemm_geglu_int8(q, K, s, W, ldw, w_scale, M, I, K, H, nullptr, nullptr, stream);
  }
  const Tokens p = tokens(x, W, ldw, w_scale, M, I, K, nullptr, H, I, true);
  const auto kernel = M <= 16 ? int8_tokens_kernel<1, false, true> : int8_tokens_kernel<2, false, true>;
  hipLaunchKernelGGL(kernel, token_grid(p, true), dim3(kNT), (size_t)p.M * p.steps * kStep, as_stream(stream), p);
  return launch_status("int8_tokens_kernel(gated)");
}

}  // extern "C"
