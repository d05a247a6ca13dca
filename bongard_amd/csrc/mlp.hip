// The gated GELU(tanh) between the MLP's gate/up and down projections as elementwise
// kernels: its forward on given pre-activations, and its backward.
//
// Forward (bongard/te_linear.py:103): h = bf16(bf16(gelu_tanh(g)) * u) on bf16 g, u.
// Autograd of that bf16 chain gives, per element:
//   a   = bf16(gelu_tanh(g))                 (the forward's activation)
//   d_a = bf16(dh * u)                       (mul backward, grad wrt a)
//   d_u = bf16(dh * a)                       (mul backward, grad wrt u)
//   d_g = bf16(d_a * F(g))                   (gelu backward, fp32 factor F of g)
// a and F come from the tables of gelu.hpp, so every value is bit-identical to torch's CPU
// chain. Each kernel is one streaming pass that also writes per-block amax partials of its
// output (|H| or |dGU|), from which the following e4m3 / e5m2 cast derives its scale.
#include <hip/hip_runtime.h>

#include <cmath>

#include "common.hpp"
#include "gelu.hpp"
#include "int8.hpp"

namespace bf8 {
namespace {

constexpr int kNT = 256;
// Every block copies the gelu tables (34 KB) into LDS first, so the streaming grids stay
// at a few blocks per CU.
constexpr int64_t kMaxBlocks = 1024;

int64_t bwd_blocks(int64_t M, int64_t I) {
  const int64_t vec = M * I / 8;
  int64_t b = (vec + kNT - 1) / kNT;
  if (b < 1) b = 1;
  return b < kMaxBlocks ? b : kMaxBlocks;
}


// H for 8 elements (4 packed pairs of g, u), with the table reads issued together.
__device__ __forceinline__ uint4 geglu_fwd8(uint4 g, uint4 u, const uint16_t* ta) {
  const uint32_t gw[4] = {g.x, g.y, g.z, g.w}, uw[4] = {u.x, u.y, u.z, u.w};
  uint32_t outside = 0, ia[4], va[8], h[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) ia[w] = gelu_index2(gw[w], outside);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    va[2 * w] = ta[ia[w] & 0xFFFFu];
    va[2 * w + 1] = ta[ia[w] >> 16];
  }
  if (__builtin_expect(__any(outside != 0), 0)) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      va[2 * w] = gelu_finish(gw[w], va[2 * w]);
      va[2 * w + 1] = gelu_finish(gw[w] >> 16, va[2 * w + 1]);
    }
  }
#pragma unroll
  for (int w = 0; w < 4; ++w) h[w] = geglu_mul_bf16x2(va[2 * w] | (va[2 * w + 1] << 16), uw[w]);
  return make_uint4(h[0], h[1], h[2], h[3]);
}

// H [M, I] = gelu(g) * u from GU [M, 2I] (gate | up), and per-block amax keys of |H|.
__global__ __launch_bounds__(kNT) void geglu_fwd_kernel(const uint16_t* __restrict__ GU,
                                                        int64_t M, int64_t I,
                                                        uint16_t* __restrict__ H,
                                                        uint32_t* __restrict__ partials) {
  __shared__ __attribute__((aligned(16))) uint16_t ta[kGeluABytes / 2];
  load_gelu_tables<kNT>(ta, nullptr);
  __syncthreads();
  const int64_t per_row = I / 8;
  const int64_t nvec = M * per_row;
  const int64_t stride = (int64_t)gridDim.x * kNT;
  uint32_t m = 0;
  for (int64_t v = (int64_t)blockIdx.x * kNT + threadIdx.x; v < nvec; v += stride) {
    const int64_t row = v / per_row;
    const int64_t col = (v - row * per_row) * 8;
    const uint4 g = *reinterpret_cast<const uint4*>(GU + row * 2 * I + col);
    const uint4 u = *reinterpret_cast<const uint4*>(GU + row * 2 * I + I + col);
    const uint4 h = geglu_fwd8(g, u, ta);
    const uint32_t k = pk_max_u16(pk_max_u16(h.x & 0x7FFF7FFFu, h.y & 0x7FFF7FFFu),
                                  pk_max_u16(h.z & 0x7FFF7FFFu, h.w & 0x7FFF7FFFu));
    m = max(m, max(k << 16, k & 0xFFFF0000u));
    *reinterpret_cast<uint4*>(H + row * I + col) = h;
  }
  m = block_max_u32<kNT>(m);
  if (threadIdx.x == 0) partials[blockIdx.x] = m;
}

// The same, and GU's checkpoint: blocks of 32 codes along its rows (gu8 [M, 2I], gu8_e [M, 2I / 32],
// I % 32 == 0), a group of four lanes a block of gates and one of ups. Bound by memory (4 B read, 4.06 written an
// element of H): [4096, 10240] 64.6 us (5.2 TB/s), [3001, 10240] 41.6.
__global__ __launch_bounds__(kNT) void geglu_fwd_mxi8_kernel(const uint16_t* __restrict__ GU, int64_t M,
                                                             int64_t I, uint16_t* __restrict__ H,
                                                             int8_t* __restrict__ gu8,
                                                             uint8_t* __restrict__ gu8_e) {
  __shared__ __attribute__((aligned(16))) uint16_t ta[kGeluABytes / 2];
  load_gelu_tables<kNT>(ta, nullptr);
  __syncthreads();
  const int64_t per_row = I / 8;
  const int64_t nvec = M * per_row;
  const int64_t stride = (int64_t)gridDim.x * kNT;
  for (int64_t v = (int64_t)blockIdx.x * kNT + threadIdx.x; v < nvec; v += stride) {
    const int64_t row = v / per_row;
    const int64_t col = (v - row * per_row) * 8;
    const int64_t at = row * 2 * I + col;
    const uint4 g = *reinterpret_cast<const uint4*>(GU + at);
    const uint4 u = *reinterpret_cast<const uint4*>(GU + at + I);
    *reinterpret_cast<uint4*>(H + row * I + col) = geglu_fwd8(g, u, ta);
    const uint32_t eg = mxi8_exponent(quad_max(absmax16(g)));
    const uint32_t eu = mxi8_exponent(quad_max(absmax16(u)));
    *reinterpret_cast<uint2*>(gu8 + at) = mxi8_codes8(g, eg);
    *reinterpret_cast<uint2*>(gu8 + at + I) = mxi8_codes8(u, eu);
    if ((v & 3) == 0) {
      gu8_e[at >> 5] = (uint8_t)eg;
      gu8_e[(at + I) >> 5] = (uint8_t)eu;
    }
  }
}

// geglu_bwd_kernel from the checkpoint: the same chain on the bf16 values that it holds. Bound by memory: 4.06
// bytes an element of H read, 4 written; [4096, 10240] 69 us, [3001, 10240] 50.
__global__ __launch_bounds__(kNT) void geglu_bwd_mxi8_kernel(const uint16_t* __restrict__ dH,
                                                             const int8_t* __restrict__ gu8,
                                                             const uint8_t* __restrict__ gu8_e,
                                                             int64_t M, int64_t I,
                                                             uint16_t* __restrict__ dGU) {
  __shared__ __attribute__((aligned(16))) uint16_t ta[kGeluABytes / 2];
  __shared__ __attribute__((aligned(16))) uint32_t tf[kGeluFBytes / 4];
  load_gelu_tables<kNT>(ta, tf);
  __syncthreads();
  const int64_t per_row = I / 8;
  const int64_t nvec = M * per_row;
  const int64_t stride = (int64_t)gridDim.x * kNT;
  for (int64_t v = (int64_t)blockIdx.x * kNT + threadIdx.x; v < nvec; v += stride) {
    const int64_t row = v / per_row;
    const int64_t col = (v - row * per_row) * 8;
    const int64_t at = row * 2 * I + col;
    const uint4 dh = *reinterpret_cast<const uint4*>(dH + row * I + col);
    const uint4 g = mxi8_values8(*reinterpret_cast<const uint2*>(gu8 + at), mxi8_step(gu8_e[at >> 5]));
    const uint4 u = mxi8_values8(*reinterpret_cast<const uint2*>(gu8 + at + I),
                                 mxi8_step(gu8_e[(at + I) >> 5]));
    const uint32_t dhw[4] = {dh.x, dh.y, dh.z, dh.w};
    const uint32_t gw[4] = {g.x, g.y, g.z, g.w};
    const uint32_t uw[4] = {u.x, u.y, u.z, u.w};
    uint32_t dg[4], du[4], m = 0;
    geglu_bwd8<true>(dhw, gw, uw, ta, tf, dg, du, m);
    *reinterpret_cast<uint4*>(dGU + at) = make_uint4(dg[0], dg[1], dg[2], dg[3]);
    *reinterpret_cast<uint4*>(dGU + at + I) = make_uint4(du[0], du[1], du[2], du[3]);
  }
}

// The same where dGU's int8 codes come next: a block takes a strip of rows by 512 columns of H, a wave eight rows
// at a time (two passes of four), so that the maxima of d_g and d_u fall to it on the way and the pass over dGU
// that would find them (4 bytes an element of H) is saved: [4096, 10240] with both copies of the codes 157 us,
// by the kernel above and the ordinary quantizer 168. Alone it is the slower one (73 us there, 10.8 against
// 5.3 at 64 rows): fewer loads in flight a wave, 2 MB of maxima, 48 bytes a lane in scratch.
constexpr int kBwdCols = 512, kBwdRows = 4;
__global__ __launch_bounds__(kNT, 4) void geglu_bwd_mxi8_maxima_kernel(
    const uint16_t* __restrict__ dH, const int8_t* __restrict__ gu8, const uint8_t* __restrict__ gu8_e, int64_t I,
    uint16_t* __restrict__ dGU, Int8Maxima p) {
  __shared__ __attribute__((aligned(16))) uint16_t ta[kGeluABytes / 2];
  __shared__ __attribute__((aligned(16))) uint32_t tf[kGeluFBytes / 4];
  load_gelu_tables<kNT>(ta, tf);
  __syncthreads();
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = p.row_tiles / 2, tc = blockIdx.x % tiles;
  const int64_t ts = blockIdx.x / tiles, r0 = ts * p.strip;
  const int64_t c = (int64_t)kBwdCols * tc + 8 * lane;
  const int left = (int)min((int64_t)p.strip, p.rows - r0);
  const uint32_t ld = (uint32_t)I, cc = (uint32_t)c;
  // the lane's offsets in a row of dH, of the codes, of their exponents and of dGU (c >= I: past its end)
  const uint32_t od = c < I ? 2 * cc : kPastEnd, oq = c < I ? cc : kPastEnd, oe = c < I ? cc >> 5 : kPastEnd;
  uint4 kg = make_uint4(0u, 0u, 0u, 0u), ku = kg;
  for (int r = 8 * wid; r < left; r += 8 * (kNT / 64)) {
    const int64_t at = r0 + r;
    Int8Rows mg, mu;
#pragma unroll
    for (int h = 0; h < 8; h += kBwdRows) {
      uint4 d[kBwdRows];
      uint2 g[kBwdRows], u[kBwdRows];
      uint32_t eg[kBwdRows], eu[kBwdRows];
#pragma unroll
      for (int i = 0; i < kBwdRows; ++i) {
        const int64_t row = at + h + i;
        const uint32_t n = r + h + i < left ? ld : 0u;  // rows past the tensor's read as zeros
        d[i] = window_load(window(dH + row * I, 2 * n), od);
        const Window wq = window(gu8 + row * 2 * I, 2 * n), we = window(gu8_e + row * (I / 16), n / 16);
        g[i] = window_load8(wq, oq);
        u[i] = window_load8(wq, oq + ld);
        eg[i] = window_load1(we, oe);
        eu[i] = window_load1(we, oe + ld / 32);
      }
#pragma unroll
      for (int i = 0; i < kBwdRows; ++i) {
        const uint4 gv = mxi8_values8(g[i], mxi8_step(eg[i])), uv = mxi8_values8(u[i], mxi8_step(eu[i]));
        const uint32_t dhw[4] = {d[i].x, d[i].y, d[i].z, d[i].w};
        const uint32_t gw[4] = {gv.x, gv.y, gv.z, gv.w};
        const uint32_t uw[4] = {uv.x, uv.y, uv.z, uv.w};
        uint32_t dg[4], du[4], m = 0;
        geglu_bwd8<true>(dhw, gw, uw, ta, tf, dg, du, m);
        const uint4 vg = make_uint4(dg[0], dg[1], dg[2], dg[3]), vu = make_uint4(du[0], du[1], du[2], du[3]);
        const Window wo = window(dGU + (at + h + i) * 2 * I, r + h + i < left ? 4 * ld : 0u);
        window_store(wo, od, vg);
        window_store(wo, od + 2 * ld, vu);
        mg.add(h + i, vg, kg);  // (rows past the tensor's: zeros, dH having read as zeros)
        mu.add(h + i, vu, ku);
        __builtin_amdgcn_sched_barrier(0);  // row by row: interleaved, the rows' values spill
      }
    }
    mg.store(p, at, tc, lane);
    mu.store(p, at, tiles + tc, lane);
  }
  __syncthreads();
  uint4(*red)[64] = reinterpret_cast<uint4(*)[64]>(tf);  // the tables have been read
  int8_column_maxima<kNT / 64>(p, red, kg, ts, c < I ? c : p.cols, wid, lane);
  __syncthreads();
  int8_column_maxima<kNT / 64>(p, red, ku, ts, c < I ? I + c : p.cols, wid, lane);
}

__global__ __launch_bounds__(kNT) void geglu_bwd_kernel(const uint16_t* __restrict__ dH,
                                                        const uint16_t* __restrict__ GU,
                                                        int64_t M, int64_t I,
                                                        uint16_t* __restrict__ dGU,
                                                        uint32_t* __restrict__ partials) {
  __shared__ __attribute__((aligned(16))) uint16_t ta[kGeluABytes / 2];
  __shared__ __attribute__((aligned(16))) uint32_t tf[kGeluFBytes / 4];
  load_gelu_tables<kNT>(ta, tf);
  __syncthreads();
  const int64_t per_row = I / 8;
  const int64_t nvec = M * per_row;
  const int64_t stride = (int64_t)gridDim.x * kNT;
  uint32_t m = 0;
  for (int64_t v = (int64_t)blockIdx.x * kNT + threadIdx.x; v < nvec; v += stride) {
    const int64_t row = v / per_row;
    const int64_t col = (v - row * per_row) * 8;
    const uint4 dh = *reinterpret_cast<const uint4*>(dH + row * I + col);
    const uint4 g = *reinterpret_cast<const uint4*>(GU + row * 2 * I + col);
    const uint4 u = *reinterpret_cast<const uint4*>(GU + row * 2 * I + I + col);
    const uint32_t dhw[4] = {dh.x, dh.y, dh.z, dh.w};
    const uint32_t gw[4] = {g.x, g.y, g.z, g.w};
    const uint32_t uw[4] = {u.x, u.y, u.z, u.w};
    uint32_t dg[4], du[4];
    geglu_bwd8(dhw, gw, uw, ta, tf, dg, du, m);
    *reinterpret_cast<uint4*>(dGU + row * 2 * I + col) = make_uint4(dg[0], dg[1], dg[2], dg[3]);
    *reinterpret_cast<uint4*>(dGU + row * 2 * I + I + col) = make_uint4(du[0], du[1], du[2], du[3]);
  }
  m = block_max_u32<kNT>(m);
  if (threadIdx.x == 0) partials[blockIdx.x] = m;
}

// The geglu backward fused with its delayed-scaling cast (for 'fp8_delayed', where dGU's
// scale is known before dGU exists): the same per-element chain as geglu_bwd_kernel, the
// bf16 d_g, d_u quantized at once with the role's delayed scale, written as fp8 rows
// [M, 2I] and/or transposed as fp8 [2I, M] (the wgrad layout), plus this step's amax
// partials of |dGU|. One 64-row x 64-column tile of I per wave: the wave streams it in
// 8-row pieces (dH, g, u: 16-byte loads, four pieces in flight), stages the fp8 d_g and
// d_u bytes in its own LDS regions and reads them back transposed (wave_transpose64_staged).
// Identical bytes to geglu_bwd_kernel followed by the delayed cast of its output.
constexpr int kTT = 64;
constexpr int kFusedWaves = kNT / 64;
constexpr int64_t kMaxFusedBlocks = 512;

int64_t fused_blocks(int64_t M, int64_t I) {
  const int64_t tiles = ((M + kTT - 1) / kTT) * (I / kTT);
  const int64_t blocks = (tiles + kFusedWaves - 1) / kFusedWaves;
  return blocks < 1 ? 1 : (blocks < kMaxFusedBlocks ? blocks : kMaxFusedBlocks);
}

template <int FMT>
__global__ __launch_bounds__(kNT) void geglu_bwd_delayed_kernel(
    const uint16_t* __restrict__ dH, const uint16_t* __restrict__ GU, int64_t M, int64_t I,
    float* __restrict__ state, int len, int pos, const uint32_t* __restrict__ prev,
    int64_t n_prev, float* __restrict__ meta_out, uint8_t* __restrict__ out,
    uint8_t* __restrict__ out_t, uint32_t* __restrict__ partials) {
  __shared__ uint32_t stage[kFusedWaves][2][kWaveTileDwords];
  __shared__ __attribute__((aligned(16))) uint16_t ta[kGeluABytes / 2];
  __shared__ __attribute__((aligned(16))) uint32_t tf[kGeluFBytes / 4];
  load_gelu_tables<kNT>(ta, tf);  // the scale step below synchronises the block
  const float scale =
      delayed_scale_block<kNT>(state, len, pos, prev, n_prev, Fp8Max<FMT>::value, meta_out,
                               blockIdx.x == 0);
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int64_t tiles_c = I / kTT;
  const int64_t ntiles = tiles_c * ((M + kTT - 1) / kTT);
  const int ch = lane & 7;  // 16-byte chunk of the piece's rows
  uint32_t* lg = stage[wid][0];
  uint32_t* lu = stage[wid][1];
  uint32_t m = 0;
  for (int64_t tile_id = (int64_t)blockIdx.x * kFusedWaves + wid; tile_id < ntiles;
       tile_id += (int64_t)gridDim.x * kFusedWaves) {
    const int64_t r0 = (tile_id / tiles_c) * kTT, c0 = (tile_id % tiles_c) * kTT;
    const int64_t c = c0 + 8 * ch;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint4 dh[4], g[4], u[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t r = r0 + 32 * half + 8 * k + (lane >> 3);
        dh[k] = g[k] = u[k] = make_uint4(0u, 0u, 0u, 0u);
        if (r < M) {
          dh[k] = *reinterpret_cast<const uint4*>(dH + r * I + c);
          g[k] = *reinterpret_cast<const uint4*>(GU + r * 2 * I + c);
          u[k] = *reinterpret_cast<const uint4*>(GU + r * 2 * I + I + c);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int lr = 32 * half + 8 * k + (lane >> 3);
        const int64_t r = r0 + lr;
        const uint32_t dhw[4] = {dh[k].x, dh[k].y, dh[k].z, dh[k].w};
        const uint32_t gw[4] = {g[k].x, g[k].y, g[k].z, g[k].w};
        const uint32_t uw[4] = {u[k].x, u[k].y, u[k].z, u[k].w};
        uint32_t dg[4], du[4];
        geglu_bwd8(dhw, gw, uw, ta, tf, dg, du, m);
        const uint2 qg = quant8_bf16<FMT>(make_uint4(dg[0], dg[1], dg[2], dg[3]), scale);
        const uint2 qu = quant8_bf16<FMT>(make_uint4(du[0], du[1], du[2], du[3]), scale);
        if (out && r < M) {
          *reinterpret_cast<uint2*>(out + r * 2 * I + c) = qg;
          *reinterpret_cast<uint2*>(out + r * 2 * I + I + c) = qu;
        }
        lg[lr * kWaveTilePitch + 2 * ch] = qg.x;
        lg[lr * kWaveTilePitch + 2 * ch + 1] = qg.y;
        lu[lr * kWaveTilePitch + 2 * ch] = qu.x;
        lu[lr * kWaveTilePitch + 2 * ch + 1] = qu.y;
      }
    }
    if (out_t) {
      const int64_t tc = r0 + (lane >> 4) * 16;  // column of out_t (a row of dGU)
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        uint4 tq[4];
        wave_transpose64_staged(which ? lu : lg, lane, tq);
        if (tc < M) {  // M % 16 == 0: whole 16-byte segments
#pragma unroll
          for (int cc = 0; cc < 4; ++cc) {
            const int64_t tr = (which ? I : 0) + c0 + 4 * (lane & 15) + cc;  // row of out_t
            *reinterpret_cast<uint4*>(out_t + tr * M + tc) = tq[cc];
          }
        }
      }
    }
  }
  m = block_max_u32<kNT>(m);
  if (threadIdx.x == 0) partials[blockIdx.x] = m;
}

// geglu_bwd_delayed_kernel without the transposed output (the K-major backward reads dGU
// as it is): a grid-stride stream over 8-element vectors of [M, I], kRowVecs per thread
// per pass with all their loads issued first, so a wave writes 512 contiguous fp8 bytes of
// d_g and of d_u per vector slot. Same chain, scale, bytes and partials count.
constexpr int kRowVecs = 4;

template <int FMT>
__global__ __launch_bounds__(kNT) void geglu_bwd_delayed_rows_kernel(
    const uint16_t* __restrict__ dH, const uint16_t* __restrict__ GU, int64_t M, int64_t I,
    float* __restrict__ state, int len, int pos, const uint32_t* __restrict__ prev,
    int64_t n_prev, float* __restrict__ meta_out, uint8_t* __restrict__ out,
    uint32_t* __restrict__ partials) {
  __shared__ __attribute__((aligned(16))) uint16_t ta[kGeluABytes / 2];
  __shared__ __attribute__((aligned(16))) uint32_t tf[kGeluFBytes / 4];
  load_gelu_tables<kNT>(ta, tf);  // the scale step below synchronises the block
  const float scale =
      delayed_scale_block<kNT>(state, len, pos, prev, n_prev, Fp8Max<FMT>::value, meta_out,
                               blockIdx.x == 0);
  const int64_t per_row = I / 8;
  const int64_t nvec = M * per_row;
  const int64_t pass = (int64_t)gridDim.x * kNT * kRowVecs;
  uint32_t m = 0;
  for (int64_t v0 = (int64_t)blockIdx.x * kNT * kRowVecs + threadIdx.x; v0 < nvec; v0 += pass) {
    uint4 dh[kRowVecs], g[kRowVecs], u[kRowVecs];
    int64_t eo[kRowVecs], go[kRowVecs];  // element offsets in dH / out and in GU
#pragma unroll
    for (int j = 0; j < kRowVecs; ++j) {
      const int64_t v = v0 + (int64_t)j * kNT;
      const int64_t vv = v < nvec ? v : nvec - 1;  // loads of a clamped vector, not stored
      const int64_t row = vv / per_row;
      const int64_t col = (vv - row * per_row) * 8;
      eo[j] = row * I + col;
      go[j] = row * 2 * I + col;
      dh[j] = *reinterpret_cast<const uint4*>(dH + eo[j]);
      g[j] = *reinterpret_cast<const uint4*>(GU + go[j]);
      u[j] = *reinterpret_cast<const uint4*>(GU + go[j] + I);
    }
#pragma unroll
    for (int j = 0; j < kRowVecs; ++j) {
      const uint32_t dhw[4] = {dh[j].x, dh[j].y, dh[j].z, dh[j].w};
      const uint32_t gw[4] = {g[j].x, g[j].y, g[j].z, g[j].w};
      const uint32_t uw[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
      uint32_t dg[4], du[4], mj = 0;
      geglu_bwd8(dhw, gw, uw, ta, tf, dg, du, mj);
      if (v0 + (int64_t)j * kNT < nvec) {
        m = max(m, mj);
        *reinterpret_cast<uint2*>(out + go[j]) =
            quant8_bf16<FMT>(make_uint4(dg[0], dg[1], dg[2], dg[3]), scale);
        *reinterpret_cast<uint2*>(out + go[j] + I) =
            quant8_bf16<FMT>(make_uint4(du[0], du[1], du[2], du[3]), scale);
      }
    }
  }
  m = block_max_u32<kNT>(m);
  if (threadIdx.x == 0) partials[blockIdx.x] = m;
}

}  // namespace
}  // namespace bf8

using namespace bf8;

extern "C" {

int64_t bf8_geglu_partials_elementwise(int64_t M, int64_t I) { return bwd_blocks(M, I); }

int bf8_geglu_bf16(const void* GU, int64_t M, int64_t I, void* H, uint32_t* partials,
                   void* stream) {
  BF8_CHECK(M >= 0 && I >= 8 && I % 8 == 0, "bf8_geglu_bf16: need I %% 8 == 0 (I=%lld)", (long long)I);
  BF8_CHECK(partials && (M == 0 || (GU && H)), "bf8_geglu_bf16: NULL pointer");  // (no rows: partials of 0)
  BF8_CHECK((((uintptr_t)GU | (uintptr_t)H) & 15) == 0,
            "bf8_geglu_bf16: pointers must be 16-byte aligned");
  const int64_t nb = bwd_blocks(M, I);
  hipLaunchKernelGGL(geglu_fwd_kernel, dim3((unsigned)nb), dim3(kNT), 0, as_stream(stream),
                     (const uint16_t*)GU, M, I, (uint16_t*)H, partials);
  return launch_status("geglu_fwd_kernel");
}

int64_t bf8_geglu_bwd_partials(int64_t M, int64_t I) { return bwd_blocks(M, I); }

int bf8_geglu_bwd(const void* dH, const void* GU, int64_t M, int64_t I, void* dGU,
                  uint32_t* partials, void* stream) {
  BF8_CHECK(M >= 0 && I >= 8 && I % 8 == 0, "bf8_geglu_bwd: need I %% 8 == 0 (I=%lld)", (long long)I);
  BF8_CHECK(partials && (M == 0 || (dH && GU && dGU)), "bf8_geglu_bwd: NULL pointer");
  BF8_CHECK((((uintptr_t)dH | (uintptr_t)GU | (uintptr_t)dGU) & 15) == 0,
            "bf8_geglu_bwd: pointers must be 16-byte aligned");
  const int64_t nb = bwd_blocks(M, I);
  hipLaunchKernelGGL(geglu_bwd_kernel, dim3((unsigned)nb), dim3(kNT), 0, as_stream(stream),
                     (const uint16_t*)dH, (const uint16_t*)GU, M, I, (uint16_t*)dGU, partials);
  return launch_status("geglu_bwd_kernel");
}

int64_t bf8_geglu_bwd_delayed_partials(int64_t M, int64_t I) { return fused_blocks(M, I); }

int bf8_geglu_bwd_delayed(const void* dH, const void* GU, int64_t M, int64_t I, float* state,
                          int len, int pos, const uint32_t* prev_partials, int64_t n_prev, int fmt,
                          float* meta_out, uint8_t* out, uint8_t* out_t, uint32_t* partials_out,
                          void* stream) {
  BF8_CHECK(fmt == BF8_E4M3 || fmt == BF8_E5M2, "bf8_geglu_bwd_delayed: bad fmt %d", fmt);
  BF8_CHECK(M >= 0 && I >= kTT && I % kTT == 0,
            "bf8_geglu_bwd_delayed: need I %% 64 == 0 (I=%lld)", (long long)I);
  BF8_CHECK(!out_t || M % 16 == 0,
            "bf8_geglu_bwd_delayed: a transposed copy needs M %% 16 == 0 (M=%lld)", (long long)M);
  BF8_CHECK(dH && GU && state && partials_out && (out || out_t),
            "bf8_geglu_bwd_delayed: NULL pointer");
  BF8_CHECK(len >= 1 && len <= 1024 && pos >= 0 && pos < len,
            "bf8_geglu_bwd_delayed: bad history length %d / slot %d", len, pos);
  BF8_CHECK(n_prev >= 0 && n_prev <= 4096 && (n_prev == 0 || prev_partials),
            "bf8_geglu_bwd_delayed: bad previous partials (%lld)", (long long)n_prev);
  BF8_CHECK((((uintptr_t)dH | (uintptr_t)GU | (uintptr_t)out | (uintptr_t)out_t) & 15) == 0,
            "bf8_geglu_bwd_delayed: pointers must be 16-byte aligned");
  if (M == 0) return BF8_OK;
  const int64_t nb = fused_blocks(M, I);
  hipStream_t s = as_stream(stream);
  const uint16_t* dh = (const uint16_t*)dH;
  const uint16_t* gu = (const uint16_t*)GU;
  if (!out_t) {
    if (fmt == BF8_E4M3)
      hipLaunchKernelGGL(geglu_bwd_delayed_rows_kernel<BF8_E4M3>, dim3((unsigned)nb), dim3(kNT), 0,
                         s, dh, gu, M, I, state, len, pos, prev_partials, n_prev, meta_out, out,
                         partials_out);
    else
      hipLaunchKernelGGL(geglu_bwd_delayed_rows_kernel<BF8_E5M2>, dim3((unsigned)nb), dim3(kNT), 0,
                         s, dh, gu, M, I, state, len, pos, prev_partials, n_prev, meta_out, out,
                         partials_out);
    return launch_status("geglu_bwd_delayed_rows_kernel");
  }
  if (fmt == BF8_E4M3)
    hipLaunchKernelGGL(geglu_bwd_delayed_kernel<BF8_E4M3>, dim3((unsigned)nb), dim3(kNT), 0, s,
                       dh, gu, M, I, state, len, pos, prev_partials, n_prev, meta_out, out, out_t,
                       partials_out);
  else
    hipLaunchKernelGGL(geglu_bwd_delayed_kernel<BF8_E5M2>, dim3((unsigned)nb), dim3(kNT), 0, s,
                       dh, gu, M, I, state, len, pos, prev_partials, n_prev, meta_out, out, out_t,
                       partials_out);
  return launch_status("geglu_bwd_delayed_kernel");
}

static int check_geglu_mxi8(const char* who, const void* in, const void* out, const void* gu8,
                            const void* gu8_e, int64_t M, int64_t I) {
  BF8_CHECK(M >= 0 && I >= 0 && I % 32 == 0, "%s: need I %% 32 == 0 (M=%lld, I=%lld)", who, (long long)M,
            (long long)I);
  if (M == 0 || I == 0) return BF8_OK;
  BF8_CHECK(in && out && gu8 && gu8_e, "%s: NULL pointer", who);
  BF8_CHECK((((uintptr_t)in | (uintptr_t)out) & 15) == 0 && ((uintptr_t)gu8 & 7) == 0,
            "%s: bf16 tensors must be 16-byte, GU8 8-byte aligned", who);
  return BF8_OK;
}

int bf8_geglu_mxint8(const void* GU, int64_t M, int64_t I, void* H, int8_t* GU8, uint8_t* GU8_exp,
                     void* stream) {
  if (const int rc = check_geglu_mxi8("bf8_geglu_mxint8", GU, H, GU8, GU8_exp, M, I)) return rc;
  if (M == 0 || I == 0) return BF8_OK;
  hipLaunchKernelGGL(geglu_fwd_mxi8_kernel, dim3((unsigned)bwd_blocks(M, I)), dim3(kNT), 0,
                     as_stream(stream), (const uint16_t*)GU, M, I, (uint16_t*)H, GU8, GU8_exp);
  return launch_status("geglu_fwd_mxi8_kernel");
}

size_t bf8_geglu_bwd_mxint8_maxima(int64_t M, int64_t I) {
  return M > 0 && I > 0 ? int8_maxima_bytes(M, 2 * I, 2) : 0;
}

int bf8_geglu_bwd_mxint8(const void* dH, const int8_t* GU8, const uint8_t* GU8_exp, int64_t M, int64_t I,
                         void* dGU, void* maxima, size_t maxima_bytes, void* stream) {
  const char* who = "bf8_geglu_bwd_mxint8";
  if (const int rc = check_geglu_mxi8(who, dH, dGU, GU8, GU8_exp, M, I)) return rc;
  BF8_CHECK(!maxima || (M < (1LL << 31) && I < (1 << 22)), "%s: M or I too large", who);
  BF8_CHECK(!maxima || (((uintptr_t)maxima & 255) == 0 && maxima_bytes >= bf8_geglu_bwd_mxint8_maxima(M, I)),
            "%s: the maxima need %zu bytes, 256-byte aligned (got %zu)", who,
            bf8_geglu_bwd_mxint8_maxima(M, I), maxima_bytes);
  if (M == 0 || I == 0) return BF8_OK;
  if (!maxima) {
    hipLaunchKernelGGL(geglu_bwd_mxi8_kernel, dim3((unsigned)bwd_blocks(M, I)), dim3(kNT), 0, as_stream(stream),
                       (const uint16_t*)dH, GU8, GU8_exp, M, I, (uint16_t*)dGU);
    return launch_status("geglu_bwd_mxi8_kernel");
  }
  const Int8Maxima p = int8_maxima(maxima, M, 2 * I, 2);
  hipLaunchKernelGGL(geglu_bwd_mxi8_maxima_kernel, dim3((unsigned)(p.strips * (p.row_tiles / 2))), dim3(kNT), 0,
                     as_stream(stream), (const uint16_t*)dH, GU8, GU8_exp, I, (uint16_t*)dGU, p);
  return launch_status("geglu_bwd_mxi8_maxima_kernel");
}

}  // extern "C"
