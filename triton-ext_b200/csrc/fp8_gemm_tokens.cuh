// Epilogue and work units shared by the kernels of fp8_gemm_tokens.cu.
//
// Those kernels compute D[n, m] = sum_k W[n, k] X[m, k]: weight rows on the 128-row side of the tensor core, tokens on
// its column side, where the tile width can follow the number of tokens in steps of 16.  The epilogue therefore gets a
// tile as [token][128 weight rows] in fp32 shared memory (one conflict-free store per value from the TMEM lanes) and
// reads it back a token at a time: a lane holds four neighbouring output columns, so residual, pre-activation and output
// are read and written 8 bytes a lane, 256 a warp, and rows of other experts are never touched.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include "activations.cuh"
#include "b2x_internal.h"
#include "b2x_ptx.cuh"
#include "fp8_gemm_common.cuh"
#include "fp8_gemm_swiglu.cuh"

namespace b2x {

constexpr int kTkRows = 128;  // weight rows per CTA tile

struct TokParams {
  int N, K, E;
  int64_t rows;            // rows of x (an upper bound where offsets are given)
  const int32_t* offsets;  // NULL: one product over all rows
  int n_tiles, k_tiles, splits;
  uint32_t idesc;          // without the column count
  int l2_w;
  // scales: 0 none, 1 one, 2 per row / per expert
  const float* scale_x;
  const float* scale_w;
  int sx_mode, sw_mode;
  // epilogue
  int half;  // fp16 instead of bf16
  const void* bias;
  int bias_type, act;
  const uint16_t* residual;
  int64_t ld_res;
  uint16_t* out;
  int64_t ld_out;
  uint16_t* pre;
  int64_t ld_pre;
  int vec_out, vec_res, vec_pre;  // rows start on 8-byte boundaries
  // SwiGLU + fp8
  uint8_t* h;
  int64_t ld_h;
  int h_e5m2;
  const float* h_scale;
  float* h_amax;
};

// Work unit: `cnt` tokens from row `row0` of expert `e` against weight tile `nt`; cnt = 0: none left.
struct TokUnit {
  int e, nt, cnt;
  int64_t row0;
};

__device__ __forceinline__ uint32_t pack2(float lo, float hi, int half) {
  if (half) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  return pack_bf16x2(lo, hi);
}
// Four values from column n of a row of N; vec: the row starts on an 8-byte boundary.
__device__ __forceinline__ void store4(uint16_t* p, const float* v, int n, int N, int half, int vec) {
  const uint32_t a = pack2(v[0], v[1], half), b = pack2(v[2], v[3], half);
  if (vec && n + 4 <= N) {
    *reinterpret_cast<uint2*>(p) = make_uint2(a, b);
    return;
  }
  if (n < N) p[0] = (uint16_t)a;
  if (n + 1 < N) p[1] = (uint16_t)(a >> 16);
  if (n + 2 < N) p[2] = (uint16_t)b;
  if (n + 3 < N) p[3] = (uint16_t)(b >> 16);
}
__device__ __forceinline__ uint2 load4(const uint16_t* p, int n, int N, int vec) {
  if (vec && n + 4 <= N) return *reinterpret_cast<const uint2*>(p);
  uint32_t a = 0, b = 0;
  if (n < N) a = p[0];
  if (n + 1 < N) a |= (uint32_t)p[1] << 16;
  if (n + 2 < N) b = p[2];
  if (n + 3 < N) b |= (uint32_t)p[3] << 16;
  return make_uint2(a, b);
}
__device__ __forceinline__ void add4(float* v, uint2 u, int half) {
  if (half) {
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&u.x)), y = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
    v[0] += x.x, v[1] += x.y, v[2] += y.x, v[3] += y.y;
  } else {
    v[0] += __uint_as_float(u.x << 16), v[1] += __uint_as_float(u.x & 0xffff0000u);
    v[2] += __uint_as_float(u.y << 16), v[3] += __uint_as_float(u.y & 0xffff0000u);
  }
}

// Factor of the row: scale_x[row] * scale_w[expert].
__device__ __forceinline__ float tok_alpha(const TokParams& p, int64_t row, float sw) {
  const float sx = p.sx_mode == 0 ? 1.0f : __ldg(p.scale_x + (p.sx_mode == 2 ? row : 0));
  return __fmul_rn(sx, sw);
}
__device__ __forceinline__ float tok_scale_w(const TokParams& p, int e) {
  return p.sw_mode == 0 ? 1.0f : __ldg(p.scale_w + (p.sw_mode == 2 ? e : 0));
}

// What a lane needs of its four columns n .. n + 3 of the weight tile at n0, for all tokens.
struct TokCols {
  int n;
  float sw;
  float bias[4];
};
__device__ __forceinline__ TokCols tok_cols(const TokParams& p, int e, int n0, int lane) {
  TokCols c;
  c.n = n0 + 4 * lane;
  c.sw = tok_scale_w(p, e);
#pragma unroll
  for (int i = 0; i < 4; ++i) c.bias[i] = p.bias && c.n + i < p.N ? load_f32(p.bias, c.n + i, p.bias_type) : 0.0f;
  return c;
}

// Finishes U tokens of a tile side by side, a warp all 128 columns of each: token u of the row `row + u * step`, where
// bit u of `live` is set.  fetch(u) gives the lane's four sums.
template <int U, typename Fetch>
__device__ __forceinline__ void tok_finish(const TokParams& p, const TokCols& c, int64_t row, int step, uint32_t live,
                                           Fetch fetch) {
  uint2 res[U];
  float alpha[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t r = row + (int64_t)u * step;
    res[u] = make_uint2(0, 0);
    if (p.residual && (live >> u & 1) && c.n < p.N) res[u] = load4(p.residual + r * p.ld_res + c.n, c.n, p.N, p.vec_res);
    alpha[u] = live >> u & 1 ? tok_alpha(p, r, c.sw) : 0.0f;
  }
  float v[4 * U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float4 f = fetch(u);
    v[4 * u] = fmaf(f.x, alpha[u], c.bias[0]);
    v[4 * u + 1] = fmaf(f.y, alpha[u], c.bias[1]);
    v[4 * u + 2] = fmaf(f.z, alpha[u], c.bias[2]);
    v[4 * u + 3] = fmaf(f.w, alpha[u], c.bias[3]);
  }
  if (p.pre) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (live >> u & 1) store4(p.pre + (row + (int64_t)u * step) * p.ld_pre + c.n, v + 4 * u, c.n, p.N, p.half, p.vec_pre);
  }
  act_all<4 * U>(p.act, v);
  if (p.residual) {
#pragma unroll
    for (int u = 0; u < U; ++u) add4(v + 4 * u, res[u], p.half);
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (live >> u & 1) store4(p.out + (row + (int64_t)u * step) * p.ld_out + c.n, v + 4 * u, c.n, p.N, p.half, p.vec_out);
}

constexpr int kTkChunk = 16;  // tokens per epilogue step of the pair kernel

// One epilogue warpgroup finishes a tile of cnt tokens whose accumulator starts at TMEM address t_row (this warp's
// lanes), in steps of 16 tokens through two halves of `stage` ([16][128] fp32 each): warp q finishes the tokens q, q + 4,
// q + 8 and q + 12 of a step.  What the tile needs is fixed at compile time; only for tiles whose 128 columns all exist
// and whose rows allow 8-byte accesses.  `release` is called when the accumulator has been read.
template <int HALF, int ACT, int RES, int PRE, typename Release>
__device__ __forceinline__ void tok_tile(const TokParams& p, const TokCols& c, uint32_t t_row, int64_t row0, int cnt, int q,
                                         int lane, uint32_t stage, uint32_t bar_id, Release release) {
  const int64_t row = row0 + q;
  uint16_t* out = p.out + row * p.ld_out + c.n;
  uint16_t* pre = PRE ? p.pre + row * p.ld_pre + c.n : nullptr;
  const uint16_t* res = RES ? p.residual + row * p.ld_res + c.n : nullptr;
  const float* sx = p.sx_mode == 2 ? p.scale_x + row : nullptr;
  const float one = p.sx_mode == 1 ? __fmul_rn(__ldg(p.scale_x), c.sw) : c.sw;
  const int64_t step_out = 4 * p.ld_out, step_pre = 4 * p.ld_pre, step_res = 4 * p.ld_res;
  const uint32_t put = stage + (q * 32 + lane) * 4, get = stage + (q * kTkRows + 4 * lane) * 4;
  uint32_t half = 0;  // byte offset of the staging half in use
  uint32_t acc[kTkChunk];
  tmem_ld_32x32b_x16(t_row, acc);
#pragma unroll 1
  for (int left = cnt; left > 0; left -= kTkChunk) {  // token 4 u of this warp exists: 4 u < left - q
    const int mine = left - q;
    uint2 r[4];
    float alpha[4] = {one, one, one, one};
    if (RES) {
#pragma unroll
      for (int u = 0; u < 4; ++u, res += step_res)
        if (4 * u < mine) r[u] = *reinterpret_cast<const uint2*>(res);
    }
    if (sx) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (4 * u < mine) alpha[u] = __fmul_rn(__ldg(sx + 4 * u), c.sw);
      sx += kTkChunk;
    }
    tmem_ld_wait();
    tmem_regs_after_wait(acc);
#pragma unroll
    for (int i = 0; i < kTkChunk; ++i) st_shared_f32(put + half + i * kTkRows * 4, __uint_as_float(acc[i]));
    tc_fence_before();
    // the other half of the staging was read before the barrier of the step before: one barrier a step
    named_bar_sync(bar_id, 128);
    if (left > kTkChunk) {
      t_row += kTkChunk;
      tmem_ld_32x32b_x16(t_row, acc);
    } else {
      release();
    }
    float v[16];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float4 f = ld_shared_f32x4(get + half + 4 * u * kTkRows * 4);
      v[4 * u] = fmaf(f.x, alpha[u], c.bias[0]);
      v[4 * u + 1] = fmaf(f.y, alpha[u], c.bias[1]);
      v[4 * u + 2] = fmaf(f.z, alpha[u], c.bias[2]);
      v[4 * u + 3] = fmaf(f.w, alpha[u], c.bias[3]);
    }
    half ^= kTkChunk * kTkRows * 4;
    if (PRE) {
#pragma unroll
      for (int u = 0; u < 4; ++u, pre += step_pre)
        if (4 * u < mine)
          __stcs(reinterpret_cast<uint2*>(pre), make_uint2(pack2(v[4 * u], v[4 * u + 1], HALF), pack2(v[4 * u + 2], v[4 * u + 3], HALF)));
    }
    if (ACT) act_all<16>(p.act, v);
#pragma unroll
    for (int u = 0; u < 4; ++u, out += step_out) {
      if (RES) add4(v + 4 * u, r[u], HALF);
      if (4 * u < mine)
        __stcs(reinterpret_cast<uint2*>(out), make_uint2(pack2(v[4 * u], v[4 * u + 1], HALF), pack2(v[4 * u + 2], v[4 * u + 3], HALF)));
    }
  }
}

__device__ __forceinline__ float tok_swiglu(float g, float u, float alpha) {
  g = __fmul_rn(g, alpha);
  return __fmul_rn(__fmul_rn(g, sigma_fast(g)), __fmul_rn(u, alpha));
}

// The same for a SwiGLU tile, whose 128 weight rows alternate 16 gate and 16 up rows: 64 columns of h.  Half a warp per
// token; max |h| is collected in `amax`.
template <typename Fetch>
__device__ __forceinline__ void tok_finish_swiglu(const TokParams& p, int e, int64_t row0, int n0, int cnt, int first,
                                                  int step, int lane, float inv, float& amax, Fetch fetch) {
  const int hc = 4 * (lane & 15);
  const int col = (hc >> 4) * 32 + (hc & 15);
  const float sw = tok_scale_w(p, e);
  const float fmax = p.h_e5m2 ? 57344.0f : 448.0f;
  for (int m0 = 2 * first; m0 < cnt; m0 += 2 * step) {
    const int m = m0 + (lane >> 4);
    if (m >= cnt) continue;
    const int64_t row = row0 + m;
    const float4 g4 = fetch(m, col), u4 = fetch(m, col + 16);
    const float alpha = tok_alpha(p, row, sw);
    const float g[4] = {g4.x, g4.y, g4.z, g4.w}, u[4] = {u4.x, u4.y, u4.z, u4.w};
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float h = tok_swiglu(g[i], u[i], alpha);
      amax = fmaxf(amax, fabsf(h));
      y[i] = swiglu_clamp(__fmul_rn(h, inv), fmax);
    }
    const uint16_t lo = p.h_e5m2 ? cvt_e5m2x2(y[0], y[1]) : cvt_e4m3x2(y[0], y[1]);
    const uint16_t hi = p.h_e5m2 ? cvt_e5m2x2(y[2], y[3]) : cvt_e4m3x2(y[2], y[3]);
    *reinterpret_cast<uint32_t*>(p.h + row * p.ld_h + n0 / 2 + hc) = (uint32_t)lo | ((uint32_t)hi << 16);
  }
}

// Expert e's rows, held within [0, rows] whatever offsets say.
__device__ __forceinline__ void tok_range(const TokParams& p, int e, int64_t& lo, int64_t& hi) {
  lo = p.offsets[e];
  hi = p.offsets[e + 1];
  lo = lo < 0 ? 0 : (lo > p.rows ? p.rows : lo);
  hi = hi < lo ? lo : (hi > p.rows ? p.rows : hi);
}

}  // namespace b2x
