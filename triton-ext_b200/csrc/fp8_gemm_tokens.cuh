// Epilogue and work units shared by the kernels of fp8_gemm_tokens.cu.
//
// Those kernels compute D[n, m] = sum_k W[n, k] X[m, k]: weight rows on the 128-row side of the tensor core, tokens on
// its column side, where the tile width can follow the number of tokens in steps of 16.  The epilogue therefore gets a
// tile as [token][128 weight rows] in fp32 shared memory (one conflict-free store per value from the TMEM lanes) and
// reads it back a token at a time: a lane holds four neighbouring output columns, so bias, residual, pre-activation and
// output are read and written 8 bytes a lane, 256 a warp, and rows of other experts are never touched.
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
__device__ __forceinline__ void store4(uint16_t* p, const float (&v)[4], int n, int N, int half, int vec) {
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
__device__ __forceinline__ void load4(const uint16_t* p, float (&v)[4], int n, int N, int half, int vec) {
  uint32_t a = 0, b = 0;
  if (vec && n + 4 <= N) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    a = u.x, b = u.y;
  } else {
    if (n < N) a = p[0];
    if (n + 1 < N) a |= (uint32_t)p[1] << 16;
    if (n + 2 < N) b = p[2];
    if (n + 3 < N) b |= (uint32_t)p[3] << 16;
  }
  if (half) {
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a)), y = __half22float2(*reinterpret_cast<const __half2*>(&b));
    v[0] = x.x, v[1] = x.y, v[2] = y.x, v[3] = y.y;
  } else {
    v[0] = __uint_as_float(a << 16), v[1] = __uint_as_float(a & 0xffff0000u);
    v[2] = __uint_as_float(b << 16), v[3] = __uint_as_float(b & 0xffff0000u);
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

// Finishes tokens first, first + step, ... < cnt of a tile: fetch(m, column) returns four values of token m from weight
// row `column` of the tile (a multiple of 4).  One warp per token.
template <typename Fetch>
__device__ __forceinline__ void tok_finish(const TokParams& p, int e, int64_t row0, int n0, int cnt, int first, int step,
                                           int lane, Fetch fetch) {
  const int n = n0 + 4 * lane;
  const float sw = tok_scale_w(p, e);
  float bias[4] = {0.f, 0.f, 0.f, 0.f};
  if (p.bias) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.N) bias[i] = load_f32(p.bias, n + i, p.bias_type);
  }
  for (int m = first; m < cnt; m += step) {
    const int64_t row = row0 + m;
    const float4 a = fetch(m, 4 * lane);
    const float alpha = tok_alpha(p, row, sw);
    float v[4] = {__fmul_rn(a.x, alpha), __fmul_rn(a.y, alpha), __fmul_rn(a.z, alpha), __fmul_rn(a.w, alpha)};
    if (p.bias) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += bias[i];
    }
    if (p.pre) store4(p.pre + row * p.ld_pre + n, v, n, p.N, p.half, p.vec_pre);
    act4(p.act, v);
    if (p.residual) {
      float r[4];
      load4(p.residual + row * p.ld_res + n, r, n, p.N, p.half, p.vec_res);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += r[i];
    }
    store4(p.out + row * p.ld_out + n, v, n, p.N, p.half, p.vec_out);
  }
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
      const float gi = __fmul_rn(g[i], alpha);
      const float h = __fmul_rn(__fdividef(gi, 1.0f + __expf(-gi)), __fmul_rn(u[i], alpha));
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
