// Dispatch and combine of a mixture of experts for sm_100a.
//
// Dispatch sorts the (token, slot) pairs stably by expert and writes each token's row, quantized to fp8 once, to all of
// its places.  The sort is a counting sort:
//   * up to kFusedPairs pairs, every CTA of the row kernel counts all pairs itself (they are a few KB) and ranks its own
//     token's: one launch;
//   * above, one cluster of 8 CTAs (moe_plan_kernel) counts and ranks contiguous eighths of the pairs, its warps
//     contiguous parts of those; counts meet in shared memory, the CTAs' over distributed shared memory.  No global
//     counters, no atomics whose order matters: the same input gives the same order.
// Row kernel: one CTA per token reads the row once (it stays in registers between the maximum and the cast) and stores
// top_k copies, 16 bytes a thread.  Bound: HBM, tokens * cols * (4 or 2) bytes in and tokens * top_k * cols out: 8191 x 7168
// bf16, top_k = 8 in 107 us (5.5 TB/s), of which the plan is 14, partly beside the rows.  16 tokens: 6.3 us.
//
// Combine reads the top_k rows of a token side by side (8 predicated 16-byte loads in flight per thread; with branches
// around them the loads went out one by one and the same case took 272 us) and adds them in the order of the slots in
// fp32.  Bound: HBM, 8191 x 7168, top_k = 8 with residual in 175 us; its gradients for 4095 tokens in 161 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include "activations.cuh"
#include "b2x_internal.h"
#include "b2x_ptx.cuh"

namespace b2x {

constexpr int kRowThreads = 128;
constexpr int kFusedPairs = 512;    // pairs that a CTA counts by itself (2048 pairs so: 19 us, in two launches 14)
constexpr int kPlanCtas = 8;
constexpr int kPlanThreads = 1024;
constexpr int kPlanDepth = 8;  // loads of a lane in flight
constexpr int kPlanWarps = kPlanThreads / 32;

struct DispatchParams {
  const void* x;
  int x_f32;
  int64_t tokens, cols, ld_x;
  const int32_t* indices;
  int k, E;
  uint8_t* q;
  int q_e5m2;
  int64_t ld_q;
  float* scale;
  const float* given;
  int32_t* offsets;
  int32_t* rows;
  int fused;  // ranks are computed here, not read from rows
  int vec_x, vec_q;  // rows start on 16-byte boundaries
};

// Exclusive sums of cnt[0..E) in place by the whole CTA; cnt[E] receives the total.
__device__ __forceinline__ void block_exclusive_scan(int* cnt, int E, int* warp_part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int carry = 0;
  for (int base = 0; base < E; base += blockDim.x) {
    const int i = base + threadIdx.x;
    const int v = i < E ? cnt[i] : 0;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    if (lane == 31) warp_part[warp] = s;
    __syncthreads();
    // sums of the warps before this one and of all, the same in every warp
    const int part = lane < warps ? warp_part[lane] : 0;
    const int before = carry + __reduce_add_sync(0xffffffffu, lane < warp ? part : 0);
    const int all = carry + __reduce_add_sync(0xffffffffu, part);
    if (i < E) cnt[i] = before + s - v;
    carry = all;
    __syncthreads();
  }
  if (threadIdx.x == 0) cnt[E] = carry;
  __syncthreads();
}

// One cluster sorts all pairs; see the top of the file.  Shared: hist[warps][E], then total[E + 1].
__global__ void __launch_bounds__(kPlanThreads)
    moe_plan_kernel(const int32_t* __restrict__ indices, int64_t pairs, int E, int32_t* __restrict__ offsets,
                    int32_t* __restrict__ rows) {
  extern __shared__ int plan_smem[];
  __shared__ int warp_part[kPlanWarps];
  int* hist = plan_smem;                 // [kPlanWarps][E]: counts, then next row of (warp, expert)
  int* total = hist + kPlanWarps * E;    // [E + 1]: this CTA's counts; peers read them
  int* start = total + E + 1;            // [E + 1]: offsets of the experts
  int* prior = start + E + 1;            // [E]: pairs of the CTAs before this one
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t rank = blockIdx.x, ctas = gridDim.x;  // one cluster
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the rows may be read and scaled meanwhile
  for (int i = threadIdx.x; i < kPlanWarps * E; i += kPlanThreads) hist[i] = 0;
  __syncthreads();
  // contiguous parts, a multiple of 32 pairs for each warp
  const int64_t per_warp = ((pairs + ctas * kPlanWarps - 1) / (ctas * kPlanWarps) + 31) / 32 * 32;
  const int64_t lo = ((int64_t)rank * kPlanWarps + warp) * per_warp;
  const int64_t hi = lo + per_warp < pairs ? lo + per_warp : pairs;
  int* mine = hist + warp * E;
  int held[kPlanDepth];  // the first pairs of the lane, for both passes; -1: dropped or none
  for (int64_t i0 = lo; i0 < hi; i0 += 32 * kPlanDepth) {
    int e[kPlanDepth];
#pragma unroll
    for (int u = 0; u < kPlanDepth; ++u) {
      const int64_t i = i0 + 32 * u + lane;
      e[u] = i < hi ? indices[i] : -1;
    }
#pragma unroll
    for (int u = 0; u < kPlanDepth; ++u) {
      if (e[u] >= E) e[u] = -1;
      if (i0 == lo) held[u] = e[u];
      if (e[u] >= 0) atomicAdd(&mine[e[u]], 1);  // a count: the order does not matter
    }
  }
  __syncthreads();
  // per expert: exclusive sums over the warps, the CTA's total
  for (int e = threadIdx.x; e < E; e += kPlanThreads) {
    int s = 0;
#pragma unroll 8
    for (int w = 0; w < kPlanWarps; ++w) {
      const int c = hist[w * E + e];
      hist[w * E + e] = s;
      s += c;
    }
    total[e] = s;
  }
  cluster_sync();
  for (int e = threadIdx.x; e < E; e += kPlanThreads) {
    int c[kPlanCtas], before = 0, all = 0;
#pragma unroll
    for (uint32_t r = 0; r < kPlanCtas; ++r) {
      c[r] = 0;
      if (r < ctas)
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(c[r]) : "r"(mapa_shared(smem_u32(&total[e]), r)) : "memory");
    }
#pragma unroll
    for (uint32_t r = 0; r < kPlanCtas; ++r) {
      if (r < rank) before += c[r];
      all += c[r];
    }
    start[e] = all;
    prior[e] = before;
  }
  __syncthreads();
  block_exclusive_scan(start, E, warp_part);
  if (rank == 0)
    for (int e = threadIdx.x; e <= E; e += kPlanThreads) offsets[e] = start[e];
  // ranks, in the order of the pairs
  for (int64_t i0 = lo; i0 < hi; i0 += 32 * kPlanDepth) {
    int e[kPlanDepth];
#pragma unroll
    for (int u = 0; u < kPlanDepth; ++u) {
      const int64_t i = i0 + 32 * u + lane;
      e[u] = i0 == lo ? held[u] : (i < hi ? indices[i] : -1);
    }
#pragma unroll
    for (int u = 0; u < kPlanDepth; ++u) {
      if (i0 + 32 * u >= hi) break;
      const int64_t i = i0 + 32 * u + lane;
      const int ex = e[u] >= 0 && e[u] < E ? e[u] : -1;
      const uint32_t same = __match_any_sync(0xffffffffu, ex);
      int row = -1;
      if (ex >= 0) row = start[ex] + prior[ex] + mine[ex] + __popc(same & ((1u << lane) - 1));
      __syncwarp();
      if (ex >= 0 && lane == 31 - __clz(same)) mine[ex] += __popc(same);
      __syncwarp();
      if (i < hi) rows[i] = row;
    }
  }
  cluster_sync();  // peers may still read this CTA's totals
}

// 16 consecutive values of a row as they are stored: 16 or 8 registers.
template <typename T>
struct Raw16 {
  uint4 v[sizeof(T)];
};
template <typename T>
__device__ __forceinline__ Raw16<T> load16(const DispatchParams& p, int64_t at, int64_t col) {
  Raw16<T> r;
  const T* s = reinterpret_cast<const T*>(p.x) + at + col;
  if (p.vec_x && col + 16 <= p.cols) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) r.v[i] = __ldcs(reinterpret_cast<const uint4*>(s) + i);
  } else {
    T e[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) e[i] = col + i < p.cols ? s[i] : T(0);
    memcpy(&r, e, sizeof(r));
  }
  return r;
}
__device__ __forceinline__ void unpack16(const Raw16<float>& r, float (&v)[16]) { memcpy(v, &r, 64); }
__device__ __forceinline__ void unpack16(const Raw16<uint16_t>& r, float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint4 u = r.v[i];
    v[8 * i] = bf16lo(u.x), v[8 * i + 1] = bf16hi(u.x), v[8 * i + 2] = bf16lo(u.y), v[8 * i + 3] = bf16hi(u.y);
    v[8 * i + 4] = bf16lo(u.z), v[8 * i + 5] = bf16hi(u.z), v[8 * i + 6] = bf16lo(u.w), v[8 * i + 7] = bf16hi(u.w);
  }
}

template <int FP8>
__device__ __forceinline__ void store16(const DispatchParams& p, const float (&v)[16], float inv, int64_t col,
                                        const int* row, int k) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = quant4<FP8>(make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]), inv);
  const bool whole = p.vec_q && col + 16 <= p.cols;
  for (int j = 0; j < k; ++j) {
    if (row[j] < 0) continue;
    uint8_t* q = p.q + (int64_t)row[j] * p.ld_q + col;
    if (whole) {
      __stcs(reinterpret_cast<uint4*>(q), make_uint4(w[0], w[1], w[2], w[3]));
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (col + i < p.cols) q[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
  }
}

// One CTA per token.  NV: 16-value pieces that a thread holds in registers (cols <= kRowThreads * 16 * NV); NV = 0:
// longer rows, read a second time (from L2) for the cast.
template <typename T, int NV, int FP8>
__global__ void __launch_bounds__(kRowThreads) moe_dispatch_kernel(const DispatchParams p) {
  extern __shared__ int row_smem[];  // row[k], mine[k]; fused: cnt[E + 1]
  __shared__ int warp_part[kRowThreads / 32];
  __shared__ float warp_max_[kRowThreads / 32];
  const int64_t t = blockIdx.x;
  int* row = row_smem;
  int* mine = row_smem + p.k;
  int* cnt = mine + p.k;
  const int64_t at = t * p.ld_x;
  Raw16<T> raw[NV ? NV : 1];
  float v[16];
  float amax = 0.0f;
  // all loads go out before anything waits for one
  constexpr int kDepth = kFusedPairs / kRowThreads;
  int pair_of[kDepth];  // fused: this thread's pairs
  if (p.fused) {
#pragma unroll
    for (int u = 0; u < kDepth; ++u) {
      const int64_t i = u * kRowThreads + threadIdx.x;
      pair_of[u] = i < p.tokens * p.k ? __ldg(p.indices + i) : -1;
    }
    for (int j = threadIdx.x; j < p.k; j += kRowThreads) row[j] = 0, mine[j] = __ldg(p.indices + t * p.k + j);
    for (int e = threadIdx.x; e < p.E; e += kRowThreads) cnt[e] = 0;
  }
  if (NV) {
#pragma unroll
    for (int n = 0; n < NV; ++n) raw[n] = load16<T>(p, at, (int64_t)(n * kRowThreads + threadIdx.x) * 16);
  }
  float s;
  if (!p.given) {
    if (NV) {
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        unpack16(raw[n], v);
#pragma unroll
        for (int i = 0; i < 16; ++i) amax = absmax_xs(amax, v[i]);
      }
    } else {
      for (int64_t c = (int64_t)threadIdx.x * 16; c < p.cols; c += kRowThreads * 16) {
        unpack16(load16<T>(p, at, c), v);
#pragma unroll
        for (int i = 0; i < 16; ++i) amax = absmax_xs(amax, v[i]);
      }
    }
    amax = fabsf(amax);
#pragma unroll
    for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if ((threadIdx.x & 31) == 0) warp_max_[threadIdx.x >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kRowThreads / 32; ++w) amax = fmaxf(amax, warp_max_[w]);
    s = __fdiv_rn(amax, Fp8Traits<FP8>::kMax);
  } else {
    s = __ldg(p.given);
  }
  const float inv = s == 0.0f ? 0.0f : __fdiv_rn(1.0f, s);
  if (p.fused) {
    const int own = (int)(t * p.k);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kDepth; ++u) {
      const int i = u * kRowThreads + threadIdx.x, e = pair_of[u];
      if (e >= 0 && e < p.E) atomicAdd(&cnt[e], 1);
      if (i < own + p.k)
        for (int j = 0; j < p.k; ++j)  // pairs before this token's j-th that go to the same expert
          if (i < own + j && e == mine[j]) atomicAdd(&row[j], 1);
    }
    __syncthreads();
    block_exclusive_scan(cnt, p.E, warp_part);
    for (int j = threadIdx.x; j < p.k; j += kRowThreads) {
      const int e = mine[j];
      const int r = e >= 0 && e < p.E ? row[j] + cnt[e] : -1;
      row[j] = r;
      p.rows[own + j] = r;
    }
    if (t == 0)
      for (int e = threadIdx.x; e <= p.E; e += kRowThreads) p.offsets[e] = cnt[e];
  } else {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the plan is there
    for (int j = threadIdx.x; j < p.k; j += kRowThreads) row[j] = p.rows[t * p.k + j];
  }
  __syncthreads();
  if (!p.given)
    for (int j = threadIdx.x; j < p.k; j += kRowThreads)
      if (row[j] >= 0) p.scale[row[j]] = s;
  if (NV) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int64_t c = (int64_t)(n * kRowThreads + threadIdx.x) * 16;
      unpack16(raw[n], v);
      if (c < p.cols) store16<FP8>(p, v, inv, c, row, p.k);
    }
  } else {
    for (int64_t c = (int64_t)threadIdx.x * 16; c < p.cols; c += kRowThreads * 16) {
      unpack16(load16<T>(p, at, c), v);
      store16<FP8>(p, v, inv, c, row, p.k);
    }
  }
}

template <typename T, int NV, int FP8>
static cudaError_t launch_dispatch_t(const DispatchParams& p, size_t smem, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.tokens, 1, 1);
  cfg.blockDim = dim3(kRowThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  // After a plan kernel the rows start beside it: reading and scaling x needs no plan.
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.fused ? 0 : 1;
  return cudaLaunchKernelEx(&cfg, moe_dispatch_kernel<T, NV, FP8>, p);
}
template <typename T, int FP8>
static cudaError_t launch_dispatch_rows(const DispatchParams& p, size_t smem, cudaStream_t st) {
  const int64_t per = (p.cols + kRowThreads * 16 - 1) / (kRowThreads * 16);
  if (per <= 1) return launch_dispatch_t<T, 1, FP8>(p, smem, st);
  if (per <= 2) return launch_dispatch_t<T, 2, FP8>(p, smem, st);
  if (per <= 4) return launch_dispatch_t<T, 4, FP8>(p, smem, st);
  return launch_dispatch_t<T, 0, FP8>(p, smem, st);
}

struct CombineParams {
  const void* y;
  int64_t y_rows, ld_y;
  const int32_t* rows;
  const float* weights;
  int64_t tokens, cols;
  int k;
  const void* residual;
  int64_t ld_res;
  void* out;  // combine: out; backward: d_y
  int64_t ld_out;
  const void* grad;
  int64_t ld_grad;
  float* d_weights;
};

// What a thread holds of a row at a time: WIDE 16 consecutive bytes, else (rows off the 16-byte grid) four values
// kRowThreads columns apart, so that a warp's accesses stay together.
template <typename T, int V>
struct Piece {
  T e[V];
};
template <typename T, bool WIDE>
struct PieceOf {
  static constexpr int V = WIDE ? 16 / (int)sizeof(T) : 4;
  static constexpr int kStep = kRowThreads * V;  // columns of a CTA's step
  __device__ static __forceinline__ int64_t first(int64_t step) { return step * kStep + (int64_t)threadIdx.x * (WIDE ? V : 1); }
};
template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  if constexpr (sizeof(T) == 4)
    return v;
  else if constexpr (__is_same(T, __half))
    return __half2float(v);
  else
    return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float f) {
  if constexpr (sizeof(T) == 4)
    return f;
  else if constexpr (__is_same(T, __half))
    return __float2half_rn(f);
  else
    return __float2bfloat16_rn(f);
}
// The piece at column c of a row, or zeros where `in` is false: a predicate, not a branch, so that several loads go out
// together.
template <typename T, bool WIDE>
__device__ __forceinline__ Piece<T, PieceOf<T, WIDE>::V> load_piece(bool in, const T* row, int64_t c, int64_t cols) {
  Piece<T, PieceOf<T, WIDE>::V> r;
  if constexpr (WIDE) {
    uint4 u;
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
        "@q ld.global.cs.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
        : "=&r"(u.x), "=&r"(u.y), "=&r"(u.z), "=&r"(u.w)
        : "l"(row + c), "r"((int)in));
    memcpy(&r, &u, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.e[i] = in && c + i * kRowThreads < cols ? row[c + i * kRowThreads] : from_f32<T>(0.0f);
  }
  return r;
}
template <typename T, bool WIDE>
__device__ __forceinline__ void store_piece(T* row, int64_t c, int64_t cols, const Piece<T, PieceOf<T, WIDE>::V>& v) {
  if constexpr (WIDE) {
    uint4 u;
    memcpy(&u, &v, 16);
    __stcs(reinterpret_cast<uint4*>(row + c), u);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i * kRowThreads < cols) row[c + i * kRowThreads] = v.e[i];
  }
}

// A CTA takes a token's columns in steps of PieceOf::kStep, `per` CTAs side by side.  MANY: more than 8 slots, their rows
// and weights read again for every step.
template <typename T, bool WIDE, bool MANY>
__global__ void __launch_bounds__(kRowThreads) moe_combine_kernel(const CombineParams p, uint32_t per) {
  using A = PieceOf<T, WIDE>;
  constexpr int U = 8;  // rows in flight
  constexpr int V = A::V;
  const int64_t t = blockIdx.x / per;
  const T* y = reinterpret_cast<const T*>(p.y);
  int r[U];
  float w[U];
  auto slots = [&](int j0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      r[u] = j0 + u < p.k ? __ldg(p.rows + t * p.k + j0 + u) : -1;
      if (r[u] >= p.y_rows) r[u] = -1;
      w[u] = r[u] < 0 ? 0.0f : (p.weights ? __ldg(p.weights + t * p.k + j0 + u) : 1.0f);
    }
  };
  if (!MANY) slots(0);
  const int64_t step = (int64_t)per * A::kStep;
  for (int64_t c = A::first(blockIdx.x % per); c < p.cols; c += step) {
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.0f;
    const Piece<T, V> res =
        load_piece<T, WIDE>(p.residual != nullptr, reinterpret_cast<const T*>(p.residual) + t * p.ld_res, c, p.cols);
    for (int j0 = 0; j0 < (MANY ? p.k : 1); j0 += U) {
      if (MANY) slots(j0);
      Piece<T, V> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = load_piece<T, WIDE>(r[u] >= 0, y + (int64_t)r[u] * p.ld_y, c, p.cols);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = fmaf(w[u], to_f32(v[u].e[i]), acc[i]);
    }
    Piece<T, V> o;
#pragma unroll
    for (int i = 0; i < V; ++i) o.e[i] = from_f32<T>(acc[i] + to_f32(res.e[i]));
    store_piece<T, WIDE>(reinterpret_cast<T*>(p.out) + t * p.ld_out, c, p.cols, o);
  }
}

// One CTA per token; 8 slots at a time (their dot products stay in registers).
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kRowThreads) moe_combine_backward_kernel(const CombineParams p) {
  using A = PieceOf<T, WIDE>;
  constexpr int KC = 8, V = A::V;
  __shared__ float part[kRowThreads / 32][KC];
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* y = reinterpret_cast<const T*>(p.y);
  const T* g = reinterpret_cast<const T*>(p.grad) + t * p.ld_grad;
  T* dy = reinterpret_cast<T*>(p.out);
  for (int j0 = 0; j0 < p.k; j0 += KC) {
    int r[KC];
    float w[KC], dot[KC];
#pragma unroll
    for (int u = 0; u < KC; ++u) {
      r[u] = j0 + u < p.k ? __ldg(p.rows + t * p.k + j0 + u) : -1;
      if (r[u] >= p.y_rows) r[u] = -1;
      w[u] = j0 + u < p.k ? __ldg(p.weights + t * p.k + j0 + u) : 0.0f;
      dot[u] = 0.0f;
    }
    for (int64_t c = A::first(0); c < p.cols; c += A::kStep) {
      Piece<T, V> v[KC];
#pragma unroll
      for (int u = 0; u < KC; ++u) v[u] = load_piece<T, WIDE>(r[u] >= 0, y + (int64_t)r[u] * p.ld_y, c, p.cols);
      const Piece<T, V> gv = load_piece<T, WIDE>(true, g, c, p.cols);
      float gf[V];
#pragma unroll
      for (int i = 0; i < V; ++i) gf[i] = to_f32(gv.e[i]);
#pragma unroll
      for (int u = 0; u < KC; ++u) {
        if (r[u] < 0) continue;
        Piece<T, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          dot[u] = fmaf(gf[i], to_f32(v[u].e[i]), dot[u]);
          o.e[i] = from_f32<T>(w[u] * gf[i]);
        }
        store_piece<T, WIDE>(dy + (int64_t)r[u] * p.ld_out, c, p.cols, o);
      }
    }
#pragma unroll
    for (int u = 0; u < KC; ++u) {
#pragma unroll
      for (int o = 16; o; o >>= 1) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], o);
      if (lane == 0) part[warp][u] = dot[u];
    }
    __syncthreads();
    if (threadIdx.x < KC && j0 + (int)threadIdx.x < p.k) {
      float s = 0.0f;
#pragma unroll
      for (int q = 0; q < kRowThreads / 32; ++q) s += part[q][threadIdx.x];
      p.d_weights[t * p.k + j0 + threadIdx.x] = s;
    }
    __syncthreads();
  }
}

template <typename T, int BACKWARD, bool WIDE>
static cudaError_t launch_combine_t(const CombineParams& p, cudaStream_t st) {
  if constexpr (BACKWARD) {
    moe_combine_backward_kernel<T, WIDE><<<(unsigned)p.tokens, kRowThreads, 0, st>>>(p);
  } else {
    // CTAs side by side on a token: one a step, until there are several times more than fit the GPU at once
    // (8191 x 7168, k = 8: 175 us with 7 CTAs a token, 180 with one; 3000 x 2049, k = 4, narrow: 63 and 43 us).
    uint32_t per = (uint32_t)((p.cols + PieceOf<T, WIDE>::kStep - 1) / PieceOf<T, WIDE>::kStep);
    while (per > 1 && p.tokens * per > (WIDE ? 65536 : 4736)) per = (per + 1) / 2;
    const unsigned grid = (unsigned)(p.tokens * per);
    if (p.k > 8)
      moe_combine_kernel<T, WIDE, true><<<grid, kRowThreads, 0, st>>>(p, per);
    else
      moe_combine_kernel<T, WIDE, false><<<grid, kRowThreads, 0, st>>>(p, per);
  }
  note_launch(1);
  return cudaGetLastError();
}

template <int BACKWARD>
static cudaError_t launch_combine(const CombineParams& p, b2x_dtype type, bool vec, cudaStream_t st) {
  if (type == B2X_F32) return vec ? launch_combine_t<float, BACKWARD, true>(p, st) : launch_combine_t<float, BACKWARD, false>(p, st);
  if (type == B2X_F16) return vec ? launch_combine_t<__half, BACKWARD, true>(p, st) : launch_combine_t<__half, BACKWARD, false>(p, st);
  return vec ? launch_combine_t<__nv_bfloat16, BACKWARD, true>(p, st) : launch_combine_t<__nv_bfloat16, BACKWARD, false>(p, st);
}

// Rows of `elem`-byte values that start on 16-byte boundaries.
static bool rows_aligned(const void* p, int64_t ld, int elem) {
  return ((uintptr_t)p % 16) == 0 && (ld * elem) % 16 == 0;
}

static bool is_float_type(b2x_dtype t) { return t == B2X_F32 || t == B2X_BF16 || t == B2X_F16; }

}  // namespace b2x

extern "C" B2X_API b2x_status b2x_moe_dispatch(const b2x_moe_dispatch_args* a, void* stream) {
  using namespace b2x;
  t_err[0] = 0;
  if (!a) return fail(B2X_ERR_INVALID_ARG, "b2x_moe_dispatch: args is NULL");
  if (a->x_type != B2X_F32 && a->x_type != B2X_BF16)
    return fail(B2X_ERR_UNSUPPORTED, "b2x_moe_dispatch: x must be fp32 or bf16");
  if (!is_fp8(a->q_type)) return fail(B2X_ERR_UNSUPPORTED, "b2x_moe_dispatch: q must be e4m3 or e5m2");
  if (a->tokens < 0 || a->cols < 0 || a->ld_x < a->cols || a->ld_q < a->cols || a->top_k < 1 || a->experts < 1)
    return fail(B2X_ERR_INVALID_ARG, "b2x_moe_dispatch: bad shape (tokens %lld, cols %lld, top_k %d, experts %lld)",
                (long long)a->tokens, (long long)a->cols, a->top_k, (long long)a->experts);
  if (a->experts > 1024 || a->top_k > 1024)
    return fail(B2X_ERR_UNSUPPORTED, "b2x_moe_dispatch: at most 1024 experts and top_k 1024");
  if (a->tokens * a->top_k >= (1LL << 31)) return fail(B2X_ERR_UNSUPPORTED, "b2x_moe_dispatch: tokens * top_k must be < 2^31");
  if (!a->offsets) return fail(B2X_ERR_INVALID_ARG, "b2x_moe_dispatch: NULL offsets");
  if (off_grid(a->x, a->x_type == B2X_F32 ? 4 : 2) || off_grid(a->indices, 4) || off_grid(a->scale, 4) || off_grid(a->given, 4) ||
      off_grid(a->offsets, 4) || off_grid(a->rows, 4))
    return fail(B2X_ERR_INVALID_ARG, "b2x_moe_dispatch: misaligned pointer");
  cudaStream_t st = (cudaStream_t)stream;
  if (a->tokens == 0) {
    cudaError_t e = cudaMemsetAsync(a->offsets, 0, (size_t)(a->experts + 1) * 4, st);
    return e == cudaSuccess ? B2X_OK : cuda_fail(e, "b2x_moe_dispatch: clearing offsets");
  }
  if (!a->indices || !a->rows || (a->cols > 0 && (!a->x || !a->q)) || (!a->given && !a->scale))
    return fail(B2X_ERR_INVALID_ARG, "b2x_moe_dispatch: NULL pointer");
  DispatchParams p{};
  p.x = a->x;
  p.x_f32 = a->x_type == B2X_F32;
  p.tokens = a->tokens;
  p.cols = a->cols;
  p.ld_x = a->ld_x;
  p.indices = a->indices;
  p.k = a->top_k;
  p.E = (int)a->experts;
  p.q = reinterpret_cast<uint8_t*>(a->q);
  p.ld_q = a->ld_q;
  p.scale = a->scale;
  p.given = a->given;
  p.offsets = a->offsets;
  p.rows = a->rows;
  const int64_t pairs = a->tokens * a->top_k;
  p.fused = pairs <= kFusedPairs;
  p.vec_x = rows_aligned(a->x, a->ld_x, p.x_f32 ? 4 : 2);
  p.vec_q = rows_aligned(a->q, a->ld_q, 1);
  if (!p.fused) {
    const int smem = (kPlanWarps * p.E + 2 * (p.E + 1) + p.E) * 4;
    cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(moe_plan_kernel), smem);
    if (e != cudaSuccess) return cuda_fail(e, "b2x_moe_dispatch: shared memory");
    // one CTA while its warps take a few rounds of pairs, else a cluster of them
    cudaLaunchConfig_t cfg = {};
    const unsigned ctas = pairs <= 8 * kPlanThreads ? 1 : kPlanCtas;
    cfg.gridDim = dim3(ctas, 1, 1);
    cfg.blockDim = dim3(kPlanThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, moe_plan_kernel, a->indices, pairs, p.E, a->offsets, a->rows);
    note_launch(1);
    if (e != cudaSuccess) return cuda_fail(e, "b2x_moe_dispatch launch (plan)");
  }
  const size_t smem = (size_t)(2 * p.k + (p.fused ? p.E + 1 : 0)) * 4;
  cudaError_t e;
  if (p.x_f32)
    e = a->q_type == B2X_E5M2 ? launch_dispatch_rows<float, 1>(p, smem, st) : launch_dispatch_rows<float, 0>(p, smem, st);
  else
    e = a->q_type == B2X_E5M2 ? launch_dispatch_rows<uint16_t, 1>(p, smem, st) : launch_dispatch_rows<uint16_t, 0>(p, smem, st);
  note_launch(1);
  return e == cudaSuccess ? B2X_OK : cuda_fail(e, "b2x_moe_dispatch launch");
}

extern "C" B2X_API b2x_status b2x_moe_combine(const void* y, int64_t y_rows, int64_t ld_y, const int32_t* rows,
                                              const float* weights, int64_t tokens, int top_k, int64_t cols,
                                              const void* residual, int64_t ld_residual, void* out, int64_t ld_out,
                                              b2x_dtype type, void* stream) {
  using namespace b2x;
  t_err[0] = 0;
  if (!is_float_type(type)) return fail(B2X_ERR_UNSUPPORTED, "b2x_moe_combine: type must be fp32, bf16 or fp16");
  if (tokens < 0 || cols < 0 || y_rows < 0 || top_k < 1 || ld_y < cols || ld_out < cols || (residual && ld_residual < cols))
    return fail(B2X_ERR_INVALID_ARG, "b2x_moe_combine: bad shape or row stride");
  if (tokens == 0 || cols == 0) return B2X_OK;
  if ((y_rows > 0 && !y) || !rows || !out) return fail(B2X_ERR_INVALID_ARG, "b2x_moe_combine: NULL pointer");
  const int elem = type == B2X_F32 ? 4 : 2;
  if (off_grid(y, elem) || off_grid(residual, elem) || off_grid(out, elem) || off_grid(rows, 4) || off_grid(weights, 4))
    return fail(B2X_ERR_INVALID_ARG, "b2x_moe_combine: misaligned pointer");
  CombineParams p{};
  p.y = y;
  p.y_rows = y_rows;
  p.ld_y = ld_y;
  p.rows = rows;
  p.weights = weights;
  p.tokens = tokens;
  p.cols = cols;
  p.k = top_k;
  p.residual = residual;
  p.ld_res = ld_residual;
  p.out = out;
  p.ld_out = ld_out;
  const bool vec = cols % (16 / elem) == 0 && rows_aligned(y, ld_y, elem) && rows_aligned(out, ld_out, elem) &&
                   (!residual || rows_aligned(residual, ld_residual, elem));
  const int64_t ctas = tokens * ((cols + kRowThreads - 1) / kRowThreads);
  if (ctas >= (1LL << 31)) return fail(B2X_ERR_UNSUPPORTED, "b2x_moe_combine: tokens * cols / 128 must be < 2^31");
  cudaError_t e = launch_combine<0>(p, type, vec, (cudaStream_t)stream);
  return e == cudaSuccess ? B2X_OK : cuda_fail(e, "b2x_moe_combine launch");
}

extern "C" B2X_API b2x_status b2x_moe_combine_backward(const void* grad, int64_t ld_grad, const void* y, int64_t y_rows,
                                                       int64_t ld_y, const int32_t* rows, const float* weights,
                                                       int64_t tokens, int top_k, int64_t cols, void* d_y,
                                                       int64_t ld_d_y, float* d_weights, b2x_dtype type, void* stream) {
  using namespace b2x;
  t_err[0] = 0;
  if (!is_float_type(type)) return fail(B2X_ERR_UNSUPPORTED, "b2x_moe_combine_backward: type must be fp32, bf16 or fp16");
  if (tokens < 0 || cols < 0 || y_rows < 0 || top_k < 1 || ld_y < cols || ld_grad < cols || ld_d_y < cols)
    return fail(B2X_ERR_INVALID_ARG, "b2x_moe_combine_backward: bad shape or row stride");
  if (tokens >= (1LL << 31)) return fail(B2X_ERR_UNSUPPORTED, "b2x_moe_combine_backward: tokens must be < 2^31");
  if (tokens == 0) return B2X_OK;
  if (!rows || !weights || !d_weights || (cols > 0 && (!grad || (y_rows > 0 && (!y || !d_y)))))
    return fail(B2X_ERR_INVALID_ARG, "b2x_moe_combine_backward: NULL pointer");
  const int elem = type == B2X_F32 ? 4 : 2;
  if (off_grid(grad, elem) || off_grid(y, elem) || off_grid(d_y, elem) || off_grid(rows, 4) || off_grid(weights, 4) || off_grid(d_weights, 4))
    return fail(B2X_ERR_INVALID_ARG, "b2x_moe_combine_backward: misaligned pointer");
  CombineParams p{};
  p.y = y;
  p.y_rows = y_rows;
  p.ld_y = ld_y;
  p.rows = rows;
  p.weights = weights;
  p.tokens = tokens;
  p.cols = cols;
  p.k = top_k;
  p.out = d_y;
  p.ld_out = ld_d_y;
  p.grad = grad;
  p.ld_grad = ld_grad;
  p.d_weights = d_weights;
  const bool vec = cols % (16 / elem) == 0 && rows_aligned(y, ld_y, elem) && rows_aligned(d_y, ld_d_y, elem) &&
                   rows_aligned(grad, ld_grad, elem);
  cudaError_t e = launch_combine<1>(p, type, vec, (cudaStream_t)stream);
  return e == cudaSuccess ? B2X_OK : cuda_fail(e, "b2x_moe_combine_backward launch");
}
