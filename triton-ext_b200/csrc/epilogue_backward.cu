// Backward pass of the GEMM epilogue for sm_100a: d_pre = grad * act'(pre) and d_bias[n] = sum_m d_pre[m, n].
//
// One pass: a thread owns one 16-byte run of columns (V values) and walks down rows, TX threads side by side and the
// rest of the CTA below one another; column sums stay in fp32 registers, meet in shared memory within the CTA and over
// distributed shared memory within a cluster of up to 8 CTAs that splits the rows.  Every sum has a fixed order, there
// is no workspace and no atomic.  Bound: HBM, three times the matrix (4000 x 28672 bf16 without an activation: 89 us),
// and with an activation the instructions of its slope (gelu_tanh 126 us, gelu 158 us).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include "activations.cuh"
#include "b2x_internal.h"
#include "b2x_ptx.cuh"

namespace b2x {

constexpr int kEbThreads = 256;
constexpr int kEbUnroll = 2;  // rows in flight per thread (1 to 4 with 2 to 6 CTAs per SM: 126 us here, 145 to 275 elsewhere)

struct EpiBwdParams {
  const void* grad;
  int64_t ld_grad;
  const void* pre;
  int64_t ld_pre;
  void* out;
  int64_t ld_out;
  float* d_bias;
  int64_t rows, cols;
};

// Plain loads: d_pre may be grad or pre.
template <typename T, int V>
__device__ __forceinline__ Piece<T, V> load_plain(const T* p) {
  if constexpr (V == 1) {
    return Piece<T, V>{{*p}};
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    Piece<T, V> r;
    memcpy(&r, &u, 16);
    return r;
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_plain(T* p, const Piece<T, V>& v) {
  if constexpr (V == 1) {
    *p = v.e[0];
  } else {
    uint4 u;
    memcpy(&u, &v, 16);
    __stcs(reinterpret_cast<uint4*>(p), u);
  }
}

// Grid: x = column blocks * cluster size; the CTAs of a cluster share their columns and split the rows.
template <typename T, int V, int ACT, int TX>
__global__ void __launch_bounds__(kEbThreads, 4) epilogue_backward_kernel(const EpiBwdParams p, int splits) {
  constexpr int TY = kEbThreads / TX, kUnroll = V == 1 ? 8 : kEbUnroll;
  __shared__ float part[TY][TX * V + 1];
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  const int split = blockIdx.x % splits;
  const int64_t c = ((int64_t)(blockIdx.x / splits) * TX + tx) * V;
  const int64_t per = (p.rows + splits - 1) / splits;
  const int64_t r0 = per * split, r1 = r0 + per < p.rows ? r0 + per : p.rows;
  float sum[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = 0.0f;
  if (c < p.cols) {
    const T* g = reinterpret_cast<const T*>(p.grad) + c;
    const T* z = reinterpret_cast<const T*>(p.pre) + c;
    T* o = reinterpret_cast<T*>(p.out) + c;
    for (int64_t r = r0 + ty; r < r1; r += TY * kUnroll) {
      Piece<T, V> gv[kUnroll], zv[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int64_t ru = r + (int64_t)u * TY;
        if (ru < r1) {
          gv[u] = load_plain<T, V>(g + ru * p.ld_grad);
          zv[u] = load_plain<T, V>(z + ru * p.ld_pre);
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int64_t ru = r + (int64_t)u * TY;
        if (ru < r1) {
          Piece<T, V> ov;
          if constexpr (V == 1) {
            float d, none;
            unpair(act_slope<ACT>(pair(to_f32(zv[u].e[0]))), d, none);
            d *= to_f32(gv[u].e[0]);
            sum[0] += d;
            ov.e[0] = from_f32<T>(d);
          } else {
#pragma unroll
            for (int i = 0; i < V; i += 2) {
              const Pair z2 = pair(to_f32(zv[u].e[i]), to_f32(zv[u].e[i + 1]));
              const Pair d2 = mul2(pair(to_f32(gv[u].e[i]), to_f32(gv[u].e[i + 1])), act_slope<ACT>(z2));
              float a, b;
              unpair(add2(pair(sum[i], sum[i + 1]), d2), sum[i], sum[i + 1]);
              unpair(d2, a, b);
              if constexpr (__is_same(T, __nv_bfloat16)) {
                const uint32_t w = pack_bf16x2(a, b);
                memcpy(&ov.e[i], &w, 4);
              } else {
                ov.e[i] = from_f32<T>(a);
                ov.e[i + 1] = from_f32<T>(b);
              }
            }
          }
          store_plain<T, V>(o + ru * p.ld_out, ov);
        }
      }
    }
  }
  if (!p.d_bias) return;  // uniform over the grid
#pragma unroll
  for (int i = 0; i < V; ++i) part[ty][tx * V + i] = sum[i];
  __syncthreads();
  for (int i = threadIdx.x; i < TX * V; i += kEbThreads) {
    float s = 0.0f;
#pragma unroll 4
    for (int y = 0; y < TY; ++y) s += part[y][i];
    part[0][i] = s;
  }
  if (splits > 1) {
    cluster_sync();
    if (split == 0) {
      for (int i = threadIdx.x; i < TX * V; i += kEbThreads) {
        float s = 0.0f;
        for (int r = 0; r < splits; ++r) {
          float f;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(mapa_shared(smem_u32(&part[0][i]), r)) : "memory");
          s += f;
        }
        part[0][i] = s;
      }
    }
    cluster_sync();  // no CTA leaves while its sums may be read
    if (split != 0) return;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < TX * V; i += kEbThreads) {
    const int64_t n = (int64_t)(blockIdx.x / splits) * TX * V + i;
    if (n < p.cols) p.d_bias[n] = part[0][i];
  }
}

template <typename T, int V, int ACT, int TX>
static cudaError_t launch_epi_bwd_t(const EpiBwdParams& p, int num_sms, cudaStream_t st) {
  const int64_t blocks = (p.cols + TX * V - 1) / (TX * V);
  // Split the rows while the grid does not fill the GPU several times over and a CTA keeps a full round of rows.
  int splits = 1;
  while (splits < 8 && blocks * splits < 8 * num_sms && p.rows >= (int64_t)2 * splits * (kEbThreads / TX) * kEbUnroll) splits *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(blocks * splits), 1, 1);
  cfg.blockDim = dim3(kEbThreads, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, epilogue_backward_kernel<T, V, ACT, TX>, p, splits);
  note_launch(1);
  return e;
}

template <typename T, int ACT>
static cudaError_t launch_epi_bwd_act(const EpiBwdParams& p, bool vec, int num_sms, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  // Threads side by side: 32 for whole 512-byte runs, fewer where the column blocks, each split over at most 8 CTAs, would
  // not give every SM two (8192 x 1024 on 32: 82 us).
  if (!vec) return launch_epi_bwd_t<T, 1, ACT, 32>(p, num_sms, st);
  const int64_t runs = (p.cols + V - 1) / V;
  if (runs / 32 * 8 >= 2 * num_sms) return launch_epi_bwd_t<T, V, ACT, 32>(p, num_sms, st);
  if (runs / 8 * 8 >= 2 * num_sms) return launch_epi_bwd_t<T, V, ACT, 8>(p, num_sms, st);
  return launch_epi_bwd_t<T, V, ACT, 4>(p, num_sms, st);
}

template <typename T>
static cudaError_t launch_epi_bwd(const EpiBwdParams& p, b2x_activation act, bool vec, int num_sms, cudaStream_t st) {
  switch (act) {
    case B2X_ACT_RELU: return launch_epi_bwd_act<T, B2X_ACT_RELU>(p, vec, num_sms, st);
    case B2X_ACT_GELU: return launch_epi_bwd_act<T, B2X_ACT_GELU>(p, vec, num_sms, st);
    case B2X_ACT_GELU_TANH: return launch_epi_bwd_act<T, B2X_ACT_GELU_TANH>(p, vec, num_sms, st);
    case B2X_ACT_SILU: return launch_epi_bwd_act<T, B2X_ACT_SILU>(p, vec, num_sms, st);
    default: return launch_epi_bwd_act<T, B2X_ACT_NONE>(p, vec, num_sms, st);
  }
}

static bool valid_activation(int a) { return a >= B2X_ACT_NONE && a <= B2X_ACT_SILU; }

}  // namespace b2x

extern "C" B2X_API b2x_status b2x_epilogue_backward(const void* grad, int64_t ld_grad, const void* pre, int64_t ld_pre,
                                                    void* d_pre, int64_t ld_d_pre, float* d_bias, b2x_dtype type,
                                                    int64_t rows, int64_t cols, b2x_activation activation, void* stream) {
  using namespace b2x;
  t_err[0] = 0;
  if (!is_float_type(type)) return fail(B2X_ERR_UNSUPPORTED, "b2x_epilogue_backward: type must be fp32, bf16 or fp16");
  if (!valid_activation(activation)) return fail(B2X_ERR_INVALID_ARG, "b2x_epilogue_backward: unknown activation %d", (int)activation);
  if (rows < 0 || cols < 0 || ld_grad < cols || ld_pre < cols || ld_d_pre < cols)
    return fail(B2X_ERR_INVALID_ARG, "b2x_epilogue_backward: bad shape or row stride");
  if (cols == 0) return B2X_OK;
  if (cols >= (1LL << 31)) return fail(B2X_ERR_UNSUPPORTED, "b2x_epilogue_backward: cols must be < 2^31");
  if (rows == 0) {
    if (!d_bias) return B2X_OK;
    cudaError_t e = cudaMemsetAsync(d_bias, 0, (size_t)cols * 4, (cudaStream_t)stream);
    return e == cudaSuccess ? B2X_OK : cuda_fail(e, "b2x_epilogue_backward: clearing d_bias");
  }
  if (!grad || !pre || !d_pre) return fail(B2X_ERR_INVALID_ARG, "b2x_epilogue_backward: NULL pointer");
  EpiBwdParams p{grad, ld_grad, pre, ld_pre, d_pre, ld_d_pre, d_bias, rows, cols};
  const int elem = type == B2X_F32 ? 4 : 2;
  const bool vec = cols % (16 / elem) == 0 && rows_aligned(grad, ld_grad, elem) && rows_aligned(pre, ld_pre, elem) &&
                   rows_aligned(d_pre, ld_d_pre, elem);
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  const int sms = device_num_sms(dev);
  cudaStream_t st = (cudaStream_t)stream;
  if (type == B2X_F32)
    e = launch_epi_bwd<float>(p, activation, vec, sms, st);
  else if (type == B2X_F16)
    e = launch_epi_bwd<__half>(p, activation, vec, sms, st);
  else
    e = launch_epi_bwd<__nv_bfloat16>(p, activation, vec, sms, st);
  return e == cudaSuccess ? B2X_OK : cuda_fail(e, "b2x_epilogue_backward launch");
}
