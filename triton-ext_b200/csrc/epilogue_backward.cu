// Backward pass of the GEMM epilogue for sm_100a: d_pre = grad * act'(pre) and d_bias[n] = sum_m d_pre[m, n].
//
// One pass: a thread owns one 16-byte run of columns (V values) and walks down rows, TX threads side by side and the
// rest of the CTA below one another; column sums stay in fp32 registers, meet in shared memory within the CTA and over
// distributed shared memory within a cluster of up to 8 CTAs that splits the rows.  Every sum has a fixed order, there
// is no workspace and no atomic.  The rows come through a ring in shared memory that each thread fills for itself ahead
// (cp.async): loads into registers left too few bytes on the way beside the slope's own registers.
// Bound: HBM, three times the matrix, and the instructions of the slope (gelu_tanh: HBM 71 %, issue slots 63 % of their peaks;
// gelu: the fp32 and the special function pipe 58 % each): 4000 x 28672 bf16 gelu_tanh 120 us (5.7 TB/s; with loads into
// registers 126, with single fp32 operations besides 248), gelu 146 us; 8192 x 1024 silu 11 us; 4000 x 28672 fp32, twice the
// bytes: gelu_tanh 226 us, gelu 221.  Columns that do not fill 16 bytes go one value at a time: 8192 x 1001 bf16 silu 26 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include "activations.cuh"
#include "b2x_internal.h"
#include "b2x_ptx.cuh"

namespace b2x {

constexpr int kEbThreads = 256;
constexpr int kEbUnroll = 2;  // rows of a stage
constexpr int kEbStages = 3;  // stages of the ring: 128 KB on the way per SM beside the one that is worked on

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

// The slope of values of type T, two at a time.
template <typename T, int ACT>
__device__ __forceinline__ Pair slope_of(Pair x) {
  if constexpr (sizeof(T) == 4 && (ACT == B2X_ACT_GELU_TANH || ACT == B2X_ACT_SILU)) {
    float a, b;
    unpair(x, a, b);
    return pair(act_slope_f32<ACT>(a), act_slope_f32<ACT>(b));
  } else {
    return act_slope<ACT>(x);
  }
}

// 16 bytes from global to shared memory, past L1 (d_pre may be grad or pre: a thread reads its values before it writes
// them, and no other thread touches them).
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Grid: x = column blocks * cluster size; the CTAs of a cluster share their columns and split the rows.
template <typename T, int V, int ACT, int TX>
__global__ void __launch_bounds__(kEbThreads, 4) epilogue_backward_kernel(const EpiBwdParams p, int splits) {
  constexpr int TY = kEbThreads / TX, U = kEbUnroll;
  // [stage][g and z of U rows][thread] on the way, and at the end the column sums [TY][TX * V + 1]
  extern __shared__ __align__(16) uint8_t eb_smem[];
  float (*part)[TX * V + 1] = reinterpret_cast<float (*)[TX * V + 1]>(eb_smem);
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
    if constexpr (V == 1) {
      constexpr int kRows = 8;  // in flight
      for (int64_t r = r0 + ty; r < r1; r += TY * kRows) {
        T gv[kRows], zv[kRows];
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
          const int64_t ru = r + (int64_t)u * TY;
          if (ru < r1) gv[u] = g[ru * p.ld_grad], zv[u] = ACT != B2X_ACT_NONE ? z[ru * p.ld_pre] : gv[u];
        }
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
          const int64_t ru = r + (int64_t)u * TY;
          if (ru < r1) {
            float d, none;
            unpair(slope_of<T, ACT>(pair(to_f32(zv[u]))), d, none);
            d *= to_f32(gv[u]);
            sum[0] += d;
            o[ru * p.ld_out] = from_f32<T>(d);
          }
        }
      }
    } else {
      // A thread copies its own pieces ahead (cp.async) and reads them back itself: no barrier.
      const uint32_t ring = smem_u32(eb_smem) + threadIdx.x * 16;
      auto slot = [&](int stage, int k) { return ring + (stage * 2 * U + k) * kEbThreads * 16; };
      auto fetch = [&](int64_t r, int stage) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t ru = r + (int64_t)u * TY;
          if (ru < r1) {
            copy_async16(slot(stage, 2 * u), g + ru * p.ld_grad);
            if (ACT != B2X_ACT_NONE) copy_async16(slot(stage, 2 * u + 1), z + ru * p.ld_pre);
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      int64_t ahead = r0 + ty;
#pragma unroll
      for (int s = 0; s < kEbStages - 1; ++s, ahead += TY * U) fetch(ahead, s);
      int stage = 0;
      for (int64_t r = r0 + ty; r < r1; r += TY * U, ahead += TY * U) {
        fetch(ahead, stage == 0 ? kEbStages - 1 : stage - 1);  // the stage that was read last
        asm volatile("cp.async.wait_group %0;" ::"n"(kEbStages - 1) : "memory");
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t ru = r + (int64_t)u * TY;
          if (ru >= r1) continue;
          const uint4 gw = ld_shared_u32x4(slot(stage, 2 * u));
          const uint4 zw = ACT != B2X_ACT_NONE ? ld_shared_u32x4(slot(stage, 2 * u + 1)) : gw;  // the slope 1 needs none
          Piece<T, V> gv, zv, ov;
          memcpy(&gv, &gw, 16);
          memcpy(&zv, &zw, 16);
#pragma unroll
          for (int i = 0; i < V; i += 2) {
            const Pair z2 = pair(to_f32(zv.e[i]), to_f32(zv.e[i + 1]));
            const Pair d2 = mul2(pair(to_f32(gv.e[i]), to_f32(gv.e[i + 1])), slope_of<T, ACT>(z2));
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
          uint4 w;
          memcpy(&w, &ov, 16);
          __stcs(reinterpret_cast<uint4*>(o + ru * p.ld_out), w);
        }
        stage = stage + 1 == kEbStages ? 0 : stage + 1;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
  }
  __syncthreads();  // the ring is done with
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
  constexpr int kSums = kEbThreads / TX * (TX * V + 1) * 4, kRing = V == 1 ? 0 : kEbStages * 2 * kEbUnroll * kEbThreads * 16;
  static_assert(kRing <= 48 << 10 && kSums <= 48 << 10, "shared memory without opting in");
  cfg.dynamicSmemBytes = kRing > kSums ? kRing : kSums;
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
  const int elem = type == B2X_F32 ? 4 : 2;
  if (off_grid(grad, elem) || off_grid(pre, elem) || off_grid(d_pre, elem) || off_grid(d_bias, 4))
    return fail(B2X_ERR_INVALID_ARG, "b2x_epilogue_backward: misaligned pointer");
  EpiBwdParams p{grad, ld_grad, pre, ld_pre, d_pre, ld_d_pre, d_bias, rows, cols};
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
