// Copies rows of bytes to rows that start on 16-byte boundaries, zeros behind the last byte: what TMA asks of operands
// whose row length is no multiple of 16.  A thread writes 16 bytes; inside a row it reads the five aligned words that hold
// them and shifts, at a row's ends it reads bytes, so nothing outside the row is touched.  Bound: HBM (one read, one write).
#include <cstdint>
#include "b2x_internal.h"

namespace b2x {

__global__ void __launch_bounds__(256) pad_rows_kernel(const uint8_t* __restrict__ src, int64_t ld_src, int64_t chunks,
                                                       uint32_t per_row, int64_t cols, uint8_t* __restrict__ dst, int64_t ld_dst) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= chunks) return;
  const int64_t r = chunks <= 0xffffffffll ? (uint32_t)i / per_row : i / per_row;
  const int64_t c = (i - r * per_row) * 16;
  const uint8_t* s = src + r * ld_src + c;
  uint32_t w[4] = {0, 0, 0, 0};
  if (c >= 4 && c + 20 <= cols) {
    const uint32_t off = (uint32_t)(uintptr_t)s & 3u;
    const uint32_t* a = reinterpret_cast<const uint32_t*>(s - off);
    uint32_t v[5];
#pragma unroll
    for (int j = 0; j < 5; ++j) v[j] = __ldcs(a + j);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(v[j], v[j + 1], 8 * off);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (c + j < cols) w[j >> 2] |= (uint32_t)s[j] << (8 * (j & 3));
  }
  *reinterpret_cast<uint4*>(dst + r * ld_dst + c) = make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace b2x

extern "C" B2X_API b2x_status b2x_pad_rows(const void* src, int64_t ld_src, int64_t rows, int64_t cols, void* dst,
                                           int64_t ld_dst, void* stream) {
  using namespace b2x;
  t_err[0] = 0;
  if (rows < 0 || cols < 0 || ld_src < cols || ld_dst < cols || ld_dst % 16 || (uintptr_t)dst % 16)
    return fail(B2X_ERR_INVALID_ARG, "b2x_pad_rows: needs ld >= cols, dst on a 16-byte boundary with ld_dst %% 16 == 0");
  if (rows == 0 || cols == 0) return B2X_OK;
  if (!src || !dst) return fail(B2X_ERR_INVALID_ARG, "b2x_pad_rows: NULL pointer");
  const int64_t per = (cols + 15) / 16;
  if (per >= (1LL << 31) || rows > ((1LL << 38) - 1) / per) return fail(B2X_ERR_UNSUPPORTED, "b2x_pad_rows: too large");
  const int64_t chunks = rows * per;
  pad_rows_kernel<<<(unsigned)((chunks + 255) / 256), 256, 0, (cudaStream_t)stream>>>(
      reinterpret_cast<const uint8_t*>(src), ld_src, chunks, (uint32_t)per, cols, reinterpret_cast<uint8_t*>(dst), ld_dst);
  note_launch(1);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? B2X_OK : cuda_fail(e, "b2x_pad_rows launch");
}
