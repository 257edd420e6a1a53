// fp8 products of a feed-forward layer for sm_100a, dense or one per expert over rows sorted by expert, with their
// epilogues (bias, activation, residual; SwiGLU and fp8).  Weight rows on the tensor core's 128-row side, tokens on its
// column side; see fp8_gemm_tokens.cuh.  The experts' row ranges are read on the device.
//
// fp8_gemm_tokens_kernel: one CTA per 128 weight rows x NT tokens x K range, two CTAs per SM (one's start and end hide
// behind the other's stream).  The K ranges of a tile are the CTAs of a cluster: each leaves its fp32 partial tile in its
// own shared memory and the cluster adds them over distributed shared memory in the order of the ranges, so there is no
// workspace, no atomic, nothing to clear, and the same inputs give the same bits.  For few tokens it is bound by reading
// the weights once: 1 x 8192 x 28672 in 42 us (5.6 TB/s), 40 rows on 64 experts of 7168 x 2048 in 71 to 75 us (5.9 TB/s).
#include <algorithm>
#include <cmath>
#include <cstdint>
#include "fp8_gemm_tokens.cuh"

namespace b2x {

constexpr int kTkThreads = 192;  // warps 0-3 read TMEM, warp 4 loads, warp 5 issues the MMAs
constexpr int kTkWarps = kTkThreads / 32;

template <int NT>
struct TkSmem {
  static constexpr int kWBytes = kTkRows * kBK;
  static constexpr int kXBytes = NT * kBK;
  static constexpr int kStageBytes = kWBytes + kXBytes;
  // two CTAs per SM: half of the shared memory each
  static constexpr int kStages = (kMaxDynSmem / 2 - 2048) / kStageBytes;
  static constexpr int kXOff = kStages * kWBytes;
  static constexpr int kBarOff = kStages * kStageBytes;
  static constexpr int kAlloc = kBarOff + (2 * kStages + 1) * 8 + 16 + 1024;
  static_assert(kStages * kStageBytes >= NT * kTkRows * 4, "the partial tile reuses the ring");
};

// Unit `unit` of the grid by one warp: experts in order, weight tiles of an expert, its token tiles innermost (so that
// the CTAs that share a weight tile run together).
template <int NT>
__device__ __forceinline__ TokUnit tok_find_unit(const TokParams& p, int unit, int lane) {
  TokUnit u{0, 0, 0, 0};
  if (!p.offsets) {
    const int mt = (int)((p.rows + NT - 1) / NT);
    u.nt = unit / mt;
    if (u.nt >= p.n_tiles) return u;
    u.row0 = (int64_t)(unit % mt) * NT;
    u.cnt = (int)min((int64_t)NT, p.rows - u.row0);
    return u;
  }
  int carry = 0;
  for (int base = 0; base < p.E; base += 32) {
    int64_t lo = 0, hi = 0;
    if (base + lane < p.E) tok_range(p, base + lane, lo, hi);
    const int mt = (int)((hi - lo + NT - 1) / NT);
    int s = mt * p.n_tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += v;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, unit < carry + s);
    if (past) {
      const int src = __ffs(past) - 1;
      const int local = unit - carry - s + mt * p.n_tiles;  // right on lane src
      const int m = mt ? local % mt : 0;
      u.e = base + src;
      u.nt = __shfl_sync(0xffffffffu, mt ? local / mt : 0, src);
      u.row0 = __shfl_sync(0xffffffffu, lo + (int64_t)m * NT, src);
      u.cnt = __shfl_sync(0xffffffffu, (int)min((int64_t)NT, hi - lo - (int64_t)m * NT), src);
      return u;
    }
    carry += __shfl_sync(0xffffffffu, s, 31);
  }
  return u;
}

// The 128 weight rows of tile nt, K block kb.  W_KIND 0: K-major [E][N, K]; 1: row-major [E][K, N]; 2: gate and up rows
// in turns of 16 (map {K, 16, gate / up, 8, blocks of 256 rows}).
template <int W_KIND>
__device__ __forceinline__ void tok_load_w(const TokParams& p, void* dst, const CUtensorMap* m, uint64_t* bar, int kb,
                                           int e, int nt, uint64_t pol) {
  if constexpr (W_KIND == 0)
    tma_load_3d(dst, m, bar, kb * kBK, nt * kTkRows, e, pol);
  else if constexpr (W_KIND == 1)
    tma_load_3d(dst, m, bar, nt * kTkRows, kb * kBK, e, pol);
  else
    tma_load_5d(dst, m, bar, kb * kBK, 0, 0, (nt & 1) * 4, e * (p.N / 256) + (nt >> 1), pol);
}

template <int NT, int W_KIND>
__global__ void __launch_bounds__(kTkThreads, 2)
    fp8_gemm_tokens_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                           const TokParams p) {
  using L = TkSmem<NT>;
  constexpr int S = L::kStages;
  constexpr uint32_t kTmemCols = NT < 32 ? 32 : NT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* empty = full + S;
  uint64_t* done = empty + S;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % p.splits;

  // every warp finds the unit itself: no shared memory, the same result in all CTAs of the cluster
  const TokUnit u = tok_find_unit<NT>(p, blockIdx.x / p.splits, lane);
  if (u.cnt == 0) return;  // the whole cluster leaves

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 4 && lane == 0) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int per = (p.k_tiles + p.splits - 1) / p.splits;
  const int k0 = min(rank * per, p.k_tiles), k1 = min(k0 + per, p.k_tiles);

  if (warp == 4) {
    if (lane == 0) {
      const uint64_t pol_w = l2_policy(p.l2_w), pol_x = policy_evict_last();
      int stage = 0;
      uint32_t phase = 0, issued = 0, pend[S];
      for (int kb = k0; kb < k1; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag, kStatusTimeoutProducer)) break;
        mbar_arrive_expect_tx(&full[stage], L::kStageBytes);
        tok_load_w<W_KIND>(p, smem + stage * L::kWBytes, &tmW, &full[stage], kb, u.e, u.nt, pol_w);
        tma_load_2d(smem + L::kXOff + stage * L::kXBytes, &tmX, &full[stage], kb * kBK, (int)u.row0, pol_x);
        issued |= 1u << stage;
        pend[stage] = phase;
        if (++stage == S) stage = 0, phase ^= 1;
      }
      for (int s = 0; s < S; ++s)
        if (issued & (1u << s)) {
          volatile int no_abort = 0;
          mbar_wait(&full[s], pend[s], &no_abort, kStatusTimeoutProducer);
        }
    }
  } else if (warp == 5) {
    if (lane == 0) {
      const uint32_t idesc = p.idesc | ((uint32_t)(NT >> 3) << 17);
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = k0; kb < k1; ++kb) {
        if (!mbar_wait(&full[stage], phase, abort_flag, kStatusTimeoutMma)) break;
        tc_fence_after();
        const uint32_t w = smem_u32(smem + stage * L::kWBytes), x = smem_u32(smem + L::kXOff + stage * L::kXBytes);
#pragma unroll
        for (int k = 0; k < kBK / 32; ++k)
          mma_f8f6f4(tmem_base,
                     W_KIND == 1 ? smem_desc_sw128(w + k * 32 * 128, 128 * kBK, 1024) : smem_desc_sw128(w + k * 32, 16, 1024),
                     smem_desc_sw128(x + k * 32, 16, 1024), idesc, (kb > k0 || k > 0) ? 1u : 0u);
        mma_commit(&empty[stage]);
        if (++stage == S) stage = 0, phase ^= 1;
      }
      mma_commit(done);
      volatile int no_abort = 0;
      mbar_wait(done, 0, &no_abort, kStatusTimeoutMma);
    }
  } else {
    // the finished partial tile -> shared memory [token][weight row], over the ring that nothing uses any more
    mbar_wait(done, 0, abort_flag, kStatusTimeoutEpilogue);
    __syncwarp();
    tc_fence_after();
    const uint32_t part = smem_u32(smem) + (warp * 32 + lane) * 4;
#pragma unroll
    for (int c0 = 0; c0 < NT; c0 += 16) {
      uint32_t v[16];
      tmem_ld_32x32b_x16(tmem_base + ((uint32_t)(warp * 32) << 16) + c0, v);
      tmem_ld_wait();
      tmem_regs_after_wait(v);
#pragma unroll
      for (int i = 0; i < 16; ++i) st_shared_f32(part + (c0 + i) * kTkRows * 4, k1 > k0 ? __uint_as_float(v[i]) : 0.0f);
    }
    tc_fence_before();
  }
  __syncwarp();
  if (p.splits > 1)
    cluster_sync();
  else
    __syncthreads();
  const uint32_t tile = smem_u32(smem);
  auto fetch4 = [&](int m, int col) {
    const uint32_t at = tile + (uint32_t)(m * kTkRows + col) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.splits == 1) {
      s = ld_shared_f32x4(at);
    } else {
      for (int r = 0; r < p.splits; ++r) {
        float4 f;
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w)
                     : "r"(mapa_shared(at, r))
                     : "memory");
        s.x += f.x, s.y += f.y, s.z += f.z, s.w += f.w;
      }
    }
    return s;
  };
  if constexpr (W_KIND == 2) {
    const float hs = __ldg(p.h_scale);
    const float inv = hs == 0.0f ? 0.0f : __fdiv_rn(1.0f, hs);
    float amax = 0.0f;
    tok_finish_swiglu(p, u.e, u.row0, u.nt * kTkRows, u.cnt, rank * kTkWarps + warp, p.splits * kTkWarps, lane, inv, amax, fetch4);
    if (p.h_amax) {
      const unsigned m = __reduce_max_sync(0xffffffffu, __float_as_uint(amax));
      if (lane == 0 && m) atomicMax(reinterpret_cast<unsigned*>(p.h_amax), m);
    }
  } else {
    const TokCols cols = tok_cols(p, u.e, u.nt * kTkRows, lane);
    for (int m = rank * kTkWarps + warp; m < u.cnt; m += p.splits * kTkWarps)
      tok_finish<1>(p, cols, u.row0 + m, 0, 1u, [&](int) { return fetch4(m, 4 * lane); });
  }
  __syncwarp();
  if (p.splits > 1)
    cluster_sync();  // peers may still read this CTA's partial tile
  else
    __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

// ---------------------------------------------------------------------------------------------------------------- pairs
//
// fp8_gemm_tokens_pair_kernel: the same products for many tokens, persistent, on CTA pairs (cta_group::2): a pair owns
// 256 weight rows x up to 256 tokens; CTA r holds weight rows 128 r .. 128 r + 127 of the tile in its TMEM and loads
// those rows and half of the tokens, 32 KB per CTA and K block where a single CTA's 128 x 256 tile needs 48 KB (no
// multicast).  The tile is as wide as its tokens need, in steps of 32.  Two accumulators let the two epilogue
// warpgroups of a CTA work behind the next tile's MMAs.  Roles as in fp8_gemm_pair.cu: warp 0 loads, warp 1 of the even
// CTA issues the MMAs, warp 2 allocates TMEM, warps 4-11 finish tiles.
//
// Units have unequal widths, so they are handed out by cluster launch control: one cluster per unit is launched, a
// running pair cancels clusters that have not started and takes their units.  Warp 3 of the even CTA asks, finds the
// unit's expert (it keeps 32 experts' ranges in its lanes, TokCursor) and passes the unit to both CTAs through a ring of
// four.  The other roles only read the ring: when each searched for its units itself, with the divisions and shuffles
// that takes, the loads and MMAs stood still for some 4000 cycles at every change of unit.
//
// Bound by the tensor cores under the power cap.  Measured (a few launches after an idle gap; back to back, at the clock that
// the cap leaves, the second takes 815 to 840 us and the experts' 600 to 620): 4000 x 28672 x 8192 in 689 us
// (the plain paired GEMM: 672), with bias, gelu_tanh and pre 739; 8192^3 in 402 (385); 20001 rows on 32 experts of
// 4096 x 7168 with SwiGLU in 511 us, of which the narrower tiles cost most: the time follows the columns, 64 to 256.

constexpr int kTpTokens = 256;    // tokens per unit
constexpr int kTpRing = 4;        // units handed out ahead
constexpr int kTpReaders = 2 + 1 + 16;  // warps that read the ring: loads of both CTAs, MMA, epilogues of both
constexpr int kTpBand = 16;       // token tiles whose X stays in L2 while the weight tiles go by

template <int STAGES>
struct TpSmem {
  static constexpr int kWBytes = kTkRows * kBK;               // 16 KB
  static constexpr int kXBytes = (kTpTokens / 2) * kBK;       // 16 KB
  static constexpr int kStageBytes = kWBytes + kXBytes;
  static constexpr int kCBytes = 2 * kTkChunk * kTkRows * 4;  // two steps of 8 KB per warpgroup
  static constexpr int kXOff = STAGES * kWBytes;
  static constexpr int kCOff = STAGES * kStageBytes;
  static constexpr int kBarOff = kCOff + 2 * kCBytes;
  static constexpr int kRingOff = (kBarOff + (2 * STAGES + 5) * 8 + 8 + 15) / 16 * 16;  // answers, barriers, units
  static constexpr int kAlloc = kRingOff + kTpRing * (2 * 16 + 3 * 8) + 1024;
};
constexpr int kTpStages = (kMaxDynSmem - 2 * TpSmem<1>::kCBytes - 1024 - 512) / TpSmem<1>::kStageBytes;

// Finds units, best in rising order; all lanes of a warp together.
struct TokCursor {
  int base, carry, total, s, mt, width;  // experts base .. base + 31; units before them, in them; lane's inclusive sum,
  int64_t lo, rows;                      // token tiles and their width; lane's range
};
__device__ __forceinline__ void tok_chunk(const TokParams& p, TokCursor& c, int n2, int lane) {
  c.lo = c.rows = 0;
  if (!p.offsets) {
    if (c.base + lane == 0) c.rows = p.rows;
  } else if (c.base + lane < p.E) {
    int64_t hi;
    tok_range(p, c.base + lane, c.lo, hi);
    c.rows = hi - c.lo;
  }
  c.mt = (int)((c.rows + kTpTokens - 1) / kTpTokens);
  c.width = c.mt ? (int)((c.rows + c.mt - 1) / c.mt + 31) / 32 * 32 : 0;  // (mt - 1) * width < rows: width <= 256
  c.s = c.mt * n2;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, c.s, o);
    if (lane >= o) c.s += v;
  }
  c.total = __shfl_sync(0xffffffffu, c.s, 31);
}
// The unit, or cnt = 0 past the last one.  nt: index of the 256-row weight tile.
__device__ __forceinline__ TokUnit tok_seek(const TokParams& p, TokCursor& c, int unit, int n2, int lane) {
  TokUnit u{0, 0, 0, 0};
  if (unit < c.carry) {
    c.base = c.carry = 0;
    tok_chunk(p, c, n2, lane);
  }
  while (unit >= c.carry + c.total) {
    if (c.base + 32 >= p.E) return u;
    c.base += 32;
    c.carry += c.total;
    tok_chunk(p, c, n2, lane);
  }
  const int src = __ffs(__ballot_sync(0xffffffffu, unit < c.carry + c.s)) - 1;
  const int mt = __shfl_sync(0xffffffffu, c.mt, src);
  const int local = unit - c.carry - (__shfl_sync(0xffffffffu, c.s, src) - mt * n2);
  const int64_t lo = __shfl_sync(0xffffffffu, c.lo, src), rows = __shfl_sync(0xffffffffu, c.rows, src);
  const int band = local / (kTpBand * n2);
  const int width = min(kTpBand, mt - band * kTpBand);
  const int r = local - band * kTpBand * n2;
  const int m = band * kTpBand + r % width;
  u.e = c.base + src;
  u.nt = r / width;
  const int tokens = __shfl_sync(0xffffffffu, c.width, src);
  u.row0 = lo + (int64_t)m * tokens;
  u.cnt = (int)min((int64_t)tokens, rows - (int64_t)m * tokens);
  return u;
}
template <int W_KIND>
__device__ __forceinline__ void tok_load_w_pair(const TokParams& p, void* dst, const CUtensorMap* m, uint32_t bar, int kb,
                                                int e, int nt, uint64_t pol) {
  if constexpr (W_KIND == 0)
    tma_load_3d_pair(dst, m, bar, kb * kBK, nt * kTkRows, e, pol);
  else if constexpr (W_KIND == 1)
    tma_load_3d_pair(dst, m, bar, nt * kTkRows, kb * kBK, e, pol);
  else
    tma_load_5d_pair(dst, m, bar, kb * kBK, 0, 0, (nt & 1) * 4, e * (p.N / 256) + (nt >> 1), pol);
}

template <int W_KIND>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_gemm_tokens_pair_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                                const __grid_constant__ CUtensorMap tmXs, const TokParams p) {
  constexpr int STAGES = kTpStages;
  using L = TpSmem<STAGES>;
  static_assert(L::kAlloc <= kMaxDynSmem, "shared memory plan exceeds the opt-in limit");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* mma_done = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint8_t* answer = smem + L::kRingOff;
  uint8_t* units = answer + kTpRing * 16;
  uint64_t* answered = reinterpret_cast<uint64_t*>(units + kTpRing * 16);
  uint64_t* ufull = answered + kTpRing;
  uint64_t* uempty = ufull + kTpRing;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kTpRing; ++s) {
      mbar_init(&answered[s], 1);
      mbar_init(&ufull[s], 1);
      mbar_init(&uempty[s], kTpReaders);  // the even CTA's is used
    }
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 2);
    }
    mbar_init(mma_done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmXs);
  }
  if (warp == 2) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // The next unit from the ring (`at` counts the reads); cnt = 0: none.  Whole warps.
  auto next_unit = [&](int& at) {
    const int s = at % kTpRing;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (mbar_wait_cluster(&ufull[s], (uint32_t)(at / kTpRing) & 1u, abort_flag, kStatusTimeoutProducer))
      v = ld_shared_u32x4(smem_u32(units + s * 16));
    __syncwarp();
    if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&uempty[s]), 0));
    ++at;
    TokUnit u;
    u.e = (int)v.x;
    u.nt = (int)v.y;
    u.row0 = (int)v.z;
    u.cnt = (int)__shfl_sync(0xffffffffu, v.w, 0);  // one answer for the warp, even where a lane gave up
    return u;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ loads (both CTAs)
    const uint64_t pol_w = l2_policy(p.l2_w), pol_x = policy_evict_last();
    int stage = 0;
    uint32_t phase = 0, issued = 0, pend = 0;  // pend: bit s = phase of stage s's last load
    bool ok = true;
    int at = 0;
    while (ok) {
      const TokUnit u = next_unit(at);
      if (u.cnt == 0) break;
      if (lane == 0) {
        const int half = (u.cnt + 31) / 32 * 16;  // tokens per CTA
        const CUtensorMap* mx = half > 64 ? &tmX : &tmXs;       // boxes of 128 or 64 tokens
        const uint32_t bytes = 2 * (L::kWBytes + (half > 64 ? 128 : 64) * kBK);
        const int x0 = (int)u.row0 + (int)rank * half;
        for (int kb = 0; kb < p.k_tiles; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag, kStatusTimeoutProducer)) {
            ok = false;
            break;
          }
          const uint32_t bar = mapa_shared(smem_u32(&full[stage]), 0);
          if (leader) mbar_arrive_expect_tx(&full[stage], bytes);
          tok_load_w_pair<W_KIND>(p, smem + stage * L::kWBytes, &tmW, bar, kb, u.e, 2 * u.nt + (int)rank, pol_w);
          tma_load_2d_pair(smem + L::kXOff + stage * L::kXBytes, mx, bar, kb * kBK, x0, pol_x);
          issued |= 1u << stage;
          pend = (pend & ~(1u << stage)) | (phase << stage);
          if (++stage == STAGES) stage = 0, phase ^= 1;
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
    }
    // the even CTA's full barriers count both CTAs' loads: none is in flight once they have completed
    if (leader && lane == 0)
      for (int s = 0; s < STAGES; ++s)
        if (issued & (1u << s)) {
          volatile int no_abort = 0;
          mbar_wait(&full[s], (pend >> s) & 1, &no_abort, kStatusTimeoutProducer);
        }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMAs (even CTA)
    if (leader) {
      const uint64_t desc_w = smem_desc_sw128(smem_u32(smem), W_KIND == 1 ? 128 * kBK : 16, 1024);
      const uint64_t desc_x = smem_desc_sw128(smem_u32(smem + L::kXOff), 16, 1024);
      int stage = 0, at = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int local = 0; ok; ++local) {
        const TokUnit u = next_unit(at);
        if (u.cnt == 0) break;
        if (lane == 0) {
          const int buf = local & 1;
          const uint32_t idesc = p.idesc | ((uint32_t)((u.cnt + 31) / 32 * 4) << 17);
          ok = mbar_wait(&tempty[buf], ((local >> 1) & 1) ^ 1, abort_flag, kStatusTimeoutMma);
          tc_fence_after();
          const uint32_t d = tmem_base + buf * kTpTokens;
          for (int kb = 0; ok && kb < p.k_tiles; ++kb) {
            if (!mbar_wait(&full[stage], phase, abort_flag, kStatusTimeoutMma)) {
              ok = false;
              break;
            }
            tc_fence_after();
            // the address fields of both descriptors move by constants: one addition each per MMA
            const uint64_t w = desc_w + (uint32_t)stage * (L::kWBytes >> 4), x = desc_x + (uint32_t)stage * (L::kXBytes >> 4);
            mma_f8f6f4_pair(d, w, x, idesc, kb > 0 ? 1u : 0u);
#pragma unroll
            for (int k = 1; k < kBK / 32; ++k)
              mma_f8f6f4_pair(d, w + k * ((W_KIND == 1 ? 32 * 128 : 32) >> 4), x + k * (32 >> 4), idesc, 1u);
            mma_commit_pair_mc(&empty[stage], 0x3);
            if (++stage == STAGES) stage = 0, phase ^= 1;
          }
          if (ok) mma_commit_pair_mc(&tfull[buf], 0x3);
        }
        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
      }
      if (lane == 0) {
        mma_commit_pair_mc(mma_done, 0x1);
        volatile int no_abort = 0;
        mbar_wait(mma_done, 0, &no_abort, kStatusTimeoutMma);
      }
    }
  } else if (warp == 3) {
    // ------------------------------------------------------------ units (even CTA)
    if (leader) {
      const int n2 = (p.n_tiles + 1) / 2;
      TokCursor cur{0, 0, 0, 0, 0, 0, 0, 0};
      tok_chunk(p, cur, n2, lane);
      int put = 0;
      for (int unit = blockIdx.x >> 1, asked = 0;; ++asked) {
        const int r = asked % kTpRing;
        if (lane == 0 && unit >= 0) {  // ask for the one after it, then pass this one on
          fence_proxy_async_smem();
          mbar_arrive_expect_tx(&answered[r], 16);
          clc_try_cancel(answer + r * 16, &answered[r]);
        }
        const TokUnit u = unit >= 0 ? tok_seek(p, cur, unit, n2, lane) : TokUnit{0, 0, 0, 0};
        int next = -1;
        if (lane == 0) {
          if (u.cnt > 0 || unit < 0) {  // clusters past the last unit are only taken out of the way
            const int s = put % kTpRing;
            if (mbar_wait_cluster(&uempty[s], ((uint32_t)(put / kTpRing) & 1u) ^ 1u, abort_flag, kStatusTimeoutProducer))
              for (uint32_t c = 0; c < 2; ++c) {
                st_cluster_v4(mapa_shared(smem_u32(units + s * 16), c), make_int4(u.e, u.nt, (int)u.row0, u.cnt));
                mbar_arrive_cluster(mapa_shared(smem_u32(&ufull[s]), c));
              }
            ++put;
          }
          if (unit >= 0) {
            volatile int no_abort = 0;
            if (mbar_wait(&answered[r], (uint32_t)(asked / kTpRing) & 1u, &no_abort, kStatusTimeoutProducer)) {
              const int cta = clc_first_ctaid_x(answer + r * 16);
              next = cta < 0 ? -1 : cta >> 1;
            }
          }
        }
        if (unit < 0) break;
        unit = __shfl_sync(0xffffffffu, next, 0);
      }
    }
  } else if (warp >= kEpiWarp0) {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int e = (warp - kEpiWarp0) >> 2, q = warp & 3;
    const uint32_t bar_id = 1 + e;
    const int wg_tid = threadIdx.x - (kEpiWarp0 + 4 * e) * 32;
    const uint32_t stage_c = smem_u32(smem + L::kCOff + e * L::kCBytes);
    const uint32_t tempty_leader = mapa_shared(smem_u32(&tempty[e]), 0);
    float inv = 0.0f, amax = 0.0f;
    if constexpr (W_KIND == 2) {
      const float hs = __ldg(p.h_scale);
      inv = hs == 0.0f ? 0.0f : __fdiv_rn(1.0f, hs);
    }
    int at = 0;
    for (int local = 0;; ++local) {
      const TokUnit u = next_unit(at);
      if (u.cnt == 0) break;
      if ((local & 1) != e) continue;
      const uint32_t t_row = tmem_base + e * kTpTokens + ((uint32_t)(q * 32) << 16);
      const int n0 = (2 * u.nt + (int)rank) * kTkRows;
      const int chunks = (u.cnt + kTkChunk - 1) / kTkChunk;
      auto release = [&]() {  // all 128 threads have read the accumulator
        if (wg_tid == 0) mbar_arrive_cluster_relaxed(tempty_leader);
      };
      auto ready = [&]() {
        const bool ok = mbar_wait(&tfull[e], (local >> 1) & 1, abort_flag, kStatusTimeoutEpilogue);
        const bool all = wg_all(ok, bar_id);
        tc_fence_after();
        return all;
      };
      if constexpr (W_KIND == 2) {
        // Lanes 0-15 hold gate rows, lanes 16-31 the up rows of the same 16 columns of h.  Of two neighbouring tokens a
        // gate lane hands the second's value over and an up lane the first's: each then has gate and up of one token.
        // The tile's codes, [256 tokens][64 bytes], fill the staging; one barrier, then whole 64-byte rows leave.
        const float sw = tok_scale_w(p, u.e);
        const float fmax = p.h_e5m2 ? 57344.0f : 448.0f;
        const int odd = lane >> 4;
        if (!ready()) break;
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
          uint32_t v[kTkChunk];
          tmem_ld_32x32b_x16(t_row + c * kTkChunk, v);
          // lane l: the factor of token l of the step
          const int m0 = min(c * kTkChunk + (lane & 15), u.cnt - 1);
          const float alpha = tok_alpha(p, u.row0 + m0, sw);
          tmem_ld_wait();
          tmem_regs_after_wait(v);
#pragma unroll
          for (int i = 0; i < kTkChunk / 2; ++i) {
            const float a = __uint_as_float(v[2 * i]), b = __uint_as_float(v[2 * i + 1]);
            const float other = __shfl_xor_sync(0xffffffffu, odd ? a : b, 16);
            const float h = tok_swiglu(odd ? other : a, odd ? b : other, __shfl_sync(0xffffffffu, alpha, 2 * i + odd));
            const int m = c * kTkChunk + 2 * i + odd;
            if (m < u.cnt) amax = fmaxf(amax, fabsf(h));
            const float y = swiglu_clamp(__fmul_rn(h, inv), fmax);
            st_shared_u8(stage_c + m * 64 + q * 16 + (lane & 15), p.h_e5m2 ? cvt_e5m2x2(y, 0.0f) : cvt_e4m3x2(y, 0.0f));
          }
        }
        tc_fence_before();
        named_bar_sync(bar_id, 128);
        release();
        for (int i = wg_tid; i < u.cnt * 4; i += 128)
          __stcs(reinterpret_cast<uint4*>(p.h + (u.row0 + (i >> 2)) * p.ld_h + n0 / 2 + (i & 3) * 16),
                 ld_shared_u32x4(stage_c + i * 16));
      } else {
        const TokCols cols = tok_cols(p, u.e, n0, lane);
        const bool fast = n0 + kTkRows <= p.N && p.vec_out && (!p.residual || p.vec_res) && (!p.pre || p.vec_pre);
        const int kind = !fast ? 16 : (p.half ? 8 : 0) + (p.act ? 4 : 0) + (p.residual ? 2 : 0) + (p.pre ? 1 : 0);
        if (!ready()) break;
        switch (kind) {
#define B2X_TILE(H, A, R, P)                                                                                              \
  case 8 * H + 4 * A + 2 * R + P:                                                                                         \
    tok_tile<H, A, R, P>(p, cols, t_row, u.row0, u.cnt, q, lane, stage_c, bar_id, release);                               \
    break;
          B2X_TILE(0, 0, 0, 0) B2X_TILE(0, 0, 0, 1) B2X_TILE(0, 0, 1, 0) B2X_TILE(0, 0, 1, 1)
          B2X_TILE(0, 1, 0, 0) B2X_TILE(0, 1, 0, 1) B2X_TILE(0, 1, 1, 0) B2X_TILE(0, 1, 1, 1)
          B2X_TILE(1, 0, 0, 0) B2X_TILE(1, 0, 0, 1) B2X_TILE(1, 0, 1, 0) B2X_TILE(1, 0, 1, 1)
          B2X_TILE(1, 1, 0, 0) B2X_TILE(1, 1, 0, 1) B2X_TILE(1, 1, 1, 0) B2X_TILE(1, 1, 1, 1)
#undef B2X_TILE
          default:  // the last columns, or rows off the 8-byte grid: one step at a time, every access checked
#pragma unroll 1
            for (int c = 0; c < chunks; ++c) {
              uint32_t v[kTkChunk];
              tmem_ld_32x32b_x16(t_row + c * kTkChunk, v);
              tmem_ld_wait();
              tmem_regs_after_wait(v);
              const uint32_t buf = stage_c + (c & 1) * kTkChunk * kTkRows * 4;
#pragma unroll
              for (int i = 0; i < kTkChunk; ++i) st_shared_f32(buf + (i * kTkRows + q * 32 + lane) * 4, __uint_as_float(v[i]));
              tc_fence_before();
              named_bar_sync(bar_id, 128);
              if (c + 1 == chunks) release();
              const int left = u.cnt - c * kTkChunk - q;
              const uint32_t live = (left > 0 ? 1u : 0u) | (left > 4 ? 2u : 0u) | (left > 8 ? 4u : 0u) | (left > 12 ? 8u : 0u);
              tok_finish<4>(p, cols, u.row0 + c * kTkChunk + q, 4, live,
                            [&](int i) { return ld_shared_f32x4(buf + ((q + 4 * i) * kTkRows + 4 * lane) * 4); });
            }
        }
      }
      named_bar_sync(bar_id, 128);  // the next tile writes the staging again
    }
    if constexpr (W_KIND == 2) {
      if (p.h_amax) {
        const unsigned m = __reduce_max_sync(0xffffffffu, __float_as_uint(amax));
        if (lane == 0 && m) atomicMax(reinterpret_cast<unsigned*>(p.h_amax), m);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync();  // no CTA leaves while its peer may still use its shared memory or barriers
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

struct TokLaunch {
  CUtensorMap tmW;
  TokParams p;
  const void* x;
  int64_t ld_x;
  int w_kind, w_fmt, x_fmt;
  int num_sms;
};

template <int NT, int W_KIND>
static cudaError_t launch_tokens_t(const TokLaunch& g, const CUtensorMap& tmX, int64_t units, cudaStream_t st) {
  using L = TkSmem<NT>;
  auto kern = fp8_gemm_tokens_kernel<NT, W_KIND>;
  cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kern), L::kAlloc);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * g.p.splits), 1, 1);
  cfg.blockDim = dim3(kTkThreads, 1, 1);
  cfg.dynamicSmemBytes = L::kAlloc;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = g.p.splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, g.tmW, tmX, g.p);
  note_launch(1);
  return e;
}

template <int NT>
static cudaError_t launch_tokens_nt(const TokLaunch& g, const CUtensorMap& tmX, int64_t units, cudaStream_t st) {
  if (g.w_kind == 0) return launch_tokens_t<NT, 0>(g, tmX, units, st);
  if (g.w_kind == 1) return launch_tokens_t<NT, 1>(g, tmX, units, st);
  return launch_tokens_t<NT, 2>(g, tmX, units, st);
}

template <int W_KIND>
static cudaError_t launch_tokens_pair_t(const TokLaunch& g, const CUtensorMap (&tmX)[2], int64_t units, cudaStream_t st) {
  using L = TpSmem<kTpStages>;
  auto kern = fp8_gemm_tokens_pair_kernel<W_KIND>;
  cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kern), L::kAlloc);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = L::kAlloc;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3((unsigned)(2 * units), 1, 1);  // one cluster per unit
  e = cudaLaunchKernelEx(&cfg, kern, g.tmW, tmX[0], tmX[1], g.p);
  note_launch(1);
  return e;
}

// Experts that get a row when `rows` fall on E experts evenly: what the grid is planned for.
static double expected_active(int64_t rows, int64_t E) { return (double)E * (1.0 - pow(1.0 - 1.0 / (double)E, (double)rows)); }

static b2x_status launch_tokens(TokLaunch& g, const char* who, cudaStream_t st) {
  TokParams& p = g.p;
  const bool moe = p.offsets != nullptr;
  const double active = moe ? expected_active(p.rows, p.E) : 1.0;
  const double mean = (double)p.rows / active;
  // Pairs or single CTAs.  Up to 32 tokens per product the weights are all there is to read, and the short single-CTA
  // tiles do that best (64 experts x 7168 x 2048, 40 rows: 80 us against 91 us on pairs; 2048 rows: 181 and 179).  Above,
  // pairs win where their units fill the GPU: twice up to 96 tokens (8 experts x 4096 x 4096, 512 rows, 128 units: 30.5
  // and 34.5; 32 experts x 4096 x 7168, 2048 rows, 512 units: 184 and 165), half of it for wider tiles, whose work per
  // byte is twice that of the single CTAs' (256 x 8192 x 8192, 32 units: 25.9 and 29.7; 384 rows, 64 units: 47.6 and 31.9).
  const int pairs = g.num_sms / 2;
  const double mean256 = ceil(mean / kTpTokens);
  const double units2 = std::max(1.0, moe ? active * mean256 : mean256) * ((p.n_tiles + 1) / 2);
  const bool pair = mean > 96 ? units2 >= pairs / 2 : (mean > 32 && units2 >= 2 * pairs);
  if (pair) {
    const int64_t most = (moe ? p.rows / kTpTokens + std::min<int64_t>(p.E, p.rows) : (p.rows + kTpTokens - 1) / kTpTokens) *
                         ((p.n_tiles + 1) / 2);
    if (2 * most >= (1LL << 31)) return fail(B2X_ERR_UNSUPPORTED, "%s: too many tiles", who);
    p.idesc = idesc_f8f6f4(g.w_fmt, g.x_fmt, g.w_kind == 1 ? 1 : 0, 0, 2 * kTkRows, 0);
    p.l2_w = 0;
    CUtensorMap tmX[2];
    for (int i = 0; i < 2; ++i) {
      b2x_status s = encode_2d(&tmX[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, g.x, (uint64_t)p.K, (uint64_t)p.rows,
                               (uint64_t)g.ld_x, 128, i ? 64 : 128, CU_TENSOR_MAP_SWIZZLE_128B, "x");
      if (s != B2X_OK) return s;
    }
    cudaError_t e = g.w_kind == 0   ? launch_tokens_pair_t<0>(g, tmX, most, st)
                    : g.w_kind == 1 ? launch_tokens_pair_t<1>(g, tmX, most, st)
                                    : launch_tokens_pair_t<2>(g, tmX, most, st);
    return e == cudaSuccess ? B2X_OK : cuda_fail(e, who);
  }
  // Token tile: the mean expert fits with room for an uneven spread.
  int nt = 128;
  if (mean <= (moe ? 10 : 16)) nt = 16;
  else if (mean <= (moe ? 20 : 32)) nt = 32;
  else if (mean <= (moe ? 48 : 64)) nt = 64;
  // Most units that any spread of the rows can give (sum of ceil(c / nt)); those past the last leave at once.
  const int64_t tok_tiles = moe ? p.rows / nt + std::min<int64_t>(p.E, p.rows) : (p.rows + nt - 1) / nt;
  const int64_t units = tok_tiles * p.n_tiles;
  const double planned = std::max(1.0, moe ? active * ceil(mean / nt) : (double)tok_tiles) * p.n_tiles;
  // K ranges: none if the tiles reach every SM, else the fewest that do, but 8 only where 4 give fewer than 64 CTAs (a little
  // under half of the SMs): a larger cluster costs more to place and to add up (1 x 28672 x 8192, 224 tiles: 42 us with one
  // range, 44, 52 and 60 with 2, 4 and 8; 1 x 8192 x 8192, 64 tiles: 23, 14.5, 11.2, 16; 1 x 1024 x 16384, 8 tiles: 41, 23,
  // 13.8, 9.5).
  p.splits = 1;
  while (p.splits < 8 && planned * p.splits < g.num_sms) {
    const int s = 2 * p.splits, per = (p.k_tiles + s - 1) / s;
    if (per < 4 || (int64_t)(s - 1) * per >= p.k_tiles) break;  // short ranges, or an empty one
    if (s == 8 && planned * 4 >= 64) break;
    p.splits = s;
  }
  if (units * p.splits >= (1LL << 31)) return fail(B2X_ERR_UNSUPPORTED, "%s: too many tiles", who);
  p.idesc = idesc_f8f6f4(g.w_fmt, g.x_fmt, g.w_kind == 1 ? 1 : 0, 0, kTkRows, 0);
  // Weights that one token tile reads, or the few token tiles of an expert side by side, and that fill more than half of L2,
  // leave it first: they would only push out what the next kernels read (in turn on one GPU: 1 x 8192 x 28672 41.5 and
  // 39.6 us, 40 rows over 64 experts of 7168 x 2048 75 and 71, two token tiles of 250 rows on an expert of 4096 x 28672 39.1 and
  // 35.4; GPUs differ by as much).  Smaller ones may still be there at the next call (1 x 1024 x 16384, 16 MB: 9.3 us, and
  // 10.0 if they leave first).
  const double weights = (moe ? std::max(1.0, active) : 1.0) * p.n_tiles * kTkRows * (double)p.K;
  p.l2_w = (moe || tok_tiles == 1) && weights > 64e6 ? 2 : 1;
  CUtensorMap tmX;
  b2x_status s = encode_2d(&tmX, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.x, (uint64_t)p.K, (uint64_t)p.rows, (uint64_t)g.ld_x, 128,
                           (uint32_t)nt, CU_TENSOR_MAP_SWIZZLE_128B, "x");
  if (s != B2X_OK) return s;
  cudaError_t e = nt == 16   ? launch_tokens_nt<16>(g, tmX, units, st)
                  : nt == 32 ? launch_tokens_nt<32>(g, tmX, units, st)
                  : nt == 64 ? launch_tokens_nt<64>(g, tmX, units, st)
                             : launch_tokens_nt<128>(g, tmX, units, st);
  return e == cudaSuccess ? B2X_OK : cuda_fail(e, who);
}

// Tensor map of the weights, [E][N, K] by strides; see tok_load_w for the kinds.
static b2x_status encode_weights(CUtensorMap* m, int kind, const void* w, int64_t E, int64_t N, int64_t K, int64_t ld_e,
                                 int64_t ld) {
  auto fn = get_encode_fn();
  if (!fn) return fail(B2X_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  cuuint32_t es[5] = {1, 1, 1, 1, 1};
  CUresult r;
  if (kind == 2) {
    cuuint64_t dims[5] = {(cuuint64_t)K, 16, 2, 8, (cuuint64_t)(E * (N / 256))};
    cuuint64_t strides[4] = {(cuuint64_t)ld, (cuuint64_t)ld * 128, (cuuint64_t)ld * 16, (cuuint64_t)ld * 256};
    cuuint32_t box[5] = {128, 16, 2, 4, 1};
    r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, const_cast<void*>(w), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  } else {
    cuuint64_t dims[3] = {(cuuint64_t)(kind ? N : K), (cuuint64_t)(kind ? K : N), (cuuint64_t)E};
    cuuint64_t strides[2] = {(cuuint64_t)ld, (cuuint64_t)(E > 1 ? ld_e : ld * (kind ? K : N))};
    cuuint32_t box[3] = {128, 128, 1};
    r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(w), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  }
  if (r != CUDA_SUCCESS)
    return fail(B2X_ERR_INVALID_ARG, "cuTensorMapEncodeTiled(weights) failed with %d (experts %lld, N %lld, K %lld)", (int)r,
                (long long)E, (long long)N, (long long)K);
  return B2X_OK;
}

// Rows of 16-bit values that start on 8-byte boundaries.
static bool even_rows(const void* p, int64_t ld) { return ((uintptr_t)p % 8) == 0 && ld % 4 == 0; }

static int b2x_device_sms(const char* who, b2x_status& s) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  s = e == cudaSuccess ? B2X_OK : cuda_fail(e, who);
  return s == B2X_OK ? device_num_sms(dev) : 0;
}

// Checks and translation shared by b2x_moe_gemm and b2x_moe_gemm_swiglu.
static b2x_status moe_gemm_params(const b2x_moe_gemm_args* a, const char* who, bool swiglu, TokLaunch& g) {
  if (!a) return fail(B2X_ERR_INVALID_ARG, "%s: args is NULL", who);
  if (!is_fp8(a->x_type) || !is_fp8(a->w_type)) return fail(B2X_ERR_UNSUPPORTED, "%s: x and w must be e4m3 or e5m2", who);
  if (a->rows < 0 || a->K < 0 || a->N < 0 || a->experts < 1)
    return fail(B2X_ERR_INVALID_ARG, "%s: bad shape (rows %lld, N %lld, K %lld, experts %lld)", who, (long long)a->rows,
                (long long)a->N, (long long)a->K, (long long)a->experts);
  if (a->rows >= (1LL << 31) || a->K >= (1LL << 31) || a->N >= (1LL << 31) || a->experts > 1024)
    return fail(B2X_ERR_UNSUPPORTED, "%s: dimensions must be < 2^31, experts at most 1024", who);
  if (a->rows == 0 || a->N == 0) return B2X_OK;
  if (a->K == 0) return fail(B2X_ERR_UNSUPPORTED, "%s: K == 0", who);
  if (!a->x || !a->w || !a->offsets) return fail(B2X_ERR_INVALID_ARG, "%s: NULL x, w or offsets", who);
  if (a->ld_x < a->K || a->ld_x % 16 || (uintptr_t)a->x % 16)
    return fail(B2X_ERR_INVALID_ARG, "%s: x must be 16-byte aligned with ld_x >= K and ld_x %% 16 == 0", who);
  int64_t ld;
  if (a->ldw_k == 1 && a->ldw_n >= a->K) {
    g.w_kind = 0;
    ld = a->ldw_n;
  } else if (a->ldw_n == 1 && a->ldw_k >= a->N) {
    g.w_kind = 1;
    ld = a->ldw_k;
  } else {
    return fail(B2X_ERR_INVALID_ARG, "%s: w strides (%lld, %lld) are not K-major or row-major", who, (long long)a->ldw_n,
                (long long)a->ldw_k);
  }
  if (ld % 16 || (uintptr_t)a->w % 16 || (a->experts > 1 && (a->ldw_e % 16 || a->ldw_e < 0)))
    return fail(B2X_ERR_INVALID_ARG, "%s: w must be 16-byte aligned with strides that are multiples of 16", who);
  if ((a->scale_x && a->scale_x_count != 1 && a->scale_x_count != a->rows) ||
      (a->scale_w && a->scale_w_count != 1 && a->scale_w_count != a->experts))
    return fail(B2X_ERR_INVALID_ARG, "%s: scale_x has one element or one per row, scale_w one or one per expert", who);
  if (off_grid(a->offsets, 4) || off_grid(a->scale_x, 4) || off_grid(a->scale_w, 4))
    return fail(B2X_ERR_INVALID_ARG, "%s: misaligned pointer", who);
  if (swiglu) {
    if (g.w_kind != 0) return fail(B2X_ERR_UNSUPPORTED, "%s: w must be K-major", who);
    if (a->N % 256) return fail(B2X_ERR_UNSUPPORTED, "%s: N (gate + up rows) must be a multiple of 256", who);
    if (a->experts > 1 && a->ldw_e != a->N * ld)
      return fail(B2X_ERR_UNSUPPORTED, "%s: the experts' weights must lie one after the other (ldw_e = N * ldw_n)", who);
    g.w_kind = 2;
  }
  b2x_status s;
  g.num_sms = b2x_device_sms(who, s);
  if (s != B2X_OK) return s;
  s = encode_weights(&g.tmW, g.w_kind, a->w, a->experts, a->N, a->K, a->ldw_e, ld);
  if (s != B2X_OK) return s;
  g.x = a->x;
  g.ld_x = a->ld_x;
  g.w_fmt = a->w_type == B2X_E4M3 ? 0 : 1;
  g.x_fmt = a->x_type == B2X_E4M3 ? 0 : 1;
  TokParams& p = g.p;
  p.N = (int)a->N;
  p.K = (int)a->K;
  p.E = (int)a->experts;
  p.rows = a->rows;
  p.offsets = a->offsets;
  p.n_tiles = (int)((a->N + kTkRows - 1) / kTkRows);
  p.k_tiles = (int)((a->K + kBK - 1) / kBK);
  p.scale_x = a->scale_x;
  p.scale_w = a->scale_w;
  p.sx_mode = !a->scale_x ? 0 : (a->scale_x_count == 1 && a->rows != 1 ? 1 : 2);
  p.sw_mode = !a->scale_w ? 0 : (a->scale_w_count == 1 ? 1 : 2);
  return B2X_OK;
}

}  // namespace b2x

extern "C" B2X_API b2x_status b2x_moe_gemm(const b2x_moe_gemm_args* a, void* y, b2x_dtype y_type, int64_t ld_y, void* stream) {
  using namespace b2x;
  t_err[0] = 0;
  if (y_type != B2X_BF16 && y_type != B2X_F16) return fail(B2X_ERR_UNSUPPORTED, "b2x_moe_gemm: y must be bf16 or fp16");
  TokLaunch g{};
  b2x_status s = moe_gemm_params(a, "b2x_moe_gemm", false, g);
  if (s != B2X_OK || a->rows == 0 || a->N == 0) return s;
  if (!y || ld_y < a->N || (uintptr_t)y % 2) return fail(B2X_ERR_INVALID_ARG, "b2x_moe_gemm: NULL y or ld_y < N");
  g.p.out = reinterpret_cast<uint16_t*>(y);
  g.p.ld_out = ld_y;
  g.p.half = y_type == B2X_F16;
  g.p.vec_out = even_rows(y, ld_y);
  return launch_tokens(g, "b2x_moe_gemm launch", (cudaStream_t)stream);
}

extern "C" B2X_API b2x_status b2x_moe_gemm_swiglu(const b2x_moe_gemm_args* a, void* h, b2x_dtype h_type, int64_t ld_h,
                                                  const float* h_scale, float* h_amax, void* stream) {
  using namespace b2x;
  t_err[0] = 0;
  if (!is_fp8(h_type)) return fail(B2X_ERR_UNSUPPORTED, "b2x_moe_gemm_swiglu: h must be e4m3 or e5m2");
  TokLaunch g{};
  b2x_status s = moe_gemm_params(a, "b2x_moe_gemm_swiglu", true, g);
  if (s != B2X_OK || a->rows == 0 || a->N == 0) return s;
  if (!h || ld_h < a->N / 2 || ld_h % 16 || (uintptr_t)h % 16)
    return fail(B2X_ERR_INVALID_ARG, "b2x_moe_gemm_swiglu: h must be 16-byte aligned with ld_h >= N/2 and ld_h %% 16 == 0");
  if (!h_scale) return fail(B2X_ERR_INVALID_ARG, "b2x_moe_gemm_swiglu: NULL h_scale");
  if (off_grid(h_scale, 4) || off_grid(h_amax, 4)) return fail(B2X_ERR_INVALID_ARG, "b2x_moe_gemm_swiglu: misaligned pointer");
  g.p.h = reinterpret_cast<uint8_t*>(h);
  g.p.ld_h = ld_h;
  g.p.h_e5m2 = h_type == B2X_E5M2;
  g.p.h_scale = h_scale;
  g.p.h_amax = h_amax;
  return launch_tokens(g, "b2x_moe_gemm_swiglu launch", (cudaStream_t)stream);
}

extern "C" B2X_API b2x_status b2x_fp8_gemm_epilogue(const b2x_gemm_args* a, const b2x_epilogue* ep, void* stream) {
  using namespace b2x;
  t_err[0] = 0;
  if (!a || !ep) return fail(B2X_ERR_INVALID_ARG, "b2x_fp8_gemm_epilogue: NULL argument");
  if (!is_fp8(a->a_type) || !is_fp8(a->b_type)) return fail(B2X_ERR_UNSUPPORTED, "b2x_fp8_gemm_epilogue: A and B must be e4m3 or e5m2");
  if (a->c_type != B2X_BF16 && a->c_type != B2X_F16) return fail(B2X_ERR_UNSUPPORTED, "b2x_fp8_gemm_epilogue: C must be bf16 or fp16");
  if (a->M < 0 || a->N < 0 || a->K < 0) return fail(B2X_ERR_INVALID_ARG, "b2x_fp8_gemm_epilogue: negative shape");
  if (a->M >= (1LL << 31) || a->N >= (1LL << 31) || a->K >= (1LL << 31))
    return fail(B2X_ERR_UNSUPPORTED, "b2x_fp8_gemm_epilogue: dimensions must be < 2^31");
  if (!valid_activation(ep->activation))
    return fail(B2X_ERR_INVALID_ARG, "b2x_fp8_gemm_epilogue: unknown activation %d", (int)ep->activation);
  if (ep->bias && !is_float_type(ep->bias_type))
    return fail(B2X_ERR_UNSUPPORTED, "b2x_fp8_gemm_epilogue: bias must be fp32, bf16 or fp16");
  if (a->scale_mode != B2X_SCALE_NONE && a->scale_mode != B2X_SCALE_TENSOR && a->scale_mode != B2X_SCALE_TENSOR_GIVEN)
    return fail(B2X_ERR_UNSUPPORTED, "b2x_fp8_gemm_epilogue: takes per-tensor scales or none");
  if (a->M == 0 || a->N == 0) return B2X_OK;
  if (a->K == 0) return fail(B2X_ERR_UNSUPPORTED, "b2x_fp8_gemm_epilogue: K == 0");
  if (!a->a || !a->b || !a->c) return fail(B2X_ERR_INVALID_ARG, "b2x_fp8_gemm_epilogue: NULL A, B or C");
  if (a->scale_mode != B2X_SCALE_NONE && (!a->scale_a || !a->scale_b))
    return fail(B2X_ERR_INVALID_ARG, "b2x_fp8_gemm_epilogue: NULL scale pointer");
  if (a->lda < a->K || a->lda % 16 || (uintptr_t)a->a % 16)
    return fail(B2X_ERR_INVALID_ARG, "b2x_fp8_gemm_epilogue: A must be 16-byte aligned with lda >= K and lda %% 16 == 0");
  TokLaunch g{};
  int64_t ld;
  if (a->ldb_k == 1 && a->ldb_n >= a->K) {
    g.w_kind = 0;
    ld = a->ldb_n;
  } else if (a->ldb_n == 1 && a->ldb_k >= a->N) {
    g.w_kind = 1;
    ld = a->ldb_k;
  } else {
    return fail(B2X_ERR_INVALID_ARG, "b2x_fp8_gemm_epilogue: B strides (%lld, %lld) are not K-major or row-major",
                (long long)a->ldb_k, (long long)a->ldb_n);
  }
  if (ld % 16 || (uintptr_t)a->b % 16)
    return fail(B2X_ERR_INVALID_ARG, "b2x_fp8_gemm_epilogue: B needs 16-byte alignment and a row stride %% 16 == 0");
  if (a->ldc < a->N || (uintptr_t)a->c % 2 || (ep->residual && ep->ld_residual < a->N) || (ep->pre && ep->ld_pre < a->N))
    return fail(B2X_ERR_INVALID_ARG, "b2x_fp8_gemm_epilogue: row strides of C, residual and pre must be >= N");
  if (off_grid(ep->residual, 2) || off_grid(ep->pre, 2) || off_grid(ep->bias, ep->bias_type == B2X_F32 ? 4 : 2) ||
      (a->scale_mode != B2X_SCALE_NONE && (off_grid(a->scale_a, 4) || off_grid(a->scale_b, 4))))
    return fail(B2X_ERR_INVALID_ARG, "b2x_fp8_gemm_epilogue: misaligned pointer");
  b2x_status s;
  g.num_sms = b2x_device_sms("b2x_fp8_gemm_epilogue", s);
  if (s != B2X_OK) return s;
  s = encode_weights(&g.tmW, g.w_kind, a->b, 1, a->N, a->K, 0, ld);
  if (s != B2X_OK) return s;
  g.x = a->a;
  g.ld_x = a->lda;
  g.w_fmt = a->b_type == B2X_E4M3 ? 0 : 1;
  g.x_fmt = a->a_type == B2X_E4M3 ? 0 : 1;
  TokParams& p = g.p;
  p.N = (int)a->N;
  p.K = (int)a->K;
  p.E = 1;
  p.rows = a->M;
  p.n_tiles = (int)((a->N + kTkRows - 1) / kTkRows);
  p.k_tiles = (int)((a->K + kBK - 1) / kBK);
  if (a->scale_mode != B2X_SCALE_NONE) {
    p.scale_x = a->scale_a;
    p.scale_w = a->scale_b;
    p.sx_mode = p.sw_mode = 1;
  }
  p.half = a->c_type == B2X_F16;
  p.bias = ep->bias;
  p.bias_type = ep->bias_type;
  p.act = ep->activation;
  p.residual = reinterpret_cast<const uint16_t*>(ep->residual);
  p.ld_res = ep->ld_residual;
  p.vec_res = even_rows(ep->residual, ep->ld_residual);
  p.out = reinterpret_cast<uint16_t*>(a->c);
  p.ld_out = a->ldc;
  p.vec_out = even_rows(a->c, a->ldc);
  p.pre = reinterpret_cast<uint16_t*>(ep->pre);
  p.ld_pre = ep->ld_pre;
  p.vec_pre = even_rows(ep->pre, ep->ld_pre);
  return launch_tokens(g, "b2x_fp8_gemm_epilogue launch", (cudaStream_t)stream);
}
