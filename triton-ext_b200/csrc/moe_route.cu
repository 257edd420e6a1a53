// Expert routing for sm_100a: scores, balance bias, groups, top-k and renormalised weights of a mixture of experts, and
// the gradient of the weights.
//
// One warp owns a token; lane l holds the logits of experts VPL l .. VPL l + VPL - 1 in registers, so a row is read once
// and a group of experts is a run of lanes.  Bound: HBM for many tokens (tokens * experts logits in), latency for few; in
// between the instructions of the selection, so that takes few.  Choices become order-preserving 32-bit keys.  The
// (k + 2)-th largest of the 32 lanes' maxima (redux.sync) is a bound that at least k + 2 keys reach and few more; those
// (almost always at most 32) are packed one to a lane in the order of their index, and each counts the better ones.  Where
// more than 32 reach the bound the choices are taken one after the other instead.  What bounds the kernel is how fast
// instructions issue (16384 x 256: 78 % of the issue slots, the integer pipe 56 %, HBM 8 %): comparisons and selections.
//
// What is compared.  Without a bias s is monotone in the logit, so the logits themselves are the keys and the choice is
// exact.  With a bias (and for sums of two) the keys are fp32 values of s + b.  s is off by at most err = 2^-20 (sigmoid) or
// (VPL + 31) 2^-24 max s.  In u = 2^-24, e^-d is off by (4 + 3 d) u of itself: 2^-22 of the instruction, the rest its
// argument's roundings.  sigma: s (1 - s) (4 + 3 |l|) u < 2 u, the sum and the reciprocal 3 u.  Softmax: the largest by 4 u, the
// sum by 4 u and 3 u of the mean distance from the maximum, at most 5 for 1024 experts (N of them at d: N d e^-d / (1 + N e^-d)),
// quotient and product by 2 u, and VPL + 5 additions.  s + b is rounded once, by u of it.  A row in which two neighbours of the
// order a, b lie closer than 2 err + 2^-23 (|a| + |b|), or in which a group that goes may be off by as much as sets it
// behind one that stays (2 err and 2^-24 of its two choices and of their sum, each), is settled in fp64: the groups alone
// (groups_exact), the candidates' order alone (rank_exact), or, where neither will do, the whole choice (choose_exact).  It is
// right to fp64, at the speed of fp32 for nearly all rows (16384 tokens, 256 experts, k = 8, sigmoid: the fp64 pipe is busy
// 0.007 % of the time; settling all doubtful rows by choose_exact took 7 us more).
//
// Measured, 16384 tokens, k = 8, 64 / 128 / 256 / 384 experts: softmax 10.1 / 10.8 / 12.5 / 14.0 us; sigmoid, bias, 8 groups by
// their two largest 18 / 21 / 26 / 32 us.  8 tokens: 2.8 to 4.5 us, launch and latency.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cfloat>
#include <cstdint>
#include "activations.cuh"
#include "b2x_internal.h"
#include "b2x_ptx.cuh"

namespace b2x {

constexpr int kRouteWarps = 4;  // tokens per CTA
constexpr uint32_t kAll = 0xffffffffu;

struct RouteParams {
  const void* logits;
  int64_t ld;
  int64_t tokens;
  int type, E, k;
  int sigmoid, renorm, groups, top_groups, top2;
  int lanes_per_group;  // where a group is a run of 2^n whole lanes, else 0
  int vec, vec_b;       // logits' rows, the biases allow 4-value loads
  float scale;
  const float* bias;
  float* weights;
  int32_t* indices;
  // backward
  const float* d_weights;
  void* d_logits;
  int64_t ld_d;
  int vec_d;
};

// Unsigned order of floats: masked (-inf) 0, then rising, NaN on top; -0 and +0 are one value (the addition also makes
// every NaN the one positive pattern).
constexpr uint32_t kNegInf = 0x007fffffu;              // -inf with its bits turned over
constexpr uint32_t kNaN = 0xffffffffu - kNegInf;
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);
  return (u ^ ((uint32_t)((int)u >> 31) | 0x80000000u)) - kNegInf;
}
__device__ __forceinline__ float key_value(uint32_t k) {  // of a key that is neither masked nor NaN
  const uint32_t u = k + kNegInf;
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {  // of numbers; NaN is ignored
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
  return v;
}

// Weights are fp32 results: unlike the scores that are only compared (and settled in fp64 where they are close) they are made
// with the library's exponential and true divisions, one or two a lane and row.
// e^(a - b), a <= b, with what the difference loses put back in first order.
__device__ __forceinline__ float exp_diff(float a, float b) {
  const float d = a - b, bb = d - a, lost = (a - (d - bb)) - (b + bb);
  const float e = expf(d);
  return d < -104.0f ? 0.0f : fmaf(e, lost, e);
}
__device__ __forceinline__ float sigma(float l) {
  const float e = expf(-fabsf(l));
  return __fdiv_rn(l < 0.0f ? e : 1.0f, 1.0f + e);
}

// sigma(l) of the chosen experts (l = -inf: none), for its quotient by their sum.  sigma(l) is e^l sigma(-l): where all are
// negative the common factor e^max is left out, so that logits of -90 or -600 give the weights that they give in 64 bits
// instead of quotients of zeros.  Below kSigmaGone even 1 / (1 + e^-l) in 64 bits is 0 (logits of the type's lowest value): 0.
constexpr float kSigmaGone = -709.78f;
__device__ __forceinline__ float sigma_parts(float l) {
  const bool there = l != -INFINITY;
  if (__any_sync(kAll, l >= 0.0f)) return there ? sigma(l) : 0.0f;
  const float top = warp_max(l);  // -inf where all are NaN
  if (!there) return 0.0f;
  return top < kSigmaGone ? 0.0f * l : __fdiv_rn(exp_diff(l, top), 1.0f + expf(l));
}

// The largest (value, lowest index) pair of the warp, in fp64; index INT_MAX: none.
__device__ __forceinline__ void warp_argmax(double& v, int& at) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const double v2 = __shfl_xor_sync(kAll, v, o);
    const int a2 = __shfl_xor_sync(kAll, at, o);
    if (v2 > v || (v2 == v && a2 < at)) v = v2, at = a2;
  }
}

// VPL consecutive logits of a row as fp32; past the last expert -inf.
template <int VPL>
__device__ __forceinline__ void load_logits(const RouteParams& p, int64_t row, int lane, float (&l)[VPL]) {
  const int e0 = lane * VPL;
  const int bytes = p.type == B2X_F32 ? 4 : 2;
  if (VPL % 4 == 0 && p.vec && e0 + VPL <= p.E) {
    const char* src = reinterpret_cast<const char*>(p.logits) + (row + e0) * bytes;
    if (p.type == B2X_F32) {
#pragma unroll
      for (int i = 0; i < VPL / 4; ++i) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(src) + i);
        l[4 * i] = f.x, l[4 * i + 1] = f.y, l[4 * i + 2] = f.z, l[4 * i + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < VPL / 4; ++i) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(src) + i);
        const uint32_t w[2] = {u.x, u.y};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (p.type == B2X_BF16) {
            l[4 * i + 2 * j] = bf16lo(w[j]), l[4 * i + 2 * j + 1] = bf16hi(w[j]);
          } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
            l[4 * i + 2 * j] = f.x, l[4 * i + 2 * j + 1] = f.y;
          }
        }
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i) l[i] = e0 + i < p.E ? load_f32(p.logits, row + e0 + i, p.type) : -INFINITY;
}

// Whether the lane's group stays, from fp64 scores of its experts: groups that are runs of 2^n lanes, the two largest by
// exchanges, the rank by counting the better groups.
template <int VPL>
__device__ __forceinline__ bool keep_exact(const RouteParams& p, const double (&s)[VPL], const bool (&off)[VPL], int lane) {
  double a1 = -INFINITY, a2 = -INFINITY;
  int n = 0;  // how many there are, up to two
#pragma unroll
  for (int i = 0; i < VPL; ++i)
    if (!off[i]) {
      if (n == 0 || s[i] > a1) a2 = a1, a1 = s[i];
      else if (n == 1 || s[i] > a2) a2 = s[i];
      n = min(n + 1, 2);
    }
  for (int o = 1; o < p.lanes_per_group; o <<= 1) {
    const double b1 = __shfl_xor_sync(kAll, a1, o), b2 = __shfl_xor_sync(kAll, a2, o);
    const int bn = __shfl_xor_sync(kAll, n, o);
    const double hi = fmax(a1, b1), lo = fmin(a1, b1);
    a2 = fmax(lo, fmax(a2, b2));
    a1 = hi;
    n = min(n + bn, 2);
  }
  const double score = p.top2 && n == 2 ? a1 + a2 : a1;
  const int g = lane / p.lanes_per_group;
  int better = 0;
  for (int i = 0; i < p.groups; ++i) {
    const double other = __shfl_sync(kAll, score, i * p.lanes_per_group);
    const int there = __shfl_sync(kAll, n, i * p.lanes_per_group);
    better += there > 0 && (other > score || (other == score && i < g));
  }
  return n > 0 && g < p.groups && better < p.top_groups;
}

// fp64 scores of the lane's experts: s, and which of them are masked.
template <int VPL>
__device__ __forceinline__ void scores_exact(const RouteParams& p, const float (&l)[VPL], int e0, double (&s)[VPL], bool (&off)[VPL]) {
  double m = 0.0, sum = 0.0;
  if (!p.sigmoid) {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < VPL; ++i) top = fmaxf(top, l[i]);
    m = (double)warp_max(top);
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    s[i] = p.sigmoid ? 1.0 / (1.0 + exp(-(double)l[i])) : exp((double)l[i] - m);
    if (l[i] == -INFINITY) s[i] = 0.0;
    sum += s[i];
  }
  if (!p.sigmoid) sum = warp_sum(sum);
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const float b = p.bias && e0 + i < p.E ? p.bias[e0 + i] : 0.0f;
    if (!p.sigmoid) s[i] /= sum;
    s[i] += (double)b;
    off[i] = e0 + i >= p.E || l[i] == -INFINITY || b == -INFINITY;
    if (s[i] != s[i]) s[i] = INFINITY;
  }
}

// The lane's group once more, where fp32 cannot tell the last group that stays from the first that goes.
template <int VPL>
__device__ __noinline__ bool groups_exact(const RouteParams& p, int64_t row, int lane) {
  float l[VPL];
  double s[VPL];
  bool off[VPL];
  load_logits<VPL>(p, row, lane, l);
  scores_exact<VPL>(p, l, lane * VPL, s, off);
  return keep_exact<VPL>(p, s, off, lane);
}

// The choice in fp64 (rows with values next to a border): lane j < k gets its expert or -1.
template <int VPL>
__device__ __noinline__ int choose_exact(const RouteParams& p, int64_t row, int lane) {
  float l[VPL];  // read again: an array handed over would live in memory for every row
  load_logits<VPL>(p, row, lane, l);
  double c[VPL], s[VPL];  // what experts are chosen by; s + b, what groups are scored by
  bool off[VPL];
  const int gs = p.E / p.groups, e0 = lane * VPL;
  scores_exact<VPL>(p, l, e0, s, off);
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    c[i] = p.bias ? s[i] : (double)l[i];
    if (c[i] != c[i]) c[i] = INFINITY;
  }
  if (p.groups > 1 && p.lanes_per_group) {
    const bool kept = keep_exact<VPL>(p, s, off, lane);
#pragma unroll
    for (int i = 0; i < VPL; ++i) off[i] = off[i] || !kept;
  } else if (p.groups > 1) {
    // lane keeps the scores of the groups VPL lane .. (groups <= experts <= 32 VPL)
    double gv[VPL];
    bool kept[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) gv[i] = -INFINITY, kept[i] = false;
    for (int g = 0; g < p.groups; ++g) {
      double total = 0.0;
      bool any = false;
      int skip = -1;
      const int lo = g * gs - e0, hi = lo + gs;
      for (int round = 0; round < (p.top2 ? 2 : 1); ++round) {
        double v = -INFINITY;
        int at = 0x7fffffff;
#pragma unroll
        for (int i = 0; i < VPL; ++i)
          if (!off[i] && i >= lo && i < hi && e0 + i != skip && (s[i] > v || at == 0x7fffffff)) v = s[i], at = e0 + i;
        warp_argmax(v, at);
        if (at != 0x7fffffff) total += v, any = true, skip = at;
      }
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (e0 + i == g && any) gv[i] = total;
    }
    for (int n = 0; n < p.top_groups; ++n) {
      double v = -INFINITY;
      int at = 0x7fffffff;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (e0 + i < p.groups && gv[i] > v) v = gv[i], at = e0 + i;
      warp_argmax(v, at);
      if (at == 0x7fffffff) break;
      const int lo = at * gs - e0, hi = lo + gs;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        if (e0 + i == at) gv[i] = -INFINITY;
        if (i >= lo && i < hi) kept[i] = true;
      }
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) off[i] = off[i] || !kept[i];
  }
  int mine = -1;
  for (int j = 0; j < p.k; ++j) {
    double v = -INFINITY;
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (!off[i] && (c[i] > v || at == 0x7fffffff)) v = c[i], at = e0 + i;
    warp_argmax(v, at);
    if (at == 0x7fffffff) break;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (e0 + i == at) off[i] = true;
    if (lane == j) mine = at;
  }
  return mine;
}

// The order of the warp's candidates (lane < n: expert `at`) in fp64: the lane's rank.
template <int VPL>
__device__ __noinline__ int rank_exact(const RouteParams& p, int64_t row, int lane, int at, bool have) {
  double m = 0.0, sum = 1.0;
  if (!p.sigmoid) {
    float l[VPL];
    load_logits<VPL>(p, row, lane, l);
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < VPL; ++i) top = fmaxf(top, l[i]);
    m = (double)warp_max(top);
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (l[i] != -INFINITY) sum += exp((double)l[i] - m);
    sum = warp_sum(sum);
  }
  double c = -INFINITY;
  if (have) {
    const double x = (double)load_f32(p.logits, row + at, p.type);
    c = (p.sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - m) / sum) + (double)p.bias[at];
    if (c != c) c = INFINITY;
  }
  const int n = __popc(__ballot_sync(kAll, have));
  int better = 0;
  for (int j = 0; j < n; ++j) {
    const double other = __shfl_sync(kAll, c, j);
    const int other_at = __shfl_sync(kAll, at, j);
    better += other > c || (other == c && other_at < at);
  }
  return better;
}

// Largest key of the warp and the lowest index that has it (the lanes hold rising runs of indexes).
template <int VPL>
__device__ __forceinline__ uint32_t take_max(const uint32_t (&key)[VPL], int lane, int& at) {
  uint32_t best = 0;
#pragma unroll
  for (int i = 0; i < VPL; ++i) best = max(best, key[i]);
  best = __reduce_max_sync(kAll, best);
  int e = 0x7fffffff;
#pragma unroll
  for (int i = VPL - 1; i >= 0; --i)
    if (key[i] == best) e = lane * VPL + i;
  at = __shfl_sync(kAll, e, __ffs(__ballot_sync(kAll, e != 0x7fffffff)) - 1);
  return best;
}

// Biases of VPL consecutive experts; past the last one 0.
template <int VPL>
__device__ __forceinline__ void load_bias(const RouteParams& p, int e0, float (&b)[VPL]) {
  if (VPL % 4 == 0 && p.vec_b && e0 + VPL <= p.E) {
#pragma unroll
    for (int i = 0; i < VPL / 4; ++i) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(p.bias + e0) + i);
      b[4 * i] = f.x, b[4 * i + 1] = f.y, b[4 * i + 2] = f.z, b[4 * i + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i) b[i] = e0 + i < p.E ? __ldg(p.bias + e0 + i) : 0.0f;
  }
}

template <int VPL>
__global__ void __launch_bounds__(kRouteWarps * 32, VPL <= 8 ? 10 : (VPL <= 16 ? 8 : 4)) moe_route_kernel(const __grid_constant__ RouteParams p) {
  __shared__ __align__(16) uint32_t pack_key[kRouteWarps][32];
  __shared__ int pack_at[kRouteWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = (int64_t)blockIdx.x * kRouteWarps + warp;
  if (t >= p.tokens) return;
  const int64_t row = t * p.ld;
  const int e0 = lane * VPL;
  float l[VPL];
  load_logits<VPL>(p, row, lane, l);

  float m = -INFINITY, sum = 1.0f;
  const bool values = p.bias || (p.groups > 1 && p.top2);  // choices or group scores are sums of rounded numbers
  const bool need_sum = !p.sigmoid && (values || !p.renorm);
  if (need_sum) {
    bool nan = false;
#pragma unroll
    for (int i = 0; i < VPL; ++i) m = fmaxf(m, l[i]), nan |= l[i] != l[i];
    m = warp_max(m);
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) sum += l[i] == -INFINITY ? 0.0f : exp_approx(l[i] - m);
    sum = warp_sum(sum);
    if (__any_sync(kAll, nan)) sum = NAN;
  }
  uint32_t key[VPL], gkey[VPL];  // what experts are chosen by, what groups are scored by
  float err = 0.0f;
  if (values) {
    const float inv = p.sigmoid ? 0.0f : __fdiv_rn(1.0f, sum);  // also the largest s
    err = p.sigmoid ? 0x1p-20f : (VPL + 31) * 0x1p-24f * inv;
    float b[VPL];
    if (p.bias) load_bias<VPL>(p, e0, b);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const float s = p.sigmoid ? sigma_fast(l[i]) : exp_approx(l[i] - m) * inv;
      gkey[i] = order_key(l[i] == -INFINITY || (p.bias && b[i] == -INFINITY) ? -INFINITY : (p.bias ? s + b[i] : s));
      key[i] = p.bias ? gkey[i] : order_key(l[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i) gkey[i] = key[i] = order_key(l[i]);
  }
  auto near = [&](uint32_t a, uint32_t b) {  // a >= b, both numbers
    const float x = key_value(a), y = key_value(b);
    return !(x - y > fmaf(0x1p-23f, fabsf(x) + fabsf(y), 2.0f * err));
  };
  // A group's score from the keys of its two best choices, and how far it may be off: each s by err, each s + b and the sum
  // of the two by 2^-24 of itself, however little of them the sum leaves (doubled, for the roundings of the limits below).
  auto group_score = [&](uint32_t a, uint32_t b, float& slack) -> uint32_t {
    if (!values || a == 0) return a;
    if (a == kNaN) return kNaN;  // b is not above a
    const float x = key_value(a), y = p.top2 && b != 0 ? key_value(b) : 0.0f;
    slack = fmaf(0x1p-22f, fabsf(x) + fabsf(y), 2.0f * err);
    return p.top2 && b != 0 ? order_key(fmaxf(x + y, -FLT_MAX)) : a;  // two of the lowest value are no masked group
  };
  constexpr uint32_t kTop = 0xffffffffu;
  auto lowest = [&](uint32_t score, float slack) { return score == kNaN ? kTop : order_key(fmaxf(key_value(score) - slack, -FLT_MAX)); };
  auto highest = [&](uint32_t score, float slack) { return score == kNaN ? kTop : order_key(key_value(score) + slack); };
  // Whether a group that goes may belong before one that stays: `last` is the least of what those may be that stay, `next`
  // the most of the others (0: there is none; kTop: NaN alone, told apart by their index).
  auto border = [&](uint32_t last, uint32_t next) { return next != 0 && next != kTop && last != kTop && last <= next; };
  bool close = false;  // something to be told apart in fp64
  if (p.groups > 1) {
    const int gs = p.E / p.groups;
    if (p.lanes_per_group) {
      // a group is a run of 2^n lanes: its two largest by n exchanges, its rank by counting the better groups
      uint32_t a = 0, b = 0;
#pragma unroll
      for (int i = 0; i < VPL; ++i) b = max(b, min(a, gkey[i])), a = max(a, gkey[i]);
      for (int o = 1; o < p.lanes_per_group; o <<= 1) {
        const uint32_t a2 = __shfl_xor_sync(kAll, a, o);
        if (p.top2) b = max(min(a, a2), max(b, __shfl_xor_sync(kAll, b, o)));
        a = max(a, a2);
      }
      float slack = 0.0f;
      const uint32_t score = group_score(a, b, slack);
      const int g = lane / p.lanes_per_group;
      int better = 0;
      for (int i = 0; i < p.groups; ++i) {
        const uint32_t other = __shfl_sync(kAll, score, i * p.lanes_per_group);
        better += other > score || (other == score && i < g);
      }
      bool kept = score != 0 && g < p.groups && better < p.top_groups;
      if (values) {
        const uint32_t last = __reduce_min_sync(kAll, kept ? lowest(score, slack) : kTop);
        const uint32_t next = __reduce_max_sync(kAll, !kept && score != 0 && g < p.groups ? highest(score, slack) : 0u);
        if (border(last, next)) kept = groups_exact<VPL>(p, row, lane);
      }
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (!kept) key[i] = 0;
    } else {
      uint32_t gk[VPL];  // lane l: groups VPL l ..
      float gs_off[VPL];
#pragma unroll
      for (int i = 0; i < VPL; ++i) gk[i] = 0, gs_off[i] = 0.0f;
      for (int g = 0; g < p.groups; ++g) {
        uint32_t a = 0, b = 0;  // the lane's two largest of the group
        const int lo = g * gs - e0, hi = lo + gs;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
          const uint32_t v = i >= lo && i < hi ? gkey[i] : 0u;
          b = max(b, min(a, v));
          a = max(a, v);
        }
        const uint32_t best = __reduce_max_sync(kAll, a);
        uint32_t second = 0;
        if (p.top2) {
          const uint32_t who = __ballot_sync(kAll, a == best);
          second = __reduce_max_sync(kAll, lane == __ffs(who) - 1 ? b : a);
        }
        float slack = 0.0f;
        const uint32_t score = group_score(best, second, slack);
#pragma unroll
        for (int i = 0; i < VPL; ++i)
          if (e0 + i == g) gk[i] = score, gs_off[i] = slack;
      }
      bool kept[VPL];
#pragma unroll
      for (int i = 0; i < VPL; ++i) kept[i] = false;
      uint32_t last = kTop;
      for (int n = 0; n < p.top_groups; ++n) {
        int at;
        if (take_max<VPL>(gk, lane, at) == 0) break;
        const int lo = at * gs - e0, hi = lo + gs;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
          if (e0 + i == at) last = min(last, lowest(gk[i], gs_off[i])), gk[i] = 0;
          if (i >= lo && i < hi) kept[i] = true;
        }
      }
      if (values) {
        uint32_t next = 0;
#pragma unroll
        for (int i = 0; i < VPL; ++i)
          if (gk[i] != 0) next = max(next, highest(gk[i], gs_off[i]));
        close = border(__reduce_min_sync(kAll, last), __reduce_max_sync(kAll, next));
      }
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (!kept[i]) key[i] = 0;
    }
  }

  // The choices in falling order, one to a lane: lane j has the (j + 1)-th key and its expert; key 0: none.
  uint32_t my_key = 0;
  int at = -1;
  uint32_t bound = 1;
  if (VPL > 1 && p.k < 32) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i) top = max(top, key[i]);
    for (int j = 0; j <= p.k + 1; ++j) {
      bound = __reduce_max_sync(kAll, top);
      if (top == bound) top = 0;
    }
    bound = max(bound, 1u);
  }
  uint32_t in = 0;
#pragma unroll
  for (int i = 0; i < VPL; ++i) in |= key[i] >= bound ? 1u << i : 0u;
  int slot = __popc(in), n = slot;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(kAll, n, o);
    if (lane >= o) n += v;
  }
  slot = n - slot;
  n = __shfl_sync(kAll, n, 31);
  if (n <= 32) {
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (in >> i & 1) {
        pack_key[warp][slot] = key[i];
        pack_at[warp][slot++] = e0 + i;
      }
    __syncwarp();
    if (lane < n) my_key = pack_key[warp][lane], at = pack_at[warp][lane];
    int better = 0;  // larger keys, and equal ones of lower index
    for (int j = 0; j < n; j += 4) {
      const uint4 k4 = *reinterpret_cast<const uint4*>(&pack_key[warp][j]);
      const uint32_t other[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (j + u < n) better += other[u] > (j + u < lane ? my_key - 1 : my_key);
    }
    __syncwarp();
    if (lane < n) pack_key[warp][better] = my_key, pack_at[warp][better] = at;
    __syncwarp();
    my_key = lane < n ? pack_key[warp][lane] : 0;
    at = lane < n ? pack_at[warp][lane] : -1;
  } else {  // more candidates than lanes: one after the other
    for (int j = 0; j <= min(p.k, 31); ++j) {
      int e;
      const uint32_t best = take_max<VPL>(key, lane, e);
      if (best == 0) break;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (e0 + i == e) key[i] = 0;
      if (lane == j) my_key = best, at = e;
    }
  }
  bool swap = false;  // neighbours to be told apart in fp64, all among the candidates
  if (p.bias) {
    // Neighbours in the order that fp32 cannot tell apart, unless logits and biases are the same: then the index decides.
    // The k-th may stand at the head of a run of such neighbours (some of them the same), and any of them may belong
    // before it: the whole run counts, and where it may go on outside the candidates what is left is compared too.
    const uint32_t next_key = __shfl_down_sync(kAll, my_key, 1);
    const int next_at = __shfl_down_sync(kAll, at, 1);
    const bool run = lane < 31 && my_key != 0 && next_key != 0 && my_key != kNaN && next_key != kNaN && near(my_key, next_key);
    bool differ = false;
    if (run) {
      const float la = load_f32(p.logits, row + at, p.type), lb = load_f32(p.logits, row + next_at, p.type);
      differ = !(la == lb && __ldg(p.bias + at) == __ldg(p.bias + next_at));
    }
    const uint32_t runs = __ballot_sync(kAll, run), differs = __ballot_sync(kAll, differ);
    const int end = p.k - 2 + __ffs(~(runs >> (p.k - 1)));  // last lane of the k-th's run
    swap = (differs & ((1u << end) - 1)) != 0;
    const uint32_t last = __shfl_sync(kAll, my_key, p.k - 1);
    if (last != 0 && last < kNaN &&
        (n > 32 ? p.k == 32 || end >= p.k : end >= p.k && bound > 1 && near(max(last, bound), bound))) {
      const int last_at = __shfl_sync(kAll, at, p.k - 1);
      const float ll = load_f32(p.logits, row + last_at, p.type), lb = __ldg(p.bias + last_at);
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (key[i] != 0 && (n > 32 || key[i] < bound) && near(last, key[i]))
          close = close || !(load_f32(p.logits, row + e0 + i, p.type) == ll && __ldg(p.bias + e0 + i) == lb);
    }
  }
  close = __any_sync(kAll, close);
  if (swap && !close) {
    const uint32_t last = __shfl_sync(kAll, my_key, p.k - 1);
    if (n > 32 || (last != 0 && last < kNaN && near(max(last, bound), bound))) {
      close = true;  // values below the bound may belong to the choice
    } else {
      const int better = rank_exact<VPL>(p, row, lane, at, lane < n);
      __syncwarp();
      if (lane < n) pack_at[warp][better] = at;
      __syncwarp();
      if (lane < n) at = pack_at[warp][lane];
    }
  }
  int mine = lane < p.k ? at : -1;
  if (close) mine = choose_exact<VPL>(p, row, lane);

  // lane j: the weight of its expert
  float w = 0.0f;
  const float lm = mine >= 0 ? load_f32(p.logits, row + mine, p.type) : -INFINITY;
  if (p.sigmoid) {
    if (p.renorm) {
      w = sigma_parts(lm);
      const float total = warp_sum(w);
      w = total == 0.0f ? 0.0f : __fdiv_rn(w, total);
    } else if (mine >= 0) {
      w = sigma(lm);
    }
  } else if (p.renorm) {  // softmax over the chosen ones: the common factor cancels
    const float top = warp_max(lm);
    if (mine >= 0) w = exp_diff(lm, top);
    const float total = warp_sum(w);
    w = mine >= 0 ? __fdiv_rn(w, total) : 0.0f;
  } else if (mine >= 0) {
    w = __fdiv_rn(exp_diff(lm, m), sum);
  }
  if (lane < p.k) {
    p.weights[t * p.k + lane] = mine >= 0 ? w * p.scale : 0.0f;
    p.indices[t * p.k + lane] = mine;
  }
}

__device__ __forceinline__ void store_f32(void* p, int64_t i, int type, float v) {
  if (type == B2X_F32)
    reinterpret_cast<float*>(p)[i] = v;
  else if (type == B2X_BF16)
    reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else
    reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
}

// VPL consecutive gradients of a row.
template <int VPL>
__device__ __forceinline__ void store_logits(const RouteParams& p, int64_t row, int lane, const float (&v)[VPL]) {
  const int e0 = lane * VPL;
  if (VPL % 4 == 0 && p.vec_d && e0 + VPL <= p.E) {
    char* dst = reinterpret_cast<char*>(p.d_logits) + (row + e0) * (p.type == B2X_F32 ? 4 : 2);
#pragma unroll
    for (int i = 0; i < VPL / 4; ++i) {
      if (p.type == B2X_F32) {
        reinterpret_cast<float4*>(dst)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      } else if (p.type == B2X_BF16) {
        reinterpret_cast<uint2*>(dst)[i] = make_uint2(pack_bf16x2(v[4 * i], v[4 * i + 1]), pack_bf16x2(v[4 * i + 2], v[4 * i + 3]));
      } else {
        const __half2 a = __floats2half2_rn(v[4 * i], v[4 * i + 1]), b = __floats2half2_rn(v[4 * i + 2], v[4 * i + 3]);
        reinterpret_cast<uint2*>(dst)[i] = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i)
    if (e0 + i < p.E) store_f32(p.d_logits, row + e0 + i, p.type, v[i]);
}

// d_logits of one token per warp.  With w_j = scale s_j (/ S, S = sum of the chosen s):
//   ds_j = scale d_j                              or  scale (d_j - sum_i d_i s_i / S) / S
//   sigmoid:  dl_e = ds_e s_e (1 - s_e); renormalised, with p_e = s_e / S,  scale p_e (d_e - sum_i p_i d_i) (1 - s_e)
//   softmax:  dl_e = s_e (ds_e - sum_i s_i ds_i); renormalised, w / scale is the softmax p over the chosen ones and
//             dl_e = scale p_e (d_e - sum_i p_i d_i), which needs the chosen logits alone.
// The chosen ones are made as the weights are; the dense part takes the approximate exponential, which is within
// (4 + 3 |l - max|) 2^-24 of s (16384 x 128: 6.9 us, with the library's 7.6).
// An expert named in two slots gets the sum of both.  The rest of the row is the dense part (0 except for the
// softmax over all experts), stored first; the chosen ones are stored over it after a __syncwarp.
template <int VPL>
__global__ void __launch_bounds__(kRouteWarps * 32) moe_route_backward_kernel(const __grid_constant__ RouteParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
  if (t >= p.tokens) return;
  const int64_t row = t * p.ld;
  int at = -1;
  float d = 0.0f, lm = -INFINITY;
  if (lane < p.k) {
    at = p.indices[t * p.k + lane];
    if (at < 0 || at >= p.E) at = -1;
    if (at >= 0) d = p.d_weights[t * p.k + lane] * p.scale, lm = load_f32(p.logits, row + at, p.type);
    if (lm == -INFINITY) at = -1, d = 0.0f;
  }
  const bool dense = !p.sigmoid && !p.renorm;
  float mine = 0.0f;
  if (dense) {
    float l[VPL];
    float m = -INFINITY, sum = 0.0f;
    load_logits<VPL>(p, row, lane, l);
#pragma unroll
    for (int i = 0; i < VPL; ++i) m = fmaxf(m, l[i]);
    m = warp_max(m);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      l[i] = l[i] == -INFINITY ? 0.0f : exp_approx(l[i] - m);
      sum += l[i];
    }
    sum = warp_sum(sum);
    const float r = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
    const float s = at >= 0 ? exp_diff(lm, m) * r : 0.0f;
    const float mean = warp_sum(at >= 0 ? s * d : 0.0f);
#pragma unroll
    for (int i = 0; i < VPL; ++i) l[i] = -l[i] * r * mean;
    store_logits<VPL>(p, t * p.ld_d, lane, l);
    float all = 0.0f;  // of every slot that names this lane's expert
    for (int j = 0; j < p.k; ++j) {
      const int aj = __shfl_sync(kAll, at, j);
      const float dj = __shfl_sync(kAll, d, j);
      if (aj == at) all += dj;
    }
    mine = s * (all - mean);
  } else {
    float zero[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) zero[i] = 0.0f;
    store_logits<VPL>(p, t * p.ld_d, lane, zero);
    float dl = 0.0f;  // this slot's part
    if (p.sigmoid) {
      const float slope = at >= 0 ? sigma(-lm) : 0.0f;  // of log s
      if (p.renorm) {
        const float v = sigma_parts(lm);
        const float total = warp_sum(v);
        const float pr = total == 0.0f ? 0.0f : __fdiv_rn(v, total);
        const float mean = warp_sum(at >= 0 ? pr * d : 0.0f);
        dl = at >= 0 ? pr * (d - mean) * slope : 0.0f;
      } else if (at >= 0) {
        dl = d * sigma(lm) * slope;
      }
    } else {
      const float top = warp_max(lm);
      float pr = at >= 0 ? exp_diff(lm, top) : 0.0f;
      const float total = warp_sum(pr);
      pr = at >= 0 ? __fdiv_rn(pr, total) : 0.0f;
      const float mean = warp_sum(at >= 0 ? pr * d : 0.0f);
      dl = at >= 0 ? pr * (d - mean) : 0.0f;
    }
    for (int j = 0; j < p.k; ++j) {
      const int aj = __shfl_sync(kAll, at, j);
      const float dj = __shfl_sync(kAll, dl, j);
      if (aj == at) mine += dj;
    }
  }
  __syncwarp();
  if (at >= 0) store_f32(p.d_logits, t * p.ld_d + at, p.type, mine);
}

template <int BACKWARD>
static cudaError_t launch_route(RouteParams p, cudaStream_t st) {
  const unsigned grid = (unsigned)((p.tokens + kRouteWarps - 1) / kRouteWarps);
  const int per = (p.E + 31) / 32;
  static constexpr int kWidths[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 32};
  int vpl = 1;
  for (int w : kWidths) {
    vpl = w;
    if (w >= per) break;
  }
  const int bytes = 4 * (p.type == B2X_F32 ? 4 : 2);  // of four values
  p.vec = (uintptr_t)p.logits % bytes == 0 && p.ld % 4 == 0;
  p.vec_b = (uintptr_t)p.bias % 16 == 0;
  p.vec_d = (uintptr_t)p.d_logits % bytes == 0 && p.ld_d % 4 == 0;
  const int gs = p.E / p.groups, lanes = gs / vpl;
  p.lanes_per_group = gs % vpl == 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
#define B2X_ROUTE(V)                                                       \
  if constexpr (BACKWARD)                                                  \
    moe_route_backward_kernel<V><<<grid, kRouteWarps * 32, 0, st>>>(p);    \
  else                                                                     \
    moe_route_kernel<V><<<grid, kRouteWarps * 32, 0, st>>>(p)
  switch (vpl) {
    case 1: B2X_ROUTE(1); break;
    case 2: B2X_ROUTE(2); break;
    case 3: B2X_ROUTE(3); break;
    case 4: B2X_ROUTE(4); break;
    case 5: B2X_ROUTE(5); break;
    case 6: B2X_ROUTE(6); break;
    case 8: B2X_ROUTE(8); break;
    case 10: B2X_ROUTE(10); break;
    case 12: B2X_ROUTE(12); break;
    case 16: B2X_ROUTE(16); break;
    default: B2X_ROUTE(32); break;
  }
#undef B2X_ROUTE
  note_launch(1);
  return cudaGetLastError();
}

// Values of `bytes` each that do not start on a multiple of it: a misaligned access.
static bool off_grid(const void* p, int bytes) { return (uintptr_t)p % bytes != 0; }

static b2x_status route_params(const b2x_moe_route_args* a, const char* who, bool backward, RouteParams& p) {
  if (!a) return fail(B2X_ERR_INVALID_ARG, "%s: args is NULL", who);
  if (a->logits_type != B2X_F32 && a->logits_type != B2X_BF16 && a->logits_type != B2X_F16)
    return fail(B2X_ERR_UNSUPPORTED, "%s: logits must be fp32, bf16 or fp16", who);
  if (a->tokens < 0 || a->experts <= 0 || a->ld_logits < a->experts)
    return fail(B2X_ERR_INVALID_ARG, "%s: bad shape (tokens %lld, experts %lld, ld %lld)", who, (long long)a->tokens,
                (long long)a->experts, (long long)a->ld_logits);
  if (a->experts > 1024 || a->top_k > 32)
    return fail(B2X_ERR_UNSUPPORTED, "%s: at most 1024 experts and top_k 32 (got %lld, %d)", who, (long long)a->experts,
                a->top_k);
  if (a->top_k < 1 || a->top_k > a->experts)
    return fail(B2X_ERR_INVALID_ARG, "%s: top_k must be in [1, experts] (got %d)", who, a->top_k);
  if (a->tokens > (int64_t)kRouteWarps * 0x7fffffff) return fail(B2X_ERR_UNSUPPORTED, "%s: too many tokens", who);
  if (!backward && (a->num_groups < 1 || a->experts % a->num_groups || a->top_groups < 1 || a->top_groups > a->num_groups))
    return fail(B2X_ERR_INVALID_ARG, "%s: num_groups (%d) must divide experts, top_groups (%d) lie in [1, num_groups]", who,
                a->num_groups, a->top_groups);
  if (a->tokens > 0 && (!a->logits || !a->indices || (!backward && !a->weights)))
    return fail(B2X_ERR_INVALID_ARG, "%s: NULL pointer", who);
  if (off_grid(a->logits, a->logits_type == B2X_F32 ? 4 : 2) || off_grid(a->bias, 4) || off_grid(a->weights, 4) ||
      off_grid(a->indices, 4))
    return fail(B2X_ERR_INVALID_ARG, "%s: misaligned pointer", who);
  p.logits = a->logits;
  p.ld = a->ld_logits;
  p.tokens = a->tokens;
  p.type = a->logits_type;
  p.E = (int)a->experts;
  p.k = a->top_k;
  p.sigmoid = a->sigmoid != 0;
  p.renorm = a->renormalize != 0;
  p.groups = backward || a->top_groups == a->num_groups ? 1 : a->num_groups;  // all groups stay: no group step
  p.top_groups = a->top_groups;
  p.top2 = a->group_top2 != 0;
  p.scale = a->scale;
  p.bias = a->bias;
  p.weights = a->weights;
  p.indices = a->indices;
  return B2X_OK;
}

}  // namespace b2x

extern "C" B2X_API b2x_status b2x_moe_route(const b2x_moe_route_args* args, void* stream) {
  using namespace b2x;
  t_err[0] = 0;
  RouteParams p{};
  b2x_status s = route_params(args, "b2x_moe_route", false, p);
  if (s != B2X_OK || p.tokens == 0) return s;
  cudaError_t e = launch_route<0>(p, (cudaStream_t)stream);
  return e == cudaSuccess ? B2X_OK : cuda_fail(e, "b2x_moe_route launch");
}

extern "C" B2X_API b2x_status b2x_moe_route_backward(const b2x_moe_route_args* args, const float* d_weights, void* d_logits,
                                                     int64_t ld_d_logits, void* stream) {
  using namespace b2x;
  t_err[0] = 0;
  RouteParams p{};
  b2x_status s = route_params(args, "b2x_moe_route_backward", true, p);
  if (s != B2X_OK) return s;
  if (ld_d_logits < p.E) return fail(B2X_ERR_INVALID_ARG, "b2x_moe_route_backward: ld_d_logits < experts");
  if (p.tokens == 0) return B2X_OK;
  if (!d_weights || !d_logits) return fail(B2X_ERR_INVALID_ARG, "b2x_moe_route_backward: NULL pointer");
  if (off_grid(d_weights, 4) || off_grid(d_logits, args->logits_type == B2X_F32 ? 4 : 2))
    return fail(B2X_ERR_INVALID_ARG, "b2x_moe_route_backward: misaligned pointer");
  p.d_weights = d_weights;
  p.d_logits = d_logits;
  p.ld_d = ld_d_logits;
  cudaError_t e = launch_route<1>(p, (cudaStream_t)stream);
  return e == cudaSuccess ? B2X_OK : cuda_fail(e, "b2x_moe_route_backward launch");
}
