// Routing of tokens to experts: scores of a row of logits, the choice of the k best experts
// (optionally steered by a per-expert bias and limited to the best groups of experts), their
// weights, and the gradient of the logits.
//
//   p = softmax(l)  or  p = 1 / (1 + e^-l);   key = p + bias;   ids = the k largest keys
//   w_j = scale * p[id_j]  or, renormalised,  scale * p[id_j] / sum_i p[id_i]
//
// A warp takes a token at a time.  The choice has to be the one that exact arithmetic makes, ties
// to the lower index.  It is made on approximate 32-bit keys first: every lane sorts the few it
// holds, then k + 1 rounds take the largest head of the 32 lists.  Where two neighbours of that
// order (or the last group kept and the first dropped) are closer than the keys' error, the row
// is decided again on 64-bit keys (about one row in a hundred with 256 sigmoid scores).  16-bit
// logits that compete without a bias need no scores: their own order is exact.
//
// Bound by instructions: some 1000 per row of 256 experts with sigmoid scores, groups and 8 choices
// (16384 rows 25 us, on 64-bit keys throughout 77; the memory traffic alone would take 3), 580 per
// row of 128 by their logits (12.5 us).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include "../api.h"
#include "../device/tile_compute.cuh"
#include "../runtime/errors.h"

namespace tileccl {
namespace {

constexpr int kWarpsPerCta = 4;
constexpr int kMaxRouted = 512;          // experts at most (a power of two)
constexpr uint32_t kAll = 0xffffffffu;

enum RouteDtype : int { kF16 = 0, kBF16 = 1, kF32 = 2 };
// What experts compete with: the logit itself (it orders like the score), or a score and a bias.
// kExact: 16-bit logits, whose keys leave room for the whole index and need no second look.
enum RouteMode : int { kByLogit = 0, kSigmoid = 1, kSoftmax = 2, kExact = 3 };

struct RouteParams {
  const void* logits;
  int64_t ld;                 // elements between rows of logits
  const float* bias;          // [experts] or null
  const uint8_t* mask;        // [tokens] (0 = the token is not routed) or null
  float* weights;             // [tokens, top_k]
  int32_t* ids;               // [tokens, top_k]
  const float* grad_weights;  // backward only
  void* grad_logits;          // backward only, [tokens, experts] contiguous
  int64_t tokens;
  int32_t experts, top_k, dtype, sigmoid, groups, top_groups, group_max, renormalize;
  int32_t fast, lane_shift;   // the groups share the lanes evenly: 2^lane_shift lanes each
  int32_t wide, wide_out;     // a lane's logits (gradients) can be moved in whole pieces
  float scale;
};

__device__ __forceinline__ float load_logit(const void* base, int64_t i, int dtype) {
  if (dtype == kF32) return static_cast<const float*>(base)[i];
  if (dtype == kBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
  return __half2float(static_cast<const __half*>(base)[i]);
}
__device__ __forceinline__ void store_logit(void* base, int64_t i, int dtype, float v) {
  if (dtype == kF32) static_cast<float*>(base)[i] = v;
  else if (dtype == kBF16) static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16(v);
  else static_cast<__half*>(base)[i] = __float2half(v);
}

template <typename T>
__device__ __forceinline__ T warp_max(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const T u = __shfl_xor_sync(kAll, v, o);
    v = u > v ? u : v;
  }
  return v;
}
template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

__device__ __forceinline__ float sigmoid_f(float x) { return 1.f / (1.f + expf(-x)); }
// sigmoid(l) * e^-min(m, 0), m the largest logit concerned: the ratio of two sigmoids keeps its
// precision where both underflow.
__device__ __forceinline__ float sigmoid_scaled(float l, float m) {
  const float s = fminf(m, 0.f);
  return (l > 0.f ? 1.f : expf(l - s)) / (1.f + expf(-fabsf(l)));
}

// Approximations for keys (denormals count as zero: far below the keys' error).
__device__ __forceinline__ float exp_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Numbers as unsigned integers of the same order.
__device__ __forceinline__ uint32_t order32(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);     // (-0 becomes +0)
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value32(uint32_t u) {
  return __uint_as_float(u ^ ((u >> 31) ? 0x80000000u : 0xffffffffu));
}
// 64-bit keys: 0 = the expert is not available (logit or bias of -inf, or outside the chosen
// groups); 1 = the key is not a number: it ranks behind every number, so ids stay distinct and
// in range.
__device__ __forceinline__ uint64_t order64(double x) {
  if (x != x) return 1;
  if (x == -CUDART_INF) return 0;
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(x == 0.0 ? 0.0 : x));
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double value64(uint64_t u) {
  return __longlong_as_double(static_cast<long long>((u >> 63) ? u & 0x7fffffffffffffffull : ~u));
}

// The row's choice on 64-bit keys (`keys`: one per expert in shared memory); lane j returns the
// j-th id.  `top` is the row's largest logit.
__device__ __noinline__ int choose_exactly(const RouteParams& p, int64_t t, float top, uint64_t* keys) {
  const int lane = threadIdx.x & 31;
  const bool by_logit = p.bias == nullptr && (p.groups == 1 || p.group_max != 0);
  double total = 1.0;
  if (!by_logit && !p.sigmoid) {
    double part = 0.0;
    for (int e = lane; e < p.experts; e += 32) {
      const float l = load_logit(p.logits, t * p.ld + e, p.dtype);
      if (l != -CUDART_INF_F) part += exp(static_cast<double>(l) - static_cast<double>(top));
    }
    total = warp_sum(part);
  }
  for (int e = lane; e < p.experts; e += 32) {
    const float l = load_logit(p.logits, t * p.ld + e, p.dtype);
    double k = l;
    if (!by_logit)
      k = p.sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(l)))
                    : exp(static_cast<double>(l) - static_cast<double>(top)) / total;
    if (p.bias != nullptr) k += static_cast<double>(p.bias[e]);
    keys[e] = l == -CUDART_INF_F ? 0 : order64(k);
  }
  __syncwarp();
  if (p.groups > 1) {
    const int per = p.experts / p.groups;
    // lane g: score of group g = its largest key, or the sum of its two largest available keys
    uint64_t score = 0;
    if (lane < p.groups) {
      uint64_t a = 0, b = 0;
      for (int i = 0; i < per; ++i) {
        const uint64_t x = keys[lane * per + i];
        if (x > a) { b = a; a = x; }
        else if (x > b) b = x;
      }
      score = p.group_max || b <= 1 ? a : order64(value64(a) + value64(b));
    }
    int ahead = 0;
    for (int g = 0; g < p.groups; ++g) {
      const uint64_t other = __shfl_sync(kAll, score, g);
      ahead += (other > score || (other == score && g < lane)) ? 1 : 0;
    }
    const uint32_t keep = __ballot_sync(kAll, lane < p.groups && ahead < p.top_groups);
    for (int e = lane; e < p.experts; e += 32)
      if (((keep >> (e / per)) & 1u) == 0) keys[e] = 0;
    __syncwarp();
  }
  int mine = -1;
  for (int j = 0; j < p.top_k; ++j) {
    uint64_t best = 0;
    int at = 0;
    for (int e = lane; e < p.experts; e += 32)
      if (keys[e] > best) { best = keys[e]; at = e; }
    const uint64_t round = warp_max(best);
    if (round == 0) break;
    const uint32_t id = __reduce_min_sync(kAll, best == round ? static_cast<uint32_t>(at) : kAll);
    if (static_cast<int>(id & 31u) == lane) keys[id] = 0;
    __syncwarp();
    if (lane == j) mine = static_cast<int>(id);
  }
  __syncwarp();
  return mine;
}

// A key in 64 bits; `total` = sum of exp(l - top) over the row (softmax).
__device__ __forceinline__ double key64(const RouteParams& p, int mode, float l, float bias, float top,
                                        double total) {
  if (mode == kByLogit) return l;      // (kExact never asks)
  const double x = static_cast<double>(l);
  const double s = mode == kSigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - static_cast<double>(top)) / total;
  return s + static_cast<double>(bias);
}
// Sum of the row's exponentials in 64 bits; lane: logits first .. first + n - 1 of the row.
__device__ __noinline__ double softmax_total(const RouteParams& p, int64_t at, int n, float top) {
  double part = 0.0;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float l = load_logit(p.logits, at + i, p.dtype);
    if (l != -CUDART_INF_F) part += exp(static_cast<double>(l) - static_cast<double>(top));
  }
  return warp_sum(part);
}
// Score of this lane's group in 64 bits; lane as above, `lanes` lanes per group.
__device__ __noinline__ uint64_t group_score64(const RouteParams& p, int mode, int64_t at, int n, int first,
                                               int lanes, float top, double total) {
  uint64_t a = 0, b = 0;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float l = load_logit(p.logits, at + i, p.dtype);
    const float bias = p.bias != nullptr ? p.bias[first + i] : 0.f;
    const uint64_t x = l == -CUDART_INF_F ? 0 : order64(key64(p, mode, l, bias, top, total));
    b = b > (a < x ? a : x) ? b : (a < x ? a : x);
    a = a > x ? a : x;
  }
  for (int o = 1; o < lanes; o <<= 1) {
    const uint64_t c = __shfl_xor_sync(kAll, a, o), d = __shfl_xor_sync(kAll, b, o);
    const uint64_t lower = a < c ? a : c, second = b > d ? b : d;
    b = lower > second ? lower : second;
    a = a > c ? a : c;
  }
  return p.group_max || b <= 1 ? a : order64(value64(a) + value64(b));
}
// Lane j holds candidate j (`id`, -1 = none).  Returns the candidates in the order of their
// 64-bit keys, the lower index first among equals.
__device__ __noinline__ int order_candidates(const RouteParams& p, int mode, int64_t row, int id, float top,
                                             double total) {
  uint64_t k = 0;
  if (id >= 0)
    k = order64(key64(p, mode, load_logit(p.logits, row + id, p.dtype), p.bias != nullptr ? p.bias[id] : 0.f,
                      top, total));
  int ahead = 0;
  for (int i = 0; i < 32; ++i) {
    const uint64_t other = __shfl_sync(kAll, k, i);
    const int other_id = __shfl_sync(kAll, id, i);
    ahead += other_id >= 0 && (other > k || (other == k && other_id < id)) ? 1 : 0;
  }
  const int lane = threadIdx.x & 31;
  int out = -1;
  for (int i = 0; i < 32; ++i) {
    const int place = __shfl_sync(kAll, id >= 0 ? ahead : -1, i);
    const int other_id = __shfl_sync(kAll, id, i);
    if (place == lane) out = other_id;
  }
  return out;
}

// Lane `lane` holds the logits first .. first + n - 1 (n <= EPL) of its row, -inf behind them.
template <int EPL>
__device__ __forceinline__ void load_logits(const RouteParams& p, int64_t at, int n, float (&l)[EPL]) {
  if (p.wide && n == EPL) {
    if (p.dtype == kF32) {
      if constexpr (EPL >= 4) {
        const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(p.logits) + at);
#pragma unroll
        for (int i = 0; i < EPL / 4; ++i) {
          const float4 v = src[i];
          l[4 * i] = v.x; l[4 * i + 1] = v.y; l[4 * i + 2] = v.z; l[4 * i + 3] = v.w;
        }
        return;
      }
    } else if constexpr (EPL >= 2) {
      alignas(16) uint32_t w[EPL / 2];
      const char* src = static_cast<const char*>(p.logits) + 2 * at;
      if constexpr (EPL == 2) w[0] = *reinterpret_cast<const uint32_t*>(src);
      else if constexpr (EPL == 4) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(src);
      else {
#pragma unroll
        for (int i = 0; i < EPL / 8; ++i)
          reinterpret_cast<uint4*>(w)[i] = reinterpret_cast<const uint4*>(src)[i];
      }
#pragma unroll
      for (int i = 0; i < EPL / 2; ++i) {
        const float2 v = unpack_16x2(p.dtype == kBF16, w[i]);
        l[2 * i] = v.x; l[2 * i + 1] = v.y;
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) l[i] = i < n ? load_logit(p.logits, at + i, p.dtype) : -CUDART_INF_F;
}

// Descending order of a lane's list (odd-even merge sort).
template <int N>
__device__ __forceinline__ void sort_descending(uint32_t (&v)[N]) {
#pragma unroll
  for (int q = 1; q < N; q <<= 1)
#pragma unroll
    for (int k = q; k >= 1; k >>= 1)
#pragma unroll
      for (int j = k % q; j + k < N; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < N && (i + j) / (2 * q) == (i + j + k) / (2 * q)) {
            const uint32_t hi = max(v[i + j], v[i + j + k]), lo = min(v[i + j], v[i + j + k]);
            v[i + j] = hi;
            v[i + j + k] = lo;
          }
}

// EPL: experts per lane (a power of two).  The lanes are shared out evenly among the groups;
// within a group lane i holds the experts i * EPL, i * EPL + 1, ...
template <int EPL, int kMode>
__global__ void __launch_bounds__(kWarpsPerCta * 32, EPL < 16 ? 8 : 4)
expert_route_kernel(const __grid_constant__ RouteParams p) {
  extern __shared__ uint64_t smem_keys[];   // [warps][experts]
  constexpr bool kByKey = kMode == kByLogit || kMode == kExact;
  // low bits of a key: the place in the lane's list, or the whole index, the lowest on top
  constexpr uint32_t kPlace = kMode == kExact ? kMaxRouted - 1u : EPL - 1u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int lanes = 1 << p.lane_shift;                            // per group
  const int per = p.fast ? p.experts / p.groups : p.experts;
  const int group = lane >> p.lane_shift;
  const int in_group = (lane - group * lanes) * EPL;
  const int first = group * per + in_group;
  const int n = min(max(per - in_group, 0), EPL);
  // Error of a pair of keys: the bits that hold the place (2^-23 EPL of each), and that of the
  // scores: sigmoid 1/4 (2 + 1.2 |l|) 2^-23, a sum and a division, below 2^-20 each; softmax,
  // whose sum carries the errors of all terms, below 2^-18 each.
  constexpr float kKeyError = kByKey ? 0.f : 4.f * EPL * 0x1p-23f;
  constexpr float kScoreError = kByKey ? 0.f : kMode == kSigmoid ? 0x1p-19f : 0x1p-17f;
  float bias[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) bias[i] = !kByKey && p.bias != nullptr && i < n ? p.bias[first + i] : 0.f;

  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kWarpsPerCta + warp; t < p.tokens;
       t += static_cast<int64_t>(gridDim.x) * kWarpsPerCta) {
    float* const out_w = p.weights + t * p.top_k;
    int32_t* const out_i = p.ids + t * p.top_k;
    if (p.mask != nullptr && p.mask[t] == 0) {
      if (lane < p.top_k) { out_w[lane] = 0.f; out_i[lane] = -1; }
      continue;
    }
    const int64_t row = t * p.ld;
    float l[EPL];
    load_logits<EPL>(p, row + first, n, l);
    float top = l[0];
    if (!p.sigmoid) {
#pragma unroll
      for (int i = 1; i < EPL; ++i) top = fmaxf(top, l[i]);
      top = value32(__reduce_max_sync(kAll, top != top ? 0u : order32(top)));
    }

    // approximate keys, packed with the place in the lane's list
    uint32_t key[EPL];
    float x[EPL];
    float inv = 1.f;
    if (kMode == kSoftmax) {
      float part = 0.f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) part += x[i] = exp_approx(l[i] - top);
      inv = rcp_approx(warp_sum(part));
    }
    float finite = 0.f;                    // NaN if a key is infinite or not a number
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      float k = l[i];
      if (kMode == kSigmoid) k = rcp_approx(1.f + exp_approx(-l[i])) + bias[i];
      if (kMode == kSoftmax) k = fmaf(x[i], inv, bias[i]);
      const bool there = l[i] != -CUDART_INF_F && (kByKey || k != -CUDART_INF_F);   // (-inf behind the row)
      finite = fmaf(there ? k : 0.f, 0.f, finite);
      const uint32_t place = kMode == kExact ? kPlace - first - i : kPlace - i;
      key[i] = there ? (order32(k) & ~kPlace) | place : 0u;
    }
    const bool odd = !p.fast || __any_sync(kAll, finite != 0.f);
    int id = -1;
    bool broken = false;                   // a row without numbers for weights
    float my_l = -CUDART_INF_F;
    if (odd) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) broken = broken || l[i] != l[i];
      broken = __any_sync(kAll, broken) || (!p.sigmoid && top == CUDART_INF_F);   // as the formula has it
      id = choose_exactly(p, t, top, smem_keys + static_cast<int64_t>(warp) * p.experts);
      if (id >= 0) my_l = load_logit(p.logits, row + id, p.dtype);
    } else {
      sort_descending(key);
      double total = 1.0;
      bool have_total = kMode != kSoftmax;
      if (p.groups > 1) {
        uint32_t a = key[0], b = EPL > 1 ? key[EPL > 1 ? 1 : 0] : 0u;
        for (int o = 1; o < lanes; o <<= 1) {
          const uint32_t c = __shfl_xor_sync(kAll, a, o), d = __shfl_xor_sync(kAll, b, o);
          b = max(min(a, c), max(b, d));
          a = max(a, c);
        }
        const float va = value32(a & ~kPlace), vb = value32(b & ~kPlace);
        const uint32_t score = a == 0 ? 0u : order32(p.group_max || b == 0 ? va : va + vb);
        int ahead = 0;
        for (int g = 0; g < p.groups; ++g) {
          const uint32_t other = __shfl_sync(kAll, score, g * lanes);
          ahead += other > score || (other == score && g < group) ? 1 : 0;
        }
        bool keep = ahead < p.top_groups;
        if (kMode != kExact) {
          const uint32_t worst = __reduce_min_sync(kAll, keep ? score : kAll);
          const uint32_t next = __reduce_max_sync(kAll, keep ? 0u : score);
          const float w = value32(worst), v = value32(next);
          const float size = fmaxf(fabsf(w), fabsf(v)) + (p.group_max ? 0.f : 2.f * fabsf(va) + 2.f * fabsf(vb));
          if (__any_sync(kAll, next != 0 && !(w - v > size * kKeyError + 2.f * kScoreError))) {
            if (!have_total) total = softmax_total(p, row + first, n, top);
            have_total = true;
            const uint64_t mine = group_score64(p, kMode, row + first, n, first, lanes, top, total);
            ahead = 0;
            for (int g = 0; g < p.groups; ++g) {
              const uint64_t other = __shfl_sync(kAll, mine, g * lanes);
              ahead += other > mine || (other == mine && g < group) ? 1 : 0;
            }
            keep = ahead < p.top_groups;
          }
        }
        if (!keep) {
#pragma unroll
          for (int i = 0; i < EPL; ++i) key[i] = 0u;
        }
      }
      // k rounds, each takes the largest head; with inexact keys they go on while the next is too
      // close to the k-th to tell them apart.
      uint32_t mine = 0;
      int from = 0;                        // lane that held this lane's choice
      float limit = -CUDART_INF_F;
      bool close = false, many = false;
      for (int j = 0;; ++j) {
        if (kMode == kExact && j == p.top_k) break;
        const uint32_t best = __reduce_max_sync(kAll, key[0]);
        if (best == 0) break;
        if (kMode != kExact && j >= p.top_k) {
          if (value32(best & ~kPlace) < limit) break;
          close = true;
          if (j == 32) { many = true; break; }
        }
        bool winner = key[0] == best;
        int at = 0;
        if (kMode != kExact) {             // (equal heads of two lanes are close: any goes first)
          at = __ffs(__ballot_sync(kAll, winner)) - 1;
          winner = lane == at;
        }
        if (lane == j) { mine = best; from = at; }
        if (winner) {
#pragma unroll
          for (int i = 0; i + 1 < EPL; ++i) key[i] = key[i + 1];
          key[EPL - 1] = 0u;
        }
        if (kMode != kExact && j == p.top_k - 1) {
          const float v = value32(best & ~kPlace);
          limit = kByKey ? v : v - (fabsf(v) * kKeyError + kScoreError);
        }
      }
      if (mine != 0) {
        const int place = static_cast<int>(kPlace - (mine & kPlace));
        id = kMode == kExact ? place : (from >> p.lane_shift) * per + (from & (lanes - 1)) * EPL + place;
        mine &= ~kPlace;
      }
      if (id >= 0) my_l = load_logit(p.logits, row + id, p.dtype);
      if (kMode != kExact) {
        const uint32_t below = __shfl_down_sync(kAll, mine, 1);
        const float w = value32(mine), v = value32(below);
        const bool pair = lane < p.top_k - 1 && below != 0 &&
                    !(w - v > fmaxf(fabsf(w), fabsf(v)) * kKeyError + kScoreError);
        if (__any_sync(kAll, pair)) {
          // two of the chosen that agree in logit and bias are equal exactly: the index decides
          const int next_id = __shfl_down_sync(kAll, id, 1);
          const float my_b = !kByKey && p.bias != nullptr && id >= 0 ? p.bias[id] : 0.f;
          const float next_l = __shfl_down_sync(kAll, my_l, 1), next_b = __shfl_down_sync(kAll, my_b, 1);
          close = close || __any_sync(kAll, pair && !(my_l == next_l && my_b == next_b && id < next_id));
        }
        if (many) {
          id = choose_exactly(p, t, top, smem_keys + static_cast<int64_t>(warp) * p.experts);
        } else if (close) {
          if (!have_total) total = softmax_total(p, row + first, n, top);
          id = order_candidates(p, kMode, row, id, top, total);
        }
        if (lane >= p.top_k) id = -1;
        if (close) my_l = id >= 0 ? load_logit(p.logits, row + id, p.dtype) : -CUDART_INF_F;
      }
    }

    // weights: lane j holds the j-th choice
    float w = 0.f;
    if (p.renormalize) {
      const float m = value32(__reduce_max_sync(kAll, my_l != my_l ? 0u : order32(my_l)));
      const float sc = id < 0 ? 0.f : p.sigmoid ? sigmoid_scaled(my_l, m) : expf(my_l - m);
      w = sc / warp_sum(sc);
    } else if (p.sigmoid) {
      w = sigmoid_f(my_l);
    } else {
      float part = 0.f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) part += i < n ? expf(l[i] - top) : 0.f;
      const float sum = warp_sum(part);
      w = expf(my_l - top) / sum;
    }
    w *= p.scale;
    if (broken) w = CUDART_NAN_F;
    if (id < 0) w = 0.f;
    if (lane < p.top_k) { out_w[lane] = w; out_i[lane] = id; }
  }
}

// dL/dl of a row from dL/dw of its k weights.  With n_j = w_j / scale and g_j = dL/dw_j:
//   softmax, renormalised   dl_i = scale n_i (g_i - sum_j g_j n_j)              i chosen
//   softmax                 dl_i = scale p_i (g_i [i chosen] - sum_j g_j p_j)   every i
//   sigmoid, renormalised   dl_i = scale n_i (1 - p_i) (g_i - sum_j g_j n_j)    i chosen
//   sigmoid                 dl_i = scale g_i p_i (1 - p_i)                      i chosen
// One warp per row; 16384 x 128 in fp32 take 8 us, 2.7 for the traffic, the rest are instructions.
template <int EPL>
__global__ void __launch_bounds__(kWarpsPerCta * 32)
expert_route_backward_kernel(const __grid_constant__ RouteParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kWarpsPerCta + warp;
  if (t >= p.tokens) return;
  const int first = lane * EPL, count = min(max(p.experts - first, 0), EPL);
  const bool dense = !p.sigmoid && !p.renormalize;     // every logit of the row counts
  int id = -1;
  float g = 0.f;
  if (lane < p.top_k) {
    id = p.ids[t * p.top_k + lane];
    g = p.grad_weights[t * p.top_k + lane];
  }
  float l[EPL];
  if (dense) load_logits<EPL>(p, t * p.ld + first, count, l);
  if (id < 0 || id >= p.experts) { id = -1; g = 0.f; }
  const bool routed = __any_sync(kAll, id >= 0);
  const float my_l = id >= 0 ? load_logit(p.logits, t * p.ld + id, p.dtype) : -CUDART_INF_F;
  float m = 0.f, sum = 0.f;
  if (dense) {
    m = l[0];
#pragma unroll
    for (int i = 1; i < EPL; ++i) m = fmaxf(m, l[i]);
    m = value32(__reduce_max_sync(kAll, m != m ? 0u : order32(m)));
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      l[i] = l[i] == -CUDART_INF_F ? 0.f : expf(l[i] - m);
      sum += l[i];
    }
    sum = warp_sum(sum);
  }
  float n = 0.f;
  if (p.renormalize) {
    const float top = value32(__reduce_max_sync(kAll, my_l != my_l ? 0u : order32(my_l)));
    const float s = id < 0 || my_l == -CUDART_INF_F ? 0.f
                    : p.sigmoid ? sigmoid_scaled(my_l, top) : expf(my_l - top);
    const float all = warp_sum(s);
    n = all > 0.f || all != all ? s / all : 0.f;
  } else if (id >= 0) {
    n = p.sigmoid ? sigmoid_f(my_l) : my_l == -CUDART_INF_F ? 0.f : expf(my_l - m) / sum;
  }
  const float dot = p.sigmoid && !p.renormalize ? 0.f : warp_sum(id >= 0 ? g * n : 0.f);
  // lane j's share of dl at its expert; the dense softmax adds -p_i * dot everywhere
  float mine = p.scale * n * (dense ? g : g - dot);
  if (p.sigmoid) mine *= sigmoid_f(-my_l);
  if (id < 0 || my_l == -CUDART_INF_F) mine = 0.f;
  float d[EPL];
  const float all = -p.scale * dot / sum;
#pragma unroll
  for (int i = 0; i < EPL; ++i) d[i] = dense && routed && l[i] != 0.f ? all * l[i] : 0.f;
  for (int j = 0; j < p.top_k; ++j) {
    const int e = __shfl_sync(kAll, id, j);
    const float v = __shfl_sync(kAll, mine, j);
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (e == first + i) d[i] += v;
  }
  const int64_t at = t * p.experts + first;
  if (p.wide_out && count == EPL) {
    if (p.dtype == kF32) {
      if constexpr (EPL >= 4) {
        float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.grad_logits) + at);
#pragma unroll
        for (int i = 0; i < EPL / 4; ++i)
          dst[i] = make_float4(d[4 * i], d[4 * i + 1], d[4 * i + 2], d[4 * i + 3]);
        return;
      }
    } else if constexpr (EPL >= 8) {
      uint4* dst = reinterpret_cast<uint4*>(static_cast<char*>(p.grad_logits) + 2 * at);
#pragma unroll
      for (int i = 0; i < EPL / 8; ++i) dst[i] = tile_cast_f32x8(p.dtype == kBF16, d + 8 * i);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if (i < count) store_logit(p.grad_logits, at + i, p.dtype, d[i]);
}

// CTAs of a forward launch: enough warps to fill the SMs, each with several rows, so that the
// bias is loaded once.
constexpr int64_t kMaxCtas = 148 * 8;

template <int EPL>
cudaError_t launch(const RouteParams& p, bool backward, cudaStream_t s) {
  const bool by_logit = p.bias == nullptr && (p.groups == 1 || p.group_max != 0);
  const int64_t blocks = (p.tokens + kWarpsPerCta - 1) / kWarpsPerCta;
  if (backward) {
    expert_route_backward_kernel<EPL><<<static_cast<unsigned>(blocks), kWarpsPerCta * 32, 0, s>>>(p);
  } else {
    const size_t smem = sizeof(uint64_t) * kWarpsPerCta * p.experts;
    const unsigned grid = static_cast<unsigned>(blocks < kMaxCtas ? blocks : kMaxCtas);
    if (by_logit && p.dtype != kF32) expert_route_kernel<EPL, kExact><<<grid, kWarpsPerCta * 32, smem, s>>>(p);
    else if (by_logit) expert_route_kernel<EPL, kByLogit><<<grid, kWarpsPerCta * 32, smem, s>>>(p);
    else if (p.sigmoid) expert_route_kernel<EPL, kSigmoid><<<grid, kWarpsPerCta * 32, smem, s>>>(p);
    else expert_route_kernel<EPL, kSoftmax><<<grid, kWarpsPerCta * 32, smem, s>>>(p);
  }
  return cudaGetLastError();
}

cudaError_t dispatch(RouteParams& p, bool backward, cudaStream_t s) {
  const int lanes = p.fast ? 32 / p.groups : 32;
  const int per = p.fast ? p.experts / p.groups : p.experts;
  const int need = (per + lanes - 1) / lanes;
  p.lane_shift = 0;
  while ((1 << p.lane_shift) < lanes) ++p.lane_shift;
  int epl = 1;
  while (epl < need) epl <<= 1;
  // every lane's piece is a power of two long; it is loaded whole if all pieces are aligned
  const int64_t elem = p.dtype == kF32 ? 4 : 2;
  const int64_t piece = epl * elem < 16 ? epl * elem : 16;
  p.wide = per % epl == 0 && (p.ld * elem) % piece == 0 &&
           reinterpret_cast<uint64_t>(p.logits) % piece == 0 ? 1 : 0;
  p.wide_out = per % epl == 0 && (p.experts * elem) % 16 == 0 ? 1 : 0;
  if (epl == 1) return launch<1>(p, backward, s);
  if (epl == 2) return launch<2>(p, backward, s);
  if (epl == 4) return launch<4>(p, backward, s);
  if (epl == 8) return launch<8>(p, backward, s);
  return launch<16>(p, backward, s);
}

int check(const RouteParams& p) {
  TCCL_CHECK_ARG(p.tokens >= 0 && p.tokens < (int64_t(1) << 31), "tokens out of range");
  TCCL_CHECK_ARG(p.experts >= 1 && p.experts <= kMaxRouted, "experts must be 1..512");
  TCCL_CHECK_ARG(p.top_k >= 1 && p.top_k <= 32 && p.top_k <= p.experts,
                 "top_k must be 1..min(32, experts)");
  TCCL_CHECK_ARG(p.dtype >= 0 && p.dtype <= 2, "dtype must be 0 (fp16), 1 (bf16) or 2 (fp32)");
  TCCL_CHECK_ARG(p.ld >= p.experts || p.tokens <= 1, "row pitch is smaller than a row");
  return kOk;
}

}  // namespace

template <int EPL>
static cudaError_t preload_route() {
  cudaFuncAttributes a;
  cudaError_t e = cudaFuncGetAttributes(&a, expert_route_kernel<EPL, kByLogit>);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, expert_route_kernel<EPL, kSigmoid>);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, expert_route_kernel<EPL, kSoftmax>);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, expert_route_kernel<EPL, kExact>);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, expert_route_backward_kernel<EPL>);
  return e;
}

cudaError_t preload_expert_route_kernels() {
  cudaError_t e = preload_route<1>();
  if (e == cudaSuccess) e = preload_route<2>();
  if (e == cudaSuccess) e = preload_route<4>();
  if (e == cudaSuccess) e = preload_route<8>();
  if (e == cudaSuccess) e = preload_route<16>();
  return e;
}

}  // namespace tileccl

using namespace tileccl;

extern "C" int tccl_expert_route(uint64_t logits, int64_t ld, uint64_t bias, uint64_t mask,
                                 uint64_t weights, uint64_t ids, int64_t tokens, int32_t experts,
                                 int32_t top_k, int32_t dtype, int32_t sigmoid, int32_t groups,
                                 int32_t top_groups, int32_t group_max, int32_t renormalize,
                                 float scale, uint64_t stream) {
  RouteParams p = {};
  p.logits = reinterpret_cast<const void*>(logits);
  p.ld = ld;
  p.bias = reinterpret_cast<const float*>(bias);
  p.mask = reinterpret_cast<const uint8_t*>(mask);
  p.weights = reinterpret_cast<float*>(weights);
  p.ids = reinterpret_cast<int32_t*>(ids);
  p.tokens = tokens;
  p.experts = experts;
  p.top_k = top_k;
  p.dtype = dtype;
  p.sigmoid = sigmoid;
  p.groups = groups;
  p.top_groups = top_groups;
  p.group_max = group_max;
  p.renormalize = renormalize;
  p.scale = scale;
  const int rc = check(p);
  if (rc) return rc;
  TCCL_CHECK_ARG(groups >= 1 && groups <= 32 && experts % groups == 0,
                 "groups must be 1..32 and divide the experts");
  TCCL_CHECK_ARG(top_groups >= 1 && top_groups <= groups, "top_groups must be 1..groups");
  p.fast = (groups & (groups - 1)) == 0 ? 1 : 0;
  if (tokens == 0) return kOk;
  TCCL_CHECK_ARG(logits != 0 && weights != 0 && ids != 0, "null argument");
  TCCL_CHECK_CUDA(dispatch(p, false, reinterpret_cast<cudaStream_t>(stream)));
  return kOk;
}

extern "C" int tccl_expert_route_backward(uint64_t grad_weights, uint64_t logits, int64_t ld,
                                          uint64_t ids, uint64_t grad_logits, int64_t tokens,
                                          int32_t experts, int32_t top_k, int32_t dtype,
                                          int32_t sigmoid, int32_t renormalize, float scale,
                                          uint64_t stream) {
  RouteParams p = {};
  p.logits = reinterpret_cast<const void*>(logits);
  p.ld = ld;
  p.ids = reinterpret_cast<int32_t*>(ids);
  p.grad_weights = reinterpret_cast<const float*>(grad_weights);
  p.grad_logits = reinterpret_cast<void*>(grad_logits);
  p.tokens = tokens;
  p.experts = experts;
  p.top_k = top_k;
  p.dtype = dtype;
  p.sigmoid = sigmoid;
  p.groups = p.fast = 1;
  p.renormalize = renormalize;
  p.scale = scale;
  const int rc = check(p);
  if (rc) return rc;
  if (tokens == 0) return kOk;
  TCCL_CHECK_ARG(logits != 0 && ids != 0 && grad_weights != 0 && grad_logits != 0, "null argument");
  TCCL_CHECK_CUDA(dispatch(p, true, reinterpret_cast<cudaStream_t>(stream)));
  return kOk;
}
