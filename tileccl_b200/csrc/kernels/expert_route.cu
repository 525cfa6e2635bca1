// Routing of tokens to experts: scores of a row of logits, the choice of the k best experts
// (optionally steered by a per-expert bias and limited to the best groups of experts), their
// weights, and the gradient of the logits.
//
//   p = softmax(l)  or  p = 1 / (1 + e^-l);   key = p + bias;   ids = the k largest keys
//   w_j = scale * p[id_j]  or, renormalised,  scale * p[id_j] / sum_i p[id_i]
//
// One warp per token; lane i holds experts i, i + 32, ...
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include "../api.h"
#include "../runtime/errors.h"

namespace tileccl {
namespace {

constexpr int kWarpsPerCta = 4;
constexpr uint32_t kAll = 0xffffffffu;

enum RouteDtype : int { kF16 = 0, kBF16 = 1, kF32 = 2 };

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
  return l > 0.f ? 1.f / (1.f + expf(-l)) : expf(l - s) / (1.f + expf(l));
}

// Keys are compared as unsigned integers of the same order.  0 = the expert is not available
// (logit or bias of -inf, or outside the chosen groups); 1 = the key is not a number: it ranks
// behind every number, so ids stay distinct and in range.
__device__ __forceinline__ uint64_t order_key(double x) {
  if (x != x) return 1;
  if (x == -CUDART_INF) return 0;
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(x == 0.0 ? 0.0 : x));
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}

template <int EPL>
__global__ void __launch_bounds__(kWarpsPerCta * 32)
expert_route_kernel(const RouteParams p) {
  extern __shared__ double smem_keys[];   // [warps][experts], only used with groups
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kWarpsPerCta + warp;
  if (t >= p.tokens) return;
  float* const out_w = p.weights + t * p.top_k;
  int32_t* const out_i = p.ids + t * p.top_k;
  if (p.mask != nullptr && p.mask[t] == 0) {
    if (lane < p.top_k) { out_w[lane] = 0.f; out_i[lane] = -1; }
    return;
  }
  float l[EPL];
  bool nan_row = false;
  float m = -CUDART_INF_F;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane + 32 * i;
    l[i] = e < p.experts ? load_logit(p.logits, t * p.ld + e, p.dtype) : -CUDART_INF_F;
    nan_row = nan_row || l[i] != l[i];
    m = fmaxf(m, l[i]);
  }
  nan_row = __any_sync(kAll, nan_row);
  m = warp_max(m);

  // The choice is made on 64-bit keys: scores of two experts may differ by less than a 32-bit
  // exponential can tell.  Without a bias the score grows with the logit, which is then the key.
  const bool by_logit = p.bias == nullptr && (p.groups == 1 || p.group_max != 0);
  double key[EPL];
  double total = 0.0;
  if (!by_logit) {
    double part = 0.0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      key[i] = p.sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(l[i])))
                         : exp(static_cast<double>(l[i]) - static_cast<double>(m));
      part += key[i];
    }
    total = warp_sum(part);
  }
  uint64_t rank[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane + 32 * i;
    double k = by_logit ? static_cast<double>(l[i]) : p.sigmoid ? key[i] : key[i] / total;
    if (p.bias != nullptr && e < p.experts) k += static_cast<double>(p.bias[e]);
    key[i] = k;
    rank[i] = (e >= p.experts || l[i] == -CUDART_INF_F) ? 0 : order_key(k);
  }
  if (p.groups > 1) {
    double* const mine = smem_keys + static_cast<int64_t>(warp) * p.experts;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = lane + 32 * i;
      if (e < p.experts) mine[e] = rank[i] == 0 ? -CUDART_INF : key[i];
    }
    __syncwarp();
    const int per = p.experts / p.groups;
    // lane g: score of group g = its largest key, or the sum of its two largest available keys
    uint64_t score = 0;
    if (lane < p.groups) {
      double a = -CUDART_INF, b = -CUDART_INF;
      bool bad = false;
      for (int i = 0; i < per; ++i) {
        const double x = mine[lane * per + i];
        if (x != x) bad = true;
        else if (x > a) { b = a; a = x; }
        else if (x > b) b = x;
      }
      const double s = p.group_max || b == -CUDART_INF ? a : a + b;
      score = a == -CUDART_INF ? (bad ? 1 : 0) : order_key(s);
    }
    int ahead = 0;
    for (int g = 0; g < p.groups; ++g) {
      const uint64_t other = __shfl_sync(kAll, score, g);
      ahead += (other > score || (other == score && g < lane)) ? 1 : 0;
    }
    const uint32_t keep = __ballot_sync(kAll, lane < p.groups && ahead < p.top_groups);
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = lane + 32 * i;
      if (e < p.experts && ((keep >> (e / per)) & 1u) == 0) rank[i] = 0;
    }
  }

  // k rounds: the warp's best remaining expert, the lowest index among equals
  int my_id = -1;
  float my_l = -CUDART_INF_F;
  for (int j = 0; j < p.top_k; ++j) {
    uint64_t best = 0;
    int at = -1;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (rank[i] > best) { best = rank[i]; at = i; }
    const uint64_t top = warp_max(best);
    if (top == 0) break;
    const uint32_t cand = best == top ? static_cast<uint32_t>(lane + 32 * at) : kAll;
    const uint32_t id = __reduce_min_sync(kAll, cand);
    float chosen = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (lane + 32 * i == static_cast<int>(id)) { rank[i] = 0; chosen = l[i]; }
    chosen = __shfl_sync(kAll, chosen, id & 31);
    if (lane == j) { my_id = static_cast<int>(id); my_l = chosen; }
  }

  // weights: lane j holds the j-th choice
  float w = 0.f;
  if (p.renormalize) {
    const float top = warp_max(my_l);
    const float s = my_id < 0 ? 0.f : p.sigmoid ? sigmoid_scaled(my_l, top) : expf(my_l - top);
    const float sum = warp_sum(s);
    w = s / sum;
  } else if (p.sigmoid) {
    w = sigmoid_f(my_l);
  } else {
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) part += lane + 32 * i < p.experts ? expf(l[i] - m) : 0.f;
    const float sum = warp_sum(part);
    w = expf(my_l - m) / sum;
  }
  w *= p.scale;
  if (nan_row || (!p.sigmoid && m == CUDART_INF_F)) w = CUDART_NAN_F;   // as the formula has it
  if (my_id < 0) w = 0.f;
  if (lane < p.top_k) { out_w[lane] = w; out_i[lane] = my_id; }
}

// dL/dl of a row from dL/dw of its k weights.  With n_j = w_j / scale and g_j = dL/dw_j:
//   softmax, renormalised   dl_i = scale n_i (g_i - sum_j g_j n_j)              i chosen
//   softmax                 dl_i = scale p_i (g_i [i chosen] - sum_j g_j p_j)   every i
//   sigmoid, renormalised   dl_i = scale n_i (1 - p_i) (g_i - sum_j g_j n_j)    i chosen
//   sigmoid                 dl_i = scale g_i p_i (1 - p_i)                      i chosen
template <int EPL>
__global__ void __launch_bounds__(kWarpsPerCta * 32)
expert_route_backward_kernel(const RouteParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kWarpsPerCta + warp;
  if (t >= p.tokens) return;
  int id = -1;
  float g = 0.f;
  if (lane < p.top_k) {
    id = p.ids[t * p.top_k + lane];
    if (id < 0 || id >= p.experts) id = -1;
    else g = p.grad_weights[t * p.top_k + lane];
  }
  const bool routed = __any_sync(kAll, id >= 0);
  float l[EPL];
  float m = -CUDART_INF_F;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane + 32 * i;
    l[i] = routed && e < p.experts ? load_logit(p.logits, t * p.ld + e, p.dtype) : -CUDART_INF_F;
    m = fmaxf(m, l[i]);
  }
  m = warp_max(m);
  float prob[EPL];
  float sum = 0.f;
  if (!p.sigmoid && !p.renormalize) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      prob[i] = l[i] == -CUDART_INF_F ? 0.f : expf(l[i] - m);
      sum += prob[i];
    }
    sum = warp_sum(sum);
  }
  const float my_l = id >= 0 ? load_logit(p.logits, t * p.ld + id, p.dtype) : -CUDART_INF_F;
  float n = 0.f;
  if (p.renormalize) {
    const float top = warp_max(my_l);
    const float s = id < 0 || my_l == -CUDART_INF_F ? 0.f
                    : p.sigmoid ? sigmoid_scaled(my_l, top) : expf(my_l - top);
    const float all = warp_sum(s);
    n = all > 0.f || all != all ? s / all : 0.f;
  } else if (id >= 0) {
    n = p.sigmoid ? sigmoid_f(my_l) : my_l == -CUDART_INF_F ? 0.f : expf(my_l - m) / sum;
  }
  const float dot = p.sigmoid && !p.renormalize ? 0.f : warp_sum(id >= 0 ? g * n : 0.f);
  // lane j's share of dl at its expert; the dense softmax adds -p_i * dot everywhere
  float mine = p.scale * n * (!p.sigmoid && !p.renormalize ? g : g - dot);
  if (p.sigmoid) mine *= sigmoid_f(-my_l);
  if (id < 0 || my_l == -CUDART_INF_F) mine = 0.f;
  float d[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    d[i] = 0.f;
    if (!p.sigmoid && !p.renormalize && routed && l[i] != -CUDART_INF_F)
      d[i] = -p.scale * (prob[i] / sum) * dot;
  }
  for (int j = 0; j < p.top_k; ++j) {
    const int e = __shfl_sync(kAll, id, j);
    const float v = __shfl_sync(kAll, mine, j);
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (e == lane + 32 * i) d[i] += v;
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane + 32 * i;
    if (e < p.experts) store_logit(p.grad_logits, t * p.experts + e, p.dtype, d[i]);
  }
}

template <int EPL>
cudaError_t launch(const RouteParams& p, bool backward, cudaStream_t s) {
  const int64_t blocks = (p.tokens + kWarpsPerCta - 1) / kWarpsPerCta;
  if (backward) {
    expert_route_backward_kernel<EPL><<<static_cast<unsigned>(blocks), kWarpsPerCta * 32, 0, s>>>(p);
  } else {
    const size_t smem = p.groups > 1 ? sizeof(double) * kWarpsPerCta * p.experts : 0;
    expert_route_kernel<EPL><<<static_cast<unsigned>(blocks), kWarpsPerCta * 32, smem, s>>>(p);
  }
  return cudaGetLastError();
}

cudaError_t dispatch(const RouteParams& p, bool backward, cudaStream_t s) {
  const int epl = (p.experts + 31) / 32;
  if (epl <= 1) return launch<1>(p, backward, s);
  if (epl <= 2) return launch<2>(p, backward, s);
  if (epl <= 4) return launch<4>(p, backward, s);
  if (epl <= 8) return launch<8>(p, backward, s);
  return launch<16>(p, backward, s);
}

int check(const RouteParams& p) {
  TCCL_CHECK_ARG(p.tokens >= 0 && p.tokens < (int64_t(1) << 31), "tokens out of range");
  TCCL_CHECK_ARG(p.experts >= 1 && p.experts <= 512, "experts must be 1..512");
  TCCL_CHECK_ARG(p.top_k >= 1 && p.top_k <= 32 && p.top_k <= p.experts,
                 "top_k must be 1..min(32, experts)");
  TCCL_CHECK_ARG(p.dtype >= 0 && p.dtype <= 2, "dtype must be 0 (fp16), 1 (bf16) or 2 (fp32)");
  TCCL_CHECK_ARG(p.ld >= p.experts || p.tokens <= 1, "row pitch is smaller than a row");
  return kOk;
}

}  // namespace

cudaError_t preload_expert_route_kernels() {
  cudaFuncAttributes a;
  cudaError_t e = cudaFuncGetAttributes(&a, expert_route_kernel<8>);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, expert_route_backward_kernel<8>);
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
  p.groups = 1;
  p.renormalize = renormalize;
  p.scale = scale;
  const int rc = check(p);
  if (rc) return rc;
  if (tokens == 0) return kOk;
  TCCL_CHECK_ARG(logits != 0 && ids != 0 && grad_weights != 0 && grad_logits != 0, "null argument");
  TCCL_CHECK_CUDA(dispatch(p, true, reinterpret_cast<cudaStream_t>(stream)));
  return kOk;
}
