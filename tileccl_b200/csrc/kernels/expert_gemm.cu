// Products of the experts over a slot map (expert_slots.cu): every slot's row times the weight
// matrix of its expert, and the gradient of those weights.
//
//   out[s] = x[row(s)] @ W[e(s)]                                row(s) = token of slot s, or s
//   SiLU gate: W's columns come as 128 gate columns followed by 128 up columns;
//              out[s] = silu(gate) * up, half as wide
//   gradient of the gate: gate and up are computed again and with dh[s] = dL/dout[s]
//              dgate = dh * up * sg * (1 + gate * (1 - sg)),  dup = dh * gate * sg,
//              sg = 1 / (1 + e^-gate), packed like W's columns
//   dW[e] = sum over the slots of e of x[row(s)]^T dy[s]
//
// 64 x 64 tiles, fp32 accumulation on the CUDA cores.
#include <cuda_runtime.h>

#include "../api.h"
#include "../device/tile_compute.cuh"
#include "../runtime/errors.h"

namespace tileccl {
namespace {

enum Epilogue : int { kNone = 0, kSiluGate = 1, kSiluGateGrad = 2 };

__device__ __forceinline__ float load16(const void* base, int64_t i, bool bf16) {
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i])
              : __half2float(static_cast<const __half*>(base)[i]);
}
__device__ __forceinline__ void store16(void* base, int64_t i, bool bf16, float v) {
  if (bf16) static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16(v);
  else static_cast<__half*>(base)[i] = __float2half(v);
}

__device__ __forceinline__ int slot_bound(const TcclExpertGemm& d, int e) {
  const int v = reinterpret_cast<const int32_t*>(d.offsets)[e];
  return v < 0 ? 0 : v > d.slots ? static_cast<int>(d.slots) : v;
}
__device__ __forceinline__ int64_t source_row(const TcclExpertGemm& d, int s) {
  if (d.token_of_slot == 0) return s;
  const int t = reinterpret_cast<const int32_t*>(d.token_of_slot)[s];
  return t >= 0 && t < d.x_rows ? t : 0;
}

__global__ void __launch_bounds__(256) expert_gemm_kernel(const TcclExpertGemm d) {
  __shared__ float xs[16][65], ws[16][65], us[16][65];
  __shared__ int tile_e, tile_row, tile_end;
  const bool bf16 = d.dtype == 1;
  if (threadIdx.x == 0) {
    int left = blockIdx.y;
    tile_e = -1;
    for (int e = 0; e < d.experts; ++e) {
      const int a = slot_bound(d, e), b = slot_bound(d, e + 1);
      const int tiles = b > a ? (b - a + 63) / 64 : 0;
      if (left < tiles) { tile_e = e; tile_row = a + left * 64; tile_end = b; break; }
      left -= tiles;
    }
  }
  __syncthreads();
  if (tile_e < 0) return;
  const bool gate = d.epilogue != kNone;
  const int n_cols = static_cast<int>(gate ? d.n / 2 : d.n);
  const int f0 = blockIdx.x * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {}, up[4][4] = {};
  const void* x = reinterpret_cast<const void*>(d.x);
  const void* w = reinterpret_cast<const void*>(d.w);
  for (int64_t k0 = 0; k0 < d.k; k0 += 16) {
    for (int i = threadIdx.x; i < 16 * 64; i += 256) {
      const int kk = i & 15, r = i >> 4;
      const int s = tile_row + r;
      xs[kk][r] = s < tile_end && k0 + kk < d.k ? load16(x, source_row(d, s) * d.ldx + k0 + kk, bf16) : 0.f;
      const int f = f0 + r;
      const int64_t c = gate ? (f / 128) * 256 + f % 128 : f;
      const bool ok = f < n_cols && k0 + kk < d.k;
      auto at = [&](int64_t col) {
        return tile_e * d.w_expert + (d.w_nk ? col * d.ldw + k0 + kk : (k0 + kk) * d.ldw + col);
      };
      ws[kk][r] = ok ? load16(w, at(c), bf16) : 0.f;
      us[kk][r] = ok && gate ? load16(w, at(c + 128), bf16) : 0.f;
    }
    __syncthreads();
    for (int kk = 0; kk < 16; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[i][j] = fmaf(xs[kk][ty * 4 + i], ws[kk][tx * 4 + j], acc[i][j]);
          if (gate) up[i][j] = fmaf(xs[kk][ty * 4 + i], us[kk][tx * 4 + j], up[i][j]);
        }
    __syncthreads();
  }
  void* out = reinterpret_cast<void*>(d.out);
  for (int i = 0; i < 4; ++i) {
    const int64_t s = tile_row + ty * 4 + i;
    if (s >= tile_end) continue;
    for (int j = 0; j < 4; ++j) {
      const int f = f0 + tx * 4 + j;
      if (f >= n_cols) continue;
      const float g = acc[i][j], u = up[i][j];
      const float sg = 1.f / (1.f + __expf(-g));
      if (d.epilogue == kNone) {
        store16(out, s * d.ldo + f, bf16, g);
      } else if (d.epilogue == kSiluGate) {
        store16(out, s * d.ldo + f, bf16, g * sg * u);
      } else {
        const int64_t c = (f / 128) * 256 + f % 128;
        const float dh = load16(reinterpret_cast<const void*>(d.dh), s * d.ld_dh + f, bf16);
        store16(out, s * d.ldo + c, bf16, dh * u * sg * (1.f + g * (1.f - sg)));
        store16(out, s * d.ldo + c + 128, bf16, dh * g * sg);
      }
    }
  }
}

// out[e][i][j] = sum over the slots of e of a[row(s)][i] * b[row'(s)][j]; one of the operands
// is gathered by token (gather_a / gather_b).
__global__ void __launch_bounds__(256) expert_weight_grad_kernel(const TcclExpertWeightGrad d) {
  __shared__ float as[16][65], bs[16][65];
  const bool bf16 = d.dtype == 1;
  const int e = blockIdx.z;
  const int32_t* offsets = reinterpret_cast<const int32_t*>(d.offsets);
  auto bound = [&](int i) { const int v = offsets[i]; return v < 0 ? 0 : v > d.slots ? static_cast<int>(d.slots) : v; };
  const int s0 = bound(e), s1 = bound(e + 1);
  const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int32_t* tok = reinterpret_cast<const int32_t*>(d.token_of_slot);
  auto row = [&](int s, bool gather, int64_t rows) -> int64_t {
    if (!gather) return s;
    const int t = tok[s];
    return t >= 0 && t < rows ? t : 0;
  };
  float acc[4][4] = {};
  for (int s = s0; s < s1; s += 16) {
    for (int i = threadIdx.x; i < 16 * 64; i += 256) {
      const int c = i & 63, r = i >> 6;
      const bool ok = s + r < s1;
      as[r][c] = ok && i0 + c < d.m ? load16(reinterpret_cast<const void*>(d.a),
                                             row(s + r, d.gather_a, d.a_rows) * d.lda + i0 + c, bf16) : 0.f;
      bs[r][c] = ok && j0 + c < d.n ? load16(reinterpret_cast<const void*>(d.b),
                                             row(s + r, d.gather_b, d.b_rows) * d.ldb + j0 + c, bf16) : 0.f;
    }
    __syncthreads();
    for (int kk = 0; kk < 16; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(as[kk][ty * 4 + i], bs[kk][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t r = i0 + ty * 4 + i, c = j0 + tx * 4 + j;
      if (r < d.m && c < d.n)
        store16(reinterpret_cast<void*>(d.out), (e * d.m + r) * d.n + c, bf16, acc[i][j]);
    }
}

}  // namespace

cudaError_t preload_expert_gemm_kernels() {
  cudaFuncAttributes a;
  cudaError_t e = cudaFuncGetAttributes(&a, expert_gemm_kernel);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, expert_weight_grad_kernel);
  return e;
}

}  // namespace tileccl

using namespace tileccl;

extern "C" int tccl_expert_gemm(const TcclExpertGemm* desc, uint64_t stream) {
  TCCL_CHECK_ARG(desc != nullptr, "null argument");
  const TcclExpertGemm& d = *desc;
  TCCL_CHECK_ARG(d.dtype == 0 || d.dtype == 1, "dtype must be 0 (fp16) or 1 (bf16)");
  TCCL_CHECK_ARG(d.epilogue >= kNone && d.epilogue <= kSiluGateGrad, "epilogue must be 0..2");
  TCCL_CHECK_ARG(d.experts >= 1 && d.experts <= 1024, "experts must be 1..1024");
  TCCL_CHECK_ARG(d.k >= 1 && d.n >= 1, "empty problem");
  TCCL_CHECK_ARG(d.k % 8 == 0, "K must be a multiple of 8 (16-byte TMA rows)");
  TCCL_CHECK_ARG(d.n % 8 == 0, "N must be a multiple of 8 (16-byte TMA rows)");
  TCCL_CHECK_ARG(d.ldx % 8 == 0 && d.ldw % 8 == 0 && d.w_expert % 8 == 0 && d.ldo % 8 == 0 &&
                     d.ld_dh % 8 == 0,
                 "leading dimensions must be multiples of 8 elements");
  TCCL_CHECK_ARG(d.x % 16 == 0 && d.w % 16 == 0 && d.out % 16 == 0 && d.dh % 16 == 0,
                 "operands must be 16-byte aligned");
  TCCL_CHECK_ARG(d.epilogue == kNone || d.n % 256 == 0,
                 "SiLU-gate epilogue needs N to be a multiple of 256");
  TCCL_CHECK_ARG(d.slots >= 0 && d.slots < (int64_t(1) << 31) && d.x_rows < (int64_t(1) << 31),
                 "too many rows");
  if (d.slots == 0) return kOk;
  TCCL_CHECK_ARG(d.x != 0 && d.w != 0 && d.out != 0 && d.offsets != 0 && d.x_rows >= 1, "null argument");
  TCCL_CHECK_ARG(d.epilogue != kSiluGateGrad || d.dh != 0, "null argument");
  const int64_t cols = d.epilogue == kNone ? d.n : d.n / 2;
  const int64_t tiles = d.slots / 64 + (d.slots < d.experts ? d.slots : d.experts);
  const dim3 grid(static_cast<unsigned>((cols + 63) / 64), static_cast<unsigned>(tiles));
  expert_gemm_kernel<<<grid, 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(d);
  TCCL_CHECK_CUDA(cudaGetLastError());
  return kOk;
}

extern "C" int tccl_expert_weight_grad(const TcclExpertWeightGrad* desc, uint64_t stream) {
  TCCL_CHECK_ARG(desc != nullptr, "null argument");
  const TcclExpertWeightGrad& d = *desc;
  TCCL_CHECK_ARG(d.dtype == 0 || d.dtype == 1, "dtype must be 0 (fp16) or 1 (bf16)");
  TCCL_CHECK_ARG(d.experts >= 1 && d.experts <= 1024, "experts must be 1..1024");
  TCCL_CHECK_ARG(d.m >= 1 && d.n >= 1, "empty problem");
  TCCL_CHECK_ARG(d.m % 8 == 0 && d.n % 8 == 0, "rows and columns must be multiples of 8");
  TCCL_CHECK_ARG(d.lda % 8 == 0 && d.ldb % 8 == 0, "leading dimensions must be multiples of 8 elements");
  TCCL_CHECK_ARG(d.a % 16 == 0 && d.b % 16 == 0 && d.out % 16 == 0, "operands must be 16-byte aligned");
  TCCL_CHECK_ARG(d.slots >= 0 && d.slots < (int64_t(1) << 31) && d.a_rows < (int64_t(1) << 31) &&
                     d.b_rows < (int64_t(1) << 31), "too many rows");
  TCCL_CHECK_ARG(d.out != 0 && d.offsets != 0, "null argument");
  TCCL_CHECK_ARG(d.slots == 0 || (d.a != 0 && d.b != 0 && d.a_rows >= 1 && d.b_rows >= 1), "null argument");
  TCCL_CHECK_ARG(!(d.gather_a || d.gather_b) || d.slots == 0 || d.token_of_slot != 0, "null argument");
  const dim3 grid(static_cast<unsigned>((d.n + 63) / 64), static_cast<unsigned>((d.m + 63) / 64),
                  static_cast<unsigned>(d.experts));
  expert_weight_grad_kernel<<<grid, 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(d);
  TCCL_CHECK_CUDA(cudaGetLastError());
  return kOk;
}
