// Weighted sum of a token's expert outputs and its gradient, and tokens' rows in slot order.
//
//   y[t] = add[t] + sum_j w[t][j] * h[slot_of[t][j]]        (choices without a slot add nothing;
//                                                           h in 16 bits or in fp32)
//   dh[slot_of[t][j]] = w[t][j] * dy[t]      dw[t][j] = <dy[t], h[slot_of[t][j]]>
//
// Sums run in fp32 in the order of the choices and are rounded once.  All three kernels are bound by
// DRAM and move 16 bytes per thread and access; CTAs of 128 threads keep the most loads in flight
// (256 threads: backward of 4096 x 8 rows of 4096 107 us instead of 90).
#include <cuda_runtime.h>

#include "../api.h"
#include "../device/symm_ptr.cuh"
#include "../device/tile_compute.cuh"
#include "../runtime/errors.h"

namespace tileccl {
namespace {

constexpr int kThreads = 128;

struct CombineParams {
  const uint4* h;            // [slots] rows of `n` 16-bit or fp32 values
  int64_t h_ld;              // 16-byte vectors between rows, likewise below
  const int32_t* slot_of;    // [tokens][top_k]
  const float* weights;      // [tokens][top_k] or null (all ones)
  const uint4* add;          // [tokens] rows or null
  int64_t add_ld;
  uint4* out;                // forward
  int64_t out_ld;
  const uint4* dy;           // backward
  int64_t dy_ld;
  uint4* dh;
  int64_t dh_ld;
  float* dw;
  int64_t tokens, slots;
  int32_t top_k, vecs, bf16;   // vecs: 16-byte vectors per row
};

// A thread sums kVecs pieces of eight values of a token's row, kThreads apart.  The rows of H are
// fetched kBatch at a time: their slots first, then all of their pieces, in flight together;
// kBatch * kVecs is 8 (4 with fp32 rows), which is what the registers of a full SM have room for.
// 16384 x 8 rows of 4096, a quarter of them elsewhere: 151 us, 6.2 TB/s; 4096 x 2 rows: 15 us with
// batches of two, 30 with batches of eight, of which two were in use.
template <int kBatch, bool kFloatRows>
__global__ void __launch_bounds__(kThreads) expert_combine_kernel(const CombineParams p) {
  constexpr int kVecs = (kFloatRows ? 4 : 8) / kBatch;
  constexpr int kWords = kFloatRows ? 2 : 1;               // 16-byte vectors per piece
  const int64_t t = blockIdx.x;
  const int v0 = blockIdx.y * (kThreads * kVecs) + threadIdx.x;
  const bool bf16 = p.bf16 != 0;
  float acc[kVecs][8] = {};
#pragma unroll
  for (int c = 0; c < kVecs; ++c)
    if (p.add != nullptr && v0 + c * kThreads < p.vecs)
      tile_accumulate_16x8(bf16, acc[c], p.add[t * p.add_ld + v0 + c * kThreads]);
  for (int j0 = 0; j0 < p.top_k; j0 += kBatch) {
    int32_t s[kBatch];
    float w[kBatch];
    uint4 x[kBatch][kVecs][kWords];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      s[j] = j0 + j < p.top_k ? p.slot_of[t * p.top_k + j0 + j] : -1;
      if (s[j] >= p.slots) s[j] = -1;
      w[j] = s[j] < 0 ? 0.f : p.weights != nullptr ? p.weights[t * p.top_k + j0 + j] : 1.f;
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
#pragma unroll
      for (int c = 0; c < kVecs; ++c)
        if (s[j] >= 0 && v0 + c * kThreads < p.vecs) {
          const uint4* src = p.h + s[j] * p.h_ld + (v0 + c * kThreads) * kWords;
#pragma unroll
          for (int i = 0; i < kWords; ++i) x[j][c][i] = ld_stream_v4(src + i);
        }
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (s[j] >= 0) {
#pragma unroll
        for (int c = 0; c < kVecs; ++c) {
          float f[8] = {};
          if (kFloatRows) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
              f[4 * i] = __uint_as_float(x[j][c][i].x);
              f[4 * i + 1] = __uint_as_float(x[j][c][i].y);
              f[4 * i + 2] = __uint_as_float(x[j][c][i].z);
              f[4 * i + 3] = __uint_as_float(x[j][c][i].w);
            }
          } else {
            tile_accumulate_16x8(bf16, f, x[j][c][0]);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[c][i] = fmaf(w[j], f[i], acc[c][i]);
        }
      }
  }
#pragma unroll
  for (int c = 0; c < kVecs; ++c)
    if (v0 + c * kThreads < p.vecs)
      p.out[t * p.out_ld + v0 + c * kThreads] = tile_cast_f32x8(bf16, acc[c]);
}

// One CTA per token.  A batch of choices at a time: dy stays in registers, every row of H is
// read once, and the dot products of the batch meet in one reduction.  4096 x 8 rows of 4096: 90
// us, 6.3 TB/s.
template <int kBatch>
__global__ void __launch_bounds__(kThreads) expert_combine_backward_kernel(const CombineParams p) {
  __shared__ float part[kThreads / 32][kBatch];
  const int64_t t = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool bf16 = p.bf16 != 0;
  for (int j0 = 0; j0 < p.top_k; j0 += kBatch) {
    int32_t s[kBatch];
    float w[kBatch], dot[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      s[j] = j0 + j < p.top_k ? p.slot_of[t * p.top_k + j0 + j] : -1;
      if (s[j] >= p.slots) s[j] = -1;
      w[j] = s[j] >= 0 ? p.weights[t * p.top_k + j0 + j] : 0.f;
      dot[j] = 0.f;
    }
    for (int v = threadIdx.x; v < p.vecs; v += kThreads) {
      uint4 x[kBatch];
      const uint4 dy = p.dy[t * p.dy_ld + v];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (s[j] >= 0) x[j] = p.h[s[j] * p.h_ld + v];
      float g[8] = {};
      tile_accumulate_16x8(bf16, g, dy);
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (s[j] >= 0) {
          float f[8] = {};
          tile_accumulate_16x8(bf16, f, x[j]);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            dot[j] = fmaf(g[i], f[i], dot[j]);
            f[i] = g[i] * w[j];
          }
          p.dh[s[j] * p.dh_ld + v] = tile_cast_f32x8(bf16, f);
        }
    }
    if (j0 > 0) __syncthreads();                 // `part` of the previous batch has been read
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
      if (lane == 0) part[warp][j] = dot[j];
    }
    __syncthreads();
    if (threadIdx.x < kBatch && j0 + threadIdx.x < p.top_k) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) sum += part[i][threadIdx.x];
      p.dw[t * p.top_k + j0 + threadIdx.x] = sum;
    }
  }
}

// out[s] = x[token of slot s]; zeros for a token that does not exist, nothing behind the last
// slot (token -1).  A CTA takes kGatherRows rows, so that as many vectors per thread are in
// flight: 8192 rows of 4096 from 4096 tokens in 16 us (6.3 TB/s).
constexpr int kGatherRows = 4;

__global__ void __launch_bounds__(kThreads) expert_gather_kernel(
    const uint4* x, int64_t x_ld, int64_t x_rows, const int32_t* token_of_slot, uint4* out,
    int64_t out_ld, int64_t slots, int32_t vecs) {
  // a product that reads the rows may set itself up meanwhile (it waits for this kernel's end)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t s0 = static_cast<int64_t>(blockIdx.x) * kGatherRows;
  const int v = blockIdx.y * kThreads + threadIdx.x;
  if (v >= vecs) return;
  int32_t t[kGatherRows];
  uint4 r[kGatherRows];
#pragma unroll
  for (int i = 0; i < kGatherRows; ++i) t[i] = s0 + i < slots ? token_of_slot[s0 + i] : -1;
#pragma unroll
  for (int i = 0; i < kGatherRows; ++i)
    r[i] = t[i] >= 0 && t[i] < x_rows ? x[t[i] * x_ld + v] : make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < kGatherRows; ++i)
    if (t[i] >= 0) out[(s0 + i) * out_ld + v] = r[i];
}

int check(const CombineParams& p) {
  TCCL_CHECK_ARG(p.tokens >= 0 && p.tokens < (int64_t(1) << 31), "tokens out of range");
  TCCL_CHECK_ARG(p.top_k >= 1 && p.vecs >= 1, "empty rows");
  TCCL_CHECK_ARG(p.vecs <= 65535 * kThreads, "rows are too long");
  return kOk;
}

}  // namespace

cudaError_t preload_expert_combine_kernels() {
  cudaFuncAttributes a;
  cudaError_t e = cudaFuncGetAttributes(&a, expert_combine_kernel<8, false>);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, expert_combine_kernel<4, false>);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, expert_combine_kernel<2, false>);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, expert_combine_kernel<4, true>);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, expert_combine_kernel<2, true>);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, expert_combine_backward_kernel<8>);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, expert_combine_backward_kernel<4>);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, expert_combine_backward_kernel<2>);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, expert_gather_kernel);
  return e;
}

}  // namespace tileccl

using namespace tileccl;

extern "C" int tccl_expert_combine(uint64_t h, int64_t h_ld, uint64_t slot_of, uint64_t weights,
                                   uint64_t add, int64_t add_ld, uint64_t out, int64_t out_ld,
                                   int64_t tokens, int64_t slots, int32_t top_k, int32_t n,
                                   int32_t dtype, int32_t h_float, uint64_t stream) {
  TCCL_CHECK_ARG(dtype == 0 || dtype == 1, "dtype must be 0 (fp16) or 1 (bf16)");
  TCCL_CHECK_ARG(n % 8 == 0 && h_ld % 8 == 0 && add_ld % 8 == 0 && out_ld % 8 == 0,
                 "row lengths and pitches must be multiples of 8 elements");
  TCCL_CHECK_ARG(h % 16 == 0 && add % 16 == 0 && out % 16 == 0, "rows must be 16-byte aligned");
  CombineParams p = {};
  p.h = reinterpret_cast<const uint4*>(h);
  p.h_ld = h_float ? h_ld / 4 : h_ld / 8;
  p.slot_of = reinterpret_cast<const int32_t*>(slot_of);
  p.weights = reinterpret_cast<const float*>(weights);
  p.add = reinterpret_cast<const uint4*>(add);
  p.add_ld = add_ld / 8;
  p.out = reinterpret_cast<uint4*>(out);
  p.out_ld = out_ld / 8;
  p.tokens = tokens;
  p.slots = slots;
  p.top_k = top_k;
  p.vecs = n / 8;
  p.bf16 = dtype;
  const int rc = check(p);
  if (rc) return rc;
  if (tokens == 0) return kOk;
  TCCL_CHECK_ARG(h != 0 && slot_of != 0 && out != 0, "null argument");
  // (few tokens: narrow pieces, so that a row is spread over more SMs)
  const int most = h_float ? 4 : 8;
  const int batch = tokens < 256 || top_k > most / 2 ? most : top_k > 2 ? 4 : 2;
  const int piece = kThreads * (most / batch);
  const dim3 grid(static_cast<unsigned>(tokens), (p.vecs + piece - 1) / piece);
  const cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
  if (h_float) {
    if (batch == 4) expert_combine_kernel<4, true><<<grid, kThreads, 0, cs>>>(p);
    else expert_combine_kernel<2, true><<<grid, kThreads, 0, cs>>>(p);
  } else {
    if (batch == 8) expert_combine_kernel<8, false><<<grid, kThreads, 0, cs>>>(p);
    else if (batch == 4) expert_combine_kernel<4, false><<<grid, kThreads, 0, cs>>>(p);
    else expert_combine_kernel<2, false><<<grid, kThreads, 0, cs>>>(p);
  }
  TCCL_CHECK_CUDA(cudaGetLastError());
  return kOk;
}

extern "C" int tccl_expert_combine_backward(uint64_t dy, int64_t dy_ld, uint64_t h, int64_t h_ld,
                                            uint64_t slot_of, uint64_t weights, uint64_t dh,
                                            int64_t dh_ld, uint64_t dw, int64_t tokens,
                                            int64_t slots, int32_t top_k, int32_t n, int32_t dtype,
                                            uint64_t stream) {
  TCCL_CHECK_ARG(dtype == 0 || dtype == 1, "dtype must be 0 (fp16) or 1 (bf16)");
  TCCL_CHECK_ARG(n % 8 == 0 && h_ld % 8 == 0 && dy_ld % 8 == 0 && dh_ld % 8 == 0,
                 "row lengths and pitches must be multiples of 8 elements");
  TCCL_CHECK_ARG(h % 16 == 0 && dy % 16 == 0 && dh % 16 == 0, "rows must be 16-byte aligned");
  CombineParams p = {};
  p.h = reinterpret_cast<const uint4*>(h);
  p.h_ld = h_ld / 8;
  p.slot_of = reinterpret_cast<const int32_t*>(slot_of);
  p.weights = reinterpret_cast<const float*>(weights);
  p.dy = reinterpret_cast<const uint4*>(dy);
  p.dy_ld = dy_ld / 8;
  p.dh = reinterpret_cast<uint4*>(dh);
  p.dh_ld = dh_ld / 8;
  p.dw = reinterpret_cast<float*>(dw);
  p.tokens = tokens;
  p.slots = slots;
  p.top_k = top_k;
  p.vecs = n / 8;
  p.bf16 = dtype;
  const int rc = check(p);
  if (rc) return rc;
  if (tokens == 0) return kOk;
  TCCL_CHECK_ARG(h != 0 && slot_of != 0 && weights != 0 && dy != 0 && dh != 0 && dw != 0,
                 "null argument");
  const cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(tokens);
  if (top_k > 4) expert_combine_backward_kernel<8><<<grid, kThreads, 0, cs>>>(p);
  else if (top_k > 2) expert_combine_backward_kernel<4><<<grid, kThreads, 0, cs>>>(p);
  else expert_combine_backward_kernel<2><<<grid, kThreads, 0, cs>>>(p);
  TCCL_CHECK_CUDA(cudaGetLastError());
  return kOk;
}

extern "C" int tccl_expert_gather(uint64_t x, int64_t x_ld, int64_t x_rows, uint64_t token_of_slot,
                                  uint64_t out, int64_t out_ld, int64_t slots, int32_t n,
                                  uint64_t stream) {
  TCCL_CHECK_ARG(n >= 8 && n % 8 == 0 && x_ld % 8 == 0 && out_ld % 8 == 0,
                 "row lengths and pitches must be multiples of 8 elements");
  TCCL_CHECK_ARG(x % 16 == 0 && out % 16 == 0, "rows must be 16-byte aligned");
  TCCL_CHECK_ARG(slots >= 0 && slots < (int64_t(1) << 31), "too many rows");
  const int vecs = n / 8;
  TCCL_CHECK_ARG(vecs <= 65535 * kThreads, "rows are too long");
  if (slots == 0) return kOk;
  TCCL_CHECK_ARG(x != 0 && token_of_slot != 0 && out != 0, "null argument");
  const dim3 grid(static_cast<unsigned>((slots + kGatherRows - 1) / kGatherRows),
                  (vecs + kThreads - 1) / kThreads);
  expert_gather_kernel<<<grid, kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      reinterpret_cast<const uint4*>(x), x_ld / 8, x_rows,
      reinterpret_cast<const int32_t*>(token_of_slot), reinterpret_cast<uint4*>(out), out_ld / 8, slots, vecs);
  TCCL_CHECK_CUDA(cudaGetLastError());
  return kOk;
}
