// Slot map of a routed batch: the (token, choice) pairs in the order of their experts, pairs of
// one expert in the order of their tokens (a stable counting sort, so that every result that
// depends on the order repeats from call to call).
//
//   offsets[e] .. offsets[e + 1]  the slots of expert e       token_of_slot[s]  token of slot s
//   slot_of[t][j]                 slot of token t's j-th choice, -1 when it has none here
//
// The entries are cut into one run per CTA and every run into one segment per warp.  A warp
// counts its segment per expert; the counts are summed over earlier warps, earlier CTAs and
// lower experts; then the warp walks its segment again, 32 entries at a time, and an entry's
// place is that start plus the number of equal entries before it (match_any).
#include <cuda_runtime.h>

#include "../api.h"
#include "../runtime/errors.h"

namespace tileccl {
namespace {

constexpr int kSlotThreads = 512;
constexpr int kSlotWarps = kSlotThreads / 32;
constexpr int kMaxExperts = 1024;
constexpr uint32_t kAll = 0xffffffffu;

struct SlotParams {
  const int32_t* ids;       // [entries]
  int64_t entries;
  int32_t top_k, experts, first;
  int32_t* offsets;         // [experts + 1]
  int32_t* token_of_slot;   // [entries]
  int32_t* slot_of;         // [entries]
  int32_t* counts;          // [CTAs][experts], null with a single CTA
  int64_t run;              // entries per CTA
};

__device__ __forceinline__ int local_expert(const SlotParams& p, int64_t i) {
  const int64_t e = static_cast<int64_t>(p.ids[i]) - p.first;
  return e >= 0 && e < p.experts ? static_cast<int>(e) : -1;
}

// cnt[w][e] = entries of expert e in warp w's segment of this CTA's run
__device__ void count_segments(const SlotParams& p, int64_t begin, int64_t end, int64_t seg,
                               int32_t* cnt) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kSlotWarps * p.experts; i += kSlotThreads) cnt[i] = 0;
  __syncthreads();
  int32_t* const mine = cnt + warp * p.experts;
  const int64_t a = begin + warp * seg, b = a + seg < end ? a + seg : end;
  for (int64_t i = a; i < b; i += 32) {
    const int e = i + lane < b ? local_expert(p, i + lane) : -1;
    if (e >= 0) atomicAdd(mine + e, 1);   // (a sum of ones: its order does not show)
  }
  __syncthreads();
}

__global__ void __launch_bounds__(kSlotThreads) expert_slot_count_kernel(const SlotParams p) {
  extern __shared__ int32_t cnt[];
  const int64_t begin = blockIdx.x * p.run;
  const int64_t end = begin + p.run < p.entries ? begin + p.run : p.entries;
  count_segments(p, begin, end, (p.run + kSlotWarps - 1) / kSlotWarps, cnt);
  for (int e = threadIdx.x; e < p.experts; e += kSlotThreads) {
    int32_t s = 0;
    for (int w = 0; w < kSlotWarps; ++w) s += cnt[w * p.experts + e];
    p.counts[static_cast<int64_t>(blockIdx.x) * p.experts + e] = s;
  }
}

__global__ void __launch_bounds__(kSlotThreads) expert_slot_place_kernel(const SlotParams p) {
  extern __shared__ int32_t cnt[];                 // [warps][experts], then [experts + 1]
  int32_t* const start = cnt + kSlotWarps * p.experts;
  __shared__ int32_t warp_total[kSlotWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t begin = blockIdx.x * p.run;
  const int64_t end = begin + p.run < p.entries ? begin + p.run : p.entries;
  const int64_t seg = (p.run + kSlotWarps - 1) / kSlotWarps;
  count_segments(p, begin, end, seg, cnt);

  // per expert: all entries, and those in the runs of earlier CTAs
  int32_t all[kMaxExperts / kSlotThreads], before[kMaxExperts / kSlotThreads];
  int32_t sum = 0;
#pragma unroll
  for (int i = 0; i < kMaxExperts / kSlotThreads; ++i) {
    const int e = threadIdx.x * (kMaxExperts / kSlotThreads) + i;
    all[i] = before[i] = 0;
    if (e < p.experts) {
      if (p.counts == nullptr) {
        for (int w = 0; w < kSlotWarps; ++w) all[i] += cnt[w * p.experts + e];
      } else {
        for (int b = 0; b < static_cast<int>(gridDim.x); ++b) {
          const int32_t c = p.counts[static_cast<int64_t>(b) * p.experts + e];
          all[i] += c;
          if (b < static_cast<int>(blockIdx.x)) before[i] += c;
        }
      }
    }
    sum += all[i];
  }
  // exclusive scan of `sum` over the threads
  int32_t scan = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int32_t v = __shfl_up_sync(kAll, scan, o);
    if (lane >= o) scan += v;
  }
  if (lane == 31) warp_total[warp] = scan;
  __syncthreads();
  int32_t base = scan - sum;
  for (int w = 0; w < warp; ++w) base += warp_total[w];
#pragma unroll
  for (int i = 0; i < kMaxExperts / kSlotThreads; ++i) {
    const int e = threadIdx.x * (kMaxExperts / kSlotThreads) + i;
    if (e < p.experts) {
      if (blockIdx.x == 0) p.offsets[e] = base;
      int32_t at = base + before[i];
      for (int w = 0; w < kSlotWarps; ++w) {       // counts become starting slots
        const int32_t c = cnt[w * p.experts + e];
        cnt[w * p.experts + e] = at;
        at += c;
      }
      base += all[i];
      if (e == p.experts - 1) start[0] = base;
    }
  }
  __syncthreads();
  const int32_t used = start[0];
  if (blockIdx.x == 0 && threadIdx.x == 0) p.offsets[p.experts] = used;

  int32_t* const mine = cnt + warp * p.experts;
  const int64_t a = begin + warp * seg, b = a + seg < end ? a + seg : end;
  for (int64_t i0 = a; i0 < b; i0 += 32) {
    const int64_t i = i0 + lane;
    const int e = i < b ? local_expert(p, i) : -1;
    const uint32_t same = __match_any_sync(kAll, e);
    const int ahead = __popc(same & ((1u << lane) - 1u));
    int32_t slot = -1;
    if (e >= 0) slot = mine[e] + ahead;
    __syncwarp();
    if (e >= 0 && ahead == 0) mine[e] += __popc(same);
    __syncwarp();
    if (i < b) {
      p.slot_of[i] = slot;
      if (slot >= 0) p.token_of_slot[slot] = static_cast<int32_t>(i / p.top_k);
      // slots behind the last one hold -1 (slot i is written by whoever owns entry i)
      if (i >= used) p.token_of_slot[i] = -1;
    }
  }
}

size_t slot_smem(int experts) { return sizeof(int32_t) * (kSlotWarps * experts + experts + 1); }

cudaError_t attrs_once() {
  static bool done[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || dev >= 64 || done[dev]) return e;
  const int bytes = static_cast<int>(slot_smem(kMaxExperts));
  e = cudaFuncSetAttribute(expert_slot_count_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(expert_slot_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done[dev] = true;
  return e;
}

// Entries one CTA takes; up to this many the map is built by a single launch of one CTA.
constexpr int64_t kRun = 4096;

int64_t slot_ctas(int64_t entries) { return entries <= kRun ? 1 : (entries + kRun - 1) / kRun; }

}  // namespace

cudaError_t preload_expert_slot_kernels() {
  cudaFuncAttributes a;
  cudaError_t e = cudaFuncGetAttributes(&a, expert_slot_count_kernel);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, expert_slot_place_kernel);
  return e;
}

}  // namespace tileccl

using namespace tileccl;

extern "C" int tccl_expert_slots_workspace(int64_t entries, int32_t experts, int64_t* bytes) {
  TCCL_CHECK_ARG(bytes != nullptr, "null argument");
  const int64_t ctas = slot_ctas(entries);
  *bytes = ctas > 1 ? ctas * experts * static_cast<int64_t>(sizeof(int32_t)) : 0;
  return kOk;
}

extern "C" int tccl_expert_slots(uint64_t ids, int64_t tokens, int32_t top_k, int32_t experts,
                                 int32_t first, uint64_t offsets, uint64_t token_of_slot,
                                 uint64_t slot_of, uint64_t workspace, uint64_t stream) {
  TCCL_CHECK_ARG(experts >= 1 && experts <= kMaxExperts, "experts must be 1..1024");
  TCCL_CHECK_ARG(top_k >= 1, "top_k must be at least 1");
  TCCL_CHECK_ARG(tokens >= 0 && tokens * top_k < (int64_t(1) << 31), "too many entries");
  TCCL_CHECK_ARG(offsets != 0, "null argument");
  SlotParams p = {};
  p.ids = reinterpret_cast<const int32_t*>(ids);
  p.entries = tokens * top_k;
  p.top_k = top_k;
  p.experts = experts;
  p.first = first;
  p.offsets = reinterpret_cast<int32_t*>(offsets);
  p.token_of_slot = reinterpret_cast<int32_t*>(token_of_slot);
  p.slot_of = reinterpret_cast<int32_t*>(slot_of);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  TCCL_CHECK_ARG(p.entries == 0 || (ids != 0 && token_of_slot != 0 && slot_of != 0), "null argument");
  const int64_t ctas = slot_ctas(p.entries);
  p.run = ctas == 1 ? (p.entries > 0 ? p.entries : 1) : kRun;
  if (ctas > 1) {
    TCCL_CHECK_ARG(workspace != 0, "this many entries need a workspace");
    p.counts = reinterpret_cast<int32_t*>(workspace);
  }
  TCCL_CHECK_CUDA(attrs_once());
  if (ctas > 1) {
    expert_slot_count_kernel<<<static_cast<unsigned>(ctas), kSlotThreads, slot_smem(experts), s>>>(p);
    TCCL_CHECK_CUDA(cudaGetLastError());
  }
  expert_slot_place_kernel<<<static_cast<unsigned>(ctas), kSlotThreads, slot_smem(experts), s>>>(p);
  TCCL_CHECK_CUDA(cudaGetLastError());
  return kOk;
}
