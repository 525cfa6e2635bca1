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
//
// Bound by latency: a handful of dependent steps per CTA (524288 entries of 128 experts: 10 us in
// two launches, 6 MB moved; 128 entries: 4.3 us in one).
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
  uint32_t entries, top_k;
  int32_t experts, first;
  int32_t* offsets;         // [experts + 1]
  int32_t* token_of_slot;   // [entries]
  int32_t* slot_of;         // [entries]
  int32_t* counts;          // [CTAs][experts], null with a single CTA
  int32_t* totals;          // [experts], null unless `counts` has been summed over the CTAs
};

// Entries a lane keeps: a warp's segment is 32 * kPerLane long, a CTA's run kRun.
constexpr int kPerLane = 8;
constexpr int64_t kRun = kSlotWarps * 32 * kPerLane;

// This lane's first entry.  Entries are counted in 32 bits: there are less than 2^31, and a 64-bit
// division per entry took a quarter of the placing kernel.
__device__ __forceinline__ uint32_t first_entry() {
  return blockIdx.x * static_cast<uint32_t>(kRun) + (threadIdx.x >> 5) * (32 * kPerLane) + (threadIdx.x & 31);
}

// This lane's entries of its warp's segment as local experts (-1: none), 32 apart.
__device__ __forceinline__ void load_entries(const SlotParams& p, int (&e)[kPerLane]) {
  const uint32_t at = first_entry();
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    // (an id below `first` wraps around to a large number)
    const int32_t id = at + 32 * i < p.entries ? p.ids[at + 32 * i] : -1;
    const uint32_t local = static_cast<uint32_t>(id) - static_cast<uint32_t>(p.first);
    e[i] = id >= 0 && local < static_cast<uint32_t>(p.experts) ? static_cast<int>(local) : -1;
  }
}

// cnt[w][e] = entries of expert e in warp w's segment of this CTA's run
__device__ __forceinline__ void count_segments(const SlotParams& p, const int (&e)[kPerLane], int32_t* cnt) {
  for (int i = threadIdx.x; i < kSlotWarps * p.experts; i += kSlotThreads) cnt[i] = 0;
  __syncthreads();
  int32_t* const mine = cnt + (threadIdx.x >> 5) * p.experts;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i)
    if (e[i] >= 0) atomicAdd(mine + e[i], 1);   // (a sum of ones: its order does not show)
  __syncthreads();
}

__global__ void __launch_bounds__(kSlotThreads) expert_slot_count_kernel(const SlotParams p) {
  extern __shared__ int32_t cnt[];
  int entry[kPerLane];
  load_entries(p, entry);
  count_segments(p, entry, cnt);
  for (int e = threadIdx.x; e < p.experts; e += kSlotThreads) {
    int32_t s = 0;
#pragma unroll
    for (int w = 0; w < kSlotWarps; ++w) s += cnt[w * p.experts + e];
    p.counts[static_cast<int64_t>(blockIdx.x) * p.experts + e] = s;
  }
}

// One CTA per expert: its counts become sums over the earlier CTAs, `totals` their total.  Up to
// kSumInPlace CTAs the placing kernel adds the rows up itself, which grows with their square.
constexpr int64_t kSumInPlace = 256;

__global__ void __launch_bounds__(kSlotThreads) expert_slot_sum_kernel(const SlotParams p, int32_t ctas) {
  __shared__ int32_t warp_total[kSlotWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int e = blockIdx.x;
  int32_t base = 0;
  for (int32_t c0 = 0; c0 < ctas; c0 += kSlotThreads) {
    const int32_t c = c0 + threadIdx.x;
    int32_t* const at = p.counts + static_cast<int64_t>(c) * p.experts + e;
    const int32_t n = c < ctas ? *at : 0;
    int32_t scan = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t v = __shfl_up_sync(kAll, scan, o);
      if (lane >= o) scan += v;
    }
    if (lane == 31) warp_total[warp] = scan;
    __syncthreads();
    int32_t before = base, all = 0;
    for (int w = 0; w < kSlotWarps; ++w) {
      if (w < warp) before += warp_total[w];
      all += warp_total[w];
    }
    if (c < ctas) *at = before + scan - n;
    base += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) p.totals[e] = base;
}

__global__ void __launch_bounds__(kSlotThreads) expert_slot_place_kernel(const SlotParams p) {
  extern __shared__ int32_t cnt[];                 // [warps][experts], [experts], [experts]
  int32_t* const all = cnt + kSlotWarps * p.experts;      // per expert: all entries
  int32_t* const before = all + p.experts;                // and those in the runs of earlier CTAs
  __shared__ int32_t warp_total[kSlotWarps], used;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int entry[kPerLane];
  load_entries(p, entry);
  for (int e = threadIdx.x; e < p.experts; e += kSlotThreads) all[e] = before[e] = 0;
  // The counts of all CTAs, as many rows at a time as the threads cover; they come in while this
  // CTA counts its own.
  const int rows = max(kSlotThreads / p.experts, 1), row = threadIdx.x / p.experts;
  const int column = threadIdx.x - row * p.experts;
  constexpr int kPer = kMaxExperts / kSlotThreads;
  int32_t sum_all[kPer] = {}, sum_before[kPer] = {};
  if (p.totals != nullptr) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = column + i * kSlotThreads;
      if (row != 0 || e >= p.experts) continue;
      sum_all[i] = p.totals[e];
      sum_before[i] = p.counts[static_cast<int64_t>(blockIdx.x) * p.experts + e];
    }
  } else if (p.counts != nullptr && row < rows) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = column + i * kSlotThreads;
      if (e >= p.experts) continue;
#pragma unroll 16
      for (int c = row; c < static_cast<int>(gridDim.x); c += rows) {
        const int32_t v = p.counts[static_cast<int64_t>(c) * p.experts + e];
        sum_all[i] += v;
        if (c < static_cast<int>(blockIdx.x)) sum_before[i] += v;
      }
    }
  }
  count_segments(p, entry, cnt);
  if (p.counts == nullptr) {
    for (int e = threadIdx.x; e < p.experts; e += kSlotThreads) {
      int32_t c = 0;
#pragma unroll
      for (int w = 0; w < kSlotWarps; ++w) c += cnt[w * p.experts + e];
      all[e] = c;
    }
  } else if (row < rows) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = column + i * kSlotThreads;
      if (e >= p.experts) continue;
      atomicAdd(all + e, sum_all[i]);
      atomicAdd(before + e, sum_before[i]);
    }
  }
  __syncthreads();
  // exclusive scan of `all` over the experts
  int32_t sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (threadIdx.x * kPer + i < p.experts) sum += all[threadIdx.x * kPer + i];
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
  for (int i = 0; i < kPer; ++i) {
    const int e = threadIdx.x * kPer + i;
    if (e < p.experts) {
      const int32_t n = all[e];
      if (blockIdx.x == 0) p.offsets[e] = base;
      int32_t at = base + before[e];
#pragma unroll
      for (int w = 0; w < kSlotWarps; ++w) {       // counts become starting slots
        const int32_t c = cnt[w * p.experts + e];
        cnt[w * p.experts + e] = at;
        at += c;
      }
      base += n;
      if (e == p.experts - 1) {
        used = base;
        if (blockIdx.x == 0) p.offsets[p.experts] = base;
      }
    }
  }
  __syncthreads();

  int32_t* const mine = cnt + warp * p.experts;
  const uint32_t at = first_entry();
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int e = entry[i];
    const uint32_t same = __match_any_sync(kAll, e);
    const int ahead = __popc(same & ((1u << lane) - 1u));
    int32_t slot = -1;
    if (e >= 0) slot = mine[e] + ahead;
    __syncwarp();
    if (e >= 0 && ahead == 0) mine[e] += __popc(same);
    __syncwarp();
    const uint32_t j = at + 32 * i;
    if (j < p.entries) {
      p.slot_of[j] = slot;
      if (slot >= 0) p.token_of_slot[slot] = static_cast<int32_t>(j / p.top_k);
      // slots behind the last one hold -1 (slot j is written by whoever owns entry j)
      if (j >= static_cast<uint32_t>(used)) p.token_of_slot[j] = -1;
    }
  }
}

size_t slot_smem(int experts) { return sizeof(int32_t) * (kSlotWarps + 2) * experts; }

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

// Up to kRun entries the map is built by a single launch of one CTA.
int64_t slot_ctas(int64_t entries) { return entries <= kRun ? 1 : (entries + kRun - 1) / kRun; }

}  // namespace

cudaError_t preload_expert_slot_kernels() {
  cudaFuncAttributes a;
  cudaError_t e = cudaFuncGetAttributes(&a, expert_slot_count_kernel);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, expert_slot_sum_kernel);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, expert_slot_place_kernel);
  return e;
}

}  // namespace tileccl

using namespace tileccl;

extern "C" int tccl_expert_slots_workspace(int64_t entries, int32_t experts, int64_t* bytes) {
  TCCL_CHECK_ARG(bytes != nullptr, "null argument");
  const int64_t ctas = slot_ctas(entries);
  const int64_t rows = ctas <= 1 ? 0 : ctas <= kSumInPlace ? ctas : ctas + 1;
  *bytes = rows * experts * static_cast<int64_t>(sizeof(int32_t));
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
  p.entries = static_cast<uint32_t>(tokens * top_k);
  p.top_k = top_k;
  p.experts = experts;
  p.first = first;
  p.offsets = reinterpret_cast<int32_t*>(offsets);
  p.token_of_slot = reinterpret_cast<int32_t*>(token_of_slot);
  p.slot_of = reinterpret_cast<int32_t*>(slot_of);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  TCCL_CHECK_ARG(p.entries == 0 || (ids != 0 && token_of_slot != 0 && slot_of != 0), "null argument");
  const int64_t ctas = slot_ctas(p.entries);
  if (ctas > 1) {
    TCCL_CHECK_ARG(workspace != 0, "this many entries need a workspace");
    p.counts = reinterpret_cast<int32_t*>(workspace);
  }
  TCCL_CHECK_CUDA(attrs_once());
  if (ctas > 1) {
    expert_slot_count_kernel<<<static_cast<unsigned>(ctas), kSlotThreads, slot_smem(experts), s>>>(p);
    TCCL_CHECK_CUDA(cudaGetLastError());
  }
  if (ctas > kSumInPlace) {
    p.totals = p.counts + ctas * experts;
    expert_slot_sum_kernel<<<static_cast<unsigned>(experts), kSlotThreads, 0, s>>>(p, static_cast<int32_t>(ctas));
    TCCL_CHECK_CUDA(cudaGetLastError());
  }
  expert_slot_place_kernel<<<static_cast<unsigned>(ctas), kSlotThreads, slot_smem(experts), s>>>(p);
  TCCL_CHECK_CUDA(cudaGetLastError());
  return kOk;
}
