// Products of the experts over a slot map (expert_slots.cu): every slot's row times the weight
// matrix of its expert, and the gradient of those weights, on the sm_100a tensor cores.
//
//   out[s] = x[s] @ W[e(s)]
//   SiLU gate: W's columns come as 128 gate columns followed by 128 up columns;
//              out[s] = silu(gate) * up, half as wide
//   gradient of the gate: gate and up are computed again and with dh[s] = dL/dout[s]
//              dgate = dh * up * sg * (1 + gate * (1 - sg)),  dup = dh * gate * sg,
//              sg = 1 / (1 + e^-gate), packed like W's columns
//   out in fp32: for sums over a token's slots that are rounded once at their end
//   dW[e] = sum over the slots s of e of a[s]^T b[s]
//
// Both kernels are persistent: a cluster of two CTAs per tile, tcgen05.mma.cta_group::2, a TMA
// ring of operand stages, two accumulators in TMEM so that the epilogue of one tile runs under
// the next tile's products.
#include <cuda.h>
#include <cuda_runtime.h>

#include "../api.h"
#include "../device/ptx.cuh"
#include "../device/tile_compute.cuh"
#include "../runtime/errors.h"

namespace tileccl {
namespace {

enum Epilogue : int { kNone = 0, kSiluGate = 1, kSiluGateGrad = 2, kFloat = 3 };

constexpr int kMaxExperts = 1024;
constexpr int kThreads = 256;            // warp 0 TMA, 1 MMA, 2 TMEM, 3 idle, 4-7 epilogue
constexpr int kCopyThreads = 128;        // warps 8-11 of the weight gradient
constexpr int kEpiThreads = 128;         // warps 4-7
constexpr int kStages = 6;               // 32 KB each
constexpr int kFewStages = 9;            // 20 KB each: with at most kFewTokens rows per tile
constexpr int kFewTokens = 64;
constexpr int kBK = 64;                  // contraction elements per stage (one 128-byte row)
constexpr int kUmmaK = 16;
constexpr int kHalfBytes = 64 * 128;     // 64 rows of 128 bytes: one TMA box, 8 KB
constexpr int kOperandBytes = 2 * kHalfBytes;
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kRingBytes = kStages * kStageBytes;
constexpr int kFewBytes = kOperandBytes + kFewTokens / 2 * 128;
static_assert(kFewStages * kFewBytes <= kRingBytes && kFewBytes % 1024 == 0, "ring of few tokens");
constexpr int kTile = 256;               // features (M) and, at most, tokens (N) of a pair's tile
constexpr int kAccCols = 256;            // TMEM columns of one accumulator
constexpr int kBand = 16;                // token tiles that share a sweep over the features
constexpr int kMinBlocks = 4;            // K blocks a pair takes at least of a shared tile
constexpr int kChunk = 16;               // tokens per epilogue step
constexpr int kStageLd = 132;            // floats between tokens of the staging buffer
constexpr int kStagingBytes = 2 * kChunk * kStageLd * 4;
constexpr int kCtlBytes = 512;
constexpr int kListBytes = 2 * 4 * (kMaxExperts + 2);
constexpr int kGemmSmem = kStages * kStageBytes + kStagingBytes + kCtlBytes + kListBytes + 1024;
constexpr int kGradStages = kStages - 1; // the sixth stage takes the copied blocks
constexpr int kGradStagingBytes = 4 * 2 * 4096;   // per epilogue warp two buffers of 32 x 64
constexpr int kGradSmem = kStages * kStageBytes + kGradStagingBytes + kCtlBytes + 1024;
static_assert(kGemmSmem <= 232448 && kGradSmem <= 232448, "shared memory of one SM");

// Status words and arrival counters of a device's products.  They are part of the module, zero when
// it is loaded: a first call needs no allocation and may be captured.
constexpr int kStatusWords = 8;
constexpr int64_t kCounterBytes = 1 << 20;
__device__ uint32_t g_status[kStatusWords];
__device__ __align__(128) uint32_t g_counters[kCounterBytes / 4];

struct GemmParams {
  CUtensorMap tma_w;          // five dimensions, see weight_map
  CUtensorMap tma_x[4];       // {K, rows}, boxes {64, 128}, {64, 64}, {64, 32}, {64, 16}
  const int32_t* offsets;
  void* out;
  const void* dh;
  float* partial;             // [pairs][2][2 CTAs][128 * partial_tokens], null = tiles stay whole
  uint32_t* counters;         // [2 * pairs][2], zero between calls
  int64_t ldo, ld_dh;
  int32_t partial_tokens;
  int32_t slots, experts, k_blocks, n, f_tiles, bf16, w_nk;
  int32_t w_halves;           // a CTA's 128 features come as two boxes
  uint32_t* status;
  uint64_t budget_ns;
};

struct GradParams {
  CUtensorMap tma_a, tma_b;   // {64, rows, columns / 64}, box {64, 64, 2}; 64 does not divide the
                              // columns: {columns, rows, 1}, box {64, 64, 1} twice
  CUtensorMap tma_out;        // {n, m, experts}, box {64, 32, 1}
  const int32_t* offsets;
  const void* a;
  const void* b;
  int64_t lda, ldb;
  int32_t slots, experts, m, n, m_tiles, n_tiles, bf16;
  int32_t a_halves, b_halves;
  uint32_t* status;
  uint64_t budget_ns;
};

__device__ __forceinline__ void tma_load_5d_pair(uint32_t dst, const CUtensorMap* m, int x, int y,
                                                 int z, int u, int v, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.tile"
      ".mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(z), "r"(u), "r"(v), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* m, int x, int y,
                                                 int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile"
      ".mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
// 16 bytes of a row, zeros instead when `take` is false (the source must be a valid address).
__device__ __forceinline__ void copy_16(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(take ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* m, int x, int y, int z,
                                             uint32_t src) {
  asm volatile(
      "cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(
          reinterpret_cast<uint64_t>(m)),
      "r"(x), "r"(y), "r"(z), "r"(src)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
// Barrier `id` of 128 threads that also agrees on a condition.
__device__ __forceinline__ bool barrier_all(int id, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %2, 0;\n\t"
      "barrier.cta.red.and.pred q, %1, 128, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(ok ? 1u : 0u)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ bool epilogue_all(bool ok) { return barrier_all(1, ok); }
__device__ __forceinline__ bool copiers_all(bool ok) { return barrier_all(2, ok); }
__device__ __forceinline__ void epilogue_sync() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }

// Shared memory of a CTA pair.  Every CTA has all barriers; in use are the leader's "full" and
// "accumulator empty" (both CTAs report to them) and both CTAs' "empty" and "accumulator full"
// (signalled by multicast commits).
struct Pipe {
  uint32_t base, staging, ctl;
  uint32_t full, empty, tail, tail_empty, acc_full, acc_empty, drain, tmem_slot;
  volatile uint32_t* words;        // generic view of tmem_slot: [0] TMEM base, [1] abort flag
  int32_t* start;                  // [experts + 1] first slot of every expert
  int32_t* tiles;                  // [experts + 1] tiles of all lower experts
};

__device__ __forceinline__ Pipe make_pipe(uint8_t* raw, int staging_bytes) {
  Pipe s;
  s.base = (smem_u32(raw) + 1023u) & ~1023u;
  s.staging = s.base + kRingBytes;
  s.ctl = s.staging + staging_bytes;
  s.full = s.ctl;
  s.empty = s.full + 8 * kFewStages;
  s.tail = s.empty + 8 * kFewStages;
  s.tail_empty = s.tail + 8;
  s.acc_full = s.tail_empty + 8;
  s.acc_empty = s.acc_full + 16;
  s.drain = s.acc_empty + 16;
  s.tmem_slot = s.drain + 8;
  uint8_t* const g = raw + (s.ctl - smem_u32(raw));
  s.words = reinterpret_cast<volatile uint32_t*>(g + (s.tmem_slot - s.ctl));
  s.start = reinterpret_cast<int32_t*>(g + kCtlBytes);
  s.tiles = s.start + kMaxExperts + 2;
  return s;
}

// Barriers and TMEM of a CTA pair: `pipe_start` sets them up, `pipe_meet` returns the TMEM base
// once both CTAs have; what a thread wrote to shared memory in between is visible to its CTA
// afterwards.
__device__ __forceinline__ void pipe_start(const Pipe& s) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < kFewStages; ++i) {
      mbar_init(s.full + 8 * i, 1);
      mbar_init(s.empty + 8 * i, 1);
    }
    mbar_init(s.tail, 2);                    // the copying warps of both CTAs
    mbar_init(s.tail_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(s.acc_full + 8 * i, 1);
      mbar_init(s.acc_empty + 8 * i, 8);     // four epilogue warps of both CTAs
    }
    mbar_init(s.drain, 1);
    s.words[1] = 0;
    mbar_fence_init();
  }
  if ((threadIdx.x >> 5) == 2) {
    tmem_alloc_pair(s.tmem_slot, 2 * kAccCols);
    tmem_relinquish_pair();
  }
}
__device__ __forceinline__ uint32_t pipe_meet(const Pipe& s) {
  tcgen05_fence_before();
  __syncthreads();
  cluster_sync_all();
  tcgen05_fence_after();
  return s.words[0];
}

__device__ __forceinline__ int slot_bound(const int32_t* offsets, int e, int slots) {
  return min(max(offsets[e], 0), slots);
}

// `pipe_start` and the list of tiles: expert e has tiles_of(rows of e) of them.  The counts per
// expert live on the GPU only, so every CTA derives the whole schedule from the offsets.
template <typename F>
__device__ __forceinline__ void list_tiles(const Pipe& s, const int32_t* offsets, int slots,
                                           int experts, F tiles_of) {
  __shared__ int32_t warp_sum[kThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kPer = kMaxExperts / kThreads;
  int32_t bound[kPer + 1], count[kPer];
  int32_t sum = 0;
#pragma unroll
  for (int i = 0; i <= kPer; ++i) {
    const int e = threadIdx.x * kPer + i;
    bound[i] = e <= experts ? offsets[e] : 0;
  }
  pipe_start(s);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = threadIdx.x * kPer + i;
    count[i] = 0;
    if (e < experts) {
      const int a = min(max(bound[i], 0), slots), b = min(max(bound[i + 1], 0), slots);
      s.start[e] = a;
      if (e == experts - 1) s.start[experts] = b;
      count[i] = tiles_of(max(b - a, 0));
    }
    sum += count[i];
  }
  int32_t scan = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int32_t v = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += v;
  }
  if (lane == 31) warp_sum[warp] = scan;
  __syncthreads();
  int32_t at = scan - sum;
  for (int w = 0; w < warp; ++w) at += warp_sum[w];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = threadIdx.x * kPer + i;
    if (e < experts) {
      s.tiles[e] = at;
      at += count[i];
      if (e == experts - 1) s.tiles[experts] = at;
    }
  }
}

// Neither CTA of a pair may retire while its partner can still read its operands or touch its
// barriers; TMEM goes back after every MMA and TMEM read is done.  After a wait that gave up,
// copies that are still on their way to either CTA get two milliseconds to land.
__device__ __forceinline__ void pipe_end(const Pipe& s, uint32_t tmem_base) {
  tcgen05_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && s.words[1] != 0) {
    const uint64_t until = globaltimer_ns() + 2000000ull;
    for (int i = 0; i < 1000000 && globaltimer_ns() < until; ++i) __nanosleep(1000);
  }
  __syncwarp();
  cluster_sync_all();
  if ((threadIdx.x >> 5) == 2) {
    tcgen05_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * kAccCols);
  }
}

// Bounded wait for arrivals of the other CTA of the pair.
__device__ __forceinline__ bool wait_cluster(uint32_t bar, uint32_t parity, const WaitBudget& wb) {
  for (uint32_t it = 0;; ++it) {
    if (mbar_try_wait_cluster(bar, parity)) return true;
    if (wb.expired(it)) {
      *wb.abort_flag = 1;
      return false;
    }
  }
}

__device__ __forceinline__ int expert_of(const Pipe& s, int experts, int t) {
  int lo = 0, hi = experts;                    // tiles[lo] <= t < tiles[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s.tiles[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ void store_row8(void* base, int64_t i, bool bf16, const float* v) {
  *reinterpret_cast<uint4*>(static_cast<char*>(base) + 2 * i) = tile_cast_f32x8(bf16, v);
}

// ---------------------------------------------------------------------------------------
// out[s] = epilogue(x[s] @ W[e(s)])
//
// The weights are the M operand (256 features per pair, 128 per CTA) and the tokens the N
// operand: M is fixed to 256 by the pair form of the instruction while N may be any multiple
// of 32, so an expert's tile is as wide as its rows need.  With the gate a CTA's 128 features
// are 64 gate columns and the 64 up columns that belong to them.  Bound by the tensor cores with
// many rows per expert (16384 rows of 8 experts, 4096 x 28672: 2.52 ms, 1530 TFLOP/s; 1270 in a
// long run, at the power limit) and by the weights' way from DRAM with few (64 rows of 64 experts,
// 4096 x 3584: 154 us; 6018 rows of 61, 1792 x 4096: 162 us, 5.9 TB/s).
//
// Schedule: tile t goes to pair t mod P.  With few tokens the time is that of streaming the
// weights, and a third of the SMs nearly draws the full memory bandwidth: only a last round with
// fewer tiles than that is worth spreading.  The first R = P + T mod P tiles (all of them when
// T < P) are then cut into P equal runs of K blocks: a pair's run covers the end of one tile,
// whole tiles, the start of another.  Parts of a tile are left in `partial` as fp32 sums;
// whichever pair comes last (a counter per tile and CTA) adds them up in the order of K, so the
// result does not depend on who that was.  Measured (us, shared / whole): one token of 1 expert of
// 14336 x 4096 27 / 46 (T = 0.2 P), 4 tokens of 2 experts 101 / 118 (T = 1.1 P); one token of 2
// experts 47 / 47 (T = 0.4 P), of 8 of 4096 x 3584 48 / 45 (T = 1.5 P) and 512 tokens of 2 experts
// 204 / 158 (wide partial tiles) stay whole.
//
// kFew: no tile is wider than kFewTokens, so the ring holds nine stages instead of six: what an SM
// draws is what it has in flight (one token of 2 experts of 14336 x 4096: 53 -> 47 us).
// ---------------------------------------------------------------------------------------
struct Item {
  int e, row0, rows, n, f0;
  int kb0, kb1;              // K blocks of this item
  int part, parts, slot;     // parts > 1: the tile is shared; slot = the tile's counter
  int first_pair;            // pair that computes part 0
};

// The items of one pair, in order; every role walks the same list.
struct Walker {
  int pos, end;              // K blocks of the shared tiles (tile * k_blocks + block)
  int unit;                  // K blocks per pair there
  int shared;                // tiles that are cut up
  int next;                  // next whole tile
};

template <int kEpi, bool kFew>
__global__ void __launch_bounds__(kThreads, 1)
expert_gemm_kernel(const __grid_constant__ GemmParams p) {
  constexpr bool kPlain = kEpi == kNone || kEpi == kFloat;
  constexpr int kRing = kFew ? kFewStages : kStages, kBytes = kFew ? kFewBytes : kStageBytes;
  extern __shared__ uint8_t smem_raw[];
  const Pipe s = make_pipe(smem_raw, kStagingBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = static_cast<int>(cluster_ctarank());
  const bool leader = cta == 0;
  if (threadIdx.x == 96) {
    tma_prefetch_desc(&p.tma_w);
    for (int i = 0; i < 4; ++i) tma_prefetch_desc(&p.tma_x[i]);
  }
  // (the offsets come in while the barriers and TMEM are set up)
  list_tiles(s, p.offsets, p.slots, p.experts,
             [&](int rows) { return (rows + kTile - 1) / kTile * p.f_tiles; });
  const uint32_t tmem_base = pipe_meet(s);
  // Behind the row copy this kernel may have been scheduled while that still runs (it touches
  // nothing but x; what came before it, the offsets among it, was complete when it began).  One
  // token of 2 experts of 4096 x 28672: 80 -> 78 us, of 8 of 4096 x 3584: 44.2 -> 43.7.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  WaitBudget wb;
  wb.start(p.budget_ns, s.words + 1);

  const int total = s.tiles[p.experts];
  const int pairs = static_cast<int>(gridDim.x >> 1), pair = static_cast<int>(blockIdx.x >> 1);
  auto walk = [&]() {
    Walker w;
    const int over = total % pairs;
    w.shared = p.partial == nullptr || over == 0 || 3 * over >= pairs ? 0 : total < pairs ? total : pairs + over;
    const int blocks = w.shared * p.k_blocks;      // (at most 2 * pairs tiles)
    w.unit = max((blocks + pairs - 1) / pairs, min(kMinBlocks, p.k_blocks));
    w.pos = min(pair * w.unit, blocks);
    w.end = min(w.pos + w.unit, blocks);
    w.next = w.shared + pair;
    return w;
  };
  // Tile t: token tiles run fastest, in bands of kBand, so that the tiles in flight share both
  // their weights and a band of tokens in L2.
  auto advance = [&](Walker& w, Item& it) {
    int t;
    if (w.pos < w.end) {
      t = w.pos / p.k_blocks;
      it.kb0 = w.pos - t * p.k_blocks;
      it.kb1 = min(p.k_blocks, it.kb0 + w.end - w.pos);
      w.pos += it.kb1 - it.kb0;
      it.first_pair = t * p.k_blocks / w.unit;
      it.part = pair - it.first_pair;
      it.parts = ((t + 1) * p.k_blocks - 1) / w.unit - it.first_pair + 1;
      it.slot = t;
    } else {
      t = w.next;
      if (t >= total) return false;
      w.next += pairs;
      it.kb0 = 0;
      it.kb1 = p.k_blocks;
      it.part = it.slot = it.first_pair = 0;
      it.parts = 1;
    }
    it.e = expert_of(s, p.experts, t);
    const int rows = s.start[it.e + 1] - s.start[it.e];
    const int tiles = (rows + kTile - 1) / kTile;
    int local = t - s.tiles[it.e];
    const int band = local / (kBand * p.f_tiles);
    local -= band * kBand * p.f_tiles;
    const int wide = min(kBand, tiles - band * kBand);
    const int ti = band * kBand + local % wide;
    it.f0 = local / wide * kTile;
    // The expert's rows in blocks of 32, shared out evenly: no tile is padded but the last.  (With
    // every tile rounded up from an equal share 8192 tokens x top 2 of 8 experts, 4096 x 28672,
    // took 2.75 ms instead of 2.52.)
    const int blocks = (rows + 31) / 32, share = blocks / tiles, more = blocks - share * tiles;
    const int first = (ti * share + min(ti, more)) * 32;
    it.row0 = s.start[it.e] + first;
    it.n = (share + (ti < more ? 1 : 0)) * 32;
    it.rows = min(it.n, rows - first);
    return true;
  };
  Walker w = walk();
  Item it;

  if (warp == 0) {
    // ------------------------------- TMA producer -------------------------------
    if (elect_one_sync()) {
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      while (ok && advance(w, it)) {
        const int mine = it.n >> 1;                          // token rows this CTA stages
        const int first = it.row0 + cta * mine;
        // this CTA's 128 features in the coordinates of weight_map
        const int f = it.f0 + cta * 128;
        const int w_inner = !kPlain ? cta * 64 : p.w_nk || p.w_halves ? f : 0;
        const int w_z = kPlain && !p.w_nk && !p.w_halves ? f / 64 : 0;
        const int w_u = kPlain ? 0 : it.f0 / kTile;
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          if (!mbar_wait(s.empty + 8 * stage, phase ^ 1u, wb)) {
            report_status(p.status, kStatusTimeoutMbarrier, 101, 0, kb, 0, it.row0);
            ok = false;
            break;
          }
          const uint32_t sa = s.base + stage * kBytes, sb = sa + kOperandBytes;
          const uint32_t bar = mapa_shared(s.full + 8 * stage, 0);
          // the bytes of both CTAs are counted on the leader's barrier
          if (leader) mbar_expect_tx(s.full + 8 * stage, 2 * (kOperandBytes + mine * 128));
          const int wx = p.w_nk ? kb * kBK : w_inner, wy = p.w_nk ? w_inner : kb * kBK;
          tma_load_5d_pair(sa, &p.tma_w, wx, wy, w_z, w_u, it.e, bar);
          if (p.w_halves) tma_load_5d_pair(sa + kHalfBytes, &p.tma_w, wx + 64, wy, w_z, w_u, it.e, bar);
          // as few boxes as the row count has binary digits: a copy keeps the TMA unit busy for
          // some 70 cycles however small it is (boxes of 16 rows throughout: 999 instead of 1549
          // TFLOP/s; the unit's own gather, four rows per copy: 460)
          int at = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (mine & (128 >> i)) {
              tma_load_2d_pair(sb + at * 128, &p.tma_x[i], kb * kBK, first + at, bar);
              at += 128 >> i;
            }
          }
          if (++stage == kRing) { stage = 0; phase ^= 1u; }
        }
      }
    }
  } else if (warp == 1 && leader) {
    // ----------------------- MMA issuer (leader CTA only) -----------------------
    if (elect_one_sync()) {
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
      bool ok = true;
      while (ok && advance(w, it)) {
        const uint32_t idesc = umma_idesc_f16(p.bf16, p.w_nk ? 0 : 1, 0, kTile, it.n);
        if (!mbar_wait(s.acc_empty + 8 * acc, acc_phase ^ 1u, wb)) {
          report_status(p.status, kStatusTimeoutMbarrier, 102, 0, 0, 0, it.row0);
          ok = false;
          break;
        }
        tcgen05_fence_after();
        const uint32_t d = tmem_base + acc * kAccCols;
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          if (!mbar_wait(s.full + 8 * stage, phase, wb)) {
            report_status(p.status, kStatusTimeoutMbarrier, 103, it.kb1, kb, 0, it.row0);
            ok = false;
            break;
          }
          tcgen05_fence_after();
          const uint32_t sa = s.base + stage * kBytes, sb = sa + kOperandBytes;
#pragma unroll
          for (int k = 0; k < kBK / kUmmaK; ++k) {
            const uint64_t da = p.w_nk ? umma_smem_desc_sw128(sa + k * kUmmaK * 2, 16, 1024)
                                       : umma_smem_desc_sw128(sa + k * kUmmaK * 128, kHalfBytes, 1024);
            const uint64_t db = umma_smem_desc_sw128(sb + k * kUmmaK * 2, 16, 1024);
            umma_f16_pair(d, da, db, idesc, kb > it.kb0 || k > 0 ? 1u : 0u);
          }
          umma_commit_pair(s.empty + 8 * stage, 3);
          if (++stage == kRing) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        umma_commit_pair(s.acc_full + 8 * acc, 3);
        acc ^= 1u;
        if (acc == 0) acc_phase ^= 1u;
      }
      if (!ok) {
        umma_commit_pair(s.drain, 1);       // outstanding MMAs end before TMEM is released
        for (int i = 0; i < 1000000 && !mbar_try_wait(s.drain, 0); ++i) {}
      }
    }
  } else if (warp >= 4) {
    // --------------------------------- epilogue ---------------------------------
    // A TMEM lane is a feature and a column a token; results are rows of features.  Sixteen
    // tokens at a time cross over through shared memory in fp32: written by feature, read back
    // by token, eight features per thread.
    const int q = warp - 4, me = threadIdx.x - 128;
    float* const staging = reinterpret_cast<float*>(smem_raw + (s.staging - smem_u32(smem_raw)));
    const bool bf16 = p.bf16 != 0;
    constexpr int kVecs = kPlain ? 16 : 8;                 // 8-feature vectors per token
    uint32_t acc = 0, acc_phase = 0, buf = 0;
    while (advance(w, it)) {
      if (!epilogue_all(mbar_wait(s.acc_full + 8 * acc, acc_phase, wb))) {
        if (me == 0) report_status(p.status, kStatusTimeoutMbarrier, 104, 0, 0, 0, it.row0);
        break;
      }
      tcgen05_fence_after();
      const uint32_t t_acc = tmem_base + acc * kAccCols + (static_cast<uint32_t>(q * 32) << 16);
      const int last_c0 = (max(it.rows, 1) - 1) / kChunk * kChunk;
      auto read_acc = [&](int c0, float (&v)[kChunk]) {
        tmem_ld_x16(t_acc + c0, v);
        if (c0 != last_c0) return;
        // every TMEM read of this accumulator is done: hand it back to the MMA warp
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(s.acc_empty + 8 * acc, 0));
      };
      // Parts of a shared tile: part q lies at pair first_pair + q, in its second place if the
      // tile starts there.  Layout: [step of 16 tokens][4][feature][4 tokens].
      auto partial_of = [&](int part) {
        const int64_t at = ((it.first_pair + part) * 2 + (part == 0 ? 1 : 0)) * 2 + cta;
        return p.partial + at * p.partial_tokens * 128 + me * 4;
      };
      if (it.parts > 1) {
        float* const mine = partial_of(it.part);
        for (int c0 = 0; c0 <= last_c0; c0 += kChunk) {
          float v[kChunk];
          read_acc(c0, v);
#pragma unroll
          for (int j = 0; j < kChunk / 4; ++j)
            __stcg(reinterpret_cast<float4*>(mine + (c0 / 4 + j) * 512),
                   make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
        }
        __threadfence();
        epilogue_sync();
        if (me == 0) {
          uint32_t* const ctr = p.counters + it.slot * 2 + cta;
          const bool last = atomicAdd(ctr, 1u) == static_cast<uint32_t>(it.parts - 1);
          if (last) *ctr = 0;                      // as the next call finds it
          s.words[2] = last ? 1u : 0u;
        }
        epilogue_sync();
        acc ^= 1u;
        if (acc == 0) acc_phase ^= 1u;
        if (s.words[2] == 0) continue;
        __threadfence();
      }
      // The gate's gradient reads dL/dout one step ahead (one vector per thread and step).
      auto load_dh = [&](int c0) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (kEpi == kSiluGateGrad && c0 + me / kVecs < it.rows)
          x = __ldg(reinterpret_cast<const uint4*>(
              static_cast<const char*>(p.dh) +
              2 * (static_cast<int64_t>(it.row0 + c0 + me / kVecs) * p.ld_dh + it.f0 / 2 + cta * 64 +
                   me % kVecs * 8)));
        return x;
      };
      uint4 dh_next = load_dh(0);
      for (int c0 = 0; c0 <= last_c0; c0 += kChunk) {
        const uint4 dh = dh_next;
        dh_next = load_dh(c0 + kChunk);
        float v[kChunk];
        if (it.parts > 1) {
          for (int i = 0; i < it.parts; ++i) {
            const float* const src = partial_of(i);
#pragma unroll
            for (int j = 0; j < kChunk / 4; ++j) {
              const float4 x = __ldcg(reinterpret_cast<const float4*>(src + (c0 / 4 + j) * 512));
              v[4 * j] = i == 0 ? x.x : v[4 * j] + x.x;
              v[4 * j + 1] = i == 0 ? x.y : v[4 * j + 1] + x.y;
              v[4 * j + 2] = i == 0 ? x.z : v[4 * j + 2] + x.z;
              v[4 * j + 3] = i == 0 ? x.w : v[4 * j + 3] + x.w;
            }
          }
        } else {
          read_acc(c0, v);
        }
        float* const sbuf = staging + buf * (kChunk * kStageLd);
        buf ^= 1u;
#pragma unroll
        for (int i = 0; i < kChunk; ++i) sbuf[i * kStageLd + q * 32 + lane] = v[i];
        epilogue_sync();       // (two buffers: one barrier per step suffices)
#pragma unroll
        for (int i = me; i < kChunk * kVecs; i += kEpiThreads) {
          const int tok = i / kVecs, vec = i % kVecs;
          if (c0 + tok >= it.rows) continue;
          const int64_t slot = it.row0 + c0 + tok;
          float a[8];
          const float4* src = reinterpret_cast<const float4*>(sbuf + tok * kStageLd + vec * 8);
          *reinterpret_cast<float4*>(a) = src[0];
          *reinterpret_cast<float4*>(a + 4) = src[1];
          if (kPlain) {
            const int f = it.f0 + cta * 128 + vec * 8;
            if (f >= p.n) continue;
            if (kEpi == kNone) {
              store_row8(p.out, slot * p.ldo + f, bf16, a);
            } else {
              float4* const dst = reinterpret_cast<float4*>(static_cast<float*>(p.out) + slot * p.ldo + f);
              dst[0] = *reinterpret_cast<const float4*>(a);
              dst[1] = *reinterpret_cast<const float4*>(a + 4);
            }
            continue;
          }
          float u[8];
          *reinterpret_cast<float4*>(u) = src[16];
          *reinterpret_cast<float4*>(u + 4) = src[17];
          const int f = it.f0 / 2 + cta * 64 + vec * 8;
          if (kEpi == kSiluGate) {
#pragma unroll
            for (int j = 0; j < 8; ++j) a[j] = apply_elementwise(kOpSilu, a[j]) * u[j];
            store_row8(p.out, slot * p.ldo + f, bf16, a);
          } else {
            float g[8] = {};
            tile_accumulate_16x8(bf16, g, dh);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float sg = apply_elementwise(kOpSigmoid, a[j]);
              const float da = g[j] * u[j] * sg * (1.f + a[j] * (1.f - sg));
              u[j] = g[j] * a[j] * sg;
              a[j] = da;
            }
            const int64_t at = slot * p.ldo + it.f0 + cta * 64 + vec * 8;
            store_row8(p.out, at, bf16, a);
            store_row8(p.out, at + 128, bf16, u);
          }
        }
      }
      if (it.parts == 1) {
        acc ^= 1u;
        if (acc == 0) acc_phase ^= 1u;
      }
    }
  }
  pipe_end(s, tmem_base);
}

// ---------------------------------------------------------------------------------------
// out[e] = sum over the slots s of e of a[s]^T b[s]
//
// 256 x 256 tiles of out[e]; the contraction runs over the expert's rows, 64 per stage, so both
// operands are MN-major (a row of 64 columns is 128 bytes of a stage).  The last, partial block of
// an expert is copied row by row, with zeros in place of the next expert's rows, into a stage of
// its own: the copies and their report to the other CTA (a release at cluster scope) take two
// microseconds, which that stage has a whole tile's time for and one of the ring's has not (8
// experts of 1024 rows, 4096 x 3584: 179 us with the copies in the ring, 168 with a stage of their
// own, 1436 TFLOP/s).  With few rows the result bounds it, which the card writes at 3.9 TB/s at
// most: 82 us for 16 to 64 rows per expert, 60 for the writes alone.
// ---------------------------------------------------------------------------------------
__global__ void __launch_bounds__(kThreads + kCopyThreads, 1)
expert_weight_grad_kernel(const __grid_constant__ GradParams p) {
  extern __shared__ uint8_t smem_raw[];
  const Pipe s = make_pipe(smem_raw, kGradStagingBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = static_cast<int>(cluster_ctarank());
  const bool leader = cta == 0;
  const int per_expert = p.m_tiles * p.n_tiles;
  if (threadIdx.x == 96) {
    tma_prefetch_desc(&p.tma_a);
    tma_prefetch_desc(&p.tma_b);
    tma_prefetch_desc(&p.tma_out);
  }
  pipe_start(s);
  const uint32_t tmem_base = pipe_meet(s);
  WaitBudget wb;
  wb.start(p.budget_ns, s.words + 1);
  const int total = p.experts * per_expert;
  const int step = static_cast<int>(gridDim.x >> 1);

  if (warp == 0) {
    // ------------------------------- TMA producer -------------------------------
    if (elect_one_sync()) {
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      for (int t = blockIdx.x >> 1; ok && t < total; t += step) {
        const int e = t / per_expert, local = t % per_expert;
        const int x_a = local / p.n_tiles * kTile + cta * 128;
        const int x_b = local % p.n_tiles * kTile + cta * 128;
        const int row0 = slot_bound(p.offsets, e, p.slots), row1 = slot_bound(p.offsets, e + 1, p.slots);
        for (int r0 = row0; r0 + kBK <= row1; r0 += kBK) {
          if (!mbar_wait(s.empty + 8 * stage, phase ^ 1u, wb)) {
            report_status(p.status, kStatusTimeoutMbarrier, 111, 0, r0, 0, t);
            ok = false;
            break;
          }
          const uint32_t sa = s.base + stage * kStageBytes, sb = sa + kOperandBytes;
          const uint32_t bar = mapa_shared(s.full + 8 * stage, 0);
          if (leader) mbar_expect_tx(s.full + 8 * stage, 2 * kStageBytes);
          auto load = [&](uint32_t dst, const CUtensorMap* map, int x, bool halves) {
            tma_load_3d_pair(dst, map, halves ? x : 0, r0, halves ? 0 : x / 64, bar);
            if (halves) tma_load_3d_pair(dst + kHalfBytes, map, x + 64, r0, 0, bar);
          };
          load(sa, &p.tma_a, x_a, p.a_halves != 0);
          load(sb, &p.tma_b, x_b, p.b_halves != 0);
          if (++stage == kGradStages) { stage = 0; phase ^= 1u; }
        }
      }
    }
  } else if (warp == 1 && leader) {
    // ----------------------- MMA issuer (leader CTA only) -----------------------
    if (elect_one_sync()) {
      const uint32_t idesc = umma_idesc_f16(p.bf16, 1, 1, kTile, kTile);
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0, tail_phase = 0;
      bool ok = true;
      for (int t = blockIdx.x >> 1; ok && t < total; t += step) {
        const int e = t / per_expert;
        const int rows = slot_bound(p.offsets, e + 1, p.slots) - slot_bound(p.offsets, e, p.slots);
        const int blocks = (max(rows, 0) + kBK - 1) / kBK;
        if (blocks == 0) continue;                       // the epilogue writes zeros
        if (!mbar_wait(s.acc_empty + 8 * acc, acc_phase ^ 1u, wb)) {
          report_status(p.status, kStatusTimeoutMbarrier, 112, 0, 0, 0, t);
          ok = false;
          break;
        }
        tcgen05_fence_after();
        const uint32_t d = tmem_base + acc * kAccCols;
        for (int kb = 0; kb < blocks; ++kb) {
          const bool copied = kb * kBK + kBK > rows;
          if (copied ? !wait_cluster(s.tail, tail_phase, wb) : !mbar_wait(s.full + 8 * stage, phase, wb)) {
            report_status(p.status, kStatusTimeoutMbarrier, copied ? 117 : 113, blocks, kb, 0, t);
            ok = false;
            break;
          }
          tcgen05_fence_after();
          const uint32_t sa = s.base + (copied ? kGradStages : stage) * kStageBytes, sb = sa + kOperandBytes;
#pragma unroll
          for (int k = 0; k < kBK / kUmmaK; ++k)
            umma_f16_pair(d, umma_smem_desc_sw128(sa + k * kUmmaK * 128, kHalfBytes, 1024),
                          umma_smem_desc_sw128(sb + k * kUmmaK * 128, kHalfBytes, 1024), idesc,
                          (kb | k) != 0 ? 1u : 0u);
          umma_commit_pair(copied ? s.tail_empty : s.empty + 8 * stage, 3);
          if (copied) tail_phase ^= 1u;
          else if (++stage == kGradStages) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        umma_commit_pair(s.acc_full + 8 * acc, 3);
        acc ^= 1u;
        if (acc == 0) acc_phase ^= 1u;
      }
      if (!ok) {
        umma_commit_pair(s.drain, 1);
        for (int i = 0; i < 1000000 && !mbar_try_wait(s.drain, 0); ++i) {}
      }
    }
  } else if (warp >= kThreads / 32) {
    // ------------- copying warps: the partial block at the end of an expert -------------
    // Thread c copies 16-byte chunk c % 8 of one half of the columns (c / 8 % 2) of the rows
    // c / 16, c / 16 + 8, ... of both operands.
    const int c = threadIdx.x - kThreads, chunk = c & 7, h = (c >> 3) & 1, row = c >> 4;
    const uint32_t dst = s.base + kGradStages * kStageBytes + h * kHalfBytes + row * 128 + ((chunk ^ row) << 4);
    uint32_t phase = 0;
    for (int t = blockIdx.x >> 1; t < total; t += step) {
      const int e = t / per_expert, local = t % per_expert;
      const int x_a = local / p.n_tiles * kTile + cta * 128 + h * 64 + chunk * 8;
      const int x_b = local % p.n_tiles * kTile + cta * 128 + h * 64 + chunk * 8;
      const int row0 = slot_bound(p.offsets, e, p.slots), row1 = slot_bound(p.offsets, e + 1, p.slots);
      const int rows = max(row1 - row0, 0);
      if (rows % kBK == 0) continue;
      if (!copiers_all(mbar_wait(s.tail_empty, phase ^ 1u, wb))) {
        if (c == 0) report_status(p.status, kStatusTimeoutMbarrier, 115, 0, 0, 0, t);
        break;
      }
      const int r0 = row0 + rows / kBK * kBK;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t r = r0 + row + 8 * i;
        const bool in_a = r < row1 && x_a < p.m, in_b = r < row1 && x_b < p.n;
        copy_16(dst + i * 1024, static_cast<const char*>(p.a) + (in_a ? 2 * (r * p.lda + x_a) : 0), in_a);
        copy_16(dst + kOperandBytes + i * 1024,
                static_cast<const char*>(p.b) + (in_b ? 2 * (r * p.ldb + x_b) : 0), in_b);
      }
      copy_wait_all();
      fence_proxy_async_smem();
      copiers_all(true);
      if (c == 0) mbar_arrive_cluster(mapa_shared(s.tail, 0));
      phase ^= 1u;
    }
  } else if (warp >= 4) {
    // --------------------------------- epilogue ---------------------------------
    // A lane is a row of out[e]: 32 rows x 64 columns at a time go through a swizzled buffer
    // into a TMA store, which clips them to the matrix.
    const int q = warp - 4;
    const uint32_t mine = s.staging + q * 2 * 4096;
    const bool bf16 = p.bf16 != 0;
    uint32_t acc = 0, acc_phase = 0, buf = 0;
    bool ok = true;
    for (int t = blockIdx.x >> 1; ok && t < total; t += step) {
      const int e = t / per_expert, local = t % per_expert;
      const int y = local / p.n_tiles * kTile + cta * 128 + q * 32, x = local % p.n_tiles * kTile;
      const bool empty = slot_bound(p.offsets, e + 1, p.slots) <= slot_bound(p.offsets, e, p.slots);
      if (!empty) {
        if (!mbar_wait(s.acc_full + 8 * acc, acc_phase, wb)) {
          if (lane == 0) report_status(p.status, kStatusTimeoutMbarrier, 114, 0, 0, 0, t);
          ok = false;
          break;
        }
        tcgen05_fence_after();
      }
      const uint32_t t_acc = tmem_base + acc * kAccCols + (static_cast<uint32_t>(q * 32) << 16);
      for (int ch = 0; ch < kTile / 64; ++ch) {
        float v[64];
        if (!empty) {
          uint32_t r0[32], r1[32];
          tmem_ld_32x32b_x32(t_acc + ch * 64, r0);
          tmem_ld_32x32b_x32(t_acc + ch * 64 + 32, r1);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            v[i] = __uint_as_float(r0[i]);
            v[32 + i] = __uint_as_float(r1[i]);
          }
          if (ch == kTile / 64 - 1) {
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(mapa_shared(s.acc_empty + 8 * acc, 0));
          }
        } else {
          tile_zeros(v);
        }
        if (lane == 0) tma_store_wait_read<1>();    // the store that last read this buffer
        __syncwarp();
        const uint32_t sbuf = mine + buf * 4096;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint4 w = tile_cast_f32x8(bf16, &v[j * 8]);
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(
                           sbuf + lane * 128 + ((j ^ (lane & 7)) << 4)),
                       "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w)
                       : "memory");
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (x + ch * 64 < p.n && y < p.m) tma_store_3d(&p.tma_out, x + ch * 64, y, e, sbuf);
          tma_store_commit();
        }
        buf ^= 1u;
      }
      if (!empty) {
        acc ^= 1u;
        if (acc == 0) acc_phase ^= 1u;
      }
    }
    if (lane == 0) tma_store_wait_all<0>();
  }
  pipe_end(s, tmem_base);
}

// ------------------------------------------------------------------------------- host side
// 16-bit tensor of `rank` dimensions (unit stride innermost) with a box of 128-byte rows.
int encode(CUtensorMap* map, bool bf16, uint64_t base, int rank, const cuuint64_t* dims,
           const cuuint64_t* strides, const cuuint32_t* box, const char* what) {
  const DriverApi& d = driver();
  cuuint32_t es[5] = {1, 1, 1, 1, 1};
  const CUresult r = d.cuTensorMapEncodeTiled(
      map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
      static_cast<cuuint32_t>(rank), reinterpret_cast<void*>(base), dims, strides, box, es,
      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(kErrCuda, std::string("cuTensorMapEncodeTiled(") + what + "): " + driver_error_string(r));
  return kOk;
}
int encode_rows(CUtensorMap* map, bool bf16, uint64_t base, uint64_t cols, uint64_t rows,
                uint64_t ld_bytes, uint32_t box_rows, const char* what) {
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {ld_bytes};
  const cuuint32_t box[2] = {64, box_rows};
  return encode(map, bf16, base, 2, dims, strides, box, what);
}

// The weights as five dimensions in which a CTA's 128 features of a K block are one box: every
// copy costs the TMA unit some 100 cycles, which shows where few tokens leave little else in a
// stage (one token of one expert of 14336 x 4096, tiles whole: 54 us with two boxes, 46 with one).
//   [N, K]           {K, N, 1, 1, E}             box {64, 128, 1, 1, 1}
//   [N, K], gate     {K, 128, 2, N / 256, E}     box {64, 64, 2, 1, 1}   64 gate and 64 up rows
//   [K, N]           {64, K, N / 64, 1, E}       box {64, 64, 2, 1, 1}   64 does not divide N:
//                    {N, K, 1, 1, E}             box {64, 64, 1, 1, 1}   twice (w_halves)
//   [K, N], gate     {128, K, 2, N / 256, E}     box {64, 64, 2, 1, 1}
int weight_map(const TcclExpertGemm& d, GemmParams* p) {
  const bool gate = d.epilogue == kSiluGate || d.epilogue == kSiluGateGrad;
  const cuuint64_t ld = d.ldw * 2, slab = d.w_expert * 2, n = d.n, k = d.k, e = d.experts;
  cuuint64_t dims[5] = {0, 0, 1, 1, e}, strides[4] = {ld, 16, 16, slab};
  cuuint32_t box[5] = {64, 64, 2, 1, 1};
  p->w_nk = d.w_nk ? 1 : 0;
  p->w_halves = 0;
  if (gate) {
    dims[0] = d.w_nk ? k : 128;
    dims[1] = d.w_nk ? 128 : k;
    dims[2] = 2;
    dims[3] = n / 256;
    strides[1] = d.w_nk ? 128 * ld : 128 * 2;
    strides[2] = 2 * strides[1];
  } else if (d.w_nk) {
    dims[0] = k;
    dims[1] = n;
    box[1] = 128;
    box[2] = 1;
  } else if (n % 64 == 0) {
    dims[0] = 64;
    dims[1] = k;
    dims[2] = n / 64;
    strides[1] = 64 * 2;
  } else {
    dims[0] = n;
    dims[1] = k;
    box[2] = 1;
    p->w_halves = 1;
  }
  return encode(&p->tma_w, d.dtype == 1, d.w, 5, dims, strides, box, "W");
}

using GemmKernel = void (*)(const GemmParams);
template <bool kFew>
GemmKernel gemm_kernel(int epilogue) {
  return epilogue == kNone           ? expert_gemm_kernel<kNone, kFew>
         : epilogue == kSiluGate     ? expert_gemm_kernel<kSiluGate, kFew>
         : epilogue == kSiluGateGrad ? expert_gemm_kernel<kSiluGateGrad, kFew>
                                     : expert_gemm_kernel<kFloat, kFew>;
}

cudaError_t attrs_once(int* sms) {
  static int count[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && count[dev] != 0) { *sms = count[dev]; return cudaSuccess; }
  e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
  for (int i = 0; i < 8 && e == cudaSuccess; ++i)
    e = cudaFuncSetAttribute(i < 4 ? gemm_kernel<false>(i) : gemm_kernel<true>(i - 4),
                             cudaFuncAttributeMaxDynamicSharedMemorySize, kGemmSmem);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(expert_weight_grad_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kGradSmem);
  if (e == cudaSuccess && dev < 64) count[dev] = *sms;
  return e;
}

template <typename P>
cudaError_t launch_pairs(void (*kernel)(const P), const P& p, int pairs, int threads, int smem,
                         cudaStream_t stream, bool chained) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs), 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = chained ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

// Tiles of a product at most: a partial tile more per expert that has rows.
int64_t most_tiles(int64_t slots, int64_t experts, int64_t n) {
  return (slots / kTile + (slots < experts ? slots : experts)) * ((n + kTile - 1) / kTile);
}
int32_t partial_tokens(int64_t slots) {
  return static_cast<int32_t>(slots < kTile ? (slots + 31) / 32 * 32 : kTile);
}

// All waits of a launch have one deadline.  Nothing waits for a peer, so it grows with the work and
// only a fault can reach it: on top of the budget 100 us for every step (K block, or tile of zeros)
// that an SM pair can be given, which takes 0.15 - 3 us.
constexpr uint64_t kWaitBudgetNs = 2000000000ull, kNsPerStep = 100000;
uint64_t deadline_ns(uint64_t budget, int64_t steps) {
  const int64_t most = int64_t(1) << 30;       // (a day; the product stays far below 2^64)
  return (budget ? budget : kWaitBudgetNs) + kNsPerStep * static_cast<uint64_t>(steps < most ? steps : most);
}

}  // namespace

cudaError_t preload_expert_gemm_kernels() {
  cudaFuncAttributes a;
  int sms = 0;
  cudaError_t e = cudaFuncGetAttributes(&a, expert_weight_grad_kernel);
  for (int i = 0; i < 8 && e == cudaSuccess; ++i)
    e = cudaFuncGetAttributes(&a, i < 4 ? gemm_kernel<false>(i) : gemm_kernel<true>(i - 4));
  if (e == cudaSuccess) e = attrs_once(&sms);
  return e;
}

}  // namespace tileccl

using namespace tileccl;

// Tiles may be shared for at most this many slots, and at least this long a contraction (see the
// schedule of expert_gemm_kernel).  What sharing gains grows with the contraction, what it costs
// with the rows of an expert (partial sums) and the parts of a tile.  Weights from DRAM, us shared /
// whole, K x N with the rows of every expert in front:
//   1 row    1024 x 4096 10.9 / 10.1   1792 x 4096 11.7 / 12.2   2048 x 4096 14.1 / 12.8
//            3584 x 4096 15.9 / 17.0   4096 x 4096 16.4 / 18.4   4096 x 19200 33.6 / 38.3
//   16 rows  2048 x 4096 14.6 / 13.1   3584 x 4096 17.2 / 17.2   4096 x 4096 16.7 / 18.7
//   32 rows  4096 x 4096 18.4 / 19.1   of each of 4 experts: 4096 x 1024 18.3 / 20.1
//   64 rows  4096 x 4096 22.1 / 19.9   6144 x 4096 25.6 / 25.5   8192 x 4096 27.7 / 31.2
//   128 rows 4096 x 4096 29.0 / 23.1   8192 x 4096 35.4 / 36.2   14336 x 4096 45.1 / 57.0
//            4096 x 1024 39.4 / 22.1   8192 x 1024 48.4 / 34.3   14336 x 1024 47.7 / 52.7
// The limits are those of the sum over experts, which the host knows: more than 32 rows of a single
// expert lose below K = 6144, and 3584 would gain with one row.
constexpr int64_t kSharedSlots = 128, kSharedK = 4096;

extern "C" int tccl_expert_gemm_scratch(int64_t slots, int64_t k, int64_t* partial_bytes,
                                        int64_t* counter_bytes) {
  TCCL_CHECK_ARG(partial_bytes != nullptr && counter_bytes != nullptr, "null argument");
  *partial_bytes = *counter_bytes = 0;
  int sms = 0;
  TCCL_CHECK_CUDA(attrs_once(&sms));
  const int64_t pairs = sms / 2;
  if (slots <= 0 || slots > kSharedSlots || k < kSharedK) return kOk;
  *partial_bytes = pairs * 4 * 128 * partial_tokens(slots) * static_cast<int64_t>(sizeof(float));
  *counter_bytes = pairs * 4 * static_cast<int64_t>(sizeof(uint32_t));
  return kOk;
}

extern "C" int tccl_expert_state(uint64_t* status, uint64_t* counters, int64_t* counter_bytes) {
  TCCL_CHECK_ARG(status != nullptr && counters != nullptr && counter_bytes != nullptr, "null argument");
  // (the first call may load the module, which a capture does not have to notice)
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  TCCL_CHECK_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
  void *s = nullptr, *c = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&s, g_status);
  if (e == cudaSuccess) e = cudaGetSymbolAddress(&c, g_counters);
  cudaThreadExchangeStreamCaptureMode(&mode);
  TCCL_CHECK_CUDA(e);
  *status = reinterpret_cast<uint64_t>(s);
  *counters = reinterpret_cast<uint64_t>(c);
  *counter_bytes = kCounterBytes;
  return kOk;
}

extern "C" int tccl_stream_id(uint64_t stream, uint64_t* id) {
  TCCL_CHECK_ARG(id != nullptr, "null argument");
  unsigned long long v = 0;
  TCCL_CHECK_CUDA(cudaStreamGetId(reinterpret_cast<cudaStream_t>(stream), &v));
  *id = v;
  return kOk;
}

extern "C" int tccl_expert_status(uint32_t* words) {
  TCCL_CHECK_ARG(words != nullptr, "null argument");
  TCCL_CHECK_CUDA(cudaMemcpyFromSymbol(words, g_status, sizeof(g_status)));
  if (words[0] == 0) return kOk;
  void *s = nullptr, *c = nullptr;
  TCCL_CHECK_CUDA(cudaGetSymbolAddress(&s, g_status));
  TCCL_CHECK_CUDA(cudaGetSymbolAddress(&c, g_counters));
  TCCL_CHECK_CUDA(cudaMemset(s, 0, sizeof(g_status)));
  TCCL_CHECK_CUDA(cudaMemset(c, 0, sizeof(g_counters)));
  TCCL_CHECK_CUDA(cudaDeviceSynchronize());          // (other streams do not wait for these)
  return kOk;
}

extern "C" int tccl_expert_gemm(const TcclExpertGemm* desc, uint64_t stream) {
  TCCL_CHECK_ARG(desc != nullptr, "null argument");
  TcclExpertGemm d = *desc;
  TCCL_CHECK_ARG(d.dtype == 0 || d.dtype == 1, "dtype must be 0 (fp16) or 1 (bf16)");
  TCCL_CHECK_ARG(d.epilogue >= kNone && d.epilogue <= kFloat, "epilogue must be 0..3");
  TCCL_CHECK_ARG(d.experts >= 1 && d.experts <= kMaxExperts, "experts must be 1..1024");
  TCCL_CHECK_ARG(d.k >= 1 && d.n >= 1 && d.k < (int64_t(1) << 31) && d.n < (int64_t(1) << 31) - kTile,
                 "K and N must be 1..2^31");
  TCCL_CHECK_ARG(d.k % 8 == 0, "K must be a multiple of 8 (16-byte TMA rows)");
  TCCL_CHECK_ARG(d.n % 8 == 0, "N must be a multiple of 8 (16-byte TMA rows)");
  TCCL_CHECK_ARG(d.ldx % 8 == 0 && d.ldw % 8 == 0 && d.w_expert % 8 == 0 && d.ldo % 8 == 0 &&
                     d.ld_dh % 8 == 0,
                 "leading dimensions must be multiples of 8 elements");
  TCCL_CHECK_ARG(d.x % 16 == 0 && d.w % 16 == 0 && d.out % 16 == 0 && d.dh % 16 == 0,
                 "operands must be 16-byte aligned");
  TCCL_CHECK_ARG(d.epilogue == kNone || d.epilogue == kFloat || d.n % 256 == 0,
                 "SiLU-gate epilogue needs N to be a multiple of 256");
  TCCL_CHECK_ARG(d.slots >= 0 && d.slots < (int64_t(1) << 31) - kTile, "too many rows");
  if (d.slots == 0) return kOk;
  TCCL_CHECK_ARG(d.x != 0 && d.w != 0 && d.out != 0 && d.offsets != 0, "null argument");
  TCCL_CHECK_ARG(d.epilogue != kSiluGateGrad || d.dh != 0, "null argument");
  TCCL_CHECK_ARG(d.token_of_slot == 0 || (d.x_slots != 0 && d.x_slots % 16 == 0 && d.x_rows >= 1),
                 "gathered rows need scratch");
  TCCL_CHECK_ARG(d.partial == 0 || (d.counters != 0 && d.partial % 16 == 0), "bad scratch");
  const int64_t f_tiles = (d.n + kTile - 1) / kTile, tiles = most_tiles(d.slots, d.experts, d.n);
  TCCL_CHECK_ARG(tiles < (int64_t(1) << 31), "too many tiles");
  TCCL_REQUIRE_DRIVER();
  if (d.token_of_slot != 0) {
    // the tokens' rows in slot order first
    const int rc = tccl_expert_gather(d.x, d.ldx, d.x_rows, d.token_of_slot, d.x_slots, d.k, d.slots,
                                      static_cast<int32_t>(d.k), stream);
    if (rc) return rc;
    d.x = d.x_slots;
    d.ldx = d.k;
  }
  const bool bf16 = d.dtype == 1;
  GemmParams p;
  int rc = weight_map(d, &p);
  if (rc) return rc;
  for (int i = 0; i < 4; ++i) {
    rc = encode_rows(&p.tma_x[i], bf16, d.x, d.k, d.slots, d.ldx * 2, 128 >> i, "X");
    if (rc) return rc;
  }
  p.offsets = reinterpret_cast<const int32_t*>(d.offsets);
  p.out = reinterpret_cast<void*>(d.out);
  p.dh = reinterpret_cast<const void*>(d.dh);
  p.ldo = d.ldo;
  p.ld_dh = d.ld_dh;
  p.slots = static_cast<int32_t>(d.slots);
  p.k_blocks = static_cast<int32_t>((d.k + kBK - 1) / kBK);
  // (K blocks of all shared tiles are counted in 32 bits)
  p.partial = p.k_blocks < (1 << 20) ? reinterpret_cast<float*>(d.partial) : nullptr;
  p.counters = reinterpret_cast<uint32_t*>(d.counters);
  p.partial_tokens = partial_tokens(d.slots);
  p.experts = d.experts;
  p.n = static_cast<int32_t>(d.n);
  p.f_tiles = static_cast<int32_t>(f_tiles);
  p.bf16 = bf16 ? 1 : 0;
  p.status = reinterpret_cast<uint32_t*>(d.status);
  int sms = 0;
  TCCL_CHECK_CUDA(attrs_once(&sms));
  // (a shared tile is cut into runs of kMinBlocks K blocks at least)
  const int64_t runs = p.partial == nullptr ? tiles : tiles * ((p.k_blocks + kMinBlocks - 1) / kMinBlocks);
  const int pairs = static_cast<int>(runs < sms / 2 ? runs : sms / 2);
  p.budget_ns = deadline_ns(d.wait_budget_ns, (tiles / pairs + 2) * (p.k_blocks + int64_t(1)));
  const GemmKernel kernel =
      d.slots <= kFewTokens ? gemm_kernel<true>(d.epilogue) : gemm_kernel<false>(d.epilogue);
  TCCL_CHECK_CUDA(launch_pairs(kernel, p, pairs,
                               kThreads, kGemmSmem,
                               reinterpret_cast<cudaStream_t>(stream), d.token_of_slot != 0));
  return kOk;
}

extern "C" int tccl_expert_weight_grad(const TcclExpertWeightGrad* desc, uint64_t stream) {
  TCCL_CHECK_ARG(desc != nullptr, "null argument");
  const TcclExpertWeightGrad& d = *desc;
  TCCL_CHECK_ARG(d.dtype == 0 || d.dtype == 1, "dtype must be 0 (fp16) or 1 (bf16)");
  TCCL_CHECK_ARG(d.experts >= 1 && d.experts <= kMaxExperts, "experts must be 1..1024");
  TCCL_CHECK_ARG(d.m >= 1 && d.n >= 1 && d.m < (int64_t(1) << 31) - kTile &&
                     d.n < (int64_t(1) << 31) - kTile, "rows and columns must be 1..2^31");
  TCCL_CHECK_ARG(d.m % 8 == 0 && d.n % 8 == 0, "rows and columns must be multiples of 8");
  TCCL_CHECK_ARG(d.lda % 8 == 0 && d.ldb % 8 == 0, "leading dimensions must be multiples of 8 elements");
  TCCL_CHECK_ARG(d.a % 16 == 0 && d.b % 16 == 0 && d.out % 16 == 0, "operands must be 16-byte aligned");
  TCCL_CHECK_ARG(d.slots >= 0 && d.slots < (int64_t(1) << 31) - kTile, "too many rows");
  TCCL_CHECK_ARG(d.out != 0 && d.offsets != 0, "null argument");
  if (d.slots == 0) {
    TCCL_CHECK_CUDA(cudaMemsetAsync(reinterpret_cast<void*>(d.out), 0, d.experts * d.m * d.n * 2,
                                    reinterpret_cast<cudaStream_t>(stream)));
    return kOk;
  }
  TCCL_CHECK_ARG(d.a != 0 && d.b != 0, "null argument");
  const int64_t m_tiles = (d.m + kTile - 1) / kTile, n_tiles = (d.n + kTile - 1) / kTile;
  const int64_t tiles = d.experts * m_tiles * n_tiles;
  TCCL_CHECK_ARG(tiles < (int64_t(1) << 31), "too many tiles");
  TCCL_REQUIRE_DRIVER();
  const bool bf16 = d.dtype == 1;
  GradParams p;
  auto operand = [&](CUtensorMap* map, uint64_t base, uint64_t cols, uint64_t ld, int32_t* halves,
                     const char* what) {
    *halves = cols % 64 != 0 ? 1 : 0;
    const cuuint64_t dims[3] = {*halves ? cols : 64, static_cast<cuuint64_t>(d.slots), *halves ? 1 : cols / 64};
    const cuuint64_t strides[2] = {ld * 2, 128};
    const cuuint32_t box[3] = {64, 64, *halves ? 1u : 2u};
    return encode(map, bf16, base, 3, dims, strides, box, what);
  };
  int rc = operand(&p.tma_a, d.a, d.m, d.lda, &p.a_halves, "A");
  if (!rc) rc = operand(&p.tma_b, d.b, d.n, d.ldb, &p.b_halves, "B");
  if (!rc) {
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(d.n), static_cast<cuuint64_t>(d.m),
                                static_cast<cuuint64_t>(d.experts)};
    const cuuint64_t strides[2] = {dims[0] * 2, dims[0] * dims[1] * 2};
    const cuuint32_t box[3] = {64, 32, 1};
    rc = encode(&p.tma_out, bf16, d.out, 3, dims, strides, box, "out");
  }
  if (rc) return rc;
  p.offsets = reinterpret_cast<const int32_t*>(d.offsets);
  p.a = reinterpret_cast<const void*>(d.a);
  p.b = reinterpret_cast<const void*>(d.b);
  p.lda = d.lda;
  p.ldb = d.ldb;
  p.slots = static_cast<int32_t>(d.slots);
  p.experts = d.experts;
  p.m = static_cast<int32_t>(d.m);
  p.n = static_cast<int32_t>(d.n);
  p.m_tiles = static_cast<int32_t>(m_tiles);
  p.n_tiles = static_cast<int32_t>(n_tiles);
  p.bf16 = bf16 ? 1 : 0;
  p.status = reinterpret_cast<uint32_t*>(d.status);
  int sms = 0;
  TCCL_CHECK_CUDA(attrs_once(&sms));
  const int pairs = static_cast<int>(tiles < sms / 2 ? tiles : sms / 2);
  // (a pair has at most m_tiles * n_tiles / pairs + 1 tiles of an expert; the experts together have
  // slots / kBK blocks of rows and one more each)
  p.budget_ns = deadline_ns(d.wait_budget_ns,
                            (m_tiles * n_tiles / pairs + 1) * (d.slots / kBK + 2 * int64_t(d.experts)));
  TCCL_CHECK_CUDA(launch_pairs(&expert_weight_grad_kernel, p, pairs, kThreads + kCopyThreads, kGradSmem,
                               reinterpret_cast<cudaStream_t>(stream), false));
  return kOk;
}
