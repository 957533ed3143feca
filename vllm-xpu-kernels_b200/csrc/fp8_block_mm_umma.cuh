// The fp8 block-scaled product on the fifth-generation tensor cores (tcgen05, kind::f8f6f4).
//
// A row of a tile is 128 bytes: 128 fp8 values, one scale group, one row of the 128-byte-swizzle layout.  A group's
// products are four MMAs of K = 32 into tensor-memory columns of their own; the epilogue threads read them, multiply by
// the product of the group's two scales and add them to fp32 accumulators in registers, while the tensor pipe works on
// the next groups.  The scales thus never meet the operands and cost one fused multiply-add per element and group.
//
// Operands come in by TMA (128-byte swizzle, plain loads): columns past K and rows past the matrix read as zeros.
// Every wait on an mbarrier is bounded; a wait that gives up sets the CTA's abort word.  The CTA runs to its end and, once none
// of its threads can wait any more, waits (bounded) for its copies and MMAs in flight, frees its tensor memory and raises
// g_block_mm_status.  Results that it could not compute are written as NaN: nobody takes them for a product.
#pragma once

#include <cuda.h>

#include "kvc_common.cuh"
#include "tensor_map.cuh"
#include "umma_sm100.cuh"

namespace kvc {
namespace {

__device__ int g_block_mm_status = 0;

struct BlockMmMaps {
  CUtensorMap a, b;  // boxes of 128 bytes x the tile's rows
};

// one box of a tiled 2-d tensor map -> shared memory of this CTA; completion is counted in bytes on `bar`
__device__ __forceinline__ void mm_tma_load(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(umma::smem_addr(bar)), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void mm_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(umma::smem_addr(bar)), "r"(bytes) : "memory");
}
// A wait by a whole warp whose lanes then go on together, whatever each of them saw.
__device__ __forceinline__ bool mm_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_word,
                                        uint32_t max_tries = umma::kMaxTries) {
  return __all_sync(0xFFFFFFFFu, umma::mbar_wait_bounded(bar, parity, abort_word, max_tries));
}
// The same for two events, with one vote.
__device__ __forceinline__ bool mm_wait(uint64_t* bar, uint32_t parity, uint64_t* bar2, uint32_t parity2, volatile uint32_t* abort_word) {
  return __all_sync(0xFFFFFFFFu, umma::mbar_wait_bounded(bar, parity, abort_word) && umma::mbar_wait_bounded(bar2, parity2, abort_word));
}
// A wait that ignores the abort word: lets what is in flight land before the CTA ends.  `times` half a second at most.
__device__ __forceinline__ void mm_wait_limited(uint64_t* bar, uint32_t parity, uint32_t times = 1) {
  for (uint32_t i = 0; i < times * umma::kMaxTries; ++i)
    if (umma::mbar_try_wait(bar, parity, umma::kTryNs)) return;
}

// Position in a ring of N slots and the parity of the slot's current round.  Two warps that take turns start at 0 and 1
// and advance by 2 (N is even then).
template <int N, int STEP = 1>
struct Ring {
  static_assert(N % STEP == 0, "a turn ends with the ring");
  uint32_t slot, parity = 0;
  __device__ __forceinline__ explicit Ring(uint32_t first = 0) : slot(first) {}
  __device__ __forceinline__ void advance() {
    slot += STEP;
    if (slot >= N) {
      slot -= N;
      parity ^= 1;
    }
  }
};

// asks L2 for a tile of a tensor map
__device__ __forceinline__ void prefetch_tile(const CUtensorMap* map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1)
               : "memory");
}

// two fp32 values in one 64-bit register, and arithmetic on both halves in one instruction (each correctly rounded)
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}
__device__ __forceinline__ void unpack2u(uint64_t v, uint32_t& lo, uint32_t& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm volatile("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// A read-only load that stays where it is written: scales are asked for a group ahead of their use, and the compiler
// would move an ordinary load down to that use.
__device__ __forceinline__ float ld_ahead(const float* p) {
  float v;
  asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// By every thread of every CTA of the cluster (its CTAs are scheduled together, so the wait ends).
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same in two halves, without ordering memory: every thread of the cluster arrives once its CTA has begun, and waits before
// its first access to another CTA's shared memory, which is not there before that CTA has begun.
__device__ __forceinline__ void cluster_begun_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_begun_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// The address that `local_addr` of this CTA's shared memory has in CTA `rank` of the cluster, and a store to it.
__device__ __forceinline__ uint32_t cluster_addr(uint32_t local_addr, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_addr), "r"(rank));
  return remote;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void st_cluster4(uint32_t addr, uint4 v) {
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// Results at addresses that are multiples of the element only.  LANES neighbouring lanes hold one 32-bit word each of a row's
// piece (lane w: element w, or elements 2w and 2w + 1); `left` of the piece's elements exist.  Where a piece of 16-bit
// elements begins in the middle of a word, every lane writes the word that ends with its first element, and the two elements
// at the piece's ends go out singly.  Without branches.  By all lanes of a warp.
__device__ __forceinline__ void st_if(bool yes, void* to, uint32_t v) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\t@q st.global.u32 [%0], %1;\n\t}" ::"l"(to), "r"(v),
               "r"(static_cast<uint32_t>(yes)) : "memory");
}
__device__ __forceinline__ void st_half_if(bool yes, void* to, uint32_t v) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\t@q st.global.u16 [%0], %1;\n\t}" ::"l"(to),
               "h"(static_cast<uint16_t>(v)), "r"(static_cast<uint32_t>(yes)) : "memory");
}
template <typename Tout>
__device__ __forceinline__ uint32_t result_word(float x, float y) {
  if constexpr (sizeof(Tout) == 4) {
    return __float_as_uint(x);
  } else {
    const Tout lo = from_f32<Tout>(x), hi = from_f32<Tout>(y);
    return *reinterpret_cast<const uint16_t*>(&lo) | static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(&hi)) << 16;
  }
}
template <typename Tout, int LANES>
__device__ __forceinline__ void store_words(uint32_t v, int w, Tout* piece, int left) {
  if constexpr (sizeof(Tout) == 4) {
    st_if(w < left, piece + w, v);
  } else {
    const uint32_t before = __shfl_up_sync(0xFFFFFFFFu, v, 1, LANES);
    const int odd = static_cast<int>(reinterpret_cast<uintptr_t>(piece) >> 1) & 1;
    const uint32_t word = odd ? __byte_perm(before, v, 0x5432) : v;
    const int e = 2 * w - odd;  // the word's first element; -1: of the piece before
    st_if(e >= 0 && e + 1 < left, piece + e, word);
    const bool first = e < 0 && left > 0, last = odd && w == LANES - 1 && left >= 2 * LANES, end = e >= 0 && e + 1 == left;
    st_half_if(first || last || end, piece + (first ? 0 : last ? 2 * LANES - 1 : e), first ? v : last ? v >> 16 : word);
  }
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// ---------------------------------------------------------------------------------------------
// few rows of a: one tile of 128 weight rows per CTA or cluster
// ---------------------------------------------------------------------------------------------
// A CTA owns 128 rows of b and TOK rows of a, and a contiguous share of the groups; the CTAs of a cluster divide the
// groups of one tile.
//   epilogue warpgroups: thread r of each owns lane r of tensor memory and, of its columns, 1 / kSplit.  Below 128 tokens
//              lanes are rows of b and columns tokens; kTurns sets of warpgroups take the groups in turn.  At 128 lanes are
//              tokens: a thread then needs one scale per group where it needs one per column otherwise, and reading those
//              (the same for all lanes, but each warp's 16 bytes per lane take four cycles of the SM's one pipe) was what a
//              group waited for: 393 ns, against 313 this way
//   kIssuers warps issue the MMAs (M = 128, N = TOK), taking the groups in turn
//   kIssuers warps issue the TMA loads, in turn as well
// In the end every thread sends its accumulators to the CTA of the cluster that owns their token (distributed shared
// memory), which adds them in the order of ranks and warpgroups and writes whole rows.
//
// An MMA this narrow takes 56 cycles whatever N is (measured), so a group of 16 KB of weights takes at least 225 where the
// SM's share of the HBM rate would allow 700: the point is to add little to that.  A warp that issues a group's MMAs
// cannot go on before the pipe has taken them, and then needs another 250 cycles for its barriers; hence two such warps.
template <int TOK>
struct ThinCfg {
  static constexpr int kCtasPerSm = TOK == 64 ? 2 : 1;
  static constexpr int kTurns = TOK <= 32 ? 2 : 1;
  static constexpr int kSplit = TOK <= 64 ? 1 : 4;
  static constexpr int kEpilogueWarps = 4 * kTurns * kSplit;
  static constexpr int kIssuers = kCtasPerSm == 1 ? 2 : 1;  // warps that issue MMAs, and as many that issue loads
  static constexpr int kThreads = (kEpilogueWarps + 2 * kIssuers) * 32;
  static constexpr bool kTokenLanes = TOK == 128;
  static constexpr int kAcc = TOK / kSplit;  // accumulators of a thread
  static constexpr int kTileB = 128 * 128;
  static constexpr int kTileA = TOK * 128;
  static constexpr int kStageBytes = kTileA + kTileB;
  static constexpr int kStages = TOK <= 32 ? 8 : TOK == 64 ? 3 : 4;
  static constexpr int kBuffers = TOK <= 32 ? 8 : 4;     // groups of products in tensor memory
  static constexpr int kCols = kBuffers * TOK;           // 128 .. 512
  static constexpr int kScaleGroups = TOK <= 32 ? 32 : TOK == 64 ? 8 : 16;  // groups whose scales are fetched at once
  static constexpr int kOffScales = kStages * kStageBytes;
  static constexpr int kScaleBytes = kScaleGroups * TOK * 4;  // two of them
  static constexpr int kOffSums = kOffScales + 2 * kScaleBytes;
  // Sums of the CTA's tokens, rows of 128 floats.  Where a thread writes 16 bytes of a row of its own, rows lie four banks
  // apart, so that eight threads meet all banks.
  static constexpr int kSumRow = kTokenLanes ? 132 : 128;
  static constexpr int kSumBytes = kTurns * (TOK + 7) * kSumRow * 4;  // splits * ceil(TOK / splits) rows
  static constexpr int kOffBar = kOffSums + kSumBytes;
  static constexpr int kBars = 2 * kStages + 2 * kBuffers + 1;
  static constexpr int kUsed = kOffBar + kBars * 8 + 16;
  // So much that kCtasPerSm CTAs fit an SM and no more: their tensor memory is then always there (CTAs of two clusters
  // could otherwise wait for each other's).
  static constexpr int kLeast = (kCtasPerSm == 1 ? 120 : 77) * 1024;
  static constexpr int kSmem = (kUsed > kLeast ? kUsed : kLeast) + 1024;
  static_assert(kSmem <= 232448 && kCtasPerSm * (kSmem + 1024) <= 233472 && (kCtasPerSm + 1) * (kSmem + 1024) > 233472, "");
  static_assert(kCtasPerSm * kCols <= 512 && kBuffers % kTurns == 0, "");
};
// Of different variants (calls on two streams) no two fit an SM together, for the same reason.
static_assert(ThinCfg<64>::kSmem + ThinCfg<16>::kSmem + 2048 > 233472 && ThinCfg<64>::kSmem + ThinCfg<32>::kSmem + 2048 > 233472 &&
                  ThinCfg<64>::kSmem + ThinCfg<128>::kSmem + 2048 > 233472 && 2 * ThinCfg<16>::kSmem + 2048 > 233472, "");
constexpr int kMaxSplits = 8;
constexpr int kPrefetchGroups = 16;

struct ThinParams {
  const float* a_scales;
  const float* b_scales;
  void* out;
  int64_t out_stride, as_stride_m, as_stride_g, bs_stride_n, bs_stride_g;
  int32_t m, n, groups, groups_per_split, splits;
  int32_t own;       // tokens a CTA of the cluster sums: ceil(TOK / splits)
  bool wide_stores;  // every 8-element piece of a row of out is aligned to 16 bytes
};

// Scales of kScaleGroups groups, [group][token], by cp.async.  Lanes run along the groups where those are closer
// together in memory than the tokens, else along the tokens.  Places of tokens past m are left as they are: their
// products are not stored.
template <int TOK>
__device__ __forceinline__ void thin_fetch_scales(const ThinParams& p, float* to, int m0, int first, int end) {
  using Cfg = ThinCfg<TOK>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tokens = min(TOK, p.m - m0), groups = min(Cfg::kScaleGroups, end - first);
  const bool along_groups = p.as_stride_g <= p.as_stride_m;
  constexpr int kSpan = TOK < 32 ? TOK : 32;               // tokens of a warp's access along the tokens
  constexpr int kGroupSpan = Cfg::kScaleGroups;            // groups of a warp's access along the groups
  const int tok0 = along_groups ? warp * (32 / kGroupSpan) + lane / kGroupSpan : lane % kSpan;
  const int tok_step = along_groups ? Cfg::kEpilogueWarps * (32 / kGroupSpan) : kSpan;
  const int g0 = along_groups ? lane % kGroupSpan : warp * (32 / kSpan) + lane / kSpan;
  const int g_step = along_groups ? kGroupSpan : Cfg::kEpilogueWarps * (32 / kSpan);
  for (int g = g0; g < groups; g += g_step) {
    const float* src = p.a_scales + (m0 + tok0) * p.as_stride_m + (first + g) * p.as_stride_g;
    uint32_t dst = umma::smem_addr(to + g * TOK + tok0);
    for (int tok = tok0; tok < tokens; tok += tok_step, src += tok_step * p.as_stride_m, dst += 4 * tok_step)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}

template <int F8, typename Tout, int TOK>
__global__ void __launch_bounds__(ThinCfg<TOK>::kThreads, ThinCfg<TOK>::kCtasPerSm)
    block_mm_thin_kernel(const __grid_constant__ BlockMmMaps maps, const __grid_constant__ ThinParams p) {
  using namespace umma;
  using Cfg = ThinCfg<TOK>;
  extern __shared__ unsigned char raw[];
  unsigned char* smem = raw + ((1024u - (smem_addr(raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  uint64_t* full = bars;
  uint64_t* empty = full + Cfg::kStages;
  uint64_t* ready = empty + Cfg::kStages;       // a group's products are in tensor memory
  uint64_t* taken = ready + Cfg::kBuffers;      // and have been read
  uint64_t* drained = taken + Cfg::kBuffers;    // after a wait that gave up: no MMA is in flight
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::kBars);
  volatile uint32_t* abort_word = tmem_slot + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kMmaWarp = Cfg::kEpilogueWarps, kLoadWarp = kMmaWarp + Cfg::kIssuers, kTakeTurns = Cfg::kIssuers;

  if (threadIdx.x == 0) {
    prefetch_map(&maps.a);
    prefetch_map(&maps.b);
    for (int i = 0; i < Cfg::kStages; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < Cfg::kBuffers; ++i) {
      mbar_init(ready + i, 1);
      mbar_init(taken + i, 4 * Cfg::kSplit);
    }
    mbar_init(drained, Cfg::kIssuers);
    *abort_word = 0;
    mbar_init_fence();
  }
  __syncwarp();
  if (p.splits > 1) cluster_begun_arrive();
  const uint32_t rank = p.splits > 1 ? cluster_rank() : 0;
  const int n_tile = blockIdx.x / p.splits;
  const int n0 = n_tile * 128, m0 = blockIdx.y * TOK;
  const int g0 = rank * p.groups_per_split;
  const int count = min(p.groups_per_split, p.groups - g0);  // >= 1
  // While the kernel before this one ends, L2 may already fetch this CTA's weights (a hint: nothing is read yet).
  if (warp == kLoadWarp && lane < min(count, kPrefetchGroups)) prefetch_tile(&maps.b, (g0 + lane) * 128, n0);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == kMmaWarp) tmem_alloc(tmem_slot, Cfg::kCols);
  fence_before_thread_sync();
  __syncthreads();
  fence_after_thread_sync();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  float* sums = reinterpret_cast<float*>(smem + Cfg::kOffSums);
  int asked = warp - kLoadWarp;  // a loading warp has asked for its groups below this one

  if (warp >= kLoadWarp) {
    Ring<Cfg::kStages, kTakeTurns> at(warp - kLoadWarp);
    for (; asked < count; asked += kTakeTurns, at.advance()) {
      // a slot is free from the start (the round "before" the first counts as finished)
      if (!mm_wait(empty + at.slot, at.parity ^ 1, abort_word)) break;
      if (elect_one()) {
        mm_expect_tx(full + at.slot, Cfg::kStageBytes);
        const uint32_t dst = smem_addr(smem + at.slot * Cfg::kStageBytes);
        mm_tma_load(dst, &maps.b, full + at.slot, (g0 + asked) * 128, n0);
        mm_tma_load(dst + Cfg::kTileB, &maps.a, full + at.slot, (g0 + asked) * 128, m0);
      }
      __syncwarp();
    }
    __syncwarp();
    if (p.splits > 1) cluster_begun_wait();
  } else if (warp >= kMmaWarp) {
    constexpr uint32_t idesc = instr_desc_f8(128, TOK, F8 == KVC_KV_FP8_E5M2);
    Ring<Cfg::kStages, kTakeTurns> at(warp - kMmaWarp);
    Ring<Cfg::kBuffers, kTakeTurns> buf(warp - kMmaWarp);
    for (int i = warp - kMmaWarp; i < count; i += kTakeTurns, at.advance(), buf.advance()) {
      if (!mm_wait(taken + buf.slot, buf.parity ^ 1, full + at.slot, at.parity, abort_word)) break;
      fence_after_thread_sync();
      if (elect_one()) {
        const uint32_t base = smem_addr(smem + at.slot * Cfg::kStageBytes);
        const uint64_t weights = smem_desc_sw128(base, 0, 1024), tokens = smem_desc_sw128(base + Cfg::kTileB, 0, 1024);
        const uint64_t da = Cfg::kTokenLanes ? tokens : weights, db = Cfg::kTokenLanes ? weights : tokens;
#pragma unroll
        for (int k = 0; k < 4; ++k) mma_f8_ss(tmem + buf.slot * TOK, da + 2 * k, db + 2 * k, idesc, k > 0);
        mma_commit(empty + at.slot);
        mma_commit(ready + buf.slot);
      }
      __syncwarp();
    }
    __syncwarp();
    if (p.splits > 1) cluster_begun_wait();
  } else {
    const int turn = (warp >> 2) % Cfg::kTurns, row = threadIdx.x & 127;
    const int col0 = (warp >> 2) / Cfg::kTurns * Cfg::kAcc;
    constexpr int kStep = Cfg::kTurns;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + col0;
    float* scales = reinterpret_cast<float*>(smem + Cfg::kOffScales);
    auto fetch = [&](int chunk) {
      thin_fetch_scales<TOK>(p, scales + (chunk & 1) * (Cfg::kScaleGroups * TOK), m0, g0 + chunk * Cfg::kScaleGroups,
                             g0 + count);
    };
    uint64_t acc[Cfg::kAcc / 2];
#pragma unroll
    for (int j = 0; j < Cfg::kAcc / 2; ++j) acc[j] = 0;
    // b's scales of the groups whose places in `scales` this thread multiplies by them, a chunk ahead of their use
    constexpr int kMine = Cfg::kScaleGroups * TOK / (Cfg::kEpilogueWarps * 32);
    const float* b_scale = p.b_scales + n_tile * p.bs_stride_n + g0 * p.bs_stride_g;
    float sb[kMine];
    auto fetch_b = [&](int chunk) {
#pragma unroll
      for (int e = 0; e < kMine; ++e) {
        const int g = chunk * Cfg::kScaleGroups + (e * (Cfg::kEpilogueWarps * 32) + static_cast<int>(threadIdx.x)) / TOK;
        sb[e] = g < count ? ld_ahead(b_scale + g * p.bs_stride_g) : 0.0f;
      }
    };
    int i = turn;  // this thread's next group
    uint32_t b = i, parity = 0;          // and its buffer
    fetch_b(0);
    fetch(0);
    fetch(1);
    for (int chunk = 0; chunk * Cfg::kScaleGroups < count; ++chunk) {
      if (chunk > 0) {  // everyone has used the chunk before: its place can be filled again
        asm volatile("bar.sync 1, %0;" ::"n"(Cfg::kEpilogueWarps * 32) : "memory");
        fetch(chunk + 1);
      }
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      asm volatile("bar.sync 1, %0;" ::"n"(Cfg::kEpilogueWarps * 32) : "memory");
      // a place holds the product of its row's and the weight block's scale from here on
#pragma unroll
      for (int e = 0; e < kMine; ++e) {
        float* place = scales + (chunk & 1) * (Cfg::kScaleGroups * TOK) + e * (Cfg::kEpilogueWarps * 32) + threadIdx.x;
        *place = __fmul_rn(*place, sb[e]);
      }
      fetch_b(chunk + 1);
      asm volatile("bar.sync 1, %0;" ::"n"(Cfg::kEpilogueWarps * 32) : "memory");
      const int end = min(count, (chunk + 1) * Cfg::kScaleGroups);
      const float* chunk_scales = scales + (chunk & 1) * (Cfg::kScaleGroups * TOK) + (Cfg::kTokenLanes ? row : col0);
      for (; i < end; i += kStep) {
        const float* group_scales = chunk_scales + (i - chunk * Cfg::kScaleGroups) * TOK;
        uint64_t lane_scale = 0;
        if constexpr (Cfg::kTokenLanes) {
          const uint32_t s = __float_as_uint(*group_scales);
          lane_scale = pack2(s, s);
        }
        mbar_wait_bounded(ready + b, parity, abort_word);
        fence_after_thread_sync();
        constexpr int kPiece = Cfg::kAcc < 32 ? Cfg::kAcc : 32;
#pragma unroll
        for (int c = 0; c < Cfg::kAcc; c += kPiece) {
          uint32_t v[kPiece];
          if constexpr (kPiece == 32) tmem_ld_32x32(lane_base + b * TOK + c, v);
          else tmem_ld_32x16(lane_base + b * TOK + c, v);
          tmem_ld_wait();
          if (c + kPiece == Cfg::kAcc) {
            fence_before_thread_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(taken + b);
          }
#pragma unroll
          for (int j = 0; j < kPiece / 4; ++j) {
            ulonglong2 s = make_ulonglong2(lane_scale, lane_scale);
            if constexpr (!Cfg::kTokenLanes) s = reinterpret_cast<const ulonglong2*>(group_scales)[c / 4 + j];
            acc[c / 2 + 2 * j] = fma_f32x2(pack2(v[4 * j], v[4 * j + 1]), s.x, acc[c / 2 + 2 * j]);
            acc[c / 2 + 2 * j + 1] = fma_f32x2(pack2(v[4 * j + 2], v[4 * j + 3]), s.y, acc[c / 2 + 2 * j + 1]);
          }
          __syncwarp();  // keeps the additions here: the compiler would move them behind the next waits
        }
        b += kStep;
        if (b >= Cfg::kBuffers) {
          b -= Cfg::kBuffers;
          parity ^= 1;
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    // Every CTA of the cluster has begun (long ago, as a rule): its shared memory can be written.  A CTA with a short last
    // share of the groups may come here while another one is still being launched.
    __syncwarp();
    if (p.splits > 1) cluster_begun_wait();
    // to the owner of the token: [rank and turn][token of the owner][row of b]
    const uint32_t part = rank * Cfg::kTurns + turn;
    if constexpr (Cfg::kTokenLanes) {
      // A thread's columns are 16-byte pieces of one row, a warp's 32 rows: in one CTA they go straight to their places.  To
      // other CTAs such stores, of 16 bytes here and there, took 1 us longer than whole rows of 128 bytes; a warp turns its
      // block in the memory of the operands, which the last product has left.
      const bool direct = p.splits == 1;
      constexpr int kBlockRow = 36;  // floats; four banks apart
      static_assert(Cfg::kAcc == 32 && Cfg::kEpilogueWarps * 32 * kBlockRow * 4 <= Cfg::kOffScales, "");
      float* block = reinterpret_cast<float*>(smem) + warp * (32 * kBlockRow);
      const uint32_t mine = smem_addr(direct ? sums + row * Cfg::kSumRow + col0 : block + lane * kBlockRow);
#pragma unroll
      for (int j = 0; j < Cfg::kAcc; j += 4) {
        uint32_t x, y, z, w;
        unpack2u(acc[j / 2], x, y);
        unpack2u(acc[j / 2 + 1], z, w);
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(mine + j * 4), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
      }
      if (!direct) {
        __syncwarp();
        const uint32_t token = (warp & 3) * 32 + (lane >> 3);
        uint32_t owner = token / p.own, tok = token - owner * p.own;
#pragma unroll
        for (int r = 0; r < 32; r += 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(block + (r + (lane >> 3)) * kBlockRow + (lane & 7) * 4);
          const uint32_t at = smem_addr(sums + (part * p.own + tok) * Cfg::kSumRow + col0 + (lane & 7) * 4);
          st_cluster4(cluster_addr(at, owner), v);
          tok += 4;
          if (tok >= static_cast<uint32_t>(p.own)) {  // own >= 16
            tok -= p.own;
            ++owner;
          }
        }
      }
    } else {
      const uint32_t local = smem_addr(sums + part * p.own * 128 + row);
      uint32_t owner = col0 / p.own, tok = col0 - owner * p.own;
      uint32_t dst = p.splits > 1 ? cluster_addr(local, owner) : local;
#pragma unroll
      for (int j = 0; j < Cfg::kAcc; ++j) {
        uint32_t lo, hi;
        unpack2u(acc[j / 2], lo, hi);
        const uint32_t v = (j & 1) ? hi : lo;
        if (p.splits > 1) st_cluster(dst + tok * 512, v);
        else asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst + tok * 512), "r"(v) : "memory");
        if (++tok == static_cast<uint32_t>(p.own)) {
          tok = 0;
          if (++owner < static_cast<uint32_t>(p.splits)) dst = cluster_addr(local, owner);
        }
      }
    }
  }
  __syncwarp();
  if (p.splits > 1) {
    if (*abort_word)  // every CTA of the cluster lacks a part then
      for (int r = 0; r < p.splits; ++r) st_cluster(cluster_addr(smem_addr(tmem_slot + 1), r), 1);
    __syncwarp();
    cluster_sync();
  } else {
    __syncthreads();
  }
  if (warp < Cfg::kEpilogueWarps) {
    const int parts = Cfg::kTurns * p.splits;
    const bool lost = *abort_word;
    const float nan = __int_as_float(0x7FFFFFFF);
    if (p.wide_stores) {
      // a thread adds up eight neighbouring columns of one token
      const int c = (threadIdx.x & 15) * 8;
      const int left = p.n - n0 - c;
      for (int tok = threadIdx.x >> 4; tok < p.own; tok += Cfg::kEpilogueWarps * 2) {
        const int m = m0 + static_cast<int>(rank) * p.own + tok;
        if (m >= p.m || static_cast<int>(rank) * p.own + tok >= TOK) break;
        const float* from = sums + tok * Cfg::kSumRow + c;
        float sum[8];
        *reinterpret_cast<float4*>(sum) = *reinterpret_cast<const float4*>(from);
        *reinterpret_cast<float4*>(sum + 4) = *reinterpret_cast<const float4*>(from + 4);
        for (int q = 1; q < parts; ++q) {
          from += p.own * Cfg::kSumRow;
          float4 v[2] = {*reinterpret_cast<const float4*>(from), *reinterpret_cast<const float4*>(from + 4)};
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[j] += reinterpret_cast<const float*>(v)[j];
        }
        Tout* out = static_cast<Tout*>(p.out) + m * p.out_stride + n0 + c;
        Chunk<8 * (int)sizeof(Tout)> piece;
#pragma unroll
        for (int j = 0; j < 8; ++j) reinterpret_cast<Tout*>(piece.b)[j] = from_f32<Tout>(lost ? nan : sum[j]);
        if (left >= 8) {
          store_chunk(out, piece, false);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < left) out[j] = reinterpret_cast<const Tout*>(piece.b)[j];
        }
      }
    } else {
      // A warp a token at a time, a thread one word of each piece of 32.  As above, with eight single elements per thread,
      // 300 x 4001 x 1024 took 13.0 us instead of 8.1.
      constexpr int kPer = 4 / (int)sizeof(Tout);
      for (int tok = warp; tok < p.own; tok += Cfg::kEpilogueWarps) {
        const int m = m0 + static_cast<int>(rank) * p.own + tok;
        if (m >= p.m || static_cast<int>(rank) * p.own + tok >= TOK) break;
        Tout* out = static_cast<Tout*>(p.out) + m * p.out_stride + n0;
#pragma unroll
        for (int c = 0; c < 128; c += 32 * kPer) {
          const float* from = sums + tok * Cfg::kSumRow + c + lane * kPer;
          float x = from[0], y = kPer == 2 ? from[kPer - 1] : 0.0f;
          for (int q = 1; q < parts; ++q) {
            from += p.own * Cfg::kSumRow;
            x += from[0];
            if constexpr (kPer == 2) y += from[kPer - 1];
          }
          store_words<Tout, 32>(lost ? result_word<Tout>(nan, nan) : result_word<Tout>(x, y), lane, out + c, p.n - n0 - c);
        }
      }
    }
  }
  __syncwarp();
  fence_before_thread_sync();
  __syncthreads();
  fence_after_thread_sync();
  if (*abort_word) {  // final by now
    if (warp >= kLoadWarp) {
      for (int j = warp - kLoadWarp; j < asked; j += kTakeTurns)
        if (j + Cfg::kStages >= asked) mm_wait_limited(full + j % Cfg::kStages, (j / Cfg::kStages) & 1);
    } else if (warp >= kMmaWarp) {
      if (elect_one()) mma_commit(drained);
      mm_wait_limited(drained, 0);
    }
    __syncwarp();
    fence_before_thread_sync();
    __syncthreads();
    fence_after_thread_sync();
  }
  if (warp == kMmaWarp) tmem_dealloc(tmem, Cfg::kCols);
  if (threadIdx.x == 0 && *abort_word) atomicMax(&g_block_mm_status, 1);
}

// ---------------------------------------------------------------------------------------------
// many rows of a: rows of a are the M operand
// ---------------------------------------------------------------------------------------------
// Persistent pairs of CTAs (clusters of two) walk tiles of 256 rows of a x 256 rows of b with MMAs that span both: each
// CTA brings in and keeps 128 rows of either operand and receives 128 rows x 256 columns of products.
//   warps 0-7  epilogue: thread r of a warpgroup owns row r of the CTA's rows of a and 128 of the 256 columns
//   warps 8-9  of the even CTA issue the MMAs (M = 256, N = 256), taking the groups in turn
//   warp 10    issues the CTA's TMA loads; they count on the even CTA's barriers
//   warp 11    fetches scales: the products of a row's and a column block's scale go to a ring in shared memory
// Tensor memory holds two groups of products (2 x 256 columns): while the epilogue threads take one, the tensor pipe
// fills the other.  Tiles are walked in bands of kWideBand row tiles, so that the pairs at work at one time share both
// operands' tiles in L2.
struct WideCfg {
  static constexpr int kTile = 128 * 128;  // 128 rows of one group of an operand
  static constexpr int kStageBytes = 2 * kTile;
  static constexpr int kStages = 6;
  static constexpr int kScaleSlots = 4;
  static constexpr int kScaleGroups = 4;                          // groups of a slot
  static constexpr int kOffScales = kStages * kStageBytes;        // [slot][column half][row][group]
  static constexpr int kOffTurn = kOffScales + kScaleSlots * 256 * kScaleGroups * 4;
  static constexpr int kOffBar = kOffTurn + 8 * 32 * 17 * 4;      // a 32 x 16 block of results per epilogue warp
  static constexpr int kBars = 2 * kStages + 4 + 2 * kScaleSlots + 1;
  static constexpr int kSmem = kOffBar + kBars * 8 + 16 + 1024;
  static_assert(kSmem <= 232448 && 2 * (kSmem + 1024) > 233472, "one CTA per SM");
};
constexpr int kWideThreads = 384;
// 384 threads leave 168 registers per thread; the epilogue threads hold 128 accumulators and 64 products
// (2 x 128 x 216 + 128 x 72 = 64512)
constexpr int kWideEpilogueRegs = 216;
constexpr int kWideOtherRegs = 72;
constexpr int kWideBand = 8;

struct WideParams {
  const float* a_scales;
  const float* b_scales;
  void* out;
  int64_t out_stride, as_stride_m, as_stride_g, bs_stride_n, bs_stride_g;
  int32_t m, n, groups;
  int32_t m_tiles, n_tiles;
  int32_t store_bytes;  // 32 or 16: the rows of out allow stores of that size; 8: words
};

__device__ __forceinline__ void wide_tile(const WideParams& p, int tile, int& mt, int& nt) {
  const int band_tiles = kWideBand * p.n_tiles;
  const int band = tile / band_tiles, rest = tile - band * band_tiles;
  const int rows = min(kWideBand, p.m_tiles - band * kWideBand);
  nt = rest / rows;
  mt = band * kWideBand + (rest - nt * rows);
}

// a TMA load into this CTA's shared memory that counts on a barrier of either CTA of the pair (no multicast)
__device__ __forceinline__ void wide_tma_load(uint32_t dst, const CUtensorMap* map, uint32_t cluster_bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(cluster_bar), "r"(c0), "r"(c1)
      : "memory");
}

// By every thread of the CTA, from wherever its role ends.
__device__ __forceinline__ void wide_cta_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kWideThreads) : "memory"); }

template <int F8, typename Tout>
__global__ void __launch_bounds__(kWideThreads, 1)
    block_mm_wide_kernel(const __grid_constant__ BlockMmMaps maps, const __grid_constant__ WideParams p) {
  using namespace umma;
  using Cfg = WideCfg;
  extern __shared__ unsigned char raw[];
  unsigned char* smem = raw + ((1024u - (smem_addr(raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  uint64_t* full = bars;                           // the even CTA's: both CTAs' tiles are there
  uint64_t* empty = full + Cfg::kStages;
  uint64_t* ready = empty + Cfg::kStages;          // a group's products are in tensor memory
  uint64_t* taken = ready + 2;                     // the even CTA's: and have been read by both CTAs
  uint64_t* scaled = taken + 2;                    // a slot's scales are there
  uint64_t* used = scaled + Cfg::kScaleSlots;      // and have been read
  uint64_t* drained = used + Cfg::kScaleSlots;     // after a wait that gave up: no MMA of the pair is in flight
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::kBars);
  volatile uint32_t* abort_word = tmem_slot + 1;
  // words 2 and 3 behind it, of the even CTA: groups that its own and the odd CTA's loading warp have asked for
  float4* scales = reinterpret_cast<float4*>(smem + Cfg::kOffScales);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();

  if (threadIdx.x == 0) {
    prefetch_map(&maps.a);
    prefetch_map(&maps.b);
    for (int i = 0; i < Cfg::kStages; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(ready + i, 1);
      mbar_init(taken + i, 16);
    }
    for (int i = 0; i < Cfg::kScaleSlots; ++i) {
      mbar_init(scaled + i, 1);
      mbar_init(used + i, 8);
    }
    mbar_init(drained, 3);
    *abort_word = 0;
    mbar_init_fence();
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == 8) tmem_alloc_pair(tmem_slot, 512);
  fence_before_thread_sync();
  __syncthreads();
  cluster_sync();
  fence_after_thread_sync();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  const int tiles = p.m_tiles * p.n_tiles;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWideEpilogueRegs));
    const int half = warp >> 2, row = threadIdx.x & 127;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + half * 128;
    const uint32_t taken_addr = cluster_addr(smem_addr(taken), 0);
    Ring<2> buf;
    Ring<Cfg::kScaleSlots> at;
    const uint32_t scale_addr = smem_addr(scales + half * 128 + row);
    for (int tile = pair; tile < tiles; tile += pairs) {
      uint64_t acc[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = 0;
      for (int g = 0; g < p.groups; ++g) {
        const int k = g & (Cfg::kScaleGroups - 1);
        if (k == 0) mbar_wait_bounded(scaled + at.slot, at.parity, abort_word);
        uint32_t s;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(s) : "r"(scale_addr + at.slot * (256 * Cfg::kScaleGroups * 4) + k * 4));
        const uint64_t s2 = pack2(s, s);
        const uint32_t b = buf.slot;
        mbar_wait_bounded(ready + b, buf.parity, abort_word);
        buf.advance();
        fence_after_thread_sync();
        // 32 columns are on their way while the 32 before them are added
        uint32_t v[2][32];
        tmem_ld_32x32(lane_base + b * 256, v[0]);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 128; c += 32) {
          if (c + 32 < 128) {
            tmem_ld_32x32(lane_base + b * 256 + c + 32, v[(c / 32 + 1) & 1]);
          } else {
            fence_before_thread_sync();
            __syncwarp();
            if (lane == 0) {
              asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(taken_addr + b * 8) : "memory");
              if (k == Cfg::kScaleGroups - 1 || g + 1 == p.groups) mbar_arrive(used + at.slot);
            }
          }
#pragma unroll
          for (int j = 0; j < 16; ++j)
            acc[c / 2 + j] = fma_f32x2(pack2(v[(c / 32) & 1][2 * j], v[(c / 32) & 1][2 * j + 1]), s2, acc[c / 2 + j]);
          __syncwarp();  // keeps the additions of these columns before the wait for the next ones
          if (c + 32 < 128) tmem_ld_wait();
        }
        if (k == Cfg::kScaleGroups - 1 || g + 1 == p.groups) at.advance();
      }
      if (*abort_word) {  // set before a wait of this tile or an earlier one returned without its event
        const uint32_t nan = 0x7FFFFFFFu;
#pragma unroll
        for (int j = 0; j < 64; ++j) acc[j] = pack2(nan, nan);
      }
      int mt, nt;
      wide_tile(p, tile, mt, nt);
      const int m = mt * 256 + static_cast<int>(rank) * 128 + row, n0 = nt * 256 + half * 128;
      Tout* out = static_cast<Tout*>(p.out) + m * p.out_stride + n0;
      const int left = p.n - n0;
      constexpr int kPiece = 32 / (int)sizeof(Tout);  // elements of a 32-byte store
      if (p.store_bytes >= 16) {
        if (m < p.m && left > 0) {
#pragma unroll
          for (int c = 0; c < 128; c += kPiece) {
            Chunk<32> piece;
#pragma unroll
            for (int j = 0; j < kPiece / 2; ++j) {
              uint32_t lo, hi;
              unpack2u(acc[c / 2 + j], lo, hi);
              reinterpret_cast<Tout*>(piece.b)[2 * j] = from_f32<Tout>(__uint_as_float(lo));
              reinterpret_cast<Tout*>(piece.b)[2 * j + 1] = from_f32<Tout>(__uint_as_float(hi));
            }
            if (c + kPiece <= left) {
              store_chunk(out + c, piece, p.store_bytes == 32);
            } else {
#pragma unroll
              for (int j = 0; j < kPiece; ++j)
                if (c + j < left) out[c + j] = reinterpret_cast<const Tout*>(piece.b)[j];
            }
          }
        }
      } else {
        // Rows at odd addresses, as words (see store_words), which a thread's own row would spread over 32 rows per access.
        // Each warp turns blocks of 32 rows x 16 words through shared memory, so that 16 lanes write a row.  Rows two apart
        // begin at the same place in a word: what a lane does is settled once per block.  (7276 x 3669 x 256: 33.7 us; with
        // single elements 46.6, 17.6 with 3664 columns, whose rows allow 32-byte stores.)
        constexpr int kPer = 4 / (int)sizeof(Tout);
        constexpr int kWords = 128 / kPer;
        uint32_t words[kWords];
#pragma unroll
        for (int j = 0; j < 64; ++j) {
          uint32_t lo, hi;
          unpack2u(acc[j], lo, hi);
          if constexpr (kPer == 2) {
            words[j] = result_word<Tout>(__uint_as_float(lo), __uint_as_float(hi));
          } else {
            words[2 * j] = lo;
            words[2 * j + 1] = hi;
          }
        }
        uint32_t* block = reinterpret_cast<uint32_t*>(smem + Cfg::kOffTurn) + warp * (32 * 17);
        const int first_row = m - lane + (lane >> 4), w = lane & 15;
        const int rows = p.m - first_row;  // row r of the block, this lane's r even, exists if r < rows
        Tout* row0 = static_cast<Tout*>(p.out) + first_row * p.out_stride + n0;
        const int odd = kPer == 2 ? static_cast<int>(reinterpret_cast<uintptr_t>(row0) >> 1) & 1 : 0;
        const int e = kPer * w - odd;
#pragma unroll
        for (int c = 0; c < kWords; c += 16) {
          const int rest = left - c * kPer;
          const bool whole = e >= 0 && e + kPer <= rest;
          const bool first = e < 0 && rest > 0, last = odd && w == 15 && rest >= 32, end = kPer == 2 && e >= 0 && e + 1 == rest;
          const bool single = first || last || end;
          const uint32_t pick = odd ? 0x5432u : 0x7654u;
          const uint32_t pick_single = last ? 0x7676u : end && odd ? 0x3232u : 0x5454u;
          Tout* to = row0 + c * kPer + e;
          const int single_at = first ? 1 : last ? 31 - e : 0;  // from `to`
#pragma unroll
          for (int j = 0; j < 16; ++j) block[lane * 17 + j] = words[c + j];
          __syncwarp();
          const uint32_t* from = block + (lane >> 4) * 17 + w;
#pragma unroll 4
          for (int r = 0; r < 32; r += 2) {
            const uint32_t v = from[r * 17];
            if constexpr (kPer == 2) {
              const uint32_t before = __shfl_up_sync(0xFFFFFFFFu, v, 1, 16);
              st_if(whole && r < rows, to, __byte_perm(before, v, pick));
              st_half_if(single && r < rows, to + single_at, __byte_perm(before, v, pick_single));
            } else {
              st_if(whole && r < rows, to, v);
            }
            to += 2 * p.out_stride;
          }
          __syncwarp();
        }
      }
    }
    // This role ends here, not where the others meet: any code behind a meeting point of all of them cost its loop time
    // (zero operands: 994 us this way, otherwise 1006 to 1042 with what stands below).
    __syncwarp();
    fence_before_thread_sync();
    wide_cta_sync();
    cluster_sync();
    return;
  }
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWideOtherRegs));
  if (warp == 10) {
    Ring<Cfg::kStages> at;
    bool ok = true;
    uint32_t asked = 0;
    for (int tile = pair; ok && tile < tiles; tile += pairs) {
      int mt, nt;
      wide_tile(p, tile, mt, nt);
      const int m0 = mt * 256 + rank * 128, n0 = nt * 256 + rank * 128;
      for (int g = 0; g < p.groups; ++g, ++asked, at.advance()) {
        ok = mm_wait(empty + at.slot, at.parity ^ 1, abort_word);
        if (!ok) break;
        if (elect_one()) {
          if (rank == 0) mm_expect_tx(full + at.slot, 2 * Cfg::kStageBytes);
          const uint32_t bar = cluster_addr(smem_addr(full + at.slot), 0);
          const uint32_t dst = smem_addr(smem + at.slot * Cfg::kStageBytes);
          wide_tma_load(dst, &maps.a, bar, g * 128, m0);
          wide_tma_load(dst + Cfg::kTile, &maps.b, bar, g * 128, n0);
        }
        __syncwarp();
      }
    }
    if (lane == 0) st_cluster(cluster_addr(smem_addr(tmem_slot + 2 + rank), 0), asked);
  } else if (warp == 11) {
    Ring<Cfg::kScaleSlots> at;
    bool ok = true;
    for (int tile = pair; ok && tile < tiles; tile += pairs) {
      int mt, nt;
      wide_tile(p, tile, mt, nt);
      // rows and column blocks past the end repeat the last one: their products are not stored
      const int last = (p.n - 1) / 128;
      const float* sb0 = p.b_scales + min(nt * 2, last) * p.bs_stride_n;
      const float* sb1 = p.b_scales + min(nt * 2 + 1, last) * p.bs_stride_n;
      for (int g = 0; g < p.groups; g += Cfg::kScaleGroups, at.advance()) {
        ok = mm_wait(used + at.slot, at.parity ^ 1, abort_word);
        if (!ok) break;
        const int m = mt * 256 + static_cast<int>(rank) * 128 + lane;
        float vb[2][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          vb[0][k] = g + k < p.groups ? ld_ahead(sb0 + (g + k) * p.bs_stride_g) : 0.0f;
          vb[1][k] = g + k < p.groups ? ld_ahead(sb1 + (g + k) * p.bs_stride_g) : 0.0f;
        }
#pragma unroll 1
        for (int r = 0; r < 4; r += 2) {  // two rows a lane at a time
          float va[2][4];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float* sa = p.a_scales + min(m + (r + i) * 32, p.m - 1) * p.as_stride_m + g * p.as_stride_g;
#pragma unroll
            for (int k = 0; k < 4; ++k) va[i][k] = g + k < p.groups ? ld_ahead(sa + k * p.as_stride_g) : 0.0f;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              scales[at.slot * 256 + h * 128 + (r + i) * 32 + lane] =
                  make_float4(__fmul_rn(va[i][0], vb[h][0]), __fmul_rn(va[i][1], vb[h][1]),
                              __fmul_rn(va[i][2], vb[h][2]), __fmul_rn(va[i][3], vb[h][3]));
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(scaled + at.slot);
      }
    }
  } else if (rank == 0) {
    constexpr uint32_t idesc = instr_desc_f8(256, 256, F8 == KVC_KV_FP8_E5M2);
    const int me = warp - 8;
    Ring<Cfg::kStages, 2> at(me);
    uint32_t parity = 0;  // of buffer `me`, the only one this warp uses
    const int mine = pair < tiles ? (tiles - 1 - pair) / pairs + 1 : 0;  // tiles of this pair
    const int64_t steps = static_cast<int64_t>(mine) * p.groups;
    for (int64_t it = me; it < steps; it += 2, at.advance(), parity ^= 1) {
      if (!mm_wait(taken + me, parity ^ 1, full + at.slot, at.parity, abort_word)) break;
      fence_after_thread_sync();
      if (elect_one()) {
        const uint32_t base = smem_addr(smem + at.slot * Cfg::kStageBytes);
        const uint64_t da = smem_desc_sw128(base, 0, 1024), db = smem_desc_sw128(base + Cfg::kTile, 0, 1024);
#pragma unroll
        for (int k = 0; k < 4; ++k) mma_f8_ss_pair(tmem + me * 256, da + 2 * k, db + 2 * k, idesc, k > 0);
        mma_commit_pair(empty + at.slot);
        mma_commit_pair(ready + me);
      }
      __syncwarp();
    }
  }
  __syncwarp();
  fence_before_thread_sync();
  wide_cta_sync();
  if (warp == 8) {  // no warp of this CTA can give up any more; the CTAs of a pair do so together
    if (*abort_word) st_cluster(cluster_addr(smem_addr(tmem_slot + 1), rank ^ 1), 1);
    __syncwarp();
  }
  cluster_sync();  // the even CTA's MMAs read the odd one's shared memory, and barriers are signalled across
  fence_after_thread_sync();
  if (*abort_word) {  // the same in both
    if (rank == 0 && warp == 10) {  // both CTAs' copies count on the even one's barriers
      const volatile uint32_t* asked = tmem_slot + 2;
      const uint32_t end = max(asked[0], asked[1]);
      for (uint32_t i = end > Cfg::kStages ? end - Cfg::kStages : 0; i < end; ++i)
        mm_wait_limited(full + i % Cfg::kStages, (i / Cfg::kStages) & 1);
      __syncwarp();
      if (lane < 2)
        asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr(smem_addr(drained), lane)) : "memory");
    } else if (rank == 0 && warp < 10) {
      if (elect_one()) mma_commit_pair(drained);
    }
    __syncwarp();
    mm_wait_limited(drained, 0, Cfg::kStages + 2);  // neither CTA ends, or gives memory back, before; longer than the waits above
    fence_after_thread_sync();
  }
  __syncwarp();
  if (warp == 8) tmem_dealloc_pair(tmem, 512);
  if (warp == 11 && lane == 0 && *abort_word) atomicMax(&g_block_mm_status, 1);
}

// Self-test of what a CTA does when a wait gives up: one warp waits, with a limit of `tries` tries (about 20 us each), for an
// arrival that nothing makes; the CTA then drains, frees its tensor memory and raises the status word as the kernels above do.
__global__ void __launch_bounds__(128) block_mm_gives_up_kernel(uint32_t tries) {
  using namespace umma;
  __shared__ __align__(8) uint64_t bar, drained;
  __shared__ uint32_t tmem_slot, abort_slot;
  volatile uint32_t* abort_word = &abort_slot;
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    mbar_init(&drained, 1);
    *abort_word = 0;
    mbar_init_fence();
  }
  __syncwarp();
  if (warp == 0) tmem_alloc(&tmem_slot, 32);
  fence_before_thread_sync();
  __syncthreads();
  fence_after_thread_sync();
  const uint32_t tmem = tmem_slot;
  if (warp == 1) mm_wait(&bar, 0, abort_word, tries);
  fence_before_thread_sync();
  __syncthreads();
  fence_after_thread_sync();
  if (*abort_word) {
    if (warp == 2) {
      if (elect_one()) mma_commit(&drained);
      mm_wait_limited(&drained, 0);
    }
    __syncwarp();
    fence_before_thread_sync();
    __syncthreads();
    fence_after_thread_sync();
  }
  if (warp == 0) tmem_dealloc(tmem, 32);
  if (threadIdx.x == 0 && *abort_word) atomicMax(&g_block_mm_status, 1);
}

}  // namespace
}  // namespace kvc
