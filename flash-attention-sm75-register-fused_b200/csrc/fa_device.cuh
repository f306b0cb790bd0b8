// Device helpers of the attention kernels' translation units: the status word and the
// bounded mbarrier waits that set it, launch shape and register split, shared and tensor
// memory layout, and the exponentials of a tile.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "fa_fwd.h"
#include "sm100_ptx.cuh"
#include "fa_softmax.cuh"

namespace fa {

// Sticky device status: high 32 bits = launch epoch, low 32 bits = error code.
// Written only when a bounded wait expires; read by fa_device_status().  (One per
// translation unit.)
static __device__ unsigned long long g_fa_status = 0ull;

// Work-item counters of persistent launches whose last rounds are dealt
// dynamically: slot sched % kSchedSlots holds (sched << 32) | items handed
// out.  A launch starts its slot by replacing a value tagged with another
// launch's number, so no reset is needed between launches; 256 slots keep
// launches whose CTAs run at the same time apart (the host numbers these
// launches on their own counter).
constexpr unsigned kSchedSlots = 256;
static __device__ unsigned long long g_fa_sched[kSchedSlots];

namespace {

constexpr int kBlockM = 128;  // query rows per tile (one TMEM lane each)
constexpr int kBlockN = 128;  // keys per K/V tile
constexpr int kThreads = 384;   // 3 warpgroups
// Warpgroup of the producer, the MMA issuer and two spare warps (8-11); the
// two softmax warpgroups are warps 0-7.
constexpr int kWarpLoad = 8;
constexpr int kWarpMma = 9;
constexpr int kWarpSoftmax0 = 0;
// Register split: launched at kLaunchRegs per thread (65536 / 384 rounded down
// to a multiple of 8); the producer/MMA warpgroup gives registers to the two
// softmax warpgroups.  256*kRegsSoftmax + 128*kRegsOther must not exceed
// 384*kLaunchRegs.
constexpr int kLaunchRegs = 168;
constexpr int kRegsSoftmax = 192;
constexpr int kRegsOther = 120;
static_assert(256 * kRegsSoftmax + 128 * kRegsOther <= kThreads * kLaunchRegs,
              "register split exceeds the launch allocation");
// Lazy rescaling: O and l keep a stale row max until the true max exceeds it
// by more than 2^15 (log2 units), so P = exp2(s - m_stale) <= 2^15 still fits
// f16 (max 65504) and bf16; results are identical up to rounding.
constexpr float kRescaleThreshold = 15.0f;

template <int D>
struct Layout {
  static constexpr int kColBlocks = D / 64;       // 128-byte swizzle column blocks
  static constexpr int kBlockBytes = kBlockM * 128;  // one 64-column block of a 128-row tile
  static constexpr int kTile = kBlockM * D * 2;   // bytes of a 128-row f16 tile
  // K and V tiles stream through one ring of tile-sized slots in load order
  // K0 V0 K1 V1 ...; a slot is refilled once the MMAs reading it completed.
  static constexpr int kSlots = (D == 128) ? 5 : 8;
  // shared memory (offsets from a 1024-aligned base)
  static constexpr int kOffQ = 0;                 // Q0, Q1
  static constexpr int kOffKV = 2 * kTile;        // ring slot s at kOffKV + s*kTile
  static constexpr int kOffBar = kOffKV + kSlots * kTile;
  // barrier indices
  static constexpr int kBarQ = 0;                       // 2
  static constexpr int kBarFull = 2;                    // kSlots (TMA tx-count)
  static constexpr int kBarEmpty = kBarFull + kSlots;   // kSlots (MMA commit)
  static constexpr int kBarS = kBarEmpty + kSlots;      // 2
  static constexpr int kBarP = kBarS + 2;               // 2
  static constexpr int kBarO = kBarP + 2;               // 2
  static constexpr int kBarDrain = kBarO + 2;           // 1
  // persistent launches (several work items per CTA): the MMAs that read Q
  // buffer b for one item have completed, so the next Q may overwrite it
  static constexpr int kBarQFree = kBarDrain + 1;       // 2
  // early part of P_g written (kPEarlyQuarters x 32 keys): the PV MMA starts
  // on it while the softmax computes the rest (128 arrivals)
  static constexpr int kBarPH = kBarQFree + 2;          // 2
  // dynamically dealt rounds: the producer publishes each round's work item
  // in a 4-entry queue (full: producer arrival; empty: every softmax thread
  // and lane 0 of the MMA warp have read it)
  static constexpr int kItemQ = 4;
  static constexpr int kBarItemFull = kBarPH + 2;               // kItemQ
  static constexpr int kBarItemEmpty = kBarItemFull + kItemQ;   // kItemQ
  static constexpr int kNumBars = kBarItemEmpty + kItemQ;
  static constexpr int kOffMisc = kOffBar + 8 * kNumBars;
  static constexpr int kOffItemQ = kOffMisc + 16;               // kItemQ ints
  // dual-tile items (d = 64): each softmax thread's (m, l) for the in-CTA
  // merge of the two groups' key halves, double-buffered by work item
  static constexpr int kOffXchg = kOffItemQ + 4 * kItemQ;
  static constexpr int kXchgBytes = (D == 64) ? 2 * 2 * kBlockM * 8 : 0;
  static constexpr int kBytes = kOffXchg + kXchgBytes;
  static constexpr int kDynBytes = kBytes + 1024;  // slack for 1024-byte alignment
  // tensor memory columns
  static constexpr uint32_t kTmemCols = 512;
  __host__ __device__ static constexpr uint32_t tS(int g) { return g ? 128u : 0u; }
  __host__ __device__ static constexpr uint32_t tO(int g) { return g ? 256u + D : 256u; }
  // d=128 fills TMEM, so P overwrites the S columns it was computed from;
  // d=64 leaves room for separate P columns.
  static constexpr bool kAliasP = (D == 128);
  __host__ __device__ static constexpr uint32_t tP(int g) {
    return kAliasP ? tS(g) : (g ? 448u : 384u);
  }
  static_assert(kDynBytes <= 227 * 1024, "shared memory budget");
};

constexpr uint32_t kSuspendNs = 100000;  // upper bound of one hardware-suspended wait

struct WaitCtl {
  volatile int* abort;        // CTA-wide abort flag in shared memory
  unsigned long long timeout_ns;
  unsigned epoch;
};

__device__ void record_error(unsigned epoch, int code) {
  const unsigned long long want =
      (static_cast<unsigned long long>(epoch) << 32) | static_cast<unsigned>(code);
  unsigned long long old = atomicAdd(&g_fa_status, 0ull);
  while (true) {
    if ((old >> 32) == epoch && (old & 0xffffffffull) != 0ull) return;  // first error wins
    const unsigned long long prev = atomicCAS(&g_fa_status, old, want);
    if (prev == old) return;
    old = prev;
  }
}

// Next work-item number of launch `sched` from its counter slot (0, 1, 2, ...
// in the order of the calls across the launch's CTAs), or -1 (error recorded,
// CTA aborting) if the counter could not be updated after many attempts.
__device__ int sched_take(unsigned sched, const WaitCtl& c) {
  unsigned long long* ctr = &g_fa_sched[sched % kSchedSlots];
  unsigned long long v = atomicAdd(ctr, 0ull);
  for (int i = 0; i < (1 << 20); ++i) {
    const bool mine = static_cast<unsigned>(v >> 32) == sched;
    const unsigned long long nv =
        mine ? v + 1ull : ((static_cast<unsigned long long>(sched) << 32) | 1ull);
    const unsigned long long prev = atomicCAS(ctr, v, nv);
    if (prev == v) return mine ? static_cast<int>(v & 0xffffffffull) : 0;
    v = prev;
  }
  *c.abort = 1;
  record_error(c.epoch, FA_ERR_TIMEOUT_BASE + 6);
  return -1;
}

__device__ __forceinline__ bool bar_wait_slow(uint32_t bar, uint32_t parity, const WaitCtl& c,
                                           int site, bool respect_abort) {
  const uint64_t t0 = ptx::global_timer_ns();
  while (true) {
    // sleeps in hardware until the phase completes or ~kSuspendNs elapse
    if (ptx::mbar_try_wait_sleep(bar, parity, kSuspendNs)) return true;
    if (respect_abort && *c.abort) return false;
    if (ptx::global_timer_ns() - t0 > c.timeout_ns) {
      *c.abort = 1;
      record_error(c.epoch, FA_ERR_TIMEOUT_BASE + site);
      return false;
    }
  }
}

// Bounded mbarrier wait.  Returns false if the CTA is aborting or the wait
// exceeded the watchdog deadline (which also records the error and aborts).
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, const WaitCtl& c, int site,
                                         bool respect_abort = true) {
  if (ptx::mbar_try_wait(bar, parity)) return true;
  return bar_wait_slow(bar, parity, c, site, respect_abort);
}

// The slow path as a call, for warps with registers to spare: their code
// stays compact around every wait.
__device__ __noinline__ bool bar_wait_slow_call(uint32_t bar, uint32_t parity, const WaitCtl& c,
                                                int site, bool respect_abort) {
  return bar_wait_slow(bar, parity, c, site, respect_abort);
}
__device__ __forceinline__ bool bar_wait_lean(uint32_t bar, uint32_t parity, const WaitCtl& c,
                                              int site, bool respect_abort = true) {
  if (ptx::mbar_try_wait(bar, parity)) return true;
  return bar_wait_slow_call(bar, parity, c, site, respect_abort);
}

// Bounded wait that polls without suspending the thread: for short waits on
// the critical path, where a suspended thread may resume late.  The timer is
// read every 256 polls.
__device__ __noinline__ bool bar_wait_spin_slow(uint32_t bar, uint32_t parity, const WaitCtl& c,
                                                int site) {
  const uint64_t t0 = ptx::global_timer_ns();
  for (uint32_t i = 1;; ++i) {
    if (ptx::mbar_test_wait(bar, parity)) return true;
    if ((i & 255u) == 0u) {
      if (*c.abort) return false;
      if (ptx::global_timer_ns() - t0 > c.timeout_ns) {
        *c.abort = 1;
        record_error(c.epoch, FA_ERR_TIMEOUT_BASE + site);
        return false;
      }
    }
  }
}

__device__ __forceinline__ bool bar_wait_spin(uint32_t bar, uint32_t parity, const WaitCtl& c,
                                              int site) {
  if (ptx::mbar_test_wait(bar, parity)) return true;
  return bar_wait_spin_slow(bar, parity, c, site);
}

// Make the values produced by tcgen05.ld visible to ordinary instructions
// only after tcgen05.wait::ld (the empty volatile asm cannot move above it).
template <int N>
__device__ __forceinline__ void pin_after_wait(uint32_t* r) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
}

// Timeline tracing for development builds (-DFA_TRACE): the first
// kTraceCtas CTAs record clock64() at fixed points of every K/V tile into
// p.trace[cta][tile][event].  Compiled out otherwise.  Events of tile j:
//   0-3   MMA warp starts issuing PV0(j), S0(j+1), PV1(j), S1(j+1)
//   4, 5  MMA warp has issued PV0(j), S0(j+1)
//   6, 7  MMA warp before / after the V_j and K_{j+1} waits
//   8-15  softmax warp w arrived on P (w = 0..7)
//   16-23 softmax warp w saw S complete
//   24-27 observer warps (d=128): S0(j), PV0(j), S1(j), PV1(j) complete
//   28-29 group 0 / 1 tile max computed (row 0)
//   30-31 producer issued the loads of V_j / K_{j+1}
//   (tile kTraceTiles-1, events 30 / 31: CTA set up / CTA done)
// Dual (decode) launches index rows by each group's running tile count
// (mod 64) and record: 2g MMA warp saw V_j, K_{j+1} of group g land; 4+g
// P_g(j) seen and PV issued; 1+2g S_g(j+1) issued; 24+g / 26+g producer
// issued K / V of the tile; 8-23, 28-29 as above.
constexpr int kTraceCtas = 8, kTraceTiles = 64, kTraceEvents = 32;
#ifdef FA_TRACE
#define FA_TRACE_AT(tile, ev)                                                          \
  do {                                                                                 \
    if (p.trace != nullptr && blockIdx.x < kTraceCtas && (tile) < kTraceTiles)         \
      p.trace[(blockIdx.x * kTraceTiles + (tile)) * kTraceEvents + (ev)] = clock64(); \
  } while (0)
#else
#define FA_TRACE_AT(tile, ev) \
  do {                        \
  } while (0)
#endif

// The first kPEarlyQuarters quarters of P (32 keys each) are announced to the
// MMA warp before the rest is computed, so the PV steps on them overlap the
// softmax's tail.
#ifndef FA_P_EARLY_QUARTERS
#define FA_P_EARLY_QUARTERS 2
#endif
constexpr int kPEarlyQuarters = FA_P_EARLY_QUARTERS;
static_assert(kPEarlyQuarters >= 1 && kPEarlyQuarters <= 3, "early part of P: 1-3 quarters");

// exp2(x * sl - m) for the 128 scores of this thread's row; the packed
// f16/bf16 values go to TMEM (P operand of the PV MMA) in four 16-column
// quarters, the first kPEarlyQuarters announced (`announce()`, an mbarrier
// arrival) as soon as they are written; returns their fp32 sum.
template <bool BF16, bool kEmulate, int kPeriod = kEmuPeriod, typename Announce>
__device__ __forceinline__ float exp_tile(const float (&x)[kBlockN], float sl, float neg_m,
                                          uint32_t tP, Announce announce) {
  float a0 = 0.f, a1 = 0.f, b0 = 0.f, b1 = 0.f;
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    uint32_t pk[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      const int i = 32 * h + 2 * c;
      float e0, e1;
      exp2_pair<kEmulate, kPeriod>(c, x[i], x[i + 1], sl, neg_m, e0, e1);
      if (c & 1)
        ptx::fadd2(b0, b1, b0, b1, e0, e1);
      else
        ptx::fadd2(a0, a1, a0, a1, e0, e1);
      pk[c] = pack2<BF16>(e0, e1);
    }
    ptx::tmem_st16(tP + 16 * h, pk);
    if (h == kPEarlyQuarters - 1) {
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      announce();
    }
  }
  ptx::fadd2(a0, a1, a0, a1, b0, b1);
  return a0 + a1;
}

// Period of the pair kernel's exponential emulation pattern (one pair in
// kPairEmuPeriod on the polynomial): 1 in 8 at d = 128, 1 in 4 at d = 64.
// Measured on B200, interleaved runs: 1 in 8 against 1 in 4 gave C5 +2.5 %,
// C4 +0.6 %, C3 (d = 64) -1.7 %; 3 in 8 and 1 in 2 were slower everywhere
// (C5 -2 % / -11 %, C3 -7 % / -16 %): every polynomial adds softmax
// instructions that compete with the MMA warp for issue slots.
#ifndef FA_EMU_PERIOD_D128
#define FA_EMU_PERIOD_D128 8
#endif
template <int D>
constexpr int kPairEmuPeriod = (D == 128) ? FA_EMU_PERIOD_D128 : kEmuPeriod;

// Reads (and clears) this translation unit's status word.
inline cudaError_t read_status_word(unsigned long long* out, bool reset) {
  cudaError_t e = cudaMemcpyFromSymbol(out, g_fa_status, sizeof(*out));
  if (e != cudaSuccess) return e;
  if (reset) {
    const unsigned long long zero = 0ull;
    e = cudaMemcpyToSymbol(g_fa_status, &zero, sizeof(zero));
  }
  return e;
}

}  // namespace
}  // namespace fa
