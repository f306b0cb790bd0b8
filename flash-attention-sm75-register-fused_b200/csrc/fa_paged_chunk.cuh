// Attention of chunks of new tokens over a paged KV cache (more query rows per
// (sequence, KV head) than the decode kernel takes).  Included by
// fa_fwd_sm100.cu, whose helpers (bounded mbarrier waits, the device status
// word, exp_tile, the register split) it uses.
//
// The pair kernel's arrangement (fa_fwd_kernel): two 128-row query tiles per
// CTA ping-pong on one tcgen05 issuer, S and P in tensor memory, lazy rescale.
// What is different:
//
//   rows   A tile holds 128 / G tokens x the G query heads of a KV head (row =
//          token * G + head), for every length: K and V are read once per
//          group, and short chunks fill their tiles.  G need not divide 128
//          (G = 7: 18 tokens, 126 rows).
//   items  (sequence, KV head, pair of tiles), found from the lengths on the device
//          in one of two ways (chosen on the host by an estimate of both).  One CTA
//          per item: the grid has room for every pair the packed rows can hold,
//          a CTA without one leaves at once, and pairs of a sequence run from its
//          end, the longest causal rows first.  Or equal runs: the key tiles of
//          all items in a row are cut into one run per SM, whatever the lengths
//          (SeqWork gives positions in closed form), one warp hands the
//          run's segments to the others through a ring, K and V of the next segment
//          load while the last one ends, and cut items are joined.  Items / runs,
//          d = 128, GQA 4, 8 KV heads: 512 tokens over 8192 keys 116 / 70 us (two
//          splits of each item, 128 CTAs: 76), over 1024 keys 23.5 / 25.3; 2 x 2048
//          over 8192 460 / 433; 200 over 200 14.3 / 22.1; 8 x 1024 over 1024 124 /
//          115; 8 x 2048 over 8192 (keys twice the L2) 1780 / 2000.
//   pages  16-bit pages: a 128-key tile is a set of TMA boxes of gcd(page, 128)
//          rows, one per lane of a producer warp (one warp for K, one for V).  A
//          box brings whole rows: the maps split d into halves of 128 bytes, laid
//          out per 8 rows (8 rows x 128 bytes of one half, then of the other),
//          which the products' descriptors take like any swizzled tile.  At B=2,
//          2048 over 8192 keys, d = 128, pages of 16: a box per half from one warp
//          551 us, whole rows 448, two warps 411 (1171 TFLOPS, as with pages of
//          128).  The rows behind the last visible key in its box are stale; V's
//          are set to zero before the tile is released, K's are masked as scores.
//          8-bit pages: paged_expand_kernel first writes the visible keys and
//          values once as 16-bit rows into the workspace (exactly, K in the
//          queries' type, V in f16, the scales beside them), so that the pairs of
//          a chunk do not widen the same keys again and again, and the kernel
//          reads plain 128-row tiles.  The softmax applies the scales in fp32:
//          K's to the scores, V's to P.
//   P      over 8-bit pages is 2^(s_ij - r_i) vs_j with a reference r_i that follows
//          the largest s_ij + log2 vs_j instead of the largest score: f16 then holds
//          the value rows that make up a result, however large or small they and
//          others are.  The row sum of exponentials is kept relative to the largest
//          score, m_i.  A bound, the tile's largest score and largest scale, says
//          where r may have to grow; only then is the maximum taken key by key.
//   joins  The parts of a cut item go to the workspace as fp32 (four columns of all
//          rows side by side, so that stores and the join's loads are whole
//          lines: 77 -> 70 us for 512 tokens over 8192 keys), and paged_join_kernel
//          merges them by a table that the runs leave.
//
// Bound by the tensor cores and what feeds them: with all SMs at work a pair's key
// tile takes 1.8 us (1.5 at the rate of a large library product), so 2 x 2048
// tokens over 8192 keys run at 1230 TFLOPS; then by the start of the work: a
// call with one item per SM costs 11 us beyond its tiles, one of equal runs 21.
#include "fa_paged.h"
#include "fa_paged_dev.cuh"

namespace fa {
namespace {

// What the kernel reads: pages, or the expanded rows of 8-bit pages.
enum { kPagesF16 = 0, kPagesBf16 = 1, kExpanded = 2 };

// A part of a work item that a CTA computes.
struct Segment {
  int b, h;              // sequence (-1: the run ends), KV head
  int c0, nq, nk, off, vis;  // of the sequence (Seq)
  int tok0;              // first token of query tile 0
  int jb, n0, n1;        // first key tile; key tiles of either query tile
  int slot;              // of the workspace, -1: the segment is the whole item
  int exp_row0;          // sequence's first row in the expanded rows
  int tiles, parity;     // key tiles before it; bit g: those of query tile g, mod 2
  int pad;
};
constexpr int kSegRing = 4;

template <int D, bool kScaled>
struct ChunkLayout {
  // register split; the scales' multiplications take 16 more in the softmax
  static constexpr int kRegsSoft = kScaled ? 208 : kRegsSoftmax;
  static constexpr int kRegsRest = kScaled ? 88 : kRegsOther;
  static_assert(256 * kRegsSoft + 128 * kRegsRest <= kThreads * kLaunchRegs,
                "register split exceeds the launch allocation");
  static constexpr int kColBlocks = D / 64;
  static constexpr int kBlockBytes = 128 * 128;           // Q: 64 columns of a tile
  static constexpr int kGroupBytes = 1024 * kColBlocks;   // K, V: 8 rows of a tile
  static constexpr int kTile = 128 * D * 2;
  static constexpr int kSlots = D == 64 ? 8 : (kScaled ? 4 : 5);
  static constexpr int kOffQ = 0;
  static constexpr int kOffKV = 2 * kTile;
  static constexpr int kOffScale = kOffKV + kSlots * kTile;
  // scales of tile j at entry j % kScaleRing: K's 128, V's 128, the 128 logarithms
  // of V's and 8 maxima of those, loaded with K_j.  K_j's slot is free only after
  // the scores of tile j - kSlots / 2 were issued for both groups, i.e. after both
  // finished the softmax of the tile before it, so entry j - kScaleRing is no
  // longer read.
  static constexpr int kScaleRing = D == 64 ? 8 : 4;
  static constexpr int kScaleEntry = (3 * 128 + 8) * 4;
  static_assert(kScaleRing >= kSlots / 2 + 1, "a scale entry outlives its tile");
  static constexpr int kOffBar = kOffScale + (kScaled ? kScaleRing * kScaleEntry : 0);
  static constexpr int kBarQ = 0;                       // 2
  static constexpr int kBarFull = 2;                    // kSlots
  static constexpr int kBarEmpty = kBarFull + kSlots;   // kSlots
  static constexpr int kBarS = kBarEmpty + kSlots;      // 2
  static constexpr int kBarP = kBarS + 2;               // 2
  static constexpr int kBarPH = kBarP + 2;              // 2
  static constexpr int kBarO = kBarPH + 2;              // 2
  static constexpr int kBarDrain = kBarO + 2;           // 1
  static constexpr int kBarTail = kBarDrain + 1;        // 1: the V tile with stale rows landed
  static constexpr int kBarQFree = kBarTail + 1;        // 2: Q read by its last scores
  static constexpr int kBarSegFull = kBarQFree + 2;     // kSegRing
  static constexpr int kBarSegEmpty = kBarSegFull + kSegRing;  // kSegRing
  static constexpr int kNumBars = kBarSegEmpty + kSegRing;
  static constexpr int kOffSeg = kOffBar + (8 * kNumBars + 15) / 16 * 16;
  static constexpr int kOffMisc = kOffSeg + kSegRing * static_cast<int>(sizeof(Segment));
  static constexpr int kBytes = kOffMisc + 16;
  static constexpr int kDynBytes = kBytes + 1024;
  static constexpr uint32_t kTmemCols = 512;
  __host__ __device__ static constexpr uint32_t tS(int g) { return g ? 128u : 0u; }
  __host__ __device__ static constexpr uint32_t tO(int g) { return g ? 256u + D : 256u; }
  __host__ __device__ static constexpr uint32_t tP(int g) {
    return D == 128 ? tS(g) : (g ? 448u : 384u);
  }
  static_assert(kDynBytes <= 227 * 1024, "shared memory budget");
};

// Four scales from shared memory; volatile, so that the loads stay where they
// are used (hoisted over the 128 scores of a row they spill).
__device__ __forceinline__ float4 load_scales(uint32_t addr) {
  float4 f;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w)
               : "r"(addr));
  return f;
}

// exp_tile (fa_fwd_sm100.cu) with P multiplied by V's scales: e = 2^(x sl - ref)
// is summed as it is, e * vs goes to tensor memory.
template <bool kEmulate, int kPeriod, typename Announce>
__device__ __forceinline__ float exp_tile_scaled(const float (&x)[kBlockN], float sl, float neg_ref,
                                                 uint32_t vs, uint32_t tP, Announce announce) {
  float a0 = 0.f, a1 = 0.f, b0 = 0.f, b1 = 0.f;
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    uint32_t pk[16];
#pragma unroll
    for (int c = 0; c < 16; c += 2) {
      const float4 f = load_scales(vs + 4 * (32 * h + 2 * c));
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int i = 32 * h + 2 * (c + y);
        float e0, e1;
        exp2_pair<kEmulate, kPeriod>(c + y, x[i], x[i + 1], sl, neg_ref, e0, e1);
        if (y)
          ptx::fadd2(b0, b1, b0, b1, e0, e1);
        else
          ptx::fadd2(a0, a1, a0, a1, e0, e1);
        ptx::fmul2(e0, e1, e0, e1, y ? f.z : f.x, y ? f.w : f.y);
        pk[c + y] = pack2<false>(e0, e1);
      }
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

// 128-row blocks of a sequence in the expanded rows.
__device__ __forceinline__ int expand_blocks(const Seq& s) { return (s.vis + kBlockN - 1) / kBlockN; }

// The pairs of query tiles of a sequence, and what they cost.  Pair i (of one
// head) sees keys [0, lim(i)), lim(i) = clamp(off + (i + 1) c, 0, vis) for c tokens
// a pair; it takes kItemCost + lim(i) positions of the work order, the key tile
// that starts at key k the one at kItemCost + k.
// (kItemCost: six ragged chunks over e4m3 pages take 271 us with 256, 260 with 384,
// 262 with 512, 273 with 1024.  kMinRun, the shortest run: 64 tokens over 8192 keys take 37.9
// us with 128, 35.5 with 512; 512 over 1024 26.9 with 128, 27.3 with 512, 31.8 with 1024)
constexpr int kItemCost = 384;
constexpr int kMinRun = 512;
struct SeqWork {
  long long off;
  int c, vis, n;  // n pairs
  int z, s;       // pairs [0, z) see no key, pairs [s, n) all of them
  __device__ __forceinline__ int lim(int i) const {
    return static_cast<int>(min(max(off + static_cast<long long>(i + 1) * c, 0ll), static_cast<long long>(vis)));
  }
  __device__ __forceinline__ int tiles(int i) const { return (lim(i) + kBlockN - 1) / kBlockN; }
  // positions of pairs [0, i)
  __device__ __forceinline__ long long before(int i) const {
    const long long s1 = min(i, s), z1 = min(i, z);
    return static_cast<long long>(i) * kItemCost + (s1 - z1) * off + c * ((s1 * (s1 + 1) - z1 * (z1 + 1)) / 2) +
           (i - s1) * vis;
  }
  // the last pair that starts at or before position x
  __device__ __forceinline__ int pair_at(long long x) const {
    int lo = 0;
    for (int hi = n; hi - lo > 1;) {
      const int mid = (lo + hi) >> 1;
      if (before(mid) <= x) lo = mid;
      else hi = mid;
    }
    return lo;
  }
};
__device__ __forceinline__ SeqWork work_of(const ChunkParams& p, const Seq& s) {
  SeqWork w;
  w.c = 2 * p.tq;
  w.vis = s.vis;
  w.off = p.a.causal == FA_CAUSAL_NONE ? s.vis : s.off;
  w.n = static_cast<long long>(s.nq) * p.a.group <= p.skip_rows ? 0 : (s.nq + w.c - 1) / w.c;
  const unsigned n = w.n, c = w.c, off = w.off;  // (differences below fit 32 bits)
  w.z = w.off < 0 ? static_cast<int>(min((0u - off) / c, n)) : 0;
  w.s = w.off < w.vis ? static_cast<int>(min((static_cast<unsigned>(w.vis) - off) / c, n)) : 0;
  w.s = max(w.s, w.z);
  return w;
}

// Where a CTA starts in the work order.
struct WorkStart {
  long long per;   // positions of a run
  long long base;  // of sequence b (p.runs: positions, else pairs)
  int b;           // -1: past the end
  int blocks;      // 128-row blocks before the sequence in the expanded rows
  Seq s;
};
// Called by all threads.  p.runs: CTA x starts at position x * per, else at pair x.
template <bool kExp>
__device__ __forceinline__ void find_start(const ChunkParams& p, int x, WorkStart* out, long long* scan_a,
                                           long long* scan_b) {
  const PagedAttn& a = p.a;
  const int share = (a.r.B + kThreads - 1) / kThreads;
  const int b0 = min(static_cast<int>(threadIdx.x) * share, a.r.B), b1 = min(b0 + share, a.r.B);
  Seq s{};  // the last one looked at
  int blocks = 0;
  auto weight = [&](int b) -> long long {
    s = load_seq(a, b);
    const bool ours = static_cast<long long>(s.nq) * a.group > p.skip_rows;
    blocks = ours ? expand_blocks(s) : 0;
    if (!p.runs) return ours ? (s.nq + 2 * p.tq - 1) / (2 * p.tq) : 0;
    const SeqWork w = work_of(p, s);
    return p.n_heads * w.before(w.n);
  };
  if (threadIdx.x == 0) out->b = -1;
  long long sum = 0, sum_blocks = 0, total, unused;
  for (int b = b0; b < b1; ++b) {
    sum += weight(b);
    sum_blocks += blocks;
  }
  long long at = block_scan<kThreads>(sum, scan_a, &total);
  long long at_blocks = kExp ? block_scan<kThreads>(sum_blocks, scan_b, &unused) : 0;
  const long long per =
      p.runs ? max((total + p.n_ctas - 1) / p.n_ctas, static_cast<long long>(kMinRun)) : 1;
  const long long v = x * per;
  if (v >= at && v < at + sum) {
    int b = b0;
    if (share > 1)
      for (;; ++b) {
        const long long w = weight(b);
        if (v < at + w) break;
        at += w;
        at_blocks += blocks;
      }
    out->per = per;
    out->base = at;
    out->blocks = static_cast<int>(at_blocks);
    out->b = b;
    out->s = s;
  }
  __syncthreads();
}

// The reference of P over 8-bit pages (log2): none yet; how far P may pass it until
// O is rescaled; and how far it may be above and below the largest score, so that
// the exponentials relative to it stay in fp32's range.  V's scales, 2^-109 to 2^121
// in what the write stores, are taken times 2^-kScaleShift: within the range from
// kRefBelow below to kRefAbove above, but for the largest ones, whose P is then up to
// 2^15, still in f16's range.
constexpr float kNoRef = -1e30f, kRefLag = 14.f, kRefAbove = 100.f, kRefBelow = 116.f;
constexpr float kScaleShift = 6.f;

// A segment as the softmax of query tile g sees it.
struct ChunkItem {
  Seq s;
  int h, tok_lo, jb, n_tiles, slot, tiles, par;
  bool last;
};

// SRC: what is read; QBF16: type of Q and O.
template <int D, int SRC, bool QBF16>
__global__ void __launch_bounds__(kThreads, 1) paged_chunk_kernel(const __grid_constant__ ChunkParams p) {
  constexpr bool kExp = SRC == kExpanded;     // the softmax applies the scales
  constexpr bool kBf16 = SRC == kPagesBf16;   // type of P and V (Q and K: QBF16)
  using L = ChunkLayout<D, kExp>;
  const PagedAttn& a = p.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  __shared__ long long sh_scan[2][kThreads / 32];
  __shared__ WorkStart start;
  const uint32_t sbase = ptx::smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 4);
  auto bar = [&](int i) -> uint32_t { return sbase + L::kOffBar + 8u * static_cast<uint32_t>(i); };
  ptx::launch_dependents();

  // ---- where does this CTA's work start?
  const int cta = static_cast<int>(blockIdx.x);
  find_start<kExp>(p, p.runs ? cta : cta / p.n_heads, &start, sh_scan[0], sh_scan[1]);
  if (p.fill) {
    fill_outside(a, D, cta, static_cast<int>(gridDim.x));
    if (a.max_q < a.r.total)
      for (int b = cta; b < a.r.B; b += static_cast<int>(gridDim.x)) fill_beyond(a, D, load_seq(a, b));
  }
  // (whatever ends this CTA early, the join finds nothing to do for it)
  if (p.runs && p.n_ctas > 1 && threadIdx.x == 0) p.ws_cuts[cta].parts = 0;
  if (start.b < 0) return;
  const int n_rows = p.tq * a.group;  // rows of a tile in use

  // ---- set-up
  int dead = 0;  // this launch failed elsewhere
  if (threadIdx.x == 0) {
    const unsigned long long st = *reinterpret_cast<volatile unsigned long long*>(&g_fa_status);
    dead = ((st >> 32) == p.epoch && (st & 0xffffffffull) != 0ull) ? 1 : 0;
    *abort_flag = 0;
    for (int i = 0; i < L::kNumBars; ++i) {
      const bool all = (i >= L::kBarP && i < L::kBarP + 2) || (i >= L::kBarPH && i < L::kBarPH + 2);
      const bool seg = i >= L::kBarSegEmpty;  // one arrival per warp that reads segments
      ptx::mbar_init(bar(i), all ? 128u : seg ? 11u : 1u);
    }
    ptx::fence_barrier_init();
  }
  if (__syncthreads_or(dead)) return;
  if (warp == kWarpMma) {
    ptx::tmem_alloc(ptx::smem_u32(tmem_slot), L::kTmemCols);
    ptx::tmem_relinquish();
    ptx::tc_fence_before();
  }
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  const WaitCtl wc{abort_flag, p.timeout_ns, p.epoch};
  volatile Segment* const segs = reinterpret_cast<volatile Segment*>(smem + L::kOffSeg);
  // Every reading warp waits for segment n, reads it and releases it.
  auto seg_ready = [&](int n) {
    return __all_sync(0xffffffffu, bar_wait(bar(L::kBarSegFull + n % kSegRing), (n / kSegRing) & 1, wc, 3));
  };
  auto seg_done = [&](int n) {
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(bar(L::kBarSegEmpty + n % kSegRing));
  };

  if (warp >= 8) {
    ptx::setmaxnreg_dec<L::kRegsRest>();
    if (warp == kWarpMma + 2) {
      // =================================================== the run's segments
      int b = start.b, n_seg = 0, tiles = 0, par = 0;
      int exp_row0 = start.blocks * kBlockN;
      bool ok = true;
      auto push = [&](const Seq& s, int h, int tok0, int jb, int n0, int n1, int slot) {
        const int e = n_seg % kSegRing;
        if (n_seg >= kSegRing &&
            !(ok = __all_sync(0xffffffffu, bar_wait(bar(L::kBarSegEmpty + e), ((n_seg / kSegRing) - 1) & 1, wc, 4))))
          return;
        if (lane == 0) {
          volatile Segment& g = segs[e];
          g.b = b;
          g.h = h;
          g.c0 = s.c0;
          g.nq = s.nq;
          g.nk = s.nk;
          g.off = s.off;
          g.vis = s.vis;
          g.tok0 = tok0;
          g.jb = jb;
          g.n0 = n0;
          g.n1 = n1;
          g.slot = slot;
          g.exp_row0 = exp_row0;
          g.tiles = tiles;
          g.parity = par;
          ptx::mbar_arrive(bar(L::kBarSegFull + e));
        }
        __syncwarp();
        ++n_seg;
        tiles += max(n0, n1);
        par ^= (n0 & 1) | ((n1 & 1) << 1);
      };
      // tiles [lo, hi) of pair i of head h
      auto take = [&](const Seq& s, int h, int i, int lo, int hi, int slot) {
        int n[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const int tok = (2 * i + g) * p.tq;
          const int lim = tok < s.nq ? row_limit(a, s, min(tok + p.tq, s.nq) - 1) : 0;
          n[g] = max(min((lim + kBlockN - 1) / kBlockN, hi) - lo, 0);
        }
        push(s, h, 2 * i * p.tq, lo, n[0], n[1], slot);
      };
      Seq s = start.s;
      SeqWork w = work_of(p, s);
      if (!p.runs) {
        // pairs of a sequence from its end, the longest causal rows first
        const int i = static_cast<int>(start.base) + w.n - 1 - cta / p.n_heads;
        take(s, p.head0 + cta % p.n_heads, i, 0, w.tiles(i), -1);
      } else {
        const long long v0 = cta * start.per, v1 = v0 + start.per;
        const long long all = w.before(w.n);
        PagedCut cut{};  // the item that this run's end cuts first
        int h = static_cast<int>((v0 - start.base) / all);
        long long at = start.base + h * all;  // of pair 0, then of pair i
        int i = w.pair_at(v0 - at);
        at += w.before(i);
        while (ok && at < v1) {
          const int n = w.tiles(i);
          const long long key0 = at + kItemCost;
          auto from = [&](long long v) {  // first tile that starts at or after v
            const long long k = v - key0;
            return k <= 0 ? 0 : static_cast<int>(min((k + kBlockN - 1) / kBlockN, static_cast<long long>(n)));
          };
          const int lo = from(v0), hi = from(v1);
          if (lo == 0 && hi > 0 && hi < n) {
            const long long last = (key0 + static_cast<long long>(n - 1) * kBlockN) / start.per;  // its last run
            cut = PagedCut{s.c0, s.nq, 2 * i * p.tq, p.head0 + h, static_cast<int>(last) - cta + 1, {0, 0, 0}};
          }
          if (lo < hi) take(s, p.head0 + h, i, lo, hi, lo > 0 ? 2 * cta : hi < n ? 2 * cta + 1 : -1);
          else if (n == 0 && at >= v0) take(s, p.head0 + h, i, 0, 0, -1);
          at = key0 + w.lim(i);
          if (++i == w.n) {
            i = 0;
            if (++h == p.n_heads) {
              h = 0;
              if (w.n > 0) exp_row0 += expand_blocks(s) * kBlockN;
              do {
                if (++b >= a.r.B) break;
                s = load_seq(a, b);
                w = work_of(p, s);
              } while (w.n == 0);
              if (b >= a.r.B) break;
            }
          }
        }
        if (ok && lane == 0 && p.n_ctas > 1) p.ws_cuts[cta] = cut;
      }
      if (ok) {
        b = -1;
        push(s, 0, 0, 0, 0, 0, -1);
      }
    } else if (warp == kWarpLoad || warp == kWarpMma + 1) {
      // ================================================ TMA producers: K (and Q), V
      const int second = warp == kWarpLoad ? 0 : 1;
      const uint64_t pol_q = ptx::policy_evict_first();
      const uint64_t pol_kv = ptx::policy_evict_last();
      if (lane == 0 && second == 0) {
        ptx::prefetch_tmap(&p.tm_q);
        ptx::prefetch_tmap(&p.tm_k);
        ptx::prefetch_tmap(&p.tm_v);
      }
      __syncwarp();
      // lane = box of the tile (the expanded rows have one of 128 rows)
      const int box = lane;
      const bool issues = box * p.box_rows < kBlockN;
      const uint32_t dst_off = box * p.box_rows * (2 * D);
      bool ok = true;
      int i = second;                   // ring entry: K_0 V_0 K_1 V_1 ..., over all segments
      int n_tail = 0, n_q[2] = {0, 0};  // stale V tiles, Q tiles loaded so far
      for (int n = 0; (ok = seg_ready(n)); ++n) {
        const volatile Segment& sg = segs[n % kSegRing];
        const int b = sg.b, h = sg.h, c0 = sg.c0, vis = sg.vis, tok0 = sg.tok0, jb = sg.jb;
        const int n_kv[2] = {sg.n0, sg.n1}, exp_row0 = sg.exp_row0;
        seg_done(n);
        if (b < 0) break;
        const int n_loop = max(n_kv[0], n_kv[1]);
        // place of this lane's box in the map's last dimension; -1 reads as zeros
        auto page_at = [&](int tile) {
          if (kExp) return h - p.head0;
          const int pos = tile * kBlockN + box * p.box_rows;
          const int page = issues && pos < vis ? a.c.lookup(b, pos) : -1;
          return page >= 0 ? page * p.page_step + h * p.head_step : -1;
        };
        int next_page = n_loop > 0 ? page_at(jb) : -1, page = -1;
        for (int g = 0; ok && g < 2 && second == 0; ++g) {
          if (n_kv[g] == 0) continue;
          if (n_q[g] > 0 &&
              !(ok = __all_sync(0xffffffffu, bar_wait(bar(L::kBarQFree + g), (n_q[g] - 1) & 1, wc, 8))))
            break;
          ++n_q[g];
          if (lane == 0) {
            ptx::mbar_arrive_expect_tx(bar(L::kBarQ + g), L::kColBlocks * n_rows * 128);
#pragma unroll
            for (int c = 0; c < L::kColBlocks; ++c)
              ptx::tma_load_3d(sbase + L::kOffQ + g * L::kTile + c * L::kBlockBytes, &p.tm_q,
                               bar(L::kBarQ + g), c * 64, h * a.group, c0 + tok0 + g * p.tq, pol_q);
          }
          __syncwarp();
        }
        for (int x = 0; ok && x < n_loop; ++x) {
          const int tile = jb + x;
          page = next_page;
          if (x + 1 < n_loop) next_page = page_at(tile + 1);
          const int slot = i % L::kSlots;
          if (i >= L::kSlots &&
              !(ok = __all_sync(0xffffffffu, bar_wait(bar(L::kBarEmpty + slot),
                                                      ((i / L::kSlots) - 1) & 1, wc, 1))))
            break;
          // stale V rows of the tile: [r0, r1)
          const int r0 = vis - tile * kBlockN;
          const int r1 = (r0 + p.box_rows - 1) / p.box_rows * p.box_rows;
          // (a run-time flag, though the expanded rows never have any: with the
          // branch compiled out ptxas schedules the softmax over 8-bit pages worse, 2
          // x 2048 tokens over 8192 keys take 3 % longer at d = 128, 4 % at d = 64)
          const bool tail = p.stale && second && r0 < kBlockN && r0 != r1;
          const uint32_t full = tail ? bar(L::kBarTail) : bar(L::kBarFull + slot);
          const bool scales = kExp && !second;
          if (lane == 0) ptx::mbar_arrive_expect_tx(full, L::kTile + (scales ? L::kScaleEntry : 0));
          __syncwarp();
          const uint32_t dst = sbase + L::kOffKV + slot * L::kTile;
          // first row: in the page, or in the expanded rows (kept inside them)
          const int row = kExp ? min(exp_row0 + tile * kBlockN, static_cast<int>(p.exp_rows) - kBlockN)
                               : a.c.row_in_page(tile * kBlockN + box * p.box_rows);
          if (issues)
            ptx::tma_load_5d(dst + dst_off, second ? &p.tm_v : &p.tm_k, full, 0, 0, 0, row >> 3, page, pol_kv);
          if (scales && lane < 4) {
            const long long at = static_cast<long long>(h - p.head0) * p.exp_rows + row;
            const float* src = lane == 0   ? p.exp_ks + at
                               : lane == 1 ? p.exp_vs + at
                               : lane == 2 ? p.exp_vl + at
                                           : p.exp_vm + at / 16;
            ptx::bulk_load(sbase + L::kOffScale + ((i >> 1) % L::kScaleRing) * L::kScaleEntry + lane * 512, src,
                           lane < 3 ? 512 : 32, full);
          }
          i += 2;
          if (tail) {
            const bool here = __all_sync(0xffffffffu, bar_wait(bar(L::kBarTail), n_tail & 1, wc, 7));
            ++n_tail;
            if (!(ok = here)) {
              i -= 2;  // (its slot is not announced)
              break;
            }
            for (int y = lane; y < (r1 - r0) * 8 * L::kColBlocks; y += 32) {
              const int r = r0 + y / (8 * L::kColBlocks), c = y % (8 * L::kColBlocks);
              *reinterpret_cast<uint4*>(smem + L::kOffKV + slot * L::kTile + (r >> 3) * L::kGroupBytes +
                                        (c >> 3) * 1024 + (r & 7) * 128 + (c & 7) * 16) =
                  make_uint4(0u, 0u, 0u, 0u);
            }
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(bar(L::kBarFull + slot));
          }
        }
        if (!ok) break;
      }
      // every copy started lands before the CTA exits
      for (int r = i - 2; r >= 0 && r >= i - L::kSlots; r -= 2)
        bar_wait(bar(L::kBarFull + r % L::kSlots), (r / L::kSlots) & 1, wc, 2, false);
      if (n_tail > 0 && !ok) bar_wait(bar(L::kBarTail), (n_tail - 1) & 1, wc, 2, false);
      for (int g = 0; g < 2; ++g)
        if (n_q[g] > 0) bar_wait(bar(L::kBarQ + g), (n_q[g] - 1) & 1, wc, 2, false);
    } else if (warp == kWarpMma) {
      // =================================================== MMA issuer (see fa_fwd_kernel)
      constexpr uint32_t idesc_qk = ptx::make_idesc_f16(kBlockM, kBlockN, QBF16 ? 1u : 0u, 0, 0);
      constexpr uint32_t idesc_pv = ptx::make_idesc_f16(kBlockM, D, kBf16 ? 1u : 0u, 0, 1);
      const uint64_t k_desc0 = ptx::smem_desc_sw128(sbase + L::kOffKV, 16, L::kGroupBytes);
      const uint64_t v_desc0 = ptx::smem_desc_sw128(sbase + L::kOffKV, 1024, L::kGroupBytes);
      const uint64_t q_desc0 = ptx::smem_desc_sw128(sbase + L::kOffQ, 16, 1024);
      const uint32_t kv_hi = static_cast<uint32_t>(k_desc0 >> 32);  // (the same for K and V)
      const uint32_t q_hi = static_cast<uint32_t>(q_desc0 >> 32);
      const uint32_t k_lo0 = static_cast<uint32_t>(k_desc0);
      const uint32_t v_lo0 = static_cast<uint32_t>(v_desc0);
      const uint32_t q_lo0 = static_cast<uint32_t>(q_desc0);
      const uint32_t q_lo1 =
          static_cast<uint32_t>(ptx::smem_desc_sw128(sbase + L::kOffQ + L::kTile, 16, 1024));
      constexpr uint32_t kSlotStep = L::kTile >> 4;
      constexpr uint32_t kVStep = 2 * L::kGroupBytes >> 4;  // 16 keys
      auto issue_s = [&](int g, int ks, uint32_t q_lo, bool last) {
        const uint32_t k_lo = k_lo0 + static_cast<uint32_t>(ks) * kSlotStep;
        if (ptx::elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t q_off = static_cast<uint32_t>(((kk / 4) * L::kBlockBytes + (kk % 4) * 32) >> 4);
            const uint32_t k_off = static_cast<uint32_t>(((kk / 4) * 1024 + (kk % 4) * 32) >> 4);
            ptx::mma_ss(tmem + L::tS(g), ptx::make_desc(q_lo + q_off, q_hi),
                        ptx::make_desc(k_lo + k_off, kv_hi), idesc_qk, kk > 0 ? 1u : 0u);
          }
          ptx::mma_commit(bar(L::kBarS + g));
          if (last) ptx::mma_commit(bar(L::kBarQFree + g));
        }
        __syncwarp();
      };
      auto commit = [&](uint32_t b) {
        if (ptx::elect_one()) ptx::mma_commit(b);
        __syncwarp();
      };
      auto wait = [&](uint32_t b, uint32_t ph, int site) {
        return __all_sync(0xffffffffu, bar_wait_lean(b, ph, wc, site));
      };
      auto issue_pv = [&](int g, int vs, bool first, uint32_t ph) -> bool {
        const uint32_t v_lo = v_lo0 + static_cast<uint32_t>(vs) * kSlotStep;
        if (!wait(bar(L::kBarPH + g), ph, 13 + 3 * g)) return false;
        ptx::tc_fence_after();
        if (ptx::elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 2 * kPEarlyQuarters; ++kk)
            ptx::mma_ts(tmem + L::tO(g), tmem + L::tP(g) + kk * 8,
                        ptx::make_desc(v_lo + kk * kVStep, kv_hi), idesc_pv, (!first || kk > 0) ? 1u : 0u);
        }
        __syncwarp();
        if (!wait(bar(L::kBarP + g), ph, 13 + 3 * g)) return false;
        ptx::tc_fence_after();
        if (ptx::elect_one()) {
#pragma unroll
          for (int kk = 2 * kPEarlyQuarters; kk < kBlockN / 16; ++kk)
            ptx::mma_ts(tmem + L::tO(g), tmem + L::tP(g) + kk * 8,
                        ptx::make_desc(v_lo + kk * kVStep, kv_hi), idesc_pv, 1u);
          ptx::mma_commit(bar(L::kBarO + g));
        }
        __syncwarp();
        return true;
      };
      bool ok = true;
      int ks = 0;                      // ring slot of the next K, its phase
      uint32_t kph = 0;
      uint32_t cnt[2] = {0, 0};        // key tiles of query tile g so far
      uint32_t n_q[2] = {0, 0};        // Q tiles used so far
      auto adv = [](int& sl, uint32_t& ph) {
        if (++sl == L::kSlots) {
          sl = 0;
          ph ^= 1u;
        }
      };
      for (int n = 0; ok && (ok = seg_ready(n)); ++n) {
        const volatile Segment& sg = segs[n % kSegRing];
        const int b = sg.b, n0 = sg.n0, n1 = sg.n1;
        seg_done(n);
        if (b < 0) break;
        const int n_loop = max(n0, n1);
        if (n_loop > 0) {
          if (n0 > 0) ok = wait(bar(L::kBarQ), n_q[0]++ & 1, 10);
          if (ok && n1 > 0) ok = wait(bar(L::kBarQ + 1), n_q[1]++ & 1, 10);
          if (ok) ok = wait(bar(L::kBarFull + ks), kph, 11);
          if (ok) {
            ptx::tc_fence_after();
            if (n0 > 0) issue_s(0, ks, q_lo0, n0 == 1);
            if (n1 > 0) issue_s(1, ks, q_lo1, n1 == 1);
            commit(bar(L::kBarEmpty + ks));
          }
        }
        for (int j = 0; ok && j < n_loop; ++j) {
          int vs = ks;
          uint32_t vph = kph;
          adv(vs, vph);
          int ns = vs;
          uint32_t nph = vph;
          adv(ns, nph);
          ks = ns;
          kph = nph;
          const bool next0 = j + 1 < n0, next1 = j + 1 < n1;
          if (!(ok = wait(bar(L::kBarFull + vs), vph, 12))) break;
          if ((next0 || next1) && !(ok = wait(bar(L::kBarFull + ns), nph, 14))) break;
          if (j < n0) {
            if (!(ok = issue_pv(0, vs, j == 0, (cnt[0] + j) & 1))) break;
            if (next0) {
              issue_s(0, ns, q_lo0, j + 2 == n0);
              if (!next1) commit(bar(L::kBarEmpty + ns));
            }
          }
          if (j < n1) {
            if (!(ok = issue_pv(1, vs, j == 0, (cnt[1] + j) & 1))) break;
          }
          commit(bar(L::kBarEmpty + vs));
          if (next1) {
            issue_s(1, ns, q_lo1, j + 2 == n1);
            commit(bar(L::kBarEmpty + ns));
          }
        }
        cnt[0] += n0;
        cnt[1] += n1;
      }
      // all products complete before tensor memory is released
      commit(bar(L::kBarDrain));
      bar_wait(bar(L::kBarDrain), 0, wc, 19, false);
      __syncwarp();
    }
  } else {
    // ===================================================== softmax groups
    ptx::setmaxnreg_inc<L::kRegsSoft>();
    const int g = warp >> 2;
    const int wq = warp & 3;
    const int r = wq * 32 + lane;  // row of the tile == TMEM lane
    const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t tS = tmem + lane_off + L::tS(g);
    const uint32_t tP = tmem + lane_off + L::tP(g);
    const uint32_t tO = tmem + lane_off + L::tO(g);
    bool ok = true;
    for (int n_seg = 0; ok && (ok = seg_ready(n_seg)); ++n_seg) {
      ChunkItem it;
      {
        const volatile Segment& sg = segs[n_seg % kSegRing];
        it.last = sg.b < 0;
        it.h = sg.h;
        it.s.c0 = sg.c0;
        it.s.nq = sg.nq;
        it.s.nk = sg.nk;
        it.s.off = sg.off;
        it.tok_lo = sg.tok0 + g * p.tq;
        it.jb = sg.jb;
        it.n_tiles = g ? sg.n1 : sg.n0;
        it.slot = sg.slot;
        it.tiles = sg.tiles;
        it.par = (sg.parity >> g) & 1;
      }
      seg_done(n_seg);
      if (it.last) break;
      const int n_tiles = it.n_tiles;
      const int tok_lo = it.tok_lo;
      const int tok = tok_lo + r / a.group;      // token of the sequence
      const int hq = it.h * a.group + r % a.group;
      const bool row_ok = r < n_rows && tok < it.s.nq;
      const float sl = a.scale_log2;
      // key limit of this row, and the smallest of the tile's rows
      const int row_end = row_limit(a, it.s, tok);
      const int tile_end = row_limit(a, it.s, tok_lo);

      float m = -INFINITY;  // running max of the scaled scores (log2 units)
      float l = 0.f;        // running sum of exp2(s - m)
      float ref = kNoRef;   // kExp: reference of P and O (else m)
      for (int j = 0; ok && j < n_tiles; ++j) {
        ok = __all_sync(0xffffffffu, bar_wait(bar(L::kBarS + g), (it.par + j) & 1, wc, 20 + g));
        if (!ok) break;
        ptx::tc_fence_after();
        float x[kBlockN];
        {
          uint32_t u0[32], u1[32], u2[32], u3[32];
          ptx::tmem_ld32(tS + 0, u0);
          ptx::tmem_ld32(tS + 32, u1);
          ptx::tmem_ld32(tS + 64, u2);
          ptx::tmem_ld32(tS + 96, u3);
          ptx::tmem_wait_ld();
          pin_after_wait<32>(u0);
          pin_after_wait<32>(u1);
          pin_after_wait<32>(u2);
          pin_after_wait<32>(u3);
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            x[c] = __uint_as_float(u0[c]);
            x[32 + c] = __uint_as_float(u1[c]);
            x[64 + c] = __uint_as_float(u2[c]);
            x[96 + c] = __uint_as_float(u3[c]);
          }
        }
        const uint32_t entry = sbase + L::kOffScale + (kExp ? ((it.tiles + j) % L::kScaleRing) * L::kScaleEntry : 0);
        if constexpr (kExp) {
#pragma unroll
          for (int c = 0; c < kBlockN; c += 4) {
            const float4 f = load_scales(entry + 4 * c);
            ptx::fmul2(x[c], x[c + 1], x[c], x[c + 1], f.x, f.y);
            ptx::fmul2(x[c + 2], x[c + 3], x[c + 2], x[c + 3], f.z, f.w);
          }
        }

        const int key0 = (it.jb + j) * kBlockN;
        const bool masked = key0 + kBlockN > tile_end;
        float m_tile;
        float sl_eff = sl;
        if (masked) {
          const int lim = row_end - key0;
#pragma unroll
          for (int c = 0; c < kBlockN; c += 2) ptx::fmul2(x[c], x[c + 1], x[c], x[c + 1], sl, sl);
#pragma unroll
          for (int c = 0; c < kBlockN; ++c)
            if (c >= lim) x[c] = -INFINITY;
          m_tile = row_extreme<kBlockN, false>(x);
          sl_eff = 1.0f;
        } else if (sl >= 0.f) {
          m_tile = row_extreme<kBlockN, false>(x) * sl;
        } else {
          m_tile = row_extreme<kBlockN, true>(x) * sl;
        }
        const float m_new = fmaxf(m, m_tile);
        auto scale_o = [&](float alpha) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            ptx::tmem_ld32(tO + c * 32, o);
            ptx::tmem_wait_ld();
            pin_after_wait<32>(o);
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float a0 = __uint_as_float(o[i]), a1 = __uint_as_float(o[i + 1]);
              ptx::fmul2(a0, a1, a0, a1, alpha, alpha);
              o[i] = __float_as_uint(a0);
              o[i + 1] = __float_as_uint(a1);
            }
            ptx::tmem_st32(tO + c * 32, o);
          }
          ptx::tmem_wait_st();
        };
        if constexpr (kExp) {
          if (m_new > m) l *= ptx::ex2_approx(m - m_new);
          m = m_new;
          const float4 v0 = load_scales(entry + 1536), v1 = load_scales(entry + 1552);
          const float vm = fmax3(fmax3(fmaxf(v0.x, v0.y), v0.z, v0.w), fmaxf(v1.x, v1.y), fmaxf(v1.z, v1.w));
          if (__any_sync(0xffffffffu, m_tile + vm > ref + kRefLag || m > ref + kRefBelow)) {
            float y = -INFINITY;  // the largest s + log2 vs
#pragma unroll
            for (int c = 0; c < kBlockN; c += 4) {
              const float4 f = load_scales(entry + 1024 + 4 * c);
              y = fmax3(y, fmaf(x[c], sl_eff, f.x), fmaf(x[c + 1], sl_eff, f.y));
              y = fmax3(y, fmaf(x[c + 2], sl_eff, f.z), fmaf(x[c + 3], sl_eff, f.w));
            }
            y = fmaxf(fminf(y, m + kRefAbove), m - kRefBelow);
            const bool grow = y > ref + kRefLag || m > ref + kRefBelow;
            if (j > 0 && __any_sync(0xffffffffu, grow)) scale_o(grow ? ptx::ex2_approx(ref - y) : 1.0f);
            if (grow) ref = y;
          }
        } else {
          const bool grow = m_new > m + kRescaleThreshold;
          if (j == 0) {
            m = m_new;
          } else {
            if (__any_sync(0xffffffffu, grow)) {
              const float alpha = grow ? ptx::ex2_approx(m - m_new) : 1.0f;
              scale_o(alpha);
              l *= alpha;
            }
            if (grow) m = m_new;
          }
        }
        const uint32_t half_bar = bar(L::kBarPH + g);
        auto announce = [half_bar] { ptx::mbar_arrive(half_bar); };
        float tile_sum;
        if constexpr (kExp) {
          tile_sum = masked ? exp_tile_scaled<false, kEmuPeriod>(x, sl_eff, -ref, entry + 512, tP, announce)
                            : exp_tile_scaled<true, kPairEmuPeriod<D>>(x, sl_eff, -ref, entry + 512, tP, announce);
          tile_sum *= m == -INFINITY ? 1.f : ptx::ex2_approx(ref - m);  // (1: no key so far, or NaN)
        } else {
          const float neg_m = (m == -INFINITY) ? 0.f : -m;
          tile_sum = masked ? exp_tile<kBf16, false>(x, sl_eff, neg_m, tP, announce)
                            : exp_tile<kBf16, true, kPairEmuPeriod<D>>(x, sl_eff, neg_m, tP, announce);
        }
        ptx::tmem_wait_st();
        ptx::tc_fence_before();
        ptx::mbar_arrive(bar(L::kBarP + g));
        l += tile_sum;
      }

      // ---- epilogue
      using T = typename std::conditional<QBF16, __nv_bfloat16, __half>::type;
      const long long row_id = static_cast<long long>(it.s.c0 + tok) * a.Hq + hq;
      const bool partial = it.slot >= 0;
      const long long ws_row = (static_cast<long long>(it.slot) * 2 + g) * kBlockM + r;
      float* lse_dst = partial ? p.ws_lse + ws_row
                       : a.lse ? a.lse + static_cast<long long>(hq) * a.r.total + it.s.c0 + tok
                               : nullptr;
      if (n_tiles == 0) {
        if (row_ok && !partial) {
          uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.o) + row_id * D);
#pragma unroll
          for (int i = 0; i < D / 8; ++i) dst[i] = make_uint4(0u, 0u, 0u, 0u);
        }
        if (row_ok && lse_dst) *lse_dst = -INFINITY;
      } else {
        if (ok) ok = __all_sync(0xffffffffu, bar_wait(bar(L::kBarO + g), (it.par + n_tiles - 1) & 1, wc, 22 + g));
        if (ok) {
          ptx::tc_fence_after();
          // (a NaN stays one; 2^(ref - m) / l as one exponent, for its parts may pass fp32's range)
          const float inv_l = l == 0.f ? 0.f : kExp ? exp2f(ref - m - __log2f(l) + kScaleShift) : l > 0.f ? 1.0f / l : l;
          const float m_use = (m == -INFINITY) ? 0.f : m;
          const float lse_row =
              l == 0.f ? -INFINITY : (m_use + __log2f(l)) * 0.69314718055994530942f;
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            ptx::tmem_ld32(tO + c * 32, o);
            ptx::tmem_wait_ld();
            pin_after_wait<32>(o);
            if (!partial) {
              uint32_t hv[16];
#pragma unroll
              for (int i = 0; i < 16; ++i)
                hv[i] = pack2<QBF16>(__uint_as_float(o[2 * i]) * inv_l, __uint_as_float(o[2 * i + 1]) * inv_l);
              if (row_ok) {
                uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.o) + row_id * D + c * 32);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  dst[i] = make_uint4(hv[4 * i], hv[4 * i + 1], hv[4 * i + 2], hv[4 * i + 3]);
              }
            } else if (row_ok) {
              // four columns of all rows side by side: a warp's stores are 512 bytes
              float4* dst = reinterpret_cast<float4*>(p.ws_o + (ws_row - r) * D) + c * 8 * kBlockM + r;
#pragma unroll
              for (int i = 0; i < 8; ++i)
                dst[i * kBlockM] =
                    make_float4(__uint_as_float(o[4 * i]) * inv_l, __uint_as_float(o[4 * i + 1]) * inv_l,
                                __uint_as_float(o[4 * i + 2]) * inv_l, __uint_as_float(o[4 * i + 3]) * inv_l);
            }
          }
          if (row_ok && lse_dst) *lse_dst = lse_row;
        }
      }
    }
  }

  // ---- teardown
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == kWarpMma) {
    __syncwarp();
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, L::kTmemCols);
  }
}

// Joins the parts of the items that the chunk kernel's runs cut: LSE = log sum_s
// exp(LSE_s), O = sum_s exp(LSE_s - LSE) O_s, parts in the order of their keys.
// Bound by latency, a dependent read of the table and of the parts: 4 to 5 us of a
// call.  Block x is for the item that the end of run x cuts first; a thread has 16
// columns of one of its 256 rows, a warp 32 rows.
constexpr int kJoinThreads = 256;
template <int D, bool BF16>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ ChunkParams p) {
  const PagedAttn& a = p.a;
  ptx::grid_dep_wait();
  const PagedCut c = p.ws_cuts[blockIdx.x];
  if (c.parts == 0) return;
  const int y = static_cast<int>(blockIdx.y * kJoinThreads + threadIdx.x);
  const int r = y % kBlockM, col = y / kBlockM % (D / 16) * 16, g = y / (kBlockM * (D / 16));
  const int tok = c.tok0 + g * p.tq + r / a.group;
  if (r >= p.tq * a.group || tok >= c.nq) return;
  // first row of query tile g in part x
  auto tile_row = [&](int x) {
    return ((x == 0 ? 2ll * blockIdx.x + 1 : 2ll * (blockIdx.x + x)) * 2 + g) * kBlockM;
  };
  float mx = -INFINITY;
#pragma unroll 4
  for (int x = 0; x < c.parts; ++x) mx = fmaxf(mx, __ldcg(p.ws_lse + tile_row(x) + r));
  float acc[16] = {}, sum = 0.f;
#pragma unroll 2
  for (int x = 0; x < c.parts; ++x) {
    const float4* src = reinterpret_cast<const float4*>(p.ws_o + tile_row(x) * D) + (col >> 2) * kBlockM + r;
    float4 o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __ldcg(src + e * kBlockM);
    const float ls = __ldcg(p.ws_lse + tile_row(x) + r);
    // (a part without a key for this row has no O; a NaN stays one)
    const float f = ls == -INFINITY ? 0.f : expf(ls - mx);
    sum += f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      acc[4 * e] = f == 0.f ? acc[4 * e] : fmaf(f, o[e].x, acc[4 * e]);
      acc[4 * e + 1] = f == 0.f ? acc[4 * e + 1] : fmaf(f, o[e].y, acc[4 * e + 1]);
      acc[4 * e + 2] = f == 0.f ? acc[4 * e + 2] : fmaf(f, o[e].z, acc[4 * e + 2]);
      acc[4 * e + 3] = f == 0.f ? acc[4 * e + 3] : fmaf(f, o[e].w, acc[4 * e + 3]);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  const int hq = c.h * a.group + r % a.group;
  const long long out = static_cast<long long>(c.c0 + tok) * a.Hq + hq;
  uint32_t w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = pack2<BF16>(acc[2 * e] * inv, acc[2 * e + 1] * inv);
  uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.o) + out * D + col);
  dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
  dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
  if (col == 0 && a.lse != nullptr)
    a.lse[static_cast<long long>(hq) * a.r.total + c.c0 + tok] = sum == 0.f ? -INFINITY : mx + logf(sum);
}

// The visible keys and values of the chunk kernel's sequences as 16-bit rows:
// sequence after sequence, each padded to 128 rows (the padding is zeros),
// [n_heads][exp_rows][d] for K (in the type of the queries) and for V (f16), with
// the scales [n_heads][exp_rows], V's logarithms and the largest of every 16 rows.
// Both types hold 8-bit values exactly.  A warp takes groups of 16 keys of one head.
// Bound by memory, much of it L2: 39 MB of e4m3 pages become 79 MB in 20 us.
constexpr int kExpandThreads = 128;

template <int D, int KV, bool kKBf16>
__global__ void __launch_bounds__(kExpandThreads) paged_expand_kernel(const __grid_constant__ ChunkParams p) {
  const PagedAttn& a = p.a;
  constexpr int L = D / 16;            // lanes per row: 8 bytes at 8 part and at d / 2 + 8 part
  constexpr int kRows = 32 / L;        // rows per pass
  constexpr int kPasses = 16 / kRows;
  __shared__ long long sh_scan[kExpandThreads / 32];
  __shared__ int sh_first[kExpandThreads];  // blocks before each thread's share of the sequences
  const int lane = threadIdx.x & 31, part = lane % L;
  const int share = (a.r.B + kExpandThreads - 1) / kExpandThreads;
  auto blocks_of = [&](int b) {
    const Seq s = load_seq(a, b);
    return static_cast<long long>(s.nq) * a.group <= p.skip_rows ? 0 : expand_blocks(s);
  };
  long long total;
  {
    const int b0 = min(static_cast<int>(threadIdx.x) * share, a.r.B), b1 = min(b0 + share, a.r.B);
    long long sum = 0;
    for (int b = b0; b < b1; ++b) sum += blocks_of(b);
    sh_first[threadIdx.x] = static_cast<int>(block_scan<kExpandThreads>(sum, sh_scan, &total));
    __syncthreads();
  }
  // units: (block, group of 16 rows in it, head), heads fastest
  const long long n_units = min(total * 8, p.exp_rows / 16) * p.n_heads;
  for (long long u = static_cast<long long>(blockIdx.x) * (kExpandThreads / 32) + (threadIdx.x >> 5);
       u < n_units; u += static_cast<long long>(gridDim.x) * (kExpandThreads / 32)) {
    const int h = static_cast<int>(u % p.n_heads);
    const long long grp = u / p.n_heads;
    const int block = static_cast<int>(grp >> 3);
    // its sequence: the last share that starts at or before the block, then on from there
    int lo = 0;
#pragma unroll
    for (int step = kExpandThreads / 2; step > 0; step >>= 1)
      if (sh_first[lo + step] <= block) lo += step;
    int b = lo * share, first = sh_first[lo];
    for (int n = blocks_of(b); b + 1 < a.r.B && block >= first + n; n = blocks_of(b)) {
      first += n;
      ++b;
    }
    const Seq s = load_seq(a, b);
    const int pos = (block - first) * kBlockN + 16 * static_cast<int>(grp & 7);
    const int left = s.vis - pos;  // rows that exist
    const int page = left > 0 ? a.c.lookup(b, pos) : -1;
    const long long prow = a.c.row_in_page(pos);
    const int head = p.head0 + h;
    const long long src0 = page * a.c.page_stride + head * a.c.head_stride + prow * a.c.row_stride;
    const long long dst0 = static_cast<long long>(h) * p.exp_rows + static_cast<long long>(grp) * 16;
    const long long sc0 = page * a.c.s_page + head * a.c.s_head + prow * a.c.s_row;
    uint2 x[2][kPasses][2];
    float sc[2][kPasses];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv)
#pragma unroll
      for (int y = 0; y < kPasses; ++y) {
        const int r = y * kRows + lane / L;
        x[kv][y][0] = x[kv][y][1] = make_uint2(0u, 0u);
        sc[kv][y] = 0.f;
        if (page >= 0 && r < left) {
          const uint2* src = reinterpret_cast<const uint2*>((kv ? a.c.v : a.c.k) + src0 + r * a.c.row_stride);
          x[kv][y][0] = __ldg(src + part);
          x[kv][y][1] = __ldg(src + D / 16 + part);
          sc[kv][y] = __ldg((kv ? a.c.vs : a.c.ks) + sc0 + r * a.c.s_row);
          if (kv) sc[kv][y] *= 1.f / (1 << static_cast<int>(kScaleShift));
        }
      }
#pragma unroll
    for (int kv = 0; kv < 2; ++kv)
#pragma unroll
      for (int y = 0; y < kPasses; ++y) {
        const long long row = dst0 + y * kRows + lane / L;
        uint4* dst = reinterpret_cast<uint4*>((kv ? p.exp_v : p.exp_k) + row * D) + part;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t w[4];
          widen<KV, false>(x[kv][y][i].x, w[0], w[1]);
          widen<KV, false>(x[kv][y][i].y, w[2], w[3]);
          if (kKBf16 && !kv) {
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              const float2 f = __half22float2(*reinterpret_cast<__half2*>(&w[z]));
              w[z] = pack2<true>(f.x, f.y);
            }
          }
          dst[i * (D / 16)] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (part == 0) (kv ? p.exp_vs : p.exp_ks)[row] = sc[kv][y];
      }
    float vm = -INFINITY;
#pragma unroll
    for (int y = 0; y < kPasses; ++y) {
      const float lg = __log2f(fabsf(sc[1][y]));
      if (part == 0) p.exp_vl[dst0 + y * kRows + lane / L] = lg;
      vm = fmaxf(vm, lg);
    }
#pragma unroll
    for (int o = L; o < 32; o <<= 1) vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, o));
    if (lane == 0) p.exp_vm[dst0 / 16] = vm;
  }
}

template <int D, int SRC, bool QBF16>
cudaError_t launch_chunk_impl(const ChunkParams& p, int grid, cudaStream_t stream) {
  auto kern = paged_chunk_kernel<D, SRC, QBF16>;
  using L = ChunkLayout<D, SRC == kExpanded>;
  static int attr_done[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_done[dev]) {
    // the setmaxnreg split is only safe with exactly kLaunchRegs per thread
    cudaFuncAttributes fa{};
    cudaError_t e = cudaFuncGetAttributes(&fa, kern);
    if (e != cudaSuccess) return e;
    if (fa.numRegs != kLaunchRegs || fa.maxThreadsPerBlock < kThreads) return cudaErrorInvalidConfiguration;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kDynBytes);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_done[dev] = 1;
  }
  kern<<<grid, kThreads, L::kDynBytes, stream>>>(p);
  return cudaGetLastError();
}

template <int D>
cudaError_t launch_chunk_d(const ChunkParams& p, int kv, bool bf16, int grid, cudaStream_t s) {
  switch (kv) {
    case FA_DTYPE_INT8:
    case FA_DTYPE_E4M3:
      return bf16 ? launch_chunk_impl<D, kExpanded, true>(p, grid, s)
                  : launch_chunk_impl<D, kExpanded, false>(p, grid, s);
    case FA_DTYPE_BF16: return launch_chunk_impl<D, kPagesBf16, true>(p, grid, s);
    default: return launch_chunk_impl<D, kPagesF16, false>(p, grid, s);
  }
}

template <int D>
cudaError_t launch_expand_d(const ChunkParams& p, int kv, bool bf16, int grid, cudaStream_t s) {
  if (kv == FA_DTYPE_INT8) {
    if (bf16) paged_expand_kernel<D, FA_DTYPE_INT8, true><<<grid, kExpandThreads, 0, s>>>(p);
    else paged_expand_kernel<D, FA_DTYPE_INT8, false><<<grid, kExpandThreads, 0, s>>>(p);
  } else {
    if (bf16) paged_expand_kernel<D, FA_DTYPE_E4M3, true><<<grid, kExpandThreads, 0, s>>>(p);
    else paged_expand_kernel<D, FA_DTYPE_E4M3, false><<<grid, kExpandThreads, 0, s>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_chunk(const ChunkParams& p, int head_dim, int kv, bool bf16, int sms,
                               cudaStream_t stream) {
  if (kv >= FA_DTYPE_INT8) {
    // enough warps to fill the GPU; they walk the rows there are
    const long long units = p.exp_rows / 16 * p.n_heads;
    const long long most = static_cast<long long>(sms) * 12;
    const long long blocks = (units + kExpandThreads / 32 - 1) / (kExpandThreads / 32);
    const int g = static_cast<int>(blocks < most ? blocks : most);
    const cudaError_t e = head_dim == 64 ? launch_expand_d<64>(p, kv, bf16, g, stream)
                                         : launch_expand_d<128>(p, kv, bf16, g, stream);
    if (e != cudaSuccess) return e;
  }
  const cudaError_t e = head_dim == 64 ? launch_chunk_d<64>(p, kv, bf16, p.n_ctas, stream)
                                       : launch_chunk_d<128>(p, kv, bf16, p.n_ctas, stream);
  if (e != cudaSuccess || !p.runs || p.n_ctas == 1) return e;
  // may start while the last runs finish; it waits for them before it reads
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.n_ctas - 1, 2 * kBlockM * (head_dim / 16) / kJoinThreads);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (head_dim == 64)
    return bf16 ? cudaLaunchKernelEx(&cfg, paged_join_kernel<64, true>, p)
                : cudaLaunchKernelEx(&cfg, paged_join_kernel<64, false>, p);
  return bf16 ? cudaLaunchKernelEx(&cfg, paged_join_kernel<128, true>, p)
              : cudaLaunchKernelEx(&cfg, paged_join_kernel<128, false>, p);
}

}  // namespace fa
