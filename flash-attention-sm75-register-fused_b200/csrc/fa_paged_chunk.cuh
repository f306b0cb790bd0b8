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
//   items  (sequence, pair of tiles, KV head, key split), found from the
//          lengths on the device: the grid has room for every pair the packed
//          rows can hold, and a CTA without one leaves at once.  Pairs of a
//          sequence run from its end, the longest causal rows first.
//   pages  16-bit pages: a 128-key tile is a set of TMA boxes of gcd(page, 128)
//          rows, one per lane of the producer warp.  The rows behind the last
//          visible key in its box are stale; V's are set to zero before the
//          tile is released, K's are masked as scores.
//          8-bit pages: three warps read 16-key groups into registers, widen
//          them to f16 (exact) and store them in the swizzled layout the
//          products read.  For bf16 results they also multiply by the row's
//          scale (two f16 roundings, 8 times finer than the result's); for f16
//          results the softmax applies the scales in fp32: K's to the scores,
//          V's to P relative to a power of two that follows the largest scale.
//   joins  With few items the keys are split; partial O and LSE go to the
//          workspace and paged_join_kernel merges them.
#include "fa_paged.h"
#include "fa_paged_dev.cuh"

namespace fa {
namespace {

template <int D, bool k8>
struct ChunkLayout {
  static constexpr int kColBlocks = D / 64;
  static constexpr int kBlockBytes = 128 * 128;
  static constexpr int kTile = 128 * D * 2;
  static constexpr int kSlots = D == 64 ? 8 : (k8 ? 4 : 5);
  static constexpr int kOffQ = 0;
  static constexpr int kOffKV = 2 * kTile;
  static constexpr int kOffScale = kOffKV + kSlots * kTile;
  // scales of tile j at entry j % kScaleRing: K's 128, V's 128, V's maximum per
  // 16 keys.  K_j's slot is free only after the scores of tile
  // j - kSlots / 2 were issued for both groups, i.e. after both finished the
  // softmax of the tile before it, so entry j - kScaleRing is no longer read.
  static constexpr int kScaleRing = D == 64 ? 8 : 4;
  static constexpr int kScaleEntry = (128 + 128 + 8) * 4;
  static_assert(kScaleRing >= kSlots / 2 + 1, "a scale entry outlives its tile");
  static constexpr int kOffBar = kOffScale + (k8 ? kScaleRing * kScaleEntry : 0);
  static constexpr int kBarQ = 0;                       // 2
  static constexpr int kBarFull = 2;                    // kSlots
  static constexpr int kBarEmpty = kBarFull + kSlots;   // kSlots
  static constexpr int kBarS = kBarEmpty + kSlots;      // 2
  static constexpr int kBarP = kBarS + 2;               // 2
  static constexpr int kBarPH = kBarP + 2;              // 2
  static constexpr int kBarO = kBarPH + 2;              // 2
  static constexpr int kBarDrain = kBarO + 2;           // 1
  static constexpr int kBarTail = kBarDrain + 1;        // 1: the V tile with stale rows landed
  static constexpr int kNumBars = kBarTail + 1;
  static constexpr int kOffMisc = kOffBar + 8 * kNumBars;
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

// exp_tile (fa_fwd_sm100.cu) with P multiplied by V's scales: e = 2^(x sl - m)
// is summed as it is, e * vs goes to tensor memory.
template <bool kEmulate, int kPeriod, typename Announce>
__device__ __forceinline__ float exp_tile_scaled(const float (&x)[kBlockN], float sl, float neg_m,
                                                 const float* vs, uint32_t tP, Announce announce) {
  float a0 = 0.f, a1 = 0.f, b0 = 0.f, b1 = 0.f;
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    uint32_t pk[16];
#pragma unroll
    for (int c = 0; c < 16; c += 2) {
      const float4 f = *reinterpret_cast<const float4*>(vs + 32 * h + 2 * c);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int i = 32 * h + 2 * (c + y);
        float e0, e1;
        exp2_pair<kEmulate, kPeriod>(c + y, x[i], x[i + 1], sl, neg_m, e0, e1);
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

// The work item of a CTA.
struct ChunkItem {
  Seq s;
  int b, h, pair, sp;
  int n_kv[2], jb, n_loop;  // key tiles of either query tile, from tile jb
};

// KV: type of the pages (FA_DTYPE_*); QBF16: type of Q and O.
template <int D, int KV, bool QBF16>
__global__ void __launch_bounds__(kThreads, 1) paged_chunk_kernel(const __grid_constant__ ChunkParams p) {
  constexpr bool k8 = KV >= FA_DTYPE_INT8;
  constexpr bool kBf16 = KV == FA_DTYPE_BF16;  // type of the products
  constexpr bool kFold = k8 && QBF16;          // scales go into the widened values
  constexpr bool kScaled = k8 && !QBF16;       // ... are applied by the softmax
  using L = ChunkLayout<D, k8>;
  const PagedAttn& a = p.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  __shared__ long long sh_scan[kThreads / 32];
  __shared__ int sh_item[2];  // sequence, pair (-1: none)
  const uint32_t sbase = ptx::smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 4);
  auto bar = [&](int i) -> uint32_t { return sbase + L::kOffBar + 8u * static_cast<uint32_t>(i); };
  ptx::launch_dependents();

  // ---- which (sequence, pair) is this CTA's?
  const int w = static_cast<int>(blockIdx.x);
  const int slot_id = w / (p.n_splits * a.c.heads);
  {
    auto pairs_of = [&](int b) {
      const Seq s = load_seq(a, b);
      return static_cast<long long>(s.nq) * a.group <= p.skip_rows ? 0 : (s.nq + 2 * p.tq - 1) / (2 * p.tq);
    };
    const int share = (a.r.B + kThreads - 1) / kThreads;
    const int b0 = min(static_cast<int>(threadIdx.x) * share, a.r.B), b1 = min(b0 + share, a.r.B);
    if (threadIdx.x == 0) sh_item[1] = -1;
    long long sum = 0, total;
    for (int b = b0; b < b1; ++b) sum += pairs_of(b);
    long long x = block_scan<kThreads>(sum, sh_scan, &total);
    if (slot_id >= x && slot_id < x + sum)
      for (int b = b0; b < b1; ++b) {
        const int n = pairs_of(b);
        if (slot_id < x + n) {
          sh_item[0] = b;
          sh_item[1] = n - 1 - static_cast<int>(slot_id - x);  // from the sequence's end
          break;
        }
        x += n;
      }
    if (p.fill_outside) {
      const int head = a.r.B > 0 ? min(max(__ldg(a.r.cu), 0), a.r.total) : a.r.total;
      const int tail = a.r.B > 0 ? min(max(__ldg(a.r.cu + a.r.B), head), a.r.total) : a.r.total;
      const int n_out = head + a.r.total - tail;
      for (int y = w; y < n_out; y += static_cast<int>(gridDim.x)) {
        const int t = y < head ? y : tail + y - head;
        for (int i = threadIdx.x; i < a.Hq * D / 2; i += kThreads)
          static_cast<uint32_t*>(a.o)[static_cast<long long>(t) * (a.Hq * D / 2) + i] = 0u;
        if (a.lse != nullptr)
          for (int i = threadIdx.x; i < a.Hq; i += kThreads)
            a.lse[static_cast<long long>(i) * a.r.total + t] = -INFINITY;
      }
    }
    __syncthreads();
  }
  ChunkItem it;
  it.pair = sh_item[1];
  if (it.pair < 0) return;
  it.b = sh_item[0];
  it.h = (w / p.n_splits) % a.c.heads;
  it.sp = w % p.n_splits;
  it.s = load_seq(a, it.b);
  const int tok0 = it.pair * 2 * p.tq;  // first token of tile 0
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int lo = tok0 + g * p.tq;
    const int lim = lo < it.s.nq ? row_limit(a, it.s, min(lo + p.tq, it.s.nq) - 1) : 0;
    it.n_kv[g] = (lim + kBlockN - 1) / kBlockN;
  }
  {
    // the pair's key tiles, in equal parts
    const int n = max(it.n_kv[0], it.n_kv[1]);
    const int tps = (n + p.n_splits - 1) / p.n_splits;
    it.jb = it.sp * tps;
#pragma unroll
    for (int g = 0; g < 2; ++g) it.n_kv[g] = max(min(it.n_kv[g] - it.jb, tps), 0);
    it.n_loop = max(it.n_kv[0], it.n_kv[1]);
  }
  const int n_rows = p.tq * a.group;  // rows of a tile in use

  // ---- set-up
  if (threadIdx.x == 0) {
    const unsigned long long st = *reinterpret_cast<volatile unsigned long long*>(&g_fa_status);
    *abort_flag = ((st >> 32) == p.epoch && (st & 0xffffffffull) != 0ull) ? 1 : 0;
    for (int i = 0; i < L::kNumBars; ++i) {
      const bool all = (i >= L::kBarP && i < L::kBarP + 2) || (i >= L::kBarPH && i < L::kBarPH + 2) ||
                       (k8 && i < 2);
      const bool full = i >= L::kBarFull && i < L::kBarFull + L::kSlots;
      ptx::mbar_init(bar(i), all ? 128u : (k8 && full) ? 8u : 1u);
    }
    ptx::fence_barrier_init();
  }
  __syncthreads();
  if (*abort_flag) return;
  if (warp == kWarpMma) {
    ptx::tmem_alloc(ptx::smem_u32(tmem_slot), L::kTmemCols);
    ptx::tmem_relinquish();
    ptx::tc_fence_before();
  }
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  const WaitCtl wc{abort_flag, p.timeout_ns, p.epoch};
  const int n_items = 2 * it.n_loop;  // K_0 V_0 K_1 V_1 ...

  if (warp >= 8) {
    ptx::setmaxnreg_dec<kRegsOther>();
    if (!k8 && warp == kWarpLoad) {
      // =================================================== TMA producer (16-bit pages)
      const uint64_t pol_q = ptx::policy_evict_first();
      const uint64_t pol_kv = ptx::policy_evict_last();
      if (lane == 0) {
        ptx::prefetch_tmap(&p.tm_q);
        ptx::prefetch_tmap(&p.tm_k);
        ptx::prefetch_tmap(&p.tm_v);
        for (int g = 0; g < 2; ++g) {
          if (it.n_kv[g] == 0) continue;
          ptx::mbar_arrive_expect_tx(bar(L::kBarQ + g), L::kColBlocks * n_rows * 128);
#pragma unroll
          for (int c = 0; c < L::kColBlocks; ++c)
            ptx::tma_load_3d(sbase + L::kOffQ + g * L::kTile + c * L::kBlockBytes, &p.tm_q,
                             bar(L::kBarQ + g), c * 64, it.h * a.group, it.s.c0 + tok0 + g * p.tq,
                             pol_q);
        }
      }
      __syncwarp();
      // lane = column block * 8 + box; a box starts at key tile * 128 + box * box_rows
      const int col = lane >> 3, box = lane & 7;
      const bool issues = col < L::kColBlocks && box * p.box_rows < kBlockN;
      const uint32_t dst_off = col * L::kBlockBytes + box * p.box_rows * 128;
      auto page_at = [&](int tile) {  // page of this lane's box; -1 reads as zeros
        const int pos = tile * kBlockN + box * p.box_rows;
        return issues && pos < it.s.vis ? a.c.lookup(it.b, pos) : -1;
      };
      int next_page = page_at(it.jb), page = -1;
      bool ok = true, tail_used = false;
      int i = 0;
      for (; i < n_items; ++i) {
        const int tile = it.jb + (i >> 1);
        if (!(i & 1)) {
          page = next_page;
          if (i + 2 < n_items) next_page = page_at(tile + 1);
        }
        const int slot = i % L::kSlots;
        if (i >= L::kSlots &&
            !(ok = __all_sync(0xffffffffu, bar_wait(bar(L::kBarEmpty + slot),
                                                    ((i / L::kSlots) - 1) & 1, wc, 1))))
          break;
        // stale V rows of the tile: [r0, r1)
        const int r0 = it.s.vis - tile * kBlockN;
        const int r1 = (r0 + p.box_rows - 1) / p.box_rows * p.box_rows;
        const bool tail = (i & 1) && r0 < kBlockN && r0 != r1;
        const uint32_t full = tail ? bar(L::kBarTail) : bar(L::kBarFull + slot);
        if (lane == 0) ptx::mbar_arrive_expect_tx(full, L::kTile);
        __syncwarp();
        const uint32_t dst = sbase + L::kOffKV + slot * L::kTile;
        if (issues)
          ptx::tma_load_4d(dst + dst_off, (i & 1) ? &p.tm_v : &p.tm_k, full, col * 64,
                      a.c.row_in_page(tile * kBlockN + box * p.box_rows), it.h, page, pol_kv);
        if (tail) {
          tail_used = true;
          if (!(ok = __all_sync(0xffffffffu, bar_wait(bar(L::kBarTail), 0, wc, 7)))) break;
          for (int x = lane; x < (r1 - r0) * 8 * L::kColBlocks; x += 32) {
            const int r = r0 + x / (8 * L::kColBlocks), c = x % (8 * L::kColBlocks);
            *reinterpret_cast<uint4*>(smem + L::kOffKV + slot * L::kTile + (c >> 3) * L::kBlockBytes +
                                      r * 128 + (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          ptx::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(bar(L::kBarFull + slot));
        }
      }
      // every copy started lands before the CTA exits
      for (int r = max(0, i - L::kSlots); r < i; ++r)
        bar_wait(bar(L::kBarFull + r % L::kSlots), (r / L::kSlots) & 1, wc, 2, false);
      if (tail_used && !ok) bar_wait(bar(L::kBarTail), 0, wc, 2, false);
      for (int g = 0; g < 2; ++g)
        if (it.n_kv[g] > 0) bar_wait(bar(L::kBarQ + g), 0, wc, 2, false);
    } else if (k8 && warp != kWarpMma) {
      // =================================================== widening warps (8-bit pages)
      // Groups of 16 keys, 8 per ring item, dealt to warps 8, 10 and 11 in turn.
      // A lane takes 16 values of a row at a time: D / 16 lanes a row.
      constexpr int kLanesRow = D / 16;
      constexpr int kLoads = 16 / (32 / kLanesRow);  // rows of the group per lane
      const int cw = warp == kWarpLoad ? 0 : warp - kWarpLoad - 1;
      const int n_groups = 8 * n_items;
      const int lr = lane / kLanesRow, lx = lane % kLanesRow;
      struct Raw {
        uint4 v[kLoads];
        float sc, sc2;  // lane < 16: scale of row `lane` (kScaled, K items: K's and V's)
      };
      auto lookup = [&](int n) {
        const int pos = (it.jb + (n >> 4)) * kBlockN + 16 * (n & 7);
        return n < n_groups && pos < it.s.vis ? a.c.lookup(it.b, pos) : -1;
      };
      auto load = [&](Raw& r, int n, int page) {
        const int pos = (it.jb + (n >> 4)) * kBlockN + 16 * (n & 7);
        const bool is_v = (n >> 3) & 1;
        const int left = page >= 0 ? it.s.vis - pos : 0;  // rows that exist
        const long long prow = a.c.row_in_page(pos);
        const uint8_t* src = (is_v ? a.c.v : a.c.k) + page * a.c.page_stride + it.h * a.c.head_stride +
                             prow * a.c.row_stride + 16 * lx;
#pragma unroll
        for (int y = 0; y < kLoads; ++y) {
          const int row = y * (32 / kLanesRow) + lr;
          r.v[y] = make_uint4(0u, 0u, 0u, 0u);
          if (row < left) r.v[y] = __ldg(reinterpret_cast<const uint4*>(src + row * a.c.row_stride));
        }
        r.sc = r.sc2 = 0.f;
        if (lane < 16 && lane < left) {
          const long long so = page * a.c.s_page + it.h * a.c.s_head + (prow + lane) * a.c.s_row;
          if constexpr (kFold) {
            r.sc = __ldg((is_v ? a.c.vs : a.c.ks) + so);
          } else if (!is_v) {
            r.sc = __ldg(a.c.ks + so);
            r.sc2 = __ldg(a.c.vs + so);
          }
        }
      };
      auto store = [&](const Raw& r, int n) -> bool {
        const int item = n >> 3, grp = n & 7;
        const int slot = item % L::kSlots;
        if (item >= L::kSlots &&
            !__all_sync(0xffffffffu, bar_wait(bar(L::kBarEmpty + slot), ((item / L::kSlots) - 1) & 1, wc, 1)))
          return false;
        uint8_t* dst = smem + L::kOffKV + slot * L::kTile;
        // f16 products of a scale below 2^-14 would lose its bits, and one above
        // 128 could overflow: such groups multiply in two steps
        bool wide = false;
        if constexpr (kFold)
          wide = __any_sync(0xffffffffu, lane < 16 && (r.sc != 0.f && (r.sc < 6.103515625e-5f || !(r.sc <= 128.f))));
#pragma unroll
        for (int y = 0; y < kLoads; ++y) {
          const int row = y * (32 / kLanesRow) + lr;
          const uint32_t in[4] = {r.v[y].x, r.v[y].y, r.v[y].z, r.v[y].w};
          uint32_t o[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) widen<KV, false>(in[i], o[2 * i], o[2 * i + 1]);
          if constexpr (kFold) {
            const float sc = __shfl_sync(0xffffffffu, r.sc, row);
            __half2 s1, s2;
            if (!wide) {
              s1 = __float2half2_rn(sc);
            } else {
              // sc = m * 2^e, 2^e in f16's range (2^-23 .. 2^7), m in [1, 2) as far as that goes
              const uint32_t eb = min(max(__float_as_uint(sc) & 0x7f800000u, 0x34000000u), 0x43000000u);
              const float e = __uint_as_float(eb), mant = sc / e;
              s1 = __float2half2_rn(mant > 65504.f ? 65504.f : mant);
              s2 = __float2half2_rn(e);
            }
            const __half2 top = __half2half2(__ushort_as_half(0x7bff));  // 65504
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              __half2 x = __hmul2(*reinterpret_cast<__half2*>(&o[i]), s1);
              if (wide) x = __hmax2_nan(__hmin2_nan(__hmul2(x, s2), top), __hneg2(top));
              o[i] = *reinterpret_cast<uint32_t*>(&x);
            }
          }
          // 16 values = 16-byte pieces 2 lx and 2 lx + 1 of the row; the right half
          // of a 128-wide row stores its odd piece first, so that the eight lanes of
          // a row hit eight bank groups
          const int row_t = 16 * grp + row;
          const int cb = D == 128 ? lx >> 2 : 0;
          const int c = (2 * lx) & 7;
          uint8_t* base = dst + cb * L::kBlockBytes + row_t * 128;
          const uint4 lo = make_uint4(o[0], o[1], o[2], o[3]), hi = make_uint4(o[4], o[5], o[6], o[7]);
          const bool odd = cb != 0;
          *reinterpret_cast<uint4*>(base + (((c + (odd ? 1 : 0)) ^ (row_t & 7)) << 4)) = odd ? hi : lo;
          *reinterpret_cast<uint4*>(base + (((c + (odd ? 0 : 1)) ^ (row_t & 7)) << 4)) = odd ? lo : hi;
        }
        if constexpr (kScaled) {
          if (!(item & 1)) {
            float* e = reinterpret_cast<float*>(smem + L::kOffScale + ((item >> 1) % L::kScaleRing) * L::kScaleEntry);
            float mx = r.sc2;
#pragma unroll
            for (int x = 8; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
            if (lane < 16) {
              e[16 * grp + lane] = r.sc;
              e[128 + 16 * grp + lane] = r.sc2;
            }
            if (lane == 0) e[256 + grp] = mx;
          }
        }
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar(L::kBarFull + slot));
        return true;
      };
      // two groups in flight, their pages looked up one step earlier
      Raw ra, rb;
      int n = cw;
      load(ra, n, lookup(n));
      load(rb, n + 3, lookup(n + 3));
      int pa = lookup(n + 6), pb = lookup(n + 9);
      for (; n < n_groups; n += 6) {
        if (!store(ra, n)) break;
        load(ra, n + 6, pa);
        pa = lookup(n + 12);
        if (n + 3 < n_groups && !store(rb, n + 3)) break;
        load(rb, n + 9, pb);
        pb = lookup(n + 15);
      }
    } else if (warp == kWarpMma) {
      // =================================================== MMA issuer (see fa_fwd_kernel)
      constexpr uint32_t fmt = kBf16 ? 1u : 0u;
      constexpr uint32_t idesc_qk = ptx::make_idesc_f16(kBlockM, kBlockN, fmt, 0, 0);
      constexpr uint32_t idesc_pv = ptx::make_idesc_f16(kBlockM, D, fmt, 0, 1);
      const uint64_t k_desc0 = ptx::smem_desc_sw128(sbase + L::kOffKV, 16, 1024);
      const uint64_t v_desc0 = ptx::smem_desc_sw128(sbase + L::kOffKV, L::kBlockBytes, 1024);
      const uint32_t d_hi = static_cast<uint32_t>(k_desc0 >> 32);
      const uint32_t v_hi = static_cast<uint32_t>(v_desc0 >> 32);
      const uint32_t k_lo0 = static_cast<uint32_t>(k_desc0);
      const uint32_t v_lo0 = static_cast<uint32_t>(v_desc0);
      const uint32_t q_lo0 = static_cast<uint32_t>(ptx::smem_desc_sw128(sbase + L::kOffQ, 16, 1024));
      const uint32_t q_lo1 =
          static_cast<uint32_t>(ptx::smem_desc_sw128(sbase + L::kOffQ + L::kTile, 16, 1024));
      constexpr uint32_t kSlotStep = L::kTile >> 4;
      auto issue_s = [&](int g, int ks, uint32_t q_lo) {
        const uint32_t k_lo = k_lo0 + static_cast<uint32_t>(ks) * kSlotStep;
        if (ptx::elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = static_cast<uint32_t>(((kk / 4) * L::kBlockBytes + (kk % 4) * 32) >> 4);
            ptx::mma_ss(tmem + L::tS(g), ptx::make_desc(q_lo + off, d_hi),
                        ptx::make_desc(k_lo + off, d_hi), idesc_qk, kk > 0 ? 1u : 0u);
          }
          ptx::mma_commit(bar(L::kBarS + g));
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
                        ptx::make_desc(v_lo + kk * 128u, v_hi), idesc_pv, (!first || kk > 0) ? 1u : 0u);
        }
        __syncwarp();
        if (!wait(bar(L::kBarP + g), ph, 13 + 3 * g)) return false;
        ptx::tc_fence_after();
        if (ptx::elect_one()) {
#pragma unroll
          for (int kk = 2 * kPEarlyQuarters; kk < kBlockN / 16; ++kk)
            ptx::mma_ts(tmem + L::tO(g), tmem + L::tP(g) + kk * 8,
                        ptx::make_desc(v_lo + kk * 128u, v_hi), idesc_pv, 1u);
          ptx::mma_commit(bar(L::kBarO + g));
        }
        __syncwarp();
        return true;
      };
      const int n0 = it.n_kv[0], n1 = it.n_kv[1];
      bool ok = true;
      int ks = 0;
      uint32_t kph = 0;
      auto adv = [](int& sl, uint32_t& ph) {
        if (++sl == L::kSlots) {
          sl = 0;
          ph ^= 1u;
        }
      };
      if (it.n_loop > 0) {
        if (n0 > 0) ok = wait(bar(L::kBarQ), 0, 10);
        if (ok && n1 > 0) ok = wait(bar(L::kBarQ + 1), 0, 10);
        if (ok) ok = wait(bar(L::kBarFull), 0, 11);
        if (ok) {
          ptx::tc_fence_after();
          if (n0 > 0) issue_s(0, ks, q_lo0);
          if (n1 > 0) issue_s(1, ks, q_lo1);
          commit(bar(L::kBarEmpty + ks));
        }
      }
      for (int j = 0; ok && j < it.n_loop; ++j) {
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
          if (!(ok = issue_pv(0, vs, j == 0, j & 1))) break;
          if (next0) {
            issue_s(0, ns, q_lo0);
            if (!next1) commit(bar(L::kBarEmpty + ns));
          }
        }
        if (j < n1) {
          if (!(ok = issue_pv(1, vs, j == 0, j & 1))) break;
        }
        commit(bar(L::kBarEmpty + vs));
        if (next1) {
          issue_s(1, ns, q_lo1);
          commit(bar(L::kBarEmpty + ns));
        }
      }
      // all products complete before tensor memory is released
      commit(bar(L::kBarDrain));
      bar_wait(bar(L::kBarDrain), 0, wc, 19, false);
      __syncwarp();
    }
  } else {
    // ===================================================== softmax groups
    ptx::setmaxnreg_inc<kRegsSoftmax>();
    const int g = warp >> 2;
    const int wq = warp & 3;
    const int r = wq * 32 + lane;  // row of the tile == TMEM lane
    const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t tS = tmem + lane_off + L::tS(g);
    const uint32_t tP = tmem + lane_off + L::tP(g);
    const uint32_t tO = tmem + lane_off + L::tO(g);
    const int n_tiles = g ? it.n_kv[1] : it.n_kv[0];
    const int tok_lo = tok0 + g * p.tq;
    const int tok = tok_lo + r / a.group;      // token of the sequence
    const int hq = it.h * a.group + r % a.group;
    const bool row_ok = r < n_rows && tok < it.s.nq;
    float sl = a.scale_log2;
    bool ok = true;
    if constexpr (k8) {
      // Q as f16 in the swizzled layout, one row per thread; a bf16 row is
      // scaled by a power of two into f16's range, undone in sl
      if (n_tiles > 0) {
        uint4 q[D / 8];
#pragma unroll
        for (int c = 0; c < D / 8; ++c) q[c] = make_uint4(0u, 0u, 0u, 0u);
        if (row_ok) {
          const uint4* src = reinterpret_cast<const uint4*>(
              a.q + static_cast<long long>(it.s.c0 + tok) * a.q_token + hq * a.q_head);
#pragma unroll
          for (int c = 0; c < D / 8; ++c) q[c] = __ldg(src + c);
        }
        if constexpr (QBF16) {
          auto f2 = [](uint32_t u) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u)); };
          float mx = 0.f;
#pragma unroll
          for (int c = 0; c < D / 8; ++c) {
            const uint32_t u[4] = {q[c].x, q[c].y, q[c].z, q[c].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, fmaxf(fabsf(f2(u[i]).x), fabsf(f2(u[i]).y)));
          }
          const uint32_t e = __float_as_uint(mx) & 0x7f800000u;
          const bool plain = e == 0u || e >= 0x7e800000u;
          const float inv = plain ? 1.f : __uint_as_float(0x7f000000u - e);
          if (!plain) sl *= __uint_as_float(e);
#pragma unroll
          for (int c = 0; c < D / 8; ++c) {
            uint32_t* u = reinterpret_cast<uint32_t*>(&q[c]);
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = pack2<false>(f2(u[i]).x * inv, f2(u[i]).y * inv);
          }
        }
        uint8_t* dst = smem + L::kOffQ + g * L::kTile + r * 128;
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
          *reinterpret_cast<uint4*>(dst + (c >> 3) * L::kBlockBytes + (((c & 7) ^ (r & 7)) << 4)) = q[c];
        ptx::fence_proxy_async_smem();
        ptx::mbar_arrive(bar(L::kBarQ + g));
      }
    }
    // key limit of this row, and the smallest of the tile's rows
    const int row_end = row_limit(a, it.s, tok);
    const int tile_end = row_limit(a, it.s, tok_lo);

    constexpr float kGrow = kScaled ? 8.0f : kRescaleThreshold;
    float m = -INFINITY;  // running max of the scaled scores (log2 units)
    float l = 0.f;        // running sum of exp2(s - m) (kScaled: times 2^-lv)
    float lv = 0.f;       // kScaled: log2 of the power of two V's scales are relative to
    for (int j = 0; ok && j < n_tiles; ++j) {
      ok = __all_sync(0xffffffffu, bar_wait(bar(L::kBarS + g), j & 1, wc, 20 + g));
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
      const float* entry = reinterpret_cast<const float*>(
          smem + L::kOffScale + (k8 ? (j % L::kScaleRing) * L::kScaleEntry : 0));
      float lv_new = lv;
      if constexpr (kScaled) {
#pragma unroll
        for (int c = 0; c < kBlockN; c += 4) {
          const float4 f = *reinterpret_cast<const float4*>(entry + c);
          ptx::fmul2(x[c], x[c + 1], x[c], x[c + 1], f.x, f.y);
          ptx::fmul2(x[c + 2], x[c + 3], x[c + 2], x[c + 3], f.z, f.w);
        }
        // P * vs stays below 2^8 * 2^6: lv follows V's largest scale (the same for
        // all threads); the first tile sets it
        const float4 f0 = *reinterpret_cast<const float4*>(entry + 256);
        const float4 f1 = *reinterpret_cast<const float4*>(entry + 260);
        const float vm = fmaxf(fmaxf(fmaxf(f0.x, f0.y), fmaxf(f0.z, f0.w)),
                               fmaxf(fmaxf(f1.x, f1.y), fmaxf(f1.z, f1.w)));
        const float e = static_cast<float>(static_cast<int>(__float_as_uint(vm) >> 23) - 127);
        if (j == 0 || e > lv + 5.f) lv_new = fmaxf(fminf(e, 100.f), -50.f);
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
      const bool grow = m_new > m + kGrow;
      if (j == 0) {
        m = m_new;
        lv = lv_new;
      } else {
        if (__any_sync(0xffffffffu, grow) || (kScaled && lv_new != lv)) {
          float alpha = grow ? ptx::ex2_approx(m - m_new) : 1.0f;
          if constexpr (kScaled) alpha *= ptx::ex2_approx(lv - lv_new);
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
          l *= alpha;
          lv = lv_new;
        }
        if (grow) m = m_new;
      }
      const float neg_m = ((m == -INFINITY) ? 0.f : -m) - lv;
      const uint32_t half_bar = bar(L::kBarPH + g);
      auto announce = [half_bar] { ptx::mbar_arrive(half_bar); };
      float tile_sum;
      if constexpr (kScaled) {
        tile_sum = masked ? exp_tile_scaled<false, kEmuPeriod>(x, sl_eff, neg_m, entry + 128, tP, announce)
                          : exp_tile_scaled<true, kPairEmuPeriod<D>>(x, sl_eff, neg_m, entry + 128, tP, announce);
      } else {
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
    const long long n_all = static_cast<long long>(a.r.total) * a.Hq;
    const bool partial = p.n_splits > 1;
    float* lse_dst = partial ? p.ws_lse + it.sp * n_all + row_id
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
      if (ok) ok = __all_sync(0xffffffffu, bar_wait(bar(L::kBarO + g), (n_tiles - 1) & 1, wc, 22 + g));
      if (ok) {
        ptx::tc_fence_after();
        const float inv_l = (l > 0.f) ? 1.0f / l : (l == 0.f ? 0.f : l);  // (a NaN stays one)
        const float m_use = (m == -INFINITY) ? 0.f : m;
        const float lse_row =
            l == 0.f ? -INFINITY : (m_use + lv + __log2f(l)) * 0.69314718055994530942f;
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
            float4* dst = reinterpret_cast<float4*>(p.ws_o + (it.sp * n_all + row_id) * D + c * 32);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              dst[i] = make_float4(__uint_as_float(o[4 * i]) * inv_l, __uint_as_float(o[4 * i + 1]) * inv_l,
                                   __uint_as_float(o[4 * i + 2]) * inv_l, __uint_as_float(o[4 * i + 3]) * inv_l);
          }
        }
        if (row_ok && lse_dst) *lse_dst = lse_row;
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

// Joins the key splits of the chunk kernel's rows, one warp per (token, query
// head): LSE = log sum_s exp(LSE_s), O = sum_s exp(LSE_s - LSE) O_s.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ ChunkParams p) {
  const PagedAttn& a = p.a;
  constexpr int E = D / 32;
  __shared__ int sh_mine[8];  // per row of the block: a sequence of the chunk kernel holds its token
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long n_all = static_cast<long long>(a.r.total) * a.Hq;
  const long long row0 = static_cast<long long>(blockIdx.x) * 8;
  if (threadIdx.x < 8) sh_mine[threadIdx.x] = 0;
  __syncthreads();
  for (int b = threadIdx.x; b < a.r.B; b += 256) {
    const Seq s = load_seq(a, b);
    if (static_cast<long long>(s.nq) * a.group <= p.skip_rows) continue;
    const long long lo = max(static_cast<long long>(s.c0) * a.Hq, row0);
    const long long hi = min((static_cast<long long>(s.c0) + s.nq) * a.Hq, row0 + 8);
    for (long long x = lo; x < hi; ++x) sh_mine[x - row0] = 1;
  }
  __syncthreads();
  ptx::grid_dep_wait();
  const long long row = row0 + warp;
  if (row >= n_all || !sh_mine[warp]) return;
  const float ls = lane < p.n_splits ? __ldcg(p.ws_lse + lane * n_all + row) : -INFINITY;
  float mx = ls;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  float wgt = ls == -INFINITY ? 0.f : expf(ls - mx);  // (a NaN stays one)
  float sum = wgt;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  float acc[E] = {};
  for (int s = 0; s < p.n_splits; ++s) {
    const float f = __shfl_sync(0xffffffffu, wgt, s);
    if (f == 0.f) continue;
    const float* src = p.ws_o + (s * n_all + row) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(f, __ldcg(src + e), acc[e]);
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.o) + row * D + lane * E);
#pragma unroll
  for (int e = 0; e < E / 2; ++e) dst[e] = pack2<BF16>(acc[2 * e] * inv, acc[2 * e + 1] * inv);
  if (lane == 0 && a.lse != nullptr)
    a.lse[row % a.Hq * a.r.total + row / a.Hq] = sum == 0.f ? -INFINITY : mx + logf(sum);
}

template <int D, int KV, bool QBF16>
cudaError_t launch_chunk_impl(const ChunkParams& p, int grid, cudaStream_t stream) {
  auto kern = paged_chunk_kernel<D, KV, QBF16>;
  constexpr int kSmem = ChunkLayout<D, (KV >= FA_DTYPE_INT8)>::kDynBytes;
  static int attr_done[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_done[dev]) {
    // the setmaxnreg split is only safe with exactly kLaunchRegs per thread
    cudaFuncAttributes fa{};
    cudaError_t e = cudaFuncGetAttributes(&fa, kern);
    if (e != cudaSuccess) return e;
    if (fa.numRegs != kLaunchRegs || fa.maxThreadsPerBlock < kThreads)
      return cudaErrorInvalidConfiguration;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_done[dev] = 1;
  }
  kern<<<grid, kThreads, kSmem, stream>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.n_splits == 1) return e;
  cudaLaunchConfig_t cfg{};
  const long long n_all = static_cast<long long>(p.a.r.total) * p.a.Hq;
  cfg.gridDim = dim3(static_cast<unsigned>((n_all + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_join_kernel<D, QBF16>, p);
}

template <int D>
cudaError_t launch_chunk_d(const ChunkParams& p, int kv, bool bf16, int grid, cudaStream_t s) {
  switch (kv) {
    case FA_DTYPE_INT8:
      return bf16 ? launch_chunk_impl<D, FA_DTYPE_INT8, true>(p, grid, s)
                  : launch_chunk_impl<D, FA_DTYPE_INT8, false>(p, grid, s);
    case FA_DTYPE_E4M3:
      return bf16 ? launch_chunk_impl<D, FA_DTYPE_E4M3, true>(p, grid, s)
                  : launch_chunk_impl<D, FA_DTYPE_E4M3, false>(p, grid, s);
    case FA_DTYPE_BF16: return launch_chunk_impl<D, FA_DTYPE_BF16, true>(p, grid, s);
    default: return launch_chunk_impl<D, FA_DTYPE_F16, false>(p, grid, s);
  }
}

}  // namespace

cudaError_t launch_paged_chunk(const ChunkParams& p, int head_dim, int kv, bool bf16, int grid,
                               cudaStream_t stream) {
  return head_dim == 64 ? launch_chunk_d<64>(p, kv, bf16, grid, stream)
                        : launch_chunk_d<128>(p, kv, bf16, grid, stream);
}

}  // namespace fa
