// Attention weight that cached keys receive from chunks of new tokens (more query
// rows per KV head than fa_paged_weights.cu streams).  Included by fa_paged_prefix.cu;
// fa_device.cuh has the bounded mbarrier waits and the device status word.
//
//   w_j = sum_i 2^(s'_ij - L'_i)    s' = scale log2(e) q_i . k_j,  L' = log2(e) LSE_i
//
// The scores are computed transposed, S^T = K Q^T on the tensor cores: keys on the rows of
// the product, so that a thread owns a key, adds the terms of all query rows in a register,
// and nothing is exchanged between threads.  A CTA takes two tiles of 128 keys of one head,
// kept in shared memory (8-bit ones widened once, exactly, to the queries' type; the key's
// scale goes into its thread's factor), and walks the query tiles that see any of them:
//
//   warps 0-15 load the keys, then the exponentials and sums: two threads per key, each
//              for half of a tile's rows (four warps per scheduler: with two, their
//              instructions' latency shows, 239 us instead of 216)
//   warp 16    TMA producer of the query tiles (128 / G tokens x the G heads of the group)
//   warp 17    tcgen05 issuer: S^T of tile t, two of four 128-column accumulators
//   warp 18    per row of a tile, -L' and its key limit, from LSE and the lengths
//
// With few key tiles a cluster of CTAs shares the query tiles of one, and its first CTA
// adds the others' sums in order: no atomics, so equal calls give equal bits.
//
// Bound by the exponentials: 128 x 256 of them take the special-function unit 2048 cycles,
// the two products about 1100.  kFmaPairs of 16 pairs go to the FMA pipe instead (0 / 2 / 4
// / 6 of 16: 239 / 226 / 216 / 235 us for 2 x 1024 tokens over 8192 keys, bf16, d = 128, GQA
// 4).  Now 201 to 207 us there (8-bit pages 201): the unit is busy for 54 %, the issue slots for 55 %;
// what is left is the latency between a tile's arrival and its last sum, and that 512 equal CTAs
// take four rounds on 148 SMs for 3.46 rounds of work.  CTAs that walk several key
// blocks, with the next one's keys loaded by a warp of their own, took as long (the
// registers that this takes spill), and so did two CTAs of one key tile per SM.
// The grid has a CTA for every 256 keys that the bounds allow every sequence, whose shared memory
// leaves room for one on an SM; those without work leave at once, but are placed: 1024
// tokens beside 31 single ones, all over 8192 keys, take 242 us, 103 and 83 by themselves.
#include "fa_paged.h"
#include "fa_paged_dev.cuh"

namespace fa {
namespace {
namespace pwc {

constexpr int kThreads = 608;
constexpr int kKeys = paged_weights_chunk_keys();  // of a CTA
constexpr int kExps = 512;   // threads of the exponentials: two per key, for half of a tile's rows each
constexpr int kWarpTma = 16, kWarpMma = 17, kWarpRows = 18;
constexpr int kRowRing = 4;
constexpr int kMaxSplit = 8;
constexpr int kFmaPairs = 4;  // of 16 pairs of exponentials, on the FMA pipe

// (y0, y1) = 2^t for two lanes on the FMA pipe, t in [-126, 127] (clamped): 2^t = 2^n
// 2^f with n the nearest integer, and 2^f a polynomial of degree 5, fitted here by a Remez
// exchange for the least relative error on [-1/2, 1/2] (7.5e-8; 2.1e-7 evaluated in fp32,
// as good as the special-function unit).
__device__ __forceinline__ void exp2_fma2(float& y0, float& y1, float t0, float t1) {
  constexpr float kRound = 12582912.0f;  // 1.5 * 2^23
  constexpr float c0 = 1.0000001192092896f, c1 = 0.6931469440460205f, c2 = 0.24022120237350464f,
                  c3 = 0.05550713092088699f, c4 = 0.009675540961325169f, c5 = 0.0013276472454890609f;
  t0 = fminf(fmaxf(t0, -126.0f), 127.0f);
  t1 = fminf(fmaxf(t1, -126.0f), 127.0f);
  float j0, j1, n0, n1, f0, f1, p0, p1;
  ptx::fadd2(j0, j1, t0, t1, kRound, kRound);
  ptx::fadd2(n0, n1, j0, j1, -kRound, -kRound);
  ptx::ffma2(f0, f1, n0, n1, -1.0f, -1.0f, t0, t1);
  ptx::ffma2(p0, p1, c5, c5, f0, f1, c4, c4);
  ptx::ffma2(p0, p1, p0, p1, f0, f1, c3, c3);
  ptx::ffma2(p0, p1, p0, p1, f0, f1, c2, c2);
  ptx::ffma2(p0, p1, p0, p1, f0, f1, c1, c1);
  ptx::ffma2(p0, p1, p0, p1, f0, f1, c0, c0);
  y0 = __uint_as_float(__float_as_uint(p0) + (__float_as_uint(j0) << 23));
  y1 = __uint_as_float(__float_as_uint(p1) + (__float_as_uint(j1) << 23));
}

template <int D>
struct Smem {
  static constexpr int kColBlocks = D / 64;
  static constexpr int kTile = 128 * D * 2;
  static constexpr int kStages = 4;                  // query tiles
  static constexpr int kOffK = 0;
  static constexpr int kOffQ = 2 * kTile;
  static constexpr int kOffRows = kOffQ + kStages * kTile;  // kRowRing x (-L'[128], limit[128])
  static constexpr int kOffRaw = kOffRows + kRowRing * 1024;  // kRowRing x LSE[128]
  static constexpr int kOffSums = kOffRaw + kRowRing * 512;
  static constexpr int kOffBar = kOffSums + 4 * kExps;
  static constexpr int kBarK = 0;
  static constexpr int kBarQFull = 1;
  static constexpr int kBarQEmpty = kBarQFull + kStages;
  static constexpr int kBarRFull = kBarQEmpty + kStages;
  static constexpr int kBarREmpty = kBarRFull + kRowRing;
  static constexpr int kBarSFull = kBarREmpty + kRowRing;   // 4: key tile + 2 (accumulator)
  static constexpr int kBarSEmpty = kBarSFull + 4;          // 4
  static constexpr int kBarDrain = kBarSEmpty + 4;
  static constexpr int kNumBars = kBarDrain + 1;
  static constexpr int kOffMin = kOffBar + 8 * kNumBars;    // kRowRing ints: least limit of a tile
  static constexpr int kOffPage = (kOffMin + 4 * kRowRing + 7) / 8 * 8;  // 16 row offsets, 16 scale offsets
  static constexpr int kOffMisc = kOffPage + 256;
  static constexpr int kBytes = kOffMisc + 16 + 1024;       // (aligned to 1024)
  static_assert(kBytes <= 227 * 1024, "shared memory budget");
};

template <int D, int KV, bool QBF16>
__global__ void __launch_bounds__(kThreads, 1) paged_weights_chunk_kernel(const __grid_constant__ WeightsChunkParams p) {
  using L = Smem<D>;
  constexpr bool k8 = KV >= FA_DTYPE_INT8;
  constexpr int kPieces = (k8 ? D : 2 * D) / 16;  // of a key row in the pages
  const PagedAttn& a = p.w.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                   ~static_cast<uintptr_t>(1023));
  const uint32_t sbase = ptx::smem_u32(smem);
  const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;
  auto bar = [&](int i) -> uint32_t { return sbase + L::kOffBar + 8u * static_cast<uint32_t>(i); };

  // ---- the CTA's keys, and the query tiles that see any of them
  const int split = p.split, rank = static_cast<int>(blockIdx.x) % split;
  const int item = static_cast<int>(blockIdx.x) / split;
  const int h = item / p.n_blocks % a.c.heads, b = item / p.n_blocks / a.c.heads;
  const int key0 = item % p.n_blocks * kKeys;
  const Seq s = load_seq(a, b);
  // (the same for all CTAs of a cluster)
  if (key0 >= s.nk || static_cast<long long>(s.nq) * a.group <= p.skip_rows) return;
  int first = 0, n_tiles = 0;
  if (key0 < s.vis) {
    if (a.causal != FA_CAUSAL_NONE) first = max(key0 - s.off, 0) / p.tq;
    n_tiles = (s.nq + p.tq - 1) / p.tq - first;
  }
  const int mine = n_tiles > rank ? (n_tiles - rank + split - 1) / split : 0;  // tiles first + rank + t split
  const int n_rows = p.tq * a.group;
  // the earlier sum of key key0 + tid (0: it has none)
  float* const dst = p.w.w + b * p.w.w_seq + h * p.w.w_head + key0 + tid;
  const bool writes = rank == 0 && tid < kKeys && key0 + tid < s.nk;
  float old = 0.f;
  if (writes && p.w.mode != FA_WEIGHTS_SET &&
      (p.w.mode == FA_WEIGHTS_ADD || key0 + tid < min(__ldg(a.r.lens + b), 3 << 29) - s.n))
    old = *dst;

  // ---- set-up
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc);
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc + 4);
  int dead = 0;  // this launch failed elsewhere
  if (tid == 0) {
    const unsigned long long st = *reinterpret_cast<volatile unsigned long long*>(&g_fa_status);
    dead = ((st >> 32) == p.epoch && (st & 0xffffffffull) != 0ull) ? 1 : 0;
    *abort_flag = 0;
    for (int i = 0; i < L::kNumBars; ++i) {
      const bool exps = i == L::kBarK || (i >= L::kBarREmpty && i < L::kBarSFull) || (i >= L::kBarSEmpty && i < L::kBarDrain);
      const unsigned n = i >= L::kBarSEmpty ? 256u : kExps;  // of a key tile, or of both
      ptx::mbar_init(bar(i), exps ? n : i >= L::kBarRFull && i < L::kBarREmpty ? 32u : 1u);
    }
    ptx::fence_barrier_init();
  }
  if (tid < kKeys / 16) {
    // pages of the 16-key groups
    const int pos = key0 + 16 * tid;
    const int page = pos < s.vis ? a.c.lookup(b, pos) : -1;
    const int row = a.c.row_in_page(pos);
    long long* const off = reinterpret_cast<long long*>(smem + L::kOffPage);
    off[tid] = page < 0 ? -1 : page * a.c.page_stride + row * a.c.row_stride + h * a.c.head_stride;
    off[kKeys / 16 + tid] = page < 0 ? 0 : page * a.c.s_page + row * a.c.s_row + h * a.c.s_head;
  }
  // rows of a query tile that no box fills
  if (n_rows < 128)
    for (int i = tid; i < L::kStages * L::kColBlocks * (128 - n_rows) * 8; i += kThreads) {
      const int r = n_rows + i / 8 % (128 - n_rows), blk = i / 8 / (128 - n_rows);
      *reinterpret_cast<uint4*>(smem + L::kOffQ + blk * 16384 + r * 128 + (i % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
  ptx::fence_proxy_async_smem();
  dead = __syncthreads_or(dead);
  if (warp == kWarpMma) {
    ptx::tmem_alloc(ptx::smem_u32(tmem_slot), 512);
    ptx::tmem_relinquish();
    ptx::tc_fence_before();
  }
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  const WaitCtl wc{abort_flag, p.timeout_ns, p.epoch};
  const int n_loop = dead ? 0 : mine;
  float total = 0.f;

  if (warp == kWarpTma) {
    const uint64_t policy = ptx::policy_evict_last();
    int t = 0;
    for (; t < n_loop; ++t) {
      const int st = t % L::kStages;
      if (t >= L::kStages &&
          !__all_sync(0xffffffffu, bar_wait(bar(L::kBarQEmpty + st), ((t / L::kStages) - 1) & 1, wc, 60)))
        break;
      if (lane == 0) {
        ptx::mbar_arrive_expect_tx(bar(L::kBarQFull + st), L::kColBlocks * n_rows * 128);
#pragma unroll
        for (int c = 0; c < L::kColBlocks; ++c)
          ptx::tma_load_3d(sbase + L::kOffQ + st * L::kTile + c * 16384, &p.tm_q, bar(L::kBarQFull + st), c * 64,
                           h * a.group, s.c0 + (first + rank + t * split) * p.tq, policy);
      }
      __syncwarp();
    }
    // every copy started lands before the CTA exits
    for (int r = t - 1; r >= 0 && r >= t - L::kStages; --r)
      bar_wait(bar(L::kBarQFull + r % L::kStages), (r / L::kStages) & 1, wc, 61, false);
  } else if (warp == kWarpMma) {
    constexpr uint32_t idesc = ptx::make_idesc_f16(128, 128, QBF16 ? 1u : 0u, 0, 0);
    const uint64_t k_desc = ptx::smem_desc_sw128(sbase + L::kOffK, 16, 1024 * L::kColBlocks);
    const uint64_t q_desc = ptx::smem_desc_sw128(sbase + L::kOffQ, 16, 1024);
    const uint32_t k_hi = static_cast<uint32_t>(k_desc >> 32), q_hi = static_cast<uint32_t>(q_desc >> 32);
    const uint32_t k_lo = static_cast<uint32_t>(k_desc), q_lo0 = static_cast<uint32_t>(q_desc);
    auto wait = [&](int i, uint32_t ph, int site) { return __all_sync(0xffffffffu, bar_wait(bar(i), ph, wc, site)); };
    bool ok = n_loop == 0 || wait(L::kBarK, 0, 62);
    for (int t = 0; ok && t < n_loop; ++t) {
      const int st = t % L::kStages, acc = t & 1;
      if (!(ok = wait(L::kBarQFull + st, (t / L::kStages) & 1, 63))) break;
      const uint32_t q_lo = q_lo0 + static_cast<uint32_t>(st * L::kTile >> 4);
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        if (t >= 2 && !(ok = wait(L::kBarSEmpty + g + 2 * acc, ((t >> 1) - 1) & 1, 64))) break;
        ptx::tc_fence_after();
        const uint32_t kg_lo = k_lo + static_cast<uint32_t>(g * L::kTile >> 4);
        if (ptx::elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            ptx::mma_ss(tmem + (g + 2 * acc) * 128,
                        ptx::make_desc(kg_lo + (((kk / 4) * 1024 + (kk % 4) * 32) >> 4), k_hi),
                        ptx::make_desc(q_lo + (((kk / 4) * 16384 + (kk % 4) * 32) >> 4), q_hi), idesc, kk > 0 ? 1u : 0u);
          ptx::mma_commit(bar(L::kBarSFull + g + 2 * acc));
          if (g == 1) ptx::mma_commit(bar(L::kBarQEmpty + st));
        }
        __syncwarp();
      }
    }
    // all products complete before tensor memory is released
    if (ptx::elect_one()) ptx::mma_commit(bar(L::kBarDrain));
    __syncwarp();
    bar_wait(bar(L::kBarDrain), 0, wc, 65, false);
    __syncwarp();
  } else if (warp == kWarpRows) {
    // This lane's four rows of every tile.  (A single warp must be done with a tile in the
    // time of its exponentials: with the divisions in the loop it took 4000 cycles a
    // tile, and the kernel 245 us.)
    int dt[4];           // token in the tile
    const float* src[4]; // LSE of the sequence's token dt
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int r = lane + 32 * y;
      dt[y] = r < n_rows ? r / a.group : 1 << 29;  // (no such token)
      src[y] = a.lse + static_cast<long long>(h * a.group + (r < n_rows ? r % a.group : 0)) * a.r.total + s.c0 +
               (r < n_rows ? dt[y] : 0);
    }
    // LSE of the next tiles is on its way (each lane reads back what it copied itself)
    const uint32_t raw = sbase + L::kOffRaw + 4 * lane;
    auto fetch = [&](int t) {
      if (t < n_loop) {
        const int tok0 = (first + rank + t * split) * p.tq;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const bool have = tok0 + dt[y] < s.nq;
          ptx::cp_async4(raw + (t % kRowRing) * 512 + 128 * y, have ? src[y] + tok0 : a.lse, have);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int t = 0; t < kRowRing - 1; ++t) fetch(t);
    for (int t = 0; t < n_loop; ++t) {
      const int e = t % kRowRing;
      const int tok0 = (first + rank + t * split) * p.tq;
      fetch(t + kRowRing - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(kRowRing - 1) : "memory");
      float l[4];
      int lim[4], least = 0x7fffffff;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int tok = tok0 + dt[y];
        l[y] = *reinterpret_cast<const volatile float*>(smem + L::kOffRaw + e * 512 + 4 * (lane + 32 * y));
        if (tok >= s.nq) l[y] = -INFINITY;
        lim[y] = l[y] == -INFINITY ? 0 : row_limit(a, s, tok);
        // (columns past n_rows are zeros; a NaN makes the tile a masked one too, for the FMA
        // pipe's exponential does not pass it on)
        if (dt[y] < 1 << 29) least = min(least, l[y] == l[y] ? lim[y] : 0);
        // (a row that adds nothing: 2^-inf)
        l[y] = l[y] == -INFINITY ? l[y] : l[y] * -1.4426950408889634f;
      }
      least = __reduce_min_sync(0xffffffffu, least);
      if (t >= kRowRing &&
          !__all_sync(0xffffffffu, bar_wait(bar(L::kBarREmpty + e), ((t / kRowRing) - 1) & 1, wc, 66)))
        break;
      float* const row = reinterpret_cast<float*>(smem + L::kOffRows + e * 1024);
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        row[lane + 32 * y] = l[y];
        reinterpret_cast<int*>(row)[128 + lane + 32 * y] = lim[y];
      }
      if (lane == 0) reinterpret_cast<int*>(smem + L::kOffMin)[e] = least;
      __syncwarp();
      ptx::mbar_arrive(bar(L::kBarRFull + e));
    }
    ptx::cp_async_wait_all();
  } else {
    // ---- the keys, in the products' layout: 8 rows x 128 bytes of one half, then of the other
    const long long* const off = reinterpret_cast<const long long*>(smem + L::kOffPage);
    float factor = a.scale_log2;
    if (n_loop > 0) {
      // (all loads before the first store)
      constexpr int kEach = kKeys * kPieces / kExps;
      uint4 x[kEach];
#pragma unroll
      for (int y = 0; y < kEach; ++y) {
        const int i = tid + y * kExps, r = i / kPieces, c = i % kPieces;
        const long long o = off[r >> 4];
        x[y] = make_uint4(0u, 0u, 0u, 0u);
        if (o >= 0 && key0 + r < s.vis) x[y] = __ldg(reinterpret_cast<const uint4*>(a.c.k + o + (r & 15) * a.c.row_stride) + c);
      }
#pragma unroll
      for (int y = 0; y < kEach; ++y) {
        const int i = tid + y * kExps, r = i / kPieces, c = i % kPieces;
        uint8_t* const row = smem + L::kOffK + (r >> 3) * (1024 * L::kColBlocks) + (r & 7) * 128;
        auto put = [&](int piece, const uint4& v) {  // 16-byte piece of the 16-bit row
          *reinterpret_cast<uint4*>(row + (piece >> 3) * 1024 + (((piece & 7) ^ (r & 7)) << 4)) = v;
        };
        if constexpr (k8) {
          const uint32_t in[4] = {x[y].x, x[y].y, x[y].z, x[y].w};
          uint32_t w[8];
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            widen<KV, false>(in[z], w[2 * z], w[2 * z + 1]);
            if constexpr (QBF16) {
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float2 f = __half22float2(*reinterpret_cast<__half2*>(&w[2 * z + e]));
                w[2 * z + e] = pack2<true>(f.x, f.y);
              }
            }
          }
          put(2 * c, make_uint4(w[0], w[1], w[2], w[3]));
          put(2 * c + 1, make_uint4(w[4], w[5], w[6], w[7]));
        } else {
          put(c, x[y]);
        }
      }
      if constexpr (k8) {
        const int r = tid % kKeys;
        const bool held = off[r >> 4] >= 0 && key0 + r < s.vis;
        factor *= held ? __ldg(a.c.ks + off[kKeys / 16 + (r >> 4)] + (r & 15) * a.c.s_row) : 0.f;
      }
      ptx::fence_proxy_async_smem();
      ptx::mbar_arrive(bar(L::kBarK));
    }
    // ---- exponentials and sums of key key0 + tid % 256, rows 64 (tid / 256) .. of every tile
    const int g = (warp >> 2) & 1, col0 = (warp >> 3) * 64;  // key tile, rows
    const uint32_t tS = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + g * 128 + col0;
    const int key = key0 + tid % kKeys, tile_end = key0 + 128 * (g + 1);
    for (int t = 0; t < n_loop; ++t) {
      const int e = t % kRowRing, acc = t & 1;
      if (!__all_sync(0xffffffffu, bar_wait(bar(L::kBarRFull + e), (t / kRowRing) & 1, wc, 67))) break;
      if (!__all_sync(0xffffffffu, bar_wait(bar(L::kBarSFull + g + 2 * acc), (t >> 1) & 1, wc, 68))) break;
      ptx::tc_fence_after();
      const float* const row = reinterpret_cast<const float*>(smem + L::kOffRows + e * 1024);
      const bool masked = reinterpret_cast<const volatile int*>(smem + L::kOffMin)[e] < tile_end;
      float a0 = 0.f, a1 = 0.f, b0 = 0.f, b1 = 0.f;
      auto half = [&](const uint32_t (&u)[32], int c0) {
        if (!masked && c0 + 32 <= n_rows) {
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const float4 l = *reinterpret_cast<const float4*>(row + c0 + c);
            float t0, t1, t2, t3;
            ptx::ffma2(t0, t1, __uint_as_float(u[c]), __uint_as_float(u[c + 1]), factor, factor, l.x, l.y);
            ptx::ffma2(t2, t3, __uint_as_float(u[c + 2]), __uint_as_float(u[c + 3]), factor, factor, l.z, l.w);
            if ((c / 4 * kFmaPairs) % 8 < kFmaPairs) {  // (spread evenly)
              exp2_fma2(t0, t1, t0, t1);
            } else {
              t0 = ptx::ex2_approx(t0);
              t1 = ptx::ex2_approx(t1);
            }
            t2 = ptx::ex2_approx(t2);
            t3 = ptx::ex2_approx(t3);
            ptx::fadd2(a0, a1, a0, a1, t0, t1);
            ptx::fadd2(b0, b1, b0, b1, t2, t3);
          }
        } else {
          const int* const lim = reinterpret_cast<const int*>(row) + 128 + c0;
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const float2 l = *reinterpret_cast<const float2*>(row + c0 + c);
            const int2 m = *reinterpret_cast<const int2*>(lim + c);
            float t0, t1;
            ptx::ffma2(t0, t1, __uint_as_float(u[c]), __uint_as_float(u[c + 1]), factor, factor, l.x, l.y);
            t0 = ptx::ex2_approx(t0);
            t1 = ptx::ex2_approx(t1);
            if (key < m.x) a0 += t0;
            if (key < m.y) a1 += t1;
          }
        }
      };
      uint32_t u0[32], u1[32];
      ptx::tmem_ld32(tS + acc * 256, u0);
      ptx::tmem_wait_ld();
      pin_after_wait<32>(u0);
      ptx::tmem_ld32(tS + acc * 256 + 32, u1);
      half(u0, col0);
      ptx::tmem_wait_ld();
      pin_after_wait<32>(u1);
      ptx::tc_fence_before();
      ptx::mbar_arrive(bar(L::kBarSEmpty + g + 2 * acc));
      half(u1, col0 + 32);
      ptx::mbar_arrive(bar(L::kBarREmpty + e));
      total += (a0 + a1) + (b0 + b1);
    }
  }

  // ---- sums of the two halves and of the cluster's CTAs, in order
  ptx::tc_fence_before();
  float* const sums = reinterpret_cast<float*>(smem + L::kOffSums);
  if (tid < kExps) sums[tid] = total;
  __syncthreads();
  if (tid < kKeys) total = sums[tid] + sums[kKeys + tid];
  if (split > 1) {
    __syncthreads();
    if (tid < kKeys) sums[tid] = total;
    ptx::cluster_sync();
    if (rank == 0 && tid < kKeys) {
      for (int r = 1; r < split; ++r) {
        float x;
        asm volatile("ld.shared::cluster.f32 %0, [%1];"
                     : "=f"(x)
                     : "r"(ptx::mapa(sbase + L::kOffSums + 4 * tid, static_cast<uint32_t>(r)))
                     : "memory");
        total += x;
      }
    }
    ptx::cluster_sync();
  }
  if (warp == kWarpMma) {
    __syncwarp();
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
  if (writes) *dst = old + total;
}

template <int D, int KV, bool QBF16>
cudaError_t launch_impl(const WeightsChunkParams& p, cudaStream_t stream) {
  auto kern = paged_weights_chunk_kernel<D, KV, QBF16>;
  static int attr_done[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::kBytes);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_done[dev] = 1;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(static_cast<long long>(p.n_blocks) * p.w.a.r.B * p.w.a.c.heads * p.split));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Smem<D>::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(p.split);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

template <int D>
cudaError_t launch_d(const WeightsChunkParams& p, int kv, bool bf16, cudaStream_t s) {
  switch (kv) {
    case FA_DTYPE_INT8: return bf16 ? launch_impl<D, FA_DTYPE_INT8, true>(p, s) : launch_impl<D, FA_DTYPE_INT8, false>(p, s);
    case FA_DTYPE_E4M3: return bf16 ? launch_impl<D, FA_DTYPE_E4M3, true>(p, s) : launch_impl<D, FA_DTYPE_E4M3, false>(p, s);
    case FA_DTYPE_BF16: return launch_impl<D, FA_DTYPE_BF16, true>(p, s);
    default: return launch_impl<D, FA_DTYPE_F16, false>(p, s);
  }
}

}  // namespace pwc
}  // namespace

cudaError_t launch_paged_weights_chunk(WeightsChunkParams p, int head_dim, int cache_dtype, bool bf16, int sms,
                                       cudaStream_t stream) {
  p.n_blocks = (p.w.a.max_k + pwc::kKeys - 1) / pwc::kKeys;
  const long long items = static_cast<long long>(p.n_blocks) * p.w.a.r.B * p.w.a.c.heads;
  // CTAs that share the query tiles of a key block.  In tiles of an SM a CTA takes its share
  // and about 6 for its start and end, and there are as many rounds of CTAs as it takes to
  // give every SM its part: few key blocks are spread over more SMs.  1024 tokens over 1024
  // keys, 8 KV heads, GQA 4: 24.6 us in clusters of 4, 55.3 in CTAs; 300 over 300: 20.5 / 24.6; 2 x
  // 1024 over 8192 (3.5 rounds): 212 in clusters of 2, 208 in CTAs.
  const int max_q = p.w.a.max_q < p.w.a.r.total ? p.w.a.max_q : p.w.a.r.total;
  const int tiles = (max_q + p.tq - 1) / p.tq;
  long long best = 0;
  for (int x = 1; x <= pwc::kMaxSplit && x <= tiles && items * x <= 0x7fffffffLL; x *= 2) {
    const long long cost = (items * x + sms - 1) / sms * (6 + (tiles + x - 1) / x);
    if (x == 1 || cost < best) {
      best = cost;
      p.split = x;
    }
  }
  if (items > 0x7fffffffLL) return cudaErrorInvalidValue;  // (refused before)
  return head_dim == 64 ? pwc::launch_d<64>(p, cache_dtype, bf16, stream)
                        : pwc::launch_d<128>(p, cache_dtype, bf16, stream);
}

}  // namespace fa
