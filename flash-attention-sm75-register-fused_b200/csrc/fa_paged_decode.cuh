// Attention of a few new tokens per sequence over a paged KV cache: at most 64
// query rows per (sequence, KV head), i.e. new tokens x query heads of a group.
// Included by fa_fwd_sm100.cu (bounded mbarrier waits, device status word).
//
//   s_ij = scale q_i . k_j,   O_i = sum_j softmax(s_i)_j v_j,
//   LSE_i = log sum_j exp(s_ij)
//
// Bound by HBM: every key and value is read once for all rows of its group.
// The kernel is therefore built around the loads.  A *unit* of work is 8 KB of
// the cache, the K and V rows of kSub consecutive keys of one head (16 keys of
// 16-bit d = 128 pages, 64 of 8-bit d = 64 pages).  All units of the batch, in
// order of sequence, head and key, are cut into equal runs, one per team of
// warps (one warp for up to 16 rows), whatever the sequences' lengths: no team
// waits for another until the end of the kernel, and ragged batches stay
// balanced.  A team streams its run through a ring of shared-memory stages,
// filled by TMA boxes of 16 rows (one per lane, each with its own page), and
// every warp keeps the online softmax of its 8 or 16 rows in registers
// (running maximum m, sum l, O rescaled when m grows):
//
//   S^T = K Q^T     m16n8k16, keys on M, query rows on N: 8 rows cost one
//                   instruction, not a 16-row tile
//   P   = exp2(S - m), transposed in registers (movmatrix) into the B operand
//   O^T += V^T P^T  V read transposed from the same stage
//
// The tensor instructions are the register-operand form: at 8 rows they need a
// tenth of their rate to keep up with HBM, and they take operands converted in
// registers, which 8-bit pages need: int8 and e4m3 both become f16 exactly, K's
// scale multiplies the score and V's scale the probability.  Because f16 has
// few exponent bits, the weights w_ij = p_ij vs_j that multiply V's 8-bit values
// have a reference of their own: with p_ij = 2^(s_ij - m_i), O_i is the sum of
// 2^(m_i - r_i) w_ij v_j, and m_i + log2 w_ij moves r_i as s_ij moves m_i.  A row
// then holds the value rows that make up its result, however large others are
// that it gives no weight to.  bf16 queries over 8-bit pages are scaled per row
// by a power of two.
//
// A team whose run covers a whole (sequence, head) writes O and LSE; otherwise
// its unnormalised O, m and l (8-bit pages: its result and the logarithm of its
// sum) go to one of its two workspace slots (its run's
// first part, which continues a head of the team before, or its last, which
// the next team continues) and paged_combine_kernel joins them in order.
//
// Short caches (DecodeParams::solo, at most 3 to 8 units per team) take one CTA per
// (sequence, head) instead, whose teams share its units and join in shared
// memory: one launch, no workspace, no plan over the batch.
//
// Measured with the join, 8 KV heads, d = 128, GQA 4, one token: 8 sequences x 8192
// keys of f16 pages 47.5 us (5.7 TB/s; a plain copy runs at 6.5), one of 65536 over
// e4m3 pages 33.1 us (4.2 TB/s): loads at HBM's rate between about 5 us until the
// first unit and 3 to 6 for the join.
#include "fa_paged.h"
#include "fa_paged_dev.cuh"

namespace fa {
namespace {
namespace pdec {

constexpr int kWarps = 4;  // per CTA
constexpr int kRowsMax = 64;
constexpr int kCombineThreads = 256;
// Reference of a row that has seen no key (no value, for r): finite, so that
// differences are never NaN, and below any score.
constexpr float kNoMax = -1e30f;
// V's scales are taken times 2^-kScaleDown, so that w stays finite for the
// largest bf16 values (p grows to 2^8).
constexpr int kScaleDown = 10;

// NT: 8-row column blocks of a warp.  Ring stages per warp: as many as the CTAs
// that share an SM leave room for.
constexpr int kMaxStages = 6;
__host__ __device__ constexpr int ctas_per_sm(int nt) { return nt == 1 ? 3 : 2; }
constexpr int stages_per_warp(int nt) { return nt == 1 ? 2 : 3; }

template <int D, int KV>
struct Cfg {
  static constexpr bool k8 = KV >= FA_DTYPE_INT8;
  static constexpr bool kBf16 = KV == FA_DTYPE_BF16;   // type of the products
  static constexpr int kRowBytes = k8 ? D : 2 * D;     // one K or V row
  static constexpr int kSub = 4096 / kRowBytes;        // keys of a unit
  static constexpr int kBoxBytes = kRowBytes < 128 ? kRowBytes : 128;  // inner extent of a box
  static constexpr int kCols = kRowBytes / kBoxBytes;  // boxes side by side
  static constexpr int kMT = kSub / 16;                // 16-key groups
  static constexpr int kBoxes = 2 * kCols * kMT;       // of a unit: (K, V) x columns x groups
  static constexpr int kKS = D / 16;                   // 16-column steps of d
  static constexpr int kScaleBytes = k8 ? kSub * 8 : 0;
  static constexpr int smem(int stages) { return 1024 + kWarps * stages * (8192 + kScaleBytes); }
  // Address of 16-byte piece c of row r of a K or V half stage: boxes of 16
  // rows in the TMA swizzle (128-byte rows: piece ^ row % 8; 64-byte rows:
  // piece ^ (row / 2) % 4), so eight rows at one piece hit eight bank groups.
  __device__ static __forceinline__ uint32_t piece(int r, int c) {
    if constexpr (kCols == 2) {
      return (c >> 3) * 2048 + r * 128 + (((c & 7) ^ (r & 7)) << 4);
    } else if constexpr (kBoxBytes == 128) {
      return r * 128 + ((c ^ (r & 7)) << 4);
    } else {
      return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
    }
  }
  static_assert(kCols == 1 || kSub == 16, "two columns: one group of rows");
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (BF16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

// load_seq for this kernel, which takes sequences of at most max_rows query
// rows per KV head (nq = vis = 0 for the others).
__device__ __forceinline__ Seq load_short(const PagedAttn& a, int b, int max_rows) {
  Seq s = load_seq(a, b);
  if (static_cast<long long>(s.nq) * a.group > max_rows) s.nq = s.vis = 0;
  return s;
}

// The runs are cut from positions, not units: a segment (sequence, head) of n
// units has kSegCost positions before its units' n, for what a team spends on a
// segment besides its units (queries, results).  Without them the teams that
// get many short sequences finish last (32 ragged sequences over int8 pages: 42 us
// without, 32 with, the kernel alone).
constexpr int kSegCost = 1;
__device__ __forceinline__ int positions_of(const PagedAttn& a, int b, int sub, int max_rows) {
  const int n = (load_short(a, b, max_rows).vis + sub - 1) / sub;
  return n > 0 ? n + kSegCost : 0;
}

// Positions of one head: in the sequences before b, and in the whole batch (a
// block-wide pass over the lengths).
struct Spot {
  long long before, total;
};

template <int kThreads>
__device__ Spot find_spot(const PagedAttn& a, int sub, int max_rows, int b, long long* sh) {
  // each thread sums a contiguous share of the sequences
  const int share = (a.r.B + kThreads - 1) / kThreads;
  const int b0 = min(static_cast<int>(threadIdx.x) * share, a.r.B), b1 = min(b0 + share, a.r.B);
  long long sum = 0;
  for (int i = b0; i < b1; ++i) sum += positions_of(a, i, sub, max_rows);
  Spot sp;
  long long x = block_scan<kThreads>(sum, sh, &sp.total);
  if (b >= b0 && b < b1) {
    for (int i = b0; i < b; ++i) x += positions_of(a, i, sub, max_rows);
    sh[kThreads / 32] = x;
  }
  __syncthreads();
  sp.before = sh[kThreads / 32];
  return sp;
}

// Workspace slots: floats [rows][D] of O, then m[rows], l[rows].  16-bit pages:
// O and l relative to 2^m; 8-bit pages: the part's own result times
// 2^-kScaleDown, with l = 1 and m the log2 of its sum of exponentials.
__host__ __device__ constexpr long long slot_floats(int rows, int d) {
  return static_cast<long long>(rows) * (d + 2);
}

// Partial result of a row over a lane's D / 32 columns.
template <int D>
struct Partial {
  static constexpr int E = D / 32;
  float m = kNoMax, l = 0.f, o[E] = {};
  __device__ __forceinline__ void add(float mi, float li, const float (&v)[E]) {
    const float mn = fmaxf(m, mi);
    const float f0 = exp2f(m - mn), f1 = exp2f(mi - mn);
    m = mn;
    l = l * f0 + li * f1;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * f0 + v[e] * f1;
  }
  // the warp writes the row, times `up`
  template <bool BF16>
  __device__ __forceinline__ void write(const PagedAttn& a, int tok, int hq, float up) const {
    const int lane = threadIdx.x & 31;
    const float inv = l == 0.f ? 0.f : up / l;
    uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.o) +
                                                (static_cast<long long>(tok) * a.Hq + hq) * D) +
                    lane * (E / 2);
#pragma unroll
    for (int e = 0; e < E; e += 2) dst[e / 2] = pack2<BF16>(o[e] * inv, o[e + 1] * inv);
    if (lane == 0 && a.lse != nullptr)
      a.lse[static_cast<long long>(hq) * a.r.total + tok] =
          l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994530942f;
  }
};

// Place of a team in its run: unit t of n of (sequence b, head h), position v.
struct Cursor {
  Seq s;
  int b, h, t, n;
  long long v;
};

template <int D, int KV, bool QBF16, int NT, int TEAM>
__global__ void __launch_bounds__(32 * kWarps, ctas_per_sm(NT))
    paged_decode_kernel(const __grid_constant__ DecodeParams p) {
  using C = Cfg<D, KV>;
  const int stages = p.stages * TEAM;  // of a team
  constexpr int kTeams = kWarps / TEAM;
  constexpr float kUp = C::k8 ? 1 << kScaleDown : 1;  // of a stored O
  const PagedAttn& a = p.a;
  extern __shared__ uint8_t smem_raw[];
  __shared__ long long sh_scan[kWarps];
  __shared__ int sh_b[kTeams];
  __shared__ long long sh_rel[kTeams];
  __shared__ __align__(8) unsigned long long sh_bar[kWarps * kMaxStages];
  __shared__ int sh_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, j = lane & 3;
  const int H = a.c.heads;
  const int team = warp / TEAM, trank = warp % TEAM;
  const int tid = static_cast<int>(blockIdx.x) * kTeams + team;
  volatile int* abort_flag = &sh_abort;
  ptx::launch_dependents();

  // ---- set-up, and the team's run [v0, v1) of the batch's positions
  int dead = 0;  // this launch failed elsewhere
  if (threadIdx.x == 0) {
    const unsigned long long st = *reinterpret_cast<volatile unsigned long long*>(&g_fa_status);
    dead = ((st >> 32) == p.epoch && (st & 0xffffffffull) != 0ull) ? 1 : 0;
    sh_abort = 0;
    // a stage is full when its boxes have landed (and, 8-bit pages, the 32
    // lanes' scales)
    for (int i = 0; i < kTeams * stages; ++i)
      ptx::mbar_init(ptx::smem_u32(&sh_bar[i]), C::k8 ? 33u : 1u);
    ptx::fence_barrier_init();
  }
  long long v1, rel;
  int b_first;
  if (p.solo) {
    // the teams take equal parts of the units of (sequence, head) blockIdx.x
    fill_outside(a, D, static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x));
    b_first = static_cast<int>(blockIdx.x) / H;
    const Seq s = load_short(a, b_first, p.max_rows);
    if (static_cast<int>(blockIdx.x) % H == 0) fill_beyond(a, D, s);
    const int n = (s.vis + C::kSub - 1) / C::kSub;
    const long long base = static_cast<long long>(static_cast<int>(blockIdx.x) % H) * (n + kSegCost) + kSegCost;
    rel = base + static_cast<long long>(n) * team / kTeams;
    v1 = base + static_cast<long long>(n) * (team + 1) / kTeams;
    if (__syncthreads_or(dead)) return;
  } else {
    const int share = (a.r.B + 32 * kWarps - 1) / (32 * kWarps);
    const int s0 = min(static_cast<int>(threadIdx.x) * share, a.r.B), s1 = min(s0 + share, a.r.B);
    long long sum = 0, total;
    for (int b = s0; b < s1; ++b) sum += positions_of(a, b, C::kSub, p.max_rows);
    const long long excl = block_scan<32 * kWarps>(sum, sh_scan, &total);
    total *= H;
    const long long per = (total + p.n_teams - 1) / p.n_teams;
    const long long lo = excl * H, hi = (excl + sum) * H;
    // the thread whose share holds a team's first position finds its sequence
    for (int w = 0; w < kTeams; ++w) {
      const long long v = per * (static_cast<long long>(blockIdx.x) * kTeams + w);
      if (v < total && v >= lo && v < hi) {
        long long x = lo;
        for (int b = s0; b < s1; ++b) {
          const long long nb = static_cast<long long>(positions_of(a, b, C::kSub, p.max_rows)) * H;
          if (v < x + nb) {
            sh_b[w] = b;
            sh_rel[w] = v - x;
            break;
          }
          x += nb;
        }
      }
    }
    if (__syncthreads_or(dead)) return;  // (one answer for the block)
    const long long v0 = min(per * tid, total);
    v1 = min(v0 + per, total);
    if (v0 >= v1) return;
    b_first = sh_b[team];
    rel = sh_rel[team];
    v1 -= v0 - rel;  // relative to the first sequence's first position, like rel
  }
  const WaitCtl wc{abort_flag, p.timeout_ns, p.epoch};
  // all warps of the team; a warp that failed makes the team leave together
  auto team_ok = [&](bool v) -> bool {
    if constexpr (TEAM == 1) {
      return __all_sync(0xffffffffu, v);
    } else {
      return ptx::bar_and(1 + team, 32 * TEAM, v);
    }
  };

  auto seek = [&](Cursor& c, int b) {  // the next sequence with units, from b
    for (; b < a.r.B; ++b) {
      c.s = load_short(a, b, p.max_rows);
      c.n = (c.s.vis + C::kSub - 1) / C::kSub;
      c.b = b;
      if (c.n > 0) break;
    }
  };
  auto advance = [&](Cursor& c) {  // to the next unit, if the run has one
    ++c.v;
    if (++c.t < c.n) return;
    c.v += kSegCost;
    if (c.v >= v1) return;
    c.t = 0;
    if (++c.h < H) return;
    c.h = 0;
    seek(c, c.b + 1);
  };
  Cursor cc;  // unit being computed
  if (p.solo) {
    cc.s = load_short(a, b_first, p.max_rows);
    cc.n = (cc.s.vis + C::kSub - 1) / C::kSub;
    cc.b = b_first;
    cc.h = static_cast<int>(blockIdx.x) % H;
    cc.t = static_cast<int>(static_cast<long long>(cc.n) * team / kTeams);
    cc.v = rel;
  } else {
    seek(cc, b_first);
    const long long seg = cc.n + kSegCost;
    cc.h = static_cast<int>(rel / seg);
    cc.t = max(static_cast<int>(rel % seg) - kSegCost, 0);
    cc.v = cc.h * seg + kSegCost + cc.t;
    if (cc.v >= v1) return;  // nothing but a segment's set-up
  }
  Cursor ci = cc;  // unit being loaded (the team's first warp)

  // ---- loads
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                   ~static_cast<uintptr_t>(1023)) +
                        team * stages * 8192;
  const uint32_t ring = ptx::smem_u32(smem);
  // scales of all stages behind the data of all teams: per key K's, V's
  const uint32_t sring = ring + (kWarps * p.stages - team * stages) * 8192 +
                         team * stages * C::kScaleBytes;
  const uint32_t bars = ptx::smem_u32(&sh_bar[team * stages]);
  const uint64_t policy = ptx::policy_evict_first();  // every key is read once
  // lane = (group * kCols + column) * 2 + (0: K, 1: V)
  const int bgrp = lane / (2 * C::kCols), bcol = (lane >> 1) % C::kCols;
  const bool boxes = lane < C::kBoxes;
  const uint32_t box_dst = (lane & 1) * 4096 + (C::kCols == 2 ? bcol * 2048 : bgrp * 16 * C::kRowBytes);
  const void* const box_map = (lane & 1) ? &p.tm_v : &p.tm_k;
  // Pages of the 16-key groups around ci: lane l holds that of group wbase + l
  // in `win` and of group wbase + 32 + l in `win_next`, loaded 32 groups ahead,
  // so a unit's pages are shuffles.  -1 (no key any row may see, or no page)
  // reads as zeros.
  int wbase = 0, win = -1, win_next = -1;
  auto load_window = [&](int first) {
    const int pos = 16 * (first + lane);
    return pos < ci.s.vis ? a.c.lookup(ci.b, pos) : -1;
  };
  auto start_window = [&] {  // at the first unit of the run in a segment
    wbase = ci.t * C::kMT;
    win = load_window(wbase);
    win_next = load_window(wbase + 32);
  };
  int wstage = 0;
  auto issue = [&] {
    if (ci.v >= v1) return;
    const uint32_t bar = bars + 8 * wstage;
    const int key0 = ci.t * C::kSub;
    int g0 = ci.t * C::kMT - wbase;  // the unit's first group in the window
    if (g0 >= 32) {
      g0 -= 32;
      wbase += 32;
      win = win_next;
      win_next = load_window(wbase + 32);
    }
    const int page = __shfl_sync(0xffffffffu, win, g0 + (boxes ? bgrp : 0));
    if (lane == 0) ptx::mbar_arrive_expect_tx(bar, 8192);
    __syncwarp();
    if (boxes)
      ptx::tma_load_4d(ring + wstage * 8192 + box_dst, box_map, bar, bcol * (C::kBoxBytes / (C::k8 ? 1 : 2)),
                       a.c.row_in_page(key0 + 16 * bgrp), ci.h * p.head_step,
                       page < 0 ? -1 : page * p.page_step, policy);
    if constexpr (C::k8) {
      const int left = ci.s.vis - key0;
#pragma unroll
      for (int x = 0; x < C::kSub / 32; ++x) {
        const int r = x * 32 + lane;
        const int pg = __shfl_sync(0xffffffffu, win, g0 + (r >> 4));
        const bool ok = r < left && pg >= 0;
        const long long o =
            ok ? static_cast<long long>(pg) * a.c.s_page + ci.h * a.c.s_head +
                     static_cast<long long>(a.c.row_in_page(key0 + (r & ~15)) + (r & 15)) * a.c.s_row
               : 0;
        const uint32_t d = sring + wstage * C::kScaleBytes + 8 * r;
        ptx::cp_async4(d, a.c.ks + o, ok);
        ptx::cp_async4(d + 4, a.c.vs + o, ok);
      }
      ptx::cp_async_arrive(bar);
    }
    if (++wstage == stages) wstage = 0;
    advance(ci);
    if (ci.t == 0 && ci.v < v1) start_window();
  };
  if (trank == 0) {
    start_window();
    for (int x = 0; x < stages - 1; ++x) issue();
  }

  // ---- the segments (sequence, head) of the run
  constexpr float kGrow = 8.f;  // O and l are rescaled when m grows by more (log2)
  // a negative scale goes into Q's sign; a zero one must not meet a masked -inf
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
  const float scale_abs = fmaxf(fabsf(a.scale_log2), 1e-30f);
  int rstage = 0;
  uint32_t rphase = 0;
  bool ok = true;
  while (ok && cc.v < v1) {
    const Seq s = cc.s;
    const int t_begin = cc.t, n_units = cc.n;
    const int t_end = static_cast<int>(min(static_cast<long long>(n_units), t_begin + (v1 - cc.v)));
    const int rows = s.nq * a.group;
    const int row0 = trank * 8 * NT;  // of this warp
    const bool active = row0 < rows;
    // Q as the B operand: row row0 + 8 nt + g, columns 16 ks + {2j, 2j + 1,
    // 8 + 2j, 9 + 2j} (8-bit pages: 16 ks + 4j .. 4j + 3, the order their
    // bytes come in)
    uint32_t q[NT][C::kKS][2];
    float cs[NT][2];  // score scale of this thread's columns
    int lim[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = row0 + nt * 8 + g;
      const int tok = r / a.group, hq = cc.h * a.group + r % a.group;
      const uint8_t* src = a.q + static_cast<long long>(s.c0 + tok) * a.q_token + hq * a.q_head;
      const bool have = r < rows;
#pragma unroll
      for (int k = 0; k < C::kKS; ++k) {
        if constexpr (C::k8) {
          uint2 w = make_uint2(0u, 0u);
          if (have) w = __ldg(reinterpret_cast<const uint2*>(src + 32 * k + 8 * j));
          q[nt][k][0] = w.x;
          q[nt][k][1] = w.y;
        } else {
          q[nt][k][0] = have ? __ldg(reinterpret_cast<const uint32_t*>(src + 32 * k + 4 * j)) : 0u;
          q[nt][k][1] = have ? __ldg(reinterpret_cast<const uint32_t*>(src + 32 * k + 16 + 4 * j)) : 0u;
        }
      }
      float unit = 1.f;
      if constexpr (C::k8 && QBF16) {
        // q / 2^e with 2^e <= max |q| < 2^(e+1), as f16
        float mx = 0.f;
#pragma unroll
        for (int k = 0; k < C::kKS; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 f = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&q[nt][k][i]));
            mx = fmaxf(mx, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const uint32_t e = __float_as_uint(mx) & 0x7f800000u;
        const bool plain = e == 0u || e >= 0x7e800000u;
        unit = plain ? 1.f : __uint_as_float(e);
        const float inv = plain ? 1.f : __uint_as_float(0x7f000000u - e);
#pragma unroll
        for (int k = 0; k < C::kKS; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 f = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&q[nt][k][i]));
            q[nt][k][i] = pack2<false>(f.x * inv, f.y * inv);
          }
      }
#pragma unroll
      for (int k = 0; k < C::kKS; ++k) {
        q[nt][k][0] ^= flip;
        q[nt][k][1] ^= flip;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        cs[nt][c] = scale_abs;
        if constexpr (C::k8 && QBF16) cs[nt][c] *= __shfl_sync(0xffffffffu, unit, (2 * j + c) * 4);
        const int rc = row0 + nt * 8 + 2 * j + c;
        lim[nt][c] = rc < rows ? row_limit(a, s, rc / a.group) : 0;
      }
    }
    const int min_lim = row_limit(a, s, 0);

    float o[NT][C::kKS][4];
    float m[NT][2], l[NT][2];
    float ref[NT][2];  // r of 8-bit pages (16-bit pages: m)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < C::kKS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nt][k][i] = 0.f;
      m[nt][0] = m[nt][1] = ref[nt][0] = ref[nt][1] = kNoMax;
      l[nt][0] = l[nt][1] = 0.f;
    }

    for (int t = t_begin; t < t_end; ++t) {
      ok = bar_wait(bars + 8 * rstage, rphase, wc, 50);
      // (also: every warp is done with the stage before, which is refilled now;
      // refilling it before the wait, so that two units are in flight while the
      // team waits, measured 1-3 % slower)
      if (!(ok = team_ok(ok))) break;
      if (trank == 0) issue();
      const uint32_t st = ring + rstage * 8192;
      const uint32_t sst = sring + rstage * C::kScaleBytes;
      uint8_t* const stage = smem + rstage * 8192;
      if (++rstage == stages) {
        rstage = 0;
        rphase ^= 1u;
      }
      const int key0 = t * C::kSub;
      const int left = s.vis - key0;
      if (KV != FA_DTYPE_INT8 && left < C::kSub) {
        // rows of V behind the last visible key are stale and might hold NaN
        // (those of a group without any visible key are zero already; int8
        // has no NaN)
        const int end = min(C::kSub, (left + 15) & ~15);
        for (int x = left * 32 + static_cast<int>(threadIdx.x % (32 * TEAM)); x < end * 32; x += 32 * TEAM) {
          const int r = x >> 5, c = x & 31;
          if (c < C::kRowBytes / 16)
            *reinterpret_cast<uint4*>(stage + 4096 + C::piece(r, c)) = make_uint4(0u, 0u, 0u, 0u);
        }
        ptx::fence_proxy_async_smem();  // before a later copy into this stage
        if (!(ok = team_ok(true))) break;
      }
      if (!active) continue;
      // S^T = K Q^T
      float sc[NT][C::kMT][4];
#pragma unroll
      for (int mt = 0; mt < C::kMT; ++mt) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[nt][mt][i] = 0.f;
        if constexpr (!C::k8) {
          const int r = mt * 16 + (lane & 15);
#pragma unroll
          for (int k = 0; k < C::kKS; ++k) {
            uint32_t f[4];
            ldsm4(st + C::piece(r, 2 * k + (lane >> 4)), f);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816<C::kBf16>(sc[nt][mt], f[0], f[1], f[2], f[3], q[nt][k][0], q[nt][k][1]);
          }
        } else {
          // two 16-column steps per ldmatrix: keys 0-7 and 8-15 of pieces k, k + 1
          const int r = mt * 16 + (lane & 15);
#pragma unroll
          for (int k = 0; k < C::kKS; k += 2) {
            uint32_t f[4];
            ldsm4(st + C::piece(r, k + (lane >> 4)), f);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              uint32_t a0, a1, a2, a3;
              widen<KV, false>(f[2 * x], a0, a2);
              widen<KV, false>(f[2 * x + 1], a1, a3);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16816<false>(sc[nt][mt], a0, a1, a2, a3, q[nt][k + x][0], q[nt][k + x][1]);
            }
          }
        }
      }
      // scores (without their common factor cs), masked, and their maxima
      float vsc[C::kMT][2];
      float vmax = 0.f;
      if constexpr (C::k8) {
#pragma unroll
        for (int mt = 0; mt < C::kMT; ++mt)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            float2 f;
            asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];"
                         : "=f"(f.x), "=f"(f.y)
                         : "r"(sst + 8 * (mt * 16 + g + 8 * hh))
                         : "memory");
            vsc[mt][hh] = f.y * (1.f / (1 << kScaleDown));
            vmax = fmaxf(vmax, fabsf(vsc[mt][hh]));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              sc[nt][mt][2 * hh] *= f.x;
              sc[nt][mt][2 * hh + 1] *= f.x;
            }
          }
      }
      if (key0 + C::kSub > min_lim) {
#pragma unroll
        for (int mt = 0; mt < C::kMT; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (key0 + mt * 16 + g + 8 * (i >> 1) >= lim[nt][i & 1]) sc[nt][mt][i] = -INFINITY;
      }
      bool grow = false;
      float top[NT][2];
      const float vlog = C::k8 ? __log2f(vmax) : 0.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = fmaxf(sc[nt][0][c], sc[nt][0][2 + c]);
#pragma unroll
          for (int mt = 1; mt < C::kMT; ++mt) x = fmaxf(x, fmaxf(sc[nt][mt][c], sc[nt][mt][2 + c]));
          top[nt][c] = x;
          grow |= fmaf(x, cs[nt][c], -m[nt][c]) > kGrow;
          // (a bound of m + log2 w: the thread's largest score and scale may be different keys')
          if constexpr (C::k8) grow |= fmaf(x, cs[nt][c], vlog) - ref[nt][c] > kGrow;
        }
      if (__any_sync(0xffffffffu, grow)) {
        auto over_keys = [](float x) {
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        };
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = fmaxf(m[nt][c], over_keys(top[nt][c]) * cs[nt][c]);
            float f = ptx::ex2_approx(m[nt][c] - x);
            m[nt][c] = x;
            l[nt][c] *= f;
            if constexpr (C::k8) {
              float y = -INFINITY;  // the largest log2 w + m
#pragma unroll
              for (int mt = 0; mt < C::kMT; ++mt)
#pragma unroll
                for (int hh = 0; hh < 2; ++hh)
                  y = fmaxf(y, fmaf(sc[nt][mt][2 * hh + c], cs[nt][c], __log2f(fabsf(vsc[mt][hh]))));
              x = fmaxf(ref[nt][c], over_keys(y));
              f = ptx::ex2_approx(ref[nt][c] - x);
              ref[nt][c] = x;
            }
#pragma unroll
            for (int k = 0; k < C::kKS; ++k) {
              o[nt][k][c] *= f;
              o[nt][k][2 + c] *= f;
            }
          }
      }
      // P and O^T += V^T P^T
      uint32_t pb[NT][C::kMT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        // (126: no value yet, all w are 0)
        const float f0 = C::k8 ? ptx::ex2_approx(fminf(m[nt][0] - ref[nt][0], 126.f)) : 1.f;
        const float f1 = C::k8 ? ptx::ex2_approx(fminf(m[nt][1] - ref[nt][1], 126.f)) : 1.f;
#pragma unroll
        for (int mt = 0; mt < C::kMT; ++mt)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            float p0 = ptx::ex2_approx(fmaf(sc[nt][mt][2 * hh], cs[nt][0], -m[nt][0]));
            float p1 = ptx::ex2_approx(fmaf(sc[nt][mt][2 * hh + 1], cs[nt][1], -m[nt][1]));
            l[nt][0] += p0;
            l[nt][1] += p1;
            if constexpr (C::k8) {
              ptx::fmul2(p0, p1, p0, p1, vsc[mt][hh], vsc[mt][hh]);  // w
              ptx::fmul2(p0, p1, p0, p1, f0, f1);
            }
            pb[nt][mt][hh] = transpose8(pack2<C::kBf16>(p0, p1));
          }
      }
      if constexpr (!C::k8) {
#pragma unroll
        for (int mt = 0; mt < C::kMT; ++mt) {
          const int r = mt * 16 + (lane & 7) + ((lane & 16) ? 8 : 0);
#pragma unroll
          for (int k = 0; k < C::kKS; ++k) {
            uint32_t f[4];
            ldsm4t(st + 4096 + C::piece(r, 2 * k + ((lane >> 3) & 1)), f);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816<C::kBf16>(o[nt][k], f[0], f[1], f[2], f[3], pb[nt][mt][0], pb[nt][mt][1]);
          }
        }
      } else {
        // rows of the A operand: M row i holds column 16k + 2i, row i + 8 column
        // 16k + 2i + 1; one ldmatrix brings 32 keys of a piece
#pragma unroll
        for (int mt = 0; mt < C::kMT; mt += 2) {
          const int r = mt * 16 + lane;
#pragma unroll
          for (int k = 0; k < C::kKS; ++k) {
            uint32_t f[4];
            ldsm4t(st + 4096 + C::piece(r, k), f);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              uint32_t a0, a1, a2, a3;
              widen<KV, true>(f[2 * x], a0, a1);
              widen<KV, true>(f[2 * x + 1], a2, a3);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16816<false>(o[nt][k], a0, a1, a2, a3, pb[nt][mt + x][0], pb[nt][mt + x][1]);
            }
          }
        }
      }
    }
    if (!ok) break;

    // ---- the segment's result
    const bool first = t_begin == 0, last = t_end == n_units;
    constexpr int kSlotRows = 8 * NT * TEAM;
    // (solo: the team's part of the ring, once all its warps have read it)
    float* const slot = p.solo ? reinterpret_cast<float*>(smem)
                               : p.ws + (2ll * tid + (first ? 1 : 0)) * slot_floats(kSlotRows, D);
    if (p.solo && !(ok = team_ok(true))) break;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x = l[nt][c];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        l[nt][c] = x;
        if constexpr (C::k8) {
          // O becomes the result times 2^-kScaleDown (one exponent: 2^(r - m) alone
          // may pass fp32's range)
          const float lg = __log2f(x);
          const float f = x == 0.f ? 0.f : exp2f(ref[nt][c] - m[nt][c] - lg);
#pragma unroll
          for (int k = 0; k < C::kKS; ++k) {
            o[nt][k][c] *= f;
            o[nt][k][2 + c] *= f;
          }
          m[nt][c] = x == 0.f ? kNoMax : m[nt][c] + lg;
          l[nt][c] = x == 0.f ? 0.f : 1.f;
        }
      }
    // column of o[..][k][2 hh + c]
    auto col = [&](int k, int hh) { return C::k8 ? 16 * k + 2 * g + hh : 16 * k + g + 8 * hh; };
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = row0 + nt * 8 + 2 * j + c;
        if (r >= rows) continue;
        if (first && last && !p.solo) {
          const int tok = s.c0 + r / a.group, hq = cc.h * a.group + r % a.group;
          const float inv = l[nt][c] == 0.f ? 0.f : kUp / l[nt][c];
          uint16_t* dst = static_cast<uint16_t*>(a.o) + (static_cast<long long>(tok) * a.Hq + hq) * D;
#pragma unroll
          for (int k = 0; k < C::kKS; ++k) {
            const uint32_t w = pack2<QBF16>(o[nt][k][c] * inv, o[nt][k][2 + c] * inv);
            if constexpr (C::k8) {
              *reinterpret_cast<uint32_t*>(dst + col(k, 0)) = w;
            } else {
              dst[col(k, 0)] = static_cast<uint16_t>(w & 0xffffu);
              dst[col(k, 1)] = static_cast<uint16_t>(w >> 16);
            }
          }
          if (g == 0 && a.lse != nullptr)
            a.lse[static_cast<long long>(hq) * a.r.total + tok] =
                l[nt][c] == 0.f ? -INFINITY : (m[nt][c] + (C::k8 ? 0.f : __log2f(l[nt][c]))) * 0.69314718055994530942f;
        } else {
          // slot 0: continues the head of an earlier team; slot 1: begins one
#pragma unroll
          for (int k = 0; k < C::kKS; ++k) {
            slot[r * D + col(k, 0)] = o[nt][k][c];
            slot[r * D + col(k, 1)] = o[nt][k][2 + c];
          }
          if (g == 0) {
            slot[kSlotRows * D + r] = m[nt][c];
            slot[kSlotRows * D + kSlotRows + r] = l[nt][c];
          }
        }
      }
    // ---- next segment
    cc.v += t_end - t_begin - 1;
    cc.t = t_end - 1;
    advance(cc);
  }
  // after a failed wait: copies in flight land before the CTA exits
  if (!ok && trank == 0) {
    for (int x = 0; x < stages; ++x) {
      bar_wait(bars + 8 * rstage, rphase, wc, 51, false);
      if (++rstage == stages) {
        rstage = 0;
        rphase ^= 1u;
      }
      if (rstage == wstage) break;
    }
    ptx::cp_async_wait_all();
  }
  if (p.solo) {
    if (__syncthreads_and(ok ? 1 : 0) == 0) return;
    // one warp joins a row of the teams' slots
    constexpr int kSlotRows = 8 * NT * TEAM;
    const Seq s = load_short(a, b_first, p.max_rows);
    const int n = (s.vis + C::kSub - 1) / C::kSub, h = static_cast<int>(blockIdx.x) % H;
    for (int row = warp; row < s.nq * a.group; row += kWarps) {
      Partial<D> all;
      for (int w = 0; w < kTeams; ++w) {
        if (static_cast<long long>(n) * w / kTeams == static_cast<long long>(n) * (w + 1) / kTeams) continue;
        const float* sl = reinterpret_cast<const float*>(smem + (w - team) * (stages * 8192));
        float v[Partial<D>::E];
#pragma unroll
        for (int e = 0; e < Partial<D>::E; ++e) v[e] = sl[row * D + lane * Partial<D>::E + e];
        all.add(sl[kSlotRows * D + row], sl[kSlotRows * D + kSlotRows + row], v);
      }
      all.template write<QBF16>(a, s.c0 + row / a.group, h * a.group + row % a.group, kUp);
    }
  }
}

// Joins the partial results of (sequence, KV head) blockIdx.x, query rows
// blockIdx.y * kRows ..: with M = max m_s over the segment's slots,
//   O = up sum 2^(m_s - M) O_s / sum 2^(m_s - M) l_s,
// slots in the order of their teams (so the result does not depend on timing).
// kRows = 8 (many rows to join, few slots each): one warp per row.  kRows = 1
// (few rows, many slots), or a segment of more than kManySlots: the block's
// warps share a row's slots and are joined at the end.
// Also writes the rows that no team of the decode kernel computes: rows of
// sequences without visible keys or beyond max_q, and packed rows of no sequence.
constexpr int kManySlots = 32;

template <int D, bool BF16, int kRows>
__global__ void __launch_bounds__(kCombineThreads)
    paged_combine_kernel(const __grid_constant__ DecodeParams p, int sub, int slot_rows, float up) {
  constexpr int kW = kCombineThreads / 32;
  constexpr int E = D / 32;
  const PagedAttn& a = p.a;
  __shared__ long long sh[kW + 1];
  __shared__ float sh_o[kW][D];
  __shared__ float sh_m[kW], sh_l[kW];
  const int b = blockIdx.x / a.c.heads, h = blockIdx.x % a.c.heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  fill_outside(a, D, static_cast<int>(blockIdx.y * gridDim.x + blockIdx.x),
               static_cast<int>(gridDim.x * gridDim.y));
  const Seq s = load_short(a, b, p.max_rows);
  if (h == 0 && blockIdx.y == 0) fill_beyond(a, D, s);
  const Spot sp = find_spot<kCombineThreads>(a, sub, p.max_rows, b, sh);
  // the decode kernel's results are complete and visible after this
  ptx::grid_dep_wait();
  const int row0 = blockIdx.y * kRows;
  const int rows = min(s.nq * a.group - row0, kRows);  // of this block
  if (rows <= 0) return;
  const int n = (s.vis + sub - 1) / sub;
  const long long total = sp.total * a.c.heads;
  const long long per = (total + p.n_teams - 1) / p.n_teams;
  const long long t0 = sp.before * a.c.heads + static_cast<long long>(h) * (n + kSegCost) + kSegCost;
  const int w0 = n > 0 ? static_cast<int>(t0 / per) : 0;
  const int w1 = n > 0 ? static_cast<int>((t0 + n - 1) / per) : -1;
  if (w0 == w1) return;  // one team had it all
  const long long stride = slot_floats(slot_rows, D);
  // slots first, first + step, ... of row `row`
  auto gather = [&](int row, int first, int step) {
    Partial<D> acc;
    constexpr int kBatch = 8;
    for (int w = w0 + first; w <= w1; w += kBatch * step) {
      float mi[kBatch], li[kBatch], v[kBatch][E];
#pragma unroll
      for (int x = 0; x < kBatch; ++x) {
        const int ww = w + x * step;
        mi[x] = kNoMax;
        li[x] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) v[x][e] = 0.f;
        if (ww <= w1) {
          const float* sl = p.ws + (2ll * ww + (ww == w0 ? 1 : 0)) * stride;
          mi[x] = __ldcg(sl + slot_rows * D + row);
          li[x] = __ldcg(sl + slot_rows * D + slot_rows + row);
          if constexpr (E == 4) {
            const float4 f = __ldcg(reinterpret_cast<const float4*>(sl + row * D) + lane);
            v[x][0] = f.x;
            v[x][1] = f.y;
            v[x][2] = f.z;
            v[x][3] = f.w;
          } else {
            const float2 f = __ldcg(reinterpret_cast<const float2*>(sl + row * D) + lane);
            v[x][0] = f.x;
            v[x][1] = f.y;
          }
        }
      }
#pragma unroll
      for (int x = 0; x < kBatch; ++x)
        if (w + x * step <= w1) acc.add(mi[x], li[x], v[x]);
    }
    return acc;
  };
  auto finish = [&](int row, const Partial<D>& r) {
    r.template write<BF16>(a, s.c0 + row / a.group, h * a.group + row % a.group, up);
  };
  if (kRows > 1 && w1 - w0 < kManySlots) {
    for (int r = warp; r < rows; r += kW) finish(row0 + r, gather(row0 + r, 0, 1));
    return;
  }
  for (int r = 0; r < rows; ++r) {
    const Partial<D> mine = gather(row0 + r, warp, kW);
    if (lane == 0) {
      sh_m[warp] = mine.m;
      sh_l[warp] = mine.l;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sh_o[warp][lane * E + e] = mine.o[e];
    __syncthreads();
    if (warp == 0) {
      Partial<D> all;
#pragma unroll
      for (int w = 0; w < kW; ++w) {
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = sh_o[w][lane * E + e];
        all.add(sh_m[w], sh_l[w], v);
      }
      finish(row0 + r, all);
    }
    __syncthreads();
  }
}

template <int D, int KV, bool QBF16, int NT, int TEAM>
cudaError_t launch_impl(const DecodeParams& p, int n_ctas, cudaStream_t stream) {
  using C = Cfg<D, KV>;
  auto kern = paged_decode_kernel<D, KV, QBF16, NT, TEAM>;
  static int attr_done[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_done[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::smem(kMaxStages));
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_done[dev] = 1;
  }
  kern<<<n_ctas, 32 * kWarps, C::smem(p.stages), stream>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.solo) return e;
  // the combine may start while the last teams finish; it waits for them
  // before it reads a slot
  cudaLaunchConfig_t cfg{};
  const unsigned segments = static_cast<unsigned>(p.a.r.B) * p.a.c.heads;
  // blocks of one row fill the device with few segments (8 heads x 64 rows: 38
  // us for the call instead of 50; 64 x 4: 86 / 90), blocks of eight with many
  // (256 x 4: 91 / 86; 128 x 64: 155 / 113); the line is at four rows for each of
  // the 148 SMs
  const bool many = static_cast<long long>(segments) * p.max_rows > 4 * 148;
  cfg.gridDim = dim3(segments, many ? (p.max_rows + 7) / 8 : p.max_rows);
  cfg.blockDim = dim3(kCombineThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, many ? paged_combine_kernel<D, QBF16, 8> : paged_combine_kernel<D, QBF16, 1>,
                            p, static_cast<int>(C::kSub), 8 * NT * TEAM,
                            C::k8 ? static_cast<float>(1 << kScaleDown) : 1.f);
}

// Rows of a team and how it is made up: one warp for 8 or 16 rows, two or four
// of 16 rows each for more.
struct Team {
  int nt, warps;
};
Team team_for(int max_rows) {
  return max_rows <= 8 ? Team{1, 1} : max_rows <= 16 ? Team{2, 1} : max_rows <= 32 ? Team{2, 2} : Team{2, 4};
}

template <int D, int KV, bool QBF16>
cudaError_t launch_rows(const DecodeParams& p, int n_ctas, cudaStream_t s) {
  if (p.max_rows <= 8) return launch_impl<D, KV, QBF16, 1, 1>(p, n_ctas, s);
  if (p.max_rows <= 16) return launch_impl<D, KV, QBF16, 2, 1>(p, n_ctas, s);
  if constexpr (D == 64 || KV >= FA_DTYPE_INT8) {
    if (p.max_rows > 32) return launch_impl<D, KV, QBF16, 2, 4>(p, n_ctas, s);
  }
  return launch_impl<D, KV, QBF16, 2, 2>(p, n_ctas, s);  // (paged_decode_rows)
}

template <int D>
cudaError_t launch_d(const DecodeParams& p, int kv, bool bf16, int n_ctas, cudaStream_t s) {
  switch (kv) {
    case FA_DTYPE_INT8:
      return bf16 ? launch_rows<D, FA_DTYPE_INT8, true>(p, n_ctas, s)
                  : launch_rows<D, FA_DTYPE_INT8, false>(p, n_ctas, s);
    case FA_DTYPE_E4M3:
      return bf16 ? launch_rows<D, FA_DTYPE_E4M3, true>(p, n_ctas, s)
                  : launch_rows<D, FA_DTYPE_E4M3, false>(p, n_ctas, s);
    case FA_DTYPE_BF16: return launch_rows<D, FA_DTYPE_BF16, true>(p, n_ctas, s);
    default: return launch_rows<D, FA_DTYPE_F16, false>(p, n_ctas, s);
  }
}

}  // namespace pdec
}  // namespace

// Query rows per (sequence, KV head) up to which this kernel is taken.  Over
// 8-bit pages always kRowsMax, for the chunk kernel has to expand them first
// (B=8, 8192 keys, 8 KV heads, d = 128, int8, 64 rows: 106 us here, 150 there; 32
// rows: 60 / 151).  16-bit pages: up to 32 rows (16: 54 / 70 us, 32: 61 / 85);
// above, teams of four warps read a unit four times from shared memory and are
// slower (48 rows: 106 / 87, 32 x 4096 keys: 210 / 137), except at d = 64 with
// less than half a CTA of the chunk kernel per SM (4 x 8 heads x 4096 keys, 48
// rows: 25 / 28 us, but 128 heads x 2048: 38 / 29).
int paged_decode_rows(long long heads, int head_dim, int kv, int sms) {
  return kv >= FA_DTYPE_INT8 || (head_dim == 64 && 2 * heads < sms) ? pdec::kRowsMax : 32;
}

namespace {
namespace pdec {
// Few units per (sequence, head): one CTA each, joined in shared memory.  What
// it saves is the join (one launch); what it costs is that few CTAs run and
// none helps another.  Time of either way, d = 128, by units per team (us, runs /
// one CTA each):
//   heads of all sequences      8          64          152         1024
//   f16  3 units            8.4 / 6.5   9.6 / 6.9  10.0 / 7.4  27.9 / 25.4
//        5                  8.5 / 8.1   9.7 / 8.2  12.1 / 8.9  37.7 / 35.4
//        8                  8.6 / 10.2 10.6 / 10.4 15.0 / 11.4 53.3 / 49.7
//        16                 9.2 / 15.7 13.1 / 15.9 20.7 / 17.3 91.5 / 87.3
//   int8 3                  9.5 / 8.6  10.8 / 8.9  12.5 / 9.8  30.8 / 31.3
//        4                  9.8 / 9.8  11.4 / 10.1 13.5 / 11.3 35.7 / 36.9
//        8                  9.7 / 14.6 12.4 / 14.9 17.1 / 17.2 55.5 / 59.8
// With a CTA for half the SMs or more 8 units, though equal lengths would allow
// 16: in a ragged batch the longest sequence has one CTA too (152 heads, lengths
// of 1 to 16 units per team: 17.1 / 16.9, mostly short ones 15.8 / 16.1).
bool is_solo(long long heads, int max_rows, int max_k, int head_dim, int kv, int sms) {
  const bool k8 = kv >= FA_DTYPE_INT8;
  const int sub = 4096 / (head_dim * (k8 ? 1 : 2));
  const int most = 2 * heads < sms ? (k8 ? 4 : 5) : !k8 || heads <= 3LL * sms ? 8 : 3;
  return (static_cast<long long>(max_k) + sub - 1) / sub <= most * (kWarps / team_for(max_rows).warps);
}
}  // namespace pdec
}  // namespace

size_t paged_decode_ws_bytes(long long heads, int max_rows, int max_k, int head_dim, int kv, int sms) {
  if (pdec::is_solo(heads, max_rows, max_k, head_dim, kv, sms)) return 0;
  const pdec::Team t = pdec::team_for(max_rows);
  const size_t teams = static_cast<size_t>(sms) * pdec::ctas_per_sm(t.nt) * (pdec::kWarps / t.warps);
  return 2 * teams * static_cast<size_t>(pdec::slot_floats(8 * t.nt * t.warps, head_dim)) * sizeof(float);
}

cudaError_t launch_paged_decode(DecodeParams p, int head_dim, int kv, bool bf16, int sms,
                                cudaStream_t stream) {
  const pdec::Team t = pdec::team_for(p.max_rows);
  const int per_cta = pdec::kWarps / t.warps;
  // no more teams than units there can be
  const int sub = 4096 / (head_dim * (kv >= FA_DTYPE_INT8 ? 1 : 2));
  const long long heads = static_cast<long long>(p.a.r.B) * p.a.c.heads;
  const long long units = heads * ((static_cast<long long>(p.a.max_k) + sub - 1) / sub);
  long long ctas = (units + per_cta - 1) / per_cta;
  const long long most = static_cast<long long>(sms) * pdec::ctas_per_sm(t.nt);
  ctas = ctas > most ? most : ctas < 1 ? 1 : ctas;
  p.n_teams = static_cast<int>(ctas) * per_cta;
  p.solo = pdec::is_solo(heads, p.max_rows, p.a.max_k, head_dim, kv, sms) ? 1 : 0;
  p.stages = pdec::stages_per_warp(t.nt);
  if (p.solo) {
    ctas = heads;
    if (ctas <= sms) p.stages = pdec::kMaxStages;
    else if (ctas <= 2LL * sms) p.stages = 3;
  }
  return head_dim == 64 ? pdec::launch_d<64>(p, kv, bf16, static_cast<int>(ctas), stream)
                        : pdec::launch_d<128>(p, kv, bf16, static_cast<int>(ctas), stream);
}

}  // namespace fa
