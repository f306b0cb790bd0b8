// Attention of a few new tokens per sequence over a paged KV cache: at most 16
// query rows per (sequence, KV head), i.e. new tokens x query heads of a group.
//
//   s_ij = scale q_i . k_j,   O_i = sum_j softmax(s_i)_j v_j,
//   LSE_i = log sum_j exp(s_ij)
//
// Bound by HBM: every key and value is read once for all rows of its group.
// The kernel is therefore built around the loads.  A *unit* of work is 8 KB of
// the cache, the K and V rows of `Sub` consecutive keys of one head (16 keys of
// 16-bit d = 128 pages, 64 of 8-bit d = 64 pages).  All units of the batch, in
// order of sequence, head and key, are cut into equal runs, one per warp,
// whatever the sequences' lengths: no warp waits for another until the end of
// the kernel, and ragged batches stay balanced.  A warp streams its run through
// a private ring of shared-memory stages filled with 16-byte asynchronous
// copies (zero-filled past the last visible key, so stale rows of a page never
// enter the arithmetic), and keeps the online softmax (running maximum m, sum
// l, O rescaled when m grows) in registers:
//
//   S^T = K Q^T     m16n8k16, keys on M, query rows on N: 8 rows cost one
//                   instruction, not a 16-row tile
//   P   = exp2(S - m), transposed in registers (movmatrix) into the B operand
//   O^T += V^T P^T  V read transposed from the same stage
//
// The warp's tensor instructions are the small register-operand form: at 8 or
// 16 rows they need a fifth to two thirds of what HBM delivers, and take
// operands converted in registers, which 8-bit pages need: int8 and e4m3 both
// become f16 exactly, K's scale multiplies the score and V's scale the
// probability.  Because f16 has few exponent bits, V's scales are taken
// relative to a power of two per warp that follows the largest one seen; bf16
// queries over 8-bit pages are scaled per row by a power of two likewise.
//
// A warp whose run covers a whole (sequence, head) writes O and LSE; otherwise
// its unnormalised O, m and l go to one of its two workspace slots (its run's
// first part, which continues a head of the warp before, or its last, which
// the next warp continues) and paged_combine_kernel joins them in order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "fa_paged.h"
#include "fa_paged_dev.cuh"
#include "sm100_ptx.cuh"

namespace fa {
namespace {

constexpr int kWarps = 4;    // per CTA
constexpr int kStages = 3;   // ring stages of 8 KB per warp
constexpr int kCtasPerSm = 2;
constexpr int kRowsMax = 16;
constexpr int kCombineThreads = 256;

template <int D, int KV>
struct Cfg {
  static constexpr bool k8 = KV >= FA_DTYPE_INT8;
  static constexpr bool kBf16 = KV == FA_DTYPE_BF16;   // type of the products
  static constexpr int kRowBytes = k8 ? D : 2 * D;     // one K or V row
  static constexpr int kSub = 4096 / kRowBytes;        // keys of a unit
  static constexpr int kChunks = kRowBytes / 16;       // 16-byte pieces of a row
  static constexpr int kRowsPerPass = 32 / kChunks;
  static constexpr int kPasses = kSub / kRowsPerPass;  // 8
  static constexpr int kMT = kSub / 16;                // 16-key tiles
  static constexpr int kKS = D / 16;                   // 16-column steps of d
  static constexpr int kScaleBytes = k8 ? kSub * 8 : 0;
  static constexpr int kStageBytes = 8192 + kScaleBytes;
  static constexpr int kSmem = kWarps * kStages * kStageBytes;
  // 16-byte piece c of row r is stored at piece c ^ swz(r): eight rows at one
  // piece lie in eight different bank groups
  __device__ static __forceinline__ int swz(int r) {
    return kChunks >= 8 ? (r & 7) : ((r >> 1) & 3);
  }
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

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

template <bool BF16>
__device__ __forceinline__ uint32_t pack2f(float lo, float hi) {
  if constexpr (BF16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
}

// load_seq for this kernel, which takes sequences of at most max_rows query
// rows per KV head (nq = vis = 0 for the others).
__device__ __forceinline__ Seq load_short(const PagedAttn& a, int b, int max_rows) {
  Seq s = load_seq(a, b);
  if (static_cast<long long>(s.nq) * a.group > max_rows) s.nq = s.vis = 0;
  return s;
}

// Units of one head: in the sequences before b, and in the whole batch (a
// block-wide pass over the lengths).
struct Spot {
  long long before, total;
};

__device__ __forceinline__ int units_of(const PagedAttn& a, int b, int sub, int max_rows) {
  return (load_short(a, b, max_rows).vis + sub - 1) / sub;
}

template <int kThreads>
__device__ Spot find_spot(const PagedAttn& a, int sub, int max_rows, int b, long long* sh) {
  // each thread sums a contiguous share of the sequences
  const int share = (a.r.B + kThreads - 1) / kThreads;
  const int b0 = min(static_cast<int>(threadIdx.x) * share, a.r.B), b1 = min(b0 + share, a.r.B);
  long long sum = 0;
  for (int i = b0; i < b1; ++i) sum += units_of(a, i, sub, max_rows);
  Spot sp;
  long long x = block_scan<kThreads>(sum, sh, &sp.total);
  if (b >= b0 && b < b1) {
    for (int i = b0; i < b; ++i) x += units_of(a, i, sub, max_rows);
    sh[kThreads / 32] = x;
  }
  __syncthreads();
  sp.before = sh[kThreads / 32];
  return sp;
}

// Workspace slots: floats [rows][D] of O, then m[rows], l[rows].
__host__ __device__ constexpr long long slot_floats(int rows, int d) {
  return static_cast<long long>(rows) * (d + 2);
}

struct DecodeParams {
  PagedAttn a;
  float* ws;
  int n_warps;   // warps of the launch that take runs
  int max_rows;  // query rows per KV head handled here (<= 8 * NT)
};

// Position of a warp in its run: the current unit's sequence, head and key.
struct Cursor {
  Seq s;
  int b, h, t, n;  // unit t of n of (b, h)
};

template <int D, int KV, bool QBF16, int NT>
__global__ void __launch_bounds__(32 * kWarps, kCtasPerSm)
    paged_decode_kernel(const __grid_constant__ DecodeParams p) {
  using C = Cfg<D, KV>;
  const PagedAttn& a = p.a;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long sh_scan[kWarps];
  __shared__ int sh_b[kWarps];
  __shared__ long long sh_rel[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, j = lane & 3;
  const int H = a.c.heads;
  ptx::launch_dependents();

  // ---- the warp's run [u0, u1) and where it starts
  long long total, per, u0, u1;
  int b_first = 0;
  long long rel = 0;
  {
    const int share = (a.r.B + 32 * kWarps - 1) / (32 * kWarps);
    const int s0 = min(static_cast<int>(threadIdx.x) * share, a.r.B), s1 = min(s0 + share, a.r.B);
    long long sum = 0;
    for (int b = s0; b < s1; ++b) sum += units_of(a, b, C::kSub, p.max_rows);
    const long long excl = block_scan<32 * kWarps>(sum, sh_scan, &total);
    total *= H;
    per = (total + p.n_warps - 1) / p.n_warps;
    const long long lo = excl * H, hi = (excl + sum) * H;
    // the thread whose share holds a warp's first unit finds its sequence
    for (int w = 0; w < kWarps; ++w) {
      const long long u = per * (static_cast<long long>(blockIdx.x) * kWarps + w);
      if (u < total && u >= lo && u < hi) {
        long long x = lo;
        for (int b = s0; b < s1; ++b) {
          const long long nb = static_cast<long long>(units_of(a, b, C::kSub, p.max_rows)) * H;
          if (u < x + nb) {
            sh_b[w] = b;
            sh_rel[w] = u - x;
            break;
          }
          x += nb;
        }
      }
    }
    __syncthreads();
    const int wid = static_cast<int>(blockIdx.x) * kWarps + warp;
    u0 = min(per * wid, total);
    u1 = min(u0 + per, total);
    if (u0 >= u1) return;
    b_first = sh_b[warp];
    rel = sh_rel[warp];
  }
  const int wid = static_cast<int>(blockIdx.x) * kWarps + warp;

  auto seek = [&](Cursor& c, int b) {  // first unit of the next sequence with keys, from b
    for (; b < a.r.B; ++b) {
      c.s = load_short(a, b, p.max_rows);
      c.n = (c.s.vis + C::kSub - 1) / C::kSub;
      c.b = b;
      if (c.n > 0) break;
    }
  };
  auto advance = [&](Cursor& c) {  // (not past the run's last unit)
    if (++c.t < c.n) return;
    c.t = 0;
    if (++c.h < H) return;
    c.h = 0;
    seek(c, c.b + 1);
  };
  Cursor cc;  // unit being computed
  seek(cc, b_first);
  cc.h = static_cast<int>(rel / cc.n);
  cc.t = static_cast<int>(rel % cc.n);
  Cursor ci = cc;  // unit being loaded

  // ---- loads
  const uint32_t ring = ptx::smem_u32(smem) + warp * (kStages * C::kStageBytes);
  const int lrow = lane / C::kChunks, lchunk = lane % C::kChunks;
  long long iu = u0;  // unit of ci
  int pages[C::kMT];  // pages of ci's 16-key groups
  auto load_pages = [&] {
#pragma unroll
    for (int m = 0; m < C::kMT; ++m) {
      const int pos = ci.t * C::kSub + 16 * m;
      pages[m] = pos < ci.s.vis ? a.c.lookup(ci.b, pos) : -1;
    }
  };
  load_pages();
  int wstage = 0;
  auto issue = [&] {
    if (iu < u1) {
      const uint32_t st = ring + wstage * C::kStageBytes;
      const int key0 = ci.t * C::kSub;
      const int left = ci.s.vis - key0;  // rows of the unit that exist
      const long long hoff = ci.h * a.c.head_stride + 16 * lchunk;
      long long off[C::kMT];
#pragma unroll
      for (int m = 0; m < C::kMT; ++m)
        off[m] = static_cast<long long>(pages[m]) * a.c.page_stride + hoff +
                 static_cast<long long>(a.c.row_in_page(key0 + 16 * m)) * a.c.row_stride;
#pragma unroll
      for (int x = 0; x < C::kPasses; ++x) {
        const int r = x * C::kRowsPerPass + lrow;  // key of the unit
        const int m = (x * C::kRowsPerPass) / 16;
        const bool ok = r < left && pages[m] >= 0;
        const long long o = ok ? off[m] + static_cast<long long>(r & 15) * a.c.row_stride : 0;
        const uint32_t d = st + r * C::kRowBytes + ((lchunk ^ C::swz(r)) << 4);
        cp16(d, a.c.k + o, ok);
        cp16(d + 4096, a.c.v + o, ok);
      }
      if constexpr (C::k8) {
#pragma unroll
        for (int x = 0; x < C::kSub / 32; ++x) {
          const int r = x * 32 + lane;
          const int page = lane < 16 ? pages[2 * x] : pages[2 * x + 1];
          const bool ok = r < left && page >= 0;
          const long long o =
              ok ? static_cast<long long>(page) * a.c.s_page + ci.h * a.c.s_head +
                       static_cast<long long>(a.c.row_in_page(key0 + (r & ~15)) + (r & 15)) * a.c.s_row
                 : 0;
          cp4(st + 8192 + 8 * r, a.c.ks + o, ok);
          cp4(st + 8192 + 8 * r + 4, a.c.vs + o, ok);
        }
      }
      if (++wstage == kStages) wstage = 0;
      if (++iu < u1) {
        advance(ci);
        load_pages();
      }
    }
    cp_commit();
  };
#pragma unroll
  for (int x = 0; x < kStages - 1; ++x) issue();

  // ---- the segments (sequence, head) of the run
  constexpr float kGrow = 8.f;        // O and l are rescaled when m grows by more (log2)
  constexpr float kTinyScale = 7.8886090522101181e-31f;  // 2^-100
  int rstage = 0;
  long long u = u0;
  while (u < u1) {
    const Seq s = cc.s;
    const int t_begin = cc.t, n_units = cc.n;
    const int t_end = static_cast<int>(min(static_cast<long long>(n_units), t_begin + (u1 - u)));
    const int rows = s.nq * a.group;
    // Q as the B operand: row 8 nt + g, columns 16 ks + {2j, 2j + 1, 8 + 2j, 9 + 2j}
    // (8-bit pages: 16 ks + 4j .. 4j + 3, the order their bytes come in)
    uint32_t q[NT][C::kKS][2];
    float colscale[NT][2];
    int lim[NT][2];
    int min_lim = 0x7fffffff;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 8 + g;
      const int tok = r / a.group, hq = cc.h * a.group + r % a.group;
      const uint8_t* src = a.q + static_cast<long long>(s.c0 + tok) * a.q_token + hq * a.q_head;
      const bool ok = r < rows;
#pragma unroll
      for (int k = 0; k < C::kKS; ++k) {
        if constexpr (C::k8) {
          uint2 w = make_uint2(0u, 0u);
          if (ok) w = __ldg(reinterpret_cast<const uint2*>(src + 32 * k + 8 * j));
          q[nt][k][0] = w.x;
          q[nt][k][1] = w.y;
        } else {
          q[nt][k][0] = ok ? __ldg(reinterpret_cast<const uint32_t*>(src + 32 * k + 4 * j)) : 0u;
          q[nt][k][1] = ok ? __ldg(reinterpret_cast<const uint32_t*>(src + 32 * k + 16 + 4 * j)) : 0u;
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
            q[nt][k][i] = pack2f<false>(f.x * inv, f.y * inv);
          }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        colscale[nt][c] = a.scale_log2;
        if constexpr (C::k8 && QBF16)
          colscale[nt][c] *= __shfl_sync(0xffffffffu, unit, (2 * j + c) * 4);
        const int rc = nt * 8 + 2 * j + c;
        lim[nt][c] = rc < rows ? row_limit(a, s, rc / a.group) : 0;
      }
    }
    min_lim = row_limit(a, s, 0);

    float o[NT][C::kKS][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < C::kKS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nt][k][i] = 0.f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }
    float vref = kTinyScale, rv = 1.f / kTinyScale;  // V scales relative to vref

    for (int t = t_begin; t < t_end; ++t) {
      cp_wait<kStages - 2>();
      __syncwarp();
      issue();
      const uint32_t st = ring + rstage * C::kStageBytes;
      if (++rstage == kStages) rstage = 0;
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
          const uint32_t row = st + r * C::kRowBytes;
#pragma unroll
          for (int k = 0; k < C::kKS; ++k) {
            uint32_t f[4];
            ldsm4(row + (((2 * k + (lane >> 4)) ^ C::swz(r)) << 4), f);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816<C::kBf16>(sc[nt][mt], f[0], f[1], f[2], f[3], q[nt][k][0], q[nt][k][1]);
          }
        } else {
          // two 16-column steps per ldmatrix: keys 0-7 and 8-15 of pieces k, k + 1
          const int r = mt * 16 + (lane & 7) + ((lane & 8) ? 8 : 0);
          const uint32_t row = st + r * C::kRowBytes;
#pragma unroll
          for (int k = 0; k < C::kKS; k += 2) {
            uint32_t f[4];
            ldsm4(row + (((k + (lane >> 4)) ^ C::swz(r)) << 4), f);
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
      // scores in log2 units, masked; do the maxima grow?
      float vsc[C::kMT][2];
      const int key0 = t * C::kSub;
      const bool masked = key0 + C::kSub > min_lim;
      bool grow = false, vgrow = false;
#pragma unroll
      for (int mt = 0; mt < C::kMT; ++mt)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          float ks = 1.f;
          const int r = mt * 16 + g + 8 * hh;
          if constexpr (C::k8) {
            float2 f;
            asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(f.x), "=f"(f.y) : "r"(st + 8192 + 8 * r) : "memory");
            ks = f.x;
            vsc[mt][hh] = f.y;
            vgrow |= f.y * rv > 64.f;
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float x = sc[nt][mt][2 * hh + c];
              if constexpr (C::k8) x *= ks;
              x *= colscale[nt][c];
              if (masked && key0 + r >= lim[nt][c]) x = -INFINITY;
              sc[nt][mt][2 * hh + c] = x;
              grow |= x > m[nt][c] + kGrow;
            }
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = m[nt][c];
#pragma unroll
            for (int mt = 0; mt < C::kMT; ++mt) x = fmaxf(x, fmaxf(sc[nt][mt][c], sc[nt][mt][2 + c]));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            const float f = x == -INFINITY ? 1.f : ptx::ex2_approx(m[nt][c] - x);
            m[nt][c] = x;
            l[nt][c] *= f;
#pragma unroll
            for (int k = 0; k < C::kKS; ++k) {
              o[nt][k][c] *= f;
              o[nt][k][2 + c] *= f;
            }
          }
      }
      if constexpr (C::k8) {
        if (__any_sync(0xffffffffu, vgrow)) {
          float x = 0.f;
#pragma unroll
          for (int mt = 0; mt < C::kMT; ++mt) x = fmaxf(x, fmaxf(vsc[mt][0], vsc[mt][1]));
#pragma unroll
          for (int w = 16; w > 0; w >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
          const float nref = __uint_as_float(__float_as_uint(x) & 0x7f800000u);
          rv = 1.f / nref;
          const float f = vref * rv;
          vref = nref;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < C::kKS; ++k)
#pragma unroll
              for (int i = 0; i < 4; ++i) o[nt][k][i] *= f;
        }
      }
      // P and O^T += V^T P^T
      uint32_t pb[NT][C::kMT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float n0 = m[nt][0] == -INFINITY ? 0.f : -m[nt][0];
        const float n1 = m[nt][1] == -INFINITY ? 0.f : -m[nt][1];
#pragma unroll
        for (int mt = 0; mt < C::kMT; ++mt)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            float p0 = ptx::ex2_approx(sc[nt][mt][2 * hh] + n0);
            float p1 = ptx::ex2_approx(sc[nt][mt][2 * hh + 1] + n1);
            l[nt][0] += p0;
            l[nt][1] += p1;
            if constexpr (C::k8) {
              const float f = vsc[mt][hh] * rv;
              p0 *= f;
              p1 *= f;
            }
            pb[nt][mt][hh] = transpose8(pack2f<C::kBf16>(p0, p1));
          }
      }
      if constexpr (!C::k8) {
#pragma unroll
        for (int mt = 0; mt < C::kMT; ++mt) {
          const int r = mt * 16 + (lane & 7) + ((lane & 16) ? 8 : 0);
          const uint32_t row = st + 4096 + r * C::kRowBytes;
#pragma unroll
          for (int k = 0; k < C::kKS; ++k) {
            uint32_t f[4];
            ldsm4t(row + (((2 * k + ((lane >> 3) & 1)) ^ C::swz(r)) << 4), f);
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
          const uint32_t row = st + 4096 + r * C::kRowBytes;
#pragma unroll
          for (int k = 0; k < C::kKS; ++k) {
            uint32_t f[4];
            ldsm4t(row + ((k ^ C::swz(r)) << 4), f);
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

    // ---- the segment's result
    const bool first = t_begin == 0, last = t_end == n_units;
    const float ov = C::k8 ? vref : 1.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x = l[nt][c];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        l[nt][c] = x;
      }
    // column of o[..][k][2 hh + c]
    auto col = [&](int k, int hh) { return C::k8 ? 16 * k + 2 * g + hh : 16 * k + g + 8 * hh; };
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = nt * 8 + 2 * j + c;
        if (r >= rows) continue;
        if (first && last) {
          const int tok = s.c0 + r / a.group, hq = cc.h * a.group + r % a.group;
          const float inv = l[nt][c] > 0.f ? ov / l[nt][c] : 0.f;
          uint16_t* dst = static_cast<uint16_t*>(a.o) + (static_cast<long long>(tok) * a.Hq + hq) * D;
#pragma unroll
          for (int k = 0; k < C::kKS; ++k) {
            const uint32_t w = pack2f<QBF16>(o[nt][k][c] * inv, o[nt][k][2 + c] * inv);
            if constexpr (C::k8) {
              *reinterpret_cast<uint32_t*>(dst + col(k, 0)) = w;
            } else {
              dst[col(k, 0)] = static_cast<uint16_t>(w & 0xffffu);
              dst[col(k, 1)] = static_cast<uint16_t>(w >> 16);
            }
          }
          if (g == 0 && a.lse != nullptr)
            a.lse[static_cast<long long>(hq) * a.r.total + tok] =
                l[nt][c] > 0.f ? (m[nt][c] + __log2f(l[nt][c])) * 0.69314718055994530942f : -INFINITY;
        } else {
          // slot 0: continues the head of an earlier warp; slot 1: begins one
          float* slot = p.ws + (2ll * wid + (first ? 1 : 0)) * slot_floats(8 * NT, D);
#pragma unroll
          for (int k = 0; k < C::kKS; ++k) {
            slot[r * D + col(k, 0)] = o[nt][k][c] * ov;
            slot[r * D + col(k, 1)] = o[nt][k][2 + c] * ov;
          }
          if (g == 0) {
            slot[8 * NT * D + r] = m[nt][c];
            slot[8 * NT * D + 8 * NT + r] = l[nt][c];
          }
        }
      }
    // ---- next segment
    u += t_end - t_begin;
    if (u < u1) {
      cc.t = t_end - 1;
      advance(cc);
    }
  }
  cp_wait<0>();
}

// Joins the partial results of (sequence, KV head) blockIdx.x, query row
// blockIdx.y: with M = max m_s over its slots in order of the warps,
//   O = sum 2^(m_s - M) O_s / sum 2^(m_s - M) l_s.
// Also writes the rows that no warp of the decode kernel computes: rows of
// sequences without visible keys and packed rows of no sequence.
template <int D, bool BF16>
__global__ void __launch_bounds__(kCombineThreads)
    paged_combine_kernel(const __grid_constant__ DecodeParams p, int sub, int slot_rows) {
  const PagedAttn& a = p.a;
  __shared__ long long sh[kCombineThreads / 32 + 1];
  __shared__ float sh_o[kCombineThreads / 32][D];
  __shared__ float sh_m[kCombineThreads / 32], sh_l[kCombineThreads / 32];
  const int b = blockIdx.x / a.c.heads, h = blockIdx.x % a.c.heads, row = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint16_t* out = static_cast<uint16_t*>(a.o);
  // rows of no sequence: before the first and after the last
  {
    const int head = min(max(__ldg(a.r.cu), 0), a.r.total);
    const int tail = min(max(__ldg(a.r.cu + a.r.B), head), a.r.total);
    const int n_out = head + a.r.total - tail;
    const int id = static_cast<int>(blockIdx.y * gridDim.x + blockIdx.x);
    for (int x = id; x < n_out; x += static_cast<int>(gridDim.x * gridDim.y)) {
      const int t = x < head ? x : tail + x - head;
      for (int i = threadIdx.x; i < a.Hq * D / 2; i += kCombineThreads)
        reinterpret_cast<uint32_t*>(out)[static_cast<long long>(t) * (a.Hq * D / 2) + i] = 0u;
      if (a.lse != nullptr)
        for (int i = threadIdx.x; i < a.Hq; i += kCombineThreads)
          a.lse[static_cast<long long>(i) * a.r.total + t] = -INFINITY;
    }
  }
  const Seq s = load_short(a, b, p.max_rows);
  const Spot sp = find_spot<kCombineThreads>(a, sub, p.max_rows, b, sh);
  // the decode kernel's results are complete and visible after this
  ptx::grid_dep_wait();
  if (row >= s.nq * a.group) return;
  const int tok = s.c0 + row / a.group, hq = h * a.group + row % a.group;
  uint16_t* dst = out + (static_cast<long long>(tok) * a.Hq + hq) * D;
  const int n = (s.vis + sub - 1) / sub;
  if (n == 0) {
    for (int i = threadIdx.x; i < D / 2; i += kCombineThreads) reinterpret_cast<uint32_t*>(dst)[i] = 0u;
    if (threadIdx.x == 0 && a.lse != nullptr)
      a.lse[static_cast<long long>(hq) * a.r.total + tok] = -INFINITY;
    return;
  }
  const long long total = sp.total * a.c.heads;
  const long long per = (total + p.n_warps - 1) / p.n_warps;
  const long long t0 = sp.before * a.c.heads + static_cast<long long>(h) * n;
  const int w0 = static_cast<int>(t0 / per), w1 = static_cast<int>((t0 + n - 1) / per);
  if (w0 == w1) return;  // one warp had it all
  const long long stride = slot_floats(slot_rows, D);
  auto slot_of = [&](int w) { return p.ws + (2ll * w + (w == w0 ? 1 : 0)) * stride; };
  // each warp joins every 8th slot, the block joins the warps
  constexpr int E = D / 32;
  float mm = -INFINITY, ll = 0.f, acc[E] = {};
  constexpr int kBatch = 4;
  for (int w = w0 + warp; w <= w1; w += kBatch * (kCombineThreads / 32)) {
    float mi[kBatch], li[kBatch], v[kBatch][E];
#pragma unroll
    for (int x = 0; x < kBatch; ++x) {
      const int ww = w + x * (kCombineThreads / 32);
      mi[x] = -INFINITY;
      li[x] = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) v[x][e] = 0.f;
      if (ww <= w1) {
        const float* sl = slot_of(ww);
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
    for (int x = 0; x < kBatch; ++x) {
      if (mi[x] == -INFINITY) continue;
      const float mn = fmaxf(mm, mi[x]);
      const float f0 = mm == -INFINITY ? 0.f : exp2f(mm - mn), f1 = exp2f(mi[x] - mn);
      mm = mn;
      ll = ll * f0 + li[x] * f1;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = acc[e] * f0 + v[x][e] * f1;
    }
  }
  if (lane == 0) {
    sh_m[warp] = mm;
    sh_l[warp] = ll;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) sh_o[warp][lane * E + e] = acc[e];
  __syncthreads();
  if (threadIdx.x < D / 2) {
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kCombineThreads / 32; ++w) M = fmaxf(M, sh_m[w]);
    float L = 0.f, x0 = 0.f, x1 = 0.f;
#pragma unroll
    for (int w = 0; w < kCombineThreads / 32; ++w) {
      const float f = sh_m[w] == -INFINITY ? 0.f : exp2f(sh_m[w] - M);
      L += f * sh_l[w];
      x0 += f * sh_o[w][2 * threadIdx.x];
      x1 += f * sh_o[w][2 * threadIdx.x + 1];
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;
    reinterpret_cast<uint32_t*>(dst)[threadIdx.x] = pack2f<BF16>(x0 * inv, x1 * inv);
    if (threadIdx.x == 0 && a.lse != nullptr)
      a.lse[static_cast<long long>(hq) * a.r.total + tok] =
          L > 0.f ? (M + log2f(L)) * 0.69314718055994530942f : -INFINITY;
  }
}

template <int D, int KV, bool QBF16, int NT>
cudaError_t launch_kv(const DecodeParams& p, int n_ctas, cudaStream_t stream) {
  using C = Cfg<D, KV>;
  auto kern = paged_decode_kernel<D, KV, QBF16, NT>;
  static int attr_done[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_done[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_done[dev] = 1;
  }
  kern<<<n_ctas, 32 * kWarps, C::kSmem, stream>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  // the combine may start while the last warps finish; it waits for them
  // before it reads a slot
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.a.r.B) * p.a.c.heads, p.max_rows);
  cfg.blockDim = dim3(kCombineThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_combine_kernel<D, QBF16>, p, static_cast<int>(C::kSub), 8 * NT);
}

template <int D, int KV, bool QBF16>
cudaError_t launch_nt(const DecodeParams& p, int n_ctas, cudaStream_t s) {
  return p.max_rows <= 8 ? launch_kv<D, KV, QBF16, 1>(p, n_ctas, s)
                         : launch_kv<D, KV, QBF16, 2>(p, n_ctas, s);
}

template <int D>
cudaError_t launch_d(const DecodeParams& p, int kv, bool bf16, int n_ctas, cudaStream_t s) {
  switch (kv) {
    case FA_DTYPE_INT8:
      return bf16 ? launch_nt<D, FA_DTYPE_INT8, true>(p, n_ctas, s)
                  : launch_nt<D, FA_DTYPE_INT8, false>(p, n_ctas, s);
    case FA_DTYPE_E4M3:
      return bf16 ? launch_nt<D, FA_DTYPE_E4M3, true>(p, n_ctas, s)
                  : launch_nt<D, FA_DTYPE_E4M3, false>(p, n_ctas, s);
    case FA_DTYPE_BF16: return launch_nt<D, FA_DTYPE_BF16, true>(p, n_ctas, s);
    default: return launch_nt<D, FA_DTYPE_F16, false>(p, n_ctas, s);
  }
}

int decode_ctas(int sms) { return sms * kCtasPerSm; }

}  // namespace

int paged_decode_rows() { return kRowsMax; }

size_t paged_decode_ws_bytes(int max_rows, int head_dim, int sms) {
  const int rows = max_rows <= 8 ? 8 : 16;
  return static_cast<size_t>(decode_ctas(sms)) * kWarps * 2 *
         static_cast<size_t>(slot_floats(rows, head_dim)) * sizeof(float);
}

cudaError_t launch_paged_decode(const PagedAttn& a, int max_rows, int head_dim, int cache_dtype,
                                bool bf16, int sms, void* workspace, cudaStream_t stream) {
  DecodeParams p;
  p.a = a;
  p.ws = static_cast<float*>(workspace);
  p.max_rows = max_rows;
  // no more warps than units there can be
  const int row_bytes = head_dim * (cache_dtype >= FA_DTYPE_INT8 ? 1 : 2);
  const int sub = 4096 / row_bytes;
  const long long units =
      static_cast<long long>(a.r.B) * a.c.heads * ((static_cast<long long>(a.max_k) + sub - 1) / sub);
  long long ctas = (units + kWarps - 1) / kWarps;
  if (ctas > decode_ctas(sms)) ctas = decode_ctas(sms);
  if (ctas < 1) ctas = 1;
  p.n_warps = static_cast<int>(ctas) * kWarps;
  return head_dim == 64 ? launch_d<64>(p, cache_dtype, bf16, static_cast<int>(ctas), stream)
                        : launch_d<128>(p, cache_dtype, bf16, static_cast<int>(ctas), stream);
}

}  // namespace fa
