// Device helpers of the paged attention kernels: a sequence's part in a call,
// the block-wide scan over sequences, 8-bit values widened to f16, the
// register-operand product and the join of two passes.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "fa_paged.h"

namespace fa {
namespace {

// Two pairs of 8-bit values of a word as f16 pairs, exactly: bytes (0, 1) and
// (2, 3), or with kCross bytes (0, 2) and (1, 3).
// int8: x ^ 0x80 = x + 128 in the low byte of the f16 1024 + (x + 128).
template <int KV, bool kCross>
__device__ __forceinline__ void widen(uint32_t w, uint32_t& p0, uint32_t& p1) {
  if constexpr (KV == FA_DTYPE_INT8) {
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t a = __byte_perm(u, 0x64646464u, kCross ? 0x4240 : 0x4140);
    const uint32_t b = __byte_perm(u, 0x64646464u, kCross ? 0x4341 : 0x4342);
    const __half2 off = __half2half2(__ushort_as_half(0x6480));  // 1152
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    p0 = *reinterpret_cast<const uint32_t*>(&x);
    p1 = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    const uint32_t u = kCross ? __byte_perm(w, 0u, 0x3120) : w;
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "mov.b32 {lo, hi}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, lo;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, hi;\n\t}\n"
        : "=r"(p0), "=r"(p1)
        : "r"(u));
  }
}

// m16n8k16 product of 16-bit registers, fp32 sums.
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

// bf16 queries over 8-bit pages are taken as f16, q / 2^e with 2^e the size of the
// row's largest element (2^e <= max |q| < 2^(e+1)): bf16's 8 bits fit f16's 11, and elements
// below 2^-14 of the largest lose at most 2^-25 of it, no more than the sum in fp32 does.
// A quad's lanes have a row, N pairs each (at(i): pair i); returns 2^e.
template <int N, typename At>
__device__ __forceinline__ float bf16_row_as_f16(At at) {
  float mx = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float2 f = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&at(i)));
    mx = fmaxf(mx, fmaxf(fabsf(f.x), fabsf(f.y)));
  }
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
  const uint32_t e = __float_as_uint(mx) & 0x7f800000u;
  const bool plain = e == 0u || e >= 0x7e800000u;
  const float inv = plain ? 1.f : __uint_as_float(0x7f000000u - e);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float2 f = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&at(i)));
    const __half2 x = __floats2half2_rn(f.x * inv, f.y * inv);
    at(i) = *reinterpret_cast<const uint32_t*>(&x);
  }
  return plain ? 1.f : __uint_as_float(e);
}

// What a sequence brings to a call.
struct Seq {
  int c0, n, nq; // first packed row; new tokens; those of them that are computed
  int nk, off;   // visible keys: key j < lim(i) = min(nk, i + off + 1) (causal) or nk;
                 // off goes by the whole length, also where bounds cut nk
  int vis;       // keys any of its rows may see
};

__device__ __forceinline__ int row_limit(const PagedAttn& a, const Seq& s, int i) {
  return a.causal == FA_CAUSAL_NONE ? s.nk : max(min(s.nk, i + s.off + 1), 0);
}

__device__ __forceinline__ Seq load_seq(const PagedAttn& a, int b) {
  Seq s;
  const int c0 = min(max(__ldg(a.r.cu + b), 0), a.r.total);
  const int c1 = min(max(__ldg(a.r.cu + b + 1), c0), a.r.total);
  // (beyond 2^30 keys and 2^28 new tokens every token sees all keys a table can hold)
  const int len = min(max(__ldg(a.r.lens + b), 0), 3 << 29);
  const int n = c1 - c0;
  s.c0 = c0;
  s.n = n;
  s.nq = min(n, a.max_q);
  s.nk = min(min(len, a.max_k), a.c.max_pages * a.c.page_size);
  s.off = a.causal == FA_CAUSAL_BOTTOM_RIGHT ? len - n : 0;
  s.vis = s.nq > 0 ? row_limit(a, s, s.nq - 1) : 0;
  return s;
}

// Result of a row of the second pass with that of the first: O = own O_2 + first
// O_1, LSE.  (Without keys in a set its weight is 0; without any, all are.  A NaN of either
// set stays one, also beside a set without keys: the maximum of NaN and -inf is -inf, so
// it does not tell rows without keys.)
struct Joined {
  float own, first, lse;
};
__device__ __forceinline__ Joined join_passes(float lse_first, float lse_own) {
  if (lse_first == -INFINITY && lse_own == -INFINITY) return {0.f, 0.f, -INFINITY};
  const float m = fmaxf(lse_first, lse_own);
  const float f1 = expf(lse_first - m), f2 = expf(lse_own - m);
  const float sum = f1 + f2;
  return {f2 / sum, f1 / sum, m + logf(sum)};
}

// O = 0, LSE = -inf in packed row t, which no kernel computes.  (Also below: all
// threads of a block call it.)
__device__ __forceinline__ void fill_row(const PagedAttn& a, int d, int t) {
  const int n = static_cast<int>(blockDim.x);
  if (kPartRows && (a.part == kPartFirst || a.part == kPartSecond)) {
    const float none = a.part == kPartFirst ? -INFINITY : __uint_as_float(kNoRow);
    for (int i = threadIdx.x; i < a.Hq * d; i += n) *a.part_at(static_cast<long long>(t) * a.Hq + i / d, i % d) = 0.f;
    for (int i = threadIdx.x; i < a.Hq; i += n) a.part_lse[static_cast<long long>(t) * a.Hq + i] = none;
    return;
  }
  const int words = a.Hq * d / 2;
  for (int i = threadIdx.x; i < words; i += n)
    static_cast<uint32_t*>(a.o)[static_cast<long long>(t) * words + i] = 0u;
  if (a.lse != nullptr)
    for (int i = threadIdx.x; i < a.Hq; i += n) a.lse[static_cast<long long>(i) * a.r.total + t] = -INFINITY;
}
// The rows of no sequence (before the first and after the last), dealt over the
// grid's blocks.
__device__ __forceinline__ void fill_outside(const PagedAttn& a, int d, int block, int n_blocks) {
  const int head = a.r.B > 0 ? min(max(__ldg(a.r.cu), 0), a.r.total) : a.r.total;
  const int tail = a.r.B > 0 ? min(max(__ldg(a.r.cu + a.r.B), head), a.r.total) : a.r.total;
  const int n_out = head + a.r.total - tail;
  for (int x = block; x < n_out; x += n_blocks) fill_row(a, d, x < head ? x : tail + x - head);
}
// The tokens of a sequence beyond max_q.
__device__ __forceinline__ void fill_beyond(const PagedAttn& a, int d, const Seq& s) {
  for (int i = a.max_q; i < s.n; ++i) fill_row(a, d, s.c0 + i);
}

// Exclusive prefix sum of `sum` over the block's threads; *total its sum.
// sh: one entry per warp.
template <int kThreads>
__device__ __forceinline__ long long block_scan(long long sum, long long* sh, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) sh[warp] = incl;
  __syncthreads();
  long long base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    const long long v = sh[w];
    if (w < warp) base += v;
    all += v;
  }
  *total = all;
  return base + incl - sum;
}

}  // namespace
}  // namespace fa
