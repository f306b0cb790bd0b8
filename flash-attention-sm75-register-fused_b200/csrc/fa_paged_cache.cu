// Writing K/V rows of new tokens into a paged cache and reading them back.
//
//   write  16-bit caches: a copy.  8-bit caches, per row x of d values:
//            a = max |x|,  scale = a / qmax,  q = round(x * (qmax / a))
//          with qmax = 127 (int8) or 448 (e4m3); fp32 arithmetic, one rounding
//          to 8 bits (4 significant bits in e4m3, 1/254 of a row's largest
//          value in int8), the scale kept in fp32.
//   read   x = q * scale in fp32, rounded once to f16 / bf16.
//
// Both move every byte once and compute little: they are bound by HBM, or by
// latency for a few tokens.  A row (d values of one token and head) is taken by
// the lanes that cover it with 16-byte loads, so the row's maximum is 3 or 4
// shuffles and both sides are coalesced.  Warps work alone: a warp takes U rows
// per lane group, finds the places of the few tokens they belong to (sequence
// by a 32-way search and ballots, page by one lookup per token: two dependent
// loads for up to 32 sequences, which overlap the source rows' own loads when
// writing) and keeps U independent 16-byte loads per lane in flight.
//
// Measured: 48 MB of bf16 rows of ragged prompts copied into pages 9.9 us (7.4 at
// the rate of a plain copy, 6.5 TB/s); 217 MB of int8 prefixes read back as bf16 38.3
// us (5.7 TB/s); eight tokens written and read back 4.8 us (two launches).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "fa_paged.h"
#include "fa_paged_dev.cuh"

namespace fa {
namespace {

constexpr int kCacheThreads = 128;
constexpr float kTinyRow = 7.8886090522101181e-31f;  // 2^-100

enum { kCopy = 0, kInt8 = 1, kE4m3 = 2 };

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t u) {
  if constexpr (BF16) {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u));
  } else {
    return __half22float2(*reinterpret_cast<__half2*>(&u));
  }
}

// max(|a|, |b|) per half of two pairs; a NaN stays.  `b` is a magnitude already.
template <bool BF16>
__device__ __forceinline__ uint32_t absmax2(uint32_t a, uint32_t b) {
  a &= 0x7fff7fffu;
  if constexpr (BF16) {
    const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  } else {
    const __half2 m = __hmax2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2_rn(float a, float b) {
  if constexpr (BF16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  }
}

// Place of one token: byte offset of its row (of head 0) in the pages, -1 if
// it has none, and offset of its scale.
struct Place {
  long long row, scale;
};
__device__ __forceinline__ long long shfl64(long long x, int src) {
  const int lo = __shfl_sync(0xffffffffu, static_cast<int>(x), src);
  const int hi = __shfl_sync(0xffffffffu, static_cast<int>(x >> 32), src);
  return (static_cast<long long>(hi) << 32) | static_cast<unsigned>(lo);
}

// Places of packed rows t0 .. t0 + n - 1 (n <= 32): lane i gets that of row
// t0 + i.  The whole warp calls it.
__device__ __forceinline__ Place find_places(const PagedCache& c, const PagedRows& r, int t0, int n) {
  const int lane = threadIdx.x & 31;
  // a sequence that starts at or before t0, by 32-way steps
  int b0 = 0;
  for (int len = r.B; len > 32;) {
    const int step = (len + 31) / 32;
    const int probe = b0 + lane * step;
    const bool le = lane * step < len && __ldg(r.cu + probe) <= t0;
    const int cnt = __popc(__ballot_sync(0xffffffffu, le));
    const int skip = max(cnt - 1, 0) * step;
    b0 += skip;
    len = min(step, len - skip);
  }
  int b = -1, pos = -1;  // of token t0 + lane
  const int t = t0 + lane;
  for (; b0 < r.B; b0 += 32) {
    int c0 = 0x7fffffff, c1 = 0, last = 0;
    if (b0 + lane < r.B) {
      c0 = max(__ldg(r.cu + b0 + lane), 0);
      c1 = min(__ldg(r.cu + b0 + lane + 1), r.total);
      last = __ldg(r.lens + b0 + lane) - c1;  // position of row t is last + t
    }
    // the sequences that have some of the rows (one or two, mostly)
    for (unsigned left = __ballot_sync(0xffffffffu, c0 < t0 + n && c1 > t0 && c0 < c1); left != 0u;
         left &= left - 1u) {
      const int src = __ffs(left) - 1;
      const int s0 = __shfl_sync(0xffffffffu, c0, src), s1 = __shfl_sync(0xffffffffu, c1, src);
      const int l = __shfl_sync(0xffffffffu, last, src);
      if (t >= s0 && t < s1 && lane < n) {
        b = b0 + src;
        pos = l + t;
      }
    }
    if (__shfl_sync(0xffffffffu, c1, 31) >= t0 + n) break;  // (0 past the last sequence)
  }
  const int page = b >= 0 && pos >= 0 ? c.lookup(b, pos) : -1;
  if (page < 0) return {-1, 0};
  const long long row = c.row_in_page(pos);
  return {page * c.page_stride + row * c.row_stride, page * c.s_page + row * c.s_row};
}

// Rows go token by token, the K heads of a token before its V heads.  A warp's
// first row has token t0 (and is `skip` rows into it); `magic` = 2^32 / (2
// heads) rounded up divides the small row numbers within a warp.
struct RowMap {
  unsigned n_rows;  // total * 2 * heads
  unsigned magic;
};
struct RowId {
  int token, kv, head;  // token: relative to t0
};
__device__ __forceinline__ RowId row_id(unsigned rel, int heads, unsigned magic) {
  const int t = static_cast<int>(__umulhi(rel, magic));
  const int rem = static_cast<int>(rel) - t * 2 * heads;
  return {t, rem >= heads ? 1 : 0, rem >= heads ? rem - heads : rem};
}

// A lane holds 8 (copies) or 16 (8-bit) values of a row: those at 8 * part and,
// for 8-bit pages, at d / 2 + 8 * part, so that every load and store of a lane
// group is one contiguous run on both sides.
template <int D, bool BF16, int KIND, int U>
__global__ void __launch_bounds__(kCacheThreads) cache_write_kernel(const PagedCache c,
                                                                   const PagedRows r,
                                                                   const PagedSource s,
                                                                   const RowMap map) {
  constexpr int kPer = KIND == kCopy ? 1 : 2;  // 16-byte loads of a lane
  constexpr int L = D / (8 * kPer);            // lanes per row
  constexpr int kRows = 32 / L;
  const int lane = threadIdx.x & 31, part = lane % L;
  const unsigned row0 = (blockIdx.x * (kCacheThreads / 32) + (threadIdx.x >> 5)) * (kRows * U);
  if (row0 >= map.n_rows) return;
  const unsigned heads2 = 2u * c.heads;
  const int t0 = static_cast<int>(row0 / heads2);
  const unsigned skip = row0 - t0 * heads2;
  const int n_tokens = row_id(skip + min(kRows * U, map.n_rows - row0) - 1u, c.heads, map.magic).token + 1;
  RowId id[U];
  uint4 x[U][kPer];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    id[u] = row_id(skip + u * kRows + lane / L, c.heads, map.magic);
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[u][i] = make_uint4(0u, 0u, 0u, 0u);
    if (row0 + u * kRows + lane / L < map.n_rows) {
      const long long t = static_cast<long long>(t0) + id[u].token;
      const uint8_t* src = id[u].kv ? s.v + t * s.v_token + id[u].head * s.v_head
                                    : s.k + t * s.k_token + id[u].head * s.k_head;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        x[u][i] = __ldcs(reinterpret_cast<const uint4*>(src) + i * (D / 16) + part);
    }
  }
  const Place pl = find_places(c, r, t0, n_tokens);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long found = shfl64(pl.row, id[u].token);
    const bool ok = found >= 0 && row0 + u * kRows + lane / L < map.n_rows;
    uint8_t* dst = const_cast<uint8_t*>(id[u].kv ? c.v : c.k) + found + id[u].head * c.head_stride;
    if constexpr (KIND == kCopy) {
      if (ok) reinterpret_cast<uint4*>(dst)[part] = x[u][0];
    } else {
      const uint32_t in8[8] = {x[u][0].x, x[u][0].y, x[u][0].z, x[u][0].w,
                               x[u][1].x, x[u][1].y, x[u][1].z, x[u][1].w};
      uint32_t m = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = absmax2<BF16>(in8[i], m);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) m = absmax2<BF16>(__shfl_xor_sync(0xffffffffu, m, o), m);
      const float2 m2 = unpack2<BF16>(m);
      const float a = m2.x != m2.x ? m2.x : (m2.y > m2.x || m2.y != m2.y ? m2.y : m2.x);
      constexpr float kQmax = KIND == kInt8 ? 127.f : 448.f;
      const bool zero = a < kTinyRow;
      const float inv = zero ? 0.f : __fdiv_rn(kQmax, a);
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 y0 = unpack2<BF16>(in8[2 * i]), y1 = unpack2<BF16>(in8[2 * i + 1]);
        const float f0 = __fmul_rn(y0.x, inv), f1 = __fmul_rn(y0.y, inv);
        const float f2 = __fmul_rn(y1.x, inv), f3 = __fmul_rn(y1.y, inv);
        if constexpr (KIND == kInt8) {
          // 1.5 * 2^23 + y rounds y to an integer (ties to even) in the low
          // mantissa bits; |y| <= 127 (1 + 2^-23), so the low byte is the value
          auto q8 = [](float y) { return __float_as_uint(__fadd_rn(y, 12582912.f)); };
          w[i] = __byte_perm(__byte_perm(q8(f0), q8(f1), 0x0040), __byte_perm(q8(f2), q8(f3), 0x0040), 0x5410);
        } else {
          const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f0, f1), __NV_SATFINITE, __NV_E4M3);
          const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f2, f3), __NV_SATFINITE, __NV_E4M3);
          w[i] = lo | (hi << 16);
        }
      }
      const long long so = shfl64(pl.scale, id[u].token);
      if (ok) {
        reinterpret_cast<uint2*>(dst)[part] = make_uint2(w[0], w[1]);
        reinterpret_cast<uint2*>(dst)[D / 16 + part] = make_uint2(w[2], w[3]);
        // (an infinite or NaN maximum makes the scale NaN)
        if (part == 0)
          (id[u].kv ? c.vs : c.ks)[so + id[u].head * c.s_head] =
              zero ? 0.f : __fdiv_rn(a, kQmax) + (a - a);
      }
    }
  }
}

template <int D, bool BF16, int KIND, int U>
__global__ void __launch_bounds__(kCacheThreads) cache_read_kernel(const PagedCache c,
                                                                  const PagedRows r,
                                                                  uint4* __restrict__ k,
                                                                  uint4* __restrict__ v,
                                                                  const RowMap map) {
  constexpr int kPer = KIND == kCopy ? 1 : 2;  // 16-byte results of a lane
  constexpr int L = D / (8 * kPer);            // lanes per row
  constexpr int kRows = 32 / L;
  const int lane = threadIdx.x & 31, part = lane % L;
  const unsigned row0 = (blockIdx.x * (kCacheThreads / 32) + (threadIdx.x >> 5)) * (kRows * U);
  if (row0 >= map.n_rows) return;
  const unsigned heads2 = 2u * c.heads;
  const int t0 = static_cast<int>(row0 / heads2);
  const unsigned skip = row0 - t0 * heads2;
  const int n_tokens = row_id(skip + min(kRows * U, map.n_rows - row0) - 1u, c.heads, map.magic).token + 1;
  const Place pl = find_places(c, r, t0, n_tokens);
  RowId id[U];
  uint4 x[U];
  float scale[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    id[u] = row_id(skip + u * kRows + lane / L, c.heads, map.magic);
    const long long found = shfl64(pl.row, id[u].token);
    const long long so = KIND != kCopy ? shfl64(pl.scale, id[u].token) : 0;
    x[u] = make_uint4(0u, 0u, 0u, 0u);
    scale[u] = 0.f;
    if (found >= 0 && row0 + u * kRows + lane / L < map.n_rows) {
      const uint8_t* src = (id[u].kv ? c.v : c.k) + found + id[u].head * c.head_stride;
      if constexpr (KIND == kCopy) {
        x[u] = __ldcs(reinterpret_cast<const uint4*>(src) + part);
      } else {
        const uint2 lo = __ldcs(reinterpret_cast<const uint2*>(src) + part);
        const uint2 hi = __ldcs(reinterpret_cast<const uint2*>(src) + D / 16 + part);
        x[u] = make_uint4(lo.x, lo.y, hi.x, hi.y);
      }
      if constexpr (KIND != kCopy) scale[u] = __ldg((id[u].kv ? c.vs : c.ks) + so + id[u].head * c.s_head);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (row0 + u * kRows + lane / L >= map.n_rows) continue;
    uint4* dst = (id[u].kv ? v : k) +
                 ((static_cast<long long>(t0) + id[u].token) * c.heads + id[u].head) * (D / 8) + part;
    if constexpr (KIND == kCopy) {
      __stcs(dst, x[u]);
    } else {
      const uint32_t in[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t p[2];  // the values as f16, exactly
        widen<KIND == kInt8 ? FA_DTYPE_INT8 : FA_DTYPE_E4M3, false>(in[i], p[0], p[1]);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float2 f = unpack2<false>(p[y]);
          w[2 * i + y] = pack2_rn<BF16>(__fmul_rn(f.x, scale[u]), __fmul_rn(f.y, scale[u]));
        }
      }
      __stcs(dst, make_uint4(w[0], w[1], w[2], w[3]));
      __stcs(dst + D / 16, make_uint4(w[4], w[5], w[6], w[7]));
    }
  }
}

// U rows per lane group, each an independent load per lane: 4 for copies, 2 for
// 8-bit pages, whose rows take more registers and instructions; few rows spread
// over more warps instead.  Measured on B200 (GPU time; 128 threads, U = 1 / 2 /
// 4): 195 MB of f16 rows read back 44 / 36 / 33 us, 217 MB of int8 45 / 39 / 44;
// 256 threads +2 %, 512 +7-15 %.
template <int KIND>
constexpr int kRowsInFlight = KIND == kCopy ? 4 : 2;
template <int kRowsPerU>
unsigned blocks_for(unsigned n_rows, int u) {
  const unsigned per = kCacheThreads / 32 * kRowsPerU * u;
  return (n_rows + per - 1) / per;
}
RowMap row_map(const PagedCache& c, const PagedRows& r) {
  const unsigned heads2 = 2u * c.heads;
  return {static_cast<unsigned>(r.total) * heads2,
          static_cast<unsigned>(((1ull << 32) + heads2 - 1) / heads2)};
}
// Few rows: up to 64 for each of the 148 SMs.  One row per lane group / more, bf16
// rows written (us): at d = 128 1024 rows 2.1 / 2.3, 9472 2.8 / 2.9, 18944 3.6 / 3.3,
// 75776 9.8 / 7.4 (int8: 2.6 / 2.9, 2.9 / 3.2, 3.6 / 3.5, 8.6 / 7.9); at d = 64 9472 2.6 /
// 2.7, 37888 3.7 / 3.3 (int8: 2.7 / 2.9, 3.5 / 3.5); reading is alike.
bool few_rows(unsigned n_rows) { return n_rows <= 148u * 64u; }

template <int D, bool BF16, int KIND>
cudaError_t write_impl(const PagedCache& c, const PagedRows& r, const PagedSource& s,
                       cudaStream_t stream) {
  const RowMap m = row_map(c, r);
  constexpr int kRows = (KIND == kCopy ? 256 : 512) / D;
  if (few_rows(m.n_rows))
    cache_write_kernel<D, BF16, KIND, 1>
        <<<blocks_for<kRows>(m.n_rows, 1), kCacheThreads, 0, stream>>>(c, r, s, m);
  else
    cache_write_kernel<D, BF16, KIND, kRowsInFlight<KIND>>
        <<<blocks_for<kRows>(m.n_rows, kRowsInFlight<KIND>), kCacheThreads, 0, stream>>>(c, r, s, m);
  return cudaGetLastError();
}

template <int D, bool BF16, int KIND>
cudaError_t read_impl(const PagedCache& c, const PagedRows& r, void* k, void* v,
                      cudaStream_t stream) {
  const RowMap m = row_map(c, r);
  constexpr int kRows = (KIND == kCopy ? 256 : 512) / D;
  uint4* k4 = static_cast<uint4*>(k);
  uint4* v4 = static_cast<uint4*>(v);
  if (few_rows(m.n_rows))
    cache_read_kernel<D, BF16, KIND, 1>
        <<<blocks_for<kRows>(m.n_rows, 1), kCacheThreads, 0, stream>>>(c, r, k4, v4, m);
  else
    cache_read_kernel<D, BF16, KIND, kRowsInFlight<KIND>>
        <<<blocks_for<kRows>(m.n_rows, kRowsInFlight<KIND>), kCacheThreads, 0, stream>>>(c, r, k4, v4, m);
  return cudaGetLastError();
}

// A copy is the same for f16 and bf16.
template <int D>
cudaError_t write_d(const PagedCache& c, const PagedRows& r, const PagedSource& s, int cache_dtype,
                    bool bf16, cudaStream_t st) {
  if (cache_dtype == FA_DTYPE_INT8)
    return bf16 ? write_impl<D, true, kInt8>(c, r, s, st) : write_impl<D, false, kInt8>(c, r, s, st);
  if (cache_dtype == FA_DTYPE_E4M3)
    return bf16 ? write_impl<D, true, kE4m3>(c, r, s, st) : write_impl<D, false, kE4m3>(c, r, s, st);
  return write_impl<D, false, kCopy>(c, r, s, st);
}

template <int D>
cudaError_t read_d(const PagedCache& c, const PagedRows& r, void* k, void* v, int cache_dtype,
                   bool bf16, cudaStream_t st) {
  if (cache_dtype == FA_DTYPE_INT8)
    return bf16 ? read_impl<D, true, kInt8>(c, r, k, v, st) : read_impl<D, false, kInt8>(c, r, k, v, st);
  if (cache_dtype == FA_DTYPE_E4M3)
    return bf16 ? read_impl<D, true, kE4m3>(c, r, k, v, st) : read_impl<D, false, kE4m3>(c, r, k, v, st);
  return read_impl<D, false, kCopy>(c, r, k, v, st);
}

}  // namespace

cudaError_t launch_cache_write(const PagedCache& c, const PagedRows& r, const PagedSource& s,
                               int head_dim, int cache_dtype, bool bf16, cudaStream_t stream) {
  return head_dim == 64 ? write_d<64>(c, r, s, cache_dtype, bf16, stream)
                        : write_d<128>(c, r, s, cache_dtype, bf16, stream);
}

cudaError_t launch_cache_read(const PagedCache& c, const PagedRows& r, void* k, void* v,
                              int head_dim, int cache_dtype, bool bf16, cudaStream_t stream) {
  return head_dim == 64 ? read_d<64>(c, r, k, v, cache_dtype, bf16, stream)
                        : read_d<128>(c, r, k, v, cache_dtype, bf16, stream);
}

}  // namespace fa
