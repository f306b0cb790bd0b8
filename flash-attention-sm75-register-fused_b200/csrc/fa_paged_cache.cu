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
// latency for a few tokens.  A row (d values of one token and head) is taken
// by d / 8 lanes, 16 bytes each on the 16-bit side, so the row's maximum is 3
// or 4 shuffles and both sides are coalesced.  A CTA takes `U` rows per lane
// group; their places (sequence, position, page) are found once per token in
// shared memory, in three dependent loads (cu_seqlens / seqlens, table) that
// overlap the source rows' own loads when writing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "fa_paged.h"

namespace fa {
namespace {

constexpr int kCacheThreads = 256;
constexpr float kTinyRow = 7.8886090522101181e-31f;  // 2^-100

enum { kCopy = 0, kInt8 = 1, kE4m3 = 2 };

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t u) {
  if constexpr (BF16) {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u));
  } else {
    return __half22float2(*reinterpret_cast<__half2*>(&u));
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

// Places of the tokens a CTA handles: page (-1: none) and row in the page.
struct Places {
  static constexpr int kMax = 2 * kCacheThreads / 8 * 4 / 2 + 2;  // see rows_per_cta
  int page[kMax];
  int row[kMax];
};

// Fills pl for packed rows [t0, t0 + n): every thread checks its share of the
// sequences for tokens of that range, then one thread per token looks up its
// page.  Ends with a barrier.
__device__ __forceinline__ void find_places(const PagedCache& c, const PagedRows& r, int t0, int n,
                                            Places& pl) {
  for (int i = threadIdx.x; i < n; i += kCacheThreads) pl.page[i] = -1;
  __syncthreads();
  for (int b = threadIdx.x; b < r.B; b += kCacheThreads) {
    const int c0 = max(__ldg(r.cu + b), 0);
    const int c1 = min(__ldg(r.cu + b + 1), r.total);
    const int last = __ldg(r.lens + b) - c1;  // position of row t is last + t
    const int hi = min(c1, t0 + n);
    for (int t = max(c0, t0); t < hi; ++t) {
      pl.page[t - t0] = b;
      pl.row[t - t0] = last + t;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kCacheThreads) {
    const int b = pl.page[i], pos = pl.row[i];
    const int page = (b >= 0 && pos >= 0) ? c.lookup(b, pos) : -1;
    pl.page[i] = page;
    pl.row[i] = page >= 0 ? c.row_in_page(pos) : 0;
  }
  __syncthreads();
}

template <int D, int U>
__host__ __device__ constexpr int rows_per_cta() {
  return kCacheThreads / (D / 8) * U;
}

// Row number -> token (relative to t0), K or V, head: rows go token by token,
// the K heads of a token before its V heads.
struct RowId {
  int token, kv, head;
};
__device__ __forceinline__ RowId row_id(long long row, int heads) {
  const long long t = row / (2 * heads);
  const int rem = static_cast<int>(row - t * (2 * heads));
  return {static_cast<int>(t), rem >= heads ? 1 : 0, rem >= heads ? rem - heads : rem};
}

template <int D, bool BF16, int KIND, int U>
__global__ void __launch_bounds__(kCacheThreads) cache_write_kernel(const PagedCache c,
                                                                   const PagedRows r,
                                                                   const PagedSource s) {
  constexpr int L = D / 8;  // lanes per row
  constexpr int kRows = kCacheThreads / L;
  __shared__ Places pl;
  const long long n_rows = static_cast<long long>(r.total) * 2 * c.heads;
  const long long row0 = static_cast<long long>(blockIdx.x) * (kRows * U);
  const int part = threadIdx.x % L;
  RowId id[U];
  uint4 x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long row = row0 + u * kRows + threadIdx.x / L;
    id[u].token = -1;
    x[u] = make_uint4(0u, 0u, 0u, 0u);
    if (row < n_rows) {
      id[u] = row_id(row, c.heads);
      const uint8_t* src =
          id[u].kv ? s.v + id[u].token * s.v_token + id[u].head * s.v_head
                   : s.k + id[u].token * s.k_token + id[u].head * s.k_head;
      x[u] = __ldcs(reinterpret_cast<const uint4*>(src) + part);
    }
  }
  const int t0 = row_id(row0, c.heads).token;
  const long long last = min(row0 + kRows * U, n_rows) - 1;
  find_places(c, r, t0, row_id(last, c.heads).token - t0 + 1, pl);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int page = id[u].token >= 0 ? pl.page[id[u].token - t0] : -1;
    const int prow = id[u].token >= 0 ? pl.row[id[u].token - t0] : 0;
    uint8_t* dst = const_cast<uint8_t*>(id[u].kv ? c.v : c.k) + page * c.page_stride +
                   id[u].head * c.head_stride + prow * c.row_stride;
    if constexpr (KIND == kCopy) {
      if (page >= 0) reinterpret_cast<uint4*>(dst)[part] = x[u];
    } else {
      float2 v[4] = {unpack2<BF16>(x[u].x), unpack2<BF16>(x[u].y), unpack2<BF16>(x[u].z),
                     unpack2<BF16>(x[u].w)};
      float a = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) a = max_nan(a, max_nan(fabsf(v[i].x), fabsf(v[i].y)));
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
      constexpr float kQmax = KIND == kInt8 ? 127.f : 448.f;
      const bool zero = a < kTinyRow;
      const float inv = zero ? 0.f : __fdiv_rn(kQmax, a);
      const float scale = zero ? 0.f : __fdiv_rn(a, kQmax);
      uint32_t w[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float y0 = __fmul_rn(v[2 * i].x, inv), y1 = __fmul_rn(v[2 * i].y, inv);
        const float y2 = __fmul_rn(v[2 * i + 1].x, inv), y3 = __fmul_rn(v[2 * i + 1].y, inv);
        if constexpr (KIND == kInt8) {
          auto q8 = [](float y) {
            return static_cast<uint32_t>(min(max(__float2int_rn(y), -127), 127)) & 0xffu;
          };
          w[i] = q8(y0) | (q8(y1) << 8) | (q8(y2) << 16) | (q8(y3) << 24);
        } else {
          const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y0, y1), __NV_SATFINITE, __NV_E4M3);
          const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y2, y3), __NV_SATFINITE, __NV_E4M3);
          w[i] = lo | (hi << 16);
        }
      }
      if (page >= 0) {
        reinterpret_cast<uint2*>(dst)[part] = make_uint2(w[0], w[1]);
        if (part == 0)
          (id[u].kv ? c.vs : c.ks)[page * c.s_page + id[u].head * c.s_head + prow * c.s_row] =
              scale;
      }
    }
  }
}

template <int D, bool BF16, int KIND, int U>
__global__ void __launch_bounds__(kCacheThreads) cache_read_kernel(const PagedCache c,
                                                                  const PagedRows r,
                                                                  uint4* __restrict__ k,
                                                                  uint4* __restrict__ v) {
  constexpr int L = D / 8;
  constexpr int kRows = kCacheThreads / L;
  __shared__ Places pl;
  const long long n_rows = static_cast<long long>(r.total) * 2 * c.heads;
  const long long row0 = static_cast<long long>(blockIdx.x) * (kRows * U);
  const int part = threadIdx.x % L;
  const int t0 = row_id(row0, c.heads).token;
  const long long last = min(row0 + kRows * U, n_rows) - 1;
  find_places(c, r, t0, row_id(last, c.heads).token - t0 + 1, pl);
  uint4 x[U];
  float scale[U];
  RowId id[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long row = row0 + u * kRows + threadIdx.x / L;
    id[u].token = -1;
    x[u] = make_uint4(0u, 0u, 0u, 0u);
    scale[u] = 0.f;
    if (row < n_rows) {
      id[u] = row_id(row, c.heads);
      const int page = pl.page[id[u].token - t0], prow = pl.row[id[u].token - t0];
      if (page >= 0) {
        const uint8_t* src = (id[u].kv ? c.v : c.k) + page * c.page_stride +
                             id[u].head * c.head_stride + prow * c.row_stride;
        if constexpr (KIND == kCopy) {
          x[u] = __ldg(reinterpret_cast<const uint4*>(src) + part);
        } else {
          const uint2 t = __ldg(reinterpret_cast<const uint2*>(src) + part);
          x[u].x = t.x;
          x[u].y = t.y;
          scale[u] = __ldg((id[u].kv ? c.vs : c.ks) + page * c.s_page + id[u].head * c.s_head +
                           prow * c.s_row);
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (id[u].token < 0) continue;
    if constexpr (KIND != kCopy) {
      uint32_t w[4];
      const uint32_t in[2] = {x[u].x, x[u].y};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t two = in[i / 2] >> (16 * (i & 1));
        float y0, y1;
        if constexpr (KIND == kInt8) {
          y0 = static_cast<float>(static_cast<int8_t>(two & 0xffu));
          y1 = static_cast<float>(static_cast<int8_t>((two >> 8) & 0xffu));
        } else {
          const __half2_raw h =
              __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xffffu), __NV_E4M3);
          const float2 f = __half22float2(__half2(h));
          y0 = f.x;
          y1 = f.y;
        }
        w[i] = pack2_rn<BF16>(__fmul_rn(y0, scale[u]), __fmul_rn(y1, scale[u]));
      }
      x[u] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    uint4* dst = (id[u].kv ? v : k) +
                 (static_cast<long long>(id[u].token) * c.heads + id[u].head) * (D / 8) + part;
    __stcs(dst, x[u]);
  }
}

// U rows per lane group: 4 keep 4 independent loads in flight per thread; few
// rows spread over more CTAs instead.
bool few_rows(long long n_rows, int head_dim) {
  return n_rows <= 2LL * 148 * (kCacheThreads / (head_dim / 8));
}

template <int D, bool BF16, int KIND>
cudaError_t write_impl(const PagedCache& c, const PagedRows& r, const PagedSource& s,
                       cudaStream_t stream) {
  const long long n_rows = static_cast<long long>(r.total) * 2 * c.heads;
  if (few_rows(n_rows, D)) {
    const unsigned grid = static_cast<unsigned>((n_rows + rows_per_cta<D, 1>() - 1) / rows_per_cta<D, 1>());
    cache_write_kernel<D, BF16, KIND, 1><<<grid, kCacheThreads, 0, stream>>>(c, r, s);
  } else {
    const unsigned grid = static_cast<unsigned>((n_rows + rows_per_cta<D, 4>() - 1) / rows_per_cta<D, 4>());
    cache_write_kernel<D, BF16, KIND, 4><<<grid, kCacheThreads, 0, stream>>>(c, r, s);
  }
  return cudaGetLastError();
}

template <int D, bool BF16, int KIND>
cudaError_t read_impl(const PagedCache& c, const PagedRows& r, void* k, void* v,
                      cudaStream_t stream) {
  const long long n_rows = static_cast<long long>(r.total) * 2 * c.heads;
  uint4* k4 = static_cast<uint4*>(k);
  uint4* v4 = static_cast<uint4*>(v);
  if (few_rows(n_rows, D)) {
    const unsigned grid = static_cast<unsigned>((n_rows + rows_per_cta<D, 1>() - 1) / rows_per_cta<D, 1>());
    cache_read_kernel<D, BF16, KIND, 1><<<grid, kCacheThreads, 0, stream>>>(c, r, k4, v4);
  } else {
    const unsigned grid = static_cast<unsigned>((n_rows + rows_per_cta<D, 4>() - 1) / rows_per_cta<D, 4>());
    cache_read_kernel<D, BF16, KIND, 4><<<grid, kCacheThreads, 0, stream>>>(c, r, k4, v4);
  }
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
