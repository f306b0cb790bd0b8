// Attention of new tokens over a paged KV cache: one CTA per (token, query
// head), four warps that take every fourth key, online softmax per warp.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "fa_paged.h"

namespace fa {
namespace {

template <bool BF16>
__device__ __forceinline__ float to_f32(uint16_t u) {
  if constexpr (BF16) return __bfloat162float(__ushort_as_bfloat16(u));
  else return __half2float(__ushort_as_half(u));
}

template <int D, bool BF16, int DTYPE>
__device__ __forceinline__ void load_row(const uint8_t* row, int lane, float scale,
                                         float (&x)[D / 32]) {
#pragma unroll
  for (int e = 0; e < D / 32; ++e) {
    const int i = lane + 32 * e;
    if constexpr (DTYPE == FA_DTYPE_INT8) {
      x[e] = static_cast<float>(static_cast<int8_t>(row[i])) * scale;
    } else if constexpr (DTYPE == FA_DTYPE_E4M3) {
      x[e] = __half2float(__half(__nv_cvt_fp8_to_halfraw(row[i], __NV_E4M3))) * scale;
    } else {
      x[e] = to_f32<BF16>(reinterpret_cast<const uint16_t*>(row)[i]);
    }
  }
}

template <int D, bool BF16, int DTYPE>
__global__ void __launch_bounds__(128) paged_simple_kernel(const PagedAttn a) {
  constexpr int E = D / 32;
  __shared__ float sm[4], sl[4], so[4][D];
  const int t = blockIdx.x, hq = blockIdx.y, h = hq / a.group;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int b = -1;
  for (int i = 0; i < a.r.B; ++i)
    if (t >= __ldg(a.r.cu + i) && t < __ldg(a.r.cu + i + 1)) b = i;
  int lim = 0;
  if (b >= 0) {
    const int c0 = __ldg(a.r.cu + b), nq = __ldg(a.r.cu + b + 1) - c0;
    const int nk = min(__ldg(a.r.lens + b), a.max_k), i = t - c0;
    lim = nk;
    if (a.causal == FA_CAUSAL_BOTTOM_RIGHT) lim = min(nk, i + nk - nq + 1);
    if (a.causal == FA_CAUSAL_TOP_LEFT) lim = min(nk, i + 1);
    if (i >= a.max_q) lim = 0;
  }
  float q[E], o[E] = {}, m = -INFINITY, l = 0.f;
  load_row<D, BF16, FA_DTYPE_F16>(a.q + t * a.q_token + hq * a.q_head, lane, 1.f, q);
  for (int j = warp; j < lim; j += 4) {
    const int page = a.c.lookup(b, j), row = a.c.row_in_page(j);
    float k[E] = {}, v[E] = {};
    if (page >= 0) {
      const long long at = page * a.c.page_stride + h * a.c.head_stride + row * a.c.row_stride;
      const long long st = page * a.c.s_page + h * a.c.s_head + row * a.c.s_row;
      load_row<D, BF16, DTYPE>(a.c.k + at, lane, a.c.ks ? a.c.ks[st] : 1.f, k);
      load_row<D, BF16, DTYPE>(a.c.v + at, lane, a.c.vs ? a.c.vs[st] : 1.f, v);
    }
    float s = 0.f;
    for (int e = 0; e < E; ++e) s = fmaf(q[e], k[e], s);
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= a.scale_log2;
    const float mn = fmaxf(m, s), f = exp2f(m - mn), p = exp2f(s - mn);
    l = l * f + p;
    for (int e = 0; e < E; ++e) o[e] = o[e] * f + p * v[e];
    m = mn;
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  for (int e = 0; e < E; ++e) so[warp][lane + 32 * e] = o[e];
  __syncthreads();
  float mx = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), sum = 0.f, w[4];
  for (int i = 0; i < 4; ++i) {
    w[i] = sm[i] == -INFINITY ? 0.f : exp2f(sm[i] - mx);
    sum += w[i] * sl[i];
  }
  const float inv = sum > 0.f ? 1.f / sum : 0.f;
  for (int i = threadIdx.x; i < D; i += 128) {
    const float r = lim > 0 ? (w[0] * so[0][i] + w[1] * so[1][i] + w[2] * so[2][i] + w[3] * so[3][i]) * inv : 0.f;
    const long long at = (static_cast<long long>(t) * a.Hq + hq) * D + i;
    if constexpr (BF16) static_cast<__nv_bfloat16*>(a.o)[at] = __float2bfloat16_rn(r);
    else static_cast<__half*>(a.o)[at] = __float2half_rn(r);
  }
  if (threadIdx.x == 0 && a.lse)
    a.lse[static_cast<long long>(hq) * a.r.total + t] =
        lim > 0 ? (mx + log2f(sum)) * 0.69314718055994530942f : -INFINITY;
}

template <int D, bool BF16>
void simple_dtype(const PagedAttn& a, int cache_dtype, dim3 grid, cudaStream_t s) {
  if (cache_dtype == FA_DTYPE_INT8) paged_simple_kernel<D, BF16, FA_DTYPE_INT8><<<grid, 128, 0, s>>>(a);
  else if (cache_dtype == FA_DTYPE_E4M3) paged_simple_kernel<D, BF16, FA_DTYPE_E4M3><<<grid, 128, 0, s>>>(a);
  else paged_simple_kernel<D, BF16, FA_DTYPE_F16><<<grid, 128, 0, s>>>(a);
}

}  // namespace

cudaError_t launch_paged_simple(const PagedAttn& a, int head_dim, int cache_dtype, bool bf16,
                                cudaStream_t stream) {
  const dim3 grid(a.r.total, a.Hq);
  if (head_dim == 64) {
    if (bf16) simple_dtype<64, true>(a, cache_dtype, grid, stream);
    else simple_dtype<64, false>(a, cache_dtype, grid, stream);
  } else {
    if (bf16) simple_dtype<128, true>(a, cache_dtype, grid, stream);
    else simple_dtype<128, false>(a, cache_dtype, grid, stream);
  }
  return cudaGetLastError();
}

}  // namespace fa
