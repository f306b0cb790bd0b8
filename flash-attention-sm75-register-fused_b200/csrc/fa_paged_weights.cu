// Attention weight that cached keys receive, summed over query rows:
//
//   w[b, h, j] = sum over the new tokens i of sequence b and the query heads of
//                KV head h of exp(scale q_i . k_j - LSE_i)
//
// with the LSE the attention returned, zero where row i does not see key j, added
// to (or replacing) the sums of earlier calls.
//
// A warp takes 16 keys and multiplies them by blocks of 32 query rows (m16n8k16,
// keys on M): S^T, one exponential per score, a sum over the rows.  Keys are
// independent of one another, so nothing is joined between warps and no sum
// depends on timing.  The columns of a row may come in any order as long as keys and
// queries agree, so a lane reads its part of a key row with 16-byte loads straight
// into the operand's registers.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "fa_paged.h"
#include "fa_paged_dev.cuh"
#include "sm100_ptx.cuh"

namespace fa {
namespace {

constexpr int kWeightThreads = 128;
constexpr int kWeightRows = 32;                    // query rows of a block
constexpr int kWeightKeys = kWeightThreads / 2;    // keys of a CTA

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
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

// An f16 pair (of 8-bit values, which both types hold exactly) in the queries' type.
template <bool BF16>
__device__ __forceinline__ uint32_t as_query_type(uint32_t x) {
  if constexpr (BF16) {
    const float2 f = __half22float2(*reinterpret_cast<__half2*>(&x));
    const __nv_bfloat162 v = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    return x;
  }
}

// Row r of (sequence, KV head): its packed token and query head.
struct QueryRow {
  int tok, hq;
};
__device__ __forceinline__ QueryRow query_row(const PagedAttn& a, const Seq& s, int h, int r) {
  return {s.c0 + r / a.group, h * a.group + r % a.group};
}

template <int D, int KV, bool QBF16>
__global__ void __launch_bounds__(kWeightThreads) paged_weights_kernel(const PagedWeights p, int n_blocks) {
  constexpr bool k8 = KV >= FA_DTYPE_INT8;
  constexpr int kRowBytes = k8 ? D : 2 * D;
  constexpr int kChunks = kRowBytes / 64;          // 16-byte pieces of a lane per key
  constexpr int kNT = kWeightRows / 8;
  constexpr int kPitch = 2 * D + (k8 ? 16 : 64);   // bytes of a query row: no bank conflicts
  const PagedAttn& a = p.a;
  __shared__ __align__(16) uint8_t sh_q[kWeightRows * kPitch];
  __shared__ float sh_lse[kWeightRows];
  __shared__ int sh_lim[kWeightRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, j = lane & 3;
  const int b = static_cast<int>(blockIdx.x / n_blocks) / a.c.heads;
  const int h = static_cast<int>(blockIdx.x / n_blocks) % a.c.heads;
  const int cta_key0 = static_cast<int>(blockIdx.x % n_blocks) * kWeightKeys;
  const Seq s = load_seq(a, b);
  if (cta_key0 >= s.nk) return;
  const int key0 = cta_key0 + warp * 16;
  const int rows = s.nq * a.group;
  // the new tokens' own positions, which have no earlier sum
  const int fresh0 = p.mode == FA_WEIGHTS_SET      ? 0
                     : p.mode == FA_WEIGHTS_APPEND ? min(__ldg(a.r.lens + b), 3 << 29) - s.n
                                                   : 0x7fffffff;

  // keys key0 + g, key0 + 8 + g: this lane's pieces
  uint4 x[2][kChunks];
  float ks[2] = {1.f, 1.f};
  const int page = key0 < s.vis ? a.c.lookup(b, key0) : -1;
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    const int r = g + 8 * y;
    const bool ok = page >= 0 && key0 + r < s.vis;
    const long long row = a.c.row_in_page(key0) + r;
    const uint8_t* src = a.c.k + page * a.c.page_stride + h * a.c.head_stride + row * a.c.row_stride;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
      x[y][c] = ok ? __ldg(reinterpret_cast<const uint4*>(src + 64 * c) + j) : make_uint4(0u, 0u, 0u, 0u);
    if constexpr (k8) ks[y] = ok ? __ldg(a.c.ks + page * a.c.s_page + h * a.c.s_head + row * a.c.s_row) : 0.f;
  }

  float sum[2] = {0.f, 0.f};
  for (int r0 = 0; r0 < rows; r0 += kWeightRows) {
    // (no row of the block sees a key of the CTA)
    if (row_limit(a, s, (min(r0 + kWeightRows, rows) - 1) / a.group) <= cta_key0) continue;
    __syncthreads();
    for (int i = threadIdx.x; i < kWeightRows * (D / 8); i += kWeightThreads) {
      const int r = i / (D / 8), c = i % (D / 8);
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (r0 + r < rows) {
        const QueryRow q = query_row(a, s, h, r0 + r);
        v = __ldg(reinterpret_cast<const uint4*>(a.q + q.tok * a.q_token + q.hq * a.q_head) + c);
      }
      *reinterpret_cast<uint4*>(sh_q + r * kPitch + 16 * c) = v;
    }
    if (threadIdx.x < kWeightRows) {
      const int r = r0 + threadIdx.x;
      float l = 0.f;
      int lim = 0;
      if (r < rows) {
        const QueryRow q = query_row(a, s, h, r);
        l = a.lse[static_cast<long long>(q.hq) * a.r.total + q.tok];
        lim = l == -INFINITY ? 0 : row_limit(a, s, r / a.group);
      }
      sh_lse[threadIdx.x] = lim > 0 ? l * 1.4426950408889634f : 0.f;
      sh_lim[threadIdx.x] = lim;
    }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      float c[4] = {0.f, 0.f, 0.f, 0.f};
      const uint8_t* qrow = sh_q + (nt * 8 + g) * kPitch;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const uint32_t k0[4] = {x[0][i].x, x[0][i].y, x[0][i].z, x[0][i].w};
        const uint32_t k1[4] = {x[1][i].x, x[1][i].y, x[1][i].z, x[1][i].w};
        if constexpr (!k8) {
          const uint4 q = *reinterpret_cast<const uint4*>(qrow + 64 * i + 16 * j);
          mma_16816<QBF16>(c, k0[0], k1[0], k0[1], k1[1], q.x, q.y);
          mma_16816<QBF16>(c, k0[2], k1[2], k0[3], k1[3], q.z, q.w);
        } else {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint4 q = *reinterpret_cast<const uint4*>(qrow + 128 * i + 32 * j + 16 * e);
            uint32_t w0[4], w1[4];
            widen<KV, false>(k0[2 * e], w0[0], w0[1]);
            widen<KV, false>(k0[2 * e + 1], w0[2], w0[3]);
            widen<KV, false>(k1[2 * e], w1[0], w1[1]);
            widen<KV, false>(k1[2 * e + 1], w1[2], w1[3]);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              w0[y] = as_query_type<QBF16>(w0[y]);
              w1[y] = as_query_type<QBF16>(w1[y]);
            }
            mma_16816<QBF16>(c, w0[0], w1[0], w0[1], w1[1], q.x, q.y);
            mma_16816<QBF16>(c, w0[2], w1[2], w0[3], w1[3], q.z, q.w);
          }
        }
      }
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = nt * 8 + 2 * j + e;
          const float t = fmaf(c[2 * y + e], a.scale_log2 * ks[y], -sh_lse[r]);
          if (key0 + g + 8 * y < sh_lim[r]) sum[y] += ptx::ex2_approx(t);
        }
    }
  }
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    sum[y] += __shfl_xor_sync(0xffffffffu, sum[y], 1);
    sum[y] += __shfl_xor_sync(0xffffffffu, sum[y], 2);
    const int key = key0 + g + 8 * y;
    if (j == 0 && key < s.nk) {
      float* dst = p.w + b * p.w_seq + h * p.w_head + key;
      *dst = key >= fresh0 ? sum[y] : *dst + sum[y];
    }
  }
}

template <int D, int KV, bool QBF16>
cudaError_t weights_impl(const PagedWeights& p, cudaStream_t stream) {
  const int n_blocks = (p.a.max_k + kWeightKeys - 1) / kWeightKeys;
  const long long grid = static_cast<long long>(n_blocks) * p.a.r.B * p.a.c.heads;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (grid == 0) return cudaSuccess;
  paged_weights_kernel<D, KV, QBF16><<<static_cast<unsigned>(grid), kWeightThreads, 0, stream>>>(p, n_blocks);
  return cudaGetLastError();
}

template <int D>
cudaError_t weights_d(const PagedWeights& p, int kv, bool bf16, cudaStream_t s) {
  switch (kv) {
    case FA_DTYPE_INT8:
      return bf16 ? weights_impl<D, FA_DTYPE_INT8, true>(p, s) : weights_impl<D, FA_DTYPE_INT8, false>(p, s);
    case FA_DTYPE_E4M3:
      return bf16 ? weights_impl<D, FA_DTYPE_E4M3, true>(p, s) : weights_impl<D, FA_DTYPE_E4M3, false>(p, s);
    case FA_DTYPE_BF16: return weights_impl<D, FA_DTYPE_BF16, true>(p, s);
    default: return weights_impl<D, FA_DTYPE_F16, false>(p, s);
  }
}

}  // namespace

cudaError_t launch_paged_weights(const PagedWeights& p, int head_dim, int cache_dtype, bool bf16, int,
                                 cudaStream_t stream) {
  return head_dim == 64 ? weights_d<64>(p, cache_dtype, bf16, stream)
                        : weights_d<128>(p, cache_dtype, bf16, stream);
}

}  // namespace fa
