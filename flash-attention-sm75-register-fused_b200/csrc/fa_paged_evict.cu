// Cutting a paged cache to a budget: per sequence and KV head, `keep` of its n > keep
// positions stay: the first `first`, the last `recent` and, of those between, the
// ones of the largest weight (equal weights: the lower position; a NaN is below
// every number).  What stays moves together in order of position, in place: keys,
// values, scales and weights; rows behind the new length keep what they hold.
//
// One block per (sequence, head).  The weight of the last one that stays is found by
// a radix selection over order-preserving integers, 8 bits a pass, so that no sort is
// needed; a second walk over the positions gives each kept one its place.  Since the
// i-th kept position is at least i, moving rows in ascending order never overwrites
// one that is still to be read, if a group of rows is loaded before any of it is stored.
#include <cuda_runtime.h>

#include <cstdint>

#include "fa_paged.h"

namespace fa {
namespace {

constexpr int kEvictThreads = 1024;

// Integer that orders as the weights do: -0 as 0, a NaN below all.
__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) return 0u;
  const uint32_t u = f == 0.f ? 0u : __float_as_uint(f);
  return u ^ (static_cast<uint32_t>(static_cast<int>(u) >> 31) | 0x80000000u);
}

// Exclusive rank of this thread among the block's threads with `v`, and their number.
__device__ __forceinline__ int block_rank(bool v, int* sh, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned m = __ballot_sync(0xffffffffu, v);
  if (lane == 0) sh[warp] = __popc(m);
  __syncthreads();
  int x = sh[lane], incl = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  *total = __shfl_sync(0xffffffffu, incl, 31);
  const int before = __shfl_sync(0xffffffffu, incl - x, warp);
  __syncthreads();
  return before + __popc(m & ((1u << lane) - 1u));
}

template <int RB, bool kScales>
__global__ void __launch_bounds__(kEvictThreads) paged_evict_kernel(const PagedEvict p) {
  __shared__ int sh_hist[256];
  __shared__ int sh_rank[32];
  __shared__ int sh_src[kEvictThreads];
  __shared__ int sh_bin, sh_want;
  const int tid = threadIdx.x;
  const int b = static_cast<int>(blockIdx.x) / p.c.heads, h = static_cast<int>(blockIdx.x) % p.c.heads;
  const int n = min(max(__ldg(p.lens + b), 0), p.c.max_pages * p.c.page_size);
  const int keep = max(p.keep != nullptr ? __ldg(p.keep + b) : p.keep_all, 0);
  if (h == 0 && tid == 0) p.new_lens[b] = min(n, keep);
  if (n <= keep || keep == 0) return;
  const int first = min(p.first, keep), recent = min(p.recent, keep - first);
  const int lo = first, hi = n - recent;
  float* const w = p.w + b * p.w_seq + h * p.w_head;

  // ---- the smallest key that stays, and how many of that value do
  uint32_t key = 0xffffffffu, mask = 0u;
  int want = keep - first - recent;  // of the positions between, fewer than there are
  if (want > 0) {
    key = 0u;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) sh_hist[tid] = 0;
      __syncthreads();
      for (int pos = lo + tid; pos < hi; pos += kEvictThreads) {
        const uint32_t u = order_key(__ldcg(w + pos));
        if ((u & mask) == key) atomicAdd(&sh_hist[(u >> shift) & 255u], 1);
      }
      __syncthreads();
      if (tid < 32) {
        // lane 31 has the highest bins
        int sum = 0;
        for (int i = 0; i < 8; ++i) sum += sh_hist[tid * 8 + i];
        int above = sum;  // in this lane's bins and the higher lanes'
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_down_sync(0xffffffffu, above, o);
          if (tid + o < 32) above += up;
        }
        const int before = above - sum;
        if (before < want && above >= want) {
          int left = want - before, i = 7;
          while (sh_hist[tid * 8 + i] < left) left -= sh_hist[tid * 8 + i--];
          sh_bin = tid * 8 + i;
          sh_want = left;
        }
      }
      __syncthreads();
      key |= static_cast<uint32_t>(sh_bin) << shift;
      mask |= 255u << shift;
      want = sh_want;
    }
  }

  // ---- the places of what stays, and the move
  constexpr int kLanes = RB / 16;                    // threads of a row
  constexpr int kRows = kEvictThreads / kLanes;      // rows in flight
  int kept = 0, ties = 0;
  for (int c0 = 0; c0 < n; c0 += kEvictThreads) {
    const int pos = c0 + tid;
    const float wt = pos < n ? __ldcg(w + pos) : 0.f;
    const uint32_t u = order_key(wt);
    const bool sure = pos < lo || pos >= hi;
    const bool tie = pos < n && !sure && u == key;
    int n_ties, n_kept;
    const int tie_rank = ties + block_rank(tie, sh_rank, &n_ties);
    const bool stays = pos < n && (sure || u > key || (tie && tie_rank < want));
    const int rank = block_rank(stays, sh_rank, &n_kept);
    if (stays) {
      sh_src[rank] = pos;
      w[kept + rank] = wt;
    }
    __syncthreads();
    for (int r0 = 0; r0 < n_kept; r0 += kRows) {
      const int r = r0 + tid / kLanes, part = tid % kLanes;
      const int src = r < n_kept ? sh_src[r] : 0, dst = kept + r;
      const bool moves = r < n_kept && src != dst;
      uint4 k = make_uint4(0u, 0u, 0u, 0u), v = k;
      float ks = 0.f, vs = 0.f;
      const int from = moves ? p.c.lookup(b, src) : -1, to = moves ? p.c.lookup(b, dst) : -1;
      if (from >= 0) {
        const long long row = p.c.row_in_page(src);
        const long long o = from * p.c.page_stride + h * p.c.head_stride + row * p.c.row_stride;
        k = __ldcg(reinterpret_cast<const uint4*>(p.c.k + o) + part);
        v = __ldcg(reinterpret_cast<const uint4*>(p.c.v + o) + part);
        if (kScales && part == 0) {
          const long long so = from * p.c.s_page + h * p.c.s_head + row * p.c.s_row;
          ks = __ldcg(p.c.ks + so);
          vs = __ldcg(p.c.vs + so);
        }
      }
      __syncthreads();
      if (to >= 0) {
        const long long row = p.c.row_in_page(dst);
        const long long o = to * p.c.page_stride + h * p.c.head_stride + row * p.c.row_stride;
        reinterpret_cast<uint4*>(const_cast<uint8_t*>(p.c.k) + o)[part] = k;
        reinterpret_cast<uint4*>(const_cast<uint8_t*>(p.c.v) + o)[part] = v;
        if (kScales && part == 0) {
          const long long so = to * p.c.s_page + h * p.c.s_head + row * p.c.s_row;
          p.c.ks[so] = ks;
          p.c.vs[so] = vs;
        }
      }
    }
    kept += n_kept;
    ties += n_ties;
    __syncthreads();
  }
}

}  // namespace

cudaError_t launch_paged_evict(const PagedEvict& p, int row_bytes, bool scales, int, cudaStream_t stream) {
  const unsigned grid = static_cast<unsigned>(p.B) * p.c.heads;
  if (row_bytes == 64) paged_evict_kernel<64, true><<<grid, kEvictThreads, 0, stream>>>(p);
  else if (row_bytes == 256) paged_evict_kernel<256, false><<<grid, kEvictThreads, 0, stream>>>(p);
  else if (scales) paged_evict_kernel<128, true><<<grid, kEvictThreads, 0, stream>>>(p);
  else paged_evict_kernel<128, false><<<grid, kEvictThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace fa
