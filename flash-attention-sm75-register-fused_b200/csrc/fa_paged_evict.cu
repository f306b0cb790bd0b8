// Cutting a paged cache to a budget: per sequence and KV head, `keep` of its n > keep
// positions stay: the first `first`, the last `recent` and, of those between, the
// ones of the largest weight (equal weights: the lower position; a NaN is below
// every number).  What stays moves together in order of position, in place: keys,
// values, scales and weights; rows behind the new length keep what they hold.
//
// One launch; a cluster of 1 to 8 CTAs per (sequence, head).
//   select  The weight of the last one that stays, by radix selection over
//           order-preserving integers, 11 bits a pass, without a sort: every CTA counts
//           its positions in shared memory, and all add up the cluster's counts.
//   place   The cluster walks the positions, 1024 per CTA and step; two ranks (of
//           equal weights, of what stays) and the CTAs' counts give every kept one
//           its place, and its position goes to the CTA that moves that place.
//   move    Places in ascending order, as many at a time as the cluster holds in
//           registers: all are loaded before any is stored, and as the i-th kept
//           position is at least i, nothing is overwritten that a later group reads.
// Bound by memory: the weights are read once (the first kCacheSteps x 1024 of a CTA stay in
// shared memory), rows that move are read and written once.  @@
#include <cuda_runtime.h>

#include <cstdint>

#include "fa_paged.h"
#include "sm100_ptx.cuh"

namespace fa {
namespace {

constexpr int kEvictThreads = 1024;
constexpr int kBins = 2048;
constexpr int kCacheSteps = 16;
constexpr int kMaxCluster = 8;

// Integer that orders as the weights do: -0 as 0, a NaN below all.
__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) return 0u;
  const uint32_t u = f == 0.f ? 0u : __float_as_uint(f);
  return u ^ (static_cast<uint32_t>(static_cast<int>(u) >> 31) | 0x80000000u);
}

__device__ __forceinline__ int load_cluster(const void* p, int rank) {
  int x;
  asm volatile("ld.shared::cluster.s32 %0, [%1];"
               : "=r"(x)
               : "r"(ptx::mapa(ptx::smem_u32(p), static_cast<uint32_t>(rank)))
               : "memory");
  return x;
}
__device__ __forceinline__ void store_cluster(const void* p, int rank, int x) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(ptx::mapa(ptx::smem_u32(p), static_cast<uint32_t>(rank))), "r"(x)
               : "memory");
}

// Sum of `x` over the block's threads before this one; *total over all.  sh: 32 entries.
__device__ __forceinline__ int block_sum_before(int x, int* sh, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) sh[warp] = incl;
  __syncthreads();
  const int mine = sh[lane];
  int all = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, all, o);
    if (lane >= o) all += up;
  }
  *total = __shfl_sync(0xffffffffu, all, 31);
  const int before = __shfl_sync(0xffffffffu, all - mine, warp);
  __syncthreads();
  return before + incl - x;
}

template <int RB, bool kScales>
__global__ void __launch_bounds__(kEvictThreads) paged_evict_kernel(const PagedEvict p, int C) {
  extern __shared__ float cache[];  // [kCacheSteps][kEvictThreads]
  __shared__ int sh_hist[2][kBins];
  __shared__ int sh_list[kEvictThreads];
  __shared__ int sh_warp[32];
  __shared__ int sh_count[2][2];
  __shared__ int sh_bin, sh_want;
  const int tid = threadIdx.x;
  const int rank = static_cast<int>(blockIdx.x) % C, item = static_cast<int>(blockIdx.x) / C;
  const int b = item / p.c.heads, h = item % p.c.heads;
  const int n = min(max(__ldg(p.lens + b), 0), p.c.max_pages * p.c.page_size);
  const int keep = max(p.keep != nullptr ? __ldg(p.keep + b) : p.keep_all, 0);
  if (h == 0 && rank == 0 && tid == 0) p.new_lens[b] = min(n, keep);
  if (n <= keep || keep == 0) return;  // (the whole cluster)
  const int first = min(p.first, keep), recent = min(p.recent, keep - first);
  const int lo = first, hi = n - recent;
  float* const w = p.w + b * p.w_seq + h * p.w_head;
  // positions of step s: [s P, (s + 1) P), this CTA's from s P + 1024 rank
  const int P = C * kEvictThreads;
  const int n_steps = (n - 1) / P + 1;
  auto pos_of = [&](int s) { return s * P + rank * kEvictThreads + tid; };
  for (int s = 0; s < n_steps && s < kCacheSteps; ++s) {
    const int pos = pos_of(s);
    cache[s * kEvictThreads + tid] = pos < n ? __ldcg(w + pos) : 0.f;
  }
  auto weight = [&](int s) {  // (a thread reads back its own)
    if (s < kCacheSteps) return cache[s * kEvictThreads + tid];
    const int pos = pos_of(s);
    return pos < n ? __ldcg(w + pos) : 0.f;
  };

  // ---- the smallest key that stays, and how many of that value do
  uint32_t key = 0xffffffffu, mask = 0u;
  int want = keep - first - recent;  // of the positions between, fewer than there are
  if (want > 0) {
    key = 0u;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t digit = pass == 2 ? 1023u : 2047u;
      int* const hist = sh_hist[pass & 1];
      hist[tid] = hist[kEvictThreads + tid] = 0;
      __syncthreads();
      for (int s = 0; s < n_steps; ++s) {
        const int pos = pos_of(s);
        const uint32_t u = order_key(weight(s));
        if (pos >= lo && pos < hi && (u & mask) == key) atomicAdd(&hist[(u >> shift) & digit], 1);
      }
      ptx::cluster_sync();
      // thread t has bins 2047 - 2 t and 2046 - 2 t: from the top down
      int c0 = 0, c1 = 0;
      const int bin = kBins - 1 - 2 * tid;
      for (int r = 0; r < C; ++r) {
        c0 += load_cluster(&hist[bin], r);
        c1 += load_cluster(&hist[bin - 1], r);
      }
      int total;
      const int before = block_sum_before(c0 + c1, sh_warp, &total);
      if (before < want && before + c0 + c1 >= want) {
        const bool second = before + c0 < want;
        sh_bin = second ? bin - 1 : bin;
        sh_want = want - before - (second ? c0 : 0);
      }
      __syncthreads();
      key |= static_cast<uint32_t>(sh_bin) << shift;
      mask |= digit << shift;
      want = sh_want;
      __syncthreads();
    }
  }

  // ---- the places of what stays, and the move
  constexpr int kLanes = RB / 16;                         // threads of a row
  constexpr int kUnits = 2;                               // rows of a thread in flight
  constexpr int kRows = kUnits * kEvictThreads / kLanes;  // ... of a CTA
  static_assert(kRows <= kEvictThreads, "list");
  const int W = C * kRows;
  int kept = 0, ties = 0;  // in the steps before
  for (int s = 0; s < n_steps && kept < keep; ++s) {
    const int pos = pos_of(s);
    const float wt = weight(s);
    const uint32_t u = order_key(wt);
    const bool sure = pos < n && (pos < lo || pos >= hi || u > key);
    const bool tie = pos >= lo && pos < hi && u == key;
    // both counts in one scan
    int both;
    const int before = block_sum_before((sure ? 1 : 0) | (tie ? 1 << 16 : 0), sh_warp, &both);
    if (tid == 0) {
      sh_count[s & 1][0] = both & 0xffff;
      sh_count[s & 1][1] = both >> 16;
    }
    ptx::cluster_sync();
    int base = 0, mine = 0, n_step = 0, tie_at = ties;  // kept before this CTA, ties before it
    int t = ties;
    for (int r = 0; r < C; ++r) {
      const int g = load_cluster(&sh_count[s & 1][0], r), e = load_cluster(&sh_count[s & 1][1], r);
      if (r == rank) {
        tie_at = t;
        base = n_step;
      }
      n_step += g + min(max(want - t, 0), e);
      t += e;
    }
    mine = tie_at + (before >> 16);  // equal weights before this one
    const bool stays = sure || (tie && mine < want);
    // kept ones of this CTA before it: the sure ones, and the ties that stay
    const int q = base + (before & 0xffff) + min(max(want - tie_at, 0), before >> 16);
    const bool still = kept == s * P && n_step == min(P, n - s * P);  // nothing has moved so far
    if (stays && !still) {
      const int sub = q / W, in = q % W;
      store_cluster(&sh_list[sub * kRows + in % kRows], in / kRows, pos);
      w[kept + q] = wt;
    }
    ptx::cluster_sync();
    for (int q0 = 0; q0 < n_step && !still; q0 += W) {
      uint4 k[kUnits], v[kUnits];
      float ks[kUnits], vs[kUnits];
      int to[kUnits];
#pragma unroll
      for (int x = 0; x < kUnits; ++x) {
        const int r = x * (kEvictThreads / kLanes) + tid / kLanes, part = tid % kLanes;
        const int place = q0 + rank * kRows + r;
        const int src = place < n_step ? sh_list[q0 / C + r] : 0;
        to[x] = place < n_step && src != kept + place ? p.c.lookup(b, kept + place) : -1;
        const int from = to[x] >= 0 ? p.c.lookup(b, src) : -1;
        k[x] = v[x] = make_uint4(0u, 0u, 0u, 0u);
        ks[x] = vs[x] = 0.f;
        if (from >= 0) {
          const long long row = p.c.row_in_page(src);
          const long long o = from * p.c.page_stride + h * p.c.head_stride + row * p.c.row_stride;
          k[x] = __ldcg(reinterpret_cast<const uint4*>(p.c.k + o) + part);
          v[x] = __ldcg(reinterpret_cast<const uint4*>(p.c.v + o) + part);
          if (kScales && part == 0) {
            const long long so = from * p.c.s_page + h * p.c.s_head + row * p.c.s_row;
            ks[x] = __ldcg(p.c.ks + so);
            vs[x] = __ldcg(p.c.vs + so);
          }
        }
      }
      ptx::cluster_sync();
#pragma unroll
      for (int x = 0; x < kUnits; ++x) {
        if (to[x] < 0) continue;
        const int r = x * (kEvictThreads / kLanes) + tid / kLanes, part = tid % kLanes;
        const long long row = p.c.row_in_page(kept + q0 + rank * kRows + r);
        const long long o = to[x] * p.c.page_stride + h * p.c.head_stride + row * p.c.row_stride;
        reinterpret_cast<uint4*>(const_cast<uint8_t*>(p.c.k) + o)[part] = k[x];
        reinterpret_cast<uint4*>(const_cast<uint8_t*>(p.c.v) + o)[part] = v[x];
        if (kScales && part == 0) {
          const long long so = to[x] * p.c.s_page + h * p.c.s_head + row * p.c.s_row;
          p.c.ks[so] = ks[x];
          p.c.vs[so] = vs[x];
        }
      }
    }
    kept += n_step;
    ties = t;
  }
  ptx::cluster_sync();  // (nobody reads the shared memory of a CTA that is gone)
}

template <int RB, bool kScales>
cudaError_t evict_impl(const PagedEvict& p, int sms, cudaStream_t stream) {
  auto kern = paged_evict_kernel<RB, kScales>;
  constexpr int kDyn = kCacheSteps * kEvictThreads * static_cast<int>(sizeof(float));
  static int attr_done[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kDyn);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_done[dev] = 1;
  }
  // CTAs of a cluster: as many as there are SMs and positions for
  const long long items = static_cast<long long>(p.B) * p.c.heads;
  const long long held = static_cast<long long>(p.c.max_pages) * p.c.page_size;
  int C = 1;
  while (C < kMaxCluster && items * 2 * C <= sms && held > static_cast<long long>(C) * kEvictThreads) C *= 2;
  if (items * C > 0x7fffffffLL) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(items * C));
  cfg.blockDim = dim3(kEvictThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(
      sizeof(float) * kEvictThreads * (held > static_cast<long long>(C) * kEvictThreads * kCacheSteps
                                           ? kCacheSteps
                                           : (held + C * kEvictThreads - 1) / (C * kEvictThreads)));
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(C);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p, C);
}

}  // namespace

cudaError_t launch_paged_evict(const PagedEvict& p, int row_bytes, bool scales, int sms, cudaStream_t stream) {
  if (row_bytes == 64) return evict_impl<64, true>(p, sms, stream);
  if (row_bytes == 256) return evict_impl<256, false>(p, sms, stream);
  return scales ? evict_impl<128, true>(p, sms, stream) : evict_impl<128, false>(p, sms, stream);
}

}  // namespace fa
