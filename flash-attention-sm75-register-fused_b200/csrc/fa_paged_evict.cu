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
//   place   The cluster walks the positions, 2048 per CTA and step; two ranks (of
//           equal weights, of what stays) and the CTAs' counts give every kept one
//           its place, and its page and position go to the list of the CTA that moves it.
//   move    Places in ascending order, a group at a time: all of a group are loaded
//           before any is stored, and as the i-th kept position is at least i, nothing
//           is overwritten that a later group reads.  So the next group's loads are on
//           their way while this one is stored.
// Bound by memory: the weights are read once (the first kCacheSteps x 2048 of a CTA stay in
// shared memory), rows that move are read and written once.  Measured on caches not cut
// before, 8 KV heads, d = 128:
// 32 ragged caches of up to 8192 bf16 positions cut to 2048, 187 MB read and written, 74 us (29 at
// the rate of a plain copy).  11 of them are longer, so 88 of the 256 clusters of two have work,
// on 176 CTAs where 296 fit; three passes of selection and the places take 16 us, then rows move
// in groups with a cluster barrier each.
// 2 x 65536 int8 positions to 16384, 144 MB, 125 us (22): of the 16 clusters of 8 that it launches 15
// are resident at a time (cudaOccupancyMaxActiveClusters), and the last one runs alone after
// them.
// 1 x 1024 to 512 17 us, all latency.
// Rows that keep their place are not moved.  Of a cache that is cut to the same number again and
// again that becomes most of them: the 32 ragged ones end at 43 us.  A CTA alone per head, with
// 1024 positions' rows moved as they are found, took 80, 328 and 19 us for a first cut.
#include <cuda_runtime.h>

#include <cstdint>

#include "fa_paged.h"
#include "sm100_ptx.cuh"

namespace fa {
namespace {

constexpr int kEvictThreads = 512;
constexpr int kBins = 2048;
constexpr int kEach = 4;                          // positions of a thread and step
constexpr int kChunk = kEach * kEvictThreads;     // ... of a CTA
constexpr int kCacheSteps = 6;
constexpr int kList = 4096;                       // places of a CTA
constexpr int kMaxCluster = 8;
// CTAs that share a head: up to this many for every SM in all (a ragged batch's short sequences
// leave at once).  32 ragged sequences x 8 heads with 2 / 4 / 8: 119 / 74 / 79 us.
constexpr long long kClusterLoad = 4;

// Integer that orders as the weights do: -0 as 0, a NaN below all.
__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) return 0u;
  const uint32_t u = f == 0.f ? 0u : __float_as_uint(f);
  return u ^ (static_cast<uint32_t>(static_cast<int>(u) >> 31) | 0x80000000u);
}

// From and to the shared memory of another CTA of the cluster.
__device__ __forceinline__ int4 load_cluster4(const void* p, int rank) {
  int4 x;
  asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];"
               : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
               : "r"(ptx::mapa(ptx::smem_u32(p), static_cast<uint32_t>(rank)))
               : "memory");
  return x;
}
__device__ __forceinline__ int2 load_cluster2(const void* p, int rank) {
  int2 x;
  asm volatile("ld.shared::cluster.v2.s32 {%0,%1}, [%2];"
               : "=r"(x.x), "=r"(x.y)
               : "r"(ptx::mapa(ptx::smem_u32(p), static_cast<uint32_t>(rank)))
               : "memory");
  return x;
}
__device__ __forceinline__ void store_cluster(const void* p, int rank, int x) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(ptx::mapa(ptx::smem_u32(p), static_cast<uint32_t>(rank))), "r"(x)
               : "memory");
}

// Sum of `x` over the block's threads before this one; *total over all.  sh: one entry a warp.
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
  const int mine = lane < kEvictThreads / 32 ? sh[lane] : 0;
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

struct Source {
  int page, pos;  // page -1: none
};

// kUnits: rows of a thread in a group.
template <int RB, bool kScales, int kUnits>
__global__ void __launch_bounds__(kEvictThreads, kUnits == 2 ? 2 : 1) paged_evict_kernel(const PagedEvict p, int C) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Source* const list = reinterpret_cast<Source*>(smem_raw);                    // [kList]
  float* const cache = reinterpret_cast<float*>(smem_raw + kList * sizeof(Source));  // [kCacheSteps][kChunk]
  __shared__ __align__(16) int sh_hist[2][kBins];
  __shared__ int sh_warp[32];
  __shared__ __align__(8) int sh_count[2][2];
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
  // Up to kChunk positions every CTA selects by itself, and the cluster shares the move alone.
  const bool alone = n <= kChunk;
  const int R = alone ? 1 : C, me = alone ? 0 : rank;
  auto sync_select = [&] {
    if (alone) __syncthreads();
    else ptx::cluster_sync();
  };
  // positions of step s: [s P, (s + 1) P), this CTA's from s P + me kChunk, a thread's four of them
  const int P = R * kChunk;
  const int n_steps = (n - 1) / P + 1;
  auto pos_of = [&](int s) { return s * P + me * kChunk + kEach * tid; };
  for (int s = 0; s < n_steps && s < kCacheSteps; ++s)
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int x = i * kEvictThreads + tid, pos = s * P + me * kChunk + x;
      cache[s * kChunk + x] = pos < n ? __ldcg(w + pos) : 0.f;
    }
  if (alone) ptx::cluster_sync();  // (all have read the weights that the first one moves)
  else __syncthreads();
  auto weights = [&](int s, float (&x)[kEach]) {
    if (s < kCacheSteps) {
      const float4 v = *reinterpret_cast<const float4*>(cache + s * kChunk + kEach * tid);
      x[0] = v.x;
      x[1] = v.y;
      x[2] = v.z;
      x[3] = v.w;
    } else {
#pragma unroll
      for (int i = 0; i < kEach; ++i) x[i] = pos_of(s) + i < n ? __ldcg(w + pos_of(s) + i) : 0.f;
    }
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
#pragma unroll
      for (int i = tid; i < kBins; i += kEvictThreads) hist[i] = 0;
      __syncthreads();
      for (int s = 0; s < n_steps; ++s) {
        float x[kEach];
        weights(s, x);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          const int pos = pos_of(s) + i;
          const uint32_t u = order_key(x[i]);
          if (pos >= lo && pos < hi && (u & mask) == key) atomicAdd(&hist[(u >> shift) & digit], 1);
        }
      }
      sync_select();
      // thread t has the four bins from 2047 - 4 t down
      static_assert(kBins == 4 * kEvictThreads, "bins of a thread");
      const int bin = kBins - 1 - 4 * tid;
      int4 part[kMaxCluster];
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r)
        part[r] = r < R ? load_cluster4(&hist[bin - 3], alone ? rank : r) : make_int4(0, 0, 0, 0);
      int c[4] = {}, sum = 0;
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) {
        c[0] += part[r].w;
        c[1] += part[r].z;
        c[2] += part[r].y;
        c[3] += part[r].x;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += c[i];
      int total;
      int before = block_sum_before(sum, sh_warp, &total);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (before < want && before + c[i] >= want) {
          sh_bin = bin - i;
          sh_want = want - before;
        }
        before += c[i];
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
  constexpr int kStride = kEvictThreads / kLanes;         // rows of a unit
  constexpr int kRows = kUnits * kStride;                 // ... of a group, in a CTA
  static_assert(kList % kRows == 0, "list");
  const int W = C * kRows;
  const int part = tid % kLanes;
  int kept = 0, ties = 0;  // in the steps before
  for (int s = 0; s < n_steps && kept < keep;) {
    // places kept .. of the next steps, as many as the lists take
    int place0 = kept, filled = 0;
    for (; s < n_steps && kept < keep && filled + P <= C * kList; ++s) {
      const int pos0 = pos_of(s);
      float x[kEach];
      weights(s, x);
      unsigned sure = 0, tie = 0;  // bit i: position pos0 + i
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int pos = pos0 + i;
        const uint32_t u = order_key(x[i]);
        const bool between = pos >= lo && pos < hi;
        sure |= (pos < n && (!between || u > key) ? 1u : 0u) << i;
        tie |= (between && u == key ? 1u : 0u) << i;
      }
      // both counts in one scan
      int both;
      const int before = block_sum_before(__popc(sure) | __popc(tie) << 16, sh_warp, &both);
      if (tid == 0) {
        sh_count[s & 1][0] = both & 0xffff;
        sh_count[s & 1][1] = both >> 16;
      }
      sync_select();
      // lane r has CTA r's counts; prefix sums over the lanes
      const int lane = tid & 31;
      const int2 counts = lane < R ? load_cluster2(sh_count[s & 1], alone ? rank : lane) : make_int2(0, 0);
      auto prefix = [&](int x) {
#pragma unroll
        for (int o = 1; o < kMaxCluster; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += up;
        }
        return x;
      };
      const int ties_end = ties + prefix(counts.y);
      const int stay = counts.x + min(max(want - (ties_end - counts.y), 0), counts.y);
      const int stay_end = prefix(stay);
      const int n_step = __shfl_sync(0xffffffffu, stay_end, kMaxCluster - 1);
      const int base = __shfl_sync(0xffffffffu, stay_end - stay, me);          // kept, equal weights
      const int tie_at = __shfl_sync(0xffffffffu, ties_end - counts.y, me);  // before this CTA
      ties = __shfl_sync(0xffffffffu, ties_end, kMaxCluster - 1);
      if (filled == 0 && kept == s * P && n_step == min(P, n - s * P)) {  // nothing has moved so far
        kept += n_step;
        place0 = kept;
        continue;
      }
      const int left = max(want - tie_at, 0);  // equal weights of this CTA that stay
      int q = filled + base + (before & 0xffff) + min(left, before >> 16), rest = left - (before >> 16);
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const bool t = (tie >> i) & 1u;
        if (((sure >> i) & 1u) || (t && rest > 0)) {
          const int in = q % W, to = in / kRows;
          Source* const at = &list[q / W * kRows + in % kRows];
          if (!alone || to == rank) {
            store_cluster(&at->page, to, p.c.lookup(b, pos0 + i));
            store_cluster(&at->pos, to, pos0 + i);
          }
          if (!alone || rank == 0) w[place0 + q] = x[i];
          ++q;
        }
        if (t) --rest;
      }
      filled += n_step;
      kept += n_step;
    }
    ptx::cluster_sync();

    struct Group {
      uint4 k[kUnits], v[kUnits];
      float ks[kUnits], vs[kUnits];
      int to[kUnits];
    };
    auto load = [&](Group& x, int q0) {
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int r = i * kStride + tid / kLanes, q = q0 + rank * kRows + r;
        x.to[i] = -1;
        x.k[i] = x.v[i] = make_uint4(0u, 0u, 0u, 0u);
        x.ks[i] = x.vs[i] = 0.f;
        if (q < filled) {
          const Source src = list[q0 / C + r];
          if (src.pos == place0 + q) continue;  // (nothing before it went)
          x.to[i] = p.c.lookup(b, place0 + q);
          if (src.page >= 0) {
            const int row = p.c.row_in_page(src.pos);
            const long long o = src.page * p.c.page_stride + h * p.c.head_stride + row * p.c.row_stride;
            x.k[i] = __ldcg(reinterpret_cast<const uint4*>(p.c.k + o) + part);
            x.v[i] = __ldcg(reinterpret_cast<const uint4*>(p.c.v + o) + part);
            if (kScales && part == 0) {
              const long long so = src.page * p.c.s_page + h * p.c.s_head + row * p.c.s_row;
              x.ks[i] = __ldcg(p.c.ks + so);
              x.vs[i] = __ldcg(p.c.vs + so);
            }
          }
        }
      }
    };
    auto store = [&](const Group& x, int q0) {
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        if (x.to[i] < 0) continue;
        const int row = p.c.row_in_page(place0 + q0 + rank * kRows + i * kStride + tid / kLanes);
        const long long o = x.to[i] * p.c.page_stride + h * p.c.head_stride + row * p.c.row_stride;
        reinterpret_cast<uint4*>(const_cast<uint8_t*>(p.c.k) + o)[part] = x.k[i];
        reinterpret_cast<uint4*>(const_cast<uint8_t*>(p.c.v) + o)[part] = x.v[i];
        if (kScales && part == 0) {
          const long long so = x.to[i] * p.c.s_page + h * p.c.s_head + row * p.c.s_row;
          p.c.ks[so] = x.ks[i];
          p.c.vs[so] = x.vs[i];
        }
      }
    };
    // (the compiler may not wait for a load before the barrier: what it returns is pinned)
    auto landed = [&](Group& x) {
#pragma unroll
      for (int i = 0; i < kUnits; ++i)
        asm volatile("" : "+r"(x.k[i].x), "+r"(x.k[i].y), "+r"(x.k[i].z), "+r"(x.k[i].w), "+r"(x.v[i].x),
                          "+r"(x.v[i].y), "+r"(x.v[i].z), "+r"(x.v[i].w), "+f"(x.ks[i]), "+f"(x.vs[i]));
    };
    Group x, y;
    if (filled > 0) load(x, 0);
    for (int q0 = 0; q0 < filled; q0 += 2 * W) {
      load(y, q0 + W);
      landed(x);
      ptx::cluster_sync();
      store(x, q0);
      if (q0 + W >= filled) break;
      load(x, q0 + 2 * W);
      landed(y);
      ptx::cluster_sync();
      store(y, q0 + W);
    }
  }
  ptx::cluster_sync();  // (nobody reads the shared memory of a CTA that is gone)
}

template <int RB, bool kScales, int kUnits>
cudaError_t evict_units(const PagedEvict& p, int C, cudaStream_t stream) {
  auto kern = paged_evict_kernel<RB, kScales, kUnits>;
  constexpr int kListBytes = kList * static_cast<int>(sizeof(Source));
  constexpr int kStepBytes = kChunk * static_cast<int>(sizeof(float));
  static int attr_done[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               kListBytes + kCacheSteps * kStepBytes);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_done[dev] = 1;
  }
  const long long P = static_cast<long long>(C) * kChunk;
  const long long steps = (static_cast<long long>(p.c.max_pages) * p.c.page_size + P - 1) / P;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(static_cast<long long>(p.B) * p.c.heads * C));
  cfg.blockDim = dim3(kEvictThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(kListBytes + kStepBytes * (steps < kCacheSteps ? steps : kCacheSteps));
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(C);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p, C);
}

template <int RB, bool kScales>
cudaError_t evict_impl(const PagedEvict& p, int sms, cudaStream_t stream) {
  const long long items = static_cast<long long>(p.B) * p.c.heads;
  const long long held = static_cast<long long>(p.c.max_pages) * p.c.page_size;
  int C = 1;
  while (C < kMaxCluster && items * 2 * C <= kClusterLoad * sms && held > 128LL * C) C *= 2;
  if (items * C > 0x7fffffffLL) return cudaErrorInvalidValue;
  return items * C <= sms ? evict_units<RB, kScales, 4>(p, C, stream) : evict_units<RB, kScales, 2>(p, C, stream);
}

}  // namespace

cudaError_t launch_paged_evict(const PagedEvict& p, int row_bytes, bool scales, int sms, cudaStream_t stream) {
  if (row_bytes == 64) return evict_impl<64, true>(p, sms, stream);
  if (row_bytes == 256) return evict_impl<256, false>(p, sms, stream);
  return scales ? evict_impl<128, true>(p, sms, stream) : evict_impl<128, false>(p, sms, stream);
}

}  // namespace fa
