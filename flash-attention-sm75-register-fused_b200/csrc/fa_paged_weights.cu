// Attention weight that cached keys receive, summed over query rows:
//
//   w[b, h, j] = sum over the new tokens i of sequence b and the query heads of
//                KV head h of exp(scale q_i . k_j - LSE_i)
//
// with the LSE the attention returned, zero where row i does not see key j, added
// to (or replacing) the sums of earlier calls.
//
// This file streams the keys for few query rows (decode, drafts);
// fa_paged_weights_chunk.cuh takes chunks.  A warp multiplies 16 keys by its query rows
// (m16n8k16, keys on M): S^T, one exponential per score, a sum over the rows.  Keys are
// independent of one another, so nothing is joined between warps and no sum
// depends on timing.  The columns of a row may come in any order as long as keys and
// queries agree, so a lane reads its part of a key row with 16-byte loads straight
// into the operand's registers.
//
// Bound by the keys' bytes.  All steps of 16 keys (32 of 8-bit pages) of the batch, in
// order of sequence, head and key, are cut into equal runs, one per warp, whatever the
// sequences' lengths.  A warp has its query rows in registers, the page ids of 32 groups of
// 16 keys in one register a lane, loaded a window ahead, and the next step's keys on
// their way while it computes this one's; nothing waits for another warp.
//
// Measured, 8 KV heads, d = 128, GQA 4: 16 sequences x 8192 keys of bf16 pages, one token,
// 48.1 us (5.8 TB/s; a plain copy runs at 6.5; one CTA per 64 keys and 32 rows, with the queries
// in shared memory, 82).  32 ragged sequences over int8 pages, 3 tokens, 26.7 us (3.6 TB/s): 290
// instructions per 16 keys, a third of them widening, and neither the issue slots (0.4 busy) nor DRAM
// (42 %) are the limit, but the latency of three warps per scheduler, whose 168 registers hold two
// steps of keys as they are read.
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

// Row r of (sequence, KV head): its packed token and query head.
struct QueryRow {
  int tok, hq;
};
__device__ __forceinline__ QueryRow query_row(const PagedAttn& a, const Seq& s, int h, int r) {
  return {s.c0 + r / a.group, h * a.group + r % a.group};
}

// Positions of the work order that a (sequence, head) takes besides its steps: its
// queries, and the wait for its first keys.
constexpr int kSegmentCost = 2;

template <int D, int KV>
struct Stream {
  static constexpr bool k8 = KV >= FA_DTYPE_INT8;
  static constexpr int kRowBytes = k8 ? D : 2 * D;
  static constexpr int kChunks = kRowBytes / 64;  // 16-byte pieces of a lane per key
  static constexpr int kTiles = k8 ? 2 : 1;       // of 16 keys in a step
  static constexpr int kKeys = 16 * kTiles;
  static constexpr int kPairs = D / 8;            // 32-bit operands of a lane per query row
};

__device__ __forceinline__ long long shfl64(long long x, int src) {
  const int lo = __shfl_sync(0xffffffffu, static_cast<int>(x), src);
  const int hi = __shfl_sync(0xffffffffu, static_cast<int>(x >> 32), src);
  return (static_cast<long long>(hi) << 32) | static_cast<unsigned>(lo);
}

template <int D, int KV>
struct KeyStep {
  using S = Stream<D, KV>;
  uint4 x[S::kTiles][2][S::kChunks];  // keys g, g + 8 of a tile
  float ks[S::kTiles][2];
  float old;                          // earlier sum of this lane's key (key_of)
};

__device__ __forceinline__ uint4 load_once(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__host__ __device__ constexpr int few_ctas_per_sm(int nt) { return nt == 1 ? 4 : nt == 2 ? 3 : 2; }

template <int D, int KV, bool QBF16, int NT>
__global__ void __launch_bounds__(kWeightThreads, few_ctas_per_sm(NT))
    paged_weights_few_kernel(const PagedWeights p, int max_rows, int n_warps) {
  using S = Stream<D, KV>;
  constexpr bool kBf16 = !S::k8 && QBF16;  // type of the products
  constexpr int kWarps = kWeightThreads / 32;
  const PagedAttn& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, j = lane & 3;
  const int H = a.c.heads;

  // ---- the warp's run [v, v1), relative to sequence b's first position
  __shared__ long long sh_scan[kWarps];
  __shared__ int sh_b[kWarps];
  __shared__ long long sh_rel[kWarps];
  auto steps_of = [&](const Seq& s) {
    return static_cast<long long>(s.nq) * a.group > max_rows ? 0 : (s.nk + S::kKeys - 1) / S::kKeys;
  };
  auto positions = [&](int b) -> long long {
    const int n = steps_of(load_seq(a, b));
    return n > 0 ? static_cast<long long>(n + kSegmentCost) * H : 0;
  };
  long long v, v1;
  int b;
  {
    const int share = (a.r.B + kWeightThreads - 1) / kWeightThreads;
    const int s0 = min(static_cast<int>(threadIdx.x) * share, a.r.B), s1 = min(s0 + share, a.r.B);
    long long sum = 0, total;
    for (int i = s0; i < s1; ++i) sum += positions(i);
    const long long lo = block_scan<kWeightThreads>(sum, sh_scan, &total);
    const long long per = (total + n_warps - 1) / n_warps;
    for (int w = 0; w < kWarps; ++w) {
      const long long first = per * (static_cast<long long>(blockIdx.x) * kWarps + w);
      if (first < total && first >= lo && first < lo + sum) {
        long long x = lo;
        for (int i = s0; i < s1; ++i) {
          const long long n = positions(i);
          if (first < x + n) {
            sh_b[w] = i;
            sh_rel[w] = first - x;
            break;
          }
          x += n;
        }
      }
    }
    __syncthreads();
    const long long v0 = per * (static_cast<long long>(blockIdx.x) * kWarps + warp);
    if (v0 >= total) return;
    b = sh_b[warp];
    v = sh_rel[warp];
    v1 = min(v0 + per, total) - v0 + v;
  }

  for (Seq s = load_seq(a, b);;) {
    const int n_all = steps_of(s), seg = n_all + kSegmentCost;
    const int h = static_cast<int>(v / seg);
    const long long at = static_cast<long long>(h) * seg + kSegmentCost;  // of the head's first step
    const int t0 = static_cast<int>(max(v - at, 0ll)), t1 = static_cast<int>(min(v1 - at, static_cast<long long>(n_all)));
    if (t0 < t1) {
      const int fresh0 = p.mode == FA_WEIGHTS_SET      ? 0
                         : p.mode == FA_WEIGHTS_APPEND ? min(__ldg(a.r.lens + b), 3 << 29) - s.n
                                                       : 0x7fffffff;
      float* const w = p.w + b * p.w_seq + h * p.w_head;
      // the key of a step whose sum this lane gets: with one tile, lanes j and j + 2 the same
      auto key_of = [&](int t) { return t * S::kKeys + (S::kTiles == 2 ? 8 * j : 8 * (j & 1)) + g; };
      // Offsets of the 16-key groups' first rows and scales (-1: no page, or no key any row may
      // see): lane l has those of group wbase + l, and the page of group wbase + 32 + l.
      int wbase = t0 * S::kTiles;
      auto page_at = [&](int first) {
        const int pos = 16 * (first + lane);
        return first + lane < t1 * S::kTiles && pos < s.vis ? a.c.lookup(b, pos) : -1;
      };
      long long win, win_scale = 0;
      int next_page = page_at(wbase);
      auto next_window = [&] {
        const int page = next_page, row = a.c.row_in_page(16 * (wbase + lane));
        win = page < 0 ? -1 : page * a.c.page_stride + row * a.c.row_stride;
        if constexpr (S::k8) win_scale = page * a.c.s_page + row * a.c.s_row;
        next_page = page_at(wbase + 32);
      };
      next_window();
      const uint8_t* const k_lane = a.c.k + h * a.c.head_stride + g * a.c.row_stride + 16 * j;
      const long long row8 = 8 * a.c.row_stride;
      const float* const ks_lane = S::k8 ? a.c.ks + h * a.c.s_head + g * a.c.s_row : nullptr;

      auto load = [&](KeyStep<D, KV>& st, int t) {
        if (t * S::kTiles >= wbase + 32) {
          wbase += 32;
          next_window();
        }
#pragma unroll
        for (int m = 0; m < S::kTiles; ++m) {
          const int key0 = t * S::kKeys + 16 * m;
          const long long off = shfl64(win, t * S::kTiles + m - wbase);
          const uint8_t* const src = k_lane + off;
          const float* sc = nullptr;
          if constexpr (S::k8) sc = ks_lane + shfl64(win_scale, t * S::kTiles + m - wbase);
          if (off >= 0 && key0 + 16 <= s.vis) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
#pragma unroll
              for (int c = 0; c < S::kChunks; ++c) st.x[m][y][c] = load_once(src + y * row8 + 64 * c);
              if constexpr (S::k8) st.ks[m][y] = __ldg(sc + 8 * y * a.c.s_row);
            }
          } else {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const bool ok = off >= 0 && key0 + g + 8 * y < s.vis;
#pragma unroll
              for (int c = 0; c < S::kChunks; ++c)
                st.x[m][y][c] = ok ? load_once(src + y * row8 + 64 * c) : make_uint4(0u, 0u, 0u, 0u);
              if constexpr (S::k8) st.ks[m][y] = ok ? __ldg(sc + 8 * y * a.c.s_row) : 0.f;
            }
          }
        }
        const int key = key_of(t);
        st.old = key < min(s.nk, fresh0) ? w[key] : 0.f;
      };

      KeyStep<D, KV> cur, next;
      load(cur, t0);

      // ---- query rows: operands, LSE and key limit of this thread's two rows per block of 8
      const int rows = s.nq * a.group;
      uint32_t q[NT][S::kPairs];
      float cs[NT][2], nlse[NT][2];
      int lim[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = nt * 8 + g;
        const QueryRow qr = query_row(a, s, h, r);
        const uint8_t* const src = a.q + static_cast<long long>(qr.tok) * a.q_token + qr.hq * a.q_head;
#pragma unroll
        for (int i = 0; i < S::kPairs / 4; ++i) {
          // 16-bit keys: the piece of 8 columns at 32 i + 8 j; 8-bit keys: the half i % 2 of the
          // 16 columns at 64 (i / 2) + 16 j
          const int byte = S::k8 ? 128 * (i / 2) + 32 * j + 16 * (i % 2) : 64 * i + 16 * j;
          const uint4 v = r < rows ? __ldg(reinterpret_cast<const uint4*>(src + byte)) : make_uint4(0u, 0u, 0u, 0u);
          q[nt][4 * i] = v.x;
          q[nt][4 * i + 1] = v.y;
          q[nt][4 * i + 2] = v.z;
          q[nt][4 * i + 3] = v.w;
        }
        float unit = 1.f;
        if constexpr (S::k8 && QBF16) {
          unit = bf16_row_as_f16<S::kPairs>([&](int i) -> uint32_t& { return q[nt][i]; });
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int rc = nt * 8 + 2 * j + c;
          const QueryRow qc = query_row(a, s, h, rc);
          float l = -INFINITY;
          if (rc < rows) l = a.lse[static_cast<long long>(qc.hq) * a.r.total + qc.tok];
          lim[nt][c] = l == -INFINITY ? 0 : row_limit(a, s, rc / a.group);
          nlse[nt][c] = l == -INFINITY ? 0.f : l * -1.4426950408889634f;
          cs[nt][c] = a.scale_log2;
          if constexpr (S::k8 && QBF16) cs[nt][c] *= __shfl_sync(0xffffffffu, unit, (2 * j + c) * 4);
        }
      }
      int all = 0x7fffffff;  // every row sees the keys below
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) all = min(all, min(lim[nt][0], lim[nt][1]));
      all = __reduce_min_sync(0xffffffffu, all);
      auto compute = [&](const KeyStep<D, KV>& st, int t) {
        float sum[S::kTiles][2];
#pragma unroll
        for (int m = 0; m < S::kTiles; ++m) {
          const int key0 = t * S::kKeys + 16 * m;
          float c[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.f;
#pragma unroll
          for (int i = 0; i < S::kChunks; ++i) {
            const uint32_t k0[4] = {st.x[m][0][i].x, st.x[m][0][i].y, st.x[m][0][i].z, st.x[m][0][i].w};
            const uint32_t k1[4] = {st.x[m][1][i].x, st.x[m][1][i].y, st.x[m][1][i].z, st.x[m][1][i].w};
            if constexpr (!S::k8) {
#pragma unroll
              for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                  mma16816<kBf16>(c[nt], k0[2 * e], k1[2 * e], k0[2 * e + 1], k1[2 * e + 1], q[nt][4 * i + 2 * e],
                                   q[nt][4 * i + 2 * e + 1]);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                uint32_t a0, a1, a2, a3;
                widen<KV, false>(k0[e], a0, a2);
                widen<KV, false>(k1[e], a1, a3);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                  mma16816<false>(c[nt], a0, a1, a2, a3, q[nt][8 * i + 2 * e], q[nt][8 * i + 2 * e + 1]);
              }
            }
          }
          float v[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              float x0 = c[nt][2 * y], x1 = c[nt][2 * y + 1];
              if constexpr (S::k8) ptx::fmul2(x0, x1, x0, x1, st.ks[m][y], st.ks[m][y]);
              ptx::ffma2(x0, x1, x0, x1, cs[nt][0], cs[nt][1], nlse[nt][0], nlse[nt][1]);
              v[nt][2 * y] = ptx::ex2_approx(x0);
              v[nt][2 * y + 1] = ptx::ex2_approx(x1);
            }
          if (key0 + 16 > all) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (key0 + g + 8 * (i >> 1) >= lim[nt][i & 1]) v[nt][i] = 0.f;
          }
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            sum[m][y] = v[0][2 * y] + v[0][2 * y + 1];
#pragma unroll
            for (int nt = 1; nt < NT; ++nt) sum[m][y] += v[nt][2 * y] + v[nt][2 * y + 1];
          }
        }
        // over the quad's lanes: each keeps the half it needs and hands on the other
        float mine[S::kTiles];
#pragma unroll
        for (int m = 0; m < S::kTiles; ++m)
          mine[m] = (j & 1 ? sum[m][1] : sum[m][0]) + __shfl_xor_sync(0xffffffffu, j & 1 ? sum[m][0] : sum[m][1], 1);
        float total;
        if constexpr (S::kTiles == 2)
          total = (j & 2 ? mine[1] : mine[0]) + __shfl_xor_sync(0xffffffffu, j & 2 ? mine[0] : mine[1], 2);
        else
          total = mine[0] + __shfl_xor_sync(0xffffffffu, mine[0], 2);
        const int key = key_of(t);
        if ((S::kTiles == 2 || j < 2) && key < s.nk) w[key] = st.old + total;
      };
      for (int t = t0; t < t1; t += 2) {
        if (t + 1 < t1) load(next, t + 1);
        compute(cur, t);
        if (t + 1 >= t1) break;
        if (t + 2 < t1) load(cur, t + 2);
        compute(next, t + 1);
      }
    }
    // ---- the next segment
    v = at + n_all;
    if (v >= v1) break;
    if (h + 1 == H) {
      v1 -= v;
      v = 0;
      do {
        if (++b >= a.r.B) return;
        s = load_seq(a, b);
      } while (steps_of(s) == 0);
    }
  }
}

template <int D, int KV, bool QBF16, int NT>
cudaError_t few_impl(const PagedWeights& p, int max_rows, int sms, cudaStream_t stream) {
  using S = Stream<D, KV>;
  constexpr int kWarps = kWeightThreads / 32;
  // no more warps than steps there can be
  const long long heads = static_cast<long long>(p.a.r.B) * p.a.c.heads;
  const long long steps = heads * ((static_cast<long long>(p.a.max_k) + S::kKeys - 1) / S::kKeys);
  const long long most = static_cast<long long>(sms) * few_ctas_per_sm(NT);
  const long long ctas = (steps + kWarps - 1) / kWarps;
  const int grid = static_cast<int>(ctas < most ? ctas : most);
  paged_weights_few_kernel<D, KV, QBF16, NT><<<grid, kWeightThreads, 0, stream>>>(p, max_rows, grid * kWarps);
  return cudaGetLastError();
}

template <int D, int KV, bool QBF16>
cudaError_t weights_impl(const PagedWeights& p, int max_rows, int sms, cudaStream_t stream) {
  if (max_rows <= 8) return few_impl<D, KV, QBF16, 1>(p, max_rows, sms, stream);
  if (max_rows <= 16) return few_impl<D, KV, QBF16, 2>(p, max_rows, sms, stream);
  return few_impl<D, KV, QBF16, 4>(p, max_rows, sms, stream);
}

template <int D>
cudaError_t weights_d(const PagedWeights& p, int n, int kv, bool bf16, int sms, cudaStream_t s) {
  switch (kv) {
    case FA_DTYPE_INT8:
      return bf16 ? weights_impl<D, FA_DTYPE_INT8, true>(p, n, sms, s) : weights_impl<D, FA_DTYPE_INT8, false>(p, n, sms, s);
    case FA_DTYPE_E4M3:
      return bf16 ? weights_impl<D, FA_DTYPE_E4M3, true>(p, n, sms, s) : weights_impl<D, FA_DTYPE_E4M3, false>(p, n, sms, s);
    case FA_DTYPE_BF16: return weights_impl<D, FA_DTYPE_BF16, true>(p, n, sms, s);
    default: return weights_impl<D, FA_DTYPE_F16, false>(p, n, sms, s);
  }
}

}  // namespace

cudaError_t launch_paged_weights(const PagedWeights& p, int max_rows, int head_dim, int cache_dtype, bool bf16, int sms,
                                 cudaStream_t stream) {
  return head_dim == 64 ? weights_d<64>(p, max_rows, cache_dtype, bf16, sms, stream)
                        : weights_d<128>(p, max_rows, cache_dtype, bf16, sms, stream);
}

}  // namespace fa
