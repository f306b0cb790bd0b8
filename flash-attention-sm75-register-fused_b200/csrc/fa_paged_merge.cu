// Joins the results of two passes over different keys of the same query rows (both
// normalised, fp32, with their natural-log LSE): with f_p = exp(LSE_p - LSE),
//   LSE = log(exp LSE_1 + exp LSE_2),   O = f_1 O_1 + f_2 O_2,
// rounded once.  Bound by latency for a decode step's rows (2 to 3 us, started while the pass
// before it ends), by memory for more: 4 d + 2 d bytes a row and pass.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "fa_paged.h"
#include "fa_paged_dev.cuh"
#include "sm100_ptx.cuh"

namespace fa {
namespace {

constexpr int kMergeThreads = 128;

// D / 4 threads a row, one 16-byte piece of either result each.
template <int D, bool BF16>
__global__ void __launch_bounds__(kMergeThreads) paged_merge_kernel(const PagedMerge p) {
  ptx::grid_dep_wait();
  const long long i = static_cast<long long>(blockIdx.x) * kMergeThreads + threadIdx.x;
  const long long row = i / (D / 4);  // token * Hq + head
  if (row >= static_cast<long long>(p.total) * p.Hq) return;
  const float4 x = __ldcg(reinterpret_cast<const float4*>(p.o1) + i);
  const float4 y = __ldcg(reinterpret_cast<const float4*>(p.o2) + i);
  const float l1 = __ldcg(p.lse1 + row), l2 = __ldcg(p.lse2 + row);
  Joined j{0.f, 0.f, -INFINITY};
  if (__float_as_uint(l2) != kNoRow) j = join_passes(l1, l2);
  float o[4] = {0.f, 0.f, 0.f, 0.f};
  // (a set without a key for this row has no O)
  if (j.own != 0.f) {
    o[0] = y.x * j.own;
    o[1] = y.y * j.own;
    o[2] = y.z * j.own;
    o[3] = y.w * j.own;
  }
  if (j.first != 0.f) {
    o[0] = fmaf(x.x, j.first, o[0]);
    o[1] = fmaf(x.y, j.first, o[1]);
    o[2] = fmaf(x.z, j.first, o[2]);
    o[3] = fmaf(x.w, j.first, o[3]);
  }
  uint2 w;
  if constexpr (BF16) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(o[0], o[1]), b = __floats2bfloat162_rn(o[2], o[3]);
    w = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
  } else {
    const __half2 a = __floats2half2_rn(o[0], o[1]), b = __floats2half2_rn(o[2], o[3]);
    w = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
  }
  static_cast<uint2*>(p.o)[i] = w;
  if (i % (D / 4) == 0 && p.lse != nullptr)
    p.lse[row % p.Hq * p.total + row / p.Hq] = j.lse;
}

}  // namespace

cudaError_t launch_paged_merge(const PagedMerge& p, int head_dim, bool bf16, cudaStream_t stream) {
  const long long n = static_cast<long long>(p.total) * p.Hq * (head_dim / 4);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((n + kMergeThreads - 1) / kMergeThreads));
  cfg.blockDim = dim3(kMergeThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (head_dim == 64)
    return bf16 ? cudaLaunchKernelEx(&cfg, paged_merge_kernel<64, true>, p)
                : cudaLaunchKernelEx(&cfg, paged_merge_kernel<64, false>, p);
  return bf16 ? cudaLaunchKernelEx(&cfg, paged_merge_kernel<128, true>, p)
              : cudaLaunchKernelEx(&cfg, paged_merge_kernel<128, false>, p);
}

}  // namespace fa
