// pybind module `flash_attn_sm75_cuda` — the reference's L3 binding
// (src/bindings/pytorch_extension.cpp:1-129) re-implemented over the C ABI in
// include/fa_b200.h.  Same four exported functions with the same argument
// lists and input checks; the kernels run asynchronously on PyTorch's
// current CUDA stream instead of the legacy stream + cudaDeviceSynchronize.
//
// Additions: native GQA (K/V may have fewer heads than Q), bf16 inputs,
// flash_attention_forward_lse returning (O, LSE), flash_attention_forward_kvcache
// (Nq != Nk: decode and chunked prefill), the paged KV cache (write, read back,
// attention, also behind shared prefixes, summed weights, eviction), and diagnostics.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>

#include "fa_b200.h"

namespace {

void check_tensor(const torch::Tensor& t, const char* name, bool allow_bf16) {
  TORCH_CHECK(t.is_cuda(), std::string(name) + " must be a CUDA tensor");
  if (allow_bf16) {
    TORCH_CHECK(t.dtype() == torch::kFloat16 || t.dtype() == torch::kBFloat16,
                std::string(name) + " must be FP16 or BF16");
  } else {
    TORCH_CHECK(t.dtype() == torch::kFloat16, std::string(name) + " must be FP16");
  }
  TORCH_CHECK(t.is_contiguous(), std::string(name) + " must be contiguous");
  TORCH_CHECK(t.dim() == 4, std::string(name) + " must be [B, H, N, D]");
}

void* stream_of(const torch::Tensor& t) {
  return static_cast<void*>(at::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

std::tuple<torch::Tensor, torch::Tensor> fwd_impl(const torch::Tensor& Q, const torch::Tensor& K,
                                                  const torch::Tensor& V, bool causal, float scale,
                                                  bool want_lse) {
  check_tensor(Q, "Q", true);
  check_tensor(K, "K", true);
  check_tensor(V, "V", true);
  TORCH_CHECK(Q.dtype() == K.dtype() && Q.dtype() == V.dtype(), "Q, K, V must share a dtype");
  TORCH_CHECK(Q.device() == K.device() && Q.device() == V.device(),
              "Q, K, V must be on the same device");
  TORCH_CHECK(Q.size(0) == K.size(0), "batch mismatch");
  TORCH_CHECK(Q.size(2) == K.size(2), "seq_len mismatch");
  TORCH_CHECK(Q.size(3) == K.size(3), "head_dim mismatch");
  TORCH_CHECK(K.sizes() == V.sizes(), "K and V must have identical shapes");
  const auto head_dim = Q.size(3);
  TORCH_CHECK(head_dim == 64 || head_dim == 128,
              "flash_attention_forward supports head_dim=64 or 128, got ", head_dim);
  TORCH_CHECK(K.size(1) > 0 && Q.size(1) % K.size(1) == 0, "GQA: Q heads (", Q.size(1),
              ") not divisible by K/V heads (", K.size(1), ")");
  TORCH_CHECK(Q.size(0) <= INT32_MAX && Q.size(1) <= INT32_MAX && Q.size(2) <= INT32_MAX,
              "size exceeds int32");

  const c10::cuda::CUDAGuard guard(Q.device());
  auto O = torch::empty_like(Q);
  torch::Tensor lse;
  if (want_lse)
    lse = torch::empty({Q.size(0), Q.size(1), Q.size(2)},
                       Q.options().dtype(torch::kFloat32));
  const int rc = fa_fwd(Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(),
                        want_lse ? lse.data_ptr<float>() : nullptr, static_cast<int>(Q.size(0)),
                        static_cast<int>(Q.size(1)), static_cast<int>(K.size(1)),
                        static_cast<int>(Q.size(2)), static_cast<int>(head_dim), scale,
                        causal ? 1 : 0,
                        Q.dtype() == torch::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16,
                        stream_of(Q));
  TORCH_CHECK(rc == FA_OK, "flash_attention_forward: ", fa_error_string(rc));
  return {O, lse};
}

// Forward into caller-provided O (and optional LSE) on the current stream;
// used by the host-buffer pipeline, which computes per-chunk slices in place.
void flash_attention_forward_out(torch::Tensor Q, torch::Tensor K, torch::Tensor V,
                                 torch::Tensor O, c10::optional<torch::Tensor> lse, bool causal,
                                 float scale) {
  check_tensor(Q, "Q", true);
  check_tensor(K, "K", true);
  check_tensor(V, "V", true);
  check_tensor(O, "O", true);
  TORCH_CHECK(Q.dtype() == K.dtype() && Q.dtype() == V.dtype() && Q.dtype() == O.dtype(),
              "Q, K, V, O must share a dtype");
  TORCH_CHECK(Q.device() == K.device() && Q.device() == V.device() && Q.device() == O.device(),
              "Q, K, V, O must be on the same device");
  TORCH_CHECK(O.sizes() == Q.sizes(), "O must have Q's shape");
  TORCH_CHECK(Q.size(0) == K.size(0) && Q.size(2) == K.size(2) && Q.size(3) == K.size(3),
              "Q and K shapes differ beyond the head count");
  TORCH_CHECK(K.sizes() == V.sizes(), "K and V must have identical shapes");
  const auto head_dim = Q.size(3);
  TORCH_CHECK(head_dim == 64 || head_dim == 128,
              "flash_attention_forward supports head_dim=64 or 128, got ", head_dim);
  TORCH_CHECK(K.size(1) > 0 && Q.size(1) % K.size(1) == 0, "GQA: Q heads (", Q.size(1),
              ") not divisible by K/V heads (", K.size(1), ")");
  float* lse_ptr = nullptr;
  if (lse.has_value() && lse->defined()) {
    TORCH_CHECK(lse->is_cuda() && lse->dtype() == torch::kFloat32 && lse->is_contiguous() &&
                    lse->dim() == 3 && lse->size(0) == Q.size(0) && lse->size(1) == Q.size(1) &&
                    lse->size(2) == Q.size(2),
                "lse must be a contiguous fp32 CUDA tensor [B, Hq, N]");
    lse_ptr = lse->data_ptr<float>();
  }
  TORCH_CHECK(Q.size(0) <= INT32_MAX && Q.size(1) <= INT32_MAX && Q.size(2) <= INT32_MAX,
              "size exceeds int32");
  const c10::cuda::CUDAGuard guard(Q.device());
  const int rc = fa_fwd(Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(), lse_ptr,
                        static_cast<int>(Q.size(0)), static_cast<int>(Q.size(1)),
                        static_cast<int>(K.size(1)), static_cast<int>(Q.size(2)),
                        static_cast<int>(head_dim), scale, causal ? 1 : 0,
                        Q.dtype() == torch::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16,
                        stream_of(Q));
  TORCH_CHECK(rc == FA_OK, "flash_attention_forward: ", fa_error_string(rc));
}

torch::Tensor flash_attention_forward(torch::Tensor Q, torch::Tensor K, torch::Tensor V,
                                      bool causal, float scale) {
  return std::get<0>(fwd_impl(Q, K, V, causal, scale, false));
}

std::tuple<torch::Tensor, torch::Tensor> flash_attention_forward_lse(torch::Tensor Q,
                                                                     torch::Tensor K,
                                                                     torch::Tensor V, bool causal,
                                                                     float scale) {
  return fwd_impl(Q, K, V, causal, scale, true);
}

// Reference ablation exports (d=64, identical shapes): one kernel serves all.
torch::Tensor d64_variant(const char* what, torch::Tensor Q, torch::Tensor K, torch::Tensor V,
                          bool causal, float scale) {
  check_tensor(Q, "Q", false);
  check_tensor(K, "K", false);
  check_tensor(V, "V", false);
  TORCH_CHECK(Q.sizes() == K.sizes() && Q.sizes() == V.sizes(),
              "Q, K, V must have identical shapes");
  TORCH_CHECK(Q.size(3) == 64, std::string(what) + " kernel supports head_dim=64 only");
  return flash_attention_forward(Q, K, V, causal, scale);
}

torch::Tensor flash_attention_forward_scalar(torch::Tensor Q, torch::Tensor K, torch::Tensor V,
                                             bool causal, float scale) {
  return d64_variant("scalar", Q, K, V, causal, scale);
}

torch::Tensor flash_attention_forward_wmma_qk(torch::Tensor Q, torch::Tensor K, torch::Tensor V,
                                              bool causal, float scale) {
  return d64_variant("wmma_qk", Q, K, V, causal, scale);
}

torch::Tensor naive_attention_forward(torch::Tensor Q, torch::Tensor K, torch::Tensor V,
                                      bool causal, float scale) {
  check_tensor(Q, "Q", false);
  check_tensor(K, "K", false);
  check_tensor(V, "V", false);
  TORCH_CHECK(Q.sizes() == K.sizes() && Q.sizes() == V.sizes(),
              "naive_attention: Q, K, V must have identical shapes");
  const c10::cuda::CUDAGuard guard(Q.device());
  auto O = torch::empty_like(Q);
  auto ws = torch::empty({Q.size(0) * Q.size(1), Q.size(2), Q.size(2)},
                         Q.options().dtype(torch::kFloat32));
  const int rc = fa_naive_fwd(Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(),
                              static_cast<int>(Q.size(0)), static_cast<int>(Q.size(1)),
                              static_cast<int>(Q.size(2)), static_cast<int>(Q.size(3)), scale,
                              causal ? 1 : 0, ws.data_ptr<float>(), stream_of(Q));
  TORCH_CHECK(rc == FA_OK, "naive_attention_forward: ", fa_error_string(rc));
  return O;
}

// Nq new queries against Nk cached keys (decode / chunked prefill); causal is
// an FA_CAUSAL_* mode.  The split-KV workspace comes from PyTorch's caching
// allocator on the current stream.  Returns (O, LSE).
std::tuple<torch::Tensor, torch::Tensor> flash_attention_forward_kvcache(
    torch::Tensor Q, torch::Tensor K, torch::Tensor V, int64_t causal, float scale) {
  check_tensor(Q, "Q", true);
  check_tensor(K, "K", true);
  check_tensor(V, "V", true);
  TORCH_CHECK(Q.dtype() == K.dtype() && Q.dtype() == V.dtype(), "Q, K, V must share a dtype");
  TORCH_CHECK(Q.device() == K.device() && Q.device() == V.device(),
              "Q, K, V must be on the same device");
  TORCH_CHECK(Q.size(0) == K.size(0), "batch mismatch");
  TORCH_CHECK(Q.size(3) == K.size(3), "head_dim mismatch");
  TORCH_CHECK(K.sizes() == V.sizes(), "K and V must have identical shapes");
  const auto head_dim = Q.size(3);
  TORCH_CHECK(head_dim == 64 || head_dim == 128,
              "flash_attention_forward supports head_dim=64 or 128, got ", head_dim);
  TORCH_CHECK(K.size(1) > 0 && Q.size(1) % K.size(1) == 0, "GQA: Q heads (", Q.size(1),
              ") not divisible by K/V heads (", K.size(1), ")");
  TORCH_CHECK(causal >= FA_CAUSAL_NONE && causal <= FA_CAUSAL_TOP_LEFT, "bad causal mode ", causal);
  TORCH_CHECK(Q.size(0) <= INT32_MAX && Q.size(1) <= INT32_MAX && Q.size(2) <= INT32_MAX &&
                  K.size(2) <= INT32_MAX,
              "size exceeds int32");
  const c10::cuda::CUDAGuard guard(Q.device());
  const int B = static_cast<int>(Q.size(0)), Hq = static_cast<int>(Q.size(1));
  const int Hkv = static_cast<int>(K.size(1)), Nq = static_cast<int>(Q.size(2));
  const int Nk = static_cast<int>(K.size(2)), d = static_cast<int>(head_dim);
  auto O = torch::empty_like(Q);
  auto lse = torch::empty({Q.size(0), Q.size(1), Q.size(2)}, Q.options().dtype(torch::kFloat32));
  const size_t ws_bytes = fa_fwd_kvcache_workspace_bytes(B, Hq, Hkv, Nq, Nk, d);
  torch::Tensor ws;
  if (ws_bytes > 0)
    ws = torch::empty({static_cast<int64_t>(ws_bytes)}, Q.options().dtype(torch::kUInt8));
  const int rc = fa_fwd_kvcache(
      Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(), lse.data_ptr<float>(), B, Hq, Hkv,
      Nq, Nk, d, scale, static_cast<int>(causal),
      Q.dtype() == torch::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16,
      ws_bytes > 0 ? ws.data_ptr() : nullptr, ws_bytes, stream_of(Q));
  TORCH_CHECK(rc == FA_OK, "flash_attention_forward_kvcache: ", fa_error_string(rc));
  return {O, lse};
}

void check_rows(const torch::Tensor& t, const char* name, int64_t n, const torch::Tensor& like) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), std::string(name) +
                                                              " must be on the inputs' device");
  TORCH_CHECK(t.dtype() == torch::kInt32 && t.dim() == 1 && t.is_contiguous() && t.size(0) == n,
              std::string(name) + " must be a contiguous int32 tensor of ", n, " entries");
}

void check_packed(const torch::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), std::string(name) + " must be a CUDA tensor");
  TORCH_CHECK(t.dtype() == torch::kFloat16 || t.dtype() == torch::kBFloat16,
              std::string(name) + " must be FP16 or BF16");
  TORCH_CHECK(t.is_contiguous(), std::string(name) + " must be contiguous");
  TORCH_CHECK(t.dim() == 3, std::string(name) + " must be [total, H, D]");
}

// Packed variable-length batch: Q [total_q, Hq, d], K/V [total_k, Hkv, d],
// cu_seqlens_* int32 [B + 1] on the device.  Returns O [total_q, Hq, d] and
// LSE fp32 [Hq, total_q].
std::tuple<torch::Tensor, torch::Tensor> flash_attention_forward_varlen(
    torch::Tensor Q, torch::Tensor K, torch::Tensor V, torch::Tensor cu_seqlens_q,
    torch::Tensor cu_seqlens_k, int64_t max_seqlen_q, int64_t max_seqlen_k, int64_t causal,
    float scale) {
  check_packed(Q, "Q");
  check_packed(K, "K");
  check_packed(V, "V");
  TORCH_CHECK(Q.dtype() == K.dtype() && Q.dtype() == V.dtype(), "Q, K, V must share a dtype");
  TORCH_CHECK(Q.device() == K.device() && Q.device() == V.device(),
              "Q, K, V must be on the same device");
  TORCH_CHECK(K.sizes() == V.sizes(), "K and V must have identical shapes");
  TORCH_CHECK(Q.size(2) == K.size(2), "head_dim mismatch");
  const auto head_dim = Q.size(2);
  TORCH_CHECK(head_dim == 64 || head_dim == 128,
              "flash_attention_forward supports head_dim=64 or 128, got ", head_dim);
  TORCH_CHECK(K.size(1) > 0 && Q.size(1) % K.size(1) == 0, "GQA: Q heads (", Q.size(1),
              ") not divisible by K/V heads (", K.size(1), ")");
  TORCH_CHECK(causal >= FA_CAUSAL_NONE && causal <= FA_CAUSAL_TOP_LEFT, "bad causal mode ", causal);
  TORCH_CHECK(cu_seqlens_q.dim() == 1 && cu_seqlens_q.size(0) >= 1,
              "cu_seqlens_q must be [B + 1]");
  const int64_t B = cu_seqlens_q.size(0) - 1;
  check_rows(cu_seqlens_q, "cu_seqlens_q", B + 1, Q);
  check_rows(cu_seqlens_k, "cu_seqlens_k", B + 1, Q);
  TORCH_CHECK(Q.size(0) <= INT32_MAX && K.size(0) <= INT32_MAX && max_seqlen_q >= 0 &&
                  max_seqlen_q <= INT32_MAX && max_seqlen_k >= 0 && max_seqlen_k <= INT32_MAX,
              "size exceeds int32");
  const c10::cuda::CUDAGuard guard(Q.device());
  auto O = torch::zeros_like(Q);
  auto lse = torch::full({Q.size(1), Q.size(0)}, -INFINITY, Q.options().dtype(torch::kFloat32));
  const int rc = fa_fwd_varlen(
      Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(), lse.data_ptr<float>(),
      cu_seqlens_q.data_ptr<int>(), cu_seqlens_k.data_ptr<int>(), static_cast<int>(B),
      static_cast<int>(Q.size(1)), static_cast<int>(K.size(1)), static_cast<int>(Q.size(0)),
      static_cast<int>(K.size(0)), static_cast<int>(max_seqlen_q), static_cast<int>(max_seqlen_k),
      static_cast<int>(head_dim), scale, static_cast<int>(causal),
      Q.dtype() == torch::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16, stream_of(Q));
  TORCH_CHECK(rc == FA_OK, "flash_attention_forward_varlen: ", fa_error_string(rc));
  return {O, lse};
}

// Padded batch: Q [B, Hq, Nq, d], K/V [B, Hkv, Nk, d] and per batch entry the
// valid query rows [q_start, q_end) and key rows [k_start, k_end) (int32 [B]
// on the device).  Rows outside a query range come back as O = 0, LSE = -inf.
std::tuple<torch::Tensor, torch::Tensor> flash_attention_forward_padded(
    torch::Tensor Q, torch::Tensor K, torch::Tensor V, torch::Tensor q_start, torch::Tensor q_end,
    torch::Tensor k_start, torch::Tensor k_end, int64_t causal, float scale) {
  check_tensor(Q, "Q", true);
  check_tensor(K, "K", true);
  check_tensor(V, "V", true);
  TORCH_CHECK(Q.dtype() == K.dtype() && Q.dtype() == V.dtype(), "Q, K, V must share a dtype");
  TORCH_CHECK(Q.device() == K.device() && Q.device() == V.device(),
              "Q, K, V must be on the same device");
  TORCH_CHECK(Q.size(0) == K.size(0), "batch mismatch");
  TORCH_CHECK(Q.size(3) == K.size(3), "head_dim mismatch");
  TORCH_CHECK(K.sizes() == V.sizes(), "K and V must have identical shapes");
  const auto head_dim = Q.size(3);
  TORCH_CHECK(head_dim == 64 || head_dim == 128,
              "flash_attention_forward supports head_dim=64 or 128, got ", head_dim);
  TORCH_CHECK(K.size(1) > 0 && Q.size(1) % K.size(1) == 0, "GQA: Q heads (", Q.size(1),
              ") not divisible by K/V heads (", K.size(1), ")");
  TORCH_CHECK(causal >= FA_CAUSAL_NONE && causal <= FA_CAUSAL_TOP_LEFT, "bad causal mode ", causal);
  const int64_t B = Q.size(0);
  check_rows(q_start, "q_start", B, Q);
  check_rows(q_end, "q_end", B, Q);
  check_rows(k_start, "k_start", B, Q);
  check_rows(k_end, "k_end", B, Q);
  TORCH_CHECK(Q.size(0) <= INT32_MAX && Q.size(1) <= INT32_MAX && Q.size(2) <= INT32_MAX &&
                  K.size(2) <= INT32_MAX,
              "size exceeds int32");
  const c10::cuda::CUDAGuard guard(Q.device());
  auto O = torch::zeros_like(Q);
  auto lse = torch::full({Q.size(0), Q.size(1), Q.size(2)}, -INFINITY,
                         Q.options().dtype(torch::kFloat32));
  const int rc = fa_fwd_padded(
      Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(), lse.data_ptr<float>(),
      q_start.data_ptr<int>(), q_end.data_ptr<int>(), k_start.data_ptr<int>(),
      k_end.data_ptr<int>(), static_cast<int>(B), static_cast<int>(Q.size(1)),
      static_cast<int>(K.size(1)), static_cast<int>(Q.size(2)), static_cast<int>(K.size(2)),
      static_cast<int>(head_dim), scale, static_cast<int>(causal),
      Q.dtype() == torch::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16, stream_of(Q));
  TORCH_CHECK(rc == FA_OK, "flash_attention_forward_padded: ", fa_error_string(rc));
  return {O, lse};
}

// Gradients of flash_attention_forward_lse: (dQ, dK, dV) from dO, the inputs,
// the forward's O and LSE.  The workspace comes from PyTorch's allocator.
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> flash_attention_backward(
    torch::Tensor dO, torch::Tensor Q, torch::Tensor K, torch::Tensor V, torch::Tensor O,
    torch::Tensor lse, bool causal, float scale) {
  check_tensor(Q, "Q", true);
  check_tensor(K, "K", true);
  check_tensor(V, "V", true);
  check_tensor(O, "O", true);
  check_tensor(dO, "dO", true);
  TORCH_CHECK(Q.dtype() == K.dtype() && Q.dtype() == V.dtype() && Q.dtype() == O.dtype() &&
                  Q.dtype() == dO.dtype(),
              "Q, K, V, O, dO must share a dtype");
  TORCH_CHECK(O.sizes() == Q.sizes() && dO.sizes() == Q.sizes(), "O and dO must have Q's shape");
  TORCH_CHECK(K.sizes() == V.sizes() && Q.size(0) == K.size(0) && Q.size(2) == K.size(2) &&
                  Q.size(3) == K.size(3),
              "K, V shapes do not match Q");
  TORCH_CHECK(lse.is_cuda() && lse.dtype() == torch::kFloat32 && lse.is_contiguous() &&
                  lse.dim() == 3 && lse.size(0) == Q.size(0) && lse.size(1) == Q.size(1) &&
                  lse.size(2) == Q.size(2),
              "lse must be a contiguous fp32 CUDA tensor [B, Hq, N]");
  const auto head_dim = Q.size(3);
  TORCH_CHECK(head_dim == 64 || head_dim == 128,
              "flash_attention_forward supports head_dim=64 or 128, got ", head_dim);
  TORCH_CHECK(K.size(1) > 0 && Q.size(1) % K.size(1) == 0, "GQA: Q heads (", Q.size(1),
              ") not divisible by K/V heads (", K.size(1), ")");
  TORCH_CHECK(Q.size(0) <= INT32_MAX && Q.size(1) <= INT32_MAX && Q.size(2) <= INT32_MAX,
              "size exceeds int32");
  const c10::cuda::CUDAGuard guard(Q.device());
  const int B = static_cast<int>(Q.size(0)), Hq = static_cast<int>(Q.size(1));
  const int N = static_cast<int>(Q.size(2));
  auto dQ = torch::empty_like(Q);
  auto dK = torch::empty_like(K);
  auto dV = torch::empty_like(V);
  const size_t ws_bytes = fa_bwd_workspace_bytes(B, Hq, N);
  auto ws = torch::empty({static_cast<int64_t>(ws_bytes > 0 ? ws_bytes : 16)},
                         Q.options().dtype(torch::kUInt8));
  const int rc = fa_bwd(Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(), dO.data_ptr(),
                        lse.data_ptr<float>(), dQ.data_ptr(), dK.data_ptr(), dV.data_ptr(), B, Hq,
                        static_cast<int>(K.size(1)), N, static_cast<int>(head_dim), scale,
                        causal ? 1 : 0, Q.dtype() == torch::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16,
                        ws.data_ptr(), ws_bytes, stream_of(Q));
  TORCH_CHECK(rc == FA_OK, "flash_attention_backward: ", fa_error_string(rc));
  return {dQ, dK, dV};
}

// Gradients of flash_attention_forward_padded (square N): (dQ, dK, dV).
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> flash_attention_backward_padded(
    torch::Tensor dO, torch::Tensor Q, torch::Tensor K, torch::Tensor V, torch::Tensor O,
    torch::Tensor lse, torch::Tensor q_start, torch::Tensor q_end, torch::Tensor k_start,
    torch::Tensor k_end, bool causal, float scale) {
  check_tensor(Q, "Q", true);
  check_tensor(K, "K", true);
  check_tensor(V, "V", true);
  check_tensor(O, "O", true);
  check_tensor(dO, "dO", true);
  TORCH_CHECK(Q.dtype() == K.dtype() && Q.dtype() == V.dtype() && Q.dtype() == O.dtype() &&
                  Q.dtype() == dO.dtype(),
              "Q, K, V, O, dO must share a dtype");
  TORCH_CHECK(O.sizes() == Q.sizes() && dO.sizes() == Q.sizes(), "O and dO must have Q's shape");
  TORCH_CHECK(K.sizes() == V.sizes() && Q.size(0) == K.size(0) && Q.size(2) == K.size(2) &&
                  Q.size(3) == K.size(3),
              "K, V shapes do not match Q (the padded backward needs Nq = Nk)");
  TORCH_CHECK(lse.is_cuda() && lse.dtype() == torch::kFloat32 && lse.is_contiguous() &&
                  lse.dim() == 3 && lse.size(0) == Q.size(0) && lse.size(1) == Q.size(1) &&
                  lse.size(2) == Q.size(2),
              "lse must be a contiguous fp32 CUDA tensor [B, Hq, N]");
  const auto head_dim = Q.size(3);
  TORCH_CHECK(head_dim == 64 || head_dim == 128,
              "flash_attention_forward supports head_dim=64 or 128, got ", head_dim);
  TORCH_CHECK(K.size(1) > 0 && Q.size(1) % K.size(1) == 0, "GQA: Q heads (", Q.size(1),
              ") not divisible by K/V heads (", K.size(1), ")");
  const int64_t B = Q.size(0);
  check_rows(q_start, "q_start", B, Q);
  check_rows(q_end, "q_end", B, Q);
  check_rows(k_start, "k_start", B, Q);
  check_rows(k_end, "k_end", B, Q);
  TORCH_CHECK(Q.size(1) <= INT32_MAX && Q.size(2) <= INT32_MAX, "size exceeds int32");
  const c10::cuda::CUDAGuard guard(Q.device());
  const int Hq = static_cast<int>(Q.size(1)), N = static_cast<int>(Q.size(2));
  auto dQ = torch::empty_like(Q);
  auto dK = torch::empty_like(K);
  auto dV = torch::empty_like(V);
  const size_t ws_bytes = fa_bwd_workspace_bytes(static_cast<int>(B), Hq, N);
  auto ws = torch::empty({static_cast<int64_t>(ws_bytes > 0 ? ws_bytes : 16)},
                         Q.options().dtype(torch::kUInt8));
  const int rc = fa_bwd_padded(
      Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(), dO.data_ptr(), lse.data_ptr<float>(),
      q_start.data_ptr<int>(), q_end.data_ptr<int>(), k_start.data_ptr<int>(), k_end.data_ptr<int>(),
      dQ.data_ptr(), dK.data_ptr(), dV.data_ptr(), static_cast<int>(B), Hq,
      static_cast<int>(K.size(1)), N, static_cast<int>(head_dim), scale, causal ? 1 : 0,
      Q.dtype() == torch::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16, ws.data_ptr(), ws_bytes,
      stream_of(Q));
  TORCH_CHECK(rc == FA_OK, "flash_attention_backward_padded: ", fa_error_string(rc));
  return {dQ, dK, dV};
}

// Gradients of flash_attention_forward_varlen for packed self-attention batches.
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> flash_attention_backward_varlen(
    torch::Tensor dO, torch::Tensor Q, torch::Tensor K, torch::Tensor V, torch::Tensor O,
    torch::Tensor lse, torch::Tensor cu_seqlens, int64_t max_seqlen, bool causal, float scale) {
  check_packed(Q, "Q");
  check_packed(K, "K");
  check_packed(V, "V");
  check_packed(O, "O");
  check_packed(dO, "dO");
  TORCH_CHECK(Q.dtype() == K.dtype() && Q.dtype() == V.dtype() && Q.dtype() == O.dtype() &&
                  Q.dtype() == dO.dtype(),
              "Q, K, V, O, dO must share a dtype");
  TORCH_CHECK(O.sizes() == Q.sizes() && dO.sizes() == Q.sizes(), "O and dO must have Q's shape");
  TORCH_CHECK(K.sizes() == V.sizes() && K.size(0) == Q.size(0) && K.size(2) == Q.size(2),
              "K, V must be [total, Hkv, d] over the same rows as Q (self-attention)");
  TORCH_CHECK(lse.is_cuda() && lse.dtype() == torch::kFloat32 && lse.is_contiguous() &&
                  lse.dim() == 2 && lse.size(0) == Q.size(1) && lse.size(1) == Q.size(0),
              "lse must be a contiguous fp32 CUDA tensor [Hq, total]");
  const auto head_dim = Q.size(2);
  TORCH_CHECK(head_dim == 64 || head_dim == 128,
              "flash_attention_forward supports head_dim=64 or 128, got ", head_dim);
  TORCH_CHECK(K.size(1) > 0 && Q.size(1) % K.size(1) == 0, "GQA: Q heads (", Q.size(1),
              ") not divisible by K/V heads (", K.size(1), ")");
  TORCH_CHECK(cu_seqlens.dim() == 1 && cu_seqlens.size(0) >= 1, "cu_seqlens must be [B + 1]");
  const int64_t B = cu_seqlens.size(0) - 1;
  check_rows(cu_seqlens, "cu_seqlens", B + 1, Q);
  TORCH_CHECK(Q.size(0) <= INT32_MAX && max_seqlen >= 0 && max_seqlen <= INT32_MAX,
              "size exceeds int32");
  const c10::cuda::CUDAGuard guard(Q.device());
  const int Hq = static_cast<int>(Q.size(1));
  auto dQ = torch::empty_like(Q);
  auto dK = torch::empty_like(K);
  auto dV = torch::empty_like(V);
  const size_t ws_bytes = fa_bwd_workspace_bytes(static_cast<int>(B), Hq, static_cast<int>(max_seqlen));
  auto ws = torch::empty({static_cast<int64_t>(ws_bytes > 0 ? ws_bytes : 16)},
                         Q.options().dtype(torch::kUInt8));
  const int rc = fa_bwd_varlen(
      Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(), dO.data_ptr(), lse.data_ptr<float>(),
      cu_seqlens.data_ptr<int>(), dQ.data_ptr(), dK.data_ptr(), dV.data_ptr(), static_cast<int>(B),
      Hq, static_cast<int>(K.size(1)), static_cast<int>(Q.size(0)), static_cast<int>(max_seqlen),
      static_cast<int>(head_dim), scale, causal ? 1 : 0,
      Q.dtype() == torch::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16, ws.data_ptr(), ws_bytes,
      stream_of(Q));
  TORCH_CHECK(rc == FA_OK, "flash_attention_backward_varlen: ", fa_error_string(rc));
  return {dQ, dK, dV};
}

// ---- paged KV cache

// Stride of a dimension, 0 where it has one entry and the stride is free.
int64_t stride_of(const torch::Tensor& t, int64_t dim) {
  return t.size(dim) > 1 ? t.stride(dim) : 0;
}

// The C description of a paged cache: pages [num_pages, Hkv, page_size, d] of
// any strides with d contiguous, block_table int32 [B, max_pages], scales fp32
// [num_pages, Hkv, page_size] for 8-bit pages.  `like` (new tokens or results)
// fixes the device and, for 16-bit pages, the type.
// (The keys alone: v = k, vs = ks.)
fa_paged_cache paged_cache(const torch::Tensor& k, const torch::Tensor& v,
                           const torch::Tensor& table, const c10::optional<torch::Tensor>& ks,
                           const c10::optional<torch::Tensor>& vs, const torch::Device& device,
                           torch::ScalarType dtype, bool writes = false) {
  TORCH_CHECK(k.is_cuda() && k.device() == device && v.device() == device,
              "k_cache and v_cache must be on the inputs' CUDA device");
  TORCH_CHECK_VALUE(k.dim() == 4 && v.dim() == 4,
                    "k_cache and v_cache must be 4D [num_pages, H_kv, page_size, D]");
  TORCH_CHECK(k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(),
              "k_cache and v_cache must share shape and dtype");
  TORCH_CHECK(k.size(3) == 64 || k.size(3) == 128,
              "flash_attention_sm75 supports head_dim=64 or 128, got ", k.size(3));
  fa_paged_cache c{};
  const auto kind = k.scalar_type();
  const bool eight = kind == torch::kInt8 || kind == torch::kFloat8_e4m3fn;
  TORCH_CHECK(eight || kind == dtype, "the pages must be int8, float8_e4m3fn or ", dtype,
              " like the rows, got ", kind);
  c.dtype = kind == torch::kInt8            ? FA_DTYPE_INT8
            : kind == torch::kFloat8_e4m3fn ? FA_DTYPE_E4M3
            : kind == torch::kBFloat16      ? FA_DTYPE_BF16
                                            : FA_DTYPE_F16;
  TORCH_CHECK(k.size(2) > 0 && k.size(2) % 16 == 0, "page_size must be a multiple of 16, got ",
              k.size(2));
  TORCH_CHECK(k.stride(3) == 1 && v.stride(3) == 1, "the pages' rows must be contiguous");
  for (int64_t i = 0; i < 3; ++i) {
    const int64_t st = stride_of(k, i);
    TORCH_CHECK(st == stride_of(v, i), "k_cache and v_cache must have the same strides");
    TORCH_CHECK(st * static_cast<int64_t>(k.element_size()) % 16 == 0,
                "the pages' strides must be multiples of 16 bytes");
    TORCH_CHECK(k.size(i) <= 1 || st > 0 || (i < 2 && !writes),
                writes ? "pages that are written cannot be broadcast tensors"
                       : "the rows of a page cannot be a broadcast dimension");
  }
  TORCH_CHECK(k.size(0) <= INT32_MAX && k.size(1) <= INT32_MAX && k.size(2) <= INT32_MAX,
              "size exceeds int32");
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.page_stride = stride_of(k, 0);
  c.head_stride = stride_of(k, 1);
  c.row_stride = stride_of(k, 2);
  TORCH_CHECK(eight == (ks.has_value() && vs.has_value()) && eight == (ks.has_value() || vs.has_value()),
              "8-bit pages need k_scale and v_scale, 16-bit pages take none");
  if (eight) {
    for (const auto* t : {&*ks, &*vs}) {
      TORCH_CHECK(t->device() == device && t->scalar_type() == torch::kFloat32 && t->dim() == 3 &&
                      t->size(0) == k.size(0) && t->size(1) == k.size(1) && t->size(2) == k.size(2),
                  "k_scale and v_scale must be fp32 [num_pages, Hkv, page_size] on the pages' device");
      for (int64_t i = 0; i < 3; ++i)
        TORCH_CHECK(stride_of(*t, i) == stride_of(*ks, i),
                    "k_scale and v_scale must have the same strides");
      for (int64_t i = 0; writes && i < 3; ++i)
        TORCH_CHECK(t->size(i) <= 1 || t->stride(i) > 0, "scales that are written cannot be broadcast tensors");
    }
    c.k_scale = ks->data_ptr<float>();
    c.v_scale = vs->data_ptr<float>();
    c.scale_page_stride = stride_of(*ks, 0);
    c.scale_head_stride = stride_of(*ks, 1);
    c.scale_row_stride = stride_of(*ks, 2);
  }
  TORCH_CHECK(table.device() == device && table.scalar_type() == torch::kInt32 &&
                  table.dim() == 2 && (table.size(1) <= 1 || table.stride(1) == 1),
              "block_table must be int32 [B, max_pages] with contiguous rows on the pages' device");
  TORCH_CHECK(table.size(0) <= INT32_MAX && table.size(1) <= INT32_MAX, "size exceeds int32");
  // (an empty table has no data: any valid pointer serves)
  c.block_table = table.numel() > 0 ? table.data_ptr<int>() : static_cast<const int*>(k.data_ptr());
  c.table_stride = stride_of(table, 0);
  c.max_pages = static_cast<int>(table.size(1));
  c.num_pages = static_cast<int>(k.size(0));
  c.kv_heads = static_cast<int>(k.size(1));
  c.page_size = static_cast<int>(k.size(2));
  c.head_dim = static_cast<int>(k.size(3));
  return c;
}

// int32 tensor with contiguous rows on `device` from a tensor (itself where it
// is one) or a sequence of ints.  `counts`: numbers that int32 does not hold become
// the largest or the least that it does (else they wrap).
torch::Tensor as_ints(pybind11::handle h, const torch::Device& device, bool counts = false) {
  torch::Tensor x;
  if (THPVariable_Check(h.ptr())) {
    x = THPVariable_Unpack(h.ptr());
  } else {
    x = pybind11::module_::import("torch").attr("as_tensor")(h).cast<torch::Tensor>();
  }
  if (counts && x.scalar_type() == torch::kInt64) x = x.clamp(INT32_MIN, INT32_MAX);
  const bool rows = x.dim() == 0 || x.size(-1) <= 1 || x.stride(-1) == 1;
  if (x.scalar_type() == torch::kInt32 && x.device() == device && rows) return x;
  return x.to(torch::TensorOptions().dtype(torch::kInt32).device(device)).contiguous();
}

// Number of sequences; checks cu_seqlens [B + 1] and seqlens_k [B] against the table.
int paged_batch(const torch::Tensor& cu, const torch::Tensor& lens, const torch::Tensor& table,
                const torch::Device& device,
                const char* agree = "block_table [B, max_pages], seqlens_k [B] and cu_seqlens [B + 1] must agree, "
                                    "got B = ") {
  TORCH_CHECK(cu.device() == device && lens.device() == device,
              "cu_seqlens and seqlens_k must be on the inputs' device");
  TORCH_CHECK(cu.scalar_type() == torch::kInt32 && lens.scalar_type() == torch::kInt32 &&
                  cu.is_contiguous() && lens.is_contiguous() && cu.dim() == 1 && lens.dim() == 1,
              "cu_seqlens and seqlens_k must be contiguous 1-D int32 tensors");
  TORCH_CHECK(lens.size(0) == table.size(0) && cu.size(0) == table.size(0) + 1,
              agree, table.size(0), ", ", lens.size(0), ", ", cu.size(0) - 1);
  return static_cast<int>(table.size(0));
}

// New rows [total, H, D], f16 / bf16, any token and head strides of 16 bytes.
void check_new_rows(const torch::Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.dim() == 3, name, " must be 3D [total, H, D]");
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == torch::kFloat16 || t.scalar_type() == torch::kBFloat16, name,
              " must be FP16 or BF16");
  TORCH_CHECK(t.size(0) <= INT32_MAX && t.size(1) <= INT32_MAX, "size exceeds int32");
}

// Uninitialised result (without the dispatcher: small calls
// are bound by host time).
torch::Tensor new_result(at::IntArrayRef sizes, torch::ScalarType dtype, const torch::Device& device) {
  return at::detail::empty_cuda(sizes, torch::TensorOptions().dtype(dtype).device(device));
}

// `t` itself if the kernels can read it in place (contiguous rows, token and
// head strides and base multiples of 16 bytes; no broadcast dimension where a
// tensor map describes it), else a contiguous copy.
torch::Tensor readable_rows(const torch::Tensor& t, bool mapped = false) {
  if (t.numel() == 0) return t;
  const bool repeats = (t.size(0) > 1 && t.stride(0) == 0) || (t.size(1) > 1 && t.stride(1) == 0);
  const bool ok = t.stride(2) == 1 && !(mapped && repeats) && stride_of(t, 0) % 8 == 0 && stride_of(t, 1) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

void kvcache_write_paged(const torch::Tensor& k_in, const torch::Tensor& v_in,
                         const torch::Tensor& k_cache, const torch::Tensor& v_cache,
                         pybind11::handle table_in, pybind11::handle cu_in,
                         pybind11::handle lens_in, const c10::optional<torch::Tensor>& ks,
                         const c10::optional<torch::Tensor>& vs) {
  check_new_rows(k_in, "k");
  check_new_rows(v_in, "v");
  const auto table = as_ints(table_in, k_in.device());
  const auto cu = as_ints(cu_in, k_in.device()), lens = as_ints(lens_in, k_in.device());
  TORCH_CHECK(k_in.sizes() == v_in.sizes() && k_in.scalar_type() == v_in.scalar_type() &&
                  k_in.device() == v_in.device(),
              "k and v must share shape, dtype and device");
  const auto c = paged_cache(k_cache, v_cache, table, ks, vs, k_in.device(), k_in.scalar_type(), /*writes=*/true);
  TORCH_CHECK(k_in.size(1) == c.kv_heads && k_in.size(2) == c.head_dim,
              "k and v must be [total, ", c.kv_heads, ", ", c.head_dim, "] for these pages");
  const int B = paged_batch(cu, lens, table, k_in.device());
  if (k_in.numel() == 0) return;
  const c10::cuda::CUDAGuard guard(k_in.device());
  const auto k = readable_rows(k_in), v = readable_rows(v_in);
  const int rc = fa_kvcache_write(
      &c, k.data_ptr(), v.data_ptr(), stride_of(k, 0), stride_of(k, 1), stride_of(v, 0),
      stride_of(v, 1), cu.data_ptr<int>(), lens.data_ptr<int>(), B, static_cast<int>(k.size(0)),
      k.scalar_type() == torch::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16, stream_of(k));
  TORCH_CHECK(rc == FA_OK, "kvcache_write_paged: ", fa_error_string(rc));
}

std::tuple<torch::Tensor, torch::Tensor> kvcache_read_paged(
    const torch::Tensor& k_cache, const torch::Tensor& v_cache, pybind11::handle table_in,
    pybind11::handle cu_in, pybind11::handle lens_in, int64_t total,
    const c10::optional<torch::Tensor>& ks, const c10::optional<torch::Tensor>& vs, bool bf16) {
  const auto table = as_ints(table_in, k_cache.device());
  const auto cu = as_ints(cu_in, k_cache.device()), lens = as_ints(lens_in, k_cache.device());
  const auto dtype = bf16 ? torch::kBFloat16 : torch::kFloat16;
  const auto c = paged_cache(k_cache, v_cache, table, ks, vs, k_cache.device(), dtype);
  TORCH_CHECK(total >= 0 && total <= INT32_MAX, "total must be a count of rows, got ", total);
  const int B = paged_batch(cu, lens, table, k_cache.device());
  const c10::cuda::CUDAGuard guard(k_cache.device());
  auto k = new_result({total, c.kv_heads, c.head_dim}, dtype, k_cache.device());
  auto v = new_result({total, c.kv_heads, c.head_dim}, dtype, k_cache.device());
  if (total == 0) return {k, v};
  const int rc = fa_kvcache_read(&c, k.data_ptr(), v.data_ptr(), cu.data_ptr<int>(),
                                 B > 0 ? lens.data_ptr<int>() : nullptr, B,
                                 static_cast<int>(total), bf16 ? FA_DTYPE_BF16 : FA_DTYPE_F16,
                                 stream_of(k_cache));
  TORCH_CHECK(rc == FA_OK, "kvcache_read_paged: ", fa_error_string(rc));
  return {k, v};
}

// O [total_q, Hq, d], or with want_lse (O, LSE fp32 [Hq, total_q]).
pybind11::object flash_attention_forward_paged(
    const torch::Tensor& q_in, const torch::Tensor& k_cache, const torch::Tensor& v_cache,
    pybind11::handle table_in, pybind11::handle cu_in, pybind11::handle lens_in,
    int64_t max_seqlen_q, int64_t max_seqlen_k, int64_t causal, c10::optional<double> scale_in,
    bool want_lse, const c10::optional<torch::Tensor>& ks, const c10::optional<torch::Tensor>& vs) {
  check_new_rows(q_in, "q");
  const auto table = as_ints(table_in, q_in.device());
  const auto cu = as_ints(cu_in, q_in.device()), lens = as_ints(lens_in, q_in.device());
  const float scale = static_cast<float>(
      scale_in.has_value() ? *scale_in : 1.0 / std::sqrt(static_cast<double>(q_in.size(2))));
  const auto c = paged_cache(k_cache, v_cache, table, ks, vs, q_in.device(), q_in.scalar_type());
  TORCH_CHECK(q_in.size(2) == c.head_dim, "head_dim mismatch");
  TORCH_CHECK(c.kv_heads > 0 && q_in.size(1) % c.kv_heads == 0, "GQA: Q heads (", q_in.size(1),
              ") not divisible by K/V heads (", c.kv_heads, ")");
  const int B = paged_batch(cu, lens, table, q_in.device());
  TORCH_CHECK(max_seqlen_q >= 0 && max_seqlen_k >= 0 && max_seqlen_q <= INT32_MAX &&
                  max_seqlen_k <= INT32_MAX,
              "max_seqlen_q and max_seqlen_k must be lengths");
  const c10::cuda::CUDAGuard guard(q_in.device());
  const auto q = readable_rows(q_in, /*mapped=*/true);
  const int Hq = static_cast<int>(q.size(1)), total = static_cast<int>(q.size(0));
  auto O = new_result(q.sizes(), q.scalar_type(), q.device());
  torch::Tensor lse;
  if (want_lse) lse = new_result({Hq, total}, torch::kFloat32, q.device());
  auto result = [&]() -> pybind11::object {
    if (!want_lse) return pybind11::cast(O);
    return pybind11::make_tuple(O, lse);
  };
  if (q.numel() == 0) return result();
  // no sequence is longer than its row of the table, whatever bound was given:
  // the plan and the workspace go by what can be
  const int mq = static_cast<int>(max_seqlen_q);
  const int mk = static_cast<int>(std::min(max_seqlen_k, static_cast<int64_t>(c.max_pages) * c.page_size));
  const size_t ws_bytes = fa_fwd_paged_workspace_bytes(&c, B, Hq, total, mq, mk);
  torch::Tensor ws;
  if (ws_bytes > 0) ws = new_result({static_cast<int64_t>(ws_bytes)}, torch::kUInt8, q.device());
  const int rc = fa_fwd_paged(&c, q.data_ptr(), stride_of(q, 0), stride_of(q, 1), O.data_ptr(),
                              want_lse ? lse.data_ptr<float>() : nullptr, cu.data_ptr<int>(),
                              B > 0 ? lens.data_ptr<int>() : nullptr, B, Hq, total, mq, mk, scale,
                              static_cast<int>(causal),
                              q.scalar_type() == torch::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16,
                              ws_bytes > 0 ? ws.data_ptr() : nullptr, ws_bytes, stream_of(q));
  TORCH_CHECK(rc == FA_OK, "flash_attention_forward_paged: ", fa_error_string(rc));
  return result();
}

// O [total_q, Hq, d], or with want_lse (O, LSE fp32 [Hq, total_q]).
pybind11::object flash_attention_forward_paged_prefix(
    const torch::Tensor& q_in, const torch::Tensor& k_cache, const torch::Tensor& v_cache,
    pybind11::handle prefix_table_in, pybind11::handle cu_prefix_in, pybind11::handle prefix_lens_in,
    pybind11::handle table_in, pybind11::handle cu_in, pybind11::handle lens_in, int64_t max_prefix_q,
    int64_t max_prefix_k, int64_t max_seqlen_q, int64_t max_seqlen_k, int64_t causal,
    c10::optional<double> scale_in, bool want_lse, const c10::optional<torch::Tensor>& ks,
    const c10::optional<torch::Tensor>& vs) {
  check_new_rows(q_in, "q");
  const auto prefix_table = as_ints(prefix_table_in, q_in.device());
  const auto cu_prefix = as_ints(cu_prefix_in, q_in.device());
  const auto prefix_lens = as_ints(prefix_lens_in, q_in.device());
  const auto table = as_ints(table_in, q_in.device());
  const auto cu = as_ints(cu_in, q_in.device()), lens = as_ints(lens_in, q_in.device());
  const float scale = static_cast<float>(
      scale_in.has_value() ? *scale_in : 1.0 / std::sqrt(static_cast<double>(q_in.size(2))));
  const auto cp = paged_cache(k_cache, v_cache, prefix_table, ks, vs, q_in.device(), q_in.scalar_type());
  const auto c = paged_cache(k_cache, v_cache, table, ks, vs, q_in.device(), q_in.scalar_type());
  TORCH_CHECK(q_in.size(2) == c.head_dim, "head_dim mismatch");
  TORCH_CHECK(c.kv_heads > 0 && q_in.size(1) % c.kv_heads == 0, "GQA: Q heads (", q_in.size(1),
              ") not divisible by K/V heads (", c.kv_heads, ")");
  const int P = paged_batch(cu_prefix, prefix_lens, prefix_table, q_in.device(), "prefix_table [P, max_pages], "
                            "prefix_lens [P] and cu_prefix_q [P + 1] must agree, got P = ");
  const int B = paged_batch(cu, lens, table, q_in.device());
  for (const int64_t x : {max_prefix_q, max_prefix_k, max_seqlen_q, max_seqlen_k})
    TORCH_CHECK(x >= 0 && x <= INT32_MAX,
                "max_prefix_q, max_prefix_k, max_seqlen_q and max_seqlen_k must be lengths");
  const c10::cuda::CUDAGuard guard(q_in.device());
  const auto q = readable_rows(q_in, /*mapped=*/true);
  const int Hq = static_cast<int>(q.size(1)), total = static_cast<int>(q.size(0));
  auto O = new_result(q.sizes(), q.scalar_type(), q.device());
  torch::Tensor lse;
  if (want_lse) lse = new_result({Hq, total}, torch::kFloat32, q.device());
  auto result = [&]() -> pybind11::object {
    if (!want_lse) return pybind11::cast(O);
    return pybind11::make_tuple(O, lse);
  };
  if (q.numel() == 0) return result();
  // bounds that are looser than the tables are cut to what these hold
  const int mpq = static_cast<int>(max_prefix_q), mq = static_cast<int>(max_seqlen_q);
  const int mpk = static_cast<int>(std::min(max_prefix_k, static_cast<int64_t>(cp.max_pages) * c.page_size));
  const int mk = static_cast<int>(std::min(max_seqlen_k, static_cast<int64_t>(c.max_pages) * c.page_size));
  const size_t ws_bytes = fa_fwd_paged_prefix_workspace_bytes(&c, P, mpq, mpk, B, Hq, total, mq, mk);
  const auto ws = new_result({static_cast<int64_t>(ws_bytes)}, torch::kUInt8, q.device());
  const int rc = fa_fwd_paged_prefix(
      &c, cp.block_table, cp.table_stride, cp.max_pages, P, cu_prefix.data_ptr<int>(),
      P > 0 ? prefix_lens.data_ptr<int>() : nullptr, mpq, mpk, q.data_ptr(), stride_of(q, 0), stride_of(q, 1),
      O.data_ptr(), want_lse ? lse.data_ptr<float>() : nullptr, cu.data_ptr<int>(),
      B > 0 ? lens.data_ptr<int>() : nullptr, B, Hq, total, mq, mk, scale, static_cast<int>(causal),
      q.scalar_type() == torch::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16, ws.data_ptr(), ws_bytes, stream_of(q));
  TORCH_CHECK(rc == FA_OK, "flash_attention_forward_paged_prefix: ", fa_error_string(rc));
  return result();
}

// Summed weights [B, Hkv, L] fp32 whose rows do not overlap, for B sequences and the cache's heads.
void check_weights(const torch::Tensor& w, int B, const fa_paged_cache& c, const torch::Device& device) {
  TORCH_CHECK(w.device() == device && w.scalar_type() == torch::kFloat32,
              "weights must be fp32 on the pages' device");
  TORCH_CHECK_VALUE(w.dim() == 3 && w.size(0) == B && w.size(1) == c.kv_heads, "weights must be [", B, ", ",
                    c.kv_heads, ", L] for this cache");
  TORCH_CHECK(w.size(2) <= INT32_MAX, "size exceeds int32");
  // (all heads of a sequence before the next sequence, or all sequences of a head before the next head)
  const int64_t last_seq = std::max<int64_t>(w.size(0) - 1, 0) * w.stride(0);
  const int64_t last_head = std::max<int64_t>(w.size(1) - 1, 0) * w.stride(1);
  TORCH_CHECK((w.size(2) <= 1 || w.stride(2) == 1) && (w.size(0) <= 1 || w.stride(0) >= w.size(2)) &&
                  (w.size(1) <= 1 || w.stride(1) >= w.size(2)) &&
                  (w.size(0) <= 1 || w.size(1) <= 1 || w.stride(0) >= last_head + w.size(2) ||
                   w.stride(1) >= last_seq + w.size(2)),
              "the rows of weights must be contiguous and must not overlap");
}

void kvcache_weights_paged(const torch::Tensor& q_in, const torch::Tensor& lse_in, const torch::Tensor& k_cache,
                           pybind11::handle table_in, pybind11::handle cu_in, pybind11::handle lens_in,
                           int64_t max_seqlen_q, int64_t max_seqlen_k, const torch::Tensor& weights, int64_t causal,
                           c10::optional<double> scale_in, int64_t mode, const c10::optional<torch::Tensor>& ks) {
  check_new_rows(q_in, "q");
  const auto table = as_ints(table_in, q_in.device());
  const auto cu = as_ints(cu_in, q_in.device()), lens = as_ints(lens_in, q_in.device());
  const float scale = static_cast<float>(
      scale_in.has_value() ? *scale_in : 1.0 / std::sqrt(static_cast<double>(q_in.size(2))));
  auto c = paged_cache(k_cache, k_cache, table, ks, ks, q_in.device(), q_in.scalar_type());
  c.v = nullptr;
  c.v_scale = nullptr;
  TORCH_CHECK(q_in.size(2) == c.head_dim, "head_dim mismatch");
  TORCH_CHECK(c.kv_heads > 0 && q_in.size(1) > 0 && q_in.size(1) % c.kv_heads == 0, "GQA: Q heads (",
              q_in.size(1), ") not divisible by K/V heads (", c.kv_heads, ")");
  TORCH_CHECK(lse_in.device() == q_in.device() && lse_in.scalar_type() == torch::kFloat32 && lse_in.dim() == 2 &&
                  lse_in.size(0) == q_in.size(1) && lse_in.size(1) == q_in.size(0),
              "lse must be fp32 [H_q, total_q] on q's device");
  const int B = paged_batch(cu, lens, table, q_in.device());
  check_weights(weights, B, c, q_in.device());
  TORCH_CHECK(max_seqlen_q >= 0 && max_seqlen_k >= 0 && max_seqlen_q <= INT32_MAX &&
                  max_seqlen_k <= INT32_MAX,
              "max_seqlen_q and max_seqlen_k must be lengths");
  const int mk = static_cast<int>(std::min(max_seqlen_k, static_cast<int64_t>(c.max_pages) * c.page_size));
  TORCH_CHECK_VALUE(weights.size(2) >= mk, "weights has ", weights.size(2), " positions, fewer than the ", mk,
                    " that max_seqlen_k and the table allow");
  if (B == 0 || mk == 0) return;
  const c10::cuda::CUDAGuard guard(q_in.device());
  const auto q = readable_rows(q_in, /*mapped=*/true);
  const auto lse = lse_in.contiguous();
  const int rc = fa_kvcache_weights(
      &c, q.data_ptr(), stride_of(q, 0), stride_of(q, 1), lse.data_ptr<float>(), cu.data_ptr<int>(),
      lens.data_ptr<int>(), B, static_cast<int>(q.size(1)), static_cast<int>(q.size(0)),
      static_cast<int>(max_seqlen_q), mk, weights.data_ptr<float>(), stride_of(weights, 0), stride_of(weights, 1),
      static_cast<int>(weights.size(2)), static_cast<int>(mode), scale, static_cast<int>(causal),
      q.scalar_type() == torch::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16, stream_of(q));
  TORCH_CHECK(rc == FA_OK, "kvcache_weights_paged: ", fa_error_string(rc));
}

// New lengths int32 [B].  keep: an int, or B of them.
torch::Tensor kvcache_evict_paged(const torch::Tensor& k_cache, const torch::Tensor& v_cache,
                                  const torch::Tensor& weights, pybind11::handle table_in, pybind11::handle lens_in,
                                  pybind11::handle keep_in, int64_t recent, int64_t first,
                                  const c10::optional<torch::Tensor>& ks, const c10::optional<torch::Tensor>& vs) {
  const auto device = k_cache.device();
  const auto table = as_ints(table_in, device), lens = as_ints(lens_in, device);
  const auto kind = k_cache.scalar_type() == torch::kBFloat16 ? torch::kBFloat16 : torch::kFloat16;
  const auto c = paged_cache(k_cache, v_cache, table, ks, vs, device, kind, /*writes=*/true);
  TORCH_CHECK(lens.device() == device && lens.is_contiguous() && lens.dim() == 1 && lens.size(0) == table.size(0),
              "seqlens_k must be [B] for block_table [B, max_pages], got B = ", table.size(0));
  const int B = static_cast<int>(table.size(0));
  check_weights(weights, B, c, device);
  const int64_t held = static_cast<int64_t>(c.max_pages) * c.page_size;
  TORCH_CHECK_VALUE(weights.size(2) >= held, "weights has ", weights.size(2), " positions, fewer than the ", held,
                    " of the table");
  torch::Tensor keep;
  int64_t keep_all = 0;
  if (pybind11::isinstance<pybind11::int_>(keep_in)) {
    keep_all = keep_in.cast<int64_t>();
  } else {
    keep = as_ints(keep_in, device, /*counts=*/true);
    if (keep.dim() == 0) keep = keep.expand({B}).contiguous();
    TORCH_CHECK(keep.is_contiguous() && keep.dim() == 1 && keep.size(0) == B,
                "keep must be one number of positions, or one for each sequence");
  }
  TORCH_CHECK_VALUE(keep_all >= 0 && first >= 0 && recent >= 0, "keep, first and recent must not be negative");
  const auto most = [](int64_t x) { return static_cast<int>(std::min<int64_t>(x, INT32_MAX)); };
  const c10::cuda::CUDAGuard guard(device);
  auto new_lens = new_result({B}, torch::kInt32, device);
  if (B == 0) return new_lens;
  const int rc = fa_kvcache_evict(
      &c, weights.data_ptr<float>(), stride_of(weights, 0), stride_of(weights, 1),
      static_cast<int>(weights.size(2)), lens.data_ptr<int>(), keep.defined() ? keep.data_ptr<int>() : nullptr,
      most(keep_all), most(first), most(recent), new_lens.data_ptr<int>(), B, stream_of(k_cache));
  TORCH_CHECK(rc == FA_OK, "kvcache_evict_paged: ", fa_error_string(rc));
  return new_lens;
}

int device_status(bool reset) { return fa_device_status(reset ? 1 : 0); }

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("naive_attention_forward", &naive_attention_forward);
  m.def("flash_attention_forward", &flash_attention_forward);
  m.def("flash_attention_forward_scalar", &flash_attention_forward_scalar);
  m.def("flash_attention_forward_wmma_qk", &flash_attention_forward_wmma_qk);
  m.def("flash_attention_forward_lse", &flash_attention_forward_lse,
        "Returns (O, LSE) with LSE fp32 [B, Hq, N]");
  m.def("flash_attention_forward_out", &flash_attention_forward_out, pybind11::arg("Q"),
        pybind11::arg("K"), pybind11::arg("V"), pybind11::arg("O"), pybind11::arg("lse"),
        pybind11::arg("causal"), pybind11::arg("scale"));
  m.def("flash_attention_backward", &flash_attention_backward,
        "(dQ, dK, dV) from dO, Q, K, V, O, LSE (fp32 [B, Hq, N]), causal, scale");
  m.def("flash_attention_forward_kvcache", &flash_attention_forward_kvcache,
        "O, LSE of Nq queries against Nk cached keys; causal: 0 none, 1 bottom-right, 2 top-left");
  m.def("flash_attention_forward_varlen", &flash_attention_forward_varlen,
        "(O [total_q, Hq, d], LSE [Hq, total_q]) of a packed variable-length batch");
  m.def("flash_attention_forward_padded", &flash_attention_forward_padded,
        "(O, LSE) of a padded batch with per-entry valid query / key row ranges");
  m.def("flash_attention_backward_padded", &flash_attention_backward_padded,
        "(dQ, dK, dV) of flash_attention_forward_padded for square padded batches");
  m.def("flash_attention_backward_varlen", &flash_attention_backward_varlen,
        "(dQ, dK, dV) of flash_attention_forward_varlen for packed self-attention batches");
  m.def("kvcache_write_paged", &kvcache_write_paged,
        "Stores K, V rows of new tokens in the pages (quantised for 8-bit pages)");
  m.def("kvcache_read_paged", &kvcache_read_paged,
        "(K, V) packed 16-bit rows of the described tokens");
  m.def("flash_attention_forward_paged", &flash_attention_forward_paged,
        "O [total_q, Hq, d], or (O, LSE [Hq, total_q]), of new tokens over a paged cache");
  m.def("flash_attention_forward_paged_prefix", &flash_attention_forward_paged_prefix,
        "O [total_q, Hq, d], or (O, LSE [Hq, total_q]), of new tokens over shared prefixes and their own keys");
  m.def("kvcache_weights_paged", &kvcache_weights_paged,
        "Attention weight of the cached keys, summed over the new tokens, into weights [B, Hkv, L]");
  m.def("kvcache_evict_paged", &kvcache_evict_paged,
        "Cuts the sequences of a paged cache to a budget by their summed weights; new lengths [B]");
  m.def("device_status", &device_status, pybind11::arg("reset") = false,
        "Error code recorded by the in-kernel watchdog (0 = none)");
  m.def("set_watchdog_ns", &fa_set_watchdog_ns);
  m.def("set_debug_flags", &fa_set_debug_flags);
  m.def("smem_bytes", &fa_smem_bytes);
  m.def("version", []() { return std::string(fa_version()); });
}
