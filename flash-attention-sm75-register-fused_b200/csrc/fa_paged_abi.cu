// C entry points of the paged KV cache (include/fa_b200.h): argument checks
// and launches.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "fa_b200.h"
#include "fa_host.h"
#include "fa_paged.h"

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool is_8bit(int dtype) { return dtype == FA_DTYPE_INT8 || dtype == FA_DTYPE_E4M3; }

// Checks the cache's description and the call's 16-bit type; fills the
// device-side view.
int check_cache(const fa_paged_cache* c, int dtype, fa::PagedCache* out) {
  if (!c) return FA_ERR_INVALID_ARG;
  if (c->head_dim != 64 && c->head_dim != 128) return FA_ERR_UNSUPPORTED_HEAD_DIM;
  if (dtype != FA_DTYPE_F16 && dtype != FA_DTYPE_BF16) return FA_ERR_DTYPE;
  if (c->dtype < FA_DTYPE_F16 || c->dtype > FA_DTYPE_E4M3) return FA_ERR_DTYPE;
  if (!is_8bit(c->dtype) && c->dtype != dtype) return FA_ERR_DTYPE;
  if (c->page_size <= 0 || c->page_size % 16 != 0) return FA_ERR_PAGE_SIZE;
  if (c->num_pages < 0 || c->max_pages < 0 || c->kv_heads <= 0) return FA_ERR_INVALID_ARG;
  const bool scales = c->k_scale != nullptr && c->v_scale != nullptr;
  if (is_8bit(c->dtype) ? !scales : (c->k_scale != nullptr || c->v_scale != nullptr))
    return FA_ERR_SCALES;
  if (!c->k || !c->v || !c->block_table) return FA_ERR_INVALID_ARG;
  const int es = is_8bit(c->dtype) ? 1 : 2;
  if (!aligned16(c->k) || !aligned16(c->v) || (c->page_stride * es) % 16 != 0 ||
      (c->head_stride * es) % 16 != 0 || (c->row_stride * es) % 16 != 0 ||
      (reinterpret_cast<uintptr_t>(c->block_table) & 3u) ||
      (reinterpret_cast<uintptr_t>(c->k_scale) & 3u) || (reinterpret_cast<uintptr_t>(c->v_scale) & 3u))
    return FA_ERR_ALIGNMENT;
  // positions are int32
  if (static_cast<long long>(c->max_pages) * c->page_size > (1LL << 30) || c->kv_heads > (1 << 16))
    return FA_ERR_TOO_LARGE;
  out->k = static_cast<const uint8_t*>(c->k);
  out->v = static_cast<const uint8_t*>(c->v);
  out->ks = c->k_scale;
  out->vs = c->v_scale;
  out->page_stride = c->page_stride * es;
  out->head_stride = c->head_stride * es;
  out->row_stride = c->row_stride * es;
  out->s_page = c->scale_page_stride;
  out->s_head = c->scale_head_stride;
  out->s_row = c->scale_row_stride;
  out->table = c->block_table;
  out->table_stride = c->table_stride;
  out->max_pages = c->max_pages;
  out->num_pages = c->num_pages;
  out->heads = c->kv_heads;
  out->page_size = c->page_size;
  out->page_shift = -1;
  for (int s = 4; s < 31; ++s)
    if (c->page_size == (1 << s)) out->page_shift = s;
  return FA_OK;
}

int check_rows(const int* cu, const int* lens, int B, int total, fa::PagedRows* out) {
  if (B < 0 || total < 0) return FA_ERR_INVALID_ARG;
  if (B > (1 << 20) || total > (1 << 28)) return FA_ERR_TOO_LARGE;
  if (B > 0 && total > 0 && (!cu || !lens)) return FA_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(cu) & 3u) || (reinterpret_cast<uintptr_t>(lens) & 3u))
    return FA_ERR_ALIGNMENT;
  *out = fa::PagedRows{cu, lens, B, total};
  return FA_OK;
}

}  // namespace

extern "C" {

int fa_kvcache_write(const fa_paged_cache* cache, const void* K, const void* V,
                     long long k_token_stride, long long k_head_stride,
                     long long v_token_stride, long long v_head_stride, const int* cu_seqlens,
                     const int* seqlens_k, int B, int total, int dtype, void* stream) {
  fa::PagedCache c;
  fa::PagedRows r;
  if (int rc = check_cache(cache, dtype, &c)) return rc;
  if (int rc = check_rows(cu_seqlens, seqlens_k, B, total, &r)) return rc;
  if (B == 0 || total == 0) return FA_OK;
  if (!K || !V) return FA_ERR_INVALID_ARG;
  if (!aligned16(K) || !aligned16(V) ||
      ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7))
    return FA_ERR_ALIGNMENT;
  if (static_cast<long long>(total) * c.heads > (1LL << 34)) return FA_ERR_TOO_LARGE;
  if (int rc = fa::host_check_device()) return rc;
  const fa::PagedSource s{static_cast<const uint8_t*>(K), static_cast<const uint8_t*>(V),
                          2 * k_token_stride, 2 * k_head_stride, 2 * v_token_stride,
                          2 * v_head_stride};
  const cudaError_t e = fa::launch_cache_write(c, r, s, cache->head_dim, cache->dtype,
                                               dtype == FA_DTYPE_BF16,
                                               static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FA_OK : FA_ERR_LAUNCH;
}

int fa_kvcache_read(const fa_paged_cache* cache, void* K, void* V, const int* cu_seqlens,
                    const int* seqlens_k, int B, int total, int dtype, void* stream) {
  fa::PagedCache c;
  fa::PagedRows r;
  if (int rc = check_cache(cache, dtype, &c)) return rc;
  if (int rc = check_rows(cu_seqlens, seqlens_k, B, total, &r)) return rc;
  if (total == 0) return FA_OK;
  if (!K || !V) return FA_ERR_INVALID_ARG;
  if (!aligned16(K) || !aligned16(V)) return FA_ERR_ALIGNMENT;
  if (static_cast<long long>(total) * c.heads > (1LL << 34)) return FA_ERR_TOO_LARGE;
  if (int rc = fa::host_check_device()) return rc;
  const cudaError_t e =
      fa::launch_cache_read(c, r, K, V, cache->head_dim, cache->dtype, dtype == FA_DTYPE_BF16,
                            static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FA_OK : FA_ERR_LAUNCH;
}

size_t fa_fwd_paged_workspace_bytes(const fa_paged_cache* cache, int B, int Hq, int total_q,
                                    int max_seqlen_q, int max_seqlen_k) {
  (void)B; (void)total_q; (void)max_seqlen_k;
  const int group = cache && cache->kv_heads > 0 ? Hq / cache->kv_heads : 1;
  const long long rows = static_cast<long long>(max_seqlen_q) * group;
  if (rows <= fa::paged_decode_rows())
    return fa::paged_decode_ws_bytes(static_cast<int>(rows), cache ? cache->head_dim : 128,
                                     fa::host_sm_count());
  return 16;
}

int fa_fwd_paged(const fa_paged_cache* cache, const void* Q, long long q_token_stride,
                 long long q_head_stride, void* O, float* lse, const int* cu_seqlens_q,
                 const int* seqlens_k, int B, int Hq, int total_q, int max_seqlen_q,
                 int max_seqlen_k, float scale, int causal, int dtype, void* workspace,
                 size_t workspace_bytes, void* stream) {
  fa::PagedAttn a;
  if (int rc = check_cache(cache, dtype, &a.c)) return rc;
  if (int rc = check_rows(cu_seqlens_q, seqlens_k, B, total_q, &a.r)) return rc;
  if (Hq < 0 || max_seqlen_q < 0 || max_seqlen_k < 0) return FA_ERR_INVALID_ARG;
  if (causal < FA_CAUSAL_NONE || causal > FA_CAUSAL_TOP_LEFT) return FA_ERR_INVALID_ARG;
  if (!std::isfinite(scale)) return FA_ERR_INVALID_ARG;
  if (Hq == 0 || total_q == 0) return FA_OK;
  if (Hq % a.c.heads != 0) return FA_ERR_GQA_DIVISIBILITY;
  if (Hq / a.c.heads > 128) return FA_ERR_GROUP;
  if (!Q || !O || !workspace) return FA_ERR_INVALID_ARG;
  if (!aligned16(Q) || !aligned16(O) || !aligned16(workspace) ||
      ((q_token_stride | q_head_stride) & 7) || (reinterpret_cast<uintptr_t>(lse) & 3u))
    return FA_ERR_ALIGNMENT;
  if (workspace_bytes <
      fa_fwd_paged_workspace_bytes(cache, B, Hq, total_q, max_seqlen_q, max_seqlen_k))
    return FA_ERR_INVALID_ARG;
  if (int rc = fa::host_check_device()) return rc;
  a.q = static_cast<const uint8_t*>(Q);
  a.q_token = 2 * q_token_stride;
  a.q_head = 2 * q_head_stride;
  a.o = O;
  a.lse = lse;
  a.Hq = Hq;
  a.group = Hq / a.c.heads;
  a.max_q = max_seqlen_q;
  a.max_k = max_seqlen_k;
  a.causal = causal;
  a.scale_log2 = scale * 1.4426950408889634f;
  const long long rows = static_cast<long long>(max_seqlen_q) * a.group;
  const bool bf16 = dtype == FA_DTYPE_BF16;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      rows <= fa::paged_decode_rows() && B > 0 && rows > 0
          ? fa::launch_paged_decode(a, static_cast<int>(rows), cache->head_dim, cache->dtype, bf16,
                                    fa::host_sm_count(), workspace, st)
          : fa::launch_paged_simple(a, cache->head_dim, cache->dtype, bf16, st);
  return e == cudaSuccess ? FA_OK : FA_ERR_LAUNCH;
}

}  // extern "C"
