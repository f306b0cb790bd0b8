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

constexpr int kMaxHeads = 1 << 14, kMaxBatch = 1 << 20, kMaxRows = 1 << 28;

// Checks the cache's description and the call's 16-bit type; fills the
// device-side view.  `writes`: no two entries may share memory.
int check_cache(const fa_paged_cache* c, int dtype, bool writes, fa::PagedCache* out) {
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
  const long long least = writes ? 1 : 0;
  if (c->row_stride <= 0 || (c->num_pages > 1 && c->page_stride < least) ||
      (c->kv_heads > 1 && c->head_stride < least))
    return FA_ERR_STRIDE;
  if (writes && is_8bit(c->dtype) &&
      (c->scale_row_stride == 0 || (c->num_pages > 1 && c->scale_page_stride == 0) ||
       (c->kv_heads > 1 && c->scale_head_stride == 0)))
    return FA_ERR_STRIDE;
  // positions are int32
  if (static_cast<long long>(c->max_pages) * c->page_size > (1LL << 30) || c->kv_heads > kMaxHeads)
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
  if (B > kMaxBatch || total > kMaxRows) return FA_ERR_TOO_LARGE;
  if (B > 0 && total > 0 && (!cu || !lens)) return FA_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(cu) & 3u) || (reinterpret_cast<uintptr_t>(lens) & 3u))
    return FA_ERR_ALIGNMENT;
  *out = fa::PagedRows{cu, lens, B, total};
  return FA_OK;
}

// Which kernels a call runs and how its keys are split.
//
// Sequences of few query rows per KV head go to the decode kernel, the others
// to the chunk kernel.  The lengths are on the device, so the host goes by
// bounds: with at most paged_decode_rows() rows every sequence is short; when
// the packed rows are exactly B full-length sequences every one is long; else
// both kernels run, the decode kernel on the sequences of at most kMixedRows
// rows.  Their limit is a team of one warp: chunks of 1024 and 512 tokens with 24
// single tokens, GQA 4, 8192 keys, take 356 us with a limit of 4 rows, 363 with
// 16, 374 with 32, 516 with 64; with 24 x 4 draft tokens 426, 374, 385, 514.
constexpr int kMixedRows = 16;

struct PagedPlan {
  bool decode = false, chunk = false;
  int decode_rows = 0;  // rows per KV head the decode kernel takes at most
  int tq = 0;           // chunk kernel: tokens of a query tile
  int slots = 0;        // ... pairs of tiles there may be
  bool runs = false;    // ... equal runs, or one CTA per (pair, head)
  int n_ctas = 0;       // ... runs
  // 8-bit pages: rows of the expanded keys, KV heads expanded at a time, and
  // bytes of one head's K (or V) rows, of a scale of every row, of their maxima
  long long exp_rows = 0;
  int exp_heads = 0;
  size_t exp_row_bytes = 0, exp_scale_bytes = 0, exp_max_bytes = 0;
  size_t ws_decode = 0, ws_o = 0, ws_lse = 0, ws_cuts = 0, ws_bytes = 0;
};

// Expanded keys and values are at most this large where several KV heads would
// make them larger: the heads then go through the chunk kernel in groups.
constexpr size_t kExpandBytes = size_t{1} << 30;

PagedPlan make_paged_plan(int B, int heads, int group, int head_dim, int dtype, int total, int max_q,
                          int max_k) {
  const bool eight = is_8bit(dtype);
  if (max_q > total) max_q = total;  // (a bound that is looser than it can be)
  PagedPlan k;
  const int sms = fa::host_sm_count();
  const long long rows = static_cast<long long>(max_q) * group;
  const long long all_heads = static_cast<long long>(B) * heads;
  const int cap = fa::paged_decode_rows(all_heads, head_dim, dtype, sms);
  k.chunk = rows > cap || B == 0 || max_q == 0;
  k.decode = !k.chunk || (rows > cap && B > 1 && group <= kMixedRows &&
                          total < static_cast<long long>(B) * max_q);
  k.decode_rows = k.chunk ? (kMixedRows / group) * group : static_cast<int>(rows);
  if (k.decode) k.ws_decode = fa::paged_decode_ws_bytes(all_heads, k.decode_rows, max_k, head_dim, dtype, sms);
  if (k.chunk) {
    k.tq = 128 / group;
    const int pair = 2 * k.tq;
    // sequences of the chunk kernel bring at least this many tokens
    const int least = k.decode ? k.decode_rows / group + 1 : 1;
    const long long n_seq = total / least < B ? total / least : B;
    const long long slots = total / pair + n_seq;
    k.slots = slots < 1 ? 1 : static_cast<int>(slots);
    k.exp_heads = heads;
    if (eight) {
      k.exp_rows = (n_seq < 1 ? 1 : n_seq) * ((static_cast<long long>(max_k) + 127) / 128 * 128);
      if (k.exp_rows < 128) k.exp_rows = 128;
      k.exp_row_bytes = static_cast<size_t>(k.exp_rows) * head_dim * 2;
      k.exp_scale_bytes = static_cast<size_t>(k.exp_rows) * sizeof(float);
      k.exp_max_bytes = static_cast<size_t>(k.exp_rows / 16) * sizeof(float);
      const size_t per_head = 2 * k.exp_row_bytes + 3 * k.exp_scale_bytes + k.exp_max_bytes;
      const size_t fit = kExpandBytes / per_head;
      if (fit < static_cast<size_t>(heads)) k.exp_heads = fit < 1 ? 1 : static_cast<int>(fit);
    }
    // A CTA per (pair, head), or equal runs of all of them: estimated in key
    // tiles of an SM, from bounds.  An item costs its tiles (from `least_t` to `tiles`
    // of a causal chunk's pairs, longest first) and 5 for its start, 3 in a run,
    // where the next item's tiles are loaded meanwhile; runs cost another 12 (parts
    // written and joined).  With all SMs at work a tile takes 15/14 of its time, and
    // runs another 9/8 where the keys outgrow the L2: the CTAs are at different
    // places of them.
    const long long tiles = max_k < 1 ? 1 : (static_cast<long long>(max_k) + 127) / 128;
    const long long drop = (max_q < max_k ? max_q : max_k) / 128;
    const long long least_t = tiles - drop, mean_t = tiles - drop / 2;
    const long long pairs = B <= 1 ? (total + pair - 1) / pair : total / pair + (n_seq + 1) / 2;
    const long long items = (pairs < 1 ? 1 : pairs) * k.exp_heads;
    long long by_item = tiles + 5, by_run = items * (mean_t + 3) * 15 / 14 / sms + 12;
    if (items > sms) {
      const long long in_waves = (items + sms - 1) / sms * (mean_t + 5);
      const long long in_order = items * (mean_t + 5) / sms + least_t + 5;
      by_item = (in_waves < in_order ? in_waves : in_order) * 15 / 14;
      // (in a ragged batch a sequence's keys are taken to go with its tokens)
      const long long keys = static_cast<long long>(total) * max_k / (max_q < 1 ? 1 : max_q);
      if (keys > (100 << 20) / 4 / heads / head_dim) by_run = by_run * 9 / 8;
    }
    k.runs = by_run < by_item;
    if (k.runs) {
      // no more runs than key tiles there can be, nor parts of an item than a
      // join reads in a few rounds
      const long long most = items * (tiles > 32 ? 32 : tiles);
      k.n_ctas = static_cast<int>(most < sms ? most : sms);
      if (k.n_ctas > 1) {
        const size_t rows = static_cast<size_t>(2 * k.n_ctas) * 256;
        k.ws_o = rows * head_dim * sizeof(float);
        k.ws_lse = rows * sizeof(float);
        k.ws_cuts = (k.n_ctas * sizeof(fa::PagedCut) + 127) / 128 * 128;
      }
    }
  }
  const size_t chunk_bytes =
      k.ws_o + k.ws_lse + k.ws_cuts +
      static_cast<size_t>(k.exp_heads) * (2 * k.exp_row_bytes + 3 * k.exp_scale_bytes + k.exp_max_bytes);
  // (the kernels run one after another, so they share the workspace)
  k.ws_bytes = k.ws_decode > chunk_bytes ? k.ws_decode : chunk_bytes;
  return k;
}

int gcd_128(int x) {  // of x (a multiple of 16) and 128
  int g = 16;
  while (g < 128 && x % (2 * g) == 0) g *= 2;
  return g;
}

// Tensor maps of the pages for the decode kernel, for boxes of `rows` rows (and
// 64 columns, or a whole 8-bit row).  Heads or pages with a stride of 0 become
// one entry, and the kernel's coordinate stays at 0; the stride of a dimension
// with one entry is free: any valid one serves.
bool page_maps(const fa_paged_cache& c, int rows, fa::DecodeParams* p) {
  const int es = is_8bit(c.dtype) ? 1 : 2;
  const unsigned long long row = static_cast<unsigned long long>(es) * c.head_dim;
  p->page_step = c.num_pages > 1 && c.page_stride > 0 ? 1 : 0;
  p->head_step = c.kv_heads > 1 && c.head_stride > 0 ? 1 : 0;
  fa::TiledMap t{};
  t.type = es == 1 ? fa::TiledMap::kBytes : c.dtype == FA_DTYPE_BF16 ? fa::TiledMap::kBf16 : fa::TiledMap::kF16;
  t.rank = 4;
  t.dims[0] = c.head_dim;
  t.dims[1] = c.page_size;
  t.dims[2] = p->head_step ? c.kv_heads : 1;
  t.dims[3] = p->page_step ? c.num_pages : 1;
  t.strides[0] = static_cast<unsigned long long>(es) * c.row_stride;
  t.strides[1] = p->head_step ? static_cast<unsigned long long>(es) * c.head_stride : row;
  t.strides[2] = p->page_step ? static_cast<unsigned long long>(es) * c.page_stride : row;
  t.box[0] = es == 1 ? c.head_dim : 64;
  t.box[1] = rows;
  t.box[2] = t.box[3] = 1;
  t.base = c.k;
  if (!fa::host_tensor_map(&p->tm_k, t)) return false;
  t.base = c.v;
  return fa::host_tensor_map(&p->tm_v, t);
}

// Tensor map of 128-byte column halves by groups of 8 rows (see ChunkParams):
// `planes` planes of `rows` rows, `plane` and `row` bytes apart.
bool tile_map(const void* base, int type, int head_dim, long long rows, unsigned long long row,
              long long planes, unsigned long long plane, int box_rows, CUtensorMap* map) {
  fa::TiledMap t{};
  t.type = type;
  t.base = base;
  t.rank = 5;
  t.dims[0] = 64;
  t.dims[1] = 8;
  t.dims[2] = head_dim / 64;
  t.dims[3] = rows / 8;
  t.dims[4] = planes;
  t.strides[0] = row;
  t.strides[1] = 128;
  t.strides[2] = 8 * row;
  t.strides[3] = plane;
  t.box[0] = 64;
  t.box[1] = 8;
  t.box[2] = head_dim / 64;
  t.box[3] = box_rows / 8;
  t.box[4] = 1;
  return fa::host_tensor_map(map, t);
}

// Maps of 16-bit pages for the chunk kernel.  Heads and pages share the last
// dimension, whose stride is the greatest common divisor of theirs (the head
// stride itself in head-major and token-major pages).
bool chunk_maps(const fa_paged_cache& c, fa::ChunkParams* p) {
  const unsigned long long row = 2ull * c.head_dim;
  const unsigned long long rs = 2ull * c.row_stride;
  const unsigned long long hs = c.kv_heads > 1 ? 2ull * c.head_stride : 0;
  const unsigned long long ps = c.num_pages > 1 ? 2ull * c.page_stride : 0;
  unsigned long long g = hs, x = ps;
  while (x != 0) {
    const unsigned long long r = g % x;
    g = x;
    x = r;
  }
  if (g == 0) g = row;  // one head of one page, or all of them the same
  const unsigned long long planes = (c.num_pages > 1 ? (c.num_pages - 1ull) * (ps / g) : 0ull) +
                                    (c.kv_heads - 1ull) * (hs / g) + 1ull;
  if (planes > 0x7fffffffull || ps / g > 0x7fffffffull || hs / g > 0x7fffffffull) return false;
  p->page_step = static_cast<int>(ps / g);
  p->head_step = static_cast<int>(hs / g);
  const int type = c.dtype == FA_DTYPE_BF16 ? fa::TiledMap::kBf16 : fa::TiledMap::kF16;
  return tile_map(c.k, type, c.head_dim, c.page_size, rs, planes, g, p->box_rows, &p->tm_k) &&
         tile_map(c.v, type, c.head_dim, c.page_size, rs, planes, g, p->box_rows, &p->tm_v);
}

// Maps of the expanded rows of 8-bit pages (a copy is the same for f16 and bf16).
bool rows_maps(fa::ChunkParams& p, int head_dim, int heads) {
  const unsigned long long row = 2ull * head_dim;
  const int type = fa::TiledMap::kF16;
  return tile_map(p.exp_k, type, head_dim, p.exp_rows, row, heads, row * p.exp_rows, 128, &p.tm_k) &&
         tile_map(p.exp_v, type, head_dim, p.exp_rows, row, heads, row * p.exp_rows, 128, &p.tm_v);
}

// Tensor map of the queries: boxes of a query tile, `tq` tokens x the heads of
// a group.
bool query_map(const fa_paged_cache& c, int tq, const void* q, long long q_token, long long q_head,
               int Hq, int total, bool bf16, CUtensorMap* map) {
  const unsigned long long row = 2ull * c.head_dim;
  fa::TiledMap t{};
  t.type = bf16 ? fa::TiledMap::kBf16 : fa::TiledMap::kF16;
  t.base = q;
  t.rank = 3;
  t.dims[0] = c.head_dim;
  t.dims[1] = Hq;
  t.dims[2] = total;
  t.strides[0] = Hq > 1 ? 2ull * q_head : row;  // (free where there is one)
  t.strides[1] = total > 1 ? 2ull * q_token : row;
  t.box[0] = 64;
  t.box[1] = Hq / c.kv_heads;
  t.box[2] = tq;
  return fa::host_tensor_map(map, t);
}

}  // namespace

extern "C" {

int fa_kvcache_write(const fa_paged_cache* cache, const void* K, const void* V,
                     long long k_token_stride, long long k_head_stride,
                     long long v_token_stride, long long v_head_stride, const int* cu_seqlens,
                     const int* seqlens_k, int B, int total, int dtype, void* stream) {
  fa::PagedCache c;
  fa::PagedRows r;
  if (int rc = check_cache(cache, dtype, true, &c)) return rc;
  if (int rc = check_rows(cu_seqlens, seqlens_k, B, total, &r)) return rc;
  if (B == 0 || total == 0) return FA_OK;
  if (!K || !V) return FA_ERR_INVALID_ARG;
  if (!aligned16(K) || !aligned16(V) ||
      ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7))
    return FA_ERR_ALIGNMENT;
  // (rows are numbered with 32 bits, in tiles of 16 tokens)
  if ((static_cast<long long>(total) + 15) * 2 * c.heads > 0xffff0000LL) return FA_ERR_TOO_LARGE;
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
  if (int rc = check_cache(cache, dtype, false, &c)) return rc;
  if (int rc = check_rows(cu_seqlens, seqlens_k, B, total, &r)) return rc;
  if (total == 0) return FA_OK;
  if (!K || !V) return FA_ERR_INVALID_ARG;
  if (!aligned16(K) || !aligned16(V)) return FA_ERR_ALIGNMENT;
  // (rows are numbered with 32 bits, in tiles of 16 tokens)
  if ((static_cast<long long>(total) + 15) * 2 * c.heads > 0xffff0000LL) return FA_ERR_TOO_LARGE;
  if (int rc = fa::host_check_device()) return rc;
  const cudaError_t e =
      fa::launch_cache_read(c, r, K, V, cache->head_dim, cache->dtype, dtype == FA_DTYPE_BF16,
                            static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FA_OK : FA_ERR_LAUNCH;
}

size_t fa_fwd_paged_workspace_bytes(const fa_paged_cache* cache, int B, int Hq, int total_q,
                                    int max_seqlen_q, int max_seqlen_k) {
  if (!cache || cache->kv_heads <= 0 || Hq <= 0 || total_q <= 0) return 0;
  const int group = Hq / cache->kv_heads;
  // what the call refuses
  if (group * cache->kv_heads != Hq || group > 128 || B < 0 || max_seqlen_q < 0 || max_seqlen_k < 0 ||
      (cache->head_dim != 64 && cache->head_dim != 128) || cache->dtype < FA_DTYPE_F16 ||
      cache->dtype > FA_DTYPE_E4M3 || cache->kv_heads > kMaxHeads || B > kMaxBatch || total_q > kMaxRows)
    return 0;
  return make_paged_plan(B, cache->kv_heads, group, cache->head_dim, cache->dtype, total_q,
                         max_seqlen_q, max_seqlen_k)
      .ws_bytes;
}

int fa_fwd_paged(const fa_paged_cache* cache, const void* Q, long long q_token_stride,
                 long long q_head_stride, void* O, float* lse, const int* cu_seqlens_q,
                 const int* seqlens_k, int B, int Hq, int total_q, int max_seqlen_q,
                 int max_seqlen_k, float scale, int causal, int dtype, void* workspace,
                 size_t workspace_bytes, void* stream) {
  fa::PagedAttn a;
  if (int rc = check_cache(cache, dtype, false, &a.c)) return rc;
  if (int rc = check_rows(cu_seqlens_q, seqlens_k, B, total_q, &a.r)) return rc;
  if (Hq < 0 || max_seqlen_q < 0 || max_seqlen_k < 0) return FA_ERR_INVALID_ARG;
  if (causal < FA_CAUSAL_NONE || causal > FA_CAUSAL_TOP_LEFT) return FA_ERR_INVALID_ARG;
  if (!std::isfinite(scale)) return FA_ERR_INVALID_ARG;
  if (Hq == 0 || total_q == 0) return FA_OK;
  if (Hq % a.c.heads != 0) return FA_ERR_GQA_DIVISIBILITY;
  if (Hq / a.c.heads > 128) return FA_ERR_GROUP;
  if (!Q || !O) return FA_ERR_INVALID_ARG;
  if (!aligned16(Q) || !aligned16(O) || !aligned16(workspace) ||
      ((q_token_stride | q_head_stride) & 7) || (reinterpret_cast<uintptr_t>(lse) & 3u))
    return FA_ERR_ALIGNMENT;
  if ((total_q > 1 && q_token_stride <= 0) || (Hq > 1 && q_head_stride <= 0)) return FA_ERR_STRIDE;
  const int group = Hq / a.c.heads;
  const bool eight = is_8bit(cache->dtype);
  const PagedPlan k = make_paged_plan(B, a.c.heads, group, cache->head_dim, cache->dtype, total_q, max_seqlen_q,
                                      max_seqlen_k);
  if (k.ws_bytes > 0 && (!workspace || workspace_bytes < k.ws_bytes)) return FA_ERR_INVALID_ARG;
  const long long grid = static_cast<long long>(k.slots) * a.c.heads;  // of all heads
  if (grid > 0x7fffffffLL || static_cast<long long>(B) * a.c.heads > 0x7fffffffLL ||
      static_cast<long long>(total_q) * Hq > (1LL << 33))
    return FA_ERR_TOO_LARGE;
  if (int rc = fa::host_check_device()) return rc;
  a.q = static_cast<const uint8_t*>(Q);
  a.q_token = 2 * q_token_stride;
  a.q_head = 2 * q_head_stride;
  a.o = O;
  a.lse = lse;
  a.Hq = Hq;
  a.group = group;
  a.max_q = max_seqlen_q;
  a.max_k = max_seqlen_k;
  a.causal = causal;
  a.scale_log2 = scale * 1.4426950408889634f;
  const bool bf16 = dtype == FA_DTYPE_BF16;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (k.decode) {
    fa::DecodeParams p;
    p.a = a;
    p.ws = static_cast<float*>(workspace);
    p.max_rows = k.decode_rows;
    p.epoch = fa::host_next_epoch();
    p.timeout_ns = fa::host_timeout_ns();
    if (!page_maps(*cache, 16, &p)) return FA_ERR_TENSOR_MAP;
    if (fa::launch_paged_decode(p, cache->head_dim, cache->dtype, bf16, fa::host_sm_count(), st) !=
        cudaSuccess)
      return FA_ERR_LAUNCH;
  }
  if (k.chunk) {
    fa::ChunkParams p;
    p.a = a;
    p.tq = k.tq;
    p.box_rows = eight ? 128 : gcd_128(cache->page_size);
    p.stale = eight ? 0 : 1;
    p.page_step = p.head_step = 0;
    p.skip_rows = k.decode ? k.decode_rows : 0;
    p.runs = k.runs ? 1 : 0;
    char* ws = static_cast<char*>(workspace);
    p.ws_o = reinterpret_cast<float*>(ws);
    p.ws_lse = reinterpret_cast<float*>(ws + k.ws_o);
    p.ws_cuts = reinterpret_cast<fa::PagedCut*>(ws + k.ws_o + k.ws_lse);
    ws += k.ws_o + k.ws_lse + k.ws_cuts;
    p.exp_rows = k.exp_rows;
    p.exp_k = reinterpret_cast<uint16_t*>(ws);
    p.exp_v = reinterpret_cast<uint16_t*>(ws + k.exp_heads * k.exp_row_bytes);
    ws += 2 * k.exp_heads * k.exp_row_bytes;
    p.exp_ks = reinterpret_cast<float*>(ws);
    p.exp_vs = reinterpret_cast<float*>(ws + k.exp_heads * k.exp_scale_bytes);
    p.exp_vl = reinterpret_cast<float*>(ws + 2 * k.exp_heads * k.exp_scale_bytes);
    p.exp_vm = reinterpret_cast<float*>(ws + 3 * k.exp_heads * k.exp_scale_bytes);
    p.timeout_ns = fa::host_timeout_ns();
    const bool maps =
        (eight ? rows_maps(p, cache->head_dim, k.exp_heads) : chunk_maps(*cache, &p)) &&
        query_map(*cache, p.tq, Q, q_token_stride, q_head_stride, Hq, total_q, bf16, &p.tm_q);
    if (!maps) return FA_ERR_TENSOR_MAP;
    for (p.head0 = 0; p.head0 < a.c.heads; p.head0 += k.exp_heads) {
      p.n_heads = a.c.heads - p.head0 < k.exp_heads ? a.c.heads - p.head0 : k.exp_heads;
      p.fill = !k.decode && p.head0 == 0 ? 1 : 0;
      p.epoch = fa::host_next_epoch();
      p.n_ctas = k.runs ? k.n_ctas : k.slots * p.n_heads;
      if (fa::launch_paged_chunk(p, cache->head_dim, cache->dtype, bf16, fa::host_sm_count(), st) !=
          cudaSuccess)
        return FA_ERR_LAUNCH;
    }
  }
  return FA_OK;
}

}  // extern "C"
