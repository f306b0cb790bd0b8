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
// device-side view.  `writes`: no two entries may share memory.  `values`: V and its
// scales are used too.
int check_cache(const fa_paged_cache* c, int dtype, bool writes, fa::PagedCache* out, bool values = true) {
  if (!c) return FA_ERR_INVALID_ARG;
  if (c->head_dim != 64 && c->head_dim != 128) return FA_ERR_UNSUPPORTED_HEAD_DIM;
  if (dtype != FA_DTYPE_F16 && dtype != FA_DTYPE_BF16) return FA_ERR_DTYPE;
  if (c->dtype < FA_DTYPE_F16 || c->dtype > FA_DTYPE_E4M3) return FA_ERR_DTYPE;
  if (!is_8bit(c->dtype) && c->dtype != dtype) return FA_ERR_DTYPE;
  if (c->page_size <= 0 || c->page_size % 16 != 0) return FA_ERR_PAGE_SIZE;
  if (c->num_pages < 0 || c->max_pages < 0 || c->kv_heads <= 0) return FA_ERR_INVALID_ARG;
  const bool scales = c->k_scale != nullptr && (c->v_scale != nullptr || !values);
  if (is_8bit(c->dtype) ? !scales : (c->k_scale != nullptr || c->v_scale != nullptr))
    return FA_ERR_SCALES;
  if (!c->k || (values && !c->v) || !c->block_table) return FA_ERR_INVALID_ARG;
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

// What attention calls have in common: head counts and bounds, queries, their strides.
int check_attention(int Hq, int max_q, int max_k, float scale, int causal) {
  if (Hq < 0 || max_q < 0 || max_k < 0) return FA_ERR_INVALID_ARG;
  if (causal < FA_CAUSAL_NONE || causal > FA_CAUSAL_TOP_LEFT) return FA_ERR_INVALID_ARG;
  return std::isfinite(scale) ? FA_OK : FA_ERR_INVALID_ARG;
}

// `other`: the call's result, or the other input by row, on `align` bytes.
int check_queries(const fa::PagedCache& c, int Hq, int total, const void* Q, const void* other,
                  long long q_token, long long q_head, unsigned align = 16) {
  if (Hq % c.heads != 0) return FA_ERR_GQA_DIVISIBILITY;
  if (Hq / c.heads > 128) return FA_ERR_GROUP;
  if (total > 0 && (!Q || !other)) return FA_ERR_INVALID_ARG;
  if (!aligned16(Q) || (reinterpret_cast<uintptr_t>(other) & (align - 1)) || ((q_token | q_head) & 7))
    return FA_ERR_ALIGNMENT;
  return FA_OK;
}

int check_query_strides(int Hq, int total, long long q_token, long long q_head) {
  return (total > 1 && q_token <= 0) || (Hq > 1 && q_head <= 0) ? FA_ERR_STRIDE : FA_OK;
}

// Summed weights: fp32 rows of at least `need` positions that do not overlap: all
// heads of a sequence before the next sequence, or all sequences of a head before
// the next head.
int check_sums(const float* w, long long seq, long long head, int len, int need, int B, int heads) {
  if (len < need || len < 0 || (B > 0 && len > 0 && !w)) return FA_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(w) & 3u) return FA_ERR_ALIGNMENT;
  if ((B > 1 && seq < len) || (heads > 1 && head < len)) return FA_ERR_STRIDE;
  const __int128 n = len;
  if (B > 1 && heads > 1 && len > 0 && seq < (heads - 1) * static_cast<__int128>(head) + n &&
      head < (B - 1) * static_cast<__int128>(seq) + n)
    return FA_ERR_STRIDE;
  return FA_OK;
}

void set_queries(fa::PagedAttn* a, const fa_paged_cache* cache, const void* Q, long long q_token, long long q_head,
                 int Hq, int max_q, int max_k, float scale, int causal) {
  a->q = static_cast<const uint8_t*>(Q);
  a->q_token = 2 * q_token;
  a->q_head = 2 * q_head;
  a->o = nullptr;
  a->lse = nullptr;
  a->Hq = Hq;
  a->group = Hq / cache->kv_heads;
  a->max_q = max_q;
  a->max_k = max_k;
  a->causal = causal;
  a->scale_log2 = scale * 1.4426950408889634f;
  a->part = fa::kPartNone;
  a->part_o = a->part_lse = nullptr;
  a->part_row = a->part_block = 0;
  a->first_o = a->first_lse = nullptr;
}

PagedPlan plan_of(const fa::PagedAttn& a, const fa_paged_cache& c) {
  return make_paged_plan(a.r.B, a.c.heads, a.group, c.head_dim, c.dtype, a.r.total, a.max_q, a.max_k);
}

int check_grid(const PagedPlan& k, const fa::PagedAttn& a) {
  const long long grid = static_cast<long long>(k.slots) * a.c.heads;  // of all heads
  return grid > 0x7fffffffLL || static_cast<long long>(a.r.B) * a.c.heads > 0x7fffffffLL ||
                 static_cast<long long>(a.r.total) * a.Hq > (1LL << 33)
             ? FA_ERR_TOO_LARGE
             : FA_OK;
}

// Sizes whose plan can be made (what the calls refuse has none).
bool sizes_ok(const fa_paged_cache* c, int B, int Hq, int total, int max_q, int max_k) {
  if (!c || c->kv_heads <= 0 || Hq <= 0 || total <= 0) return false;
  const int group = Hq / c->kv_heads;
  return group * c->kv_heads == Hq && group <= 128 && B >= 0 && max_q >= 0 && max_k >= 0 &&
         (c->head_dim == 64 || c->head_dim == 128) && c->dtype >= FA_DTYPE_F16 && c->dtype <= FA_DTYPE_E4M3 &&
         c->kv_heads <= kMaxHeads && B <= kMaxBatch && total <= kMaxRows;
}

// fp32 results of a first pass: O and LSE.
size_t part_bytes(int total, int Hq, int head_dim) {
  return (static_cast<size_t>(total) * Hq * (head_dim + 1) * sizeof(float) + 127) / 128 * 128;
}

// How the second of two passes joins its rows with the first's.  The chunk kernel does it as it
// writes them, and the decode kernel where a CTA has one (sequence, head).  Where teams end
// many short segments they would wait there for what they read (64 tokens over 64 sequences: 60
// us instead of 30 for the pass), so the combine does it; and where both kernels run their
// results go to the workspace and a kernel of its own joins them.
int join_mode(const PagedPlan& k) {
  if (k.chunk) return k.decode ? fa::kPartSecond : fa::kPartJoin;
  return k.ws_decode == 0 ? fa::kPartJoin : fa::kPartRuns;
}
int part_buffers(const PagedPlan& second) { return join_mode(second) == fa::kPartJoin ? 1 : 2; }

// The kernels of one pass.  `early`: it may start while the kernels before it end.
int run_paged(const fa::PagedAttn& a, const fa_paged_cache& cache, const PagedPlan& k, const void* Q,
              long long q_token_stride, long long q_head_stride, int dtype, void* workspace, void* stream,
              bool early = false) {
  const bool eight = is_8bit(cache.dtype);
  const bool bf16 = dtype == FA_DTYPE_BF16;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (k.decode) {
    fa::DecodeParams p;
    p.a = a;
    p.ws = static_cast<float*>(workspace);
    p.max_rows = k.decode_rows;
    p.early = early ? 1 : 0;
    p.epoch = fa::host_next_epoch();
    p.timeout_ns = fa::host_timeout_ns();
    if (!page_maps(cache, 16, &p)) return FA_ERR_TENSOR_MAP;
    const auto launch = a.part == fa::kPartNone ? fa::launch_paged_decode : fa::launch_paged_decode_part;
    if (launch(p, cache.head_dim, cache.dtype, bf16, fa::host_sm_count(), st) != cudaSuccess) return FA_ERR_LAUNCH;
  }
  if (k.chunk) {
    fa::ChunkParams p;
    p.a = a;
    p.tq = k.tq;
    p.box_rows = eight ? 128 : gcd_128(cache.page_size);
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
        (eight ? rows_maps(p, cache.head_dim, k.exp_heads) : chunk_maps(cache, &p)) &&
        query_map(cache, p.tq, Q, q_token_stride, q_head_stride, a.Hq, a.r.total, bf16, &p.tm_q);
    if (!maps) return FA_ERR_TENSOR_MAP;
    for (p.head0 = 0; p.head0 < a.c.heads; p.head0 += k.exp_heads) {
      p.n_heads = a.c.heads - p.head0 < k.exp_heads ? a.c.heads - p.head0 : k.exp_heads;
      p.fill = !k.decode && p.head0 == 0 ? 1 : 0;
      p.epoch = fa::host_next_epoch();
      p.n_ctas = k.runs ? k.n_ctas : k.slots * p.n_heads;
      const long long most = static_cast<long long>(k.slots) * p.n_heads;
      p.max_items = most < 0x7fffffffLL ? static_cast<int>(most) : 0x7fffffff;
      const auto launch = a.part == fa::kPartNone ? fa::launch_paged_chunk : fa::launch_paged_chunk_part;
      if (launch(p, cache.head_dim, cache.dtype, bf16, fa::host_sm_count(), st) != cudaSuccess) return FA_ERR_LAUNCH;
    }
  }
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
  if (!sizes_ok(cache, B, Hq, total_q, max_seqlen_q, max_seqlen_k)) return 0;
  return make_paged_plan(B, cache->kv_heads, Hq / cache->kv_heads, cache->head_dim, cache->dtype, total_q,
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
  if (int rc = check_attention(Hq, max_seqlen_q, max_seqlen_k, scale, causal)) return rc;
  if (Hq == 0 || total_q == 0) return FA_OK;
  if (int rc = check_queries(a.c, Hq, total_q, Q, O, q_token_stride, q_head_stride)) return rc;
  if (!aligned16(workspace) || (reinterpret_cast<uintptr_t>(lse) & 3u)) return FA_ERR_ALIGNMENT;
  if (int rc = check_query_strides(Hq, total_q, q_token_stride, q_head_stride)) return rc;
  set_queries(&a, cache, Q, q_token_stride, q_head_stride, Hq, max_seqlen_q, max_seqlen_k, scale, causal);
  a.o = O;
  a.lse = lse;
  const PagedPlan k = plan_of(a, *cache);
  if (k.ws_bytes > 0 && (!workspace || workspace_bytes < k.ws_bytes)) return FA_ERR_INVALID_ARG;
  if (int rc = check_grid(k, a)) return rc;
  if (int rc = fa::host_check_device()) return rc;
  return run_paged(a, *cache, k, Q, q_token_stride, q_head_stride, dtype, workspace, stream);
}

size_t fa_fwd_paged_prefix_workspace_bytes(const fa_paged_cache* cache, int n_prefixes,
                                           int max_prefix_q, int max_prefix_k, int B, int Hq,
                                           int total_q, int max_seqlen_q, int max_seqlen_k) {
  if (!sizes_ok(cache, B, Hq, total_q, max_seqlen_q, max_seqlen_k) ||
      !sizes_ok(cache, n_prefixes, Hq, total_q, max_prefix_q, max_prefix_k))
    return 0;
  const int group = Hq / cache->kv_heads;
  const PagedPlan first = make_paged_plan(n_prefixes, cache->kv_heads, group, cache->head_dim, cache->dtype,
                                          total_q, max_prefix_q, max_prefix_k);
  const PagedPlan second = make_paged_plan(B, cache->kv_heads, group, cache->head_dim, cache->dtype, total_q,
                                           max_seqlen_q, max_seqlen_k);
  return part_buffers(second) * part_bytes(total_q, Hq, cache->head_dim) + first.ws_bytes + second.ws_bytes;
}

int fa_fwd_paged_prefix(const fa_paged_cache* cache, const int* prefix_table,
                        long long prefix_table_stride, int prefix_max_pages, int n_prefixes,
                        const int* cu_prefix_q, const int* prefix_lens, int max_prefix_q,
                        int max_prefix_k, const void* Q, long long q_token_stride,
                        long long q_head_stride, void* O, float* lse, const int* cu_seqlens_q,
                        const int* seqlens_k, int B, int Hq, int total_q, int max_seqlen_q,
                        int max_seqlen_k, float scale, int causal, int dtype, void* workspace,
                        size_t workspace_bytes, void* stream) {
  fa::PagedAttn a, first;
  if (int rc = check_cache(cache, dtype, false, &a.c)) return rc;
  fa_paged_cache of_prefixes = *cache;
  of_prefixes.block_table = prefix_table;
  of_prefixes.table_stride = prefix_table_stride;
  of_prefixes.max_pages = prefix_max_pages;
  if (int rc = check_cache(&of_prefixes, dtype, false, &first.c)) return rc;
  if (int rc = check_rows(cu_seqlens_q, seqlens_k, B, total_q, &a.r)) return rc;
  if (int rc = check_rows(cu_prefix_q, prefix_lens, n_prefixes, total_q, &first.r)) return rc;
  if (int rc = check_attention(Hq, max_seqlen_q, max_seqlen_k, scale, causal)) return rc;
  if (int rc = check_attention(Hq, max_prefix_q, max_prefix_k, scale, FA_CAUSAL_NONE)) return rc;
  if (Hq == 0 || total_q == 0) return FA_OK;
  if (int rc = check_queries(a.c, Hq, total_q, Q, O, q_token_stride, q_head_stride)) return rc;
  if (!aligned16(workspace) || (reinterpret_cast<uintptr_t>(lse) & 3u)) return FA_ERR_ALIGNMENT;
  if (int rc = check_query_strides(Hq, total_q, q_token_stride, q_head_stride)) return rc;
  set_queries(&a, cache, Q, q_token_stride, q_head_stride, Hq, max_seqlen_q, max_seqlen_k, scale, causal);
  set_queries(&first, cache, Q, q_token_stride, q_head_stride, Hq, max_prefix_q, max_prefix_k, scale,
              FA_CAUSAL_NONE);
  a.o = O;
  a.lse = lse;
  const PagedPlan k1 = plan_of(first, of_prefixes), k2 = plan_of(a, *cache);
  const size_t part = part_bytes(total_q, Hq, cache->head_dim);
  const size_t parts = part_buffers(k2) * part;
  // (the second pass may start while the first still uses its workspace: each has its own)
  const size_t need = parts + k1.ws_bytes + k2.ws_bytes;
  if (!workspace || workspace_bytes < need) return FA_ERR_INVALID_ARG;
  if (int rc = check_grid(k1, first)) return rc;
  if (int rc = check_grid(k2, a)) return rc;
  if (int rc = fa::host_check_device()) return rc;
  char* const ws = static_cast<char*>(workspace) + parts;
  const size_t rows = static_cast<size_t>(total_q) * Hq;
  first.part_o = static_cast<float*>(workspace);
  first.part_lse = first.part_o + rows * cache->head_dim;
  first.part = fa::kPartFirst;
  first.part_row = a.part_row = cache->head_dim;
  first.part_block = a.part_block = 4;
  a.part = join_mode(k2);
  a.first_o = first.part_o;
  a.first_lse = first.part_lse;
  if (a.part == fa::kPartJoin) {
    a.part_o = first.part_o;
    a.part_lse = first.part_lse;
    if (k2.chunk) {  // a thread of the chunk kernel has a row: the same columns of the rows side by side
      first.part_row = a.part_row = 4;
      first.part_block = a.part_block = 4 * static_cast<long long>(rows);
    }
  } else {
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + part);
    a.part_lse = a.part_o + rows * cache->head_dim;
  }
  if (int rc = run_paged(first, of_prefixes, k1, Q, q_token_stride, q_head_stride, dtype, ws, stream)) return rc;
  if (int rc = run_paged(a, *cache, k2, Q, q_token_stride, q_head_stride, dtype, ws + k1.ws_bytes, stream,
                         /*early=*/true))
    return rc;
  if (a.part != fa::kPartSecond) return FA_OK;
  const fa::PagedMerge m{first.part_o, first.part_lse, a.part_o, a.part_lse, O, lse, total_q, Hq};
  const cudaError_t e = fa::launch_paged_merge(m, cache->head_dim, dtype == FA_DTYPE_BF16,
                                               static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FA_OK : FA_ERR_LAUNCH;
}

int fa_kvcache_weights(const fa_paged_cache* cache, const void* Q, long long q_token_stride,
                       long long q_head_stride, const float* lse, const int* cu_seqlens_q,
                       const int* seqlens_k, int B, int Hq, int total_q, int max_seqlen_q,
                       int max_seqlen_k, float* weights, long long w_seq_stride,
                       long long w_head_stride, int weights_len, int mode, float scale, int causal,
                       int dtype, void* stream) {
  fa::PagedWeights p;
  if (int rc = check_cache(cache, dtype, false, &p.a.c, /*values=*/false)) return rc;
  if (int rc = check_rows(cu_seqlens_q, seqlens_k, B, total_q, &p.a.r)) return rc;
  // (a sequence without new tokens has sums too)
  if (B > 0 && (!cu_seqlens_q || !seqlens_k)) return FA_ERR_INVALID_ARG;
  if (int rc = check_attention(Hq, max_seqlen_q, max_seqlen_k, scale, causal)) return rc;
  if (mode < FA_WEIGHTS_SET || mode > FA_WEIGHTS_APPEND) return FA_ERR_INVALID_ARG;
  const long long held = static_cast<long long>(cache->max_pages) * cache->page_size;
  const int keys = static_cast<int>(max_seqlen_k < held ? max_seqlen_k : held);
  if (int rc = check_sums(weights, w_seq_stride, w_head_stride, weights_len, keys, B, p.a.c.heads)) return rc;
  if (Hq == 0) return FA_ERR_INVALID_ARG;
  if (B == 0 || keys == 0) return FA_OK;
  if (int rc = check_queries(p.a.c, Hq, total_q, Q, lse, q_token_stride, q_head_stride, 4)) return rc;
  if (int rc = check_query_strides(Hq, total_q, q_token_stride, q_head_stride)) return rc;
  if (static_cast<long long>(B) * p.a.c.heads > 0x7fffffffLL || static_cast<long long>(total_q) * Hq > (1LL << 33))
    return FA_ERR_TOO_LARGE;
  // Sequences of few query rows are streamed, the others go through the tensor cores; both
  // where the bounds allow both (see kMixedRows).
  const int most = max_seqlen_q < total_q ? max_seqlen_q : total_q, group = Hq / p.a.c.heads;
  const bool chunk = static_cast<long long>(most) * group > fa::paged_weights_rows();
  const bool few = !chunk || (B > 1 && group <= kMixedRows && total_q < static_cast<long long>(B) * most);
  const int few_rows = chunk ? kMixedRows / group * group : most * group;
  const long long blocks = (static_cast<long long>(keys) + fa::paged_weights_chunk_keys() - 1) / fa::paged_weights_chunk_keys();
  if (chunk && blocks * B * p.a.c.heads > 0x7fffffffLL) return FA_ERR_TOO_LARGE;
  if (int rc = fa::host_check_device()) return rc;
  set_queries(&p.a, cache, Q, q_token_stride, q_head_stride, Hq, max_seqlen_q, keys, scale, causal);
  p.a.lse = const_cast<float*>(lse);
  p.w = weights;
  p.w_seq = w_seq_stride;
  p.w_head = w_head_stride;
  p.mode = mode;
  const bool bf16 = dtype == FA_DTYPE_BF16;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // (everything that can be refused is, before the first kernel changes a sum: with "add" or
  // "append" the call could not be made again)
  fa::WeightsChunkParams c;
  if (chunk) {
    c.w = p;
    c.tq = 128 / group;
    c.skip_rows = few ? few_rows : -1;
    c.epoch = fa::host_next_epoch();
    c.timeout_ns = fa::host_timeout_ns();
    if (!query_map(*cache, c.tq, Q, q_token_stride, q_head_stride, Hq, total_q, bf16, &c.tm_q))
      return FA_ERR_TENSOR_MAP;
  }
  if (few && fa::launch_paged_weights(p, few_rows, cache->head_dim, cache->dtype, bf16, fa::host_sm_count(), st) !=
                 cudaSuccess)
    return FA_ERR_LAUNCH;
  if (chunk &&
      fa::launch_paged_weights_chunk(c, cache->head_dim, cache->dtype, bf16, fa::host_sm_count(), st) != cudaSuccess)
    return FA_ERR_LAUNCH;
  return FA_OK;
}

int fa_kvcache_evict(const fa_paged_cache* cache, float* weights, long long w_seq_stride,
                     long long w_head_stride, int weights_len, const int* seqlens_k,
                     const int* keep, int keep_all, int first, int recent, int* new_lens, int B,
                     void* stream) {
  fa::PagedEvict p;
  if (!cache) return FA_ERR_INVALID_ARG;
  const bool eight = is_8bit(cache->dtype);
  if (int rc = check_cache(cache, eight ? FA_DTYPE_F16 : cache->dtype, true, &p.c)) return rc;
  if (B < 0 || first < 0 || recent < 0) return FA_ERR_INVALID_ARG;
  if (B > kMaxBatch || static_cast<long long>(B) * p.c.heads > 0x7fffffffLL) return FA_ERR_TOO_LARGE;
  if (B == 0) return FA_OK;
  if (!seqlens_k || !new_lens || new_lens == seqlens_k || new_lens == keep) return FA_ERR_INVALID_ARG;
  if (((reinterpret_cast<uintptr_t>(seqlens_k) | reinterpret_cast<uintptr_t>(keep) |
        reinterpret_cast<uintptr_t>(new_lens)) & 3u) != 0)
    return FA_ERR_ALIGNMENT;
  if (int rc = check_sums(weights, w_seq_stride, w_head_stride, weights_len, p.c.max_pages * p.c.page_size, B,
                          p.c.heads))
    return rc;
  if (int rc = fa::host_check_device()) return rc;
  p.w = weights;
  p.w_seq = w_seq_stride;
  p.w_head = w_head_stride;
  p.lens = seqlens_k;
  p.keep = keep;
  p.keep_all = keep_all;
  p.first = first;
  p.recent = recent;
  p.new_lens = new_lens;
  p.B = B;
  const cudaError_t e = fa::launch_paged_evict(p, cache->head_dim * (eight ? 1 : 2), eight, fa::host_sm_count(),
                                               static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FA_OK : FA_ERR_LAUNCH;
}

}  // extern "C"
