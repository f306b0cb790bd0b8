// Device-side view of a paged KV cache and of the new tokens of a call, and
// the launchers of the paged kernels (fa_paged_cache.cu, fa_paged_decode.cuh, fa_paged_chunk.cuh).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "fa_b200.h"

namespace fa {

struct PagedCache {
  const uint8_t* k;  // pages (element size 2, or 1 in 8-bit caches)
  const uint8_t* v;
  float* ks;         // scales of an 8-bit cache
  float* vs;
  long long page_stride, head_stride, row_stride;  // bytes
  long long s_page, s_head, s_row;                 // scale elements
  const int* table;
  long long table_stride;
  int max_pages, num_pages, heads, page_size;
  int page_shift;    // log2(page_size), or -1 if it is no power of two

  __device__ __forceinline__ int page_of(int pos) const {
    return page_shift >= 0 ? pos >> page_shift : pos / page_size;
  }
  // Page id that holds position pos (>= 0) of sequence b, -1 if none does.
  __device__ __forceinline__ int lookup(int b, int pos) const {
    const int i = page_of(pos);
    if (i >= max_pages) return -1;
    const int page = __ldg(table + static_cast<long long>(b) * table_stride + i);
    return static_cast<unsigned>(page) < static_cast<unsigned>(num_pages) ? page : -1;
  }
  __device__ __forceinline__ int row_in_page(int pos) const {
    return page_shift >= 0 ? pos & (page_size - 1) : pos % page_size;
  }
};

// New tokens: sequence b owns packed rows [cu[b], cu[b+1]) and ends at
// position lens[b] of its cache.
struct PagedRows {
  const int* cu;
  const int* lens;
  int B;
  int total;  // packed rows
};

// K/V rows of new tokens (strides in bytes).
struct PagedSource {
  const uint8_t* k;
  const uint8_t* v;
  long long k_token, k_head, v_token, v_head;
};

struct PagedAttn {
  PagedCache c;
  PagedRows r;
  const uint8_t* q;           // strides in bytes
  long long q_token, q_head;
  void* o;                    // [total, Hq, d]
  float* lse;                 // [Hq, total] or nullptr
  int Hq, group;              // group = Hq / heads
  int max_q, max_k;
  int causal;                 // FA_CAUSAL_*
  float scale_log2;           // scale * log2(e)
};

// An item of the chunk kernel that the end of a run cuts: its sequence's first row
// and tokens, its first token, KV head and parts (0: none is cut).
struct alignas(16) PagedCut {
  int c0, nq, tok0, h, parts, pad[3];
};

struct alignas(64) ChunkParams {
  CUtensorMap tm_q;  // (d, Hq, T), box (64, G, tq)
  // (64 columns, 8 rows, d / 64, row groups of 8, planes), box (64, 8, d / 64,
  // box_rows / 8, 1): a plane is a head of a page, at page * page_step + head *
  // head_step; 8-bit pages: a head's expanded rows
  CUtensorMap tm_k;
  CUtensorMap tm_v;
  PagedAttn a;
  int tq;            // tokens of a 128-row tile: 128 / group
  int box_rows;
  int page_step, head_step;
  int stale;         // tiles may end in stale rows (pages do, the expanded rows do not)
  int skip_rows;     // sequences with at most this many rows per KV head are not ours
  int runs;          // 1: CTAs take equal runs of the work order, 0: a (pair, head) each
  int n_ctas;
  int fill;          // write the rows that no kernel computes
  int head0, n_heads;  // KV heads of this launch
  // 8-bit pages: 16-bit rows and scales of the launch's heads (paged_expand_kernel)
  long long exp_rows;
  uint16_t* exp_k;   // [n_heads][exp_rows][d], the type of the queries
  uint16_t* exp_v;   // f16
  float* exp_ks;     // [n_heads][exp_rows]
  float* exp_vs;     // ... times 2^-kScaleShift
  float* exp_vl;     // ... log2 of its magnitude
  float* exp_vm;     // [n_heads][exp_rows / 16], the largest exp_vl of 16 rows
  // parts of cut items, two slots per run: [2 n_ctas][2 query tiles][d / 4][128
  // rows][4] fp32, normalised, and [2 n_ctas][2][128], natural log
  float* ws_o;
  float* ws_lse;
  PagedCut* ws_cuts;  // [n_ctas]
  unsigned epoch;
  unsigned long long timeout_ns;
};

cudaError_t launch_cache_write(const PagedCache& c, const PagedRows& r, const PagedSource& s,
                               int head_dim, int cache_dtype, bool bf16, cudaStream_t stream);
cudaError_t launch_cache_read(const PagedCache& c, const PagedRows& r, void* k, void* v,
                              int head_dim, int cache_dtype, bool bf16, cudaStream_t stream);

struct alignas(64) DecodeParams {
  CUtensorMap tm_k;  // (d, page rows, heads, pages), box (min(row, 128 bytes), 16, 1, 1)
  CUtensorMap tm_v;
  int page_step, head_step;  // 1, or 0 where the map has one entry for all of them
  PagedAttn a;
  float* ws;
  // set by launch_paged_decode: teams of the launch, one CTA per (sequence,
  // head), ring stages per warp
  int n_teams, solo, stages;
  int max_rows;  // query rows per KV head of the sequences handled
  unsigned epoch;
  unsigned long long timeout_ns;
};

// Decode kernel: sequences with at most max_rows <= paged_decode_rows() query
// rows (new tokens x group) per KV head, and the rows of sequences without
// visible keys or of no sequence.  Sequences with more rows are left alone.
// heads: sequences x KV heads.
int paged_decode_rows(long long heads, int head_dim, int cache_dtype, int sms);
size_t paged_decode_ws_bytes(long long heads, int max_rows, int max_k, int head_dim, int cache_dtype, int sms);
cudaError_t launch_paged_decode(DecodeParams p, int head_dim, int cache_dtype, bool bf16, int sms,
                                cudaStream_t stream);
// Chunk kernel (after the expansion of 8-bit pages) over the KV heads of p, and
// the join of the items that its runs cut.
cudaError_t launch_paged_chunk(const ChunkParams& p, int head_dim, int cache_dtype, bool bf16, int sms,
                               cudaStream_t stream);

}  // namespace fa
