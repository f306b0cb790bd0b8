/*
 * fa_b200.h — C ABI of the B200 (sm_100a) FlashAttention forward.
 *
 * Drop-in boundary for the reference's attention-forward path
 * (JohnScheuer/flash-attention-sm75-register-fused).  Every entry point takes
 * plain device pointers and sizes; no framework types cross this boundary.
 *
 * Layout (all entry points): Q [B, Hq, N, d], K/V [B, Hkv, N, d], O like Q,
 * row-major and contiguous, f16 (or bf16 where a dtype argument exists).
 * LSE (optional) is fp32 [B, Hq, N], natural log:  LSE = log sum_j exp(s_ij).
 * Causal masking is top-left aligned: query i attends keys j <= i.
 * GQA: query head h reads KV head h / (Hq / Hkv) (repeat_interleave order).
 *
 * Pointer arguments are typed void* here; the reference declares the legacy
 * launchers with `half*`, which is the same C ABI, so the reference binding
 * (src/bindings/pytorch_extension.cpp:4-19) links against this library as is.
 */
#ifndef FA_B200_H
#define FA_B200_H

#include <stdbool.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes returned by the int-returning entry points ---- */
enum {
  FA_OK = 0,
  FA_ERR_INVALID_ARG = 1,          /* null pointer, negative size, bad causal/dtype flag */
  FA_ERR_UNSUPPORTED_HEAD_DIM = 2, /* head_dim not in {64, 128} */
  FA_ERR_GQA_DIVISIBILITY = 3,     /* Hq % Hkv != 0 */
  FA_ERR_ALIGNMENT = 4,            /* a pointer is not 16-byte aligned */
  FA_ERR_DTYPE = 5,                /* dtype not FA_DTYPE_F16 / FA_DTYPE_BF16 */
  FA_ERR_TENSOR_MAP = 6,           /* cuTensorMapEncodeTiled rejected a shape */
  FA_ERR_LAUNCH = 7,               /* kernel launch failed (see cudaGetLastError) */
  FA_ERR_DEVICE = 8,               /* current device is not sm_100 */
  FA_ERR_CUDA = 9,                 /* another CUDA runtime call failed */
  FA_ERR_TOO_LARGE = 10,           /* a size overflows the kernel's index types */
  FA_ERR_SCRATCH_LIMIT = 11,       /* fa_naive_fwd_noalloc: problem larger than its static scratch */
  FA_ERR_PAGE_SIZE = 12,           /* paged cache: page_size not a positive multiple of 16 */
  FA_ERR_GROUP = 13,               /* paged attention: more than 128 query heads per KV head */
  FA_ERR_SCALES = 14,              /* 8-bit cache without scales, or a 16-bit cache with them */
  FA_ERR_STRIDE = 15,              /* paged cache or its queries: a stride that cannot be used */
  FA_ERR_TIMEOUT_BASE = 100        /* device watchdog: 100 + wait site id */
};

enum {
  FA_DTYPE_F16 = 0,
  FA_DTYPE_BF16 = 1,
  FA_DTYPE_INT8 = 2, /* paged caches only: value = int8 * scale of its row */
  FA_DTYPE_E4M3 = 3  /* paged caches only: value = e4m3 * scale of its row */
};

/* Causal alignment for fa_fwd_kvcache (fa_fwd takes 0/1; for Nq == Nk both
 * alignments are the reference's top-left mask, attention_ref.py:33-40). */
enum {
  FA_CAUSAL_NONE = 0,
  FA_CAUSAL_BOTTOM_RIGHT = 1, /* key j visible to query i iff j <= i + Nk - Nq (KV cache) */
  FA_CAUSAL_TOP_LEFT = 2      /* key j visible to query i iff j <= i (SDPA is_causal) */
};

/* Test hooks (fa_set_debug_flags). */
enum {
  FA_DEBUG_SKIP_Q_LOAD = 1, /* producer never loads Q: the consumers' wait must time out */
  FA_DEBUG_PAIR_KERNEL = 2, /* square / chunked prefill always on the pair kernel (two Q
                               tiles per CTA), for comparisons */
  FA_DEBUG_TILE_SPLIT2 = 4, /* tile kernel with each tile's keys split between 2 softmax
                               warpgroups instead of 4, for comparisons */
  FA_DEBUG_TILE_KERNEL = 8, /* square / chunked prefill always on the tile kernel (one Q
                               tile per CTA, S double-buffered), for comparisons */
  FA_DEBUG_PAIR2_KERNEL = 16, /* d = 128 square / chunked prefill on CTA pairs (one product
                                for two SMs) wherever they apply (opt-in) */
  FA_DEBUG_NO_TAIL_SPLIT = 32, /* keep a pair-kernel launch's half-empty last wave on the pair
                                 kernel instead of the tile kernel, for comparisons */
  FA_DEBUG_NO_PERSIST = 64,     /* one CTA per pair-kernel work item instead of persistent
                                 CTAs, for comparisons */
  FA_DEBUG_STATIC_DEAL = 128,   /* persistent pair-kernel CTAs deal every round in the fixed
                                 boustrophedon order (the last rounds too), for comparisons */
  FA_DEBUG_DUAL_TILES = 256     /* d = 64 square launches as one-Q-tile items whose two softmax
                                 groups split the keys and merge in the CTA, wherever they apply
                                 (by default only non-causal launches of one to two waves of Q
                                 pairs; FA_DEBUG_PAIR_KERNEL keeps Q pairs there) */
};

/*
 * fa_fwd — asynchronous attention forward on `stream` (cudaStream_t; NULL =
 * legacy default stream).  Returns FA_OK or an FA_ERR_* code; argument errors
 * are reported before anything is launched.  B == 0, Hq == 0 or N == 0 is a
 * no-op.  `lse` may be NULL.
 *
 * Replaces: launch_flash_attention_forward
 *   (reference src/kernels/flash_attention_forward.cu:795-817) with native
 *   GQA (reference expands K/V in src/flash_attention_sm75/ops.py:6-27),
 *   an LSE output, bf16, a caller stream and an error code.
 */
int fa_fwd(const void* Q, const void* K, const void* V, void* O, float* lse, int B, int Hq,
           int Hkv, int N, int head_dim, float scale, int causal, int dtype, void* stream);

/*
 * fa_fwd_kvcache — attention of Nq new queries against Nk cached keys
 * (decode: Nq = 1; chunked prefill: Nq < Nk).  Q/O are [B, Hq, Nq, d], K/V
 * [B, Hkv, Nk, d], LSE [B, Hq, Nq]; `causal` is an FA_CAUSAL_* value.  Rows
 * that see no key (bottom-right with Nq > Nk) get O = 0 and LSE = -inf.
 * When the call alone would not fill the GPU, the key range is split across
 * CTAs and merged by a second kernel; that needs `workspace` (16-byte aligned)
 * of at least fa_fwd_kvcache_workspace_bytes() bytes, otherwise (NULL or
 * smaller) the call runs unsplit.  Asynchronous on `stream`.
 *
 * No reference counterpart: the reference's HF patch sends these calls to
 * PyTorch SDPA (reference src/flash_attention_sm75/llama_attention_replacement.py:63-65,
 * reason "kvcache_decode").
 */
int fa_fwd_kvcache(const void* Q, const void* K, const void* V, void* O, float* lse, int B,
                   int Hq, int Hkv, int Nq, int Nk, int head_dim, float scale, int causal,
                   int dtype, void* workspace, size_t workspace_bytes, void* stream);

/* Workspace bytes fa_fwd_kvcache needs to split this problem (0: no split). */
size_t fa_fwd_kvcache_workspace_bytes(int B, int Hq, int Hkv, int Nq, int Nk, int head_dim);

/*
 * fa_fwd_varlen — attention over a packed batch of variable-length sequences
 * (the cu_seqlens layout): Q/O [total_q, Hq, d], K/V [total_k, Hkv, d], all
 * contiguous.  Sequence b owns query rows [cu_seqlens_q[b], cu_seqlens_q[b+1])
 * and key rows [cu_seqlens_k[b], cu_seqlens_k[b+1]); the offsets are int32
 * DEVICE arrays of B + 1 non-decreasing entries (clamped to [0, total]).
 * max_seqlen_q / max_seqlen_k bound the lengths (query rows of a longer
 * sequence past max_seqlen_q, rounded up to 256, are not computed).
 * `causal`: FA_CAUSAL_BOTTOM_RIGHT (key j visible to query i of a sequence iff
 * j <= i + nk - nq), FA_CAUSAL_TOP_LEFT (j <= i) or FA_CAUSAL_NONE.  LSE (may be
 * NULL) is fp32 [Hq, total_q].  Rows that see no key get O = 0, LSE = -inf.
 * Keys past a sequence's end are masked; the V rows that follow it in the
 * packed buffer (the next sequence's) are multiplied by exactly 0, so they
 * must be finite.  Asynchronous on `stream`.
 *
 * No reference counterpart: the reference's HF patch sends masked (padded /
 * varlen) batches to PyTorch SDPA (reference
 * src/flash_attention_sm75/llama_attention_replacement.py:61-62, reason
 * "has_attn_mask").
 */
int fa_fwd_varlen(const void* Q, const void* K, const void* V, void* O, float* lse,
                  const int* cu_seqlens_q, const int* cu_seqlens_k, int B, int Hq, int Hkv,
                  int total_q, int total_k, int max_seqlen_q, int max_seqlen_k, int head_dim,
                  float scale, int causal, int dtype, void* stream);

/*
 * fa_fwd_padded — attention of a padded batch in the fixed layout (Q/O
 * [B, Hq, Nq, d], K/V [B, Hkv, Nk, d], LSE [B, Hq, Nq]): batch entry b's valid
 * queries are rows [q_start[b], q_end[b]) and its valid keys rows
 * [k_start[b], k_end[b]) (int32 DEVICE arrays of B entries, clamped to
 * [0, Nq] / [0, Nk]).  Padding keys are never attended; rows of O and LSE
 * outside a query range are not written.  `causal` follows fa_fwd_kvcache on
 * the full padded rows (BOTTOM_RIGHT: key j visible to query i iff
 * j <= i + Nk - Nq; TOP_LEFT: j <= i), restricted to the valid keys; valid
 * rows that then see no key get O = 0, LSE = -inf.  Covers left padding
 * (start > 0), right padding (end < N) and both.  Asynchronous on `stream`.
 *
 * No reference counterpart (reference llama_attention_replacement.py:61-62).
 */
int fa_fwd_padded(const void* Q, const void* K, const void* V, void* O, float* lse,
                  const int* q_start, const int* q_end, const int* k_start, const int* k_end,
                  int B, int Hq, int Hkv, int Nq, int Nk, int head_dim, float scale, int causal,
                  int dtype, void* stream);

/*
 * fa_bwd — gradients of fa_fwd (square, causal 0/1 top-left, GQA): from Q, K, V,
 * the forward's O and LSE ([B, Hq, N] fp32, natural log) and dO = dL/dO, writes
 * dQ [B, Hq, N, d], dK and dV [B, Hkv, N, d] (GQA: summed over each group's
 * query heads).  `workspace` (16-byte aligned) needs fa_bwd_workspace_bytes()
 * bytes.  Asynchronous on `stream`; same error codes as fa_fwd.
 *
 * No reference counterpart: the reference's autograd Function raises in
 * backward (reference src/flash_attention_sm75/ops.py:47-52).
 */
int fa_bwd(const void* Q, const void* K, const void* V, const void* O, const void* dO,
           const float* lse, void* dQ, void* dK, void* dV, int B, int Hq, int Hkv, int N,
           int head_dim, float scale, int causal, int dtype, void* workspace,
           size_t workspace_bytes, void* stream);

/* Workspace bytes of fa_bwd: two fp32 values per query row (from LSE and rowsum(dO*O)) and two
 * 4 KB operand tiles per 128-row query tile, rows padded to 128. */
size_t fa_bwd_workspace_bytes(int B, int Hq, int N);

/*
 * fa_bwd_padded — gradients of fa_fwd_padded for square padded batches
 * (Nq = Nk = N): batch entry b's valid query rows are [q_start[b], q_end[b]) and
 * valid keys [k_start[b], k_end[b]) (int32 device arrays of B entries); O and
 * LSE come from fa_fwd_padded (rows outside a query range: O = 0, LSE = -inf, as
 * the Python API returns them).  Padding keys get dK = dV = 0 and query rows
 * outside the ranges dQ = 0.  `causal` 0/1 (bottom-right = top-left for square
 * inputs).  Workspace, errors and stream as fa_bwd.
 *
 * No reference counterpart (reference llama_attention_replacement.py:61-62).
 */
int fa_bwd_padded(const void* Q, const void* K, const void* V, const void* O, const void* dO,
                  const float* lse, const int* q_start, const int* q_end, const int* k_start,
                  const int* k_end, void* dQ, void* dK, void* dV, int B, int Hq, int Hkv, int N,
                  int head_dim, float scale, int causal, int dtype, void* workspace,
                  size_t workspace_bytes, void* stream);

/*
 * fa_bwd_varlen — gradients of fa_fwd_varlen for packed self-attention batches
 * (the same cu_seqlens for queries and keys): Q, K, V, O, dO, dQ, dK, dV in the
 * packed layout ([total, H, d]), LSE fp32 [Hq, total] from fa_fwd_varlen,
 * cu_seqlens int32 device array of B + 1 offsets, max_seqlen >= every length.
 * `causal` 0/1.  Workspace: fa_bwd_workspace_bytes(B, Hq, max_seqlen).
 * Errors and stream as fa_bwd.
 *
 * No reference counterpart (reference llama_attention_replacement.py:61-62).
 */
int fa_bwd_varlen(const void* Q, const void* K, const void* V, const void* O, const void* dO,
                  const float* lse, const int* cu_seqlens, void* dQ, void* dK, void* dV, int B,
                  int Hq, int Hkv, int total, int max_seqlen, int head_dim, float scale,
                  int causal, int dtype, void* workspace, size_t workspace_bytes, void* stream);

/* ---- paged KV cache ----
 *
 * A cache of `num_pages` pages of `page_size` tokens.  Element (page, head,
 * row, c) of K lies at k[page * page_stride + head * head_stride +
 * row * row_stride + c] (strides in elements; V the same from v), so head-major
 * pages [num_pages, kv_heads, page_size, d], token-major pages
 * [num_pages, page_size, kv_heads, d] and slices of a larger array all fit.
 * Pointers are 16-byte aligned and the strides multiples of 16 bytes; the row
 * stride is positive, the others not negative (where a dimension has one entry,
 * its stride is not used).  A head or page stride of 0, the same rows seen as
 * several heads or pages, is for reading alone: writes refuse it, and a scale
 * stride of 0, with FA_ERR_STRIDE.
 *
 * Position p of sequence b is row p % page_size of page
 * block_table[b * table_stride + p / page_size] (int32, on the device).  Table
 * entries outside [0, num_pages) are skipped by writes and read as rows of
 * zeros; nothing outside the cache is addressed whatever the tables hold.
 *
 * 8-bit caches (dtype FA_DTYPE_INT8 / FA_DTYPE_E4M3) hold one fp32 scale per
 * token and head for K and for V, at k_scale[page * scale_page_stride +
 * head * scale_head_stride + row * scale_row_stride]; 16-bit caches have none
 * (k_scale = v_scale = NULL).
 *
 * Every entry point takes the same description of new tokens: sequence b
 * brings n_b = cu_seqlens[b+1] - cu_seqlens[b] of them (rows cu_seqlens[b] ..
 * of the packed arrays), the last of which is position seqlens_k[b] - 1, so
 * token i is position seqlens_k[b] - n_b + i.  cu_seqlens (B + 1 entries, from
 * 0 up, non-decreasing) and seqlens_k (B entries) are int32 DEVICE arrays; the
 * kernels clamp what they read to the arrays' bounds.  Positions below 0 or
 * beyond max_pages * page_size hold nothing.
 */
typedef struct fa_paged_cache {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  long long page_stride, head_stride, row_stride;
  long long scale_page_stride, scale_head_stride, scale_row_stride;
  const int* block_table;
  long long table_stride;
  int max_pages; /* entries of one table row */
  int num_pages;
  int kv_heads;
  int page_size; /* a multiple of 16 */
  int head_dim;  /* 64 or 128 */
  int dtype;     /* FA_DTYPE_* of the pages */
} fa_paged_cache;

/*
 * fa_kvcache_write — stores the K and V rows of new tokens in their pages.
 * K/V: f16 or bf16 (`dtype`), token t's row of head h at t * token_stride +
 * h * head_stride (elements, multiples of 8; 16-byte aligned).  A 16-bit cache
 * must have the same dtype (the rows are copied); an 8-bit cache stores
 *   a = max |x| of the row, scale = a / qmax, q = round(x * (qmax / a))
 * with qmax = 127 (int8, ties to even) or 448 (e4m3, nearest even); rows with
 * a < 2^-100 are stored as zeros with scale 0, and a row that holds an
 * infinity or a NaN reads back as NaN.  Asynchronous on `stream`.  Two tokens
 * must not have the same place.
 *
 * No reference counterpart: the reference has no KV cache (reference
 * src/flash_attention_sm75/llama_attention_replacement.py:63-65 leaves cached
 * decode to PyTorch SDPA).
 */
int fa_kvcache_write(const fa_paged_cache* cache, const void* K, const void* V,
                     long long k_token_stride, long long k_head_stride,
                     long long v_token_stride, long long v_head_stride, const int* cu_seqlens,
                     const int* seqlens_k, int B, int total, int dtype, void* stream);

/*
 * fa_kvcache_read — the reverse: K/V rows [total, kv_heads, d] (contiguous,
 * f16 or bf16; a 16-bit cache's own dtype) of the described tokens, e.g. of
 * whole prefixes (cu_seqlens = running sums of seqlens_k), in the layout
 * fa_fwd_varlen takes.  8-bit values are multiplied by their scale in fp32 and
 * rounded once.  Rows of tokens without a place, and of no sequence, are zero.
 * Asynchronous on `stream`.
 */
int fa_kvcache_read(const fa_paged_cache* cache, void* K, void* V, const int* cu_seqlens,
                    const int* seqlens_k, int B, int total, int dtype, void* stream);

/*
 * fa_fwd_paged — attention of new tokens over a paged cache that already holds
 * their own keys and values: Q row (t, h) at t * q_token_stride +
 * h * q_head_stride (elements, multiples of 8, positive where there is more than
 * one token / head; 16-byte aligned), O
 * [total_q, Hq, d] contiguous, LSE (may be NULL) fp32 [Hq, total_q].  Sequence
 * b's queries see keys j < seqlens_k[b], with `causal` FA_CAUSAL_BOTTOM_RIGHT
 * those with j <= i + seqlens_k[b] - n_b, with FA_CAUSAL_TOP_LEFT j <= i.  Rows
 * that see no key, and rows of no sequence, get O = 0, LSE = -inf.  Keys that
 * no query may see have no effect, whatever their rows of the pages hold.
 * `dtype` (f16 / bf16) is that of Q and O; a 16-bit cache has the same.
 * 8-bit keys and values are used exactly, with their scales in fp32.  The
 * probabilities are rounded to f16 (16-bit pages: to their type), over 8-bit pages
 * after their product with the value's scale and relative to a row's largest one.
 * For few tokens bf16 queries over 8-bit pages are rounded to f16 relative to the
 * row's largest magnitude (exact down to 2^-17 of it).
 * max_seqlen_q / max_seqlen_k bound n_b and seqlens_k: tokens beyond them get O =
 * 0, LSE = -inf, keys beyond them are not seen.  The kernels and the workspace are chosen by
 * max_seqlen_k as it is given, so it should be no more than the longest sequence
 * there may be, and never more than max_pages * page_size.  Hq / kv_heads is at most 128.
 * `workspace` (16-byte aligned) needs fa_fwd_paged_workspace_bytes() bytes (may
 * be NULL where that is 0).  Asynchronous on `stream`.
 *
 * No reference counterpart (reference llama_attention_replacement.py:63-65).
 */
int fa_fwd_paged(const fa_paged_cache* cache, const void* Q, long long q_token_stride,
                 long long q_head_stride, void* O, float* lse, const int* cu_seqlens_q,
                 const int* seqlens_k, int B, int Hq, int total_q, int max_seqlen_q,
                 int max_seqlen_k, float scale, int causal, int dtype, void* workspace,
                 size_t workspace_bytes, void* stream);

/* Workspace bytes of fa_fwd_paged (a function of its sizes alone): partial
 * results of split keys, and for chunks over 8-bit pages the keys and values as
 * f16 (at most about 1 GiB, or one KV head's if that is more); 0 for a few new
 * tokens over short caches, and for what the call refuses. */
size_t fa_fwd_paged_workspace_bytes(const fa_paged_cache* cache, int B, int Hq, int total_q,
                                    int max_seqlen_q, int max_seqlen_k);

/*
 * fa_fwd_paged_prefix — fa_fwd_paged for a batch whose sequences share long
 * prefixes, each computed once for all its tokens.  Prefix g of n_prefixes has
 * prefix_lens[g] keys in the pages of row g of `prefix_table` (rows of
 * prefix_max_pages entries, prefix_table_stride apart; the same pages as the
 * sequences', which hold what follows the prefix), and packed rows
 * [cu_prefix_q[g], cu_prefix_q[g+1]) see all of them besides their own
 * sequence's keys, for which `causal` and everything else is as in fa_fwd_paged.
 * cu_prefix_q (n_prefixes + 1 entries, non-decreasing) and prefix_lens are int32
 * DEVICE arrays, clamped to their bounds; rows outside every range have no prefix.
 * max_prefix_q / max_prefix_k bound the tokens and keys of a prefix: tokens beyond
 * the first max_prefix_q of a range do not see it, keys beyond max_prefix_k are not seen.
 * The two sets of keys are computed one after the other and joined in fp32; the
 * result is rounded once.  `workspace` (16-byte aligned) needs
 * fa_fwd_paged_prefix_workspace_bytes() bytes.  Asynchronous on `stream`.
 *
 * No reference counterpart (reference llama_attention_replacement.py:63-65).
 */
int fa_fwd_paged_prefix(const fa_paged_cache* cache, const int* prefix_table,
                        long long prefix_table_stride, int prefix_max_pages, int n_prefixes,
                        const int* cu_prefix_q, const int* prefix_lens, int max_prefix_q,
                        int max_prefix_k, const void* Q, long long q_token_stride,
                        long long q_head_stride, void* O, float* lse, const int* cu_seqlens_q,
                        const int* seqlens_k, int B, int Hq, int total_q, int max_seqlen_q,
                        int max_seqlen_k, float scale, int causal, int dtype, void* workspace,
                        size_t workspace_bytes, void* stream);

/* Workspace bytes of fa_fwd_paged_prefix (a function of its sizes alone): fp32 results
 * of one pass or of both, and the sum of the two passes' workspaces (the second may start
 * while the first still uses its own); 0 for what the call refuses. */
size_t fa_fwd_paged_prefix_workspace_bytes(const fa_paged_cache* cache, int n_prefixes,
                                           int max_prefix_q, int max_prefix_k, int B, int Hq,
                                           int total_q, int max_seqlen_q, int max_seqlen_k);

/* What fa_kvcache_weights does with the sums of earlier calls. */
enum {
  FA_WEIGHTS_SET = 0,   /* they are replaced */
  FA_WEIGHTS_ADD = 1,   /* added to */
  FA_WEIGHTS_APPEND = 2 /* added to, but the new tokens' own positions, which have none, are set */
};

/*
 * fa_kvcache_weights — the attention weight that cached keys received: for the
 * positions j < min(seqlens_k[b], max_seqlen_k) of every sequence b and KV head h
 *   weights[b * w_seq_stride + h * w_head_stride + j]  = or +=
 *     sum over its new tokens i and the query heads of h of exp(scale q_i.k_j - LSE_i),
 * keys that a row may not see (`causal`) adding 0.  Q, cu_seqlens_q, seqlens_k,
 * the bounds, scale and causal are those of the attention call whose LSE (fp32
 * [Hq, total_q]) is given; a row whose LSE is -inf adds nothing.  Only the keys of
 * `cache` are read (v and v_scale may be NULL).  `weights` is fp32, a row holds
 * weights_len >= min(max_seqlen_k, max_pages * page_size) positions and rows do not
 * overlap; positions from there on, and those of other rows, are left as they are.
 * All sums are fp32, in an order that does not depend on timing.  Asynchronous
 * on `stream`.
 *
 * No reference counterpart (reference llama_attention_replacement.py:63-65).
 */
int fa_kvcache_weights(const fa_paged_cache* cache, const void* Q, long long q_token_stride,
                       long long q_head_stride, const float* lse, const int* cu_seqlens_q,
                       const int* seqlens_k, int B, int Hq, int total_q, int max_seqlen_q,
                       int max_seqlen_k, float* weights, long long w_seq_stride,
                       long long w_head_stride, int weights_len, int mode, float scale, int causal,
                       int dtype, void* stream);

/*
 * fa_kvcache_evict — cuts every sequence of a cache to its budget, for each KV
 * head by itself.  Of a sequence of n = seqlens_k[b] > keep positions (keep[b], an
 * int32 DEVICE array, or keep_all for all where keep is NULL; negative: 0) stay
 * the first f = min(first, keep), the last r = min(recent, keep - f) and, of those
 * between, the keep - f - r with the largest weights (equal weights: the lower
 * position; a NaN is less than every number).  Their rows of K and V, scales and
 * weights move together in order of position to positions 0 .. keep - 1, in place;
 * what lies behind is left as it is.  new_lens[b] (int32 DEVICE array, not
 * seqlens_k) = min(n, keep).  `weights` as in fa_kvcache_weights, with weights_len >=
 * max_pages * page_size.  No page may belong to two sequences, nor twice to one.
 * Rows without a page read as zeros, and are not written.  Asynchronous on `stream`.
 *
 * No reference counterpart (reference llama_attention_replacement.py:63-65).
 */
int fa_kvcache_evict(const fa_paged_cache* cache, float* weights, long long w_seq_stride,
                     long long w_head_stride, int weights_len, const int* seqlens_k,
                     const int* keep, int keep_all, int first, int recent, int* new_lens, int B,
                     void* stream);

/* ---- reference-compatible launchers (void, fp16, blocking) ----
 * Same signatures and conventions as the reference: errors are printed to
 * stderr, the work runs on the legacy default stream and the call ends with
 * cudaDeviceSynchronize(). */

/* reference src/kernels/flash_attention_forward.cu:795-817 */
void launch_flash_attention_forward(const void* Q, const void* K, const void* V, void* O,
                                    int batch, int heads, int seq_len, int head_dim, float scale,
                                    bool causal);
/* reference src/kernels/flash_attention_forward.cu:819-833 (d=64 only) */
void launch_flash_attention_forward_scalar(const void* Q, const void* K, const void* V, void* O,
                                           int batch, int heads, int seq_len, int head_dim,
                                           float scale, bool causal);
/* reference src/kernels/flash_attention_forward.cu:835-849 (d=64 only) */
void launch_flash_attention_forward_wmma_qk(const void* Q, const void* K, const void* V, void* O,
                                            int batch, int heads, int seq_len, int head_dim,
                                            float scale, bool causal);
/* reference src/kernels/naive_attention.cu:115-164; workspace holds
 * batch*heads*seq_len*seq_len floats (the materialised score matrix). */
void launch_naive_attention(const void* Q, const void* K, const void* V, void* O, int batch,
                            int heads, int seq_len, int head_dim, float scale, bool causal,
                            float* workspace);

/* Stream-ordered form of launch_naive_attention used by the Python binding
 * (same math, no device synchronisation, returns a status code). */
int fa_naive_fwd(const void* Q, const void* K, const void* V, void* O, int batch, int heads,
                 int seq_len, int head_dim, float scale, int causal, float* workspace,
                 void* stream);

/* fa_naive_fwd_noalloc — the materialised attention of fa_naive_fwd for
 * callers that cannot allocate device memory while they run: hosts whose
 * allocator is closed after start-up, real-time or embedded loops, runtimes
 * that own all device memory and forbid cudaMalloc from libraries.  It has no
 * counterpart in the reference (the reference's binding allocates the
 * workspace with torch::empty per call, pytorch_extension.cpp:37-40).
 *   - The score workspace is a file-scope device array of 4Mi floats
 *     (16 MiB), so batch*heads*seq_len*seq_len must be <= 4194304; larger
 *     problems return FA_ERR_SCRATCH_LIMIT and launch nothing.  Every GPU that
 *     loads this library holds those 16 MiB until the process exits.
 *   - Nothing is allocated or freed: no cudaMalloc/cudaFree, no allocating
 *     library call.  Every call looks up the array's device address
 *     (cudaGetSymbolAddress) for the calling thread's current device, so the
 *     address stays right after a cudaDeviceReset; the first call on a device
 *     may also load this library's module there, so make that first call
 *     before any stream capture on the device.
 *   - All calls on a device share the one array and it keeps the last call's
 *     contents (every score is rewritten before it is read, so nothing needs
 *     clearing).  Calls whose work overlaps on the GPU race on the array:
 *     order them on one stream or synchronise between them.
 * Arguments, layout (fp16), stream semantics and results as fa_naive_fwd. */
int fa_naive_fwd_noalloc(const void* Q, const void* K, const void* V, void* O, int batch,
                         int heads, int seq_len, int head_dim, float scale, int causal,
                         void* stream);

/* ---- standalone-kernel launchers ----
 * reference flash-attention-sm75-fused/src/flash_mha_flatargs.cu:231-252
 * (full attention, d = 64).  Asynchronous on `stream`. */
int flatargs_launch(const void* Q, const void* K, const void* V, void* O, int B, int H, int N,
                    float scale, void* stream);
/* reference flash-attention-sm75-fused/src/flash_mha_v2.cu:366-392
 * (d = 64; mode 0 = FULL, 1 = CAUSAL).  Asynchronous on `stream`. */
int launch_v2(const void* Q, const void* K, const void* V, void* O, int B, int H, int N,
              float scale, int mode, void* stream);

/* ---- diagnostics ---- */
/* Error code recorded by the device watchdog on the current device (0 if
 * none); `reset` clears it.  Synchronous (reads device memory). */
int fa_device_status(int reset);
/* Watchdog deadline for every in-kernel wait, in ns (default 1e9). */
void fa_set_watchdog_ns(unsigned long long ns);
/* FA_DEBUG_* bits applied to subsequent launches (tests only; default 0). */
void fa_set_debug_flags(int flags);
/* Development hook: device buffer (8*64*32 int64) that builds compiled with
 * FA_TRACE fill with per-tile clock64() samples; NULL disables.  No effect in
 * regular builds. */
void fa_set_trace_buffer(void* buf);
/* Human-readable text for a status code. */
const char* fa_error_string(int code);
/* Dynamic shared memory one CTA of the kernel uses for this head_dim. */
int fa_smem_bytes(int head_dim);
/* Library version string. */
const char* fa_version(void);

#ifdef __cplusplus
}
#endif

#endif /* FA_B200_H */
