"""Paged KV cache: writing new tokens, reading them back, attention over it (also
for batches behind shared prefixes), the attention weight its keys receive, and
eviction of those that receive little (no reference counterpart; the reference leaves cached decode to PyTorch SDPA,
llama_attention_replacement.py:63-65).

A cache is a pair of tensors ``[num_pages, H_kv, page_size, D]`` for keys and
values, in any memory order with contiguous rows (token-major pages are passed
as ``pages.transpose(1, 2)``), of fp16 / bf16, or of int8 / float8_e4m3fn with
fp32 scales ``[num_pages, H_kv, page_size]`` (one per token and head, any
strides).  Position ``p`` of sequence ``b`` is row ``p % page_size`` of page
``block_table[b, p // page_size]``.  Pages (and scales) broadcast over heads can
be read and attended over, not written.

The functions describe tokens in the same way: sequence ``b`` has the
packed rows ``[cu_seqlens[b], cu_seqlens[b + 1])``, and the last of them is
position ``seqlens_k[b] - 1``.  A serving step writes its tokens' K and V, then
attends, with one set of ``block_table``, ``cu_seqlens`` and ``seqlens_k``.
"""
import torch

import flash_attn_sm75_cuda as _C

from .ops import _CAUSAL_MODES


# The binding checks the arguments; integer arguments may be tensors of any type
# and device or sequences, and are used in place where they are int32 on the
# inputs' device.


def kvcache_write_paged(k, v, k_cache, v_cache, block_table, cu_seqlens, seqlens_k, k_scale=None,
                        v_scale=None):
    """Store the keys and values of new tokens in a paged cache, in place.

    Args:
        k, v: [total, H_kv, D]  float16 / bfloat16, cuda (slices of a fused
            projection are read in place)
        k_cache, v_cache: [num_pages, H_kv, page_size, D]; 16-bit pages have
            k's dtype, 8-bit pages (int8, float8_e4m3fn) also need
        k_scale, v_scale: fp32 [num_pages, H_kv, page_size], written with them
        block_table: int32 [B, max_pages]
        cu_seqlens: B + 1 row offsets (int32 tensor or ints)
        seqlens_k: B lengths of the sequences including the new tokens

    8-bit rows are scaled by their largest magnitude: x is held as
    round(x * qmax / max|x|) with scale max|x| / qmax, qmax = 127 (int8) or
    448 (e4m3).  Tokens without a place (position below 0 or past the table,
    a table entry outside the cache) are not stored.
    """
    _C.kvcache_write_paged(k, v, k_cache, v_cache, block_table, cu_seqlens,
                           seqlens_k, k_scale, v_scale)


def kvcache_read_paged(k_cache, v_cache, block_table, cu_seqlens, seqlens_k, total, k_scale=None,
                       v_scale=None, dtype=None):
    """Keys and values of a paged cache as packed rows.

    Args:
        k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens,
            seqlens_k: as ``kvcache_write_paged``; cu_seqlens = running sums of
            seqlens_k reads whole sequences
        total: rows of the result (cu_seqlens[-1])
        dtype: torch.float16 or torch.bfloat16 (default: the pages' own type;
            bfloat16 for 8-bit pages)

    Returns:
        k, v: [total, H_kv, D], the layout ``flash_attention_varlen_forward``
        takes.  Rows of tokens without a place, and of no sequence, are zero.
    """
    if dtype is None:
        dtype = k_cache.dtype if k_cache.element_size() == 2 else torch.bfloat16
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"dtype must be torch.float16 or torch.bfloat16, got {dtype}")
    return _C.kvcache_read_paged(k_cache, v_cache, block_table, cu_seqlens,
                                 seqlens_k, total, k_scale, v_scale,
                                 dtype is torch.bfloat16)


def flash_attention_forward_paged(q, k_cache, v_cache, block_table, cu_seqlens_q, seqlens_k,
                                  max_seqlen_q, max_seqlen_k, causal=False, scale=None,
                                  return_lse=False, causal_alignment="bottom_right", k_scale=None,
                                  v_scale=None):
    """Attention of new tokens over a paged cache that holds their own keys
    and values too; forward only.

    Args:
        q: [total_q, H_q, D]  float16 / bfloat16, cuda; H_kv divides H_q
        k_cache, v_cache, k_scale, v_scale, block_table, seqlens_k: as
            ``kvcache_write_paged``
        cu_seqlens_q: B + 1 row offsets of q (int32 tensor or ints); one
            token per sequence, a few, chunks, or any mixture
        max_seqlen_q, max_seqlen_k: upper bounds of the new tokens and of
            seqlens_k (loose ones cost: over 8-bit pages the workspace of a
            chunk grows with B x max_seqlen_k, up to what the table can hold)
        causal, causal_alignment: "bottom_right" (token i of a sequence sees
            keys j <= i + n_k - n_q: the tokens are the cache's last ones) or
            "top_left" (j <= i)
        scale: float (default 1/sqrt(D))
        return_lse: also return LSE [H_q, total_q] fp32 (natural log)

    Rows that see no key, rows of no sequence and tokens beyond max_seqlen_q
    return O = 0, LSE = -inf.
    """
    mode = 0
    if causal:
        mode = _CAUSAL_MODES.get(causal_alignment)
        if mode is None:
            raise ValueError(f"causal_alignment must be one of {sorted(_CAUSAL_MODES)}")
    return _C.flash_attention_forward_paged(q, k_cache, v_cache, block_table, cu_seqlens_q, seqlens_k,
                                            max_seqlen_q, max_seqlen_k, mode, scale, return_lse,
                                            k_scale, v_scale)


def flash_attention_forward_paged_prefix(q, k_cache, v_cache, prefix_table, cu_prefix_q, prefix_lens,
                                         block_table, cu_seqlens_q, seqlens_k, max_prefix_q,
                                         max_prefix_k, max_seqlen_q, max_seqlen_k, causal=False,
                                         scale=None, return_lse=False,
                                         causal_alignment="bottom_right", k_scale=None, v_scale=None):
    """``flash_attention_forward_paged`` of a batch whose sequences share long
    prefixes (a system prompt, a document): each prefix is computed once for all
    the tokens behind it, instead of once per sequence; forward only.

    Args:
        q, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens_q,
            seqlens_k, max_seqlen_q, max_seqlen_k, causal, causal_alignment,
            scale, return_lse: as ``flash_attention_forward_paged``; the block
            table and the lengths are those of what follows the prefix
        prefix_table: int32 [P, max_pages], the pages of the prefixes in the
            same cache
        cu_prefix_q: P + 1 row offsets (int32 tensor or ints): the tokens in
            rows [cu_prefix_q[g], cu_prefix_q[g + 1]) see prefix g; rows
            outside have none
        prefix_lens: P lengths of the prefixes
        max_prefix_q, max_prefix_k: upper bounds of a prefix's tokens and keys
            (tokens beyond do not see it, keys beyond are not seen)

    It pays where many sequences of few tokens share a long prefix, also beside a
    chunk (64 tokens behind 8192 keys: 61 us instead of 135 with the prefix's
    pages at the head of every table; 512 tokens and 31 single ones behind 8192:
    130 / 192).  Tables that begin with the prefix's (whole) pages are faster for a
    few sequences behind a short one (8 behind 1024: 19 / 15), for drafts of d = 64
    behind several (32 x 4 behind three of up to 4096: 41 / 31) and for chunks that
    fill tiles by themselves (8 x 512 behind 8192: 522 to 593 / 498 to 551, from run to
    run; 4 x 512 over e4m3 pages 346 / 325).

    A token sees all keys of its prefix, and those of its own sequence that
    ``causal`` leaves.  Rows that see no key, rows of no sequence and tokens
    beyond max_seqlen_q return O = 0, LSE = -inf.
    """
    mode = 0
    if causal:
        mode = _CAUSAL_MODES.get(causal_alignment)
        if mode is None:
            raise ValueError(f"causal_alignment must be one of {sorted(_CAUSAL_MODES)}")
    return _C.flash_attention_forward_paged_prefix(q, k_cache, v_cache, prefix_table, cu_prefix_q,
                                                   prefix_lens, block_table, cu_seqlens_q, seqlens_k,
                                                   max_prefix_q, max_prefix_k, max_seqlen_q,
                                                   max_seqlen_k, mode, scale, return_lse, k_scale,
                                                   v_scale)


_WEIGHT_MODES = {"set": 0, "add": 1, "append": 2}


def kvcache_weights_paged(q, lse, k_cache, block_table, cu_seqlens_q, seqlens_k, max_seqlen_q,
                          max_seqlen_k, weights, causal=False, scale=None, mode="append",
                          causal_alignment="bottom_right", k_scale=None):
    """Attention weight that cached keys received from new tokens, summed over
    these and over the query heads of a KV head, in place in ``weights``.

    Args:
        q: [total_q, H_q, D]  float16 / bfloat16, cuda
        lse: fp32 [H_q, total_q], what ``flash_attention_forward_paged`` (or
            ``..._paged_prefix``) returned for these queries
        k_cache, k_scale, block_table, cu_seqlens_q, seqlens_k, max_seqlen_q,
            max_seqlen_k, causal, causal_alignment, scale: as that call's (the
            weight of prefix keys: its prefix_table, cu_prefix_q, prefix_lens,
            max_prefix_q and max_prefix_k, with causal=False and mode="add")
        weights: fp32 [B, H_kv, L], L at least max_seqlen_k or the positions of
            a table row, with contiguous rows; weights[b, h, j] is the sum of
            position j of sequence b
        mode: "append" (added to the sums there, but the new tokens' own
            positions, which have none yet, are set), "add" or "set" (all of a
            sequence's positions)

    Positions from a sequence's length (or max_seqlen_k) on are left as they are.
    Chunks (more than 32 query rows per KV head) take a block for every 256 keys that
    max_seqlen_k allows every sequence of the batch, so a bound near the lengths is
    faster, and a chunk beside many long sequences pays for theirs (1024 tokens and 31
    single ones, all over 8192 keys: 242 us; 103 and 83 by themselves).
    """
    if mode not in _WEIGHT_MODES:
        raise ValueError(f"mode must be one of {sorted(_WEIGHT_MODES)}, got {mode!r}")
    rule = 0
    if causal:
        rule = _CAUSAL_MODES.get(causal_alignment)
        if rule is None:
            raise ValueError(f"causal_alignment must be one of {sorted(_CAUSAL_MODES)}")
    _C.kvcache_weights_paged(q, lse, k_cache, block_table, cu_seqlens_q, seqlens_k, max_seqlen_q,
                             max_seqlen_k, weights, rule, scale, _WEIGHT_MODES[mode], k_scale)


def kvcache_evict_paged(k_cache, v_cache, weights, block_table, seqlens_k, keep, recent=0, first=0,
                        k_scale=None, v_scale=None):
    """Cut the sequences of a paged cache to ``keep`` positions, in place, each KV
    head by its own weights; returns the new lengths.

    Args:
        k_cache, v_cache, k_scale, v_scale, block_table, seqlens_k: as
            ``kvcache_write_paged``; no page may belong to two sequences
        weights: fp32 [B, H_kv, L] (``kvcache_weights_paged``), L at least the
            positions of a table row
        keep: positions that stay, one int for all or B of them (of these a
            negative one counts as 0)
        recent, first: the last `recent` and the first `first` positions stay
            whatever their weight (`first` comes first where keep is too small)

    Of the others those of the largest weight stay (equal weights: the lower
    position; a NaN is less than every number).  Keys, values, scales and
    weights of what stays move to positions 0 .. keep - 1 in their order;
    positions behind keep what they hold.

    Returns:
        int32 [B]: min(seqlens_k, keep), the lengths from now on (the next
        tokens are written behind them).
    """
    return _C.kvcache_evict_paged(k_cache, v_cache, weights, block_table, seqlens_k, keep, recent, first,
                                  k_scale, v_scale)
