"""Paged KV cache: writing new tokens, reading them back, and attention over it
(no reference counterpart; the reference leaves cached decode to PyTorch SDPA,
llama_attention_replacement.py:63-65).

A cache is a pair of tensors ``[num_pages, H_kv, page_size, D]`` for keys and
values, in any memory order with contiguous rows (token-major pages are passed
as ``pages.transpose(1, 2)``), of fp16 / bf16, or of int8 / float8_e4m3fn with
fp32 scales ``[num_pages, H_kv, page_size]`` (one per token and head, any
strides).  Position ``p`` of sequence ``b`` is row ``p % page_size`` of page
``block_table[b, p // page_size]``.  Pages (and scales) broadcast over heads can
be read and attended over, not written.

All three functions describe tokens in the same way: sequence ``b`` has the
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
