"""Shared prefixes, summed weights and eviction, host side: the C entry points'
argument errors and workspace query (no GPU is touched), and the plain forms that the
GPU tests compare with, pinned against other ways to the same values."""
import ctypes
import math

import pytest
import torch

import flash_attention_sm75 as fa
from tests import abi_ctypes as abi
from tests.paged_plain import Paged, attention
from tests.serving_plain import evicted, evicted_whole, prefix_attention, summed_weights, with_prefixes
from tests.test_paged_cpu import P16, _cache

EIGHT = dict(dtype=2, k_scale=P16, v_scale=P16, scale_page_stride=32, scale_head_stride=16, scale_row_stride=1)


def _prefix(c, table=P16, pages=4, n=1, mpq=3, mpk=64, total=3, dtype=0, Q=P16, Hq=4, scale=1.0, causal=1, ws=P16,
            nbytes=1 << 62, qs=256, max_q=3, max_k=64, cup=P16, plens=P16, lse=None):
    return abi.load().fa_fwd_paged_prefix(ctypes.byref(c) if c else None, table, 4, pages, n, cup, plens, mpq, mpk,
                                          Q, qs, 64, P16, lse, P16, P16, 1, Hq, total, max_q, max_k, scale, causal,
                                          dtype, ws, nbytes, None)


def _weights(c, total=3, dtype=0, Q=P16, Hq=4, scale=1.0, causal=1, qs=256, max_q=3, max_k=64, w=P16, ws=256, wh=64,
             L=64, mode=2, lse=P16, cu=P16, B=2):
    return abi.load().fa_kvcache_weights(ctypes.byref(c) if c else None, Q, qs, 64, lse, cu, P16, B, Hq, total,
                                         max_q, max_k, w, ws, wh, L, mode, scale, causal, dtype, None)


def _evict(c, w=P16, ws=256, wh=64, L=64, lens=P16, keep=None, keep_all=8, first=0, recent=0, new=2 * P16, B=2):
    return abi.load().fa_kvcache_evict(ctypes.byref(c) if c else None, w, ws, wh, L, lens, keep, keep_all, first,
                                       recent, new, B, None)


@pytest.mark.parametrize("call", [_prefix, _weights, _evict])
def test_cache_argument_errors(call):
    assert call(None) == 1
    assert call(_cache(head_dim=96)) == 2
    assert call(_cache(dtype=4)) == 5
    assert call(_cache(page_size=24)) == 12
    assert call(_cache(kv_heads=0)) == 1
    assert call(_cache(dtype=2)) == 14                   # 8-bit pages without scales
    assert call(_cache(k_scale=P16, v_scale=P16)) == 14  # 16-bit pages with scales
    assert call(_cache(k=0)) == 1
    assert call(_cache(block_table=0)) == 1
    assert call(_cache(k=P16 + 8)) == 4
    assert call(_cache(row_stride=65)) == 4
    assert call(_cache(row_stride=0)) == 15
    assert call(_cache(max_pages=1 << 28)) == 10


def test_prefix_argument_errors():
    assert _prefix(_cache(), table=0) == 1
    assert _prefix(_cache(), table=P16 + 2) == 4
    assert _prefix(_cache(), pages=-1) == 1
    assert _prefix(_cache(), pages=1 << 28) == 10
    assert _prefix(_cache(), n=-1) == 1
    assert _prefix(_cache(), n=1 << 21) == 10
    assert _prefix(_cache(), cup=0) == 1 and _prefix(_cache(), plens=0) == 1
    assert _prefix(_cache(), cup=P16 + 1) == 4
    for kw in (dict(mpq=-1), dict(mpk=-1), dict(max_q=-1), dict(max_k=-1), dict(causal=3), dict(scale=math.nan),
               dict(Q=0), dict(ws=0), dict(nbytes=0)):
        assert _prefix(_cache(), **kw) == 1, kw
    assert _prefix(_cache(), dtype=2) == 5 and _prefix(_cache(dtype=1), dtype=0) == 5
    assert _prefix(_cache(), Hq=3) == 3 and _prefix(_cache(), Hq=258) == 13
    assert _prefix(_cache(), qs=260) == 4 and _prefix(_cache(), ws=P16 + 4) == 4 and _prefix(_cache(), lse=2) == 4
    assert _prefix(_cache(), qs=-256) == 15
    assert _prefix(_cache(), total=0) == 0               # nothing to do
    # one byte less than the query says
    f = abi.load().fa_fwd_paged_prefix_workspace_bytes
    n = f(ctypes.byref(_cache()), 1, 3, 64, 1, 4, 3, 3, 64)
    assert n >= 3 * 4 * 65 * 4
    assert _prefix(_cache(), nbytes=n - 1) == 1


def test_prefix_workspace_depends_on_sizes_alone():
    f = abi.load().fa_fwd_paged_prefix_workspace_bytes
    plain = abi.load().fa_fwd_paged_workspace_bytes
    for first, second in (((1, 1, 64), (1, 4, 1, 1, 64)), ((2, 40, 8192), (64, 4, 64, 1, 1000)),
                          ((1, 700, 4096), (3, 4, 700, 512, 512)), ((0, 0, 0), (8, 4, 8, 1, 8192))):
        n = f(ctypes.byref(_cache()), *first, *second)
        assert n == f(ctypes.byref(_cache(k=P16 * 2, block_table=P16 * 4)), *first, *second)
        B, Hq, total, max_q, max_k = second
        part = total * Hq * 65 * 4
        passes = (plain(ctypes.byref(_cache()), first[0], Hq, total, first[1], first[2]) +
                  plain(ctypes.byref(_cache()), *second))
        # the results of the first pass, and of the second unless it joins them as it writes
        assert any(0 <= n - passes - x * part < 256 for x in (1, 2))
    for first, second in (((-1, 1, 64), (1, 4, 1, 1, 64)), ((1, -1, 64), (1, 4, 1, 1, 64)),
                          ((1, 1, 64), (1, 258, 9, 9, 64)), ((1, 1, 64), (1, 4, -9, 9, 64)),
                          ((1, 1, -64), (1, 4, 9, 9, 64)), ((1 << 21, 1, 64), (1, 4, 9, 9, 64))):
        assert f(ctypes.byref(_cache()), *first, *second) == 0
    assert f(None, 1, 1, 64, 1, 4, 9, 9, 64) == 0


def test_weights_argument_errors():
    for kw in (dict(mode=-1), dict(mode=3), dict(causal=3), dict(scale=math.inf), dict(max_q=-1), dict(max_k=-1),
               dict(w=0), dict(L=63), dict(L=-1), dict(Q=0), dict(lse=0), dict(cu=0),
               dict(Hq=0)):
        assert _weights(_cache(), **kw) == 1, kw
    assert _weights(_cache(), dtype=2) == 5
    assert _weights(_cache(), Hq=3) == 3 and _weights(_cache(), Hq=258) == 13
    assert _weights(_cache(), qs=260) == 4 and _weights(_cache(), w=P16 + 2) == 4 and _weights(_cache(), lse=P16 + 2) == 4
    assert _weights(_cache(), qs=0) == 15
    # rows of sums that overlap
    assert _weights(_cache(), ws=63) == 15 and _weights(_cache(), wh=0) == 15
    # keys alone: no values and no scales of values
    assert _weights(_cache(v=0), B=0) == 0
    assert _weights(_cache(**{**EIGHT, "v": 0, "v_scale": 0}), B=0) == 0
    assert _weights(_cache(dtype=2, v=0, v_scale=0)) == 14
    # nothing to do; the bound counts no more than the table holds
    assert _weights(_cache(), max_k=0, L=0, w=0) == 0
    assert _weights(_cache(max_pages=0), max_k=1 << 30, L=0, w=0) == 0


def test_evict_argument_errors():
    for kw in (dict(w=0), dict(L=63), dict(lens=0), dict(new=0), dict(new=P16), dict(keep=2 * P16), dict(first=-1),
               dict(recent=-1), dict(B=-1)):
        assert _evict(_cache(), **kw) == 1, kw
    assert _evict(_cache(), w=P16 + 2) == 4 and _evict(_cache(), lens=P16 + 2) == 4
    assert _evict(_cache(), new=2 * P16 + 1) == 4 and _evict(_cache(), keep=P16 + 2) == 4
    assert _evict(_cache(), ws=63) == 15 and _evict(_cache(), wh=0) == 15
    # broadcast pages and scales are not written
    assert _evict(_cache(head_stride=0)) == 15 and _evict(_cache(page_stride=0)) == 15
    assert _evict(_cache(**{**EIGHT, "scale_row_stride": 0})) == 15
    assert _evict(_cache(), B=1 << 21) == 10
    assert _evict(_cache(), B=0) == 0


def test_python_choices_are_checked():
    q = torch.zeros(1, 4, 64)
    with pytest.raises(ValueError, match="mode must be one of"):
        fa.kvcache_weights_paged(q, None, None, None, None, None, 1, 1, None, mode="replace")
    with pytest.raises(ValueError, match="causal_alignment"):
        fa.kvcache_weights_paged(q, None, None, None, None, None, 1, 1, None, causal=True, causal_alignment="left")
    with pytest.raises(ValueError, match="causal_alignment"):
        fa.flash_attention_forward_paged_prefix(q, *[None] * 8, 1, 1, 1, 1, causal=True, causal_alignment="left")


def test_plain_prefix_attention_is_attention_over_both_sets():
    """Prefix pages put before a sequence's own in its table: the same as paged_plain.attention,
    which is pinned against PyTorch's."""
    P = with_prefixes([(5, 37), (1, 16), (9, 9)], [48, 16], 2, 64, 16, torch.float16, seed=1)
    q = P.new(6)
    rows = [P.cu[0], P.cu[2], P.cu[3]]
    for mode in (0, 1):
        o, lse, _, _ = prefix_attention(P, q, 6, rows, mode)
        J = with_prefixes(P.lens[:3], P.prefixes, 2, 64, 16, torch.float16, seed=1)
        J.lens = [(m, n + (48 if b < 2 else 16)) for b, (m, n) in enumerate(P.lens[:3])]
        pages = [[*P.table[3 + (b == 2), :3 if b < 2 else 1].tolist(), *P.table[b].tolist()] for b in range(3)]
        J.table = torch.tensor([(p + [-1] * 3)[:7] for p in pages], dtype=torch.int32)
        o2, lse2, _, _ = attention(J, q, 6, mode)
        assert (o - o2).abs().max() < 1e-12 and (lse - lse2).abs().max() < 1e-12


def test_plain_weights_sum_to_the_rows():
    """Over all keys of a head, the weights of R rows sum to R; and each is the probability's column sum."""
    P = Paged([(5, 37), (1, 16), (3, 2)], 2, 64, 16, torch.float16, seed=2)
    q = P.new(6)
    _, lse, _, _ = attention(P, q, 6, 1)
    old = torch.zeros(3, 2, 48)
    w, _ = summed_weights(P, q, lse, 6, 1, old, "set")
    seen = [(lse[:, P.cu[b]:P.cu[b + 1]] > -math.inf).sum().item() / 2 for b in range(3)]
    assert torch.allclose(w.sum(-1), torch.tensor(seen, dtype=torch.float64)[:, None].expand(3, 2), atol=1e-9)
    assert (w[0, :, 37:] == 0).all()


def test_plain_eviction():
    P = Paged([(0, 20), (0, 5)], 1, 64, 16, torch.float16, seed=3)
    w = torch.zeros(2, 1, 48)
    w[0, 0, :20] = torch.tensor([1, 9, 2, 9, 2, 9, float("nan"), 9, 0, -1, 9, 9, 3, 3, 3, 0, 0, 0, 0, 0])
    k, v, _, _, w2, lens = evicted(P, w, 8, 2, 1)
    assert lens == [8, 5]
    at = [0, 1, 3, 5, 7, 10, 18, 19]  # the first, the five earliest nines, the last two
    assert torch.equal(w2[0, 0, :8], w[0, 0, at])
    for i, j in enumerate(at):
        (pg, row), (dpg, drow) = P.place(0, j), P.place(0, i)
        assert torch.equal(v[dpg, 0, drow], P.v[pg, 0, row])


@pytest.mark.parametrize("call", [_weights, _evict])
def test_rows_of_sums_that_overlap(call):
    """Strides of at least a row, but rows of one sequence on those of another: refused.  One after
    the other, in either order, they are accepted (no work here: no sequences)."""
    for ws, wh in ((64, 64), (100, 64), (64, 100), (127, 64), (64, 127), (1 << 62, 1 << 62)):
        overlap = not (ws >= wh + 64 or wh >= ws + 64)
        assert overlap and call(_cache(kv_heads=2), ws=ws, wh=wh) == 15, (ws, wh)
    assert call(_cache(kv_heads=2), ws=64, wh=64, B=0) == 0
    if not torch.cuda.is_available():  # (the check of the device comes after that of the strides)
        for ws, wh in ((128, 64), (64, 128), (1 << 62, 64)):
            assert call(_cache(kv_heads=2), ws=ws, wh=wh) not in (0, 15), (ws, wh)


def test_weights_of_more_key_blocks_than_a_grid_has():
    """2^20 sequences x 16 heads x 2^16 keys (or one head of 2^30): chunks would take 2^32 blocks of 256
    keys.  Refused before any kernel runs (single tokens come first where a batch has both)."""
    many = dict(B=1 << 20, L=1 << 16, max_k=1 << 16, ws=1 << 40, wh=1 << 17)
    big = dict(kv_heads=16, max_pages=1 << 12)
    assert _weights(_cache(**big), Hq=64, total=3000, max_q=1000, **many) == 10
    assert _weights(_cache(**big), Hq=64, total=1000, max_q=1000, **many) == 10
    one = dict(B=1 << 10, L=1 << 30, max_k=1 << 30, ws=1 << 40, wh=1 << 31)
    assert _weights(_cache(kv_heads=1, max_pages=1 << 26), Hq=4, total=3000, max_q=1000, **one) == 10
    if not torch.cuda.is_available():  # streams of few rows have no such limit (the device is checked afterwards)
        assert _weights(_cache(**big), Hq=64, total=1 << 20, max_q=1, **many) not in (0, 10)


@pytest.mark.parametrize("keep,recent,first", [(64, 10, 2), (1, 0, 0), (0, 3, 3), (150, 400, 20), (299, 0, 1)])
def test_plain_evictions_agree(keep, recent, first):
    """The vectorised form against the one that goes row by row, with every kind of weight."""
    P = Paged([(0, 300), (0, 77), (0, 0)], 2, 64, 16, torch.int8, seed=5)
    g = torch.Generator().manual_seed(keep)
    w = torch.randn(3, 2, P.width * P.page, generator=g)
    r = torch.rand(w.shape, generator=g)
    for i, x in enumerate((0.0, -0.0, 1.5, math.nan, math.inf, -math.inf)):
        w[(r > i / 10) & (r < (i + 1) / 10)] = x
    k, v, ks, vs, w2, _ = evicted(P, w, keep, recent, first)
    got, w3 = evicted_whole(dict(k=P.k, v=P.v, ks=P.ks, vs=P.vs), P.table, w, P.nk, keep, recent, first, P.page)
    assert torch.equal(w2.view(torch.int32), w3.view(torch.int32))
    for a, b in ((got["k"].view(torch.uint8), k), (got["v"].view(torch.uint8), v),
                 (got["ks"].view(torch.int32), ks.view(torch.int32)), (got["vs"].view(torch.int32), vs.view(torch.int32))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("cache", [dict(), EIGHT], ids=["f16", "int8"])
@pytest.mark.parametrize("B,total,max_q", [(64, 64, 1), (4, 2048, 512), (9, 300, 200), (1, 1, 1)])
def test_prefix_workspace_holds_both_passes_at_once(cache, B, total, max_q):
    """The second pass may start while the first still runs: fp32 rows of one pass or of both (d + 1
    numbers for every token and query head, in whole 128 bytes) and both passes' own workspaces."""
    lib, c = abi.load(), _cache(**cache)
    c.max_pages = 1 << 10
    first = lib.fa_fwd_paged_workspace_bytes(ctypes.byref(c), 1, 8, total, total, 8192)
    own = lib.fa_fwd_paged_workspace_bytes(ctypes.byref(c), B, 8, total, max_q, 900)
    rows = -(-total * 8 * 65 * 4 // 128) * 128
    both = lib.fa_fwd_paged_prefix_workspace_bytes(ctypes.byref(c), 1, total, 8192, B, 8, total, max_q, 900)
    assert both - first - own in (rows, 2 * rows)
    assert first > 0
