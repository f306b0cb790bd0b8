"""Paged KV cache, host side: the C entry points' argument errors and workspace
query (no GPU is touched), and the plain forms that the GPU tests compare with,
pinned against PyTorch's scaled_dot_product_attention."""
import ctypes

import pytest
import torch
import torch.nn.functional as F

from tests import abi_ctypes as abi
from tests.paged_plain import Paged, attention, quantise

P16 = 0x10000  # an aligned address that is never read


def _cache(**kw):
    c = abi.PagedCache()
    c.k = c.v = P16
    c.page_stride, c.head_stride, c.row_stride = 2 * 16 * 64, 16 * 64, 64
    c.block_table, c.table_stride, c.max_pages = P16, 4, 4
    c.num_pages, c.kv_heads, c.page_size, c.head_dim, c.dtype = 9, 2, 16, 64, 0
    for name, x in kw.items():
        setattr(c, name, x)
    return c


def _write(c, total=3, dtype=0, K=P16, ts=128):
    return abi.load().fa_kvcache_write(ctypes.byref(c) if c else None, K, P16, ts, 64, 128, 64, P16, P16,
                                       1, total, dtype, None)


def _read(c, total=3, dtype=0, K=P16):
    return abi.load().fa_kvcache_read(ctypes.byref(c) if c else None, K, P16, P16, P16, 1, total, dtype, None)


def _attend(c, total=3, dtype=0, Q=P16, Hq=4, scale=1.0, causal=1, ws=P16, nbytes=1 << 62, qs=256,
            max_q=3, max_k=64):
    return abi.load().fa_fwd_paged(ctypes.byref(c) if c else None, Q, qs, 64, P16, None, P16, P16, 1, Hq,
                                   total, max_q, max_k, scale, causal, dtype, ws, nbytes, None)


@pytest.mark.parametrize("call", [_write, _read, _attend])
def test_cache_argument_errors(call):
    assert call(None) == 1
    assert call(_cache(head_dim=96)) == 2
    assert call(_cache(dtype=4)) == 5
    assert call(_cache(), dtype=2) == 5
    assert call(_cache(dtype=1), dtype=0) == 5           # 16-bit pages of another type
    assert call(_cache(page_size=0)) == 12
    assert call(_cache(page_size=24)) == 12
    assert call(_cache(kv_heads=0)) == 1
    assert call(_cache(num_pages=-1)) == 1
    assert call(_cache(dtype=2)) == 14                   # 8-bit pages without scales
    assert call(_cache(dtype=3, k_scale=P16)) == 14
    assert call(_cache(k_scale=P16, v_scale=P16)) == 14  # 16-bit pages with scales
    assert call(_cache(k=0)) == 1
    assert call(_cache(block_table=0)) == 1
    assert call(_cache(k=P16 + 8)) == 4
    assert call(_cache(row_stride=65)) == 4
    assert call(_cache(max_pages=1 << 28)) == 10
    assert call(_cache(), total=-1) == 1
    assert call(_cache(), total=1 << 30) == 10
    assert call(_cache(), total=0) == 0                  # nothing to do


def test_call_argument_errors():
    assert _write(_cache(), K=0) == 1
    assert _write(_cache(), K=P16 + 2) == 4
    assert _write(_cache(), ts=65) == 4
    assert _read(_cache(), K=P16 + 2) == 4
    assert _attend(_cache(), Hq=3) == 3
    assert _attend(_cache(), Hq=258) == 13
    assert _attend(_cache(), scale=float("nan")) == 1
    assert _attend(_cache(), causal=3) == 1
    assert _attend(_cache(), Q=0) == 1
    assert _attend(_cache(), qs=260) == 4
    assert _attend(_cache(), ws=0, max_q=99, total=99, max_k=8192) == 1
    assert _attend(_cache(), ws=P16 + 4) == 4
    assert _attend(_cache(), nbytes=0, max_q=99, total=99, max_k=8192) == 1
    assert _attend(_cache(), max_q=-1) == 1
    for code in (12, 13, 14):
        assert abi.load().fa_error_string(code) not in (b"ok", b"unknown error")


def test_workspace_depends_on_sizes_alone():
    f = abi.load().fa_fwd_paged_workspace_bytes
    # a short cache needs none; splits, and chunks over 8-bit pages, do
    for args, some in (((1, 4, 1, 1, 64), False), ((8, 4, 8, 1, 8192), True),
                       ((3, 4, 700, 512, 4096), True), ((0, 4, 5, 1, 1), False)):
        n = f(ctypes.byref(_cache()), *args)
        assert (n > 0) == some
        assert n == f(ctypes.byref(_cache(k=P16 * 2, block_table=P16 * 4)), *args)
    eight = dict(dtype=2, k_scale=P16, v_scale=P16)
    assert f(ctypes.byref(_cache(**eight)), 1, 4, 700, 700, 700) >= 2 * 2 * 768 * 64 * 2
    # a batch whose expanded keys pass 1 GiB goes head by head
    assert f(ctypes.byref(_cache(kv_heads=16, **eight)), 64, 64, 1 << 16, 1024, 1 << 14) < 2 << 30
    # sizes that the call itself refuses: no crash
    for args in ((1, 258, 9, 9, 64), (-1, 4, 9, 9, 64), (1, 4, -9, 9, 64), (1, 4, 9, -1, 64)):
        assert f(ctypes.byref(_cache()), *args) == 0
    assert f(None, 1, 4, 9, 9, 64) == 0 and f(ctypes.byref(_cache(kv_heads=0)), 1, 4, 9, 9, 64) == 0


@pytest.mark.parametrize("mode", [0, 1, 2])
def test_plain_attention_matches_sdpa(mode):
    P = Paged([(5, 37), (1, 16), (9, 9)], 2, 64, 16, torch.float16, seed=mode)
    q = P.new(6)
    o, lse, _, _ = attention(P, q, 6, mode)
    for b, (m, n) in enumerate(P.lens):
        i, j = torch.arange(m)[:, None], torch.arange(n)[None]
        see = torch.ones(m, n, dtype=torch.bool) if mode == 0 else j <= i + (n - m if mode == 1 else 0)
        rows = slice(P.cu[b], P.cu[b + 1])
        k, v = (P.held(x, b, n).repeat_interleave(3, 1).transpose(0, 1) for x in ("k", "v"))
        ref = F.scaled_dot_product_attention(q[rows].double().transpose(0, 1), k, v, attn_mask=see)
        assert (o[rows].transpose(0, 1) - ref).abs().max() < 1e-12


@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
def test_plain_quantise(kind):
    x = torch.randn(50, 64, generator=torch.Generator().manual_seed(1))
    x[3] = 0
    y, s = quantise(x, kind)
    back = y.double() * s.double().unsqueeze(-1)
    a = x.abs().amax(-1, keepdim=True).double()
    step = a / 254 if kind == torch.int8 else torch.maximum(x.abs().double() * 2 ** -4, a / 448 * 2 ** -10)
    assert ((back - x).abs() <= step * (1 + 1e-5)).all()
