"""Paged KV cache on the GPU: writing, reading back and attention against
plain 64-bit forms (tests/paged_plain.py, which derives the tolerances), through
the Python API and the C ABI.

Every cache row that no sequence owns holds NaN (8-bit pages: NaN scales and
the byte 0x7f, an e4m3 NaN), and the block table's unused entries point outside
the cache, so a kernel that lets either into a result fails.
"""
import math

import pytest
import torch

import flash_attention_sm75 as fa
from tests import abi_ctypes as abi
from tests.paged_plain import QMAX, UNIT, Paged, attention, bits, quantise

pytestmark = pytest.mark.gpu

F16, BF16, I8, E4M3 = torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn


def _attend(P, q, Hq, mode, c=None, slack=0, **kw):
    c = c or P.cuda()
    max_q = max([m for m, _ in P.lens] + [0]) + slack
    max_k = max([n for _, n in P.lens] + [0]) + slack
    return fa.flash_attention_forward_paged(
        q.cuda() if not q.is_cuda else q, c["k_cache"], c["v_cache"], c["table"], c["cu"], c["lens"],
        max_q, max_k, causal=mode != 0, causal_alignment="top_left" if mode == 2 else "bottom_right",
        k_scale=c["k_scale"], v_scale=c["v_scale"], return_lse=True, **kw)


def _check(P, q, Hq, mode, got, scale=None):
    o, lse, tol, tol_lse = attention(P, q, Hq, mode, scale)
    go, gl = got[0].double().cpu(), got[1].double().cpu()
    assert torch.isfinite(go).all()
    bad = (go - o).abs() > tol
    assert not bad.any(), ((go - o).abs() / tol.clamp(min=1e-12)).max().item()
    fin = torch.isfinite(lse)
    assert torch.equal(gl == -math.inf, ~fin)
    assert ((gl - lse).abs()[fin] <= tol_lse[fin]).all(), (gl - lse).abs()[fin].max().item()
    assert (go[(~fin).T] == 0).all()


# lengths (new, cached), query heads, KV heads, d, page
ATTEND = [
    ([(1, 1)], 1, 1, 64, 16),
    ([(1, 300)], 32, 8, 128, 16),
    ([(1, 17), (1, 1), (1, 500), (0, 40), (1, 64), (1, 0)], 8, 2, 128, 16),
    ([(1, 1000), (3, 777), (2, 33)], 6, 2, 64, 48),              # 3 heads a group, page 48
    ([(4, 129), (4, 640), (4, 4)], 8, 2, 128, 32),               # 16 rows a KV head
    ([(2, 90), (1, 411)], 14, 2, 64, 16),                        # 7 heads a group
    ([(5, 60), (17, 200), (1, 900)], 4, 4, 128, 64),
    ([(40, 40), (3, 3), (129, 300)], 4, 1, 64, 16),
    ([(64, 64)], 8, 1, 128, 128),
    ([(300, 513), (1, 700), (0, 0), (33, 33)], 8, 2, 128, 16),
    ([(513, 513), (20, 1500)], 6, 1, 128, 48),                   # 6 heads a group
    ([(50, 20), (7, 3)], 4, 2, 64, 16),                          # more new tokens than cached
    ([(260, 700)], 5, 5, 64, 256),
    ([(9, 2000), (1, 2500)], 40, 1, 128, 16),                    # 40 heads a group
]


@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("kind", [(F16, F16), (BF16, BF16), (F16, I8), (BF16, E4M3)],
                         ids=["f16", "bf16", "f16-int8", "bf16-e4m3"])
@pytest.mark.parametrize("case", ATTEND, ids=[str(i) for i in range(len(ATTEND))])
def test_attention_matches_plain(sm100, case, kind, mode):
    lens, Hq, Hkv, d, page = case
    io, cache = kind
    order = "token" if (len(lens) + mode) % 2 else "head"
    P = Paged(lens, Hkv, d, page, cache, io=io, order=order, seed=len(lens) + 7 * mode)
    q = P.new(Hq)
    _check(P, q, Hq, mode, _attend(P, q, Hq, mode))
    assert abi.load().fa_device_status(1) == 0


@pytest.mark.parametrize("kind", [(BF16, I8), (F16, E4M3), (BF16, BF16)],
                         ids=["bf16-int8", "f16-e4m3", "bf16"])
@pytest.mark.parametrize("nq,nk,G,d", [(1, 9000, 4, 128), (2, 5000, 8, 64), (100, 4100, 4, 128),
                                       (1, 20000, 1, 64), (33, 3000, 3, 128)])
def test_attention_long(sm100, nq, nk, G, d, kind):
    """Key ranges that are split between many warps or CTAs and joined."""
    P = Paged([(nq, nk), (1, 5)], 2, d, 16, kind[1], io=kind[0], seed=nk)
    q = P.new(2 * G)
    _check(P, q, 2 * G, 1, _attend(P, q, 2 * G, 1))


@pytest.mark.parametrize("nq", [1, 40])
@pytest.mark.parametrize("cache", [F16, I8])
def test_attention_large_and_growing_scores(sm100, nq, cache):
    """Keys whose scores climb along the cache (the running maximum grows late)
    and large logits; a negative scale."""
    P = Paged([(nq, 700), (nq, 130)], 2, 128, 16, cache, seed=3)
    q = P.new(8, spread=3.0)
    ramp = torch.linspace(0.2, 6.0, 700)
    for b, (_, n) in enumerate(P.lens):
        x = torch.randn(n, 2, 128, generator=P.g) * ramp[:n, None, None]
        if cache in QMAX:
            x8, s = quantise(x, cache)
            P.put("k", b, range(n), x8, s)
        else:
            P.put("k", b, range(n), x.half(), None)
    for scale in (None, -0.07, 0.0):
        _check(P, q, 8, 1, _attend(P, q, 8, 1, scale=scale), scale)


@pytest.mark.parametrize("nq", [1, 40])
@pytest.mark.parametrize("cache", [I8, E4M3])
def test_attention_scales_of_very_different_size(sm100, nq, cache):
    """Value rows whose scales span six decades, with an all-zero row: what a
    small row adds is held to the size of the rows around it."""
    P = Paged([(nq, 400)], 1, 64, 16, cache, seed=5)
    mult = 10.0 ** (torch.arange(400) % 7 - 3).double()
    x = (torch.randn(400, 1, 64, generator=P.g) * mult[:, None, None].float()).half().float()
    x[13] = 0
    x8, s = quantise(x, cache)
    P.put("v", 0, range(400), x8, s)
    q = P.new(4)
    _check(P, q, 4, 1, _attend(P, q, 4, 1))


@pytest.mark.parametrize("nq", [1, 40])
def test_rows_of_no_sequence(sm100, nq):
    """Rows before cu_seqlens[0] and after its last entry: O = 0, LSE = -inf;
    looser length bounds than needed change nothing."""
    P = Paged([(nq, 90), (nq, 200)], 2, 64, 16, F16, seed=1, first=3, tail=5)
    q = P.new(4)
    got = _attend(P, q, 4, 1)
    _check(P, q, 4, 1, got)
    again = _attend(P, q, 4, 1, slack=900)
    _check(P, q, 4, 1, again)


@pytest.mark.parametrize("io", [F16, BF16])
def test_expanded_keys_go_head_group_by_head_group(sm100, io):
    """A bound on the lengths whose expanded 8-bit keys would pass 1 GiB for all
    heads: the chunk kernel runs a few heads at a time, with the same result."""
    P = Paged([(150, 700), (90, 90)], 6, 128, 32, I8, io=io, seed=21)
    q = P.new(12)
    c = P.cuda()
    args = (q.cuda(), c["k_cache"], c["v_cache"], c["table"], c["cu"], c["lens"], 150)
    kw = dict(causal=True, k_scale=c["k_scale"], v_scale=c["v_scale"], return_lse=True)
    got = fa.flash_attention_forward_paged(*args, 1 << 18, **kw)
    _check(P, q, 12, 1, got)


def test_single_token_calls_without_workspace(sm100):
    """Short caches: one kernel, also for more (sequence, head) pairs than SMs and
    more ring stages than units."""
    for B, nk, cache in ((1, 300, F16), (40, 90, I8), (70, 512, BF16)):
        io = BF16 if cache == BF16 else F16
        P = Paged([(1, 1 + (nk * (b + 1)) // B) for b in range(B - 1)] + [(1, nk)], 4, 128, 16, cache,
                  io=io, seed=B)
        q = P.new(8)
        _check(P, q, 8, 1, _attend(P, q, 8, 1))


def test_max_seqlen_k_limits_the_keys(sm100):
    """Keys past max_seqlen_k are not seen (no causal rule here)."""
    for nq in (1, 40):
        P = Paged([(nq, 200)], 1, 64, 16, F16, seed=2)
        q = P.new(4)
        c = P.cuda()
        got = fa.flash_attention_forward_paged(q.cuda(), c["k_cache"], c["v_cache"], c["table"], c["cu"],
                                               c["lens"], nq, 100, return_lse=True)
        P.lens = [(nq, 100)]
        _check(P, q, 4, 0, got)


@pytest.mark.parametrize("nq", [1, 3, 60])
def test_missing_pages_read_as_zero_rows(sm100, nq):
    """A table entry outside the cache within a sequence: keys and values of
    zeros (score 0), nothing outside the cache is touched."""
    for cache in (F16, I8):
        P = Paged([(nq, 150)], 2, 64, 16, cache, seed=4)
        q = P.new(8)
        c = P.cuda()
        c["table"][0, 3] = -7
        c["table"][0, 5] = P.pages
        for name in ("k", "v"):
            pos = [p for p in range(150) if p // 16 in (3, 5)]
            z = torch.zeros(len(pos), 2, 64).to(cache)
            P.put(name, 0, pos, z, torch.zeros(len(pos), 2) if cache in QMAX else None)
        _check(P, q, 8, 1, _attend(P, q, 8, 1, c=c))


@pytest.mark.parametrize("nq", [1, 30])
def test_strided_queries_streams_and_repeats(sm100, nq):
    """q as a slice of a wider projection, on a stream of its own; the same
    call again gives the same bits."""
    P = Paged([(nq, 1200), (nq, 77)], 2, 128, 16, BF16, io=BF16, order="token", seed=9)
    wide = (torch.randn(P.total, 12, 128, generator=P.g)).to(BF16).cuda()
    q = wide[:, 2:10]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    c = P.cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        a = _attend(P, q, 8, 1, c=c)
        b = _attend(P, q, 8, 1, c=c)
    st.synchronize()
    _check(P, q.cpu(), 8, 1, a)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_attention_in_a_cuda_graph(sm100):
    """Captured once, replayed on new lengths within the same bounds."""
    P = Paged([(1, 100), (1, 700)], 2, 128, 16, F16, seed=8)
    q = P.new(8)
    c = P.cuda()
    qd = q.cuda()
    call = lambda: fa.flash_attention_forward_paged(  # noqa: E731
        qd, c["k_cache"], c["v_cache"], c["table"], c["cu"], c["lens"], 1, 700, causal=True,
        return_lse=True)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for lens in ([(1, 100), (1, 700)], [(1, 31), (1, 699)]):
        P.lens = lens
        c["lens"].copy_(torch.tensor([n for _, n in lens], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        _check(P, q, 8, 1, out)


# ------------------------------------------------------------------ write and read back

WRITE = [
    ([(1, 1)], 1, 64, 16),
    ([(1, 300), (1, 17), (0, 9), (1, 16)], 8, 128, 16),
    ([(70, 70), (5, 200), (33, 1000)], 2, 64, 48),
    ([(300, 700), (1, 700), (129, 129)], 3, 128, 32),
    ([(6, 4), (2, 90)], 2, 64, 16),                     # two tokens before position 0
]


@pytest.mark.parametrize("order", ["head", "token"])
@pytest.mark.parametrize("kind", [(F16, F16), (BF16, BF16), (F16, I8), (BF16, I8), (F16, E4M3),
                                  (BF16, E4M3)],
                         ids=["f16", "bf16", "f16-int8", "bf16-int8", "f16-e4m3", "bf16-e4m3"])
@pytest.mark.parametrize("case", WRITE, ids=[str(i) for i in range(len(WRITE))])
def test_write_and_read_back(sm100, case, kind, order):
    lens, Hkv, d, page = case
    io, cache = kind
    P = Paged(lens, Hkv, d, page, cache, io=io, order=order, seed=11, first=2, tail=3)
    c = P.cuda()
    kv = torch.randn(P.total, 2 * Hkv + 1, d, generator=P.g)
    kv[0] *= 1e-3
    if P.total > 6:
        kv[5] = 0
    kv = kv.to(io).cuda()
    k, v = kv[:, :Hkv], kv[:, Hkv:2 * Hkv]  # strided slices
    before = {n: c[n].clone() if c[n] is not None else None
              for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    fa.kvcache_write_paged(k, v, c["k_cache"], c["v_cache"], c["table"], c["cu"], c["lens"],
                           k_scale=c["k_scale"], v_scale=c["v_scale"])
    rk, rv = fa.kvcache_read_paged(c["k_cache"], c["v_cache"], c["table"], c["cu"], c["lens"], P.total,
                                   k_scale=c["k_scale"], v_scale=c["v_scale"], dtype=io)
    torch.cuda.synchronize()
    for name, x, back in (("k", k.cpu(), rk.cpu()), ("v", v.cpu(), rv.cpu())):
        pages = c[name + "_cache"].cpu()
        sc = c[name + "_scale"].cpu() if cache in QMAX else None
        want = bits(before[name + "_cache"].cpu()).clone()
        want_s = before[name + "_scale"].cpu().clone() if sc is not None else None
        if sc is not None:
            x8, s = quantise(x, cache)
        stored = torch.zeros(P.total, dtype=torch.bool)
        for b, (m, n) in enumerate(lens):
            for i in range(m):
                p, t = n - m + i, P.cu[b] + i
                if p < 0:
                    continue
                pg, row = P.place(b, p)
                want[pg, :, row] = bits(x8 if sc is not None else x)[t]
                if sc is not None:
                    want_s[pg, :, row] = s[t]
                stored[t] = True
        # the pages hold exactly the defined bits, and nothing else changed
        same = bits(pages) == want if sc is not None else (pages == want) | (pages.isnan() & want.isnan())
        assert same.all()
        if sc is not None:
            assert torch.equal(torch.nan_to_num(sc, nan=-1.0), torch.nan_to_num(want_s, nan=-1.0))
        # read back: within the rounding of 8 bits and of the 16-bit result
        assert (back[~stored] == 0).all()
        y, ref = back[stored].double(), x[stored].double()
        if sc is None:
            assert torch.equal(back[stored], x[stored])
            continue
        a = ref.abs().amax(-1, keepdim=True)
        step = a / 254 if cache == I8 else torch.maximum(ref.abs() * 2 ** -4, a / 448 * 2 ** -10)
        u = UNIT[io]
        floor = 2.0 ** -25 if io == F16 else 0.0  # f16 results below 2^-14 are subnormal
        assert ((y - ref).abs() <= step * (1 + 2 ** -10) + ref.abs() * u + step * u + floor).all()


def test_read_whole_prefixes_feeds_the_varlen_entry(sm100):
    P = Paged([(1, 130), (1, 5), (1, 64)], 2, 64, 16, F16, seed=6)
    c = P.cuda()
    n = [x for _, x in P.lens]
    cu = [0, n[0], n[0] + n[1], sum(n)]
    k, v = fa.kvcache_read_paged(c["k_cache"], c["v_cache"], c["table"], cu, c["lens"], sum(n))
    q = P.new(4)
    o, lse = fa.flash_attention_varlen_forward(q.cuda(), k, v, P.cu, cu, 1, max(n), causal=True,
                                               return_lse=True)
    _check(P, q, 4, 1, (o, lse))
    for b in range(3):
        assert torch.equal(k[cu[b]:cu[b + 1]].cpu().double(), P.held("k", b, n[b]))


@pytest.mark.parametrize("cache", [I8, E4M3])
def test_rows_with_infinities_read_back_as_nan(sm100, cache):
    """A row with an infinity or a NaN reads back as NaN; its neighbours, and
    rows of the smallest values, do not change."""
    P = Paged([(4, 4)], 1, 64, 16, cache, io=BF16, seed=12)
    c = P.cuda()
    x = torch.randn(4, 1, 64, generator=P.g)
    x[1, 0, 7], x[2, 0, 9] = float("inf"), float("nan")
    x[3] = 1e-38
    x = x.to(BF16).cuda()
    fa.kvcache_write_paged(x, x, c["k_cache"], c["v_cache"], c["table"], c["cu"], c["lens"],
                           k_scale=c["k_scale"], v_scale=c["v_scale"])
    k, _ = fa.kvcache_read_paged(c["k_cache"], c["v_cache"], c["table"], c["cu"], c["lens"], 4,
                                 k_scale=c["k_scale"], v_scale=c["v_scale"])
    k = k.float().cpu()
    assert k.dtype == torch.float32 and torch.isfinite(k[0]).all() and (k[3] == 0).all()
    assert k[1].isnan().all() and k[2].isnan().all()


def test_large_cache_offsets_pass_32_bits(sm100):
    """Pages whose element offsets need more than 32 bits (5 GB of pages)."""
    pages, Hkv, page, d = 20000, 8, 128, 128
    kc = torch.empty(pages, Hkv, page, d, dtype=I8, device="cuda")
    vc = torch.empty_like(kc)
    ks = torch.zeros(pages, Hkv, page, device="cuda")
    vs = torch.zeros_like(ks)
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(0)
    x = torch.randn(300, 2 * Hkv, d, generator=g).half()
    xd = x.cuda()
    fa.kvcache_write_paged(xd[:, :Hkv], xd[:, Hkv:], kc, vc, table, [0, 300], [300], k_scale=ks,
                           v_scale=vs)
    k, v = fa.kvcache_read_paged(kc, vc, table, [0, 300], [300], 300, k_scale=ks, v_scale=vs, dtype=F16)
    for got, want in ((k, x[:, :Hkv]), (v, x[:, Hkv:])):
        y, s = quantise(want, I8)
        assert torch.equal(got.cpu(), (y.float() * s.unsqueeze(-1)).half())
    for nq in (1, 40):
        q = torch.randn(nq, 32, d, generator=g).half()
        o = fa.flash_attention_forward_paged(q.cuda(), kc, vc, table, [0, nq], [300], nq, 300, causal=True,
                                             k_scale=ks, v_scale=vs)
        ref = fa.flash_attention_varlen_forward(q.cuda(), k, v, [0, nq], [0, 300], nq, 300, causal=True)
        # two kernels on values of at most ~3, each within 2^-11 relative of the sums they round
        assert (o.float() - ref.float()).abs().max().item() <= 4e-3


# ------------------------------------------------------------------ refusals

def test_refusals(sm100):
    P = Paged([(1, 20), (2, 30)], 2, 64, 16, F16, seed=0)
    c = P.cuda()
    q = P.new(4).cuda()
    kv = P.new(2).cuda()

    def attend(**kw):
        a = dict(q=q, k_cache=c["k_cache"], v_cache=c["v_cache"], block_table=c["table"],
                 cu_seqlens_q=c["cu"], seqlens_k=c["lens"], max_seqlen_q=2, max_seqlen_k=30)
        a.update(kw)
        return fa.flash_attention_forward_paged(**a)

    def write(**kw):
        a = dict(k=kv, v=kv, k_cache=c["k_cache"], v_cache=c["v_cache"], block_table=c["table"],
                 cu_seqlens=c["cu"], seqlens_k=c["lens"])
        a.update(kw)
        return fa.kvcache_write_paged(**a)

    with pytest.raises(ValueError, match="3D"):
        attend(q=q[0])
    with pytest.raises(ValueError, match="4D"):
        attend(k_cache=c["k_cache"][0])
    with pytest.raises(RuntimeError, match="head_dim=64 or 128"):
        attend(k_cache=c["k_cache"][..., :32], v_cache=c["v_cache"][..., :32], q=q[..., :32])
    with pytest.raises(RuntimeError, match="not divisible"):
        attend(q=q[:, :3])
    with pytest.raises(ValueError, match="causal_alignment"):
        attend(causal=True, causal_alignment="middle")
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        attend(q=q.cpu())
    with pytest.raises(RuntimeError, match="FP16 or BF16"):
        attend(q=q.float())
    with pytest.raises(RuntimeError, match="like the rows"):
        attend(q=q.bfloat16())
    with pytest.raises(RuntimeError, match="take none"):
        attend(k_scale=torch.ones(P.pages, 2, 16, device="cuda"),
               v_scale=torch.ones(P.pages, 2, 16, device="cuda"))
    with pytest.raises(RuntimeError, match="need k_scale"):
        attend(k_cache=c["k_cache"].to(I8), v_cache=c["v_cache"].to(I8))
    with pytest.raises(RuntimeError, match="multiple of 16"):
        attend(k_cache=c["k_cache"][:, :, :8], v_cache=c["v_cache"][:, :, :8])
    with pytest.raises(RuntimeError, match="must agree"):
        attend(seqlens_k=c["lens"][:1])
    with pytest.raises(RuntimeError, match="lengths"):
        attend(max_seqlen_q=-1)
    with pytest.raises(RuntimeError, match="128 query heads"):
        attend(q=torch.zeros(3, 258, 64, dtype=F16, device="cuda"))
    odd = torch.zeros(P.pages, 2, 16, 66, dtype=F16, device="cuda")[..., :64]
    with pytest.raises(RuntimeError, match="16 bytes"):
        attend(k_cache=odd, v_cache=odd)
    with pytest.raises(RuntimeError, match="same strides"):
        write(v_cache=c["v_cache"].transpose(1, 2).contiguous().transpose(1, 2))
    with pytest.raises(RuntimeError, match="for these pages"):
        write(k=kv[:, :1], v=kv[:, :1])
    with pytest.raises(RuntimeError, match="share shape"):
        write(v=kv[:, :1])
    with pytest.raises(RuntimeError, match="must be fp32"):
        z = torch.ones(P.pages, 2, 8, device="cuda")
        write(k_cache=c["k_cache"].to(I8), v_cache=c["v_cache"].to(I8), k_scale=z, v_scale=z)
    with pytest.raises(ValueError, match="dtype"):
        fa.kvcache_read_paged(c["k_cache"], c["v_cache"], c["table"], c["cu"], c["lens"], 3,
                              dtype=torch.float32)
    with pytest.raises(RuntimeError, match="count of rows"):
        fa.kvcache_read_paged(c["k_cache"], c["v_cache"], c["table"], c["cu"], c["lens"], -1)


def test_empty_calls(sm100):
    P = Paged([(1, 20)], 2, 64, 16, F16, seed=0)
    c = P.cuda()
    none = torch.empty(0, 4, 64, dtype=F16, device="cuda")
    zero = torch.zeros(2, dtype=torch.int32, device="cuda")
    o, lse = fa.flash_attention_forward_paged(none, c["k_cache"], c["v_cache"], c["table"], zero,
                                              c["lens"], 0, 20, return_lse=True)
    assert o.shape == (0, 4, 64) and lse.shape == (4, 0)
    fa.kvcache_write_paged(none[:, :2], none[:, :2], c["k_cache"], c["v_cache"], c["table"], zero, c["lens"])
    k, v = fa.kvcache_read_paged(c["k_cache"], c["v_cache"], c["table"], zero, c["lens"], 0)
    assert k.shape == v.shape == (0, 2, 64)
    # a batch without sequences: every row is of no sequence
    t0 = torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    e = torch.zeros(0, dtype=torch.int32, device="cuda")
    q = torch.ones(3, 4, 64, dtype=F16, device="cuda")
    o, lse = fa.flash_attention_forward_paged(q, c["k_cache"], c["v_cache"], t0, zero[:1], e, 1, 1,
                                              return_lse=True)
    assert (o == 0).all() and (lse == -math.inf).all()
    k, v = fa.kvcache_read_paged(c["k_cache"], c["v_cache"], t0, zero[:1], e, 2)
    assert (k == 0).all() and (v == 0).all()


@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("kind", [(BF16, BF16), (F16, E4M3)], ids=["bf16", "f16-e4m3"])
def test_key_tiles_of_many_items_in_equal_runs(sm100, kind, mode):
    """A few long sequences between short, empty and keyless ones, more query
    rows than the decode kernel takes: runs that cover several items, items that
    several runs cut, items without keys, pairs whose second tile is empty."""
    lens = [(90, 3000), (0, 0), (70, 70), (300, 100), (129, 129), (65, 5000), (40, 0), (257, 2300)]
    P = Paged(lens, 2, 128, 32, kind[1], io=kind[0], seed=31)
    q = P.new(2 * 2)
    got = _attend(P, q, 4, mode)
    _check(P, q, 4, mode, got)
    again = _attend(P, q, 4, mode)
    assert all(torch.equal(x, y) for x, y in zip(got, again))


def test_one_long_item_cut_by_many_runs(sm100):
    """One KV head, one pair of query tiles, 150 key tiles: parts of a few tiles."""
    P = Paged([(70, 19111)], 1, 64, 64, F16, seed=33)
    q = P.new(1)
    _check(P, q, 1, 1, _attend(P, q, 1, 1))


def test_many_sequences_without_keys(sm100):
    """A batch bound to hold no keys at all: O = 0, LSE = -inf everywhere."""
    P = Paged([(70, 0)] * 200, 2, 64, 16, F16, seed=35)
    q = P.new(4)
    _check(P, q, 4, 0, _attend(P, q, 4, 0))
