"""Paged KV cache on the GPU, at the edges: broadcast tensors, loose and tight
bounds, scales of very different size, large caches, many heads and sequences,
captured graphs, and the C entry points.  Compared with the plain 64-bit forms
and tolerances of tests/paged_plain.py."""
import math

import pytest
import torch

import flash_attention_sm75 as fa
from tests import abi_ctypes as abi
from tests.paged_plain import QMAX, UNIT, Paged, attention, quantise
from tests.test_paged_gpu import BF16, E4M3, F16, I8, _attend, _check

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ broadcast tensors

@pytest.mark.parametrize("nq", [1, 40])
@pytest.mark.parametrize("kind", [(F16, F16), (BF16, BF16), (F16, I8), (BF16, E4M3)],
                         ids=["f16", "bf16", "f16-int8", "bf16-e4m3"])
def test_queries_broadcast_over_heads_and_tokens(sm100, nq, kind):
    """Queries expanded over heads, over tokens, and over both."""
    P = Paged([(nq, 300), (nq, 77)], 2, 64, 16, kind[1], io=kind[0], seed=41)
    one = (torch.randn(P.total, 8, 64, generator=P.g)).to(kind[0]).cuda()
    for q in (one[:, :1].expand(-1, 8, -1), one[:1].expand(P.total, -1, -1),
              one[:1, :1].expand(P.total, 8, -1)):
        _check(P, q.cpu(), 8, 1, _attend(P, q, 8, 1))


@pytest.mark.parametrize("nq", [1, 40])
@pytest.mark.parametrize("kind", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, I8)],
                         ids=["f16", "bf16", "f16-e4m3", "bf16-int8"])
def test_pages_broadcast_over_heads(sm100, nq, kind):
    """One KV head of pages seen as several: attention and reading back."""
    P = Paged([(nq, 300), (nq, 77)], 1, 128, 32, kind[1], io=kind[0], seed=42)
    c = P.cuda()
    for name in ("k_cache", "v_cache"):
        c[name] = c[name].expand(-1, 3, -1, -1)
    for name in ("k_scale", "v_scale"):
        c[name] = None if c[name] is None else c[name].expand(-1, 3, -1)
    q = P.new(6)
    got = _attend(P, q, 6, 1, c=c)
    _check(P, q, 6, 1, got)  # (the same values under one head)
    n = [x for _, x in P.lens]
    k, _ = fa.kvcache_read_paged(c["k_cache"], c["v_cache"], c["table"], [0, n[0], sum(n)], c["lens"], sum(n),
                                 k_scale=c["k_scale"], v_scale=c["v_scale"], dtype=kind[0])
    want = torch.cat([P.held("k", b, n[b]) for b in range(2)]).float().to(kind[0])
    assert torch.equal(k.cpu(), want.expand(-1, 3, -1))


@pytest.mark.parametrize("nq", [1, 40])
def test_pages_broadcast_over_pages(sm100, nq):
    """One page seen as several."""
    P = Paged([(nq, 16)], 2, 64, 16, F16, seed=43, spare=0)
    c = P.cuda()
    c["k_cache"], c["v_cache"] = c["k_cache"].expand(9, -1, -1, -1), c["v_cache"].expand(9, -1, -1, -1)
    c["table"] = torch.tensor([[0, 7, 3, 8, -1, 2]], dtype=torch.int32, device="cuda")
    c["lens"].fill_(90)
    P.table, P.lens = torch.tensor([[0, 0, 0, 0, 1, 0]], dtype=torch.int32), [(nq, 90)]
    P.k, P.v = (torch.cat([x, torch.zeros_like(x)]) for x in (P.k, P.v))  # (no page: zeros)
    q = P.new(4)
    _check(P, q, 4, 1, _attend(P, q, 4, 1, c=c))


def test_new_rows_broadcast_into_the_cache(sm100):
    """New keys and values expanded over heads are written as any others."""
    P = Paged([(5, 40), (3, 3)], 4, 64, 16, F16, seed=44)
    c = P.cuda()
    x = torch.randn(P.total, 1, 64, generator=P.g).half().cuda()
    fa.kvcache_write_paged(x.expand(-1, 4, -1), x.expand(-1, 4, -1), c["k_cache"], c["v_cache"], c["table"],
                           c["cu"], c["lens"])
    for got in fa.kvcache_read_paged(c["k_cache"], c["v_cache"], c["table"], c["cu"], c["lens"], P.total):
        assert torch.equal(got, x.expand(-1, 4, -1))


def test_writes_into_broadcast_pages_are_refused(sm100):
    P = Paged([(2, 20)], 1, 64, 16, I8, seed=45)
    c = P.cuda()
    x = P.new(2).cuda()

    def write(heads_c, heads_s, x):
        fa.kvcache_write_paged(x, x, c["k_cache"].expand(-1, heads_c, -1, -1), c["v_cache"].expand(-1, heads_c, -1, -1),
                               c["table"], c["cu"], c["lens"], k_scale=c["k_scale"].expand(-1, heads_s, -1),
                               v_scale=c["v_scale"].expand(-1, heads_s, -1))

    with pytest.raises(RuntimeError, match="pages that are written"):
        write(2, 2, x)
    own = [c[n].expand(-1, 2, -1, -1).contiguous() for n in ("k_cache", "v_cache")]
    c["k_cache"], c["v_cache"] = own
    with pytest.raises(RuntimeError, match="scales that are written"):
        fa.kvcache_write_paged(x, x, *own, c["table"], c["cu"], c["lens"], k_scale=c["k_scale"].expand(-1, 2, -1),
                               v_scale=c["v_scale"].expand(-1, 2, -1))
    row = torch.zeros(3, 2, 1, 64, dtype=F16, device="cuda").expand(-1, -1, 16, -1)
    with pytest.raises(RuntimeError, match="rows of a page"):
        fa.flash_attention_forward_paged(x, row, row, c["table"], c["cu"], c["lens"], 2, 20)


# ------------------------------------------------------------------ lengths and their bounds

@pytest.mark.parametrize("nq", [1, 40])
@pytest.mark.parametrize("cache", [F16, I8], ids=["f16", "int8"])
def test_loose_bounds_cost_no_memory(sm100, nq, cache):
    """Bounds far above what the batch and its table can hold."""
    P = Paged([(nq, 300), (nq, 77)], 2, 128, 16, cache, seed=50)
    q = P.new(8).cuda()
    c = P.cuda()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = fa.flash_attention_forward_paged(q, c["k_cache"], c["v_cache"], c["table"], c["cu"], c["lens"], 1 << 30,
                                           1 << 30, causal=True, k_scale=c["k_scale"], v_scale=c["v_scale"],
                                           return_lse=True)
    assert torch.cuda.max_memory_allocated() - before < 256 << 20
    _check(P, q.cpu(), 8, 1, got)


@pytest.mark.parametrize("io", [F16, BF16])
def test_wide_tables_go_head_group_by_head_group(sm100, io):
    """A table whose sequences' expanded 8-bit keys would pass 1 GiB for all heads: the
    chunk kernel runs a few heads at a time."""
    P = Paged([(150, 700), (90, 90)], 6, 128, 32, I8, io=io, seed=21)
    q = P.new(12)
    c = P.cuda()
    wide = torch.full((2, 1 << 13), -1, dtype=torch.int32, device="cuda")
    wide[:, :c["table"].size(1)] = c["table"]
    got = fa.flash_attention_forward_paged(q.cuda(), c["k_cache"], c["v_cache"], wide, c["cu"], c["lens"], 150,
                                           1 << 18, causal=True, k_scale=c["k_scale"], v_scale=c["v_scale"],
                                           return_lse=True)
    _check(P, q, 12, 1, got)


def _plain_rows(P, q, Hq, limits):
    """O and LSE in 64 bits where token i of sequence b sees its keys j < limits[b][i]."""
    o = torch.zeros(P.total, Hq, P.d, dtype=torch.float64)
    lse = torch.full((Hq, P.total), -math.inf, dtype=torch.float64)
    for b, lim in enumerate(limits):
        for i, n in enumerate(lim):
            if n <= 0:
                continue
            t = P.cu[b] + i
            k, v = (P.held(x, b, n).repeat_interleave(Hq // P.Hkv, 1).transpose(0, 1) for x in ("k", "v"))
            s = (k @ q[t].double().unsqueeze(-1)).squeeze(-1) / math.sqrt(P.d)
            lse[:, t] = torch.logsumexp(s, -1)
            o[t] = (torch.softmax(s, -1).unsqueeze(1) @ v).squeeze(1)
    return o, lse


def _close(got, want, io):
    """Values of a few units: P and O are each rounded once to 11 or 8 bits, and the
    exponential is good to 1e-4; |V| and |O| stay below 6 here."""
    o, lse = want
    assert (got[0].double().cpu() - o).abs().max() <= 6 * (3 * UNIT[io] + 2e-4)
    fin = torch.isfinite(lse)
    gl = got[1].double().cpu()
    assert torch.equal(gl == -math.inf, ~fin) and (gl - lse).abs()[fin].max() <= 2e-4
    assert (got[0].cpu()[(~fin).T] == 0).all()


@pytest.mark.parametrize("nq", [1, 5, 40])
@pytest.mark.parametrize("kind", [(F16, F16), (BF16, BF16)], ids=["f16", "bf16"])
def test_key_bounds_do_not_move_the_causal_rule(sm100, nq, kind):
    """Keys that max_seqlen_k or the table's width leaves out are not seen; which of the
    others a token sees goes by its own position."""
    P = Paged([(nq, 200), (nq, 60)], 2, 64, 16, kind[1], io=kind[0], seed=51)
    q = P.new(4)
    c = P.cuda()

    def limits(most):
        return [[min(n - nq + i + 1, most) for i in range(nq)] for n in (200, 60)]

    def call(table, max_k):
        return fa.flash_attention_forward_paged(q.cuda(), c["k_cache"], c["v_cache"], table, c["cu"], c["lens"],
                                                nq, max_k, causal=True, return_lse=True)

    _close(call(c["table"], 170), _plain_rows(P, q, 4, limits(170)), kind[0])
    _close(call(c["table"][:, :11], 200), _plain_rows(P, q, 4, limits(176)), kind[0])


@pytest.mark.parametrize("B,nq", [(3, 4), (2, 90), (40, 3)])
def test_rows_beyond_max_seqlen_q(sm100, B, nq):
    """Tokens past max_seqlen_q are not computed: O = 0, LSE = -inf; the others' results
    are those of the whole call."""
    P = Paged([(nq, 100 + b) for b in range(B)], 2, 64, 16, F16, seed=52, first=1, tail=2)
    q = P.new(8)
    c = P.cuda()
    full = _attend(P, q, 8, 1)
    for most in (nq - 1, 1, 0):
        junk = [torch.full((P.total, 8, 64), float("nan"), dtype=F16, device="cuda") for _ in range(3)]
        del junk  # (memory that a result may get is not zero)
        o, lse = fa.flash_attention_forward_paged(q.cuda(), c["k_cache"], c["v_cache"], c["table"], c["cu"],
                                                  c["lens"], most, 200, causal=True, return_lse=True)
        i = torch.arange(P.total, device="cuda") - 1
        keep = (i >= 0) & (i < B * nq) & (i % nq < most)
        assert (o[~keep] == 0).all() and (lse[:, ~keep] == -math.inf).all()
        # (other kernels may take the shorter sequences: two roundings of P and O, values below 6)
        assert keep.sum() == B * most
        if most:
            assert (o[keep].float() - full[0][keep].float()).abs().max() <= 6 * 6 * UNIT[F16]


def test_rows_beyond_max_seqlen_q_in_a_mixed_batch(sm100):
    """The same where both kernels run: a chunk is cut, single tokens are whole."""
    lens = [(300, 400), (1, 50), (2, 60), (250, 250)]
    P = Paged(lens, 2, 64, 16, F16, seed=53)
    q = P.new(8)
    c = P.cuda()
    full = _attend(P, q, 8, 1)
    junk = [torch.full((P.total, 8, 64), float("nan"), dtype=F16, device="cuda") for _ in range(3)]
    del junk
    o, lse = fa.flash_attention_forward_paged(q.cuda(), c["k_cache"], c["v_cache"], c["table"], c["cu"], c["lens"],
                                              200, 400, causal=True, return_lse=True)
    keep = torch.cat([torch.arange(m) < 200 for m, _ in lens]).cuda()
    assert (o[~keep] == 0).all() and (lse[:, ~keep] == -math.inf).all()
    assert (o[keep].float() - full[0][keep].float()).abs().max() <= 6 * 6 * UNIT[F16]


# ------------------------------------------------------------------ scales of very different size

def _check_relative(P, q, Hq, mode, got):
    """_check without an absolute term, for 8-bit pages whose keys and queries are used
    exactly: with A = sum p |v| an element of O is off by at most
        u_out |O| + A (2 u + 4e-4),   u = 2^-11 (P is f16; the exponential, the scores in fp32),
    and by P's smallest step: p times a row's scale is an f16 relative to a largest one
    W = max_j p_j scale_j, good to 2^-25 W, so 2^-25 W sum_j |v_j / scale_j| (and half a step of
    f16 results below 2^-14)."""
    d, io = P.d, P.io
    go, gl = got[0].double().cpu(), got[1].double().cpu()
    assert torch.isfinite(go).all()
    for b, (m, n) in enumerate(P.lens):
        rows = slice(P.cu[b], P.cu[b + 1])
        k, v = (P.held(x, b, n).repeat_interleave(Hq // P.Hkv, 1).transpose(0, 1) for x in ("k", "v"))
        pos = torch.arange(n)
        vs = P.vs[P.table[b].long()[pos // P.page], :, pos % P.page].double()
        vs = vs.repeat_interleave(Hq // P.Hkv, 1).transpose(0, 1)              # [Hq, n]
        s = q[rows].double().transpose(0, 1) @ k.transpose(1, 2) / math.sqrt(d)
        see = torch.arange(n)[None] <= torch.arange(m)[:, None] + n - m if mode else torch.ones(m, n, dtype=bool)
        s = s.masked_fill(~see, -math.inf)
        z = torch.logsumexp(s, -1)
        p = torch.exp(s - z[..., None])
        o, a = p @ v, p @ v.abs()
        w = (p * vs[:, None]).amax(-1, keepdim=True)
        v8 = (v / vs.clamp(min=1e-300)[..., None]).abs()
        steps = w * (see.double() @ v8)
        tol = UNIT[io] * o.abs() + a * (2 * UNIT[F16] + 4e-4) + 2.0 ** -25 * steps
        if io == F16:
            tol = tol + 2.0 ** -25
        off = (go[rows].transpose(0, 1) - o).abs()
        assert (off <= tol).all(), (off / tol).max().item()
        assert ((gl[:, rows] - z).abs() <= 1e-4 + z.abs() * 2.0 ** -20).all()


@pytest.mark.parametrize("nq", [1, 6, 40])
@pytest.mark.parametrize("kind", [(F16, I8), (F16, E4M3), (BF16, I8), (BF16, E4M3)],
                         ids=["f16-int8", "f16-e4m3", "bf16-int8", "bf16-e4m3"])
@pytest.mark.parametrize("late", [True, False], ids=["late", "early"])
def test_small_value_row_takes_the_weight(sm100, nq, kind, late):
    """A key whose value row is millions of times smaller than others' takes nearly all
    the weight, behind the large ones and before them, alone and within one tile."""
    io, cache = kind
    P = Paged([(nq, 700), (nq, 90)], 1, 64, 16, cache, io=io, seed=61)
    q0 = torch.randn(64, generator=P.g)
    q = (q0 + 0.01 * torch.randn(P.total, 4, 64, generator=P.g)).to(io)
    big, small = (3e3, 2e-3) if io == F16 else (1e7, 1e-6)
    for b, (_, n) in enumerate(P.lens):
        k = torch.randn(n, 1, 64, generator=P.g) * 0.1
        v = torch.randn(n, 1, 64, generator=P.g) * small
        at = n - nq - 5 if late else 3
        other = 20 if late else n - nq - 9
        k[at, 0] = q0 * 8          # its score is about 64 above the others'
        v[other] = torch.randn(1, 64, generator=P.g) * big
        v[at + 1] = torch.randn(1, 64, generator=P.g) * big
        for name, x in (("k", k), ("v", v)):
            P.put(name, b, range(n), *quantise(x, cache))
    _check_relative(P, q, 4, 1, _attend(P, q, 4, 1))


@pytest.mark.parametrize("nq", [1, 40])
@pytest.mark.parametrize("cache", [I8, E4M3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("size", [2e-30, 1e-20, 1e-7, 1e-4, 1e6, 1e20, 1e36])
def test_bf16_results_hold_their_range(sm100, nq, cache, size):
    """Values (and keys, with queries to match) far outside f16's range."""
    P = Paged([(nq, 300), (nq, 50)], 2, 128, 16, cache, io=BF16, seed=62)
    for b, (_, n) in enumerate(P.lens):
        for name in ("k", "v"):
            P.put(name, b, range(n), *quantise(torch.randn(n, 2, 128, generator=P.g) * size, cache))
    q = P.new(8, spread=1 / size)
    _check_relative(P, q, 8, 1, _attend(P, q, 8, 1))


@pytest.mark.parametrize("nq", [1, 40])
def test_lse_over_8_bit_pages_is_held_in_32_bits(sm100, nq):
    """Scores come from the stored bits and their fp32 scales: the LSE of bf16 results is
    as good as that of f16 ones."""
    for io in (F16, BF16):
        for cache in (I8, E4M3):
            P = Paged([(nq, 2000)], 2, 128, 32, cache, io=io, seed=63)
            q = P.new(8)
            gl = _attend(P, q, 8, 1)[1].double().cpu()
            lse = attention(P, q, 8, 1)[1]
            # one exponential is good to 2^-13 at worst (its approximation's error has both
            # signs over the sum), fp32 sums and scores to 1e-6: 2e-5 is a tenth of what f16 keys cost
            assert (gl - lse).abs().max() <= 2e-5


# ------------------------------------------------------------------ many heads, many sequences, large caches

@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("kind", [(F16, F16), (BF16, BF16), (F16, I8), (BF16, E4M3)],
                         ids=["f16", "bf16", "f16-int8", "bf16-e4m3"])
@pytest.mark.parametrize("G,d", [(64, 64), (65, 128), (100, 64), (128, 128), (128, 64)])
def test_groups_up_to_128_heads(sm100, G, d, kind, mode):
    """Query tiles of one token (more than 64 heads per KV head), full and not, and of two."""
    P = Paged([(1, 150), (5, 5), (0, 9), (2, 300), (1, 0)], 2, d, 16, kind[1], io=kind[0], seed=71)
    q = P.new(2 * G)
    _check(P, q, 2 * G, mode, _attend(P, q, 2 * G, mode))


def test_one_token_of_128_heads(sm100):
    """A decode step with a full one-token tile, keys split between many CTAs."""
    P = Paged([(1, 6000)], 1, 128, 64, BF16, io=BF16, seed=72)
    q = P.new(128)
    _check(P, q, 128, 1, _attend(P, q, 128, 1))


@pytest.mark.parametrize("cache", [F16, I8], ids=["f16", "int8"])
@pytest.mark.parametrize("B", [33, 100, 1500])
def test_write_and_read_many_sequences(sm100, B, cache):
    """More sequences than one warp looks at at once, some of them without tokens."""
    g = torch.Generator().manual_seed(B)
    new = [int(x) for x in torch.randint(0, 4, (B,), generator=g)]
    new[B // 2:B // 2 + 20] = [0] * len(new[B // 2:B // 2 + 20])
    new[3] = 70
    P = Paged([(m, m + b % 5) for b, m in enumerate(new)], 1, 64, 16, cache, seed=73, first=2, tail=1, poison=False)
    c = P.cuda()
    x = torch.randn(P.total, 2, 64, generator=P.g).half()
    xd = x.cuda()
    fa.kvcache_write_paged(xd[:, :1], xd[:, 1:], c["k_cache"], c["v_cache"], c["table"], c["cu"], c["lens"],
                           k_scale=c["k_scale"], v_scale=c["v_scale"])
    got = fa.kvcache_read_paged(c["k_cache"], c["v_cache"], c["table"], c["cu"], c["lens"], P.total,
                                k_scale=c["k_scale"], v_scale=c["v_scale"], dtype=F16)
    pages = [c["k_cache"].cpu(), c["v_cache"].cpu()]
    inside = torch.zeros(P.total, dtype=torch.bool)
    inside[P.cu[0]:P.cu[-1]] = True
    for kv in range(2):
        want = x[:, kv:kv + 1]
        if cache == I8:
            y, s = quantise(want, I8)
            want = (y.float() * s.unsqueeze(-1)).half()
        back = got[kv].cpu()
        assert torch.equal(back[inside], want[inside]) and (back[~inside] == 0).all()
        for b in (0, 3, 31, 32, B - 1):  # and the right pages hold them
            m, n = P.lens[b]
            for i in range(m):
                pg, row = P.place(b, n - m + i)
                stored = y[P.cu[b] + i] if cache == I8 else want[P.cu[b] + i]
                assert torch.equal(pages[kv][pg, :, row], stored)


@pytest.mark.parametrize("cache", [F16, I8], ids=["f16", "int8"])
def test_byte_offsets_pass_32_bits(sm100, cache):
    """Pages that lie more than 2^32 bytes into each tensor: written, read back, and
    attended over by both kernels."""
    page, Hkv, d = 128, 8, 128
    pages = (1 << 32) // (page * Hkv * d * (1 if cache == I8 else 2)) + 40
    kc = torch.zeros(pages, Hkv, page, d, dtype=cache, device="cuda")
    vc = torch.zeros_like(kc)
    assert (pages - 5) * kc.stride(0) * kc.element_size() > 1 << 32
    s = {n: torch.zeros(pages, Hkv, page, device="cuda") for n in ("k_scale", "v_scale")} if cache == I8 else {}
    table = torch.tensor([[pages - 1, 3, pages - 3], [pages - 2, pages - 5, 7]], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(0)
    n = [300, 270]
    x = torch.randn(sum(n), 2 * Hkv, d, generator=g).half()
    xd = x.cuda()
    cu = [0, n[0], sum(n)]
    fa.kvcache_write_paged(xd[:, :Hkv], xd[:, Hkv:], kc, vc, table, cu, n, **s)
    k, v = fa.kvcache_read_paged(kc, vc, table, cu, n, sum(n), dtype=F16, **s)
    for got, want in ((k, x[:, :Hkv]), (v, x[:, Hkv:])):
        if cache == I8:
            y, sc = quantise(want, I8)
            want = (y.float() * sc.unsqueeze(-1)).half()
        assert torch.equal(got.cpu(), want)
    # the rows' own bytes are where the table says, and nowhere 2^32 bytes before
    assert torch.equal(kc[pages - 1, :, 0].cpu(), (quantise(x[0, :Hkv], I8)[0] if cache == I8 else x[0, :Hkv]))
    assert not kc[39].any() and not kc[35].any()
    for nq in (1, 40):
        q = torch.randn(2 * nq, 32, d, generator=g).half().cuda()
        o = fa.flash_attention_forward_paged(q, kc, vc, table, [0, nq, 2 * nq], n, nq, 300, causal=True, **s)
        ref = fa.flash_attention_varlen_forward(q, k, v, [0, nq, 2 * nq], cu, nq, 300, causal=True)
        # two kernels on values of at most ~3, each within 2^-11 relative of the sums they round
        assert (o.float() - ref.float()).abs().max().item() <= 4e-3


# ------------------------------------------------------------------ captured graphs, C entry points

@pytest.mark.parametrize("kind", [(F16, F16), (BF16, E4M3), (F16, I8)], ids=["f16", "bf16-e4m3", "f16-int8"])
def test_chunks_in_a_cuda_graph(sm100, kind):
    """Captured once, replayed on other lengths and another split of the rows within the same
    bounds: chunks beside single tokens, more keys, fewer rows in use."""
    lens = [(120, 1500), (1, 900), (29, 400)]
    P = Paged(lens, 2, 128, 16, kind[1], io=kind[0], seed=81)
    q = P.new(8)
    c = P.cuda()
    qd = q.cuda()
    call = lambda: fa.flash_attention_forward_paged(  # noqa: E731
        qd, c["k_cache"], c["v_cache"], c["table"], c["cu"], c["lens"], 120, 1500, causal=True,
        k_scale=c["k_scale"], v_scale=c["v_scale"], return_lse=True)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for now in (lens, [(1, 1), (1, 900), (100, 400)], [(0, 3), (2, 2), (3, 3)], [(100, 1500), (20, 20), (30, 31)], lens):
        P.lens = now
        P.cu = [0, now[0][0], now[0][0] + now[1][0], sum(m for m, _ in now)]
        c["lens"].copy_(torch.tensor([n for _, n in now], dtype=torch.int32))
        c["cu"].copy_(torch.tensor(P.cu, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        _check(P, q, 8, 1, out)


@pytest.mark.parametrize("nq", [1, 50])
@pytest.mark.parametrize("kind", [(F16, F16), (BF16, I8)], ids=["f16", "bf16-int8"])
def test_c_entry_points(sm100, nq, kind):
    """The same calls through the C ABI: write, read back, attend."""
    io, cache = kind
    P = Paged([(nq, 170), (nq, nq)], 2, 64, 16, cache, io=io, order="token", seed=91)
    c = P.cuda()
    pc = abi.paged_cache(c["k_cache"], c["v_cache"], c["table"], c["k_scale"], c["v_scale"])
    new = torch.randn(P.total, 5, 64, generator=P.g).to(io)
    nd = new.cuda()
    assert abi.fa_kvcache_write(pc, nd[:, :2], nd[:, 2:4], c["cu"], c["lens"]) == 0
    k, v = (torch.full((P.total, 2, 64), float("nan"), dtype=io, device="cuda") for _ in range(2))
    assert abi.fa_kvcache_read(pc, k, v, c["cu"], c["lens"]) == 0
    for got, name, x in ((k, "k", new[:, :2]), (v, "v", new[:, 2:4])):
        y, s = quantise(x, cache) if cache in QMAX else (x, None)
        for b, (m, n) in enumerate(P.lens):
            rows = slice(P.cu[b], P.cu[b + 1])
            P.put(name, b, range(n - m, n), y[rows], s[rows] if s is not None else None)
        want = (y.float() * s.unsqueeze(-1)).to(io) if s is not None else x
        assert torch.equal(got.cpu(), want)
    q = P.new(6)
    o = torch.full((P.total, 6, 64), float("nan"), dtype=io, device="cuda")
    lse = torch.full((6, P.total), float("nan"), device="cuda")
    for causal in (1, 2):
        assert abi.fa_fwd_paged(pc, q.cuda(), o, lse, c["cu"], c["lens"], nq, 170, causal=causal) == 0
        torch.cuda.synchronize()
        _check(P, q, 6, causal, (o, lse))
    o2 = torch.empty_like(o)
    assert abi.fa_fwd_paged(pc, q.cuda(), o2, None, c["cu"], c["lens"], nq, 170, causal=2) == 0
    assert torch.equal(o, o2) and abi.load().fa_device_status(1) == 0
