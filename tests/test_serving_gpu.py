"""Attention behind shared prefixes, summed attention weights and eviction over a
paged cache on the GPU, against plain 64-bit forms (tests/serving_plain.py, which
derives the tolerances).  Cache rows that no sequence owns hold NaN and unused
table entries point outside the cache (tests/paged_plain.py)."""
import math

import pytest
import torch

import flash_attention_sm75 as fa
from tests import abi_ctypes as abi
from tests.paged_plain import QMAX, Paged, attention, bits, quantise
from tests.serving_plain import evicted, prefix_attention, split, summed_weights, with_prefixes

pytestmark = pytest.mark.gpu

F16, BF16, I8, E4M3 = torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn
KINDS = [(F16, F16), (BF16, BF16), (F16, I8), (BF16, E4M3), (BF16, I8)]
KIND_IDS = ["f16", "bf16", "f16-int8", "bf16-e4m3", "bf16-int8"]
NAMES = {1: "bottom_right", 2: "top_left"}


def _rule(mode):
    return dict(causal=mode != 0, causal_alignment=NAMES.get(mode, "bottom_right"))


def _scales(c):
    return dict(k_scale=c["k_scale"], v_scale=c["v_scale"])


# ---------------------------------------------------------------- shared prefixes

def _attend(P, q, rows, mode, c=None, slack=0, max_prefix_q=None, max_prefix_k=None, **kw):
    c = c or P.cuda()
    s = split(P, c)
    lens = P.lens[:P.B]
    mpq = max([b - a for a, b in zip(rows, rows[1:])] + [0]) if max_prefix_q is None else max_prefix_q
    mpk = max(P.prefixes + [0]) if max_prefix_k is None else max_prefix_k
    return fa.flash_attention_forward_paged_prefix(
        q.cuda() if not q.is_cuda else q, c["k_cache"], c["v_cache"], s["prefix_table"],
        torch.tensor(rows, dtype=torch.int32, device="cuda"), s["prefix_lens"], s["table"], s["cu"], s["lens"],
        mpq + slack, mpk + slack, max([m for m, _ in lens] + [0]) + slack, max([n for _, n in lens] + [0]) + slack,
        return_lse=True, **_rule(mode), **_scales(c), **kw)


def _check(P, q, Hq, rows, mode, got, scale=None, **kw):
    o, lse, tol, tol_lse = prefix_attention(P, q, Hq, rows, mode, scale, **kw)
    go, gl = got[0].double().cpu(), got[1].double().cpu()
    assert torch.isfinite(go).all()
    bad = (go - o).abs() > tol
    assert not bad.any(), ((go - o).abs() / tol.clamp(min=1e-12)).max().item()
    fin = torch.isfinite(lse)
    assert torch.equal(gl == -math.inf, ~fin)
    assert ((gl - lse).abs()[fin] <= tol_lse[fin]).all(), (gl - lse).abs()[fin].max().item()
    assert (go[(~fin).T] == 0).all()


# own lengths (new, cached), the sequences where prefixes start and the last one
# ends, prefix lengths, query heads, KV heads, d, page
PREFIX = [
    ([(1, 1)], [0, 1], [40], 1, 1, 64, 16),
    ([(1, 7), (1, 0), (1, 90)], [0, 3], [300], 8, 2, 128, 16),
    ([(1, 20)] * 40, [0, 40], [700], 8, 2, 128, 16),                      # 160 rows a KV head: tiles
    ([(1, 300), (1, 5), (1, 64)] * 9, [0, 5, 20, 27], [513, 1, 200], 16, 2, 64, 32),
    ([(130, 130), (70, 90), (1, 1)], [0, 3], [260], 4, 2, 128, 16),       # chunks in both passes
    ([(2, 5), (0, 9), (200, 200), (3, 0), (1, 17)], [0, 2, 4], [90, 129], 6, 2, 64, 48),
    ([(3, 3), (1, 2000)], [0, 1], [1500], 14, 2, 128, 16),                # 7 heads a group, one without
    ([(4, 0), (1, 0)], [0, 1, 2], [0, 33], 4, 4, 64, 16),                 # rows without any key
    ([(33, 40)], [0, 1], [5000], 40, 1, 128, 64),                         # 40 heads a group
    ([(1, 30)] * 70, [0, 70], [3000], 4, 1, 64, 16),
]


@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("case", PREFIX, ids=[str(i) for i in range(len(PREFIX))])
def test_prefix_matches_plain(sm100, case, kind, mode):
    lens, cuts, prefixes, Hq, Hkv, d, page = case
    io, cache = kind
    order = "token" if (len(lens) + mode) % 2 else "head"
    P = with_prefixes(lens, prefixes, Hkv, d, page, cache, io=io, order=order, seed=len(lens) + mode)
    q = P.new(Hq)
    rows = [P.cu[x] for x in cuts]
    _check(P, q, Hq, rows, mode, _attend(P, q, rows, mode))
    assert abi.load().fa_device_status(1) == 0


@pytest.mark.parametrize("cache", [F16, E4M3])
@pytest.mark.parametrize("nq", [1, 40])
def test_prefix_bounds_and_rows_of_no_sequence(sm100, nq, cache):
    """Rows before and after the sequences, a prefix over rows of no sequence and over parts of
    one; looser bounds change nothing, tighter ones cut what the documentation says."""
    P = with_prefixes([(nq, 90), (nq, 70)], [200, 130], 2, 64, 16, cache, seed=4, first=3, tail=5)
    q = P.new(8)
    for rows in ([0, 3 + nq, P.total], [2, 3 + nq // 2, 3 + nq + 1], [5, 5, 6]):
        _check(P, q, 8, rows, 1, _attend(P, q, rows, 1))
        _check(P, q, 8, rows, 1, _attend(P, q, rows, 1, slack=900))
    rows = [3, 3 + nq, 3 + 2 * nq]
    for mq, mk in ((nq // 2, 200), (nq, 100), (0, 200), (nq, 0)):
        got = _attend(P, q, rows, 1, max_prefix_q=mq, max_prefix_k=mk)
        _check(P, q, 8, rows, 1, got, max_prefix_q=mq, max_prefix_k=mk)


@pytest.mark.parametrize("nq", [1, 33])
@pytest.mark.parametrize("cache", [F16, I8])
def test_prefix_large_scores(sm100, nq, cache):
    """Rows that one of the two sets dominates by far, a negative and a zero scale."""
    P = with_prefixes([(nq, 150), (nq, 40)], [300], 2, 128, 16, cache, seed=5, spread=3.0)
    q = P.new(8, spread=4.0)
    rows = [0, P.total]
    for scale in (None, -0.3, 0.0):
        _check(P, q, 8, rows, 1, _attend(P, q, rows, 1, scale=scale), scale)


def test_prefix_without_prefixes_or_sequences(sm100):
    P = with_prefixes([(2, 30), (1, 9)], [], 2, 64, 16, F16, seed=6)
    q = P.new(4)
    c = P.cuda()
    s = split(P, c)
    empty = torch.empty(0, 3, dtype=torch.int32, device="cuda")
    got = fa.flash_attention_forward_paged_prefix(
        q.cuda(), c["k_cache"], c["v_cache"], empty, [0], [], s["table"], s["cu"], s["lens"], 3, 30, 2, 30,
        causal=True, return_lse=True)
    _check(P, q, 4, [0], 1, got)
    o, lse = fa.flash_attention_forward_paged_prefix(
        q.cuda(), c["k_cache"], c["v_cache"], s["table"], [0, 2, 3], [30, 9], empty, [0], [], 2, 30, 0, 0,
        causal=True, return_lse=True)
    assert (o == 0).all() and (lse == -math.inf).all()
    none = fa.flash_attention_forward_paged_prefix(
        q.cuda()[:0], c["k_cache"], c["v_cache"], s["table"], [0, 0, 0], [30, 9], s["table"], [0, 0, 0], s["lens"], 0,
        30, 0, 30)
    assert none.shape == (0, 4, 64)


def test_prefix_strided_inputs_and_outputs_alone(sm100):
    """Queries as slices of a projection, tables as slices of wider ones, 64-bit tables and lists;
    without return_lse the same O."""
    P = with_prefixes([(1, 50), (3, 20)] * 4, [170, 64], 2, 128, 16, BF16, io=BF16, order="token", seed=7)
    q = P.new(8)
    rows = [0, P.cu[5], P.total]
    c = P.cuda()
    s = split(P, c)
    want = _attend(P, q, rows, 1, c)
    _check(P, q, 8, rows, 1, want)
    wide = torch.zeros(P.total, 12, 128, dtype=BF16, device="cuda")
    wide[:, :8] = q.cuda()
    big = torch.full((2, 40), 1 << 30, dtype=torch.int32, device="cuda")
    w = s["prefix_table"].size(1)
    big[:, 5:5 + w] = s["prefix_table"]
    got = fa.flash_attention_forward_paged_prefix(
        wide[:, :8], c["k_cache"], c["v_cache"], big[:, 5:5 + w], rows, s["prefix_lens"].long().cpu(),
        s["table"].long(), s["cu"].tolist(), s["lens"].cpu(), rows[1], 170, 3, 50, causal=True)
    assert torch.equal(got, want[0])
    # every other head, a broadcast token: copied
    odd = fa.flash_attention_forward_paged_prefix(
        q.cuda()[:1].expand(P.total, -1, -1), c["k_cache"], c["v_cache"], s["prefix_table"], rows, s["prefix_lens"],
        s["table"], s["cu"], s["lens"], rows[1], 170, 3, 50, causal=True, return_lse=True)
    _check(P, q[:1].expand(P.total, -1, -1), 8, rows, 1, odd)


@pytest.mark.parametrize("cache", [F16, I8])
@pytest.mark.parametrize("tokens", [1, 60])
def test_prefix_in_a_graph_and_on_another_stream(sm100, tokens, cache):
    """A captured call replayed with other lengths, prefixes and queries in the same buffers, beside
    a second graph of the same call."""
    lens = [(tokens, 64), (tokens, 200), (tokens, 130)]
    A = with_prefixes(lens, [300, 90], 2, 64, 16, cache, seed=8)
    c = A.cuda()
    s = split(A, c)
    q = A.new(8).cuda()
    cup = torch.tensor([0, tokens, 3 * tokens], dtype=torch.int32, device="cuda")

    def call():
        return fa.flash_attention_forward_paged_prefix(
            q, c["k_cache"], c["v_cache"], s["prefix_table"], cup, s["prefix_lens"], s["table"], s["cu"], s["lens"],
            3 * tokens, 300, tokens, 200, causal=True, return_lse=True, **_scales(c))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        eager = call()
    stream.synchronize()
    _check(A, q.cpu(), 8, cup.tolist(), 1, eager)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(graphs[0][1], eager))
    cup.copy_(torch.tensor([0, 2 * tokens, 3 * tokens]))
    A.prefixes = [17, 0]
    s["prefix_lens"].copy_(torch.tensor(A.prefixes))
    A.lens[:3] = [(tokens, 64), (tokens, 60), (tokens, tokens)]
    s["lens"].copy_(torch.tensor([n for _, n in A.lens[:3]]))
    q.copy_(A.new(8).cuda())
    for g, out in (graphs[1], graphs[0]):
        g.replay()
        torch.cuda.synchronize()
        _check(A, q.cpu(), 8, cup.tolist(), 1, out)


def test_prefix_c_entry_point_with_a_soiled_workspace(sm100):
    for lens, prefixes, cache in (([(1, 40)] * 50, [900], F16), ([(90, 90), (1, 3)], [400], BF16),
                                  ([(1, 40)] * 50, [900], I8), ([(90, 90), (1, 3)], [400], E4M3)):
        io = BF16 if cache == BF16 else F16
        P = with_prefixes(lens, prefixes, 2, 128, 16, cache, io=io, seed=9)
        c = P.cuda()
        s = split(P, c)
        q = P.new(8).cuda()
        pc = abi.paged_cache(c["k_cache"], c["v_cache"], s["table"], c["k_scale"], c["v_scale"])
        rows = torch.tensor([0, P.total], dtype=torch.int32, device="cuda")
        want = _attend(P, q, [0, P.total], 1, c)
        for soil in (0xff, 0x7f):
            ws = torch.full((64 << 20,), soil, dtype=torch.uint8, device="cuda")
            o, lse = torch.full_like(q, math.nan), torch.full((8, P.total), math.nan, device="cuda")
            rc = abi.fa_fwd_paged_prefix(pc, s["prefix_table"], rows, s["prefix_lens"], P.total, max(prefixes), q, o, lse,
                                         s["cu"], s["lens"], max(m for m, _ in lens), max(n for _, n in lens), causal=1,
                                         workspace=ws)
            assert rc == 0
            torch.cuda.synchronize()
            assert torch.equal(o, want[0]) and torch.equal(lse, want[1])


def test_prefix_refusals(sm100):
    P = with_prefixes([(1, 20)], [32], 2, 64, 16, F16, seed=1)
    c = P.cuda()
    s = split(P, c)
    q = P.new(4).cuda()

    def call(q=q, prefix_table=s["prefix_table"], cup=(0, 1), plens=(32,), kc=c["k_cache"], table=s["table"], mpq=1):
        return fa.flash_attention_forward_paged_prefix(q, kc, c["v_cache"], prefix_table, cup, plens, table, [0, 1], [20],
                                                       mpq, 32, 1, 20, causal=True)

    call()
    for kw in (dict(q=q[0]), dict(q=q.cpu()), dict(q=q.float()), dict(q=q[:, :3]), dict(cup=(0, 1, 1)),
               dict(plens=(32, 1)), dict(kc=c["k_cache"].bfloat16()), dict(kc=c["k_cache"].cpu()), dict(mpq=-1),
               dict(prefix_table=s["prefix_table"][0])):
        with pytest.raises((RuntimeError, ValueError)):
            call(**kw)


# ---------------------------------------------------------------- summed weights

def _old(P, seed=0, extra=5):
    g = torch.Generator().manual_seed(seed)
    return torch.rand(len(P.lens), P.Hkv, P.width * P.page + extra, generator=g) * 3


def _weights(P, q, lse, old, mode, kind, c=None, max_q=None, max_k=None, **kw):
    c = c or P.cuda()
    w = old.cuda().clone()
    fa.kvcache_weights_paged(q.cuda(), lse.cuda().float(), c["k_cache"], c["table"], c["cu"], c["lens"],
                             max([m for m, _ in P.lens] + [0]) if max_q is None else max_q,
                             max([n for _, n in P.lens] + [0]) if max_k is None else max_k, w, mode=kind,
                             k_scale=c["k_scale"], **_rule(mode), **kw)
    return w


def _check_weights(P, q, lse, Hq, mode, old, kind, got, scale=None, **kw):
    w, tol = summed_weights(P, q, lse.float(), Hq, mode, old, kind, scale, **kw)
    err = (got.double().cpu() - w).abs()
    assert (err <= tol).all(), (err / tol.clamp(min=1e-30)).max().item()
    held = torch.zeros_like(old, dtype=torch.bool)
    for b, (_, n) in enumerate(P.lens):
        held[b, :, :n if kw.get("max_k") is None else min(n, kw["max_k"])] = True
    assert torch.equal(got.cpu()[~held], old[~held])


WEIGHTS = [
    ([(1, 1)], 1, 1, 64, 16),
    ([(1, 300)], 32, 8, 128, 16),
    ([(1, 17), (1, 1), (1, 500), (0, 40), (1, 64), (1, 0)], 8, 2, 128, 16),
    ([(1, 1000), (3, 777), (2, 33)], 6, 2, 64, 48),
    ([(4, 129), (4, 640), (4, 4)], 8, 2, 128, 32),
    ([(2, 90), (1, 411)], 14, 2, 64, 16),
    ([(5, 60), (17, 200), (1, 900)], 4, 4, 128, 64),
    ([(300, 513), (1, 700), (0, 0), (33, 33)], 8, 2, 128, 16),
    ([(513, 513), (20, 1500)], 6, 1, 128, 48),
    ([(50, 20), (7, 3)], 4, 2, 64, 16),                          # more new tokens than cached
    ([(260, 700)], 5, 5, 64, 256),
    ([(9, 2000), (1, 2500)], 40, 1, 128, 16),
    ([(1, 60), (2, 130)], 128, 1, 64, 16),                       # 128 heads a group
]


@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("case", WEIGHTS, ids=[str(i) for i in range(len(WEIGHTS))])
def test_weights_match_plain(sm100, case, kind, mode):
    lens, Hq, Hkv, d, page = case
    io, cache = kind
    order = "token" if (len(lens) + mode) % 2 else "head"
    P = Paged(lens, Hkv, d, page, cache, io=io, order=order, seed=len(lens) + 7 * mode)
    q = P.new(Hq)
    _, lse, _, _ = attention(P, q, Hq, mode)
    old = _old(P)
    how = ("append", "add", "set")[mode]
    _check_weights(P, q, lse, Hq, mode, old, how, _weights(P, q, lse, old, mode, how))
    assert abi.load().fa_device_status(1) == 0


@pytest.mark.parametrize("nq", [1, 7, 100])
def test_weights_modes_bounds_and_rows_of_no_sequence(sm100, nq):
    P = Paged([(nq, 130), (0, 50), (nq, 100)], 2, 64, 16, F16, seed=2, first=3, tail=5)
    q = P.new(8)
    _, lse, _, _ = attention(P, q, 8, 1)
    old = _old(P)
    for how in ("append", "add", "set"):
        _check_weights(P, q, lse, 8, 1, old, how, _weights(P, q, lse, old, 1, how))
        _check_weights(P, q, lse, 8, 1, old, how, _weights(P, q, lse, old, 1, how, max_q=nq + 900, max_k=4000))
        # a bound on the tokens cuts the sequence's last ones, one on the keys its last ones
        mq, mk = max(nq // 2, 1), 77
        _check_weights(P, q, lse, 8, 1, old, how, _weights(P, q, lse, old, 1, how, max_q=mq, max_k=mk), max_q=mq,
                       max_k=mk)


def test_weights_without_queries(sm100):
    """A step without tokens: the sums stay, or are set to 0."""
    P = Paged([(0, 130), (0, 7), (0, 0)], 2, 64, 16, F16, seed=2)
    q, lse, old = P.new(8), torch.zeros(8, 0), _old(P)
    assert q.size(0) == 0
    for how in ("append", "add", "set"):
        _check_weights(P, q, lse, 8, 1, old, how, _weights(P, q, lse, old, 1, how))


@pytest.mark.parametrize("nq", [1, 150])
def test_weights_masked_rows_and_places(sm100, nq):
    """Rows whose LSE is -inf add nothing, whatever keys hold; NaN keys that no row may see do
    not show; a NaN key gets NaN alone."""
    P = Paged([(nq, 300)], 2, 128, 16, BF16, io=BF16, seed=3)
    q = P.new(4)
    _, lse, _, _ = attention(P, q, 4, 1)
    lse[:, ::3] = -math.inf
    old = _old(P)
    _check_weights(P, q, lse, 4, 1, old, "append", _weights(P, q, lse, old, 1, "append"))
    P.put("k", 0, [299], torch.full((1, 2, 128), math.nan).bfloat16(), None)
    got = _weights(P, q, lse, old, 2, "set").cpu()      # top-left: key 299 is seen by no row
    if nq < 300:
        assert (got[0, :, 299] == 0).all() and torch.isfinite(got[0, :, :300]).all()
    P.put("k", 0, [5], torch.full((1, 2, 128), math.nan).bfloat16(), None)
    got = _weights(P, q, lse, old, 0, "set").cpu()
    dead = torch.isinf(lse).all()
    bad = torch.isnan(got[0, :, :300])
    want = torch.zeros(2, 300, dtype=torch.bool)
    if not dead:
        want[:, [5, 299]] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("cache", [F16, I8, E4M3])
@pytest.mark.parametrize("nq", [1, 130])
def test_weights_large_scores_and_scales(sm100, nq, cache):
    """Logits up to hundreds (most terms underflow), a negative and a zero scale."""
    P = Paged([(nq, 700), (nq, 150)], 2, 128, 16, cache, seed=4, spread=3.0)
    q = P.new(8, spread=4.0)
    old = _old(P)
    for scale in (None, -0.3, 0.0):
        _, lse, _, _ = attention(P, q, 8, 1, scale)
        got = _weights(P, q, lse, old, 1, "append", scale=scale)
        _check_weights(P, q, lse, 8, 1, old, "append", got, scale)


def test_weights_strided_arguments_and_repeats(sm100):
    """Sums as a transposed slice of a larger tensor, queries as slices, lse of wider memory: the
    rows beside stay; equal calls give equal bits; the same page twice in a table."""
    P = Paged([(3, 200), (1, 90)], 2, 64, 16, F16, seed=5)
    q = P.new(8)
    _, lse, _, _ = attention(P, q, 8, 1)
    old = _old(P)
    want = _weights(P, q, lse, old, 1, "append")
    assert torch.equal(want, _weights(P, q, lse, old, 1, "append"))
    c = P.cuda()
    big = torch.full((2, 3, old.size(2) + 7), 5.0, device="cuda")
    big[:, :2, 3:-4] = old.cuda().transpose(0, 1)
    w = big[:, :2, 3:-4].transpose(0, 1)
    wq = torch.zeros(P.total, 20, 64, dtype=F16, device="cuda")
    wq[:, 8:16] = q.cuda()
    wl = torch.zeros(8, P.total + 3, device="cuda")
    wl[:, :P.total] = lse.cuda()
    fa.kvcache_weights_paged(wq[:, 8:16], wl[:, :P.total], c["k_cache"], c["table"], P.cu, P.nk, 3, 200, w, causal=True)
    assert torch.equal(w, want)
    assert (big[:, 2] == 5).all() and (big[..., :3] == 5).all() and (big[..., -4:] == 5).all()
    # two sequences over the same pages: each its own sums
    t = c["table"].clone()
    t[1] = t[0]
    P.table = t.cpu()
    _, lse, _, _ = attention(P, q, 8, 1)
    w = old.cuda().clone()
    fa.kvcache_weights_paged(q.cuda(), lse.cuda().float(), c["k_cache"], t, c["cu"], c["lens"], 3, 200, w, causal=True)
    _check_weights(P, q, lse, 8, 1, old, "append", w)
    # broadcast heads of a cache and of queries are read
    kc = c["k_cache"][:, :1].expand(-1, 2, -1, -1)
    P.k[:, 1] = P.k[:, 0]
    P.v[:, 1] = P.v[:, 0]
    _, lse, _, _ = attention(P, q, 8, 1)
    w = old.cuda().clone()
    fa.kvcache_weights_paged(q.cuda(), lse.cuda().float(), kc, t, c["cu"], c["lens"], 3, 200, w, causal=True)
    _check_weights(P, q, lse, 8, 1, old, "append", w)


@pytest.mark.parametrize("nq", [1, 70])
def test_weights_in_a_graph(sm100, nq):
    P = Paged([(nq, 300), (nq, 128)], 2, 128, 16, BF16, io=BF16, seed=6)
    c = P.cuda()
    q = P.new(8)
    _, lse, _, _ = attention(P, q, 8, 1)
    old = _old(P)
    qd, ld, w = q.cuda(), lse.cuda().float(), old.cuda().clone()

    def call():
        fa.kvcache_weights_paged(qd, ld, c["k_cache"], c["table"], c["cu"], c["lens"], nq, 300, w, causal=True)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    stream.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    P.lens = [(nq, 250), (nq, nq)]
    P.nk = [250, nq]
    c["lens"].copy_(torch.tensor(P.nk))
    q = P.new(8)
    _, lse, _, _ = attention(P, q, 8, 1)
    qd.copy_(q)
    ld.copy_(lse)
    w.copy_(old)
    g.replay()
    torch.cuda.synchronize()
    _check_weights(P, q, lse, 8, 1, old, "append", w)


def test_weights_refusals(sm100):
    P = Paged([(1, 20)], 2, 64, 16, I8, seed=1)
    c = P.cuda()
    q, lse, w = P.new(4).cuda(), torch.zeros(4, 1, device="cuda"), torch.zeros(1, 2, 48, device="cuda")

    def call(q=q, lse=lse, k=c["k_cache"], table=c["table"], w=w, ks=c["k_scale"], max_k=20, max_q=1, **kw):
        fa.kvcache_weights_paged(q, lse, k, table, [0, 1], [20], max_q, max_k, w, causal=True, k_scale=ks, **kw)

    call()
    for kw in (dict(q=q[0]), dict(q=q[:, :3], lse=lse[:3]), dict(lse=lse[:3]), dict(lse=lse.double()),
               dict(lse=lse.cpu()), dict(ks=None), dict(w=w.double()), dict(w=w.cpu()), dict(w=w[0]),
               dict(w=w[:, :1].expand(-1, 2, -1)), dict(w=w[..., :19]), dict(w=w.transpose(1, 2).contiguous().transpose(1, 2)),
               dict(max_k=-1), dict(max_q=1 << 40), dict(mode="sum")):
        with pytest.raises((RuntimeError, ValueError)):
            call(**kw)


# ---------------------------------------------------------------- eviction

def _sums(P, seed=0, ties=True, extra=3):
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(2 * torch.randn(len(P.lens), P.Hkv, P.width * P.page + extra, generator=g))
    if ties:
        w[torch.rand(w.shape, generator=g) < 0.3] = 0
        w[torch.rand(w.shape, generator=g) < 0.2] = 1.5
        w[torch.rand(w.shape, generator=g) < 0.02] = -0.0
    return w


def _evict(P, w, keep, recent=0, first=0, c=None):
    c = c or P.cuda()
    wd = w.cuda().clone()
    lens = fa.kvcache_evict_paged(c["k_cache"], c["v_cache"], wd, c["table"], c["lens"],
                                  keep if isinstance(keep, int) else torch.tensor(keep, device="cuda"), recent=recent,
                                  first=first, **_scales(c))
    return c, wd, lens


def _check_evict(P, w, keep, recent, first, got):
    c, wd, lens = got
    k, v, ks, vs, w2, n2 = evicted(P, w, keep, recent, first)
    for name, want in (("k_cache", k), ("v_cache", v), ("k_scale", ks), ("v_scale", vs)):
        if want is not None:
            x = bits(c[name]).cpu()
            x, want = (x.view(torch.int32), want.view(torch.int32)) if x.dtype == torch.float32 else \
                (x.view(torch.int16), want.view(torch.int16)) if x.element_size() == 2 else (x, want)
            assert torch.equal(x, want), name
    assert torch.equal(wd.cpu().view(torch.int32), w2.view(torch.int32))
    assert lens.dtype == torch.int32 and lens.tolist() == n2


EVICT = [  # lengths, KV heads, d, page, keep, recent, first
    ([20], 1, 64, 16, 8, 2, 1),
    ([1, 2, 0, 33], 2, 128, 16, 1, 0, 0),
    ([300, 17, 128, 129, 1025], 2, 128, 16, 128, 16, 4),
    ([2100, 700], 3, 64, 48, 1024, 0, 0),
    ([2100, 700], 3, 64, 48, 1025, 1025, 0),                     # the recent ones alone
    ([900, 40], 2, 64, 32, 33, 100, 4),                          # more asked for than stays
    ([900, 40], 2, 64, 32, 3, 0, 7),
    ([5000], 1, 128, 256, 4999, 10, 0),                          # one goes
    ([5000], 2, 128, 16, 0, 10, 2),                              # all go
    ([3000, 3000], 2, 64, 16, [700, 2999], 64, 4),
]


@pytest.mark.parametrize("kind", [F16, BF16, I8, E4M3], ids=["f16", "bf16", "int8", "e4m3"])
@pytest.mark.parametrize("case", EVICT, ids=[str(i) for i in range(len(EVICT))])
def test_evict_matches_plain(sm100, case, kind):
    lens, Hkv, d, page, keep, recent, first = case
    P = Paged([(0, n) for n in lens], Hkv, d, page, kind, order="token" if len(lens) % 2 else "head", seed=len(lens))
    for ties in (True, False):
        w = _sums(P, seed=3, ties=ties)
        _check_evict(P, w, keep, recent, first, _evict(P, w, keep, recent, first))


def test_evict_odd_weights(sm100):
    """NaN, infinities, negative sums, all equal, all zero, subnormal."""
    P = Paged([(0, 500)], 2, 64, 16, F16, seed=4)
    n = P.width * P.page
    g = torch.Generator().manual_seed(1)
    rows = [torch.full((n,), 2.0), torch.zeros(n), -torch.rand(n, generator=g), torch.arange(n) * 1e-42,
            torch.randn(n, generator=g)]
    rows[4][::3] = math.nan
    rows[4][1::5] = -math.inf
    rows[4][2::7] = math.inf
    for a in rows:
        for b in (rows[0], rows[4]):
            w = torch.stack([a, b])[None].clone()
            for keep in (1, 130, 499):
                _check_evict(P, w, keep, 1, 0, _evict(P, w, keep, 1, 0))


def test_evict_leaves_missing_pages_and_other_rows_alone(sm100):
    """Table entries outside the cache: rows read as zeros and are not written."""
    P = Paged([(0, 200), (0, 90)], 2, 64, 16, BF16, seed=5)
    w = _sums(P, seed=6, ties=False)
    c = P.cuda()
    c["table"][0, 3] = -1
    c["table"][0, 7] = 1 << 29
    k0 = c["k_cache"].clone()
    _, wd, lens = _evict(P, w, 100, 8, 0, c)
    assert lens.tolist() == [100, 90]
    _, _, _, _, w2, _ = evicted(P, w, 100, 8, 0)
    assert torch.equal(wd.cpu(), w2)
    gone = {int(P.table[0, 3]), int(P.table[0, 7])}
    for pg in gone:  # pages without an entry, and the other sequence's
        assert torch.equal(c["k_cache"][pg].view(torch.int16), k0[pg].view(torch.int16))
    for pg in P.table[1, :6].tolist():
        assert torch.equal(c["k_cache"][pg].view(torch.int16), k0[pg].view(torch.int16))
    kr, _ = fa.kvcache_read_paged(c["k_cache"], c["v_cache"], c["table"][:1], [0, 100], [100], 100)
    assert (kr[48:64] == 0).all() and torch.isfinite(kr).all()


def test_evict_in_a_graph_and_strided_sums(sm100):
    P = Paged([(0, 400), (0, 300)], 2, 128, 16, F16, seed=7)
    w = _sums(P, seed=8)
    c = P.cuda()
    keep = torch.tensor([64, 200], dtype=torch.int32, device="cuda")
    big = torch.full((2, 2, w.size(2) + 9), 7.0, device="cuda")
    ws = big[..., 4:-5].transpose(0, 1)
    k0, v0, l0 = c["k_cache"].clone(), c["v_cache"].clone(), c["lens"].clone()

    def call():
        return fa.kvcache_evict_paged(c["k_cache"], c["v_cache"], ws, c["table"], c["lens"], keep, recent=10, first=2)

    ws.copy_(w)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        lens = call()
    stream.synchronize()
    _check_evict(P, w, [64, 200], 10, 2, (c, ws.contiguous(), lens))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for ks in ([30, 31], [64, 500]):
        keep.copy_(torch.tensor(ks))
        c["k_cache"].copy_(k0)
        c["v_cache"].copy_(v0)
        c["lens"].copy_(l0)
        ws.copy_(w)
        g.replay()
        torch.cuda.synchronize()
        _check_evict(P, w, ks, 10, 2, (c, ws.contiguous(), out))
    assert (big[..., :4] == 7).all() and (big[..., -5:] == 7).all()


def test_evict_long(sm100):
    """A cache longer than one block's first look, by heads of different weights."""
    P = Paged([(0, 20000), (0, 9000)], 2, 64, 64, I8, seed=9)
    w = _sums(P, seed=10)
    _check_evict(P, w, 8191, 100, 4, _evict(P, w, 8191, 100, 4))


def test_evict_refusals(sm100):
    P = Paged([(0, 40)], 2, 64, 16, I8, seed=1)
    c = P.cuda()
    w = torch.zeros(1, 2, 64, device="cuda")

    def call(k=c["k_cache"], v=c["v_cache"], w=w, lens=(40,), keep=8, ks=c["k_scale"], vs=c["v_scale"], **kw):
        return fa.kvcache_evict_paged(k, v, w, c["table"], lens, keep, k_scale=ks, v_scale=vs, **kw)

    call()
    for kw in (dict(k=c["k_cache"][:, :1].expand(-1, 2, -1, -1), v=c["v_cache"][:, :1].expand(-1, 2, -1, -1)),
               dict(ks=c["k_scale"][:1].expand_as(c["k_scale"]), vs=c["v_scale"][:1].expand_as(c["v_scale"])),
               dict(ks=None), dict(w=w.half()), dict(w=w[..., :63]), dict(w=w[:, :1].expand(-1, 2, -1)), dict(lens=(40, 1)),
               dict(keep=(1, 2)), dict(keep=-1), dict(first=-1), dict(recent=-1), dict(w=w[0]), dict(k=c["k_cache"].cpu())):
        with pytest.raises((RuntimeError, ValueError)):
            call(**kw)


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
def test_weights_of_prefix_and_own_keys_sum_to_the_rows(sm100, kind):
    """Each row's weights over its prefix and its own keys sum to 1: the LSE of the two passes and
    the sums of two calls belong together."""
    io, cache = kind
    P = with_prefixes([(1, 60), (40, 70), (3, 3)], [200, 77], 2, 128, 16, cache, io=io, seed=12)
    q = P.new(8).cuda()
    c = P.cuda()
    s = split(P, c)
    cup = torch.tensor([0, P.cu[2], P.total], dtype=torch.int32, device="cuda")
    _, lse = _attend(P, q, cup.tolist(), 1, c)
    own = torch.zeros(3, 2, P.width * 16, device="cuda")
    pre = torch.zeros(2, 2, P.width * 16, device="cuda")
    fa.kvcache_weights_paged(q, lse, c["k_cache"], s["table"], s["cu"], s["lens"], 40, 70, own, causal=True,
                             k_scale=c["k_scale"])
    fa.kvcache_weights_paged(q, lse, c["k_cache"], s["prefix_table"], cup, s["prefix_lens"], P.cu[2], 200, pre,
                             mode="add", k_scale=c["k_scale"])
    o, p = own.sum(-1).cpu(), pre.sum(-1).cpu()
    # (LSE is good to 1e-4 and, 8-bit pages, f16 rounding of a score of about 10; 164 rows)
    assert torch.allclose(o[0] + o[1] + p[0], torch.full((2,), 4.0 * 41), rtol=2e-3)
    assert torch.allclose(o[2] + p[1], torch.full((2,), 4.0 * 3), rtol=2e-3)


@pytest.mark.parametrize("cache", [F16, I8])
def test_byte_offsets_past_4_gib(sm100, cache):
    """The same pages at the end of a cache of more than 2^32 bytes: equal bits."""
    P = with_prefixes([(1, 300), (60, 90), (2, 40)], [150], 2, 128, 16, cache, seed=13)
    q = P.new(8).cuda()
    c = P.cuda()
    s = split(P, c)
    n, size = P.pages, 2 * 16 * 128 * c["k_cache"].element_size()
    big = (1 << 32) // size + 1000

    def far(x):
        if x is None:
            return None
        y = torch.empty((big + n, *x.shape[1:]), dtype=x.dtype, device="cuda")
        bits(y)[big:] = bits(x)
        return y

    b = dict(c, **{k: far(c[k]) for k in ("k_cache", "v_cache", "k_scale", "v_scale")})
    b["table"] = torch.where((c["table"] >= 0) & (c["table"] < n), c["table"] + big, c["table"])
    P.pages += big
    rows = [0, P.total]
    near, there = _attend(P, q, rows, 1, c), _attend(P, q, rows, 1, b)
    assert torch.equal(near[0], there[0]) and torch.equal(near[1], there[1])
    out = []
    for x in (c, b):
        t = x["table"][:3].contiguous()
        w = torch.ones(3, 2, P.width * 16, device="cuda")
        fa.kvcache_weights_paged(q, near[1], x["k_cache"], t, s["cu"], s["lens"], 60, 300, w, causal=True,
                                 k_scale=x["k_scale"])
        lens = fa.kvcache_evict_paged(x["k_cache"], x["v_cache"], w, t, s["lens"], 70, recent=9, **_scales(x))
        out.append((w, lens, bits(x["k_cache"])[-n:], bits(x["v_cache"])[-n:]))
    for x, y in zip(*out):
        assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))


@pytest.mark.parametrize("kind", [F16, I8])
def test_many_sequences(sm100, kind):
    """More sequences than threads of a block; ragged, some without tokens or keys."""
    g = torch.Generator().manual_seed(5)
    n = torch.randint(0, 30, (700,), generator=g).tolist()
    lens = [(min(x, int(torch.randint(0, 4, (1,), generator=g))), x) for x in n]
    P = with_prefixes(lens, [33, 0, 100], 1, 64, 16, kind, seed=14)
    q = P.new(3)
    rows = [P.cu[10], P.cu[300], P.cu[310], P.cu[650]]
    c = P.cuda()
    got = _attend(P, q, rows, 1, c)
    _check(P, q, 3, rows, 1, got)
    P.lens, P.cu, P.nk = P.lens[:700], P.cu[:701], P.nk[:700]
    c["table"], c["cu"], c["lens"] = c["table"][:700].contiguous(), c["cu"][:701].contiguous(), c["lens"][:700].contiguous()
    old = _old(P)
    lse = got[1].cpu()
    _check_weights(P, q, lse, 3, 1, old, "append", _weights(P, q, lse, old, 1, "append", c))
    w = _sums(P, seed=15)
    _check_evict(P, w, 9, 2, 1, _evict(P, w, 9, 2, 1, c))


@pytest.mark.parametrize("kind", [F16, I8], ids=["f16", "int8"])
def test_a_serving_run(sm100, kind):
    """Steps of two requests behind one prompt as they would be served: write, attend, sum the
    weights, cut the caches when they are long; every step's results, sums and lengths against
    the plain forms over what the cache then holds."""
    Hq, Hkv, d, page = 8, 2, 64, 16
    P = with_prefixes([(0, 0), (0, 0)], [90], Hkv, d, page, kind, seed=11, spare=40)
    P.table = torch.full((3, 12), -1, dtype=torch.int32)
    P.table[2, :6] = torch.arange(6)
    P.table[0], P.table[1] = torch.arange(6, 18), torch.arange(18, 30)
    P.width = 12
    used = [0, 0]
    for b, n in ((2, 90),):
        for name in ("k", "v"):
            x = torch.randn(n, Hkv, d, generator=P.g)
            P.put(name, b, range(n), *(quantise(x, kind) if kind in QMAX else (x.to(kind), None)))
    c = P.cuda()
    table = c["table"][:2].contiguous()
    sums = torch.full((2, Hkv, 12 * page), math.nan, device="cuda")
    plain = sums.cpu().clone()
    for step, new in enumerate(([40, 3], [1, 1], [9, 60], [1, 1], [1, 30], [70, 1], [1, 1])):
        used = [u + n for u, n in zip(used, new)]
        P.lens = [(n, u) for n, u in zip(new, used)] + [(0, 90)]
        P.cu = [0, new[0], sum(new), sum(new)]
        P.total, P.nk = sum(new), used + [90]
        cu = torch.tensor(P.cu[:3], dtype=torch.int32, device="cuda")
        lens = torch.tensor(used, dtype=torch.int32, device="cuda")
        qkv = torch.randn(P.total, Hq + 2 * Hkv, d, generator=P.g).half()
        q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        fa.kvcache_write_paged(k.cuda(), v.cuda(), c["k_cache"], c["v_cache"], table, cu, lens, **_scales(c))
        o, lse = fa.flash_attention_forward_paged_prefix(
            q.cuda(), c["k_cache"], c["v_cache"], c["table"][2:], [0, P.total], [90], table, cu, lens, P.total, 90,
            max(new), max(used), causal=True, return_lse=True, **_scales(c))
        fa.kvcache_weights_paged(q.cuda(), lse, c["k_cache"], table, cu, lens, max(new), max(used), sums, causal=True,
                                 k_scale=c["k_scale"])
        # the plain forms over the cache as it is now
        for name in ("k", "v"):
            getattr(P, name).copy_(c[name + "_cache"].cpu())
            if kind in QMAX:
                getattr(P, name + "s").copy_(c[name + "_scale"].cpu())
        _check(P, q, Hq, [0, P.total], 1, (o, lse))
        Q = P
        both, Q.lens, Q.cu = P.lens, P.lens[:2], P.cu
        want, tol = summed_weights(Q, q, lse.cpu(), Hq, 1, plain, "append")
        Q.lens = both
        held = ~torch.isnan(want)
        assert torch.equal(torch.isnan(sums.cpu()), ~held)
        assert ((sums.cpu().double() - want).abs()[held] <= tol[held]).all()
        plain = sums.cpu().clone()
        if max(used) > 64:
            P.lens = P.lens[:2]
            w2 = evicted(P, plain, 48, 16, 4)
            got = fa.kvcache_evict_paged(c["k_cache"], c["v_cache"], sums, table, lens, 48, recent=16, first=4,
                                         **_scales(c))
            _k = bits(c["k_cache"]).cpu()
            assert torch.equal(_k.view(torch.uint8), w2[0].view(torch.uint8))
            assert torch.equal(sums.cpu().view(torch.int32), w2[4].view(torch.int32))
            used = got.tolist()
            assert used == w2[5]
            plain = sums.cpu().clone()


@pytest.mark.parametrize("pages", ["same", "int8", "e4m3"])
def test_example_with_a_budget(sm100, pages):
    """examples/paged_serving.py with caches cut to 64 tokens: every request ends, no request's
    cache stays a quarter beyond the budget, and each step's attention is that over the keys held."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_serving.py")
    spec = importlib.util.spec_from_file_location("paged_serving", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    seen = []
    plain = example.evict

    def evict(cache, batch, budget):
        plain(cache, batch, budget)
        seen.extend(r.length for r in batch)
        for r in batch:
            assert len(r.pages) == -(-r.length // example.PAGE)
            # every position that is left has a sum, from the tokens that saw it
            assert torch.isfinite(r.sums[:, :r.length]).all() and (r.sums[:, :r.length] > 0).all()
        assert len(cache.free) + sum(len(r.pages) for r in batch) == 512

    example.evict = evict
    drawn, worst = example.serve(pages, steps=60, verbose=False, budget=64)
    assert sorted(len(d) for d in drawn) == [4, 8, 12, 20, 30]
    assert max(seen) <= 80 and 64 in seen
    # values of a few units: bf16 results and bf16 keys read back differ by a few roundings of 2^-8
    assert worst <= 0.06


# ---------------------------------------------------------------- what is not a number

# tokens: some behind the prefix alone, behind both, with own keys alone, without any
NAN = [
    ([(1, 0), (1, 200), (1, 200), (1, 0)], [0, 2], [300], 8, 2),                                # a CTA per head joins
    ([(1, 0), (1, 200)] * 40 + [(1, 200), (1, 0)] * 40, [0, 80], [700], 8, 2),                  # runs, combined
    ([(200, 200), (1, 0), (200, 0), (200, 200), (1, 0), (200, 0)], [0, 3], [300], 8, 2),        # chunks
    ([(200, 200), (1, 0), (1, 200), (200, 200), (1, 0), (1, 200), (9, 0)], [0, 3], [300], 8, 2),  # both kernels, merged
]


@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("case", NAN, ids=["solo", "runs", "chunks", "both"])
def test_prefix_passes_nan_on(sm100, case, kind):
    """A NaN query returns NaN from whichever set of keys it sees, as from the plain call; without any
    key it returns O = 0, LSE = -inf; the other rows do not change."""
    lens, cuts, prefixes, Hq, Hkv = case
    io, cache = kind
    P = with_prefixes(lens, prefixes, Hkv, 128, 16, cache, io=io, seed=21)
    q = P.new(Hq)
    rows = [P.cu[x] for x in cuts]
    c = P.cuda()
    clean = _attend(P, q, rows, 0, c)
    _check(P, q, Hq, rows, 0, clean)
    q[:, 1] = math.nan
    q[::2, 5, 7] = math.nan
    o, lse = _attend(P, q, rows, 0, c)
    sees = torch.isfinite(clean[1]).cpu()                              # [Hq, total]
    bad = q.isnan().any(-1).T & sees
    assert bad.any() and (~sees).any()
    assert torch.equal(lse.isnan().cpu(), bad)
    assert o.isnan().all(-1).cpu()[bad.T].all()
    ok = ~bad.cuda()
    assert torch.equal(lse[ok], clean[1][ok]) and torch.equal(o[ok.T], clean[0][ok.T])


@pytest.mark.parametrize("where", ["list", "cpu", "cuda"])
def test_evict_budgets_beyond_int32(sm100, where):
    """A number of positions that int32 does not hold keeps everything, alone or for each sequence."""
    P = Paged([(0, 40), (0, 90), (0, 33)], 2, 64, 16, F16, seed=2)
    w = _sums(P, seed=2)
    for big in (1 << 31, 1 << 32, (1 << 32) + 5, 1 << 62):
        keep = [big, 20, big]
        c = P.cuda()
        wd = w.cuda()
        lens = fa.kvcache_evict_paged(c["k_cache"], c["v_cache"], wd, c["table"], c["lens"],
                                      keep if where == "list" else torch.tensor(keep, device=where), recent=3)
        _check_evict(P, w, keep, 3, 0, (c, wd, lens))
        c = P.cuda()
        lens = fa.kvcache_evict_paged(c["k_cache"], c["v_cache"], wd, c["table"], c["lens"], big)
        assert lens.tolist() == [40, 90, 33]
