"""The kernels of summed weights and of eviction where they go round more than once: caches and
batches so long that a warp of the streamed weights takes many windows of pages, a CTA of the chunk
weights goes round its rings of query tiles, and an eviction takes several steps and lists.  The
plain forms here are vectorised (64 bits; eviction bit for bit)."""
import math

import pytest
import torch

import flash_attention_sm75 as fa
from tests import abi_ctypes as abi
from tests.paged_plain import QMAX, Paged, attention, quantise
from tests.serving_plain import evicted_whole, with_prefixes
from tests.test_serving_gpu import BF16, E4M3, F16, I8, KIND_IDS, KINDS, _attend, _check_weights, _old, _weights

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- shared prefixes

# own lengths, the sequences where prefixes start and the last one ends, prefix lengths
PREFIX = [
    ([(1, 64)] * 8, [0, 8], [1024]),                                            # a CTA per head joins
    ([(1, 900), (1, 30)] * 32, [0, 64], [4096]),                                # runs, combined
    ([(256, 256)] * 4, [0, 4], [2048]),                                         # chunks
    ([(256, 256), (1, 900), (1, 5)] * 8, [0, 9, 24], [1500, 700]),              # both kernels, merged
]


@pytest.mark.parametrize("kind", [(F16, F16), (BF16, E4M3)], ids=["f16", "bf16-e4m3"])
@pytest.mark.parametrize("case", PREFIX, ids=["solo", "runs", "chunks", "both"])
def test_prefix_calls_repeat_exactly(sm100, case, kind):
    """The second pass may start while the first one ends: equal calls give equal bits, one after the
    other without a pause, after a pause, and beside other work on the GPU."""
    lens, cuts, prefixes = case
    io, cache = kind
    P = with_prefixes(lens, prefixes, 4, 128, 16, cache, io=io, seed=31)
    q = P.new(16).cuda()
    rows = [P.cu[x] for x in cuts]
    c = P.cuda()
    want = _attend(P, q, rows, 1, c)
    torch.cuda.synchronize()
    side, x = torch.cuda.Stream(), torch.randn(2048, 2048, device="cuda")
    for pause in (False, True):
        got = []
        for i in range(12):
            if pause:
                torch.cuda.synchronize()
                with torch.cuda.stream(side):
                    x @ x
            got.append(_attend(P, q, rows, 1, c))
        torch.cuda.synchronize()
        for o, lse in got:
            assert torch.equal(o, want[0]) and torch.equal(lse, want[1])


# ---------------------------------------------------------------- streamed weights

# new tokens, query heads, d: 1, 16 and 24 query rows per KV head (blocks of 8, 16 and 32)
ROWS = [(1, 2, 64), (1, 32, 128), (3, 16, 64)]


@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("case", ROWS, ids=["1", "16", "24"])
def test_streamed_weights_of_long_sequences(sm100, case, kind):
    """3.2 million keys: 84 groups of 16 for each of 2368 warps (148 SMs), which start inside of heads; a
    window has 32.  The pages repeat, so the cache is small; some entries have no page (their keys
    read as zeros).  The bound is that of serving_plain.summed_weights."""
    m, Hq, d = case
    io, cache = kind
    Hkv, page, pages = 2, 16, 40
    G = Hq // Hkv
    lens = [900011, 3, 700003]
    g = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    k, ks = rnd(pages, Hkv, page, d), None
    if cache in QMAX:
        k, ks = (x.cuda() for x in quantise(k.cpu(), cache))
    else:
        k = k.to(cache)
    width = -(-max(lens) // page)
    table = torch.randint(0, pages, (3, width), generator=g, device="cuda").to(torch.int32)
    table[torch.rand(table.shape, generator=g, device="cuda") < 0.02] = -1
    L = width * page
    old = torch.rand((3, Hkv, L), generator=g, device="cuda") * 1e-5
    q = rnd(3 * m, Hq, d).to(io)
    held = k.cpu().double() if ks is None else k.cpu().double() * ks.cpu().double()[..., None]
    held = torch.cat([held.cuda(), torch.zeros(1, Hkv, page, d, dtype=torch.float64, device="cuda")])
    scale = 1 / math.sqrt(d)
    lse = torch.full((Hq, 3 * m), -math.inf, device="cuda")
    want, tol = old.double().clone(), torch.zeros(3, Hkv, L, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        at = (torch.where(table[b] < 0, pages, table[b]).long()[:, None] * page + torch.arange(page, device="cuda"))
        at = at.view(-1)[:n]
        see = torch.arange(n, device="cuda") <= torch.arange(m, device="cuda").repeat_interleave(G)[:, None] + (n - m)
        for h in range(Hkv):
            x = q[b * m:(b + 1) * m, h * G:(h + 1) * G].double().reshape(m * G, d)
            key = held[:, h].reshape(-1, d)
            s = (x @ key.T * scale)[:, at]
            size = (x.abs() @ key.abs().T * scale)[:, at]
            z = torch.logsumexp(s.masked_fill(~see, -math.inf), -1).float()
            lse[h * G:(h + 1) * G, b * m:(b + 1) * m] = z.view(m, G).T
            z = z.double()[:, None]
            p = torch.where(see, torch.exp(s - torch.where(z == -math.inf, 0, z)), 0.0)
            new = p.sum(0)
            base = old[b, h, :n].double()
            base[max(n - m, 0):] = 0
            want[b, h, :n] = base + new
            rel = d * 2.0 ** -23 * size + 2.0 ** -22 * (s.abs() + z.abs()) + 2.0 ** -21
            tol[b, h, :n] = torch.where(see, p * rel, 0.0).sum(0) + (m * G + 1) * 2.0 ** -24 * (base + new) + m * G * 2.0 ** -126
    w = old.clone()
    fa.kvcache_weights_paged(q, lse, k, table, [0, m, 2 * m, 3 * m], lens, m, max(lens), w, causal=True, k_scale=ks)
    err = (w.double() - want).abs()
    assert (err <= tol).all(), (err / tol.clamp(min=1e-30)).max().item()


# ---------------------------------------------------------------- weights of chunks

# lengths, query heads, KV heads, d, page; query tiles, and CTAs that share them on 148 SMs
CHUNKS = [
    ([(160, 2040), (153, 2048)], 40, 5, 128, 16),       # 10 tiles for a CTA
    ([(640, 1025), (577, 1300)], 16, 8, 64, 32),        # 10
    ([(320, 3000), (1, 2000)], 64, 8, 128, 64),         # 20 for clusters of 2, and a single token beside
    ([(2390, 250)], 4, 1, 128, 16),                     # 75 for a cluster of 8 (more tokens than keys)
    ([(2400, 2400)], 4, 1, 64, 16),                     # 75 for clusters of 8, fewer for the later keys
]


@pytest.mark.parametrize("kind", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("case", CHUNKS, ids=[str(i) for i in range(len(CHUNKS))])
def test_chunk_weights_of_many_query_tiles(sm100, case, kind):
    """Rings of four query tiles, LSE rows and accumulators that are used again and again."""
    lens, Hq, Hkv, d, page = case
    io, cache = kind
    P = Paged(lens, Hkv, d, page, cache, io=io, order="token", seed=len(lens))
    q = P.new(Hq)
    old = _old(P)
    for mode in (0, 1):
        _, lse, _, _ = attention(P, q, Hq, mode)
        how = ("add", "append")[mode]
        got = _weights(P, q, lse, old, mode, how)
        _check_weights(P, q, lse, Hq, mode, old, how, got)
        assert torch.equal(got, _weights(P, q, lse, old, mode, how))
    assert abi.load().fa_device_status(1) == 0


# ---------------------------------------------------------------- eviction

def _long_cache(lens, Hkv, d, page, kind, seed):
    """A cache of random bits (every value, NaN too), pages in a random order."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages, width = sum(need) + 3, max(need)
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    size = torch.tensor([], dtype=kind).element_size()
    raw = dict(dtype=torch.uint8 if size == 1 else torch.int16, device="cuda", generator=g)
    c = {x: torch.randint(0, 256, (pages, Hkv, page, d), **raw) * (1 if size == 1 else 129) for x in ("k", "v")}
    for x in ("k_scale", "v_scale"):
        c[x] = torch.rand((pages, Hkv, page), generator=g, device="cuda") if size == 1 else None
    w = torch.exp(2 * torch.randn((len(lens), Hkv, width * page), generator=g, device="cuda"))
    r = torch.rand(w.shape, generator=g, device="cuda")
    w[r < 0.25] = 0.0
    w[(r > 0.25) & (r < 0.3)] = -0.0
    w[(r > 0.3) & (r < 0.45)] = 1.5
    w[(r > 0.45) & (r < 0.46)] = math.nan
    w[(r > 0.46) & (r < 0.47)] = math.inf
    w[(r > 0.47) & (r < 0.48)] = -math.inf
    return c, table, w


EVICT_LONG = [  # sequences, upper length, keep, recent, first, KV heads, d, page, pages; CTAs of a cluster on 148 SMs
    (75, 8200, 4500, 100, 4, 4, 64, 16, F16),               # 1: lists of 4096 places are filled twice
    (75, 8200, 7900, 0, 5000, 4, 64, 64, E4M3),             # 1: whole steps stay where they are
    (75, 16000, 9000, 512, 0, 4, 64, 48, I8),               # 1: steps beyond the weights held in shared memory
    (40, 9000, 6000, 64, 4, 4, 128, 16, BF16),              # 2
    (38, 27000, 20000, 1000, 0, 4, 64, 32, I8),             # 2: beyond the held weights, several lists
    (20, 20000, 17000, 64, 4, 4, 64, 16, F16),              # 4: several lists
    (3, 5000, 2100, 10, 0, 1, 128, 16, BF16),               # 8
    (1, 120000, 40000, 1000, 20000, 2, 64, 64, I8),         # 8: all of it, the first step in place
    (1, 110001, 110000, 0, 0, 1, 64, 256, F16),             # 8: one goes
]


@pytest.mark.parametrize("case", EVICT_LONG, ids=[str(i) for i in range(len(EVICT_LONG))])
def test_evict_in_several_steps(sm100, case):
    B, top, keep, recent, first, Hkv, d, page, kind = case
    g = torch.Generator().manual_seed(B)
    lens = [top] + [int(torch.randint(top // 2, top + 1, (1,), generator=g)) for _ in range(B - 1)]
    c, table, w = _long_cache(lens, Hkv, d, page, kind, seed=B)
    want, w2 = evicted_whole(c, table, w, lens, keep, recent, first, page)
    n2 = fa.kvcache_evict_paged(c["k"].view(kind), c["v"].view(kind), w, table, lens, keep, recent=recent, first=first,
                                k_scale=c["k_scale"], v_scale=c["v_scale"])
    assert n2.tolist() == [min(n, keep) for n in lens]
    assert torch.equal(w.view(torch.int32), w2.view(torch.int32))
    for x in want:
        if want[x] is not None:
            assert torch.equal(c[x], want[x]), x
