"""Measured cases of three further operators over the paged KV cache.

  prefix   attention of a batch whose sequences share long prefixes: the packed
           rows [cu_prefix[g], cu_prefix[g + 1]) see all keys of prefix g and
           their own sequence's keys (causally: those up to their own position)
  weights  the attention weight every cached key received from the new tokens,
           summed over them and over the query heads of its KV head, added to
           the sums of earlier steps
  evict    per sequence and KV head the cache is cut to `keep` positions: the
           first few, the most recent ones and, of the rest, those of the largest
           summed weight (ties: the earlier position); their rows move together
           in order of position

Position p of sequence b (or prefix g) is row p % page of page table[b, p //
page]; sequence b brings n_b = cu[b + 1] - cu[b] new tokens, its last ones.
"""
import math
import os
import random
import sys

import torch

own = False

_QMAX = {"int8": 127.0, "e4m3": 448.0}
_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8,
          "e4m3": torch.float8_e4m3fn}


def _package():
    """This repository's package (its folder is not a package name)."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    folder = os.path.join(root, "flash-attention-sm75-register-fused_b200")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import flash_attention_sm75
    return flash_attention_sm75


# ------------------------------------------------------------------ cases

def _case(name, op, B, Hq, Hkv, d, nq, nk, page, io, cache, order="head", ragged=0, **more):
    """B sequences of nq new tokens and nk own keys with them (ragged != 0: upper
    bounds, drawn per sequence from this number); io: type of q and results, cache:
    type of the pages; order: "head" pages are [Hkv, page, d] in memory, "token"
    pages [page, Hkv, d].  prefix: `prefixes` of up to `length` keys, `loose`
    sequences at the end without one.  weights: `mode`, `causal`.  evict: `keep`,
    `recent`, `first`."""
    c = dict(op=op, B=B, Hq=Hq, Hkv=Hkv, d=d, nq=nq, nk=nk, page=page, io=io, cache=cache,
             order=order, ragged=ragged, **more)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # eight users behind one short system prompt, first answers: latency
        _case("prefix-decode-b8-1k", "prefix", 8, 32, 8, 128, 1, 64, 16, "f16", "f16",
              prefixes=1, length=1024, loose=0),
        # a decode step of 64 users behind an 8k prompt, turns of different lengths
        _case("prefix-decode-b64-8k", "prefix", 64, 32, 8, 128, 1, 1024, 16, "bf16", "bf16", ragged=3,
              prefixes=1, length=8192, loose=0),
        # samples of a long document in 8-bit pages
        _case("prefix-decode-b48-16k-e4m3", "prefix", 48, 32, 8, 128, 1, 400, 64, "bf16", "e4m3", ragged=5,
              prefixes=1, length=16384, loose=0),
        # three prompts of different lengths, draft tokens, requests without a prompt, d = 64
        _case("prefix-groups-draft4-d64", "prefix", 32, 16, 16, 64, 4, 900, 32, "f16", "f16", order="token",
              ragged=7, prefixes=3, length=4096, loose=3),
        # the questions of eight users prefilled behind a common 8k prompt
        _case("prefix-chunks-8x512-8k", "prefix", 8, 32, 8, 128, 512, 512, 16, "bf16", "bf16",
              prefixes=1, length=8192, loose=0),
        # one user, a short prompt, one token: latency
        _case("weights-token-b1-short", "weights", 1, 32, 8, 128, 1, 300, 16, "f16", "f16",
              mode="append", causal=True),
        # a decode step of sixteen users at 8k
        _case("weights-token-b16-8k", "weights", 16, 32, 8, 128, 1, 8192, 16, "bf16", "bf16",
              mode="append", causal=True),
        # continuous batching over int8 pages, a few draft tokens, grouped heads
        _case("weights-draft3-b32-int8", "weights", 32, 32, 8, 128, 3, 8192, 16, "bf16", "int8", ragged=9,
              mode="append", causal=True),
        # prompts in chunks: the last 1024 tokens of 8k
        _case("weights-chunk1024-b2-8k", "weights", 2, 32, 8, 128, 1024, 8192, 16, "bf16", "bf16",
              mode="append", causal=True),
        # one user's cache halved
        _case("evict-b1-1k", "evict", 1, 32, 8, 128, 1, 1024, 16, "f16", "f16", keep=512, recent=64, first=4),
        # ragged long caches cut to a budget
        _case("evict-b32-8k-to-2k", "evict", 32, 32, 8, 128, 1, 8192, 16, "bf16", "bf16", ragged=11,
              keep=2048, recent=256, first=4),
        # one very long int8 cache, read back afterwards
        _case("evict-read-b2-64k-int8", "evict", 2, 32, 8, 128, 1, 65536, 64, "bf16", "int8",
              keep=16384, recent=1024, first=0),
    ]


def _log_int(r, lo, hi):
    n = int(round(math.exp(r.uniform(math.log(lo), math.log(hi))))) if hi > lo else lo
    return max(lo, min(hi, n))


def _some_int(r, hi):
    """A length in 1 .. hi: mostly spread evenly, sometimes over the logarithm."""
    return _log_int(r, 1, hi) if r.random() < 0.3 else r.randint(1, hi)


def _lengths(case):
    """[(new tokens, own keys with them)] of the case's sequences."""
    B, nq, nk = case["B"], case["nq"], case["nk"]
    if not case["ragged"]:
        return [(nq, nk)] * B
    r = random.Random(case["ragged"])
    out = []
    for b in range(B):
        n, m = _some_int(r, nk), _some_int(r, nq)
        if b == 0:
            n, m = nk, nq
        m = min(m, n)
        if b > 2 and r.random() < 0.08:
            m, n = 0, 0  # a slot of the batch without a sequence
        out.append((m, n))
    return out


def _groups(case):
    """[(first sequence, past the last, prefix length)]: equal shares of the
    sequences with a prefix (ragged: cut at random places, lengths drawn)."""
    n = case["B"] - case["loose"]
    P = case["prefixes"]
    if not case["ragged"]:
        cuts = [n * g // P for g in range(P + 1)]
        return [(cuts[g], cuts[g + 1], case["length"]) for g in range(P)]
    r = random.Random(case["ragged"] + 1)
    cuts = [0] + sorted(r.randint(0, n) for _ in range(P - 1)) + [n]
    return [(cuts[g], cuts[g + 1], case["length"] if g == 0 else _some_int(r, case["length"]))
            for g in range(P)]


def draw(rng):
    top = max(_cost(c) for c in listed())
    while True:
        d = rng.choice((64, 128, 128))
        Hkv = rng.choice((1, 2, 4, 8, 8, 16))
        G = rng.choice((1, 2, 3, 4, 4, 7, 8))
        io = rng.choice(("f16", "bf16"))
        cache = rng.choice((io, io, "int8", "e4m3"))
        page = rng.choice((16, 16, 32, 48, 64, 128, 256))
        order = rng.choice(("head", "head", "token"))
        op = rng.choice(("prefix", "weights", "evict"))
        B = _log_int(rng, 1, 128 if op == "prefix" else 64)
        ragged = rng.randrange(1, 1 << 20) if B > 1 and rng.random() < 0.7 else 0
        nq = rng.choice((1, 1, _log_int(rng, 2, 8), _log_int(rng, 9, 1024)))
        more = {}
        if op == "prefix":
            nk = _log_int(rng, 1, 2048)
            loose = rng.choice((0, 0, B // 8))
            more = dict(prefixes=min(rng.choice((1, 1, 2, 3, 5)), B - loose), length=_log_int(rng, 16, 16384),
                        loose=loose)
        elif op == "weights":
            nk = _log_int(rng, 1, 65536 if B == 1 else 8192)
            more = dict(mode=rng.choice(("append", "append", "add", "set")), causal=rng.random() < 0.9)
        else:
            nk = _log_int(rng, 16, 65536 if B <= 2 else 8192)
            keep = _log_int(rng, 1, nk)
            more = dict(keep=keep, recent=rng.randint(0, keep) // rng.choice((1, 4, 16)),
                        first=rng.choice((0, 0, 4, 16)))
            nq = 1
        c = _case(None, op, B, G * Hkv, Hkv, d, min(nq, nk), nk, page, io, cache, order, ragged, **more)
        keys = B * nk + (more["prefixes"] * more["length"] if op == "prefix" else 0)
        scores = 0
        if op == "prefix":
            scores = B * G * Hkv * c["nq"] * (nk + more["length"]) * 4
        elif op == "weights":
            scores = B * G * Hkv * c["nq"] * nk * 4
        if _cost(c) <= top and scores <= 6 << 30 and keys * Hkv * d <= 1 << 29:
            return c


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)


def work(case):
    """The bytes and flops no implementation does without."""
    lens = _lengths(case)
    Hq, Hkv, d = case["Hq"], case["Hkv"], case["d"]
    row = d + 4 if case["cache"] in _QMAX else d * 2  # one cached row of K or V
    tokens = sum(m for m, _ in lens)
    keys = sum(n for m, n in lens if m)
    pairs = sum(m * (n - m) + m * (m + 1) // 2 for m, n in lens)
    if case["op"] == "prefix":
        for b0, b1, n in _groups(case):
            m = sum(m for m, _ in lens[b0:b1])
            keys += n if m else 0
            pairs += m * n
        return {"bytes": keys * Hkv * 2 * row + tokens * Hq * (2 * 2 * d + 4), "flops": 4 * d * Hq * pairs}
    if case["op"] == "weights":
        if not case["causal"]:
            pairs = sum(m * n for m, n in lens)
        rw = 4 if case["mode"] == "set" else 8
        return {"bytes": keys * Hkv * (row + rw) + tokens * Hq * (2 * d + 4), "flops": 2 * d * Hq * pairs}
    cut = [n for _, n in lens if n > case["keep"]]
    moved = len(cut) * max(case["keep"] - case["first"], 0)
    out = sum(cut) * Hkv * 4 + moved * Hkv * (2 * 2 * row + 4)
    if case["cache"] in _QMAX:  # and read back
        out += sum(min(n, case["keep"]) for _, n in lens) * Hkv * 2 * (row + 2 * d)
    return {"bytes": out, "flops": 0}


# ------------------------------------------------------------------ inputs

def _quantise(x, kind):
    """(8-bit values, scales) of rows x[..., d]."""
    a = x.float().abs().amax(-1)
    y = x.float() * (_QMAX[kind] / a)[..., None]
    if kind == "int8":
        return torch.round(y).clamp(-127, 127).to(torch.int8), a / _QMAX[kind]
    return y.clamp(-448, 448).to(torch.float8_e4m3fn), a / _QMAX[kind]


def _table(need, perm, first):
    """Block table of sequences of `need` pages out of perm[first:]; unused entries are 0."""
    dev = perm.device
    width = max(max(need), 1)
    start = torch.tensor([first + sum(need[:b]) for b in range(len(need))], device=dev)
    col = torch.arange(width, device=dev)
    used = col[None] < torch.tensor(need, device=dev)[:, None]
    at = (start[:, None] + col[None]).clamp(max=perm.numel() - 1)
    return torch.where(used, perm[at], torch.zeros_like(perm[at]))


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    lens = _lengths(case)
    B, Hq, Hkv, d, page = (case[k] for k in ("B", "Hq", "Hkv", "d", "page"))
    io = _TYPES[case["io"]]
    tokens = sum(m for m, _ in lens)
    groups = _groups(case) if case["op"] == "prefix" else []
    need = [-(-n // page) for _, n in lens]
    need_p = [-(-n // page) for _, _, n in groups]
    pages = sum(need) + sum(need_p) + 1
    perm = torch.randperm(pages, generator=g, device=dev).to(torch.int32)

    def cache(kind):
        """One cache [pages, Hkv, page, d] in the case's memory order, with stale rows of
        earlier requests in it; keys have a few large channels as trained models do."""
        shape = (pages, Hkv, page, d) if case["order"] == "head" else (pages, page, Hkv, d)
        x = torch.randn(shape, generator=g, device=dev, dtype=torch.float32)
        if kind == "k":
            x[..., ::17] *= 3.0
        if case["cache"] in _QMAX:
            y, s = _quantise(x, case["cache"])
        else:
            y, s = x.to(io), None
        if case["order"] == "token":
            y = y.transpose(1, 2)
            s = s.transpose(1, 2) if s is not None else None
        return y, s

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    kc, ks = cache("k")
    vc, vs = cache("v")
    cu = [sum(m for m, _ in lens[:b]) for b in range(B + 1)]
    st = dict(case=case, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, table=_table(need, perm, 0),
              tokens=tokens, cu=ints(cu), lens=ints([n for _, n in lens]), max_q=max(m for m, _ in lens),
              max_k=max(n for _, n in lens), io=io)
    if case["op"] == "prefix":
        st["prefix_table"] = _table(need_p, perm, sum(need))
        st["rows"] = [cu[b] for b, _, _ in groups] + [cu[groups[-1][1]]]
        st["cu_prefix"] = ints(st["rows"])
        st["prefix_sizes"] = [n for _, _, n in groups]
        st["prefix_lens"] = ints(st["prefix_sizes"])
        st["max_prefix_q"] = max(b - a for a, b in zip(st["rows"], st["rows"][1:]))
        st["max_prefix_k"] = max(st["prefix_sizes"])
    if case["op"] != "evict":
        st["q"] = torch.randn((tokens, Hq, d), generator=g, device=dev).to(io)
    if case["op"] == "weights":
        # what the attention before this call returned, and the sums of earlier steps
        s, see, _, at, live = _scores(st)
        lse = torch.logsumexp(s.masked_fill(~see, float("-inf")), -1)     # [B, h, g, q]
        st["lse"] = torch.full((Hq, tokens), float("-inf"), device=dev)
        st["lse"][:, at[live]] = lse.permute(1, 2, 0, 3).reshape(Hq, B, st["max_q"])[:, live]
    if case["op"] != "prefix":
        # sums over many steps: a few keys have most of the weight, some underflowed
        w = torch.randn((B, Hkv, st["table"].size(1) * page), generator=g, device=dev).mul_(2.0).exp_()
        w[torch.rand(w.shape, generator=g, device=dev) < 0.05] = 0.0
        st["weights"] = w
    if case["op"] == "evict":
        st["kept"] = [min(n, case["keep"]) for _, n in lens]
        st["cu_kept"] = ints([sum(st["kept"][:b]) for b in range(B + 1)])
    return st


# ------------------------------------------------------------------ plain forms

def _rows(st, cache, scale, pg, row):
    """fp32 rows of the cache at (page, row): [..., Hkv, d]."""
    if scale is None:
        return cache[pg, :, row].float()
    # (indexing is not defined for 8-bit floats: their bytes are gathered)
    y = cache.view(torch.int8)[pg, :, row].view(cache.dtype).float()
    return y * scale[pg, :, row][..., None]


def _scores(st):
    """Scores [B, Hkv, G, q, k] of the new tokens with their own keys (padded), which
    of them count, the keys' places, and the packed row of (sequence, token) with those
    that exist."""
    c = st["case"]
    dev = st["cu"].device
    B, Hq, Hkv, d, page = (c[k] for k in ("B", "Hq", "Hkv", "d", "page"))
    nq = (st["cu"][1:] - st["cu"][:-1]).long()
    nk = st["lens"].long()
    qi = torch.arange(st["max_q"], device=dev)
    ki = torch.arange(st["max_k"], device=dev)
    live = qi[None] < nq[:, None]                                  # [B, q]
    at = (st["cu"][:-1].long()[:, None] + qi[None]).clamp(max=max(st["tokens"] - 1, 0))
    q = st["q"][at].float().view(B, st["max_q"], Hkv, Hq // Hkv, d)
    pg, row = st["table"][:, ki // page].long(), (ki % page).expand(B, -1)
    k = _rows(st, st["k_cache"], st["k_scale"], pg, row)           # [B, k, Hkv, d]
    s = torch.einsum("bqhgd,bkhd->bhgqk", q, k) * (1.0 / math.sqrt(d))
    held = ki[None] < nk[:, None]                                  # [B, k]
    see = held[:, None, :] & live[:, :, None]
    if c.get("causal", True):
        see = see & (ki[None, None] <= qi[None, :, None] + (nk - nq)[:, None, None])
    return s, see[:, None, None], (pg, row, held), at, live


def _softmax_parts(s, see):
    """Row maxima (0 where there is no key), exponentials and their sums."""
    s = s.masked_fill(~see, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    return m[..., 0], p, p.sum(-1)


def _plain_prefix(st):
    c = st["case"]
    dev = st["cu"].device
    B, Hq, Hkv, d, page = (c[k] for k in ("B", "Hq", "Hkv", "d", "page"))
    G = Hq // Hkv
    T = st["tokens"]
    # own keys: maximum, sum and unnormalised result of every packed row
    s, see, (pg, row, held), at, live = _scores(st)
    m1, p, l1 = _softmax_parts(s, see)
    v = _rows(st, st["v_cache"], st["v_scale"], pg, row) * held[:, :, None, None]
    o1 = torch.einsum("bhgqk,bkhd->bqhgd", p, v)
    del s, p
    m = torch.full((T, Hkv, G), float("-inf"), device=dev)
    l = torch.zeros((T, Hkv, G), device=dev)
    o = torch.zeros((T, Hkv, G, d), device=dev)
    m[at[live]] = m1.permute(0, 3, 1, 2)[live]
    l[at[live]] = l1.permute(0, 3, 1, 2)[live]
    o[at[live]] = o1[live]
    # the prefix of every group of rows, once for all of them
    for i, n in enumerate(st["prefix_sizes"]):
        rows = slice(st["rows"][i], st["rows"][i + 1])
        ki = torch.arange(n, device=dev)
        pg, row = st["prefix_table"][i, ki // page].long(), ki % page
        k = _rows(st, st["k_cache"], st["k_scale"], pg, row)
        v = _rows(st, st["v_cache"], st["v_scale"], pg, row)
        q = st["q"][rows].float().view(-1, Hkv, G, d)
        s = torch.einsum("thgd,khd->thgk", q, k) * (1.0 / math.sqrt(d))
        m2, p, l2 = _softmax_parts(s, torch.ones((), dtype=torch.bool, device=dev))
        o2 = torch.einsum("thgk,khd->thgd", p, v)
        top = torch.maximum(m[rows], m2)
        f1, f2 = torch.exp(m[rows] - top), torch.exp(m2 - top)
        m[rows] = top
        l[rows] = l[rows] * f1 + l2 * f2
        o[rows] = o[rows] * f1[..., None] + o2 * f2[..., None]
    o = o / torch.where(l > 0, l, torch.ones_like(l))[..., None]
    return o.view(T, Hq, d).to(st["io"]), (m + torch.log(l)).view(T, Hq).T.contiguous()


def _plain_weights(st):
    c = st["case"]
    B, Hq, Hkv = c["B"], c["Hq"], c["Hkv"]
    s, see, (_, _, held), at, live = _scores(st)
    lse = st["lse"][:, at].view(Hkv, Hq // Hkv, B, -1).permute(2, 0, 1, 3)
    see = see & (lse != float("-inf"))[..., None]
    p = torch.exp((s - lse[..., None]).masked_fill(~see, float("-inf")))
    new = p.sum((2, 3))                                            # [B, Hkv, k]
    w = st["weights"][:, :, :st["max_k"]]
    nq = (st["cu"][1:] - st["cu"][:-1]).long()
    ki = torch.arange(st["max_k"], device=w.device)
    if c["mode"] == "set":
        old = torch.zeros_like(w)
    elif c["mode"] == "add":
        old = w
    else:  # the new tokens' own positions start at 0
        old = torch.where((ki[None] < (st["lens"] - nq)[:, None])[:, None], w, torch.zeros_like(w))
    w.copy_(torch.where(held[:, None], old + new, w))


def _plain_evict(st):
    c = st["case"]
    dev = st["lens"].device
    B, Hkv, page, keep = c["B"], c["Hkv"], c["page"], c["keep"]
    n = st["lens"].long()
    L = st["max_k"]
    pos = torch.arange(L, device=dev)
    first = min(c["first"], keep)
    recent = min(c["recent"], keep - first)
    w = st["weights"][:, :, :L]
    w = torch.where(w.isnan(), torch.full_like(w, float("-inf")), w)
    # rank: always kept, then by weight (a stable order: ties to the lower position), then
    # what is not held
    sure = (pos[None] < first) | (pos[None] >= (n - recent)[:, None])
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices
    cls = torch.where(pos[None] >= n[:, None], 2, torch.where(sure, 0, 1))[:, None].expand(B, Hkv, L)
    by_class = torch.sort(cls.gather(-1, order), dim=-1, stable=True).indices
    order = order.gather(-1, by_class)
    width = min(keep, L)
    kept = torch.sort(order[..., :width], dim=-1).values           # [B, Hkv, width]
    dst = torch.arange(width, device=dev)
    new_len = torch.minimum(n, torch.full_like(n, keep))
    ok = (dst[None] < new_len[:, None]) & (n > keep)[:, None]      # rows that may move
    b, h, i = ok[:, None].expand(B, Hkv, width).nonzero(as_tuple=True)
    src = kept[b, h, i]
    spg, srow = st["table"][b, src // page].long(), src % page
    dpg, drow = st["table"][b, i // page].long(), i % page
    for x in (st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"]):
        if x is not None:
            x = x.view(torch.int8) if x.element_size() == 1 else x
            x[dpg, h, drow] = x[spg, h, srow]
    st["weights"][b, h, i] = st["weights"][b, h, src]
    return new_len.to(torch.int32)


def _plain_read_kept(st):
    page = st["case"]["page"]
    dev = st["lens"].device
    n = torch.tensor(st["kept"], device=dev)
    b = torch.repeat_interleave(torch.arange(len(st["kept"]), device=dev), n)
    pos = torch.arange(b.numel(), device=dev) - st["cu_kept"].long()[b]
    pg, row = st["table"][b, pos // page].long(), pos % page
    return (_rows(st, st["k_cache"], st["k_scale"], pg, row).to(st["io"]),
            _rows(st, st["v_cache"], st["v_scale"], pg, row).to(st["io"]))


# ------------------------------------------------------------------ one pass

def run(state):
    c = state["case"]
    op = c["op"]
    eight = c["cache"] in _QMAX
    scales = dict(k_scale=state["k_scale"], v_scale=state["v_scale"])
    if not own:
        if op == "prefix":
            return dict(zip(("o", "lse"), _plain_prefix(state)))
        if op == "weights":
            _plain_weights(state)
            return {"weights": state["weights"]}
        lens = _plain_evict(state)
        out = (dict(zip(("k", "v"), _plain_read_kept(state))) if eight else
               {"k_cache": state["k_cache"], "v_cache": state["v_cache"]})
        return {**out, "weights": state["weights"], "lens": lens}
    fa = _package()
    if op == "prefix":
        o, lse = fa.flash_attention_forward_paged_prefix(
            state["q"], state["k_cache"], state["v_cache"], state["prefix_table"], state["cu_prefix"],
            state["prefix_lens"], state["table"], state["cu"], state["lens"], state["max_prefix_q"],
            state["max_prefix_k"], state["max_q"], state["max_k"], causal=True, return_lse=True, **scales)
        return {"o": o, "lse": lse}
    if op == "weights":
        fa.kvcache_weights_paged(state["q"], state["lse"], state["k_cache"], state["table"], state["cu"],
                                 state["lens"], state["max_q"], state["max_k"], state["weights"],
                                 causal=c["causal"], mode=c["mode"], k_scale=state["k_scale"])
        return {"weights": state["weights"]}
    lens = fa.kvcache_evict_paged(state["k_cache"], state["v_cache"], state["weights"], state["table"],
                                  state["lens"], c["keep"], recent=c["recent"], first=c["first"], **scales)
    if not eight:
        return {"k_cache": state["k_cache"], "v_cache": state["v_cache"], "weights": state["weights"],
                "lens": lens}
    k, v = fa.kvcache_read_paged(state["k_cache"], state["v_cache"], state["table"], state["cu_kept"], lens,
                                 sum(state["kept"]), dtype=state["io"], **scales)
    return {"k": k, "v": v, "weights": state["weights"], "lens": lens}


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    lens = _lengths(case)
    Hq, Hkv, d, page = (case[k] for k in ("Hq", "Hkv", "d", "page"))
    G = Hq // Hkv
    starts = [sum(m for m, _ in lens[:b]) for b in range(len(lens))]

    def held(name, table, b, n):
        """[Hkv, n, d] values that the first n positions of a row of `table` stand for."""
        p = torch.arange(n, device="cuda")
        pg, row = table[b].long()[p // page], p % page
        x, s = st[name + "_cache"], st[name + "_scale"]
        if s is None:
            return x[pg, :, row].double().transpose(0, 1)
        y = x.view(torch.uint8)[pg, :, row].view(x.dtype).double()
        return (y * s[pg, :, row].double().unsqueeze(-1)).transpose(0, 1)

    def queries(b):
        """[Hkv, G m, d], token after token, of sequence b."""
        x = st["q"][starts[b]:starts[b] + lens[b][0]].double()
        return x.view(-1, Hkv, G, d).permute(1, 0, 2, 3).reshape(Hkv, -1, d)

    def own_scores(b, causal):
        m, n = lens[b]
        s = queries(b) @ held("k", st["table"], b, n).transpose(1, 2) / math.sqrt(d)
        if causal:
            i = torch.arange(m, device="cuda").repeat_interleave(G).unsqueeze(1)
            s[:, torch.arange(n, device="cuda") > i + (n - m)] = -math.inf
        return s

    if case["op"] == "prefix":
        o = torch.zeros(st["tokens"], Hq, d, dtype=torch.float64, device="cuda")
        lse = torch.full((Hq, st["tokens"]), -math.inf, dtype=torch.float64, device="cuda")
        prefix = [None] * len(lens)
        for i, (b0, b1, n) in enumerate(_groups(case)):
            kv = (held("k", st["prefix_table"], i, n), held("v", st["prefix_table"], i, n))
            prefix[b0:b1] = [kv] * (b1 - b0)
        for b, (m, n) in enumerate(lens):
            if m == 0:
                continue
            s, v = own_scores(b, True), held("v", st["table"], b, n)
            if prefix[b] is not None:
                s = torch.cat([queries(b) @ prefix[b][0].transpose(1, 2) / math.sqrt(d), s], -1)
                v = torch.cat([prefix[b][1], v], 1)
            z = torch.logsumexp(s, -1)
            x = torch.exp(s - z.unsqueeze(-1)) @ v                 # [Hkv, m G, d]
            rows = slice(starts[b], starts[b] + m)
            o[rows] = x.view(Hkv, m, G, d).transpose(0, 1).reshape(m, Hq, d)
            lse[:, rows] = z.view(Hkv, m, G).transpose(1, 2).reshape(Hq, m)
        return {"o": o, "lse": lse}
    if case["op"] == "weights":
        w = st["weights"].double()
        for b, (m, n) in enumerate(lens):
            total = torch.zeros(Hkv, n, dtype=torch.float64, device="cuda")
            if m:
                z = st["lse"][:, starts[b]:starts[b] + m].double().view(Hkv, G, m).transpose(1, 2)
                total = torch.exp(own_scores(b, case["causal"]) - z.reshape(Hkv, -1, 1)).sum(1)
            base = {"set": 0, "add": n, "append": n - m}[case["mode"]]  # sums that are kept
            w[b, :, base:n] = 0
            w[b, :, :n] += total
        return {"weights": w}
    # evict: the kept positions of one sequence and head at a time
    keep, first = case["keep"], min(case["first"], case["keep"])
    recent = min(case["recent"], keep - first)
    w = st["weights"].double()
    caches = [x.view(torch.uint8).clone().view(x.dtype) if x.element_size() == 1 else x.clone()
              for x in (st["k_cache"], st["v_cache"])]
    rows = {"k": [], "v": []}
    for b, (_, n) in enumerate(lens):
        total = min(n, keep)
        at = []
        for h in range(Hkv):
            mid = w[b, h, first:n - recent] if n > keep else w[b, h, :0]
            best = torch.sort(-mid, stable=True).indices[:keep - first - recent] + first
            ends = [torch.arange(first, device="cuda"), torch.arange(n - recent, n, device="cuda")]
            at.append(torch.sort(torch.cat([*ends, best])).values if n > keep
                      else torch.arange(n, device="cuda"))
        if total == 0:
            continue
        at = torch.stack(at)                                       # [Hkv, total]
        dst = torch.arange(total, device="cuda")
        dpg, drow = st["table"][b].long()[dst // page], dst % page
        for name, cache in zip(("k", "v"), caches):
            x = held(name, st["table"], b, n).gather(1, at.unsqueeze(-1).expand(-1, -1, d))
            if case["cache"] in _QMAX:
                rows[name].append(x.transpose(0, 1))
            else:
                cache[dpg, :, drow] = x.transpose(0, 1).to(cache.dtype)
        w[b, :, :total] = w[b].gather(1, at)
    out = ({name: torch.cat(x) for name, x in rows.items()} if case["cache"] in _QMAX else
           {"k_cache": caches[0].double(), "v_cache": caches[1].double()})
    return {**out, "weights": w, "lens": torch.tensor([min(n, keep) for _, n in lens], device="cuda")}
