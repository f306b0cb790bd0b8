"""Measured cases of the paged KV cache operators.

Three operators over one paged cache (pages of `page` tokens, found through a
block table): writing the keys and values of new tokens (16-bit copies, or
8 bits with one fp32 scale per token and head), reading them back as packed
16-bit rows, and attention of the new tokens over the cached ones (single
tokens, a few draft tokens, chunks, mixtures).

Token i of sequence b, which brings n_b = cu[b+1] - cu[b] tokens, lies at
position nk_b - n_b + i of the sequence; position p is row p % page of page
table[b, p // page].
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
_TINY = 2.0 ** -100  # rows below it are stored as zeros


def _package():
    """This repository's package (its folder is not a package name)."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    folder = os.path.join(root, "flash-attention-sm75-register-fused_b200")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import flash_attention_sm75
    return flash_attention_sm75


# ------------------------------------------------------------------ cases

def _case(name, op, B, Hq, Hkv, d, nq, nk, page, io, cache, order="head", ragged=0, causal=True):
    """B sequences of nq new tokens that end at position nk (ragged != 0: nq
    and nk are upper bounds, drawn per sequence from this number); io: type of
    the new tokens and results, cache: type of the pages; order: "head" pages
    are [Hkv, page, d] in memory, "token" pages [page, Hkv, d]."""
    c = dict(op=op, B=B, Hq=Hq, Hkv=Hkv, d=d, nq=nq, nk=nk, page=page, io=io, cache=cache,
             order=order, ragged=ragged, causal=causal)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one decode step of eight sequences quantised into the cache and read back: latency
        _case("write-read-token-b8-int8", "write_read", 8, 32, 8, 128, 1, 8192, 16, "f16", "int8"),
        # a prefill batch of four prompts copied into bf16 pages
        _case("write-prompts-bf16", "write", 4, 32, 8, 128, 4096, 4096, 16, "bf16", "bf16", ragged=3),
        # the same into e4m3 pages, read back for a model that wants plain rows
        _case("write-read-prompts-e4m3", "write_read", 4, 32, 8, 128, 4096, 8192, 64, "bf16", "e4m3",
              ragged=5),
        # whole ragged int8 prefixes expanded to packed bf16 rows
        _case("read-prefixes-int8", "read", 16, 32, 8, 128, 8192, 8192, 16, "bf16", "int8", ragged=7),
        # token-major f16 pages gathered at d = 64
        _case("read-prefixes-f16-d64", "read", 16, 16, 16, 64, 4096, 4096, 32, "f16", "f16",
              order="token", ragged=9),
        # the shortest attention call: one user, a short prompt, one token
        _case("decode-b1-short", "attend", 1, 32, 8, 128, 1, 300, 16, "f16", "f16"),
        # a decode step of eight users at 8k, grouped heads
        _case("decode-b8-gqa4-8k", "attend", 8, 32, 8, 128, 1, 8192, 16, "f16", "f16"),
        # one long context in 8 bits
        _case("decode-b1-64k-e4m3", "attend", 1, 32, 8, 128, 1, 65536, 64, "bf16", "e4m3"),
        # continuous batching: 32 users of very different lengths, int8 pages
        _case("decode-b32-ragged-int8", "attend", 32, 32, 8, 128, 1, 8192, 16, "bf16", "int8",
              ragged=11),
        # four draft tokens to verify, one KV head per query head, d = 64
        _case("draft4-b16-mha-4k-d64", "attend", 16, 16, 16, 64, 4, 4096, 16, "bf16", "bf16"),
        # a 512-token chunk of a prompt behind an 8k prefix
        _case("chunk512-8k-bf16", "attend", 1, 32, 8, 128, 512, 8192, 16, "bf16", "bf16"),
        # a serving step that mixes chunks, draft tokens and single tokens over 8-bit pages
        _case("mixed-chunks-8k-e4m3", "attend", 6, 32, 8, 128, 1024, 8192, 32, "f16", "e4m3",
              ragged=13),
    ]


def _lengths(case):
    """[(new tokens, cached tokens with them)] of the case's sequences."""
    B, nq, nk = case["B"], case["nq"], case["nk"]
    if not case["ragged"]:
        return [(nq, nk)] * B
    r = random.Random(case["ragged"])
    out = []
    for b in range(B):
        n, m = _some_int(r, nk), _some_int(r, nq)
        if b == 0:
            n, m = nk, nq
        m = n if case["op"] == "read" else min(m, n)  # read: the whole prefix
        if b > 2 and r.random() < 0.08:
            m, n = 0, 0  # a slot of the batch without a sequence
        out.append((m, n))
    return out


def _some_int(r, hi):
    """A length in 1 .. hi: mostly spread evenly, sometimes over the logarithm."""
    n = _log_int(r, 1, hi) if r.random() < 0.3 else r.randint(1, hi)
    return n if n != 3072 else 3071


def _log_int(r, lo, hi):
    n = int(round(math.exp(r.uniform(math.log(lo), math.log(hi))))) if hi > lo else lo
    n = max(lo, min(hi, n))
    return n if n != 3072 else 3071


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
        op = rng.choice(("write", "read", "attend", "attend", "attend", "attend"))
        if op == "write" and cache in _QMAX:
            op = "write_read"
        B = _log_int(rng, 1, 64)
        nk = _log_int(rng, 16, 65536 if B == 1 else 8192)
        if op == "read":
            nq = nk
        elif op == "attend":
            nq = rng.choice((1, 1, _log_int(rng, 2, 8), _log_int(rng, 9, 1024)))
        else:
            nq = rng.choice((1, _log_int(rng, 2, 4096), _log_int(rng, 256, 8192)))
        nq = min(nq, nk)
        ragged = rng.randrange(1, 1 << 20) if B > 1 and rng.random() < 0.7 else 0
        causal = rng.random() < 0.9
        c = _case(None, op, B, G * Hkv, Hkv, d, nq, nk, page, io, cache, order, ragged, causal)
        scores = B * G * Hkv * nq * nk * 4 if op == "attend" else 0
        if _cost(c) <= top and scores <= 6 << 30 and B * nk * Hkv * d <= 1 << 29:
            return c


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)


def work(case):
    """The bytes and flops no implementation does without."""
    lens = _lengths(case)
    Hq, Hkv, d = case["Hq"], case["Hkv"], case["d"]
    row = d * 1 + 4 if case["cache"] in _QMAX else d * 2  # one cached row of K or V
    tokens = sum(m for m, _ in lens)
    if case["op"] == "write":
        return {"bytes": tokens * Hkv * 2 * (2 * d + row), "flops": 0}
    if case["op"] == "read":
        return {"bytes": tokens * Hkv * 2 * (2 * d + row), "flops": 0}
    if case["op"] == "write_read":
        return {"bytes": tokens * Hkv * 2 * 2 * (2 * d + row), "flops": 0}
    keys = sum(n for m, n in lens if m)
    if case["causal"]:
        pairs = sum(m * (n - m) + m * (m + 1) // 2 for m, n in lens)
    else:
        pairs = sum(m * n for m, n in lens)
    return {"bytes": keys * Hkv * 2 * row + tokens * Hq * (2 * 2 * d + 4),
            "flops": 4 * d * Hq * pairs}


# ------------------------------------------------------------------ inputs

def _quantise(x, kind):
    """(8-bit values, scales) of rows x[..., d]."""
    a = x.float().abs().amax(-1)
    keep = a >= _TINY
    inv = torch.where(keep, _QMAX[kind] / a, torch.zeros_like(a))
    scale = torch.where(keep, a / _QMAX[kind], torch.zeros_like(a))
    y = x.float() * inv[..., None]
    if kind == "int8":
        return torch.round(y).clamp(-127, 127).to(torch.int8), scale
    return y.clamp(-448, 448).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    lens = _lengths(case)
    B, Hq, Hkv, d, page = (case[k] for k in ("B", "Hq", "Hkv", "d", "page"))
    io = _TYPES[case["io"]]
    tokens = sum(m for m, _ in lens)
    need = [-(-n // page) for _, n in lens]
    width = max(max(need), 1)
    pages = sum(need) + 1
    # each sequence owns a random set of pages; unused table entries are 0
    perm = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    first = torch.tensor([sum(need[:b]) for b in range(B)], device=dev)
    col = torch.arange(width, device=dev)
    used = col[None] < torch.tensor(need, device=dev)[:, None]
    at = (first[:, None] + col[None]).clamp(max=pages - 1)
    table = torch.where(used, perm[at], torch.zeros_like(perm[at]))

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

    kc, ks = cache("k")
    vc, vs = cache("v")
    st = dict(case=case, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, table=table, tokens=tokens,
              cu=torch.tensor([sum(m for m, _ in lens[:b]) for b in range(B + 1)],
                              dtype=torch.int32, device=dev),
              lens=torch.tensor([n for _, n in lens], dtype=torch.int32, device=dev),
              max_q=max(m for m, _ in lens), max_k=max(n for _, n in lens), io=io)
    # new rows as slices of one projection's output, as a model has them
    if case["op"] == "attend":
        st["q"] = torch.randn((tokens, Hq, d), generator=g, device=dev).to(io)
    if case["op"] in ("write", "write_read"):
        kv = torch.randn((tokens, 2 * Hkv, d), generator=g, device=dev)
        kv[:, :Hkv, ::17] *= 3.0
        kv = kv.to(io)
        st["k"], st["v"] = kv[:, :Hkv], kv[:, Hkv:]
    return st


# ------------------------------------------------------------------ plain forms

def _owner(st):
    """Sequence and position of every new token."""
    i = torch.arange(st["tokens"], device=st["cu"].device)
    b = torch.searchsorted(st["cu"][1:].contiguous(), i.to(torch.int32), right=True)
    n = (st["cu"][1:] - st["cu"][:-1])[b]
    return b, (st["lens"][b] - n + i - st["cu"][b]).long()


def _plain_write(st):
    b, pos = _owner(st)
    page = st["case"]["page"]
    pg, row = st["table"][b, pos // page].long(), pos % page
    for new, cache, scale in ((st["k"], st["k_cache"], st["k_scale"]),
                              (st["v"], st["v_cache"], st["v_scale"])):
        if scale is None:
            cache[pg, :, row] = new
            continue
        y, s = _quantise(new, st["case"]["cache"])
        # (indexing is not defined for 8-bit floats: their bytes are stored)
        cache.view(torch.int8)[pg, :, row] = y.view(torch.int8)
        scale[pg, :, row] = s


def _rows(st, cache, scale, pg, row):
    """fp32 rows of the cache at (page, row): [..., Hkv, d]."""
    if scale is None:
        return cache[pg, :, row].float()
    y = cache.view(torch.int8)[pg, :, row].view(cache.dtype).float()
    return y * scale[pg, :, row][..., None]


def _plain_read(st):
    b, pos = _owner(st)
    page = st["case"]["page"]
    pg, row = st["table"][b, pos // page].long(), pos % page
    return (_rows(st, st["k_cache"], st["k_scale"], pg, row).to(st["io"]),
            _rows(st, st["v_cache"], st["v_scale"], pg, row).to(st["io"]))


def _plain_attend(st):
    c = st["case"]
    dev = st["cu"].device
    B, Hq, Hkv, d, page = (c[k] for k in ("B", "Hq", "Hkv", "d", "page"))
    G = Hq // Hkv
    nq = (st["cu"][1:] - st["cu"][:-1]).long()
    nk = st["lens"].long()
    qi = torch.arange(st["max_q"], device=dev)
    ki = torch.arange(st["max_k"], device=dev)
    live = qi[None] < nq[:, None]                                  # [B, q]
    at = (st["cu"][:-1].long()[:, None] + qi[None]).clamp(max=st["tokens"] - 1)
    q = st["q"][at].float().view(B, st["max_q"], Hkv, G, d)
    pg, row = st["table"][:, ki // page].long(), (ki % page).expand(B, -1)
    k = _rows(st, st["k_cache"], st["k_scale"], pg, row)           # [B, k, Hkv, d]
    v = _rows(st, st["v_cache"], st["v_scale"], pg, row)
    held = ki[None] < nk[:, None]                                  # [B, k]
    v = v * held[:, :, None, None]
    s = torch.einsum("bqhgd,bkhd->bhgqk", q, k) * (1.0 / math.sqrt(d))
    see = held[:, None, :] & live[:, :, None]
    if c["causal"]:
        see = see & (ki[None, None] <= qi[None, :, None] + (nk - nq)[:, None, None])
    s = s.masked_fill(~see[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    p = torch.exp(s - m)
    l = p.sum(-1)                                                  # [B, h, g, q]
    o = torch.einsum("bhgqk,bkhd->bqhgd", p, v)
    o = o / torch.where(l > 0, l, torch.ones_like(l)).permute(0, 3, 1, 2)[..., None]
    lse = m[..., 0] + torch.log(l)
    out = torch.zeros_like(st["q"])
    out[at[live]] = o.reshape(B, st["max_q"], Hq, d)[live].to(st["io"])
    lse_out = torch.full((Hq, st["tokens"]), float("-inf"), device=dev)
    lse_out[:, at[live]] = lse.permute(1, 2, 0, 3).reshape(Hq, B, st["max_q"])[:, live]
    return out, lse_out


# ------------------------------------------------------------------ one pass

def run(state):
    op = state["case"]["op"]
    if not own:
        if op == "attend":
            return dict(zip(("o", "lse"), _plain_attend(state)))
        if op in ("write", "write_read"):
            _plain_write(state)
        if op == "write":
            return {"k_cache": state["k_cache"], "v_cache": state["v_cache"]}
        return dict(zip(("k", "v"), _plain_read(state)))
    fa = _package()
    if op == "attend":
        o, lse = fa.flash_attention_forward_paged(
            state["q"], state["k_cache"], state["v_cache"], state["table"], state["cu"],
            state["lens"], state["max_q"], state["max_k"], causal=state["case"]["causal"],
            k_scale=state["k_scale"], v_scale=state["v_scale"], return_lse=True)
        return {"o": o, "lse": lse}
    if op in ("write", "write_read"):
        fa.kvcache_write_paged(state["k"], state["v"], state["k_cache"], state["v_cache"],
                               state["table"], state["cu"], state["lens"],
                               k_scale=state["k_scale"], v_scale=state["v_scale"])
    if op == "write":
        return {"k_cache": state["k_cache"], "v_cache": state["v_cache"]}
    k, v = fa.kvcache_read_paged(state["k_cache"], state["v_cache"], state["table"], state["cu"],
                                 state["lens"], state["tokens"], k_scale=state["k_scale"],
                                 v_scale=state["v_scale"], dtype=state["io"])
    return {"k": k, "v": v}


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    lens = _lengths(case)
    Hq, Hkv, d, page = (case[k] for k in ("Hq", "Hkv", "d", "page"))
    starts = [sum(m for m, _ in lens[:b]) for b in range(len(lens))]

    def places(b, lo, hi):
        p = torch.arange(lo, hi, device="cuda")
        return st["table"][b].long()[p // page], p % page

    def held(name, b, lo, hi):
        """[Hkv, n, d] values that positions [lo, hi) of sequence b stand for."""
        pg, row = places(b, lo, hi)
        x, s = st[name + "_cache"], st[name + "_scale"]
        bits = x if s is None else x.view(torch.uint8)
        y = bits[pg, :, row]
        y = (y if s is None else y.view(x.dtype)).double()
        if s is not None:
            y = y * s[pg, :, row].double().unsqueeze(-1)
        return y.transpose(0, 1)

    def stands_for(x):
        """64-bit values that rows x stand for once quantised."""
        x = x.double()
        a = x.abs().amax(-1, keepdim=True)
        unit = a / _QMAX[case["cache"]]
        y = torch.where(a >= _TINY, x / unit, torch.zeros_like(x))
        if case["cache"] == "int8":
            return torch.round(y) * unit
        # e4m3: 4 significant bits, smallest exponent -6
        e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
        q = torch.exp2(e - 3)
        return torch.round(y / q) * q * unit

    if case["op"] == "write":
        out = {}
        for name in ("k", "v"):
            c = st[name + "_cache"].double()
            for b, (m, n) in enumerate(lens):
                pg, row = places(b, n - m, n)
                c[pg, :, row] = st[name][starts[b]:starts[b] + m].double()
            out[name + "_cache"] = c
        return out
    if case["op"] == "write_read":
        return {name: stands_for(st[name]) for name in ("k", "v")}
    if case["op"] == "read":
        return {name: torch.cat([held(name, b, n - m, n).transpose(0, 1)
                                 for b, (m, n) in enumerate(lens)]) for name in ("k", "v")}
    o = torch.zeros(st["tokens"], Hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((Hq, st["tokens"]), -math.inf, dtype=torch.float64, device="cuda")
    for b, (m, n) in enumerate(lens):
        if m == 0 or n == 0:
            continue
        k, v = held("k", b, 0, n), held("v", b, 0, n)
        rows = slice(starts[b], starts[b] + m)
        for h in range(Hq):
            s = st["q"][rows, h].double() @ k[h * Hkv // Hq].T / math.sqrt(d)
            if case["causal"]:
                i = torch.arange(m, device="cuda").unsqueeze(1)
                s[torch.arange(n, device="cuda") > i + (n - m)] = -math.inf
            z = torch.logsumexp(s, -1)
            lse[h, rows] = z
            o[rows, h] = torch.exp(s - z.unsqueeze(-1)) @ v[h * Hkv // Hq]
    return {"o": o, "lse": lse}
