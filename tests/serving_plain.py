"""Plain 64-bit forms of attention behind shared prefixes, of summed attention
weights and of eviction over a paged cache (CPU; no code of the package).  The caches
are those of tests/paged_plain.py; prefixes are further sequences of them without
new tokens, rows B .. of the table."""
import math

import torch

from tests.paged_plain import QMAX, UNIT, Paged, bits


def with_prefixes(lens, prefixes, *args, **kw):
    """A cache that holds the sequences `lens` and prefixes of the given lengths."""
    P = Paged(list(lens) + [(0, n) for n in prefixes], *args, **kw)
    P.B, P.prefixes = len(lens), list(prefixes)
    return P


def split(P, c):
    """The arguments of a call from P.cuda(): the sequences' and the prefixes' tables."""
    B = P.B
    return dict(table=c["table"][:B], cu=c["cu"][:B + 1].contiguous(), lens=c["lens"][:B].contiguous(),
                prefix_table=c["table"][B:], prefix_lens=c["lens"][B:].contiguous())


def see_mask(m, n, mode):
    i, j = torch.arange(m)[:, None], torch.arange(n)[None]
    if mode == 0:
        return torch.ones(m, n, dtype=torch.bool)
    return j <= i + (n - m if mode == 1 else 0)


def prefix_attention(P, q, Hq, rows, mode, scale=None, max_prefix_q=None, max_prefix_k=None):
    """O [total, Hq, d], LSE [Hq, total] in 64 bits with the bounds on their errors
    (derived in paged_plain.attention: P rounded to 16 bits, O once, exponentials good
    to 1e-4, 8-bit queries or keys rounded to f16 once).  Two passes are joined
    in fp32, which adds some units of 2^-24 to weights that sum to 1: below the 1e-6
    and 1e-4 that the bounds end with.  That bound takes a score for exact; its products are,
    but their sum in fp32, in any order and with truncation, is off by at most d 2^-23
    sum |q k|, and its scaling, the conversion to log2 units and back by 2^-22 |s|:
    `ds` has these too, for scores of a hundred and more they are most of it.  `rows`: prefix g is seen by rows [rows[g], rows[g + 1])."""
    d = P.d
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    eight = P.cache in QMAX
    u = UNIT[torch.float16] if eight else UNIT[P.io]
    G = Hq // P.Hkv
    o = torch.zeros(P.total, Hq, d, dtype=torch.float64)
    lse = torch.full((Hq, P.total), -math.inf, dtype=torch.float64)
    tol = torch.zeros_like(o)
    tol_lse = torch.full_like(lse, 1e-4)

    def keys(b, n):
        return tuple(P.held(x, b, n).repeat_interleave(G, 1).transpose(0, 1) for x in ("k", "v"))

    for b in range(P.B):
        m, n = P.lens[b]
        if m == 0:
            continue
        own = see_mask(m, n, mode)
        for g in [None] + list(range(len(P.prefixes))):
            # the tokens of b that see prefix g (None: no prefix)
            t = torch.arange(P.cu[b], P.cu[b + 1])
            owner = torch.full_like(t, -1)
            for x in range(len(P.prefixes)):
                end = rows[x + 1] if max_prefix_q is None else min(rows[x + 1], rows[x] + max_prefix_q)
                owner[(t >= rows[x]) & (t < end)] = x
            mine = owner == (-1 if g is None else g)
            if not mine.any():
                continue
            k, v = keys(b, n)
            see = own[mine]
            if g is not None:
                np_ = P.prefixes[g] if max_prefix_k is None else min(P.prefixes[g], max_prefix_k)
                k2, v2 = keys(P.B + g, np_)
                k, v = torch.cat([k2, k], 1), torch.cat([v2, v], 1)
                see = torch.cat([torch.ones(see.size(0), np_, dtype=torch.bool), see], 1)
            if k.size(1) == 0:
                continue
            at = t[mine]
            x = q[at].double().transpose(0, 1)
            s = (x @ k.transpose(1, 2) * scale).masked_fill(~see, -math.inf)
            z = torch.logsumexp(s, -1)
            p = torch.exp(s - torch.where(z == -math.inf, torch.zeros_like(z), z)[..., None])
            ob, a = p @ v, p @ v.abs()
            size = (x.abs() @ k.abs().transpose(1, 2)).masked_fill(~see, 0).amax(-1) * abs(scale)
            ds = size * (d * 2.0 ** -23 + 2.0 ** -22 + (u if eight else 0))
            o[at], lse[:, at] = ob.transpose(0, 1), z
            tol[at] = (UNIT[P.io] * ob.abs() + a * (2 * u + 2e-4 + 4 * ds)[..., None] + 1e-6).transpose(0, 1)
            tol_lse[:, at] = 1e-4 + 2 * ds
    return o, lse, tol, tol_lse


def summed_weights(P, q, lse, Hq, mode, old, kind, scale=None, max_q=None, max_k=None):
    """weights [B, Hkv, L] in 64 bits after the call, and the bound on their errors.

    A term is 2^(s' - L'), s' and L' the score and the LSE times log2 e.  The
    products of 16-bit values are exact in fp32; their sum over d, in any order and
    with truncation, is off by at most d 2^-23 sum |q k|.  Scaling, the conversion
    of the LSE and the difference round three times, 2^-24 (|s| + |LSE|) each (and
    8-bit keys' scale once more); the exponential is good to 2^-22.  So a term p is
    off by p (d 2^-23 |scale| sum |q k| + 2^-22 (|s| + |LSE|) + 2^-21), and adding R
    terms and the old sum by (R + 1) 2^-24 of them.  Terms below 2^-126 may be 0."""
    d, G = P.d, Hq // P.Hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    w = old.double().clone()
    tol = torch.zeros_like(w)
    for b, (m, n) in enumerate(P.lens):
        nk = n if max_k is None else min(n, max_k)
        mq = m if max_q is None else min(m, max_q)
        see = see_mask(m, n, mode)[:mq, :nk]
        k = P.held("k", b, nk).transpose(0, 1)                              # [Hkv, nk, d]
        rows = slice(P.cu[b], P.cu[b] + mq)
        x = q[rows].double().view(mq, P.Hkv, G, d).permute(1, 0, 2, 3)      # [Hkv, mq, G, d]
        z = lse[:, rows].double().view(P.Hkv, G, mq).transpose(1, 2)        # [Hkv, mq, G]
        s = torch.einsum("hmgd,hkd->hmgk", x, k) * scale
        size = torch.einsum("hmgd,hkd->hmgk", x.abs(), k.abs()) * abs(scale)
        ok = see[None, :, None] & (z != -math.inf)[..., None]
        zz = torch.where(z == -math.inf, torch.zeros_like(z), z)[..., None]
        p = torch.where(ok, torch.exp(s - zz), torch.zeros_like(s))
        rel = d * 2.0 ** -23 * size + 2.0 ** -22 * (s.abs() + zz.abs()) + 2.0 ** -21
        new = p.sum((1, 2))
        fresh = {"set": 0, "add": n, "append": max(n - m, 0)}[kind]
        base = w[b, :, :nk].clone()
        base[:, fresh:] = 0
        w[b, :, :nk] = base + new
        R = mq * G
        tol[b, :, :nk] = ((p * torch.where(ok, rel, torch.zeros_like(rel))).sum((1, 2)) +
                          (R + 1) * 2.0 ** -24 * (base.abs() + new) + R * 2.0 ** -126)
    return w, tol


def evicted(P, weights, keep, recent, first):
    """(k, v, k_scale, v_scale, weights, lens) after the call, bit by bit."""
    out = [None if x is None else bits(x).clone() for x in (P.k, P.v, P.ks, P.vs)]
    w = weights.clone()
    lens = []
    for b, (_, n) in enumerate(P.lens):
        kp = max(keep if isinstance(keep, int) else int(keep[b]), 0)
        lens.append(min(n, kp))
        if n <= kp:
            continue
        f = min(first, kp)
        r = min(recent, kp - f)
        for h in range(P.Hkv):
            mid = list(range(f, n - r))
            key = {j: -math.inf if math.isnan(weights[b, h, j]) else float(weights[b, h, j]) for j in mid}
            # (a NaN is below every number, -inf too)
            mid.sort(key=lambda j: (math.isnan(weights[b, h, j]), -key[j], j))
            at = sorted(list(range(f)) + mid[:kp - f - r] + list(range(n - r, n)))
            rows = [P.place(b, j) for j in at]
            for x, src in zip(out, (P.k, P.v, P.ks, P.vs)):
                if x is None:
                    continue
                held = bits(src)
                for i, (pg, row) in enumerate(rows):
                    dpg, drow = P.place(b, i)
                    x[dpg, h, drow] = held[pg, h, row]
            w[b, h, :kp] = weights[b, h, at]
    return (*out, w, lens)


def evicted_whole(c, table, w, lens, keep, recent, first, page):
    """The same for long caches: whole sequences at a time, bit by bit.  c: name -> [pages, Hkv, page,
    ...] (or None) on any device; returns (caches, weights)."""
    out = {x: None if y is None else y.clone() for x, y in c.items()}
    w2 = w.clone()
    h = torch.arange(w.size(1), device=w.device)[:, None]
    for b, n in enumerate(lens):
        if n <= keep:
            continue
        f = min(first, keep)
        r = min(recent, keep - f)
        x = w[b, :, :n].double() + 0.0  # (-0 is 0)
        # (beyond every fp32 number: what stays whatever its weight above +inf, a NaN below -inf)
        x = torch.where(x == math.inf, 1e39, torch.where(x == -math.inf, -1e39, x))
        x = torch.where(x.isnan(), -math.inf, x)
        x[:, :f] = math.inf
        x[:, n - r:] = math.inf
        best = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :keep]
        at = torch.sort(best, dim=-1).values
        dst = torch.arange(keep, device=w.device)
        pg = table[b].long()
        for name, src in c.items():
            if src is not None:
                out[name][pg[dst // page], h, dst % page] = src[pg[at // page], h, at % page]
        w2[b, :, :keep] = w[b].gather(1, at)
    return out, w2
