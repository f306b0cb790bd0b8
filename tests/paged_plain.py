"""Plain 64-bit forms of the paged-cache operators and the inputs their tests
share (CPU; no code of the package)."""
import math

import torch

QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
# largest relative error of rounding to 11 (f16) or 8 (bf16) significant bits
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def bits(x):
    """8-bit tensors as bytes (indexing is not defined for 8-bit floats)."""
    return x.view(torch.uint8) if x.element_size() == 1 else x


class Paged:
    """A batch over a paged cache: lengths [(new, cached)], pages in a random
    order, every row that no sequence owns poisoned with NaN."""

    def __init__(self, lens, Hkv, d, page, cache, io=torch.float16, order="head", seed=0,
                 spare=2, first=0, tail=0, poison=True, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.Hkv, self.d, self.page = lens, Hkv, d, page
        self.io, self.cache, self.order = io, cache, order
        need = [-(-n // page) for _, n in lens]
        self.pages = max(sum(need) + spare, 1)
        self.width = max(need + [1]) + 1
        perm = torch.randperm(self.pages, generator=g).tolist()
        # entries past a sequence's end point outside the cache
        self.table = torch.full((len(lens), self.width), -1, dtype=torch.int32)
        self.table[:, -1] = 1 << 30
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = torch.tensor(perm[at:at + n], dtype=torch.int32)
            at += n
        self.cu = [first]
        for m, _ in lens:
            self.cu.append(self.cu[-1] + m)
        self.total = self.cu[-1] + tail
        self.nk = [n for _, n in lens]
        shape = (self.pages, Hkv, page, d)
        eight = cache in QMAX
        self.k = torch.zeros(shape).to(cache)
        self.v = torch.zeros(shape).to(cache)
        self.ks = torch.full(shape[:3], float("nan")) if eight else None
        self.vs = torch.full(shape[:3], float("nan")) if eight else None
        if poison and not eight:
            self.k.fill_(float("nan"))
            self.v.fill_(float("nan"))
        elif poison:
            bits(self.k).fill_(0x7f)
            bits(self.v).fill_(0x7f)
        for b, (_, n) in enumerate(lens):
            for name in ("k", "v"):
                x = torch.randn(n, Hkv, d, generator=g) * spread
                if eight:
                    x8, s = quantise(x, cache)
                    self.put(name, b, range(n), x8, s)
                else:
                    self.put(name, b, range(n), x.to(cache), None)
        self.g = g

    def place(self, b, pos):
        return int(self.table[b, pos // self.page]), pos % self.page

    def put(self, name, b, positions, x, s):
        c, sc = getattr(self, name), getattr(self, name + "s")
        for i, p in enumerate(positions):
            pg, row = self.place(b, p)
            bits(c)[pg, :, row] = bits(x)[i]
            if s is not None:
                sc[pg, :, row] = s[i]

    def held(self, name, b, n, caches=None):
        """[n, Hkv, d] 64-bit values of the first n positions of sequence b."""
        c, sc = caches or (getattr(self, name), getattr(self, name + "s"))
        pos = torch.arange(n)
        pg, row = self.table[b].long()[pos // self.page], pos % self.page
        x = bits(c)[pg, :, row]
        x = x.view(c.dtype).double() if c.element_size() == 1 else x.double()
        return x * sc[pg, :, row].double().unsqueeze(-1) if sc is not None else x

    def new(self, heads, spread=1.0):
        return (torch.randn(self.total, heads, self.d, generator=self.g) * spread).to(self.io)

    def cuda(self):
        """(k_cache, v_cache, table, cu, lens, scales) on the GPU in the memory order."""
        def page_order(x):
            if x is None:
                return None
            if self.order == "token":
                return x.transpose(1, 2).contiguous().cuda().transpose(1, 2)
            return x.contiguous().cuda()

        i32 = dict(dtype=torch.int32, device="cuda")
        return dict(k_cache=page_order(self.k), v_cache=page_order(self.v),
                    table=self.table.cuda(), cu=torch.tensor(self.cu, **i32),
                    lens=torch.tensor(self.nk, **i32), k_scale=page_order(self.ks),
                    v_scale=page_order(self.vs))


def quantise(x, kind):
    """8-bit rows and scales as the operator defines them, in fp32."""
    a = x.float().abs().amax(-1)
    keep = ~(a < 2.0 ** -100)
    q = torch.tensor(QMAX[kind])
    inv = torch.where(keep, q / a, torch.zeros(()))
    s = torch.where(keep, a / q, torch.zeros(()))
    y = x.float() * inv.unsqueeze(-1)
    if kind == torch.int8:
        return torch.round(y).clamp(-127, 127).to(torch.int8), s
    return y.clamp(-448, 448).to(torch.float8_e4m3fn), s


def attention(P, q, Hq, mode, scale=None):
    """O [total, Hq, d], LSE [Hq, total] in 64 bits and the bound on O's and
    LSE's errors that the kernels' roundings allow.

    The kernels round P to 16 bits and O once; the exponential is good to 1e-4
    relative; 8-bit keys and values may be rounded to f16 once, which moves a
    score by at most u * sum|q k| * scale =: ds (relative error of each p: 2 ds).
    With A = sum p |v| the error of O is at most
        u_out |O| + A * (2 u + 2e-4 + 4 ds),   u = unit of the 16-bit products
    (p and the row sum each carry the exponential's and the score's error), and
    that of LSE 1e-4 + 2 ds.  8-bit caches are computed in f16 whatever q's type.
    """
    d = P.d
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    eight = P.cache in QMAX
    u = UNIT[torch.float16] if eight else UNIT[P.io]
    o = torch.zeros(P.total, Hq, d, dtype=torch.float64)
    lse = torch.full((Hq, P.total), -math.inf, dtype=torch.float64)
    tol = torch.zeros_like(o)
    tol_lse = torch.full_like(lse, 1e-4)
    for b, (m, n) in enumerate(P.lens):
        if m == 0 or n == 0:
            continue
        rows = slice(P.cu[b], P.cu[b + 1])
        k = P.held("k", b, n).repeat_interleave(Hq // P.Hkv, 1).transpose(0, 1)
        v = P.held("v", b, n).repeat_interleave(Hq // P.Hkv, 1).transpose(0, 1)
        x = q[rows].double().transpose(0, 1)                       # [Hq, m, d]
        s = x @ k.transpose(1, 2) * scale
        i, j = torch.arange(m)[:, None], torch.arange(n)[None]
        see = torch.ones(m, n, dtype=torch.bool)
        if mode:
            see = j <= i + (n - m if mode == 1 else 0)
        s = s.masked_fill(~see, -math.inf)
        z = torch.logsumexp(s, -1)
        p = torch.exp(s - torch.where(z == -math.inf, torch.zeros_like(z), z)[..., None])
        ob = p @ v
        ds = (x.abs() @ k.abs().transpose(1, 2)).masked_fill(~see, 0).amax(-1) * abs(scale) * u
        ds = ds if eight else torch.zeros_like(ds)
        a = p @ v.abs()
        t = UNIT[P.io] * ob.abs() + a * (2 * u + 2e-4 + 4 * ds)[..., None] + 1e-6
        o[rows], lse[:, rows] = ob.transpose(0, 1), z
        tol[rows], tol_lse[:, rows] = t.transpose(0, 1), 1e-4 + 2 * ds
    return o, lse, tol, tol_lse
