"""Paged caches for the tests, and the paged operators from their definitions in 64 bits."""
import math

import torch

D = 128
E4, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def exponents(x):
    """The least e >= -117 with max|x| <= 448 * 2^e, by comparison; 128 for rows with an infinity or NaN."""
    top = x.double().abs().amax(-1)
    e = torch.ceil(torch.log2(top / 448)).clamp(min=-117)
    e = torch.where(top <= 448 * torch.exp2(e - 1), e - 1, e)  # log2 of a number next to a power of two
    e = torch.where(top > 448 * torch.exp2(e), e + 1, e).clamp(min=-117)
    return torch.where(torch.isfinite(top), e, 128.0)


def rounded(x, bits, least):
    """x (64 bits) to `bits` significant bits, to even on ties, in steps of at least 2^least."""
    step = torch.exp2((torch.frexp(x)[1] - bits).clamp(min=least).double())
    return torch.round(x / step) * step


def stored(x, e4m3):
    """What a cache holds of rows x [..., 128], in 64 bits."""
    x = x.double()
    if not e4m3:
        return torch.where(torch.isfinite(x), rounded(x, 8, -133), x)
    e = exponents(x)
    unit = torch.exp2(e)[..., None]
    return torch.where((e == 128)[..., None], math.nan, rounded(x / unit, 4, -9) * unit)


def values(pages, scales):
    """The numbers that pages stand for, in 64 bits."""
    if scales is None:
        return pages.double()
    byte = scales.view(torch.uint8).double()
    return torch.where((byte == 255)[..., None], math.nan, pages.float().double() * torch.exp2(byte - 127)[..., None])


class Pool:
    """Pages in any order, `layout` one of plain, joint ([pages, 2, ...]) and rows ([pages, page_size, heads, 128])."""

    def __init__(self, seqs, entries, page_size, heads, e4m3, device, layout="plain", extra=3, seed=0, fill=True):
        self.n, self.ps, self.h, self.e4m3, self.dev = seqs * entries + extra, page_size, heads, e4m3, device
        self.gen = torch.Generator().manual_seed(seed)
        order = torch.randperm(self.n, generator=self.gen)[:seqs * entries]
        self.tables = order.view(seqs, entries).int().to(device)
        n, h, p = self.n, heads, page_size
        kind = E4 if e4m3 else torch.bfloat16

        def make(shape, byte):
            if e4m3:
                return torch.full(shape, byte, dtype=torch.uint8, device=device)
            return torch.zeros(shape, dtype=torch.bfloat16, device=device)

        if layout == "joint":
            both = make((n, 2, h, p, D), 0).view(kind)
            self.k, self.v = both[:, 0], both[:, 1]
        elif layout == "rows":
            self.k, self.v = (make((n, p, h, D), 0).view(kind).transpose(1, 2) for _ in range(2))
        else:
            self.k, self.v = (make((n, h, p, D), 0).view(kind) for _ in range(2))
        self.ks = self.vs = None
        if e4m3:
            self.ks, self.vs = (torch.full((n, h, p), 127, dtype=torch.uint8, device=device).view(E8) for _ in range(2))
        if fill:
            self.fill()

    def fill(self, scale=1.0):
        """Random rows of magnitudes that differ from row to row."""
        g = torch.Generator(device=self.dev).manual_seed(int(torch.randint(1 << 30, (1,), generator=self.gen)))
        for pages, scales in ((self.k, self.ks), (self.v, self.vs)):
            x = torch.randn(pages.shape, generator=g, device=self.dev) * scale
            if self.e4m3:
                e = torch.randint(-3, 2, scales.shape, generator=g, device=self.dev)
                x = x * 20
                pages.copy_(x.to(E4))
                scales.view(torch.uint8).copy_((e + 123).to(torch.uint8))
            else:
                pages.copy_(x.to(torch.bfloat16))

    def rows(self, which, s, first, count):
        """Positions first .. first + count - 1 of sequence s in 64 bits, [count, heads, 128]."""
        pages, scales = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        at = torch.arange(first, first + count, device=self.dev)
        page = self.tables[s].long()[at // self.ps]
        if scales is None:
            return pages[page, :, at % self.ps].double()
        b = scales.view(torch.uint8)[page, :, at % self.ps].double()
        x = pages.view(torch.uint8)[page, :, at % self.ps].view(E4).float().double()
        return torch.where((b == 255)[..., None], math.nan, x * torch.exp2(b - 127)[..., None])

    def args(self):
        return self.k, self.v, self.tables

    def scales(self):
        return self.ks, self.vs


def attention(pool, q, lengths):
    """The attention in 64 bits, and how far the operator may be off: see test_gpu_paged."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    off = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    g = q.shape[1] // pool.h
    for s, n in enumerate(lengths):
        if n == 0:
            continue
        k, v = pool.rows("k", s, 0, n), pool.rows("v", s, 0, n)
        for h in range(pool.h):
            qq = q[s, h * g:(h + 1) * g].double()
            w = qq @ k[:, h].t().contiguous() / math.sqrt(D)
            out[s, h * g:(h + 1) * g] = torch.softmax(w, 1) @ v[:, h].contiguous()
            size = (qq.abs() @ k[:, h].abs().t().contiguous() / math.sqrt(D)).amax(1)  # of a score's products
            adds = 11 * math.ceil(n / 32) + 64
            off[s, h * g:(h + 1) * g] = ((2.0 ** -21 * size + 4 * 2.0 ** -24 * math.sqrt(adds)) *
                                         v[:, h].abs().max())[:, None]
            if q.dtype == torch.bfloat16:
                off[s, h * g:(h + 1) * g] += 2.0 ** -16 * v[:, h].abs().max()
    if q.dtype == torch.bfloat16:
        off += 2.0 ** -8 * (out.abs() + off)
    return out, off
