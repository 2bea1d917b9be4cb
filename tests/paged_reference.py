"""A paged cache and its three operators in 64 bits on the CPU, slot by slot, and how far a
kernel's results may be from them."""
import math

import torch

EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def to_e4m3(x):
    """Nearest e4m3 value (ties to even) of 64-bit x, |x| <= 448: steps of 2^-9 up to 2^-6,
    an eighth of the octave above."""
    octave = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(octave - 3)
    return torch.round(x / step) * step


def quantise(x):
    """(values, scale exponents e) of rows [..., D] in 64 bits: e = -127 for zeros, 128 for a row that is not finite."""
    x = x.double()
    amax = x.abs().amax(-1)
    bad = ~torch.isfinite(amax)
    a = torch.where(bad | (amax == 0), torch.ones_like(amax) * 448, amax)
    e = torch.ceil(torch.log2(a / 448))
    e = torch.where(a > 448 * torch.exp2(e), e + 1, e)
    e = torch.where(a <= 448 * torch.exp2(e - 1), e - 1, e)
    e = torch.where(amax == 0, torch.full_like(e, -127), e).clamp(min=-127)
    v = to_e4m3(torch.where(bad[..., None], torch.zeros_like(x), x) / torch.exp2(e)[..., None])
    return v, torch.where(bad, torch.full_like(e, 128), e)


def stored(x, dtype, quantized):
    """What the cache stands for after `x` went in, in 64 bits."""
    if not quantized:
        return x.to(dtype).double()
    v, e = quantise(x)
    return torch.where((e == 128)[..., None], torch.full_like(v, math.nan), v * torch.exp2(e)[..., None])


class Case:
    """A batch over a cache whose every other slot is poisoned: NaN pages, NaN scales, table
    entries behind a row's last page that name no page."""

    def __init__(self, seed, batch, tokens, held, new, heads, kv_heads, d, page, dtype, quantized, spare=3, loud=1.0):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.quantized, self.page, self.d = dtype, quantized, page, d
        self.held, self.new, self.tokens = held, new, tokens
        n = lambda *s: torch.randn(s, generator=g)
        self.q = n(batch, tokens, heads, d).to(dtype)
        total = [h + m for h, m in zip(held, new)]
        self.keys = [(n(t, kv_heads, d) * loud).to(dtype) for t in total]
        self.values = [n(t, kv_heads, d).to(dtype) for t in total]
        used = [-(-t // page) for t in total]
        self.pages = sum(used) + spare
        order = torch.randperm(self.pages, generator=g).tolist()
        width = max(max(used), 1) + 2
        self.table = torch.randint(0, 2 ** 30, (batch, width), generator=g, dtype=torch.int32) * 2 + 2 ** 30
        self.table[:, ::2] = -7
        at = 0
        for b, u in enumerate(used):
            self.table[b, :u] = torch.tensor(order[at:at + u], dtype=torch.int32)
            at += u
        shape = (self.pages, page, kv_heads, d)
        if quantized:
            self.k = torch.full(shape, 0x7f, dtype=torch.uint8).view(torch.float8_e4m3fn)
            self.v = self.k.clone()
            self.ks = torch.full((self.pages, kv_heads, page), 255, dtype=torch.uint8).view(torch.float8_e8m0fnu)
            self.vs = self.ks.clone()
        else:
            self.k = torch.full(shape, math.nan, dtype=dtype)
            self.v = self.k.clone()
            self.ks = self.vs = None

    def put(self, first, last):
        """Tokens [first[b], last[b]) of every row into the CPU pages, by the definition."""
        for b, (lo, hi) in enumerate(zip(first, last)):
            for x, pages, scales in ((self.keys[b], self.k, self.ks), (self.values[b], self.v, self.vs)):
                p = torch.arange(lo, hi)
                at, slot = self.table[b, p // self.page].long(), p % self.page
                if not self.quantized:
                    pages[at, slot] = x[lo:hi]
                    continue
                v, e = quantise(x[lo:hi])
                pages.view(torch.uint8)[at, slot] = v.float().to(torch.float8_e4m3fn).view(torch.uint8)
                scales.view(torch.uint8)[at, :, slot] = (e + 127).to(torch.uint8)
        return self

    def attention(self, causal=True, window=None, scale=None):
        """(o, lse, bound): the result in 64 bits and how far a kernel's may be off, element
        by element: the output's own rounding, weights rounded to `weights` of their size
        (both in the sum with the values and in their total), and what 32-bit scores of D
        products leave, which an exponential passes on as a relative error."""
        B, T, H, D = self.q.shape
        hk = self.keys[0].shape[1]
        scale = 1 / math.sqrt(D) if scale is None else scale
        o = torch.zeros(B, T, H, D, dtype=torch.float64)
        lse = torch.full((B, H, T), -math.inf, dtype=torch.float64)
        bound = torch.zeros_like(o)
        # weights in the stream type or better (8-bit pages: in pieces, 2^-9 beside a bf16 stream, 2^-12 beside f16)
        weights = EPS[self.dtype]
        for b in range(B):
            n = self.new[b]
            if n == 0:
                continue
            k = stored(self.keys[b], self.dtype, self.quantized)
            v = stored(self.values[b], self.dtype, self.quantized)
            i = self.held[b] + torch.arange(n)[:, None]
            j = torch.arange(k.shape[0])
            seen = torch.ones(n, k.shape[0], dtype=torch.bool)
            if causal:
                seen &= j <= i
            if window is not None:
                seen &= (j >= i - window[0]) & (j <= i + window[1])
            for h in range(H):
                kk, vv, qq = k[:, h // (H // hk)], v[:, h // (H // hk)], self.q[b, :n, h].double()
                s = (qq @ kk.T * scale).masked_fill(~seen, -math.inf)
                size = (qq.abs() @ kk.abs().T * abs(scale)).masked_fill(~seen, 0).amax(-1, keepdim=True)
                lse[b, h, :n] = torch.logsumexp(s, -1)
                p = torch.softmax(s, -1).nan_to_num(0.0)
                o[b, :n, h] = p @ vv
                mass = p @ vv.abs()
                rel = 2 * weights + 2 * (D + 8) * 2.0 ** -24 * size + 2.0 ** -18
                bound[b, :n, h] = EPS[self.dtype] * (o[b, :n, h].abs() + rel * mass) + rel * mass + 2.0 ** -25
        return o, lse, bound
