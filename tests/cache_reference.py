"""Plain 64-bit statements of the cache and attention ops, and inputs for their tests. CPU only: torch and loops.

A cache side is ``values [blocks, T, heads, dim]`` with, for e4m3, ``scales [blocks, T, heads]``.
"""
import math

import torch

FP8 = torch.float8_e4m3fn
STEP = {torch.bfloat16: torch.finfo(torch.bfloat16).eps / 2, torch.float16: torch.finfo(torch.float16).eps / 2}


def quantise(x):
    """(e4m3 values, float32 scales of the last dimension), from the definition: the smallest power of two s with
    max |x| <= 448 s over the finite values, x / s to nearest even, infinities to the ends, NaN kept."""
    x = x.double()
    size = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    scale = torch.ones_like(size)
    for e in range(-126, 120):
        scale = torch.where((size > 448.0 * 2.0 ** (e - 1)) & (size > 0), 2.0 ** e, scale)
    # a row smaller than any step of the loop: the smallest scale
    scale = torch.where((size > 0) & (size <= 448.0 * 2.0 ** -127), 2.0 ** -126, scale)
    return (x / scale[..., None]).clamp(-448.0, 448.0).float().to(FP8), scale.float()


def dequantise(values, scales, kind):
    """What reading the cache back gives, in `kind`."""
    x = values.double() * scales.double()[..., None]
    return x.clamp(-torch.finfo(kind).max, torch.finfo(kind).max).to(kind)


class Cache:
    """Both sides of a layer's cache. Every token the test does not fill is NaN."""

    def __init__(self, blocks, T, heads, dim, kind, cache_kind, order="thd", seed=0):
        self.gen = torch.Generator().manual_seed(seed)
        self.blocks, self.T, self.heads, self.dim, self.kind, self.cache_kind = blocks, T, heads, dim, kind, cache_kind
        self.fp8 = cache_kind == FP8

        def plane(*tail):
            if order == "thd":
                return lambda fill, dtype: torch.full((blocks, T, heads) + tail, fill, dtype=torch.float32).to(dtype)
            return lambda fill, dtype: torch.full((blocks, heads, T) + tail, fill, dtype=torch.float32).to(dtype).transpose(1, 2)

        self.k, self.v = (plane(dim)(float("nan"), cache_kind) for _ in "kv")
        self.ks, self.vs = (plane()(1.0, torch.float32) if self.fp8 else None for _ in "kv")

    def fill(self, slots, k=None, v=None, size=1.0):
        """Random tokens (or those given) into `slots`."""
        n = len(slots)
        b, o = slots // self.T, slots % self.T
        for x, values, scales in ((k, self.k, self.ks), (v, self.v, self.vs)):
            if x is None:
                x = (torch.randn(n, self.heads, self.dim, generator=self.gen) * size).to(self.kind)
            if self.fp8:
                q, s = quantise(x)
                values.view(torch.uint8)[b, o] = q.view(torch.uint8)
                scales[b, o] = s
            else:
                values[b, o] = x

    def rows(self, slots):
        """(k, v) in 64 bits, as read back in the queries' type."""
        b, o = slots // self.T, slots % self.T
        out = []
        for values, scales in ((self.k, self.ks), (self.v, self.vs)):
            if self.fp8:
                x = values.view(torch.uint8)[b, o].view(FP8)
                out.append(dequantise(x, scales[b, o], self.kind).double())
            else:
                out.append(values[b, o].double())
        return out

    def to(self, device):
        """(k, v, k scales, v scales) on a device, strides kept."""
        def move(t):
            if t is None:
                return None
            d = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=device)
            (d.view(torch.uint8) if self.fp8 and t.dtype == FP8 else d).copy_(t.view(torch.uint8) if t.dtype == FP8 else t)
            return d
        return move(self.k), move(self.v), move(self.ks), move(self.vs)


def tables(gen, lengths, T, blocks, first=0, width=None):
    """A block table of distinct shuffled blocks (from `first` on) and each sequence's slots in order."""
    width = max(1, max(-(-n // T) for n in lengths)) if width is None else width
    ids = torch.randperm(blocks - first, generator=gen) + first
    table = torch.zeros(len(lengths), width, dtype=torch.int64)
    at, slots = 0, []
    for b, n in enumerate(lengths):
        need = -(-n // T)
        table[b, :need] = ids[at:at + need]
        at += need
        j = torch.arange(n)
        slots.append(table[b, j // T] * T + j % T)
    return table, slots


def attend(q, k, v, visible, scale):
    """One sequence. q [n, Hq, D], k and v [L, H, D] in 64 bits, visible [n, L]. Returns out, lse and what bounds a kernel's
    error: sum of w |v| per element, and the largest sum of |q k| of a row's visible keys."""
    n, Hq, D = q.shape
    L, H = k.shape[0], k.shape[1]
    G = Hq // H
    out, size = torch.zeros(n, Hq, D, dtype=torch.float64), torch.zeros(n, Hq, D, dtype=torch.float64)
    lse, reach = torch.full((n, Hq), -math.inf, dtype=torch.float64), torch.zeros(n, Hq, dtype=torch.float64)
    for h in range(Hq):
        kh, vh = k[:, h // G], v[:, h // G]
        s = (q[:, h] @ kh.t() * scale).masked_fill(~visible, -math.inf)
        seen = visible.any(-1)
        if L == 0 or not bool(seen.any()):
            continue
        lse[:, h] = torch.logsumexp(s, -1)
        w = torch.where(seen[:, None], torch.softmax(s, -1), 0.0)
        out[:, h] = w @ vh
        size[:, h] = w @ vh.abs()
        reach[:, h] = (q[:, h].abs() @ kh.abs().t() * visible).amax(-1) * scale
    return out, lse, size, reach


def bounds(want, lse, size, reach, kind, dim, keys):
    """How far a kernel with 32-bit scores, statistics and sums and weights rounded to `kind` may be off.

    u = half a step of `kind`, e = 2^-24. A score is a sum of `dim` exact products: off by (dim + 8) e of their sizes'
    sum (additions, the scaling, the subtraction of the maximum), and so is the weight, relatively; twice that because the maximum's
    own error enters too. exp2, its argument's rounding and one rescaling per tile of 32 keys: (keys / 32 + 64) 2 e.
    The weight's rounding: u, and the result's own: u of the result. fp16 weights end at 2^-24 of at most 1 / 2^6 of the
    largest: keys * 2^-31 of the largest |v| covers it, which stays below size * keys * 2^-24 for the sizes tested."""
    u, e = STEP[kind], 2.0 ** -24
    rel = 2 * (dim + 8) * e * reach + (keys / 32 + 64) * 2 * e
    out = u * want.abs() + (u + u * u + rel)[..., None] * size + 1e-30
    return out, rel + 4 * e * lse.abs().clamp(max=1e30)
