"""cache_write and cache_read on the GPU against their definitions in 64 bits: types, layouts, strides, head sizes that
take the vectorised path and ones that do not, padded rows, special values. Results are exact: every bit is compared."""
import pytest
import torch

import heterofusedkernels_amd  # noqa: F401
import pcie_through  # noqa: F401
from cache_reference import FP8, dequantise, quantise
from gpu_helpers import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16
ops = torch.ops.pcie_through


def bits(t):
    t = t.cpu().contiguous()
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def empty_plane(blocks, T, H, D, kind, order, fill):
    shape = (blocks, T, H) if order == "thd" else (blocks, H, T)
    p = torch.full(shape + (D,), fill, dtype=torch.uint8, device=DEV).view(kind) if kind == FP8 else \
        torch.full(shape + (D,), float(fill), dtype=kind, device=DEV)
    s = torch.full(shape, float(fill), dtype=torch.float32, device=DEV) if kind == FP8 else None
    return (p, s) if order == "thd" else (p.transpose(1, 2), s.transpose(1, 2) if s is not None else None)


def wanted(before, scales_before, x, slots, T):
    """The cache after the write, on the CPU."""
    cache = before.cpu().contiguous().clone()
    scales = scales_before.cpu().contiguous().clone() if scales_before is not None else None
    ok = (slots >= 0) & (slots < cache.shape[0] * T)
    b, o = slots[ok] // T, slots[ok] % T
    if scales is not None:
        q, s = quantise(x[ok])
        cache.view(torch.uint8)[b, o] = q.view(torch.uint8)
        scales[b, o] = s
    else:
        cache[b, o] = x[ok]
    return cache, scales


def same_codes(got, want):
    """e4m3 codes are equal, or both are NaN (either sign)."""
    g, w = bits(got).int(), bits(want).int()
    return bool(((g == w) | (((g & 0x7f) == 0x7f) & ((w & 0x7f) == 0x7f))).all())


CASES = [  # n, heads, dim, T, order
    (1, 8, 128, 16, "thd"), (3, 1, 64, 16, "htd"), (129, 8, 128, 16, "htd"), (1000, 1, 576, 64, "thd"), (77, 5, 96, 32, "thd"),
    (40, 3, 80, 3, "htd"), (33, 2, 8, 16, "thd"), (9, 2, 1024, 16, "thd"), (61, 3, 37, 5, "thd"), (17, 2, 1, 16, "htd"), (300, 16, 128, 1, "thd"),
]


@pytest.mark.parametrize("kind,cache_kind", [(BF16, FP8), (FP16, FP8), (BF16, BF16), (FP16, FP16)])
@pytest.mark.parametrize("n,H,D,T,order", CASES)
def test_write_then_read(n, H, D, T, order, kind, cache_kind):
    announce("cache write/read n=%d H=%d D=%d T=%d %s %s %s" % (n, H, D, T, order, kind, cache_kind))
    gen = torch.Generator().manual_seed(n * 1000 + D)
    blocks = -(-n // T) + 3
    slots = torch.randperm(blocks * T, generator=gen)[:n]
    if n > 8:      # padded rows and slots behind the cache
        slots[n // 2], slots[n - 1], slots[2] = -1, blocks * T, 2 ** 40
    x = [(torch.randn(n, H, D, generator=gen) * torch.exp2(torch.randint(-12, 12, (n, H, 1), generator=gen).float())).to(kind)
         for _ in "kv"]
    x[0][0, 0] = 0.0
    planes = [empty_plane(blocks, T, H, D, cache_kind, order, 7) for _ in "kv"]
    want = [wanted(p, s, y, slots, T) for (p, s), y in zip(planes, x)]
    slots_d = slots.to(DEV)
    ops.cache_write(x[0].to(DEV), planes[0][0], slots_d, x[1].to(DEV), planes[1][0], planes[0][1], planes[1][1])
    torch.cuda.synchronize()
    for (p, s), (wp, ws) in zip(planes, want):
        assert torch.equal(bits(p), bits(wp))
        assert s is None or torch.equal(bits(s), bits(ws))

    # back, with repeated slots; rows without a slot keep what they held
    again = torch.cat([slots, slots[:3]])
    out = [torch.full((n + 3 if n >= 3 else 2 * n, H, D), 3.0, dtype=kind, device=DEV) for _ in "kv"]
    ops.cache_read(planes[0][0], out[0], again.to(DEV), planes[1][0], out[1], planes[0][1], planes[1][1])
    torch.cuda.synchronize()
    ok = (again >= 0) & (again < blocks * T)
    for y, (wp, ws) in zip(out, want):
        b, o = again[ok] // T, again[ok] % T
        rows = dequantise(wp.view(torch.uint8)[b, o].view(FP8), ws[b, o], kind) if cache_kind == FP8 else wp[b, o]
        assert torch.equal(bits(y[ok.to(DEV)]), bits(rows))
        assert bool((y[~ok.to(DEV)] == 3.0).all())


@pytest.mark.parametrize("kind", [BF16, FP16])
@pytest.mark.parametrize("D", [128, 37])
def test_special_values(kind, D):
    """Infinities, NaN, zeros, the largest and the smallest values, rows of one kind each and mixed ones; both paths."""
    announce("cache write special values %s D=%d" % (kind, D))
    inf, nan, big, tiny = float("inf"), float("nan"), torch.finfo(kind).max, torch.finfo(kind).smallest_normal
    rows = [[0.0], [-0.0, 0.0], [inf], [-inf, 1.0], [nan], [nan, 2.0, inf], [big], [-big, big / 3], [tiny], [tiny / 8, tiny], [1.75], [1.7578125],
            [448.0, -448.0], [449.0, 1.0], [61440.0, 65504.0], [57344.0], [1.0, 2.0 ** -9, 2.0 ** -10, 2.0 ** -11, 3 * 2.0 ** -10]]
    n = len(rows)
    x = torch.stack([torch.tensor((r * D)[:D], dtype=torch.float32) for r in rows]).to(kind)[:, None]
    plane, scales = empty_plane(3, 16, 1, D, FP8, "thd", 5)
    before, sb = plane.clone(), scales.clone()
    slots = torch.arange(n) + 7
    ops.cache_write(x.to(DEV), plane, slots.to(DEV), None, None, scales)
    want, ws = wanted(before, sb, x, slots, 16)
    torch.cuda.synchronize()
    assert same_codes(plane, want)
    assert torch.equal(bits(scales), bits(ws))
    out = torch.zeros_like(x, device=DEV)
    ops.cache_read(plane, out, slots.to(DEV), None, None, scales)
    rows = dequantise(want.view(torch.uint8)[slots // 16, slots % 16].view(FP8), ws[slots // 16, slots % 16], kind)
    got = out.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(rows))
    assert torch.equal(got.nan_to_num(0.0), rows.nan_to_num(0.0))
    assert bool(torch.isfinite(got[~torch.isnan(rows)]).all())


@pytest.mark.parametrize("kind", [BF16, FP16])
def test_every_code_under_every_scale(kind):
    announce("cache read: 256 codes x 246 scales, %s" % kind)
    exponents = torch.arange(-126, 120)
    codes = torch.arange(256, dtype=torch.uint8).repeat(len(exponents), 1)
    plane = codes.to(DEV).view(FP8).view(1, len(exponents), 1, 256)
    scales = torch.exp2(exponents.double()).float().to(DEV).view(1, -1, 1)
    out = torch.zeros(len(exponents), 1, 256, dtype=kind, device=DEV)
    ops.cache_read(plane, out, torch.arange(len(exponents), device=DEV), None, None, scales)
    want = dequantise(codes.view(FP8)[:, None], scales.cpu()[0], kind)
    got = out.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


def test_strided_rows_and_sides_of_their_own_shape():
    """Rows out of a fused projection (strided, and unaligned by one value), a latent side next to a narrower one."""
    announce("cache write strided rows, k [1, 576], v [2, 64]")
    gen = torch.Generator().manual_seed(5)
    n, T, blocks = 50, 16, 6
    slots = torch.randperm(blocks * T, generator=gen)[:n]
    for shift in (0, 1):
        fused = torch.randn(n, 2, 800 + shift, generator=gen).to(BF16).to(DEV)
        k, v = fused[:, :1, shift:576 + shift], fused[:, :, 600 + shift:664 + shift]
        for cache_kind in (FP8, BF16):
            (kp, ks), (vp, vs) = empty_plane(blocks, T, 1, 576, cache_kind, "thd", 1), empty_plane(blocks, T, 2, 64, cache_kind, "htd", 2)
            want_k, want_v = wanted(kp, ks, k.cpu(), slots, T), wanted(vp, vs, v.cpu(), slots, T)
            ops.cache_write(k, kp, slots.to(DEV), v, vp, ks, vs)
            torch.cuda.synchronize()
            for got, got_s, (w, ws) in ((kp, ks, want_k), (vp, vs, want_v)):
                assert torch.equal(bits(got), bits(w))
                assert ws is None or torch.equal(bits(got_s), bits(ws))
