"""cache_write and cache_read drawn at random: head sizes on every path, alignments, strides, sides of their own shape, blocks of any
size, padded rows. Every bit is compared, of the cache, of its scales and of what lies around the rows."""
import random

import pytest
import torch

import heterofusedkernels_amd  # noqa: F401
import pcie_through  # noqa: F401
from cache_reference import FP8, dequantise
from gpu_helpers import announce
from test_gpu_cache_ops import bits, wanted

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16
ops = torch.ops.pcie_through


def view_in(rng, sizes, order, kind, fill, odd):
    """A tensor of these sizes, dims laid out in `order`, inside a longer buffer: gaps behind each dim and before the first value, of
    whole 16 bytes or (odd) of single values."""
    step = rng.choice([1, 3]) if odd else 16
    stride, at = [0] * len(sizes), 1
    for i, d in enumerate(reversed(order)):
        stride[d] = at
        at *= sizes[d]
        if i != 0 or rng.random() < 0.5:
            at += step * rng.choice([0, 0, 1, 2]) if odd or at % 16 == 0 else 0
    first = step * rng.choice([0, 1, 2])
    buffer = torch.full((first + at + 32,), fill, dtype=torch.float32).to(kind)
    return buffer, first, stride


def on_device(buffer, first, sizes, stride):
    d = torch.empty(buffer.shape, dtype=buffer.dtype, device=DEV)
    (d.view(torch.uint8) if d.element_size() == 1 else d).copy_(buffer.view(torch.uint8) if d.element_size() == 1 else buffer)
    return d, d.as_strided(sizes, stride, first)


@pytest.mark.parametrize("seed", range(80))
def test_drawn_writes_and_reads(seed):
    rng = random.Random(seed)
    gen = torch.Generator().manual_seed(seed)
    kind = rng.choice([BF16, FP16])
    cache_kind = rng.choice([kind, FP8])
    T, n = rng.choice([1, 2, 3, 7, 16, 16, 64, 100]), rng.choice([1, 2, 5, 33, 100, 300])
    blocks = -(-n // T) + rng.randrange(4)
    sides = rng.choice([1, 2, 2])
    shapes = [(rng.choice([1, 2, 3, 4, 8, 13]), rng.choice([1, 2, 7, 8, 16, 24, 37, 64, 72, 80, 96, 128, 128, 200, 256, 264, 512, 520, 576, 768, 1000, 1023, 1024]))
              for _ in range(sides)]
    if rng.random() < 0.6:
        shapes = [shapes[0]] * sides
    odd = rng.random() < 0.3
    announce("seed %d: %d tokens, %d blocks of %d, %s, %s into %s, %s" % (seed, n, blocks, T, shapes, kind, cache_kind, "odd strides" if odd else "whole strides"))
    slots = torch.randperm(blocks * T, generator=gen)[:n]
    slots[torch.rand(n, generator=gen) < rng.choice([0.0, 0.2])] = rng.choice([-1, blocks * T, -(1 << 62), 1 << 62])
    args, kept = [], []
    for H, D in shapes:
        buffer, first, stride = view_in(rng, (n, H, D), rng.choice([(0, 1, 2), (1, 0, 2)]), kind, 3.0, odd)
        rows = buffer.as_strided((n, H, D), stride, first)
        size = torch.exp2(torch.randint(-14, 14, (n, H, 1), generator=gen).float())
        rows.copy_((torch.randn(n, H, D, generator=gen) * size).to(kind))
        plane = view_in(rng, (blocks, T, H, D), rng.choice([(0, 1, 2, 3), (0, 2, 1, 3), (1, 0, 2, 3)]), cache_kind, 7.0, odd)
        scale = view_in(rng, (blocks, T, H), rng.choice([(0, 1, 2), (0, 2, 1)]), torch.float32, 7.0, odd) if cache_kind == FP8 else None
        r_d = on_device(buffer, first, (n, H, D), stride)
        p_d = on_device(plane[0], plane[1], (blocks, T, H, D), plane[2])
        s_d = on_device(scale[0], scale[1], (blocks, T, H), scale[2]) if scale is not None else (None, None)
        args.append((r_d[1], p_d[1], s_d[1]))
        kept.append((rows, plane, scale, r_d, p_d, s_d))
    slots_d = slots.to(DEV)
    k, v = args[0], args[1] if sides == 2 else (None, None, None)
    want = [wanted(p_d[1], s_d[1], rows.contiguous(), slots, T) for rows, _, _, _, p_d, s_d in kept]
    ops.cache_write(k[0], k[1], slots_d, v[0], v[1], k[2], v[2])
    torch.cuda.synchronize()
    for (rows, plane, scale, r_d, p_d, s_d), (wp, ws), (H, D) in zip(kept, want, shapes):
        whole = plane[0].clone()
        inside = whole.as_strided((blocks, T, H, D), plane[2], plane[1])
        (inside.view(torch.uint8) if cache_kind == FP8 else inside).copy_(wp.view(torch.uint8) if cache_kind == FP8 else wp)
        assert torch.equal(bits(p_d[0]), bits(whole)), "the plane, or what lies between its values"
        if scale is not None:
            whole = scale[0].clone()
            whole.as_strided((blocks, T, H), scale[2], scale[1]).copy_(ws)
            assert torch.equal(bits(s_d[0]), bits(whole)), "the scales, or what lies between them"

    # back into rows of another layout, slots repeated
    again = torch.cat([slots, slots[: n // 2]]) if rng.random() < 0.5 else slots
    m, ok = len(again), (again >= 0) & (again < blocks * T)
    back = []
    for H, D in shapes:
        buffer, first, stride = view_in(rng, (m, H, D), rng.choice([(0, 1, 2), (1, 0, 2)]), kind, 5.0, odd)
        back.append((buffer, first, stride) + on_device(buffer, first, (m, H, D), stride))
    ops.cache_read(k[1], back[0][4], again.to(DEV), v[1], back[1][4] if sides == 2 else None, k[2], v[2])
    torch.cuda.synchronize()
    b, o = again[ok] // T, again[ok] % T
    for (buffer, first, stride, d, _), (wp, ws), (H, D) in zip(back, want, shapes):
        rows = dequantise(wp.view(torch.uint8)[b, o].view(FP8), ws[b, o], kind) if cache_kind == FP8 else wp[b, o]
        buffer.as_strided((m, H, D), stride, first)[ok] = rows
        assert torch.equal(bits(d), bits(buffer)), "the rows, or what lies between them"
