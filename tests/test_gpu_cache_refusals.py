"""Calls that the cache and attention ops refuse by name before anything is launched, and ones beside them that they take."""
import pytest
import torch

import heterofusedkernels_amd  # noqa: F401
import pcie_through  # noqa: F401
from cache_reference import FP8
from gpu_helpers import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16
ops = torch.ops.pcie_through


def refused(match):
    return pytest.raises(RuntimeError, match=match)


def cache_of(kind):
    """(values, scales or None)"""
    return torch.zeros(4, 16, 2, 64, dtype=kind, device=DEV), torch.ones(4, 16, 2, device=DEV) if kind == FP8 else None


@pytest.mark.parametrize("k_kind,v_kind", [(BF16, FP8), (FP8, BF16), (FP16, FP8), (BF16, FP16)])
def test_sides_of_two_types(k_kind, v_kind):
    announce("keys in %s, values in %s" % (k_kind, v_kind))
    (k, ks), (v, vs) = cache_of(k_kind), cache_of(v_kind)
    x, slots = torch.ones(3, 2, 64, dtype=BF16, device=DEV), torch.arange(3, device=DEV)
    with refused("kCache and vCache must have one type"):
        ops.cache_write(x, k, slots, x, v, ks, vs)
    with refused("kCache and vCache must have one type"):
        ops.cache_read(k, x, slots, v, x.clone(), ks, vs)
    with refused("one shape and one type"):
        ops.prefix_attention(x, k, v, slots[:0], slots[:1], slots[:, None], slots, torch.zeros_like(x), 0.1, ks, vs)
    torch.cuda.synchronize()
    for t in (k, v):
        assert not bool(t.view(torch.uint8).any())
    assert bool((x == 1).all())


def in_memory_of(t, dtype, *shape):
    """A dense tensor in t's memory."""
    n = 1
    for s in shape:
        n *= s
    return t.view(-1).view(torch.uint8)[:n * torch.empty(0, dtype=dtype).element_size()].view(dtype).view(*shape)


def test_written_tensors_that_share_memory():
    """Everything that is written against everything else: no call of these is made sound by the order of its workgroups."""
    announce("written tensors in memory that is read")
    k, v = torch.zeros(4, 16, 2, 64, dtype=BF16, device=DEV), torch.zeros(4, 16, 2, 64, dtype=BF16, device=DEV)
    (f, fs), (g, gs) = cache_of(FP8), cache_of(FP8)
    x, slots = torch.zeros(3, 2, 64, dtype=BF16, device=DEV), torch.arange(3, device=DEV)
    with refused("kCache and k must not overlap"):
        ops.cache_write(k.view(64, 2, 64)[:3], k, slots + 10)
    with refused("vCache and k must not overlap"):
        ops.cache_write(v.view(64, 2, 64)[:3], k, slots, x, v)
    with refused("kCache and v must not overlap"):
        ops.cache_write(x, k, slots, k.view(64, 2, 64)[5:8], v)
    with refused("kCache and slots must not overlap"):
        ops.cache_write(x, k, in_memory_of(k, torch.int64, 3))
    with refused("kCache and kScales must not overlap"):
        ops.cache_write(x, f, slots, None, None, in_memory_of(f, torch.float32, 4, 16, 2))
    with refused("vCache and kScales must not overlap"):
        ops.cache_write(x, f, slots, x.clone(), g, in_memory_of(g, torch.float32, 4, 16, 2), gs)
    with refused("kScales and k must not overlap"):
        ops.cache_write(in_memory_of(fs, BF16, 1, 2, 64), f, slots[:1], None, None, fs)
    with refused("k and kCache must not overlap"):
        ops.cache_read(k, k.view(64, 2, 64)[:3], slots)
    with refused("v and kCache must not overlap"):
        ops.cache_read(k, x, slots, v, k.view(64, 2, 64)[20:23])
    with refused("k and kScales must not overlap"):
        ops.cache_read(f, in_memory_of(fs, BF16, 1, 2, 64), slots[:1], None, None, fs)
    with refused("k and slots must not overlap"):
        many = torch.zeros(64, dtype=torch.int64, device=DEV)
        ops.cache_read(k, in_memory_of(many, BF16, 1, 2, 64), many[:1])

    q, out = torch.zeros(3, 4, 64, dtype=BF16, device=DEV), torch.zeros(3, 4, 64, dtype=BF16, device=DEV)
    table, starts, lens = torch.zeros(1, 96, dtype=torch.int64, device=DEV), torch.tensor([0, 3], device=DEV), torch.tensor([5], device=DEV)
    many, each = table.repeat(3, 1), lens.repeat(3)
    lse = torch.zeros(3, 4, device=DEV)

    def both(match, q=q, k=k, v=v, out=out, ks=None, vs=None, lse=lse):
        with refused(match):
            ops.prompt_attention(q, k, v, table, starts, lens, out, 0.1, True, ks, vs, lse)
        with refused(match):
            ops.prefix_attention(q, k, v, table[0], lens, many, each, out, 0.1, ks, vs, lse)

    both("out and kCache must not overlap", out=in_memory_of(k, BF16, 3, 4, 64))
    both("out and vCache must not overlap", out=in_memory_of(v, BF16, 3, 4, 64))
    both("out and kCache must not overlap", q=in_memory_of(k, BF16, 3, 4, 64), out=in_memory_of(k, BF16, 3, 4, 64))
    wide = torch.zeros(8, 16, 2, 64, dtype=FP8, device=DEV), torch.ones(8, 16, 2, device=DEV)
    both("out and kScales must not overlap", q=q[:1], k=wide[0], v=wide[0], ks=wide[1], vs=wide[1].clone(), out=in_memory_of(wide[1], BF16, 1, 4, 64), lse=None)
    both("lse and vScales must not overlap", k=f, v=g, ks=fs, vs=gs, lse=in_memory_of(gs, torch.float32, 3, 4))
    both("lse and kCache must not overlap", lse=in_memory_of(k, torch.float32, 3, 4))
    both("lse and q must not overlap", lse=in_memory_of(q, torch.float32, 3, 4))
    both("out and lse must not overlap", lse=in_memory_of(out, torch.float32, 3, 4))
    with refused("out and blockTable must not overlap"):
        ops.prompt_attention(q[:1], k, v, table, starts, lens, in_memory_of(table, BF16, 1, 4, 64), 0.1)
    with refused("lse and kvLens must not overlap"):
        ops.prompt_attention(q[:1, :2], k, v, table, starts, lens, out[:1, :2], 0.1, True, None, None, in_memory_of(lens, torch.float32, 1, 2))
    with refused("lse and queryStarts must not overlap"):
        ops.prompt_attention(q[:1], k, v, table, starts, lens, out[:1], 0.1, True, None, None, in_memory_of(starts, torch.float32, 1, 4))
    with refused("lse and prefixLen must not overlap"):
        ops.prefix_attention(q[:1, :2], k, v, table[0], lens, table, each[:1], out[:1, :2], 0.1, None, None, in_memory_of(lens, torch.float32, 1, 2))
    with refused("out and prefixBlocks must not overlap"):
        ops.prefix_attention(q[:1], k, v, table[0], lens, many[:1], each[:1], in_memory_of(table, BF16, 1, 4, 64), 0.1)
    torch.cuda.synchronize()


def test_neighbours_in_one_memory_are_no_overlap():
    """Keys and values of one allocation, interleaved or one behind the other; queries and results of one buffer; e4m3 values and
    scales in one block; a cache that is nothing but one block."""
    announce("neighbours in one memory")
    x, slots = torch.ones(3, 2, 64, dtype=BF16, device=DEV), torch.arange(3, device=DEV)
    for both in (torch.zeros(2, 4, 16, 2, 64, dtype=BF16, device=DEV), torch.zeros(4, 2, 16, 2, 64, dtype=BF16, device=DEV).transpose(0, 1),
                 torch.zeros(4, 2, 2, 16, 64, dtype=BF16, device=DEV).permute(1, 0, 3, 2, 4)):
        k, v = both
        ops.cache_write(x, k, slots, 2 * x, v)
        back = torch.zeros(2, 3, 2, 64, dtype=BF16, device=DEV)
        ops.cache_read(k, back[0], slots, v, back[1])
        assert bool((back[0] == 1).all()) and bool((back[1] == 2).all())
        work = torch.ones(2, 3, 4, 64, dtype=BF16, device=DEV)
        table, lens = torch.zeros(1, 1, dtype=torch.int64, device=DEV), torch.tensor([3], device=DEV)
        ops.prompt_attention(work[0], k, v, table, torch.tensor([0, 3], device=DEV), lens, work[1], 0.1)
        assert bool((work[1] == 2).all())
        mixed = torch.ones(3, 8, 64, dtype=BF16, device=DEV)      # q and out interleaved
        ops.prefix_attention(mixed[:, :4], k, v, table[0], lens, table.repeat(3, 1), lens.repeat(3), mixed[:, 4:], 0.1)
        assert bool((mixed[:, 4:] == 2).all()) and bool((mixed[:, :4] == 1).all())
    for blocks in (1, 4):
        raw = torch.zeros(2, blocks, pcie_through.fp8_block_bytes(16, 2, 64), dtype=torch.uint8, device=DEV)
        (k, ks), (v, vs) = (pcie_through.fp8_cache_views(p, 16, 2, 64) for p in raw)
        ops.cache_write(x, k, slots, 2 * x, v, ks, vs)
        back = torch.zeros(2, 3, 2, 64, dtype=BF16, device=DEV)
        ops.cache_read(k, back[0], slots, v, back[1], ks, vs)
        assert bool((back[0] == 1).all()) and bool((back[1] == 2).all())


def test_gradients_of_scales_and_of_the_logarithm():
    """A gradient would have to flow through e4m3 scales and through lse as through the values."""
    announce("scales and lse that require a gradient")
    (f, fs), (g, gs) = cache_of(FP8), cache_of(FP8)
    x, slots = torch.zeros(3, 2, 64, dtype=BF16, device=DEV), torch.arange(3, device=DEV)
    q, out, lse = torch.zeros(3, 4, 64, dtype=BF16, device=DEV), torch.zeros(3, 4, 64, dtype=BF16, device=DEV), torch.zeros(3, 4, device=DEV)
    table, starts, lens = torch.zeros(1, 2, dtype=torch.int64, device=DEV), torch.tensor([0, 3], device=DEV), torch.tensor([5], device=DEV)

    def calls(ks, vs, lse):
        yield "write", lambda: ops.cache_write(x, f, slots, x.clone(), g, ks, vs)
        yield "read", lambda: ops.cache_read(f, x, slots, g, x.clone(), ks, vs)
        yield "prompt", lambda: ops.prompt_attention(q, f, g, table, starts, lens, out, 0.1, True, ks, vs, lse)
        yield "prefix", lambda: ops.prefix_attention(q, f, g, table[0], lens, table.repeat(3, 1), lens.repeat(3), out, 0.1, ks, vs, lse)

    for what, change in (("kScales", dict(ks=fs.clone().requires_grad_())), ("vScales", dict(vs=gs.clone().requires_grad_())),
                         ("lse", dict(lse=lse.clone().requires_grad_()))):
        for name, call in calls(**{**dict(ks=fs, vs=gs, lse=lse), **change}):
            if what == "lse" and name in ("write", "read"):
                continue
            with refused(what + " requires a gradient"):
                call()
            with torch.no_grad():
                call()
    torch.cuda.synchronize()


def test_tangents_of_forward_mode():
    """The ops have no derivative in either direction: a tangent is refused, not dropped."""
    import torch.autograd.forward_ad as forward

    announce("tangents")
    (k, _), (v, _) = cache_of(BF16), cache_of(BF16)
    (f, fs), (g, gs) = cache_of(FP8), cache_of(FP8)
    x, slots = torch.zeros(3, 2, 64, dtype=BF16, device=DEV), torch.arange(3, device=DEV)
    q, out, lse = torch.zeros(3, 4, 64, dtype=BF16, device=DEV), torch.zeros(3, 4, 64, dtype=BF16, device=DEV), torch.zeros(3, 4, device=DEV)
    table, starts, lens = torch.zeros(1, 2, dtype=torch.int64, device=DEV), torch.tensor([0, 3], device=DEV), torch.tensor([5], device=DEV)

    def attend(q=q, k=k, v=v, out=out, lse=lse, ks=None, vs=None):
        yield lambda: ops.prompt_attention(q, k, v, table, starts, lens, out, 0.1, True, ks, vs, lse)
        yield lambda: ops.prefix_attention(q, k, v, table[0], lens, table.repeat(3, 1), lens.repeat(3), out, 0.1, ks, vs, lse)

    def dual(t):
        return forward.make_dual(t, torch.ones_like(t))

    with forward.dual_level():
        for name, t in (("q", q), ("k", k), ("v", v), ("out", out), ("lse", lse)):
            for call in attend(**{name: dual(t)}):
                with refused({"k": "kCache", "v": "vCache"}.get(name, name) + " carries a tangent"):
                    call()
        for name, t in (("ks", fs), ("vs", gs)):
            for call in attend(**{**dict(k=f, v=g, ks=fs, vs=gs), name: dual(t)}):
                with refused(name[0] + "Scales carries a tangent"):
                    call()
        with refused("k carries a tangent"):
            ops.cache_write(dual(x), k, slots)
        with refused("v carries a tangent"):
            ops.cache_write(x, k, slots, dual(x.clone()), v)
        with refused("vCache carries a tangent"):
            ops.cache_read(k, x, slots, dual(v), x.clone())
        with torch.no_grad():      # which does not switch forward mode off
            with refused("k carries a tangent"):
                ops.cache_write(dual(x), k, slots)
        for call in attend(q=forward.unpack_dual(dual(q)).primal):
            call()
    torch.cuda.synchronize()


def test_views_that_begin_at_one_address():
    """Strided views share memory for certain where they begin at one address, whatever their strides: e4m3 blocks that carry their
    scales, given for both sides; results that begin where the queries do but lie otherwise."""
    announce("strided views of one address")
    x, slots = torch.zeros(3, 2, 64, dtype=BF16, device=DEV), torch.arange(3, device=DEV)
    raw = torch.zeros(4, pcie_through.fp8_block_bytes(16, 2, 64), dtype=torch.uint8, device=DEV)
    (k, ks), (again, again_s) = pcie_through.fp8_cache_views(raw, 16, 2, 64), pcie_through.fp8_cache_views(raw, 16, 2, 64)
    other = torch.ones(4, 16, 2, device=DEV)
    with refused("kCache and vCache must not overlap"):
        ops.cache_write(x, k, slots, x.clone(), again, ks, other)
    (far, _), = [pcie_through.fp8_cache_views(raw.clone(), 16, 2, 64)]
    with refused("kScales and vScales must not overlap"):
        ops.cache_write(x, k, slots, x.clone(), far, ks, again_s)
    wide = torch.zeros(3, 2, 128, dtype=BF16, device=DEV)
    with refused("k and v must not overlap"):
        ops.cache_read(k, wide[..., :64], slots, far, wide[..., :64], ks, other)

    buffer = torch.zeros(3, 8, 128, dtype=BF16, device=DEV)
    q = buffer[:, :4, :64]
    table, starts, lens = torch.zeros(1, 2, dtype=torch.int64, device=DEV), torch.tensor([0, 3], device=DEV), torch.tensor([5], device=DEV)
    cache = torch.zeros(4, 16, 2, 64, dtype=BF16, device=DEV)
    for out in (buffer[:, ::2, :64], buffer.view(6, 4, 128)[:3, :, :64]):
        with refused("out and q, unless they are one tensor, must not overlap"):
            ops.prompt_attention(q, cache, cache, table, starts, lens, out, 0.1)
        with refused("out and q, unless they are one tensor, must not overlap"):
            ops.prefix_attention(q, cache, cache, table[0], lens, table.repeat(3, 1), lens.repeat(3), out, 0.1)
    # one view of a wider buffer in place of another of the same strides: results in place of the queries; a stride of one row is no stride
    ops.prompt_attention(q, cache, cache, table, starts, lens, buffer[:, :4, :64], 0.1)
    one = buffer[:1, :4, :64]
    ops.prefix_attention(one, cache, cache, table[0], lens, table, lens, one.as_strided((1, 4, 64), (64, 128, 1)), 0.1)
    torch.cuda.synchronize()
