"""The cache and attention entry points as far as they go without a GPU: schemas, struct layouts, refusals (all of them come
before a launch), workspace sizes, the views of e4m3 blocks, and the plain statements the GPU tests compare with."""
import os
import subprocess

import pytest
import torch

import heterofusedkernels_amd  # noqa: F401
import pcie_through
from cache_reference import FP8, dequantise, quantise
from heterofusedkernels_amd import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_schemas():
    want = {
        "cache_write": "pcie_through::cache_write(Tensor k, Tensor(a!) kCache, Tensor slots, Tensor? v=None, Tensor(b!)? vCache=None, "
                       "Tensor(c!)? kScales=None, Tensor(d!)? vScales=None) -> ()",
        "cache_read": "pcie_through::cache_read(Tensor kCache, Tensor(a!) k, Tensor slots, Tensor? vCache=None, Tensor(b!)? v=None, "
                      "Tensor? kScales=None, Tensor? vScales=None) -> ()",
        "prompt_attention": "pcie_through::prompt_attention(Tensor q, Tensor kCache, Tensor vCache, Tensor blockTable, Tensor queryStarts, "
                            "Tensor kvLens, Tensor(a!) out, float scale, bool causal=True, Tensor? kScales=None, Tensor? vScales=None, "
                            "Tensor(b!)? lse=None) -> ()",
        "prefix_attention": "pcie_through::prefix_attention(Tensor q, Tensor kCache, Tensor vCache, Tensor prefixBlocks, Tensor prefixLen, "
                            "Tensor blockTable, Tensor kvLens, Tensor(a!) out, float scale, Tensor? kScales=None, Tensor? vScales=None, "
                            "Tensor(b!)? lse=None) -> ()",
    }
    for name, schema in want.items():
        assert str(getattr(torch.ops.pcie_through, name).default._schema) == schema


def test_no_cpu_fallback():
    x, cache, slots = torch.zeros(1, 1, 16), torch.zeros(1, 1, 1, 16), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(NotImplementedError):
        torch.ops.pcie_through.cache_write(x, cache, slots)
    with pytest.raises(NotImplementedError):
        torch.ops.pcie_through.prompt_attention(x, cache, cache, slots[None], torch.tensor([0, 1]), slots, x, 1.0)


def test_structs_match_the_header(tmp_path):
    import ctypes

    src = tmp_path / "s.c"
    names = {"hfk_cache_plane": capi.CachePlane, "hfk_token_rows": capi.TokenRows, "hfk_attention": capi.Attention}
    lines = ["printf(\"%%zu\\n\", sizeof(%s));" % n for n in names]
    for n, c in names.items():
        lines += ["printf(\"%%zu\\n\", offsetof(%s, %s));" % (n, f[0]) for f in c._fields_]
    src.write_text("#include <stdio.h>\n#include \"hfk.h\"\nint main(void) { %s return 0; }\n" % " ".join(lines))
    exe = tmp_path / "s"
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Werror", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    got = [int(x) for x in subprocess.check_output([str(exe)], text=True).split()]
    want = [ctypes.sizeof(c) for c in names.values()] + [getattr(c, f[0]).offset for c in names.values() for f in c._fields_]
    assert got == want


def plane(values=4096, scales=0, blocks=8, T=16, heads=2, dim=64, kind=capi.BF16, strides=None):
    b, t, h = strides or (T * heads * dim, heads * dim, dim)
    return capi.CachePlane(values, scales, b, t, h, T * heads, heads, 1, blocks, T, heads, dim, kind)


def rows(data=4096, heads=2, dim=64, kind=capi.BF16, strides=None):
    t, h = strides or (heads * dim, dim)
    return capi.TokenRows(data, t, h, kind)


def test_cache_entry_points_refuse():
    """Addresses are made up: nothing is launched, so nothing reads them."""
    for call in (capi.cache_write, capi.cache_read):
        assert call(None, rows(), None, None, 8, 1) == -1
        assert call(plane(), None, None, None, 8, 1) == -1
        assert call(plane(), rows(), plane(), None, 8, 1) == -1
        assert call(plane(), rows(), None, None, 0, 1) == -1                                     # slots
        assert call(plane(values=0), rows(), None, None, 8, 1) == -1
        assert call(plane(), rows(data=0), None, None, 8, 1) == -1
        assert call(plane(kind=capi.FP8_E4M3), rows(), None, None, 8, 1) == -1                   # scales
        assert call(plane(kind=7), rows(), None, None, 8, 1) == capi.ERR_BAD_TYPE
        assert call(plane(), rows(kind=capi.FP8_E4M3), None, None, 8, 1) == capi.ERR_BAD_TYPE
        assert call(plane(), rows(kind=capi.FP16), None, None, 8, 1) == capi.ERR_BAD_TYPE
        assert call(plane(), rows(), plane(kind=capi.FP8_E4M3, scales=64), rows(), 8, 1) == capi.ERR_BAD_TYPE
        assert call(plane(T=0), rows(), None, None, 8, 1) == -2
        assert call(plane(dim=0), rows(), None, None, 8, 1) == -2
        assert call(plane(strides=(-1, 128, 64)), rows(), None, None, 8, 1) == -2
        assert call(plane(strides=(1 << 41, 128, 64)), rows(), None, None, 8, 1) == -2
        assert call(plane(), rows(), plane(blocks=9), rows(), 8, 1) == -2
        assert call(plane(dim=1040), rows(dim=1040), None, None, 8, 1) == -3
        assert call(plane(), rows(), None, None, 8, 1 << 31) == -3
        assert call(plane(heads=60000), rows(heads=60000), None, None, 8, 1 << 20) == -3
        assert call(plane(values=4097), rows(), None, None, 8, 1) == capi.ERR_BAD_ALIGNMENT
        assert call(plane(kind=capi.FP8_E4M3, scales=66), rows(), None, None, 8, 1) == capi.ERR_BAD_ALIGNMENT
        assert call(plane(), rows(), None, None, 0, 0) == 0                                      # nothing to do
        assert call(plane(values=0, blocks=0), rows(), None, None, 8, 1) == 0                    # no slot anywhere
    for rc, word in ((capi.ERR_BAD_TYPE, "type"), (capi.ERR_BAD_ALIGNMENT, "16 bytes"), (capi.ERR_WORKSPACE_TOO_SMALL, "workspace")):
        assert word in capi.status_string(rc)


def attention(n=4, q_heads=4, scale=0.125, k=None, v=None, q=None, out=None, lse=0):
    k = plane() if k is None else k
    return capi.Attention(k, k if v is None else v, q or rows(heads=q_heads, dim=k.head_dim), out or rows(heads=q_heads, dim=k.head_dim), lse, n, q_heads,
                          scale)


def test_attention_entry_points_refuse():
    def both(a):
        got = {capi.prompt_attention(a, 8, 1, 4, 8, 8, True), capi.prefix_attention(a, 8, 4, 8, 8, 4, 8),
               capi.prompt_attention_workspace(a, 1, 4)[0], capi.prefix_attention_workspace(a, 4, 4)[0]}
        assert len(got) == 1, got
        return got.pop()

    assert both(None) == -1
    assert both(attention(q_heads=3)) == -2
    assert both(attention(q_heads=0)) == -2
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert both(attention(scale=scale)) == -2
    assert both(attention(k=plane(dim=72, strides=(16 * 144, 144, 72)))) == -2                   # no multiple of 16
    assert both(attention(k=plane(dim=272, strides=(16 * 544, 544, 272)))) == -2                 # beyond 256
    assert both(attention(v=plane(T=8))) == -2
    assert both(attention(v=plane(blocks=9))) == -2
    assert both(attention(v=plane(kind=capi.FP16))) == capi.ERR_BAD_TYPE
    assert both(attention(out=rows(heads=4, kind=capi.FP16))) == capi.ERR_BAD_TYPE
    assert both(attention(k=plane(kind=capi.FP16))) == capi.ERR_BAD_TYPE
    assert both(attention(q=rows(heads=4, strides=(260, 65)))) == capi.ERR_BAD_ALIGNMENT
    assert both(attention(out=rows(data=4104, heads=4))) == capi.ERR_BAD_ALIGNMENT
    assert both(attention(k=plane(values=4104))) == capi.ERR_BAD_ALIGNMENT
    assert both(attention(lse=4098)) == capi.ERR_BAD_ALIGNMENT
    assert both(attention(n=1 << 31)) == -3
    assert both(attention(k=plane(strides=(1 << 33, 128, 64)))) == -3                            # a block beyond 32 bits
    good = attention()
    assert capi.prompt_attention(good, 0, 1, 4, 8, 8, True) == -1
    assert capi.prompt_attention(good, 8, 1, 4, 0, 8, True) == -1
    assert capi.prefix_attention(good, 0, 4, 8, 8, 4, 8, 256, 1 << 40) == -1
    assert capi.prefix_attention(good, 8, 4, 0, 8, 4, 8, 256, 1 << 40) == -1
    assert capi.prompt_attention(good, 8, 1, 1 << 31, 8, 8, True) == -3                          # keys of one sequence
    assert capi.prefix_attention(good, 8, 4, 8, 8, 4, 8, 0, 0) == -1                             # its workspace
    assert capi.prefix_attention(good, 8, 4, 8, 8, 4, 8, 256, 16) == capi.ERR_WORKSPACE_TOO_SMALL
    assert capi.prefix_attention(good, 8, 4, 8, 8, 4, 8, 264, 1 << 40) == capi.ERR_BAD_ALIGNMENT
    # nothing to do
    assert capi.prompt_attention(attention(n=0), 8, 1, 4, 8, 8, True) == 0
    assert capi.prompt_attention(good, 8, 0, 4, 8, 8, True) == 0
    assert capi.prefix_attention(attention(n=0), 8, 4, 8, 8, 4, 8) == 0
    assert capi.prompt_attention_workspace(attention(n=0), 1, 4) == (0, 0) == capi.prompt_attention_workspace(good, 0, 4)
    assert capi.prefix_attention_workspace(attention(n=0), 4, 4) == (0, 0) == capi.prefix_attention_workspace(attention(n=0), 0, 0)


def test_workspace_sizes():
    """Many rows need none; few rows over many keys some, and never more than a share of the rows for every resident workgroup."""
    rc, size = capi.prompt_attention_workspace(attention(n=100000), 1, 10000)
    assert rc == 0 and size == 0
    rc, size = capi.prompt_attention_workspace(attention(n=4), 1, 10000)
    assert rc == 0 and 0 < size <= 257 * 4 * 4 * (64 + 2) * 4 + 512
    assert capi.prompt_attention_workspace(attention(n=4), 1, 8)[1] == 0                          # 128 keys: not worth a split
    for n in (1, 5, 300):
        for width in (0, 1, 77, 100000):
            rc, size = capi.prefix_attention_workspace(attention(n=n), 0, width)
            assert rc == 0 and size % 256 == 0
            assert size <= (512 + n) * 4 * (64 + 2) * 4 + 512
            assert capi.prefix_attention_workspace(attention(n=n), 50, width)[1] > size


def test_views_of_blocks_that_carry_their_scales():
    T, H, D = 16, 3, 32
    size = pcie_through.fp8_block_bytes(T, H, D)
    assert size == T * H * (D + 4)
    pool = torch.zeros(2, 5, size, dtype=torch.uint8)
    for plane_ in pool.unbind(0):      # the second has an offset into the pool's memory
        v, s = pcie_through.fp8_cache_views(plane_, T, H, D)
        assert v.shape == (5, T, H, D) and v.dtype == FP8 and s.shape == (5, T, H) and s.dtype == torch.float32
        v.view(torch.uint8)[3, 2, 1, 7] = 9
        s[3, 15, 2] = 4.0
        assert plane_[3, (2 * H + 1) * D + 7] == 9
        assert plane_[3, T * H * D:].view(torch.float32)[15 * H + 2] == 4.0
        assert int((plane_ != 0).sum()) == 3      # the value, and two bytes of 4.0 (0x40800000)
    for bad in (pool[0].float(), pool[0][:, :-16], pool[0].t().contiguous().t()):
        with pytest.raises(ValueError):
            pcie_through.fp8_cache_views(bad, T, H, D)
    with pytest.raises(ValueError):
        pcie_through.fp8_block_bytes(16, 2, 40)
    with pytest.raises(ValueError):
        pcie_through.fp8_cache_views(torch.zeros(2, pcie_through.fp8_block_bytes(1, 3, 32), dtype=torch.uint8), 1, 3, 32)


def test_plain_quantiser_follows_its_definition():
    x = torch.tensor([[0.0, 0.0], [448.0, 1.0], [449.0, 1.0], [float("inf"), 3.0], [float("nan"), 3.0], [2.0 ** -130, 0.0], [3.0e38, 0.0]])
    q, s = quantise(x)
    assert s.tolist() == [1.0, 1.0, 2.0, 2.0 ** -7, 2.0 ** -7, 2.0 ** -126, 2.0 ** 119]
    assert q.float()[1].tolist() == [448.0, 1.0] and q.float()[2].tolist() == [224.0, 0.5]
    assert q.float()[3].tolist() == [448.0, 384.0] and torch.isnan(q.float()[4, 0])
    assert dequantise(q, s, torch.float16)[6, 0] == torch.finfo(torch.float16).max
    gen = torch.Generator().manual_seed(0)
    y = torch.randn(50, 64, generator=gen)
    q, s = quantise(y)
    assert bool(((dequantise(q, s, torch.float32) - y).abs() <= y.abs() * 2.0 ** -4 + s[:, None] * 2.0 ** -10).all())


def test_scales_of_scores_beyond_the_range_are_refused():
    """At its ends the running maximum's threshold, or the scale in base 2, would leave 32 bits."""
    for scale in (1e-39, 2.0 ** -101, 2.0 ** 101, 3e38):
        assert capi.prompt_attention_workspace(attention(scale=scale), 1, 4)[0] == -2
        assert capi.prefix_attention_workspace(attention(scale=scale), 4, 4)[0] == -2
    for scale in (2.0 ** -100, 2.0 ** 100):
        assert capi.prompt_attention_workspace(attention(scale=scale), 1, 4)[0] == 0
