"""What no query sees does not count, whatever it holds: e4m3 scales of tokens that were never written are as arbitrary as
their values. Tolerances: cache_reference.bounds."""
import pytest
import torch

import heterofusedkernels_amd  # noqa: F401
import pcie_through  # noqa: F401
from cache_reference import FP8, Cache, attend, bounds, tables
from gpu_helpers import announce
from test_gpu_attention import check_prefix, check_prompt, close, visible_of

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16
ops = torch.ops.pcie_through
SCALES = {"nan": float("nan"), "inf": float("inf"), "largest": 3.0e38, "zero": 0.0}


def unwritten(cache, slots, scale, code):
    """Every token outside `slots` holds this scale and this e4m3 code; the cache's first token is one of them."""
    owned = torch.zeros(cache.blocks * cache.T, dtype=torch.bool)
    owned[torch.cat(slots)] = True
    assert not bool(owned[0])
    rest = torch.nonzero(~owned)[:, 0]
    for values, scales in ((cache.k, cache.ks), (cache.v, cache.vs)):
        values.view(torch.uint8)[rest // cache.T, rest % cache.T] = code
        scales[rest // cache.T, rest % cache.T] = scale


@pytest.mark.parametrize("code", [0x7f, 0x00, 0x7e], ids=["nan", "zero", "448"])
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("prefix,own,Hq,H,D,T", [(0, [5, 0, 700, 33, 1], 8, 4, 128, 16), (45, [3, 40], 8, 1, 64, 16), (300, [9] * 30, 8, 2, 96, 5),
                                                 (20, [31, 97], 6, 2, 256, 32)])
def test_scales_of_unwritten_tokens_under_a_prefix(prefix, own, Hq, H, D, T, scale, code):
    announce("prefix %d + %s, %d heads over %d of %d, unwritten scales %s, codes %d" % (prefix, own, Hq, H, D, scale, code))
    for kind in (BF16, FP16):
        gen = torch.Generator().manual_seed(prefix + D)
        blocks = 1 + sum(-(-n // T) for n in own) + -(-prefix // T)
        cache = Cache(blocks, T, H, D, kind, FP8, "htd" if T == 16 else "thd", prefix)
        table, slots = tables(gen, [prefix] + own, T, blocks, first=1)
        cache.fill(torch.cat(slots))
        unwritten(cache, slots, SCALES[scale], code)
        width = max(-(-n // T) for n in own)
        check_prefix(cache, table[0, :-(-prefix // T)].contiguous(), slots[0], table[1:, :width].contiguous(), slots[1:], own,
                     torch.randn(len(own), Hq, D, generator=gen).to(kind), D ** -0.5)


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("q_lens,kv_lens,Hq,H,D,T", [([33], [33], 8, 2, 128, 16), ([5, 40, 1], [70, 900, 3], 8, 2, 64, 16), ([20], [77], 4, 2, 256, 32)])
def test_scales_of_unwritten_tokens_behind_prompts(q_lens, kv_lens, Hq, H, D, T, scale):
    announce("prompts %s of %s, %d heads over %d of %d, unwritten scales %s" % (q_lens, kv_lens, Hq, H, D, scale))
    for kind in (BF16, FP16):
        gen = torch.Generator().manual_seed(D)
        blocks = 1 + sum(-(-n // T) for n in kv_lens)
        cache = Cache(blocks, T, H, D, kind, FP8, "thd", 3)
        table, slots = tables(gen, kv_lens, T, blocks, first=1)
        cache.fill(torch.cat(slots))
        unwritten(cache, slots, SCALES[scale], 0x7f)
        q = torch.randn(sum(q_lens) + 2, Hq, D, generator=gen).to(kind)
        starts = torch.tensor([0] + torch.tensor(q_lens).cumsum(0).tolist())
        check_prompt(cache, table, slots, q, starts, kv_lens, True, D ** -0.5)


@pytest.mark.parametrize("scale", SCALES)
def test_scales_of_unwritten_tokens_beside_a_missing_block(scale):
    """Tokens of a table entry outside the cache are given the first token's place, which holds nothing that was written."""
    announce("missing blocks, unwritten scales %s" % scale)
    T, H, Hq, D, L = 16, 4, 8, 128, 200
    gen = torch.Generator().manual_seed(4)
    blocks = 2 + -(-L // T)
    cache = Cache(blocks, T, H, D, BF16, FP8, "thd", 8)
    table, slots = tables(gen, [L], T, blocks, first=1)
    cache.fill(slots[0])
    table[0, 1], table[0, 6] = -1, blocks
    j = torch.arange(L)
    known = (table[0, j // T] >= 0) & (table[0, j // T] < blocks)
    unwritten(cache, [slots[0][known]], SCALES[scale], 0x7f)
    kk, vv = (torch.zeros(L, H, D, dtype=torch.float64) for _ in "kv")
    kk[known], vv[known] = cache.rows(slots[0][known])
    k, v, ks, vs = cache.to(DEV)
    q = torch.randn(7, Hq, D, generator=gen).to(BF16)
    out, lse = torch.zeros(q.shape, dtype=BF16, device=DEV), torch.zeros(q.shape[:2], device=DEV)
    ops.prompt_attention(q.to(DEV), k, v, table.to(DEV), torch.tensor([0, 7], device=DEV), torch.tensor([L], device=DEV), out, 0.1, True, ks, vs, lse)
    want, wl, size, reach = attend(q.double(), kk, vv, visible_of(7, L, True) & known[None], 0.1)
    o_ok, l_ok = bounds(want, wl, size, reach, BF16, D, L)
    close(out, want, o_ok, "prompt")
    close(lse, wl, l_ok, "prompt lse")
    ops.prefix_attention(q.to(DEV), k, v, table[0].to(DEV), torch.tensor([L], device=DEV), table.repeat(7, 1).contiguous()[:, :2].contiguous().to(DEV),
                         torch.tensor([0, 1, 16, 17, 20, 31, 32], device=DEV), out, 0.1, ks, vs, lse)
    for row, n in enumerate((0, 1, 16, 17, 20, 31, 32)):
        seen = torch.cat([known, known[:n]])[None]
        want, wl, size, reach = attend(q[row:row + 1].double(), torch.cat([kk, kk[:n]]), torch.cat([vv, vv[:n]]), seen, 0.1)
        o_ok, l_ok = bounds(want, wl, size, reach, BF16, D, L + n)
        close(out[row:row + 1], want, o_ok, "prefix row %d" % row)
        close(lse[row:row + 1], wl, l_ok, "prefix lse row %d" % row)
