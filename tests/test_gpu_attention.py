"""prompt_attention and prefix_attention on the GPU against a plain 64-bit statement, at the lengths, head layouts and
masks where they can go wrong. Tolerances: cache_reference.bounds. Tokens no sequence owns are NaN in every cache."""
import pytest
import torch

import heterofusedkernels_amd  # noqa: F401
import pcie_through  # noqa: F401
from cache_reference import FP8, Cache, attend, bounds, tables
from gpu_helpers import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16
ops = torch.ops.pcie_through


def close(got, want, allowed, what):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    off = (got - want).abs()
    bad = ~((off <= allowed) | (got == want) | torch.isnan(want))
    assert not bool(bad.any()), "%s: %d of %d off, worst %.3g of %.3g allowed" % (
        what, int(bad.sum()), bad.numel(), float(off[bad].max()), float(allowed.expand_as(off)[bad].min()))


def visible_of(n, L, causal):
    i, j = torch.arange(n)[:, None], torch.arange(L)[None]
    return j <= L - n + i if causal else torch.ones(n, L, dtype=torch.bool)


def prompt_case(q_lens, kv_lens, Hq, H, D, T, kind, cache_kind, causal=True, order="thd", behind=3, seed=0, spare=2):
    gen = torch.Generator().manual_seed(seed + 17)
    blocks = sum(-(-n // T) for n in kv_lens) + spare
    cache = Cache(blocks, T, H, D, kind, cache_kind, order, seed)
    table, slots = tables(gen, kv_lens, T, blocks)
    cache.fill(torch.cat(slots) if slots else torch.zeros(0, dtype=torch.int64))
    total = sum(q_lens) + behind
    q = torch.randn(total, Hq, D, generator=gen).to(kind)
    starts = torch.tensor([0] + torch.tensor(q_lens).cumsum(0).tolist())
    return cache, table, slots, q, starts


def check_prompt(cache, table, slots, q, starts, kv_lens, causal, scale, q_d=None, out=None):
    kind, D = cache.kind, cache.dim
    k, v, ks, vs = cache.to(DEV)
    out = torch.full(q.shape, 5.0, dtype=kind, device=DEV) if out is None else out
    lse = torch.full(q.shape[:2], 5.0, device=DEV)
    ops.prompt_attention(q.to(DEV) if q_d is None else q_d, k, v, table.to(DEV), starts.to(DEV), torch.tensor(kv_lens).to(DEV), out, scale, causal, ks, vs, lse)
    torch.cuda.synchronize()
    for b, L in enumerate(kv_lens):
        first, last = int(starts[b]), int(starts[b + 1])
        kk, vv = cache.rows(slots[b])
        want, wl, size, reach = attend(q[first:last].double(), kk, vv, visible_of(last - first, L, causal), scale)
        o_ok, l_ok = bounds(want, wl, size, reach, kind, D, L)
        close(out[first:last], want, o_ok, "out of sequence %d" % b)
        close(lse[first:last], wl, l_ok, "lse of sequence %d" % b)
    end = int(starts[-1])
    assert bool((out[end:] == 5.0).all()) and bool((lse[end:] == 5.0).all()), "rows behind the last sequence"


PROMPTS = [  # q lens, kv lens, Hq, H, D, T
    ([1], [1], 4, 4, 64, 16),
    ([33], [33], 8, 2, 128, 16),
    ([130, 1, 0, 64, 7], [130, 70, 40, 64, 300], 8, 2, 128, 16),
    ([5, 40], [3, 0], 4, 1, 64, 16),                       # rows that see nothing
    ([257], [257], 6, 2, 64, 64),
    ([19, 100], [200, 161], 7, 1, 96, 5),                  # groups and blocks that are no powers of two
    ([66, 3], [66, 90], 4, 2, 256, 32),
    ([70], [111], 4, 2, 208, 16),
    ([2, 2, 2], [2, 3, 65], 64, 8, 128, 1),
    ([40], [1500], 8, 1, 128, 16),                         # few rows, many keys: split
    ([1, 4, 1], [700, 1200, 3], 16, 2, 64, 16),
    ([600], [600], 4, 1, 16, 16),
]


@pytest.mark.parametrize("kind,cache_kind", [(BF16, BF16), (FP16, FP16), (BF16, FP8), (FP16, FP8)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", PROMPTS, ids=str)
def test_prompt_attention(case, causal, kind, cache_kind):
    q_lens, kv_lens, Hq, H, D, T = case
    announce("prompt %s causal=%s %s %s" % (case, causal, kind, cache_kind))
    order = "htd" if T in (16, 5) else "thd"
    cache, table, slots, q, starts = prompt_case(q_lens, kv_lens, Hq, H, D, T, kind, cache_kind, causal, order)
    check_prompt(cache, table, slots, q, starts, kv_lens, causal, D ** -0.5)


PREFIXES = [  # prefix, own lens, Hq, H, D, T
    (0, [1], 4, 4, 64, 16),
    (0, [5, 0, 700, 33, 1], 8, 2, 128, 16),
    (20, [0, 3, 17], 8, 2, 128, 16),
    (333, [40] * 3, 8, 2, 128, 16),                        # prefix and own tokens by one launch
    (333, [40, 0, 1, 90, 77] * 5, 16, 2, 64, 16),          # the prefix by the wide kernel
    (700, [9] * 10, 6, 1, 128, 16),                        # 60 rows: four row blocks
    (65, [30, 31], 28, 4, 96, 5),
    (129, [64, 128, 129], 40, 2, 128, 32),
    (100, [200, 10], 6, 2, 256, 16),
    (100, [7] * 9, 8, 1, 208, 16),
    (1, [1] * 70, 4, 4, 16, 16),
    (0, [300] * 2, 80, 1, 64, 64),                         # a group of 80: more than one row tile
    (0, [2500], 4, 1, 128, 16),                            # split
]


@pytest.mark.parametrize("kind,cache_kind", [(BF16, BF16), (FP16, FP16), (BF16, FP8), (FP16, FP8)])
@pytest.mark.parametrize("case", PREFIXES, ids=str)
def test_prefix_attention(case, kind, cache_kind):
    prefix, own, Hq, H, D, T = case
    announce("prefix %s %s %s" % (case, kind, cache_kind))
    gen = torch.Generator().manual_seed(prefix + 3)
    blocks = sum(-(-n // T) for n in own) + -(-prefix // T) + 2
    cache = Cache(blocks, T, H, D, kind, cache_kind, "htd" if T == 16 else "thd", prefix)
    table, slots = tables(gen, [prefix] + own, T, blocks)
    cache.fill(torch.cat(slots))
    prefix_blocks = table[0, :-(-prefix // T)].contiguous()
    width = max(-(-n // T) for n in own)
    check_prefix(cache, prefix_blocks, slots[0], table[1:, :width].contiguous(), slots[1:], own,
                 torch.randn(len(own), Hq, D, generator=gen).to(kind), D ** -0.5)


def check_prefix(cache, prefix_blocks, prefix_slots, table, slots, own, q, scale):
    k, v, ks, vs = cache.to(DEV)
    out = torch.full(q.shape, 5.0, dtype=cache.kind, device=DEV)
    lse = torch.full(q.shape[:2], 5.0, device=DEV)
    ops.prefix_attention(q.to(DEV), k, v, prefix_blocks.to(DEV), torch.tensor([len(prefix_slots)], device=DEV), table.to(DEV),
                         torch.tensor(own, device=DEV), out, scale, ks, vs, lse)
    torch.cuda.synchronize()
    for b, n in enumerate(own):
        kk, vv = cache.rows(torch.cat([prefix_slots, slots[b]]))
        keys = len(prefix_slots) + n
        want, wl, size, reach = attend(q[b:b + 1].double(), kk, vv, torch.ones(1, keys, dtype=torch.bool), scale)
        o_ok, l_ok = bounds(want, wl, size, reach, cache.kind, cache.dim, keys)
        close(out[b:b + 1], want, o_ok, "out of row %d" % b)
        close(lse[b:b + 1], wl, l_ok, "lse of row %d" % b)
