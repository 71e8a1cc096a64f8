"""Long walks of one workgroup over its keys: so many cache heads that the keys are not split, so many keys that every stage and
every kept place is taken again and again, for each head size and type. Tolerances: cache_reference.bounds."""
import pytest
import torch

import heterofusedkernels_amd  # noqa: F401
import pcie_through  # noqa: F401
from cache_reference import FP8, attend, bounds
from gpu_helpers import announce
from heterofusedkernels_amd import capi
from test_cache_boundary_cpu import attention, plane
from test_gpu_attention import check_prompt, close, prompt_case, visible_of

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16
ops = torch.ops.pcie_through
TYPES = [(BF16, BF16), (FP16, FP16), (BF16, FP8), (FP16, FP8)]


def unsplit(q_lens, kv_lens, Hq, H, D, T):
    """No workspace is asked for where every row's keys are walked by one workgroup."""
    a = attention(n=sum(q_lens) + 3, q_heads=Hq, k=plane(heads=H, dim=D, T=T, blocks=1 << 20))
    return capi.prompt_attention_workspace(a, len(q_lens), max(-(-n // T) for n in kv_lens)) == (0, 0)


@pytest.mark.parametrize("kind,cache_kind", TYPES)
@pytest.mark.parametrize("D,L", [(64, 1357), (128, 1357), (256, 805), (80, 1301), (208, 737)])
def test_one_prompt(D, L, kind, cache_kind):
    """21 tiles of 64 keys, or 26 of 32; queries whose last tiles are cut by the causal edge."""
    announce("one prompt of 70 behind %d, 260 heads over 130 of %d, %s %s" % (L - 70, D, kind, cache_kind))
    assert unsplit([70], [L], 260, 130, D, 16)
    cache, table, slots, q, starts = prompt_case([70], [L], 260, 130, D, 16, kind, cache_kind, order="htd" if D == 128 else "thd", seed=D)
    check_prompt(cache, table, slots, q, starts, [L], D != 80, D ** -0.5)


@pytest.mark.parametrize("kind,cache_kind", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_several_prompts(D, kind, cache_kind):
    """Row tiles of walks of different lengths, from one tile to 19 or 38, beside each other."""
    q_lens, kv_lens = [300, 1, 40, 0, 5], [1190, 700, 901, 33, 5]
    announce("prompts %s of %s, 44 heads of %d, %s %s" % (q_lens, kv_lens, D, kind, cache_kind))
    assert unsplit(q_lens, kv_lens, 44, 44, D, 16)
    cache, table, slots, q, starts = prompt_case(q_lens, kv_lens, 44, 44, D, 16, kind, cache_kind, seed=D + 1)
    check_prompt(cache, table, slots, q, starts, kv_lens, True, D ** -0.5)


@pytest.mark.parametrize("kind,cache_kind", [(BF16, BF16), (FP16, FP8)])
@pytest.mark.parametrize("D,prefix", [(64, 1357), (128, 1357), (256, 805)])
def test_a_wide_prefix(D, prefix, kind, cache_kind):
    announce("70 rows under a prefix of %d, 130 heads of %d, %s %s" % (prefix, D, kind, cache_kind))
    rows, H = 70, 130
    cache, table, slots, q, _ = prompt_case([rows], [prefix], H, H, D, 16, kind, cache_kind, behind=0, seed=D + 2)
    k, v, ks, vs = cache.to(DEV)
    out, lse = torch.zeros(q.shape, dtype=kind, device=DEV), torch.zeros(q.shape[:2], device=DEV)
    table, none = table.to(DEV), torch.zeros(rows, dtype=torch.int64, device=DEV)
    ops.prefix_attention(q.to(DEV), k, v, table[0], torch.tensor([prefix], device=DEV), table[:, :1].repeat(rows, 1), none, out, D ** -0.5, ks, vs, lse)
    want, wl, size, reach = attend(q.double(), *cache.rows(slots[0]), torch.ones(rows, prefix, dtype=torch.bool), D ** -0.5)
    o_ok, l_ok = bounds(want, wl, size, reach, kind, D, prefix)
    close(out, want, o_ok, "out")
    close(lse, wl, l_ok, "lse")


@pytest.mark.parametrize("cache_kind", [BF16, FP8])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_rising_scores_and_values_that_are_no_numbers(D, cache_kind):
    """The running maximum moves from tile to tile; a NaN lies in a tile that every row sees, another far behind in one that the
    causal edge cuts."""
    L, n, H = 1000, 90, 130
    announce("rising scores and NaN values over %d keys, %d heads of %d, %s" % (L, H, D, cache_kind))
    cache, table, slots, q, _ = prompt_case([n], [L], H, H, D, 16, BF16, cache_kind, behind=0, seed=D + 3)
    assert unsplit([n], [L], H, H, D, 16)
    k = torch.randn(L, H, D, generator=cache.gen) * 0.2 + torch.linspace(-2, 2, L)[:, None, None]
    v = torch.randn(L, H, D, generator=cache.gen)
    cache.fill(slots[0], k=k.to(BF16), v=v.to(BF16))
    kk, vv = cache.rows(slots[0])
    early, late = 500, L - 40
    odd = v.clone()
    odd[early, :, 3], odd[late, :, 5] = float("nan"), float("nan")
    cache.fill(slots[0], k=k.to(BF16), v=odd.to(BF16))
    if cache_kind == FP8:      # the row's scale does not know of a NaN, but may of what it replaced
        _, with_odd = cache.rows(slots[0])
        vv = torch.where(torch.isnan(with_odd), 0.0, with_odd)
    kd, vd, ks, vs = cache.to(DEV)
    q = q.abs().clamp(max=2.0) + 0.5
    out, lse = torch.zeros(q.shape, dtype=BF16, device=DEV), torch.zeros(q.shape[:2], device=DEV)
    scale = 16.0 / D
    ops.prompt_attention(q.to(DEV), kd, vd, table.to(DEV), torch.tensor([0, n], device=DEV), torch.tensor([L], device=DEV), out, scale, True, ks, vs, lse)
    want, wl, size, reach = attend(q.double(), kk, vv, visible_of(n, L, True), scale)
    want[:, :, 3] = float("nan")
    want[n - (L - late):, :, 5] = float("nan")
    o_ok, l_ok = bounds(want.nan_to_num(0.0), wl, size, reach, BF16, D, L)
    close(out, want, o_ok, "out")
    close(lse, wl, l_ok, "lse")
