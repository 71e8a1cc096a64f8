"""Keys that are cut into parts and joined give what they give in one part: what is no number counts in whichever part it lies,
however small that part's weights are beside another's."""
import pytest
import torch

import heterofusedkernels_amd  # noqa: F401
import pcie_through  # noqa: F401
from gpu_helpers import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16
ops = torch.ops.pcie_through


def answers(q, k, v, keys, scale):
    """(name, out, lse) of each way to attend `q` [rows, heads, D] over the first `keys` tokens of a cache."""
    T, rows = k.shape[1], q.shape[0]
    table = torch.arange(k.shape[0], device=DEV)[None]
    many = table.repeat(rows, 1)
    starts, lens = torch.tensor([0, rows], device=DEV), torch.full((rows,), keys, device=DEV)
    half = keys // 2 // T
    rest = torch.full((rows,), keys - half * T, device=DEV)
    none = torch.zeros(rows, dtype=torch.int64, device=DEV)
    calls = {
        "prompt": lambda o, l: ops.prompt_attention(q, k, v, table, starts, lens[:1], o, scale, False, None, None, l),
        "own keys": lambda o, l: ops.prefix_attention(q, k, v, table[0, :0], none[:1], many, lens, o, scale, None, None, l),
        "prefix": lambda o, l: ops.prefix_attention(q, k, v, table[0], lens[:1], many[:, :0], none, o, scale, None, None, l),
        "both": lambda o, l: ops.prefix_attention(q, k, v, table[0, :half], torch.tensor([half * T], device=DEV), many[:, half:].contiguous(), rest, o, scale,
                                                  None, None, l),
    }
    for name, call in calls.items():
        out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], device=DEV)
        call(out, lse)
        yield name, out.cpu().float(), lse.cpu()


def filled(keys, D, seed):
    gen = torch.Generator().manual_seed(seed)
    blocks = -(-keys // 16)
    k, v = (torch.randn(blocks, 16, 1, D, generator=gen) for _ in "kv")
    return gen, k, v


@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("all_of_the_part", [False, True], ids=["one key", "all keys around"])
@pytest.mark.parametrize("keys", [50, 2900, 20000])
def test_nan_scores_in_a_part_of_small_weights(keys, all_of_the_part, rows):
    """One key (or some thousand around it) is NaN, another one's scores pass all the others' by 400: NaN, as in one part."""
    announce("NaN keys beside large scores, %d keys, %d rows, %s" % (keys, rows, "many" if all_of_the_part else "one"))
    D = 64
    gen, k, v = filled(keys, D, keys)
    q = torch.ones(rows, 2, D) + torch.rand(rows, 2, D, generator=gen)
    at, large = keys // 5, keys * 4 // 5
    k.view(-1, D)[large] = 40.0
    if all_of_the_part:
        k.view(-1, D)[at - keys // 8:at + keys // 8] = float("nan")
    else:
        k.view(-1, D)[at, 3] = float("nan")
    for name, out, lse in answers(q.to(BF16).to(DEV), k.to(BF16).to(DEV), v.to(BF16).to(DEV), keys, 0.125):
        assert bool(torch.isnan(out).all()) and bool(torch.isnan(lse).all()), name


@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_values_that_are_no_numbers_in_a_part_of_small_weights(value, rows):
    """Their column is no number (the weight is none but in 32 bits); the other columns and lse know nothing of them."""
    announce("values %s beside large scores, %d rows" % (value, rows))
    D, keys = 64, 2900
    gen, k, v = filled(keys, D, 7)
    q = torch.ones(rows, 2, D) + torch.rand(rows, 2, D, generator=gen)
    k.view(-1, D)[keys * 4 // 5] = 40.0
    odd = v.clone()
    odd.view(-1, D)[keys // 5, 9] = value
    q, k = q.to(BF16).to(DEV), k.to(BF16).to(DEV)
    for (name, out, lse), (_, clean, clean_lse) in zip(answers(q, k, odd.to(BF16).to(DEV), keys, 0.125), answers(q, k, v.to(BF16).to(DEV), keys, 0.125)):
        assert not bool(torch.isfinite(out[:, :, 9]).any()), name
        assert torch.equal(lse, clean_lse), name
        out[:, :, 9] = clean[:, :, 9]
        assert torch.equal(out, clean), name
