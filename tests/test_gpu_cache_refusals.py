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
