"""Table entries outside the cache, wherever in a tile of keys they lie: their tokens are not seen. Tolerances:
cache_reference.bounds."""
import pytest
import torch

import heterofusedkernels_amd  # noqa: F401
import pcie_through  # noqa: F401
from cache_reference import FP8, attend, bounds
from gpu_helpers import announce
from test_gpu_attention import close, prompt_case, visible_of

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16
ops = torch.ops.pcie_through


def check(cache, table, slots, q, L, causal, scale, prompt_only=False):
    """Both ops over a table some of whose entries are outside the cache."""
    n, T, kind, D = q.shape[0], cache.T, cache.kind, cache.dim
    j = torch.arange(L)
    known = (table[0, j // T] >= 0) & (table[0, j // T] < cache.blocks)
    kk, vv = (torch.where(known[:, None, None], x, 0.0) for x in cache.rows(slots[0]))
    k, v, ks, vs = cache.to(DEV)
    q_d, table_d, len_d = q.to(DEV), table.to(DEV), torch.tensor([L], device=DEV)
    out, lse = torch.zeros(q.shape, dtype=kind, device=DEV), torch.zeros(q.shape[:2], device=DEV)
    ops.prompt_attention(q_d, k, v, table_d, torch.tensor([0, n], device=DEV), len_d, out, scale, causal, ks, vs, lse)
    want, wl, size, reach = attend(q.double(), kk, vv, visible_of(n, L, causal) & known[None], scale)
    o_ok, l_ok = bounds(want, wl, size, reach, kind, D, L)
    close(out, want, o_ok, "prompt")
    close(lse, wl, l_ok, "prompt lse")
    if prompt_only:
        return
    want, wl, size, reach = attend(q.double(), kk, vv, known[None].expand(n, L), scale)
    o_ok, l_ok = bounds(want, wl, size, reach, kind, D, L)
    none = torch.zeros(n, dtype=torch.int64, device=DEV)
    many = table_d.repeat(n, 1)
    for name, call in (("prefix", lambda: ops.prefix_attention(q_d, k, v, table_d[0], len_d, many[:, :0], none, out, scale, ks, vs, lse)),
                       ("own keys", lambda: ops.prefix_attention(q_d, k, v, table_d[0, :0], none[:1], many, len_d.repeat(n), out, scale, ks, vs, lse))):
        call()
        close(out, want, o_ok, name)
        close(lse, wl, l_ok, name + " lse")


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("missing", range(9))
def test_one_missing_block_at_each_place_of_a_tile(missing, D):
    announce("block %d of 9 is missing, heads of %d" % (missing, D))
    for cache_kind in (BF16, FP8):
        cache, table, slots, q, _ = prompt_case([20], [140], 8, 4, D, 16, BF16, cache_kind, behind=0, seed=missing)
        table[0, missing] = (-1, cache.blocks, 2 ** 40)[missing % 3]
        check(cache, table, slots, q, 140, True, D ** -0.5)


@pytest.mark.parametrize("kind,cache_kind", [(BF16, BF16), (FP16, FP16), (BF16, FP8), (FP16, FP8)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T,share", [(1, 0.3), (4, 0.5), (5, 0.1), (32, 0.4)])
def test_missing_blocks_at_random(T, share, D, kind, cache_kind):
    """Blocks of one token to 32, so that any set of a tile's keys is missing; many tiles, one part and several."""
    announce("blocks of %d, %.0f %% missing, heads of %d, %s %s" % (T, 100 * share, D, kind, cache_kind))
    for n, L, Hq, H in ((70, 333, 4, 2), (3, 1500, 2, 1), (90, 700, 130, 130)):
        if H == 130 and (D == 64 or T != 4):      # so many heads that the keys are not split
            continue
        cache, table, slots, q, _ = prompt_case([n], [L], Hq, H, D, T, kind, cache_kind, behind=0, seed=T, order="htd" if T == 4 else "thd")
        gone = torch.rand(table.shape, generator=cache.gen) < share
        table[gone] = torch.where(torch.rand(table.shape, generator=cache.gen) < 0.5, -1, cache.blocks)[gone]
        check(cache, table, slots, q, L, T != 5, D ** -0.5, prompt_only=H == 130)
