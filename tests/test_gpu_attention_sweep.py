"""Attention calls drawn at random over what the header allows: lengths, heads, head sizes, blocks, layouts and types; tables wider
than needed with anything in the entries behind a sequence's last block; entries outside the cache; lengths and query starts outside
their range. Every token no sequence owns is NaN, its scale too. Tolerances: cache_reference.bounds."""
import math
import random

import pytest
import torch

import heterofusedkernels_amd  # noqa: F401
import pcie_through  # noqa: F401
from cache_reference import FP8, Cache, attend, bounds
from gpu_helpers import announce
from test_gpu_attention import close, visible_of

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16
ops = torch.ops.pcie_through


def log_uniform(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


class Drawn:
    """A cache, the tables of `lens` sequences (an entry in eight outside the cache at times), and their slots and visibility."""

    def __init__(self, rng, lens, T, H, D, kind, cache_kind, order):
        self.gen = torch.Generator().manual_seed(rng.randrange(1 << 30))
        need = [-(-n // T) for n in lens]
        blocks = 1 + sum(need) + rng.randrange(3)
        self.cache = Cache(blocks, T, H, D, kind, cache_kind, order, rng.randrange(1 << 30))
        ids = torch.randperm(blocks - 1, generator=self.gen) + 1      # the first block is nobody's
        width = max(need) + rng.choice([0, 0, 1, 5]) if lens else 1
        # behind a sequence's last block: anything
        self.table = torch.randint(-(1 << 62), 1 << 62, (len(lens), width), generator=self.gen)
        self.table[torch.rand(self.table.shape, generator=self.gen) < 0.5] = 0
        self.known, self.slots, at = [], [], 0
        missing = rng.choice([0.0, 0.0, 0.12])
        for b, n in enumerate(lens):
            self.table[b, :need[b]] = ids[at:at + need[b]]
            at += need[b]
            j = torch.arange(n)
            self.slots.append(self.table[b, j // T] * T + j % T)
            gone = torch.rand(need[b], generator=self.gen) < missing
            self.table[b, :need[b]][gone] = rng.choice([-1, blocks, 1 << 40])
            self.known.append(~gone[j // T])
        owned = torch.cat([s[k] for s, k in zip(self.slots, self.known)] + [torch.zeros(0, dtype=torch.int64)])
        if len(owned):
            self.cache.fill(owned)
        if cache_kind == FP8:
            rest = torch.ones(blocks * T, dtype=torch.bool)
            rest[owned] = False
            for scales in (self.cache.ks, self.cache.vs):
                scales[rest.view(blocks, T)] = rng.choice([float("nan"), float("inf")])

    def rows(self, b):
        """(k, v) of a sequence in 64 bits, zeros where a token is not known."""
        return [torch.where(self.known[b][:, None, None], x, 0.0) for x in self.cache.rows(torch.where(self.known[b], self.slots[b], 0))]


def shape(rng):
    H = rng.choice([1, 2, 3, 4, 5, 8, 16])
    G = rng.choice([1, 1, 2, 3, 4, 7, 8, 16, 33]) if H < 5 else rng.choice([1, 2, 4, 5])
    D = rng.choice([16, 32, 48, 64, 64, 80, 96, 128, 128, 128, 160, 192, 256])
    kind = rng.choice([BF16, FP16])
    return H, G, D, rng.choice([1, 2, 3, 5, 8, 16, 16, 16, 32, 64, 100]), kind, rng.choice([kind, FP8]), rng.choice(["thd", "htd"])


@pytest.mark.parametrize("seed", range(60))
def test_drawn_prompts(seed):
    rng = random.Random(seed)
    H, G, D, T, kind, cache_kind, order = shape(rng)
    n_seqs = log_uniform(rng, 1, 20)
    q_lens = [rng.choice([0, 1, 1, 2]) if rng.random() < 0.3 else log_uniform(rng, 1, 260) for _ in range(n_seqs)]
    kv_lens = [max(0, n + rng.choice([0, 0, -3, 1])) if rng.random() < 0.4 else n + log_uniform(rng, 1, 1500 // n_seqs + 2) for n in q_lens]
    causal, given = rng.random() < 0.75, list(kv_lens)
    announce("seed %d: prompts %s of %s, %d x %d heads of %d, T %d, %s %s %s, causal %s" % (seed, q_lens, kv_lens, H, G, D, T, kind, cache_kind, order, causal))
    x = Drawn(rng, kv_lens, T, H, D, kind, cache_kind, order)
    first, behind = rng.choice([0, 0, 3]), rng.choice([0, 2])
    total = first + sum(q_lens) + behind
    q = torch.randn(total, H * G, D, generator=x.gen).to(kind)
    starts = [first]
    for n in q_lens:
        starts.append(starts[-1] + n)
    for b, n in enumerate(kv_lens):      # a length beyond its table is cut to it; one below zero is none
        if n == x.table.shape[1] * T and rng.random() < 0.5:
            given[b] = n + rng.choice([1, 1 << 40])
        elif n == 0 and rng.random() < 0.5:
            given[b] = -rng.choice([1, 1 << 40])
    k, v, ks, vs = x.cache.to(DEV)
    out = torch.full(q.shape, 5.0, dtype=kind, device=DEV)
    lse = torch.full(q.shape[:2], 5.0, device=DEV)
    scale = D ** -0.5 * rng.choice([0.1, 1.0, 1.0, 4.0])
    ops.prompt_attention(q.to(DEV), k, v, x.table.to(DEV), torch.tensor(starts, device=DEV), torch.tensor(given, device=DEV), out, scale, causal, ks, vs, lse)
    torch.cuda.synchronize()
    for b, L in enumerate(kv_lens):
        i, end = starts[b], starts[b + 1]
        seen = visible_of(end - i, L, causal) & x.known[b][None]
        want, wl, size, reach = attend(q[i:end].double(), *x.rows(b), seen, scale)
        o_ok, l_ok = bounds(want, wl, size, reach, kind, D, L)
        close(out[i:end], want, o_ok, "out of sequence %d" % b)
        close(lse[i:end], wl, l_ok, "lse of sequence %d" % b)
    for rest in (slice(0, first), slice(starts[-1], total)):
        assert bool((out[rest] == 5.0).all()) and bool((lse[rest] == 5.0).all()), "rows of no sequence"


@pytest.mark.parametrize("seed", range(60))
def test_drawn_prefixes(seed):
    rng = random.Random(1000 + seed)
    H, G, D, T, kind, cache_kind, order = shape(rng)
    rows = log_uniform(rng, 1, 40)
    prefix = 0 if rng.random() < 0.25 else log_uniform(rng, 1, 1500)
    own = [0 if rng.random() < 0.15 else log_uniform(rng, 1, 3000 // rows + 40) for _ in range(rows)]
    announce("seed %d: prefix %d, own %s, %d x %d heads of %d, T %d, %s %s %s" % (seed, prefix, own, H, G, D, T, kind, cache_kind, order))
    x = Drawn(rng, [prefix] + own, T, H, D, kind, cache_kind, order)
    q = torch.randn(rows, H * G, D, generator=x.gen).to(kind)
    k, v, ks, vs = x.cache.to(DEV)
    out = torch.full(q.shape, 5.0, dtype=kind, device=DEV)
    lse = torch.full(q.shape[:2], 5.0, device=DEV)
    scale = D ** -0.5 * rng.choice([0.1, 1.0, 1.0, 4.0])
    blocks = x.table[0, :-(-prefix // T) + rng.choice([0, 0, 2])].contiguous()
    width = max(-(-n // T) for n in own) + rng.choice([0, 0, 2])
    ops.prefix_attention(q.to(DEV), k, v, blocks.to(DEV), torch.tensor([prefix], device=DEV), x.table[1:, :width].contiguous().to(DEV),
                         torch.tensor(own, device=DEV), out, scale, ks, vs, lse)
    torch.cuda.synchronize()
    shared = x.rows(0)
    for b, n in enumerate(own):
        kk, vv = (torch.cat([s, o]) for s, o in zip(shared, x.rows(1 + b)))
        seen = torch.cat([x.known[0], x.known[1 + b]])[None]
        want, wl, size, reach = attend(q[b:b + 1].double(), kk, vv, seen, scale)
        o_ok, l_ok = bounds(want, wl, size, reach, kind, D, prefix + n)
        close(out[b:b + 1], want, o_ok, "out of row %d" % b)
        close(lse[b:b + 1], wl, l_ok, "lse of row %d" % b)
