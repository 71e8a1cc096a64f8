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


LONG = [  # q lens, kv lens, Hq, H: more sequences than a wave has lanes, more splits than a wave takes at a time
    ([1 + i % 7 for i in range(150)], [3 + (i * 37) % 90 for i in range(150)], 4, 2),
    ([3], [20000], 2, 1),
    ([2, 1], [33, 9000], 3, 3),
]


@pytest.mark.parametrize("cache_kind", [BF16, FP8])
@pytest.mark.parametrize("case", LONG, ids=["150 sequences", "20000 keys", "splits of one sequence only"])
def test_prompt_attention_long(case, cache_kind):
    q_lens, kv_lens, Hq, H = case
    announce("prompt long %d sequences, most %d keys, %s" % (len(q_lens), max(kv_lens), cache_kind))
    cache, table, slots, q, starts = prompt_case(q_lens, kv_lens, Hq, H, 64, 16, BF16, cache_kind)
    check_prompt(cache, table, slots, q, starts, kv_lens, True, 0.125)


@pytest.mark.parametrize("kind,cache_kind", [(BF16, BF16), (FP16, FP8)])
@pytest.mark.parametrize("prefix,own,Hq,H", [(0, [(i * 131) % 400 for i in range(200)], 4, 4), (0, [20000], 2, 1), (9000, [1, 0], 3, 3),
                                             (0, [5, 7000, 0, 0, 3], 8, 4), (5000, [64] * 40, 8, 4)],
                         ids=["200 rows", "20000 keys", "9000 keys of prefix", "one long row", "wide prefix"])
def test_prefix_attention_long(prefix, own, Hq, H, kind, cache_kind):
    announce("prefix long %d + %d rows, most %d keys, %s %s" % (prefix, len(own), max(own), kind, cache_kind))
    T, D = 16, 64
    gen = torch.Generator().manual_seed(11)
    blocks = sum(-(-n // T) for n in own) + -(-prefix // T) + 2
    cache = Cache(blocks, T, H, D, kind, cache_kind, "thd", 5)
    table, slots = tables(gen, [prefix] + own, T, blocks)
    cache.fill(torch.cat(slots))
    width = max(-(-n // T) for n in own)
    check_prefix(cache, table[0, :-(-prefix // T)].contiguous(), slots[0], table[1:, :width].contiguous(), slots[1:], own,
                 torch.randn(len(own), Hq, D, generator=gen).to(kind), D ** -0.5)


@pytest.mark.parametrize("kind,cache_kind", [(BF16, BF16), (FP16, FP16), (FP16, FP8)])
def test_scores_that_rise_and_fall(kind, cache_kind):
    """Scores over a range of +-200 that rise from tile to tile, and that fall: the running maximum moves at every tile, and never."""
    announce("rising and falling scores %s %s" % (kind, cache_kind))
    n, D, H = 700, 64, 1
    for falling in (False, True):
        cache, table, slots, q, starts = prompt_case([n], [n], 2, H, D, 16, kind, cache_kind, seed=3)
        steps = torch.linspace(-25, 25, n)
        steps = steps.flip(0) if falling else steps
        k = (torch.randn(n, H, D, generator=cache.gen) * 0.1 + steps[:, None, None] / 4).to(kind)
        cache.fill(slots[0], k=k)
        q = q.abs().clamp(max=2.0) + 0.5
        check_prompt(cache, table, slots, q, starts, [n], True, 0.5)
        check_prefix(cache, table[0, :20].contiguous(), slots[0][:320], table[:, 20:].contiguous(), [slots[0][320:]], [n - 320], q[:1], 0.5)


@pytest.mark.parametrize("cache_kind", [BF16, FP8])
def test_values_that_are_no_numbers(cache_kind):
    """NaN and infinities in tokens that only the later queries see: the earlier ones' results do not know of them, the later
    ones' columns become what the sums say. Direct results and split ones."""
    announce("NaN and infinities in the future, %s" % cache_kind)
    for q_lens, L, Hq, H in (([200], 200, 4, 2), ([50], 900, 1, 1)):
        n, D, T = q_lens[0], 64, 16
        cache, table, slots, q, starts = prompt_case(q_lens, [L], Hq, H, D, T, BF16, cache_kind, order="htd")
        v = torch.randn(L, H, D, generator=cache.gen).to(BF16)
        k = torch.randn(L, H, D, generator=cache.gen).to(BF16)
        special = BF16 if cache_kind == BF16 else None
        v[L - 30, 0, 3] = float("nan")
        if special:      # e4m3 has no infinities
            v[L - 20, H - 1, 7] = float("inf")
            v[L - 10, H - 1, 7] = float("-inf")
        k[L - 5, 0, 1] = float("nan")
        cache.fill(slots[0], k=k, v=v)
        kd, vd, ks, vs = cache.to(DEV)
        out = torch.zeros(q.shape, dtype=BF16, device=DEV)
        lse = torch.zeros(q.shape[:2], device=DEV)
        ops.prompt_attention(q.to(DEV), kd, vd, table.to(DEV), starts.to(DEV), torch.tensor([L], device=DEV), out, 0.125, True, ks, vs, lse)
        got, lse = out.cpu().double()[:n], lse.cpu()[:n]
        first = lambda token: n - (L - token)      # the first query that sees this token
        for h in range(Hq):
            of0, last = h * H // Hq == 0, h * H // Hq == H - 1
            want = torch.zeros(n, D)               # 0: finite
            if of0:
                want[first(L - 30):, 3] = float("nan")
                want[first(L - 5):] = float("nan")
            if special and last:
                want[first(L - 20):, 7] = torch.where(torch.isnan(want[first(L - 20):, 7]), want[first(L - 20):, 7], torch.tensor(float("inf")))
                want[first(L - 10):, 7] = float("nan")
            assert torch.equal(torch.isnan(got[:, h]), torch.isnan(want)), h
            assert torch.equal(got[:, h] == float("inf"), want == float("inf")), h
            assert torch.equal(torch.isnan(lse[:, h]), torch.arange(n) >= (first(L - 5) if of0 else n)), h
        # what saw nothing of it is right, too
        clean = first(L - 30)
        kk, vv = cache.rows(slots[0][:L - n + clean])
        want, wl, size, reach = attend(q[:clean].double(), kk, vv, visible_of(clean, L - n + clean, True), 0.125)
        o_ok, l_ok = bounds(want, wl, size, reach, BF16, D, L)
        close(out[:clean], want, o_ok, "queries before the first")


def test_a_row_whose_only_key_is_nan():
    announce("one key, NaN")
    for value, D in ((float("nan"), 64),):
        k = torch.full((1, 16, 1, D), value, dtype=BF16, device=DEV)
        v = torch.ones(1, 16, 1, D, dtype=BF16, device=DEV)
        q = torch.ones(1, 1, D, dtype=BF16, device=DEV)
        zero, one = torch.zeros(1, 1, dtype=torch.int64, device=DEV), torch.ones(1, dtype=torch.int64, device=DEV)
        for call in (lambda o, l: ops.prompt_attention(q, k, v, zero, torch.tensor([0, 1], device=DEV), one, o, 1.0, True, None, None, l),
                     lambda o, l: ops.prefix_attention(q, k, v, zero[0, :0], zero[0], zero, one, o, 1.0, None, None, l),
                     lambda o, l: ops.prefix_attention(q, k, v, zero[0], one, zero[:, :0], zero[0], o, 1.0, None, None, l)):
            out, lse = torch.zeros(1, 1, D, dtype=BF16, device=DEV), torch.zeros(1, 1, device=DEV)
            call(out, lse)
            assert bool(torch.isnan(out).all()) and bool(torch.isnan(lse).all())


@pytest.mark.parametrize("cache_kind", [BF16, FP8])
def test_blocks_outside_the_cache_are_not_seen(cache_kind):
    """A table entry outside the cache hides its block's tokens; lengths outside the table are cut; both in both ops."""
    announce("bad block ids, %s" % cache_kind)
    T, H, Hq, D = 16, 2, 8, 128
    for n, L in ((40, 200), (3, 1400)):
        cache, table, slots, q, starts = prompt_case([n], [L], Hq, H, D, T, BF16, cache_kind)
        table[0, 1], table[0, 4] = -1, cache.blocks
        if L > 1000:
            table[0, 40:60] = 2 ** 40
        j = torch.arange(L)
        known = (table[0, j // T] >= 0) & (table[0, j // T] < cache.blocks)
        kk, vv = cache.rows(slots[0])
        kk, vv = torch.where(known[:, None, None], kk, 0.0), torch.where(known[:, None, None], vv, 0.0)
        kd, vd, ks, vs = cache.to(DEV)
        out, lse = torch.zeros(q.shape, dtype=BF16, device=DEV), torch.zeros(q.shape[:2], device=DEV)
        ops.prompt_attention(q.to(DEV), kd, vd, table.to(DEV), starts.to(DEV), torch.tensor([L], device=DEV), out, 0.1, True, ks, vs, lse)
        want, wl, size, reach = attend(q[:n].double(), kk, vv, visible_of(n, L, True) & known[None], 0.1)
        o_ok, l_ok = bounds(want, wl, size, reach, BF16, D, L)
        close(out[:n], want, o_ok, "prompt")
        close(lse[:n], wl, l_ok, "prompt lse")
        cut = table.shape[1] - 3
        ops.prefix_attention(q[:1].to(DEV), kd, vd, table[0, :3].contiguous().to(DEV), torch.tensor([3 * T + 99], device=DEV),
                             table[:, 3:3 + cut].contiguous().to(DEV), torch.tensor([L - 3 * T], device=DEV), out[:1], 0.1, ks, vs, lse[:1])
        want, wl, size, reach = attend(q[:1].double(), kk, vv, known[None], 0.1)
        o_ok, l_ok = bounds(want, wl, size, reach, BF16, D, L)
        close(out[:1], want, o_ok, "prefix")
        close(lse[:1], wl, l_ok, "prefix lse")
    # nothing at all: negative lengths, a table of no width, a cache of no blocks
    none = torch.zeros(0, T, H, D, dtype=BF16, device=DEV)
    for kv, tab, cache_k in ((-5, table, kd.to(BF16)), (7, table[:, :0], kd.to(BF16)), (7, table, none)):
        for call in (lambda o, l: ops.prompt_attention(q[:4].to(DEV), cache_k, cache_k, tab.contiguous().to(DEV), torch.tensor([0, 4], device=DEV),
                                                       torch.tensor([kv], device=DEV), o, 1.0, True, None, None, l),
                     lambda o, l: ops.prefix_attention(q[:4].to(DEV), cache_k, cache_k, tab[0].contiguous().to(DEV), torch.tensor([kv], device=DEV),
                                                       tab.repeat(4, 1).contiguous().to(DEV), torch.tensor([kv] * 4, device=DEV), o, 1.0, None, None, l)):
            o, l = torch.ones(4, Hq, D, dtype=BF16, device=DEV), torch.ones(4, Hq, device=DEV)
            call(o, l)
            assert bool((o == 0).all()) and bool((l == float("-inf")).all())


def test_sequences_out_of_order_are_skipped():
    announce("query starts out of order")
    cache, table, slots, q, starts = prompt_case([4, 4, 4], [9, 9, 9], 2, 1, 64, 16, BF16, BF16, behind=0)
    k, v, _, _ = cache.to(DEV)
    bad = torch.tensor([0, 4, 2, 100], device=DEV)      # the second runs backwards, the third ends behind the last row
    out = torch.full(q.shape, 5.0, dtype=BF16, device=DEV)
    ops.prompt_attention(q.to(DEV), k, v, table.to(DEV), bad, torch.tensor([9, 9, 9], device=DEV), out, 0.125)
    torch.cuda.synchronize()
    kk, vv = cache.rows(slots[0])
    want, wl, size, reach = attend(q[:4].double(), kk, vv, visible_of(4, 9, True), 0.125)
    close(out[:4], want, bounds(want, wl, size, reach, BF16, 64, 9)[0], "the sound sequence")
    assert bool((out[4:] == 5.0).all())


def test_strided_queries_and_results():
    """q as a part of a fused projection, out as a part of a wider buffer; what lies between is left alone."""
    announce("strided q and out")
    cache, table, slots, q, starts = prompt_case([50, 20], [50, 300], 6, 2, 64, 16, FP16, FP16, behind=0)
    fused = torch.zeros(70, 10, 72, dtype=FP16, device=DEV)
    fused[:, 1:7, 8:] = q.to(DEV)
    wide = torch.full((70, 9, 128), 5.0, dtype=FP16, device=DEV)
    check_prompt(cache, table, slots, q, starts, [50, 300], True, 0.125, q_d=fused[:, 1:7, 8:], out=wide[:, 2:8, 32:96])
    assert bool((wide[:, :2] == 5.0).all() and (wide[:, 8:] == 5.0).all() and (wide[:, :, :32] == 5.0).all() and (wide[:, :, 96:] == 5.0).all())


@pytest.mark.parametrize("cache_kind", [BF16, FP8])
def test_a_cache_of_more_than_4_gib(cache_kind):
    announce("cache beyond 4 GiB, %s" % cache_kind)
    T, H, D = 16, 8, 128
    size = 1 if cache_kind == FP8 else 2
    blocks = (5 << 30) // (T * H * D * size)
    k = torch.empty(blocks, T, H, D * size, dtype=torch.uint8, device=DEV).view(cache_kind)
    v = torch.empty(blocks, T, H, D * size, dtype=torch.uint8, device=DEV).view(cache_kind)
    ks, vs = (torch.ones(blocks, T, H, device=DEV) if cache_kind == FP8 else None for _ in "kv")
    gen = torch.Generator().manual_seed(1)
    n = 90
    table = torch.tensor([[blocks - 1, 7, blocks - 2, (4 << 30) // (T * H * D * size), blocks - 9, blocks // 2]])
    j = torch.arange(n)
    slots = table[0, j // T] * T + j % T
    small = Cache(6, T, H, D, BF16, cache_kind)
    own = torch.arange(6)[j // T] * T + j % T
    x = [torch.randn(n, H, D, generator=gen).to(BF16) for _ in "kv"]
    small.fill(own, k=x[0], v=x[1])
    ops.cache_write(x[0].to(DEV), k, slots.to(DEV), x[1].to(DEV), v, ks, vs)
    back = [torch.zeros(n, H, D, dtype=BF16, device=DEV) for _ in "kv"]
    ops.cache_read(k, back[0], slots.to(DEV), v, back[1], ks, vs)
    kk, vv = small.rows(own)
    assert torch.equal(back[0].cpu().double(), kk) and torch.equal(back[1].cpu().double(), vv)
    q = torch.randn(n, 16, D, generator=gen).to(BF16)
    out = torch.zeros(q.shape, dtype=BF16, device=DEV)
    ops.prompt_attention(q.to(DEV), k, v, table.to(DEV), torch.tensor([0, n], device=DEV), torch.tensor([n], device=DEV), out, 0.1, True, ks, vs)
    want, wl, s, reach = attend(q.double(), kk, vv, visible_of(n, n, True), 0.1)
    close(out, want, bounds(want, wl, s, reach, BF16, D, n)[0], "prompt")
    ops.prefix_attention(q[:1].to(DEV), k, v, table[0, :2].contiguous().to(DEV), torch.tensor([32], device=DEV), table[:, 2:].contiguous().to(DEV),
                         torch.tensor([n - 32], device=DEV), out[:1], 0.1, ks, vs)
    want, wl, s, reach = attend(q[:1].double(), kk, vv, torch.ones(1, n, dtype=torch.bool), 0.1)
    close(out[:1], want, bounds(want, wl, s, reach, BF16, D, n)[0], "prefix")
    if cache_kind == BF16:      # one block longer than 32-bit offsets reach
        with pytest.raises(RuntimeError, match="exceeds"):
            ops.prompt_attention(q.to(DEV), k.view(1, blocks * T, H, D), v.view(1, blocks * T, H, D), table[:, :1].to(DEV),
                                 torch.tensor([0, n], device=DEV), torch.tensor([n], device=DEV), out, 0.1)


@pytest.mark.parametrize("rows", [1, 3, 20])
def test_infinite_values_that_are_seen(rows):
    """An infinity in V gives infinity in its column, whatever the weight's rounding, in every kernel a row can go through."""
    announce("infinite values, %d rows" % rows)
    T, D, n = 16, 64, 40
    gen = torch.Generator().manual_seed(rows)
    k, v = (torch.randn(4, T, 1, D, generator=gen).to(BF16) for _ in "kv")
    v[0, 0, 0, 5], v[1, 3, 0, 9], v[2, 1, 0, 9] = float("inf"), float("-inf"), float("inf")
    k, v = k.to(DEV), v.to(DEV)
    table = torch.arange(4)[None].to(DEV)
    q = torch.randn(rows, 4, D, generator=gen).to(BF16).to(DEV)
    want = torch.zeros(D)
    want[5], want[9] = float("inf"), float("nan")
    lens = torch.full((rows,), n, device=DEV)
    none = torch.zeros(rows, dtype=torch.int64, device=DEV)
    out = [torch.zeros_like(q) for _ in range(4)]
    ops.prompt_attention(q, k, v, table, torch.tensor([0, rows], device=DEV), lens[:1], out[0], 0.125, False)
    ops.prefix_attention(q, k, v, table[0, :0], none[:1], table.repeat(rows, 1), lens, out[1], 0.125)
    ops.prefix_attention(q, k, v, table[0], lens[:1], table[:, :0].repeat(rows, 1), none, out[2], 0.125)
    many = table.repeat(1, 40)      # the same blocks again and again: many tiles, splits
    ops.prompt_attention(q, k, v, many, torch.tensor([0, rows], device=DEV), torch.tensor([160 * T], device=DEV), out[3], 0.125, False)
    for i, o in enumerate(out):
        o = o.cpu().float()
        assert bool((torch.isnan(o) == torch.isnan(want)).all()), i
        assert bool(((o == float("inf")) == (want == float("inf"))).all()) and not bool((o == float("-inf")).any()), i


@pytest.mark.parametrize("rows,keys", [(3, 300), (1, 2900)])
@pytest.mark.parametrize("causal", [True, False])
def test_values_that_are_no_numbers_around_a_missing_block(rows, keys, causal):
    """Keys beside a block that is not there, keys of whole tiles and keys of the last, ragged one: each counts wherever it lies."""
    announce("no numbers around a missing block, %d rows, %d keys, causal %s" % (rows, keys, causal))
    T, D = 16, 64
    n = -(-keys // T)
    gen = torch.Generator().manual_seed(keys)
    k, v = (torch.randn(n, T, 1, D, generator=gen).to(BF16) for _ in "kv")
    inf, nan = float("inf"), float("nan")
    odd = v.clone()
    for token, column, value in ((5, 4, inf), (5, 3, inf), (130, 3, nan), (130, 7, inf), (keys - rows, 6, -inf), (keys - rows, 8, inf), (50, 8, -inf)):
        odd[token // T, token % T, 0, column] = value
    want = {3: nan, 4: inf, 6: -inf, 7: inf, 8: nan}
    table = torch.arange(n)[None].clone()
    table[0, 2] = -1
    table = table.to(DEV)
    q = torch.randn(rows, 2, D, generator=gen).to(BF16).to(DEV)
    clean, out = torch.zeros_like(q), torch.zeros_like(q)
    for values, to in ((v, clean), (odd, out)):
        ops.prompt_attention(q, k.to(DEV), values.to(DEV), table, torch.tensor([0, rows], device=DEV), torch.tensor([keys], device=DEV), to, 0.125, causal)
    clean, out = clean.cpu(), out.cpu().float()
    for column in range(D):
        got = out[:, :, column]
        if column not in want:
            assert torch.equal(got, clean[:, :, column].float()), column
        else:
            assert torch.equal(got, torch.full_like(got, want[column])) or bool(torch.isnan(got).all()) and want[column] != want[column], (column, got)
