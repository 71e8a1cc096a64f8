"""The cache and attention ops as a serving loop uses them: together, with the block swap, on streams, in graphs, and their
refusals. Figures are compared with the plain 64-bit statements or, where two ways must agree, bit by bit."""
import pytest
import torch

import heterofusedkernels_amd  # noqa: F401
import pcie_through
from cache_reference import FP8, attend, bounds, dequantise, quantise
from gpu_helpers import announce
from heterofusedkernels import memory

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16
ops = torch.ops.pcie_through


def off(got, want, allowed):
    return float(((got.double().cpu() - want).abs() - allowed).max())


def test_a_prefix_is_written_swapped_out_and_in_and_answered_from():
    """A prompt's keys and values enter e4m3 blocks that carry their scales; the blocks go to pinned host memory and come back
    elsewhere; sequences answer under them as a shared prefix, and a second prompt continues behind them."""
    announce("write, swap out, swap in, read, attend")
    T, H, D, Hq, blocks, n = 16, 4, 64, 16, 64, 150
    gen = torch.Generator().manual_seed(2)
    size = pcie_through.fp8_block_bytes(T, H, D)
    planes = [torch.zeros(blocks, size, dtype=torch.uint8, device=DEV) for _ in "kv"]
    (k, ks), (v, vs) = (pcie_through.fp8_cache_views(p, T, H, D) for p in planes)
    need = -(-n // T)
    at = torch.randperm(blocks, generator=gen)[:need]
    j = torch.arange(n)
    x = [torch.randn(n, H, D, generator=gen).to(BF16) for _ in "kv"]
    ops.cache_write(x[0].to(DEV), k, (at[j // T] * T + j % T).to(DEV), x[1].to(DEV), v, ks, vs)
    seen = [dequantise(*quantise(y), BF16).double() for y in x]

    host = memory.alloc_numa_pinned_tensor(2 * blocks * size).view(torch.uint8).view(2, blocks, size)
    dev_tab, host_tab = pcie_through.plane_pointer_table(planes, DEV), pcie_through.plane_pointer_table(list(host.unbind(0)), DEV)
    slots_host = torch.randperm(blocks, generator=gen)[:need]
    pcie_through.swap_blocks(host_tab, dev_tab, torch.stack([at, slots_host], 1).to(DEV), size, size, size, blocks, blocks)
    for p in planes:
        p.zero_()
    back = torch.randperm(blocks, generator=gen)[:need]
    pcie_through.swap_blocks(dev_tab, host_tab, torch.stack([slots_host, back], 1).to(DEV), size, size, size, blocks, blocks)

    out = [torch.zeros(n, H, D, dtype=BF16, device=DEV) for _ in "kv"]
    ops.cache_read(k, out[0], (back[j // T] * T + j % T).to(DEV), v, out[1], ks, vs)
    assert torch.equal(out[0].cpu().double(), seen[0]) and torch.equal(out[1].cpu().double(), seen[1])

    # three sequences under the prefix (its last block partly theirs to share), each with tokens of its own
    free = torch.tensor([b for b in range(blocks) if b not in back.tolist()])
    own = [20, 0, 5]
    table = free[:6].view(3, 2).contiguous()
    new = [torch.randn(sum(own), H, D, generator=gen).to(BF16) for _ in "kv"]
    where = torch.cat([table[b, torch.arange(m) // T] * T + torch.arange(m) % T for b, m in enumerate(own)])
    ops.cache_write(new[0].to(DEV), k, where.to(DEV), new[1].to(DEV), v, ks, vs)
    new = [dequantise(*quantise(y), BF16).double() for y in new]
    q = torch.randn(3, Hq, D, generator=gen).to(BF16)
    got = torch.zeros(3, Hq, D, dtype=BF16, device=DEV)
    ops.prefix_attention(q.to(DEV), k, v, back.to(DEV), torch.tensor([n], device=DEV), table.to(DEV), torch.tensor(own, device=DEV), got,
                         0.125, ks, vs)
    first = 0
    for b, m in enumerate(own):
        kk, vv = (torch.cat([seen[i], new[i][first:first + m]]) for i in (0, 1))
        first += m
        want, wl, s, reach = attend(q[b:b + 1].double(), kk, vv, torch.ones(1, n + m, dtype=torch.bool), 0.125)
        assert off(got[b:b + 1], want, bounds(want, wl, s, reach, BF16, D, n + m)[0]) <= 0

    # a second prompt of 30 tokens behind the prefix: the table goes on where the prefix's blocks end
    m = 30
    cont = torch.cat([back, free[6:8]])[None]
    p = n + torch.arange(m)
    more = [torch.randn(m, H, D, generator=gen).to(BF16) for _ in "kv"]
    ops.cache_write(more[0].to(DEV), k, (cont[0, p // T] * T + p % T).to(DEV), more[1].to(DEV), v, ks, vs)
    more = [dequantise(*quantise(y), BF16).double() for y in more]
    q = torch.randn(m, Hq, D, generator=gen).to(BF16)
    got = torch.zeros(m, Hq, D, dtype=BF16, device=DEV)
    ops.prompt_attention(q.to(DEV), k, v, cont.to(DEV), torch.tensor([0, m], device=DEV), torch.tensor([n + m], device=DEV), got, 0.125, True, ks, vs)
    kk, vv = (torch.cat([seen[i], more[i]]) for i in (0, 1))
    visible = torch.arange(n + m)[None] <= n + torch.arange(m)[:, None]
    want, wl, s, reach = attend(q.double(), kk, vv, visible, 0.125)
    assert off(got, want, bounds(want, wl, s, reach, BF16, D, n + m)[0]) <= 0


class Step:
    """One step of a loop with fixed buffers: tokens written, read back, a prompt chunk and a decoding step answered. The shapes
    take workspaces in both attention ops."""

    def __init__(self, seed):
        self.gen = torch.Generator(device=DEV).manual_seed(seed)
        self.T, self.H, self.D, self.blocks, self.n, self.B = 16, 2, 64, 160, 1000, 6
        self.k, self.v = (torch.zeros(self.blocks, 16, 2, 64, dtype=FP8, device=DEV) for _ in "kv")
        self.ks, self.vs = (torch.ones(self.blocks, 16, 2, device=DEV) for _ in "kv")
        self.x = [torch.zeros(self.n, 2, 64, dtype=BF16, device=DEV) for _ in "kv"]
        self.table = torch.randperm(self.blocks, generator=self.gen, device=DEV)[None].contiguous()
        j = torch.arange(self.n, device=DEV)
        self.slots = self.table[0, j // 16] * 16 + j % 16
        self.q, self.one = torch.zeros(20, 8, 64, dtype=BF16, device=DEV), torch.zeros(self.B, 8, 64, dtype=BF16, device=DEV)
        self.starts, self.len = torch.tensor([0, 20], device=DEV), torch.tensor([self.n], device=DEV)
        self.prefix_len = torch.tensor([640], device=DEV)
        self.own = self.table[:, 40:].repeat(self.B, 1).contiguous()
        self.own_lens = torch.tensor([0, 1, 300, 17, 360, 5], device=DEV)
        self.results = [torch.zeros_like(self.x[0]), torch.zeros_like(self.x[0]), torch.zeros_like(self.q), torch.zeros(20, 8, device=DEV),
                        torch.zeros_like(self.one), torch.zeros(self.B, 8, device=DEV)]

    def refill(self):
        for t in self.x + [self.q, self.one]:
            t.normal_(generator=self.gen)
        self.own_lens.copy_(torch.randint(0, 361, (self.B,), generator=self.gen, device=DEV))
        self.prefix_len.copy_(torch.randint(1, 641, (1,), generator=self.gen, device=DEV))

    def run(self):
        r = self.results
        ops.cache_write(self.x[0], self.k, self.slots, self.x[1], self.v, self.ks, self.vs)
        ops.cache_read(self.k, r[0], self.slots, self.v, r[1], self.ks, self.vs)
        ops.prompt_attention(self.q, self.k, self.v, self.table, self.starts, self.len, r[2], 0.125, True, self.ks, self.vs, r[3])
        ops.prefix_attention(self.one, self.k, self.v, self.table[0, :40], self.prefix_len, self.own, self.own_lens, r[4], 0.125,
                             self.ks, self.vs, r[5])

    def copies(self):
        return [t.clone() for t in self.results + [self.k.view(torch.uint8), self.v.view(torch.uint8), self.ks, self.vs]]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_the_step_replays_in_a_hip_graph():
    announce("HIP graph of the step, replayed with eager work in between")
    s = Step(1)
    s.refill()
    s.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run()
    for _ in range(4):
        s.refill()
        s.run()                                    # eager
        want = s.copies()
        for t in s.results:
            t.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert same(s.copies(), want)


def test_two_graphs_and_eager_calls_on_streams_of_their_own():
    announce("two graphs on two streams beside eager calls on a third")
    steps = [Step(k) for k in range(3)]
    for s in steps:
        s.refill()
        s.run()
    torch.cuda.synchronize()
    want = [s.copies() for s in steps]
    graphs = []
    for s in steps[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.run()
        graphs.append(g)
    for s in steps:
        for t in s.results:
            t.fill_(9.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                graphs[i].replay() if i < 2 else steps[2].run()
    torch.cuda.synchronize()
    for s, w in zip(steps, want):
        assert same(s.copies(), w)


def test_the_same_call_gives_the_same_bits():
    announce("ten equal calls")
    s = Step(7)
    s.refill()
    s.run()
    want = s.copies()
    for _ in range(9):
        s.run()
        assert same(s.copies(), want)


def test_refusals():
    """Every refusal names its argument and comes before anything is launched."""
    announce("refusals")
    k = torch.zeros(4, 16, 2, 64, dtype=BF16, device=DEV)
    f = torch.zeros(4, 16, 2, 64, dtype=FP8, device=DEV)
    fs = torch.ones(4, 16, 2, device=DEV)
    x, slots = torch.zeros(3, 2, 64, dtype=BF16, device=DEV), torch.arange(3, device=DEV)
    refused = lambda match: pytest.raises(RuntimeError, match=match)      # noqa: E731
    with refused("slots must be int64"):
        ops.cache_write(x, k, slots.int())
    with refused("slots must be on the cache's device"):
        ops.cache_write(x, k, slots.cpu())
    with refused(r"k must be \[3, 2, 64\]"):
        ops.cache_write(x[:, :1], k, slots)
    with refused("its scales are needed"):
        ops.cache_write(x, f, slots)
    with refused("only a float8_e4m3fn cache has scales"):
        ops.cache_write(x, k, slots, None, None, fs)
    with refused(r"scales must be \[blocks"):
        ops.cache_write(x, f, slots, None, None, fs[:3])
    with refused("v and vCache go together"):
        ops.cache_write(x, k, slots, x)
    with refused("element type"):
        ops.cache_write(x.half(), k, slots)
    with refused("must be bfloat16 or float16"):
        ops.cache_write(x.float(), k, slots)
    with refused("must not overlap itself"):
        ops.cache_write(x, k[:1].expand(4, 16, 2, 64), slots)
    with refused("must be contiguous"):
        ops.cache_read(k, x, torch.arange(6, device=DEV)[::2])
    with refused("values of a head must be contiguous"):
        ops.cache_read(k.transpose(2, 3).contiguous().transpose(2, 3), x, slots)

    q, out = torch.zeros(3, 4, 64, dtype=BF16, device=DEV), torch.zeros(3, 4, 64, dtype=BF16, device=DEV)
    table, starts, lens = torch.zeros(1, 2, dtype=torch.int64, device=DEV), torch.tensor([0, 3], device=DEV), torch.tensor([5], device=DEV)

    def prompt(q=q, k=k, v=k, table=table, starts=starts, lens=lens, out=out, scale=0.1, **more):
        ops.prompt_attention(q, k, v, table, starts, lens, out, scale, **more)

    prompt()
    with refused("no multiple of the cache's"):
        prompt(q=q[:, :3], out=out[:, :3])
    with refused("must hold q's type"):
        prompt(k=k.half(), v=k.half())
    with refused("out must have q's type"):
        prompt(out=out.half())
    with refused("one shape and one type"):
        prompt(v=k[:3])
    with refused("multiple of 16"):
        prompt(q=q[..., :40], k=k[..., :40], v=k[..., :40], out=out[..., :40])
    with refused("multiple of 16 bytes"):
        prompt(q=torch.zeros(3, 4, 68, dtype=BF16, device=DEV)[..., 2:66])
    with refused("multiple of 16 bytes"):
        prompt(k=torch.zeros(4, 16, 2, 68, dtype=BF16, device=DEV)[..., :64], v=torch.zeros(4, 16, 2, 68, dtype=BF16, device=DEV)[..., :64])
    with refused("one row and queryStarts one entry more"):
        prompt(starts=torch.tensor([0, 1, 3], device=DEV))
    for scale in (0.0, -1.0, float("nan"), float("inf"), 1e300):
        with refused("scale must be positive and finite"):
            prompt(scale=scale)
    with refused("lse must be a contiguous float32"):
        prompt(lse=torch.zeros(3, 4, dtype=torch.float64, device=DEV))
    with refused("must not overlap itself"):
        prompt(out=out[:1].expand(3, 4, 64))
    with refused("blockTable must have 2"):
        prompt(table=table[0])
    with refused("prefixLen must hold one"):
        ops.prefix_attention(q, k, k, table[0], lens.repeat(2), table.repeat(3, 1), lens.repeat(3), out, 0.1)
    with refused("one row per row of q"):
        ops.prefix_attention(q, k, k, table[0], lens, table, lens, out, 0.1)
    # nothing to do is no error
    prompt(q=q[:0], out=out[:0], starts=torch.tensor([0, 0], device=DEV))
    prompt(table=table[:0], starts=starts[:1], lens=lens[:0])
    ops.prefix_attention(q[:0], k, k, table[0], lens, table[:0], lens[:0], out[:0], 0.1)
    ops.cache_write(x[:0], k, slots[:0])
    torch.cuda.synchronize()


def test_refusals_of_overlaps_and_gradients():
    """Two written sides in one memory, results half in the queries, gradients that nobody would compute."""
    announce("refusals of overlaps and gradients")
    k = torch.zeros(4, 16, 2, 64, dtype=BF16, device=DEV)
    f, fs = torch.zeros(4, 16, 2, 64, dtype=FP8, device=DEV), torch.ones(4, 16, 2, device=DEV)
    x, slots = torch.zeros(4, 2, 64, dtype=BF16, device=DEV), torch.arange(3, device=DEV)
    with pytest.raises(RuntimeError, match="kCache and vCache must not overlap"):
        ops.cache_write(x[:3], k, slots, x[:3], k)
    with pytest.raises(RuntimeError, match="kScales and vScales must not overlap"):
        ops.cache_write(x[:3], f, slots, x[:3], f.clone(), fs, fs)
    with pytest.raises(RuntimeError, match="k and v must not overlap"):
        ops.cache_read(k, x[:3], slots, k, x[1:])
    q = torch.zeros(4, 4, 64, dtype=BF16, device=DEV)
    table, starts, lens = torch.zeros(1, 2, dtype=torch.int64, device=DEV), torch.tensor([0, 3], device=DEV), torch.tensor([5], device=DEV)
    with pytest.raises(RuntimeError, match="out and q, unless they are one tensor, must not overlap"):
        ops.prompt_attention(q[:3], k, k, table, starts, lens, q[1:], 0.1)
    with pytest.raises(RuntimeError, match="q requires a gradient"):
        ops.prompt_attention(q[:3].clone().requires_grad_(), k, k, table, starts, lens, q[:3], 0.1)
    with pytest.raises(RuntimeError, match="kCache requires a gradient"):
        ops.prefix_attention(q, k.clone().requires_grad_(), k, table[0], lens, table.repeat(4, 1), lens.repeat(4), q, 0.1)
    with pytest.raises(RuntimeError, match="v requires a gradient"):
        ops.cache_write(x[:3], k, slots, x[:3].clone().requires_grad_(), k.clone())
    with torch.no_grad():
        ops.prompt_attention(q[:3].clone().requires_grad_(), k, k, table, starts, lens, q[:3], 0.1)
    torch.cuda.synchronize()


@pytest.mark.parametrize("rows,keys", [(300, 300), (5, 40), (5, 2000)])
def test_results_in_place_of_the_queries(rows, keys):
    announce("results in place of the queries, %d rows, %d keys" % (rows, keys))
    gen = torch.Generator().manual_seed(rows)
    k, v = (torch.randn(-(-keys // 16), 16, 2, 64, generator=gen).to(BF16).to(DEV) for _ in "kv")
    q = torch.randn(rows, 8, 64, generator=gen).to(BF16).to(DEV)
    table = torch.arange(len(k), device=DEV)[None]
    starts, lens = torch.tensor([0, rows], device=DEV), torch.tensor([keys], device=DEV)
    want = [torch.empty_like(q) for _ in range(2)]
    got = [q.clone() for _ in range(2)]
    for to, of in zip((want, got), ([q, q], got)):
        ops.prompt_attention(of[0], k, v, table, starts, lens, to[0], 0.125)
        ops.prefix_attention(of[1], k, v, table[0, :2], lens.clamp(max=20), table.repeat(rows, 1), lens.repeat(rows), to[1], 0.125)
    assert same(got, want)


def test_refused_calls_have_no_effect_and_capture_goes_on():
    """A refused call inside a capture leaves the capture sound."""
    announce("a refusal inside a capture")
    s = Step(4)
    s.refill()
    s.run()
    want = s.copies()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError):
            ops.cache_read(s.k, s.results[0], s.slots, None, None, None, None)
        s.run()
    for t in s.results:
        t.fill_(9.0)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert same(s.copies(), want)


def test_c_entry_points_take_their_own_workspace():
    """hfk_prompt_attention through the C-ABI: too small a workspace is refused before anything is launched, the stated size is
    enough and nothing behind it is touched."""
    import ctypes

    from heterofusedkernels_amd import capi

    announce("C entry points and their workspace")
    s = Step(3)
    s.refill()
    s.run()
    want = s.copies()

    def plane(t, sc):
        return capi.CachePlane(t.data_ptr(), sc.data_ptr(), t.stride(0), t.stride(1), t.stride(2), sc.stride(0), sc.stride(1), sc.stride(2),
                               t.shape[0], t.shape[1], t.shape[2], t.shape[3], capi.FP8_E4M3)

    def rows(t):
        return capi.TokenRows(t.data_ptr(), t.stride(0), t.stride(1), capi.BF16)

    stream = torch.cuda.current_stream().cuda_stream
    for q, out, lse, prompt in ((s.q, s.results[2], s.results[3], True), (s.one, s.results[4], s.results[5], False)):
        a = capi.Attention(plane(s.k, s.ks), plane(s.v, s.vs), rows(q), rows(out), lse.data_ptr(), q.shape[0], 8, 0.125)
        prefix = s.table[0, :40]
        rc, size = capi.prompt_attention_workspace(a, 1, s.table.shape[1]) if prompt else capi.prefix_attention_workspace(a, 40, s.own.shape[1])
        assert rc == 0 and size > 0 and size % 256 == 0
        space = torch.full((size + 4096,), 77, dtype=torch.uint8, device=DEV)
        assert space.data_ptr() % 256 == 0

        def call(pointer, n):
            if prompt:
                return capi.prompt_attention(a, s.table.data_ptr(), 1, s.table.shape[1], s.starts.data_ptr(), s.len.data_ptr(), True, pointer, n, stream)
            return capi.prefix_attention(a, prefix.data_ptr(), 40, s.prefix_len.data_ptr(), s.own.data_ptr(), s.own.shape[1], s.own_lens.data_ptr(),
                                         pointer, n, stream)

        out.fill_(9.0)
        lse.fill_(9.0)
        assert call(space.data_ptr(), size - 1) == capi.ERR_WORKSPACE_TOO_SMALL
        assert call(0, size) == -1
        assert call(space.data_ptr() + 16, size) == capi.ERR_BAD_ALIGNMENT
        torch.cuda.synchronize()
        assert bool((out == 9.0).all())
        assert call(space.data_ptr(), size) == 0
        torch.cuda.synchronize()
        assert bool((space[size:] == 77).all())
    assert same(s.copies(), want)
    assert ctypes.sizeof(capi.CachePlane) == 2 * 8 + 6 * 8 + 8 + 4 * 4
