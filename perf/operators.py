"""Workloads of the cache and attention operators: ``cache_write``, ``cache_read``, ``prompt_attention``, ``prefix_attention``.

``run`` computes a case in plain torch operations, or, with ``own`` set, through ``torch.ops.pcie_through``. A cache plane is
``[blocks, T, heads, D]``, stored tokens-first like the caches of ``swap_blocks`` or heads-first like the layers of
``multi_layer_block_transfer``; a slot is ``block * T + offset``. Every sequence length is a function of the case alone.
"""
import math

import torch

own = False

BF16, FP16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
TYPES = {"bf16": BF16, "fp16": FP16, "fp8": FP8}
DEV = "cuda"


def listed():
    return [
        # one token of one sequence enters an fp8 cache: the smallest call of a decoding step
        dict(name="write-fp8-1", op="write", n=1, heads=8, dim=128, block=16, type="bf16", cache="fp8", order="thd", padded=0),
        # a long prompt enters an fp8 cache, heads-first as the block transfer lays its layers out
        dict(name="write-fp8-8192", op="write", n=8192, heads=8, dim=128, block=16, type="bf16", cache="fp8", order="htd", padded=0),
        # an odd number of latent rows (one head of 576, no values), the batch padded at its end
        dict(name="write-latent-1000", op="write", n=1000, heads=1, dim=576, block=64, type="bf16", cache="bf16", order="thd", padded=24),
        # a short prefix read back in fp16
        dict(name="read-fp8-77", op="read", n=77, heads=8, dim=64, block=16, type="fp16", cache="fp8", order="thd", padded=0),
        # a long swapped-in prefix read back for a pass that wants it dense
        dict(name="read-fp8-32768", op="read", n=32768, heads=8, dim=128, block=16, type="bf16", cache="fp8", order="thd", padded=0),
        # one short prompt, everything new
        dict(name="prompt-33", op="prompt", seqs=1, q_max=33, past=0, q_heads=16, heads=4, dim=64, block=16, type="fp16", cache="fp16", order="thd", causal=True),
        # one long prompt, everything new: compute-bound
        dict(name="prompt-8192", op="prompt", seqs=1, q_max=8192, past=0, q_heads=32, heads=8, dim=128, block=16, type="bf16", cache="bf16", order="thd", causal=True),
        # a ragged batch of prompts from one token to 1999, each behind a cached past
        dict(name="prompt-ragged", op="prompt", seqs=9, q_max=1999, past=700, q_heads=32, heads=8, dim=128, block=16, type="bf16", cache="bf16", order="htd", causal=True),
        # a chunk of a prompt behind a long fp8 past: few queries, many keys
        dict(name="prompt-chunk-fp8", op="prompt", seqs=1, q_max=250, past=16000, q_heads=32, heads=8, dim=128, block=16, type="bf16", cache="fp8", order="thd", causal=True),
        # one sequence, short prefix: latency
        dict(name="prefix-1", op="prefix", batch=1, prefix=500, own_max=20, q_heads=32, heads=8, dim=128, block=16, type="fp16", cache="fp16", order="thd"),
        # a batch of 64 under one system prompt of 16384 tokens
        dict(name="prefix-64", op="prefix", batch=64, prefix=16384, own_max=1023, q_heads=32, heads=8, dim=128, block=16, type="bf16", cache="bf16", order="thd"),
        # no prefix in common: the ordinary paged decoding step over long fp8 caches
        dict(name="decode-24-fp8", op="prefix", batch=24, prefix=0, own_max=16001, q_heads=64, heads=8, dim=128, block=64, type="bf16", cache="fp8", order="thd"),
    ]


def _log(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    op = rng.choice(["write", "read", "prompt", "prefix"])
    kind = rng.choice(["bf16", "fp16"])
    cache = rng.choice([kind, "fp8"])
    block, order = rng.choice([16, 32, 64]), rng.choice(["thd", "htd"])
    if op in ("write", "read"):
        heads, dim = rng.choice([(1, 576), (1, 128), (2, 128), (4, 64), (5, 96), (8, 64), (8, 128), (16, 128)])
        n = _log(rng, 1, 8192 if op == "write" else 32768) // (2 if heads == 16 else 1) + 1
        return dict(op=op, n=n, heads=heads, dim=dim, block=block, type=kind, cache=cache, order=order, padded=rng.choice([0, 0, n // 9]))
    heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 8]) if heads == 8 else rng.choice([1, 3, 4, 7, 8])
    dim = rng.choice([64, 128])
    if op == "prompt":
        seqs, q_max, past = _log(rng, 1, 16), _log(rng, 1, 6000), _log(rng, 1, 16000) - 1
        while seqs * q_max * (q_max + past) * heads * group > 6000 * 6000 * 32 or seqs * (q_max + past) > 120000:
            seqs, q_max, past = max(1, seqs - 1), max(1, q_max * 3 // 4), past * 3 // 4
        return dict(op=op, seqs=seqs, q_max=q_max, past=past, q_heads=heads * group, heads=heads, dim=dim, block=block, type=kind, cache=cache, order=order, causal=rng.random() < 0.85)
    batch, prefix, most = _log(rng, 1, 96), rng.choice([0, 1, 1, 1]) * _log(rng, 1, 20000), _log(rng, 1, 16000)
    while batch * most > 300000:
        most = most * 3 // 4
    return dict(op=op, batch=batch, prefix=prefix, own_max=most, q_heads=heads * group, heads=heads, dim=dim, block=block, type=kind, cache=cache, order=order)


def _spread(count, most):
    """`count` lengths between 0 or 1 and `most`, uneven, the longest first, one of them 1."""
    return [max(1, most - (i * 2654435761 % 1000003) * most // 1000003) if i else most for i in range(count - 1)] + [1] if count > 1 else [most]


def _lengths(case):
    """(queries, keys) of each sequence of a prompt case: a past of its own before each."""
    q = _spread(case["seqs"], case["q_max"])
    past = _spread(case["seqs"], case["past"]) if case["past"] else [0] * case["seqs"]
    return q, [a + b for a, b in zip(q, past)]


def _plane(blocks, case):
    """An empty plane of `blocks` blocks as [blocks, T, heads, D], its scales, in the case's order."""
    T, H, D, kind = case["block"], case["heads"], case["dim"], TYPES[case["cache"]]
    if case["order"] == "thd":
        return torch.zeros(blocks, T, H, D, dtype=kind, device=DEV), torch.ones(blocks, T, H, device=DEV)
    return (torch.zeros(blocks, H, T, D, dtype=kind, device=DEV).permute(0, 2, 1, 3),
            torch.ones(blocks, H, T, device=DEV).permute(0, 2, 1))


def _filled(blocks, case, gen, outlier):
    """A plane of random tokens; keys have a few channels far larger than the others, as trained models' keys do."""
    plane, scales = _plane(blocks, case)
    x = torch.randn(plane.shape, generator=gen, device=DEV, dtype=torch.float32)
    if outlier:
        x[..., ::37] *= 4.0
    x = x.to(TYPES[case["type"]])
    if case["cache"] == "fp8":
        x, s = _quantised(x)
        scales.copy_(s)
        plane.view(torch.uint8).copy_(x.view(torch.uint8))
    else:
        plane.copy_(x)
    return plane, scales


def _quantised(x):
    """(e4m3 values, scales of the last dim): the smallest power of two that brings the largest finite value to 448 or less."""
    x = x.float()
    size = x.abs()
    most = torch.where(torch.isfinite(size), size, 0.0).amax(-1)
    part, exponent = torch.frexp(most)            # most = part * 2 ** exponent, part in [0.5, 1), and 448 = 0.875 * 2 ** 9
    exponent = (exponent - 9 + (part > 0.875).to(exponent.dtype)).clamp(-126, 119)
    scale = torch.where(most > 0, torch.ldexp(torch.ones_like(most), exponent), 1.0)
    return (x / scale[..., None]).clamp(-448.0, 448.0).to(FP8), scale


def _random(gen, kind, *shape):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(TYPES[kind])


def _table(lengths, T, ids):
    """Block table of sequences of these lengths out of shuffled block ids."""
    width = max(1, max(-(-n // T) for n in lengths))
    return ids[: len(lengths) * width].view(len(lengths), width).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = dict(case=case)
    T, H, D = case["block"], case["heads"], case["dim"]
    if case["op"] in ("write", "read"):
        n = case["n"]
        need = -(-n // T)
        blocks = need + need // 4 + 2
        # tokens of a sequence lie one behind the other in shuffled blocks; those of the padding have no slot
        order = torch.randperm(blocks, generator=gen, device=DEV)[:need]
        slots = (order[:, None] * T + torch.arange(T, device=DEV)).reshape(-1)[:n].contiguous()
        if case["padded"]:
            slots[n - case["padded"]:] = -1
        s["slots"] = slots
        s["sides"] = 1 if case["dim"] == 576 else 2
        if case["op"] == "write":
            for side in "kv"[: s["sides"]]:
                whole, scales = _plane(blocks + 1, case)   # the last block is no part of the cache: it takes the plain form's padding
                s[side] = _random(gen, case["type"], n, H, D)
                s[side + "_whole"], s[side + "_whole_scales"] = whole, scales
                s[side + "_cache"], s[side + "_scales"] = whole[:blocks], scales[:blocks]
        else:
            for side in "kv"[: s["sides"]]:
                s[side + "_cache"], s[side + "_scales"] = _filled(blocks, case, gen, side == "k")
                s[side] = torch.zeros(n, H, D, dtype=TYPES[case["type"]], device=DEV)
        return s
    if case["op"] == "prompt":
        q, kv = _lengths(case)
        total, longest = sum(q), max(kv)
        starts = [0]
        for n in q:
            starts.append(starts[-1] + n)
        s.update(starts=torch.tensor(starts, device=DEV), q_max=max(q), kv_max=longest)
        needed = len(kv) * -(-longest // T)
    else:
        kv = _spread(case["batch"], case["own_max"])
        total, longest = case["batch"], max(kv)
        pre = -(-case["prefix"] // T)
        needed = len(kv) * -(-longest // T) + pre
        s["prefix_len"] = torch.tensor([case["prefix"]], device=DEV)
        s.update(kv_max=longest, prefix_max=case["prefix"])
    blocks = needed + needed // 8 + 1
    ids = torch.randperm(blocks, generator=gen, device=DEV)
    s["table"] = _table(kv, T, ids)
    if case["op"] == "prefix":
        s["prefix_blocks"] = ids[needed - pre: needed].contiguous()
    s["kv"] = torch.tensor(kv, device=DEV)
    s["q"] = _random(gen, case["type"], total, case["q_heads"], D)
    s["k_cache"], s["k_scales"] = _filled(blocks, case, gen, True)
    s["v_cache"], s["v_scales"] = _filled(blocks, case, gen, False)
    s["out"] = torch.zeros_like(s["q"])
    s["lse"] = torch.zeros(total, case["q_heads"], device=DEV)
    s["scale"] = D ** -0.5
    return s


def run(s):
    return _through_the_ops(s) if own else _plainly(s)


def _through_the_ops(s):
    import heterofusedkernels_amd  # noqa: F401
    import pcie_through  # noqa: F401

    ops, case = torch.ops.pcie_through, s["case"]
    ks, vs = (s["k_scales"], s.get("v_scales")) if case["cache"] == "fp8" else (None, None)
    if case["op"] == "write":
        ops.cache_write(s["k"], s["k_cache"], s["slots"], s.get("v"), s.get("v_cache"), ks, vs)
        return {name: s[name] for name in _written(s)}
    if case["op"] == "read":
        ops.cache_read(s["k_cache"], s["k"], s["slots"], s.get("v_cache"), s.get("v"), ks, vs)
        return {side: s[side] for side in "kv"[: s["sides"]]}
    if case["op"] == "prompt":
        ops.prompt_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["starts"], s["kv"], s["out"], s["scale"], case["causal"], ks, vs, s["lse"])
    else:
        ops.prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["prefix_blocks"], s["prefix_len"], s["table"], s["kv"], s["out"], s["scale"], ks, vs, s["lse"])
    return {"out": s["out"], "lse": s["lse"]}


def _written(s):
    names = [side + "_cache" for side in "kv"[: s["sides"]]]
    return names + [side + "_scales" for side in "kv"[: s["sides"]]] if s["case"]["cache"] == "fp8" else names


def _plainly(s):
    return {"write": _write, "read": _read, "prompt": _prompt, "prefix": _prefix}[s["case"]["op"]](s)


def _write(s):
    T, fp8 = s["case"]["block"], s["case"]["cache"] == "fp8"
    slots = torch.where(s["slots"] >= 0, s["slots"], s["k_cache"].shape[0] * T)
    at = (slots // T, slots % T)
    _write_side(s, "k", at, fp8)
    if s["sides"] == 2:
        _write_side(s, "v", at, fp8)
    return {name: s[name] for name in _written(s)}


def _write_side(s, side, at, fp8):
    if fp8:
        values, scales = _quantised(s[side])
        s[side + "_whole"].view(torch.uint8).index_put_(at, values.view(torch.uint8))
        s[side + "_whole_scales"].index_put_(at, scales)
    else:
        s[side + "_whole"].index_put_(at, s[side])


def _read(s):
    T = s["case"]["block"]
    slots = s["slots"].clamp(min=0)
    at, keep = (slots // T, slots % T), (s["slots"] >= 0)[:, None, None]
    got = {"k": _read_side(s, "k", at, keep)}
    if s["sides"] == 2:
        got["v"] = _read_side(s, "v", at, keep)
    return got


def _read_side(s, side, at, keep):
    x, kind = _rows(s, side, *at), s[side].dtype
    return torch.where(keep, x.clamp(-torch.finfo(kind).max, torch.finfo(kind).max).to(kind), s[side])


def _rows(s, side, block, offset):
    """Rows of the cache in 32 bits."""
    if s["case"]["cache"] == "fp8":
        values = s[side + "_cache"].view(torch.uint8)[block, offset].view(FP8).float()
        return values * s[side + "_scales"][block, offset][..., None]
    return s[side + "_cache"][block, offset].float()


def _paged(s, side, table, count):
    """The first `count` tokens of each row of a block table: [rows, heads, count, D]."""
    j = torch.arange(count, device=DEV)
    T = s["case"]["block"]
    return _rows(s, side, table[:, j // T], (j % T).expand(table.shape[0], count)).transpose(1, 2)


def _weights(scores, seen):
    """exp(scores - their largest) of the seen keys, its sum, and the largest."""
    scores = scores.masked_fill(~seen, -math.inf)
    most = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(scores - most)
    return p, p.sum(-1, keepdim=True), most


def _finish(o, total, most):
    lse = torch.where(total > 0, most + torch.log(total), -math.inf)
    return torch.where(total > 0, o / total, 0.0), lse[..., 0]


def _prompt(s):
    case, starts, kv = s["case"], s["starts"], s["kv"]
    H, D, G = case["heads"], case["dim"], case["q_heads"] // case["heads"]
    n, Q, L = kv.shape[0], s["q_max"], s["kv_max"]
    count = starts[1:] - starts[:-1]
    i, j = torch.arange(Q, device=DEV), torch.arange(L, device=DEV)
    at = (starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[at].view(n, Q, H, G, D).permute(0, 2, 3, 1, 4).reshape(n * H, G * Q, D)
    k = _paged(s, "k", s["table"], L).reshape(n * H, L, D)
    v = _paged(s, "v", s["table"], L).reshape(n * H, L, D)
    scores = (torch.bmm(q, k.transpose(1, 2)) * s["scale"]).view(n, H, G, Q, L)
    limit = (kv - count)[:, None] + i if case["causal"] else (kv - 1)[:, None].expand(n, Q)
    p, total, most = _weights(scores, (j <= limit[..., None])[:, None, None])
    o = torch.bmm(p.view(n * H, G * Q, L), v).view(n, H, G, Q, D)
    o, lse = _finish(o, total, most)
    # the padded batch back to packed rows: row r is query r - starts[b] of its sequence b
    r = torch.arange(s["q"].shape[0], device=DEV)
    b = torch.searchsorted(starts, r, right=True) - 1
    r = r - starts[b]
    return {"out": o[b, :, :, r].flatten(1, 2).to(s["q"].dtype), "lse": lse[b, :, :, r].flatten(1, 2)}


def _prefix(s):
    case, kv = s["case"], s["kv"]
    H, D, G = case["heads"], case["dim"], case["q_heads"] // case["heads"]
    B, P, L = case["batch"], s["prefix_max"], s["kv_max"]
    q = s["q"].float().view(B, H, G, D)
    # the prefix: one product for the whole batch
    shared_q = q.permute(1, 0, 2, 3).reshape(H, B * G, D)
    shared_k, shared_v = (_paged(s, side, s["prefix_blocks"][None], P)[0] for side in "kv")
    shared = torch.bmm(shared_q, shared_k.transpose(1, 2)).view(H, B, G, P).permute(1, 0, 2, 3)
    # the sequences' own tokens
    k, v = (_paged(s, side, s["table"], L).reshape(B * H, L, D) for side in "kv")
    alone = torch.bmm(q.reshape(B * H, G, D), k.transpose(1, 2)).view(B, H, G, L)
    j = torch.arange(P + L, device=DEV)
    seen = (j < P + kv[:, None])[:, None, None]
    p, total, most = _weights(torch.cat([shared, alone], -1) * s["scale"], seen)
    o = torch.bmm(p[..., P:].reshape(B * H, G, L), v).view(B, H, G, D)
    o = o + torch.bmm(p[..., :P].permute(1, 0, 2, 3).reshape(H, B * G, P), shared_v).view(H, B, G, D).transpose(0, 1)
    o, lse = _finish(o, total, most)
    return {"out": o.reshape(B, H * G, D).to(s["q"].dtype), "lse": lse.reshape(B, H * G)}


def work(case):
    H, D = case["heads"], case["dim"]
    size, cached = 2, 1 if case["cache"] == "fp8" else 2
    scale = 4 if case["cache"] == "fp8" else 0
    if case["op"] in ("write", "read"):
        n, sides = case["n"] - case["padded"], 1 if D == 576 else 2
        return {"bytes": 8 * case["n"] + sides * n * H * (D * (size + cached) + scale), "flops": sides * n * H * D * (2 if scale else 0)}
    row = 2 * H * (D * cached + scale)      # a token's keys and values
    if case["op"] == "prompt":
        q, kv = _lengths(case)
        pairs = sum(n * (L - n) + n * (n + 1) // 2 if case["causal"] else n * L for n, L in zip(q, kv))
        queries, tokens = sum(q), sum(kv)
    else:
        kv = _spread(case["batch"], case["own_max"])
        queries, tokens, pairs = case["batch"], case["prefix"] + sum(kv), case["batch"] * case["prefix"] + sum(kv)
    return {"bytes": tokens * row + queries * case["q_heads"] * (2 * D * size + 4), "flops": 4 * D * case["q_heads"] * pairs}


def _exact_rows(s, side, slots):
    T = s["case"]["block"]
    x = s[side + "_cache"][slots // T, slots % T].double() if s["case"]["cache"] != "fp8" else (
        s[side + "_cache"].view(torch.uint8)[slots // T, slots % T].view(FP8).double() * s[side + "_scales"][slots // T, slots % T].double()[..., None])
    return x


def exact(case, seed):
    s = prepare(case, seed)
    T, D = case["block"], case["dim"]
    sides = "kv"[: s.get("sides", 2)]
    if case["op"] == "write":
        got = {}
        keep = s["slots"] >= 0
        slots = s["slots"][keep]
        for side in sides:
            cache, scales = s[side + "_cache"].double(), s[side + "_scales"].double()
            x = s[side][keep].double()
            if case["cache"] == "fp8":
                most = x.abs().amax(-1)
                scale = torch.exp2(torch.ceil(torch.log2(most / 448.0)))
                scales[slots // T, slots % T] = scale
                x = x / scale[..., None]
                got[side + "_scales"] = scales
            cache[slots // T, slots % T] = x
            got[side + "_cache"] = cache
        return got
    if case["op"] == "read":
        got = {}
        for side in sides:
            x = s[side].double()
            keep = s["slots"] >= 0
            x[keep] = _exact_rows(s, side, s["slots"][keep])
            got[side] = x
        return got
    H, G = case["heads"], case["q_heads"] // case["heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device=DEV)
    tables, lens = s["table"], s["kv"].tolist()
    starts = s["starts"].tolist() if case["op"] == "prompt" else list(range(case["batch"] + 1))
    shared = torch.zeros(0, dtype=torch.int64, device=DEV)
    if case["op"] == "prefix":
        j = torch.arange(case["prefix"], device=DEV)
        shared = s["prefix_blocks"][j // T] * T + j % T
    for b, length in enumerate(lens):
        j = torch.arange(length, device=DEV)
        slots = torch.cat([shared, tables[b, j // T] * T + j % T])
        k, v = _exact_rows(s, "k", slots), _exact_rows(s, "v", slots)
        first, last = starts[b], starts[b + 1]
        for h in range(H):
            q = s["q"][first:last, h * G:(h + 1) * G].double().transpose(0, 1)      # [G, n, D]
            scores = torch.matmul(q, k[:, h].t().contiguous()) * s["scale"]
            if case["op"] == "prompt" and case["causal"]:
                hidden = torch.ones(last - first, length, dtype=torch.bool, device=DEV).triu(length - (last - first) + 1)
                scores.masked_fill_(hidden, -math.inf)
            lse[first:last, h * G:(h + 1) * G] = torch.logsumexp(scores, -1).t()
            out[first:last, h * G:(h + 1) * G] = torch.matmul(torch.softmax(scores, -1), v[:, h].contiguous()).transpose(0, 1)
    return {"out": out, "lse": lse}
