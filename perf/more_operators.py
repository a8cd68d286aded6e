"""Attention over a paged cache, as cases that can be timed and whose outputs can be compared.

Three operators: rotary positions with several axes (on their own, or with the turned keys and the values written into the
cache), attention of one new token over the cache, and what keeps its pages (taking over, extending, moving together).  Heads
of 64 on 20 and images of 832 x 1216 and 1024 x 1024 are those of SDXL, prompts have 77 tokens; the rest is generic.  Queries,
keys and values ~ N(0, 1), as norms in front of the projections leave them.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
E4M3 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": E4M3}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}


def listed():
    return [
        # The image tokens of a guidance pair at 832 x 1216, q and k as slices of one projection's output.
        dict(name="rotary_2x3952_20_heads", op="rotary", rows=7904, heads=20, kv_heads=20, d=64, sections="8,12,12", pairs=True,
             dtype="bf16", fused=True, fractions=False),
        # Sixteen frames of 32 x 32 tokens at fractions of a second, in 32 bits.
        dict(name="rotary_16384_fp32", op="rotary", rows=16384, heads=16, kv_heads=8, d=128, sections="16,24,24", pairs=False,
             dtype="fp32", fused=False, fractions=True),
        # One token of a guidance pair: the smallest call.
        dict(name="append_2_tokens", op="append", lengths="77,77", new="1,1", pool=2, heads=20, kv_heads=20, d=64, sections="32",
             pairs=False, dtype="bf16", cache="bf16", page=16, layers=1),
        # One token each of 64 requests into pages of 8-bit numbers; the other slots are not of this step.
        dict(name="append_64_tokens_e4m3", op="append", lengths=",".join(str(1 + 83 * i % 2000) for i in range(64)), new=",".join("1" * 64),
             pool=96, heads=32, kv_heads=8, d=128, sections="16,24,24", pairs=True, dtype="bf16", cache="e4m3", page=32, layers=2),
        # Prompts of mixed lengths, pages and heads that no tile divides, a part of each head turned.
        dict(name="append_8184_rows_fp16", op="append", lengths="4500,77,0,1023,4093,1,640,2355", new="4096,77,0,1023,64,1,568,2355", pool=8, heads=16,
             kv_heads=8, d=80, sections="24", pairs=False, dtype="fp16", cache="fp16", page=24, layers=1),
        # One token of a guidance pair over its prompts.
        dict(name="attention_2x77_20_heads", op="attention", lengths="77,77", pool=2, heads=20, kv_heads=20, d=64, page=16, window=0,
             dtype="bf16", cache="bf16", layers=1),
        # One token each of 64 requests of mixed lengths, an empty one among them.
        dict(name="attention_64_requests", op="attention", lengths=",".join(str([8192, 0, 1, 77, 4096, 640, 2355, 5000][i % 8] + (i // 8) * (i % 8 > 2)) for i in range(64)),
             pool=96, heads=32, kv_heads=8, d=128, page=32, window=0, dtype="bf16", cache="bf16", layers=2),
        # One long sequence, on few key heads.
        dict(name="attention_131072_tokens", op="attention", lengths="131071", pool=1, heads=16, kv_heads=2, d=128, page=64, window=0,
             dtype="fp16", cache="fp16", layers=1),
        # A window over an 8-bit cache, no size a multiple of any tile.
        dict(name="attention_13_window_e4m3", op="attention", lengths="5000,1,999,1000,1001,0,77,23,24,25,3100,2047,4095", pool=13, heads=15, kv_heads=3, d=80,
             page=24, window=1000, dtype="bf16", cache="e4m3", layers=1),
        # Four beams of one prompt that go on from the same tokens.
        dict(name="fork_4_beams", op="fork", parents="77", children=3, pool=4, kv_heads=20, d=64, page=16, grow=4, cache="bf16", layers=2),
        # Six answers to each of eight prompts, through the layers of a model.
        dict(name="fork_48_of_8_24_layers", op="fork", parents="4100,77,2355,1023,31,640,8191,2000", children=6, pool=64, kv_heads=8, d=128, page=32, grow=40, cache="bf16",
             layers=24),
        # A pool of which a good half is in use, moved to its lower end.
        dict(name="compact_2048_pages", op="compact", pages=2048, live=0.6, pool=40, kv_heads=8, d=128, page=32, cache="bf16", layers=4),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _sections(rng, d):
    turned = rng.choice([d, d, d // 2 // 8 * 8]) // 2
    if rng.random() < 0.4:
        return str(turned)
    first = max(1, turned // 4)
    second = (turned - first) // 2
    return "%d,%d,%d" % (first, second, turned - first - second) if rng.random() < 0.7 else "%d,%d" % (first, turned - first)


def draw(rng):
    op = rng.choice(["rotary", "append", "append", "attention", "attention", "attention", "fork", "compact"])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8, 10, 20])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8]) if kv_heads < 10 else kv_heads
    d = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    page = rng.choice([8, 16, 16, 24, 32, 64, 100, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    cache = rng.choice([dtype, dtype, "e4m3"])
    if op == "rotary":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        rows = _log_int(rng, 1, max(1, 16384 * 24 * 128 // ((heads + kv_heads) * d)))
        return dict(op=op, rows=rows, heads=heads, kv_heads=kv_heads, d=d, sections=_sections(rng, d), pairs=rng.random() < 0.5, dtype=dtype,
                    fused=rng.random() < 0.5, fractions=rng.random() < 0.3)
    if op == "append":
        count = _log_int(rng, 1, 128)
        longest = max(1, 8192 * 16 * 80 // (count * heads * d))
        new = [1] * count if rng.random() < 0.5 else [rng.choice([0, 1, _log_int(rng, 1, longest), longest]) for _ in range(count)]
        new[0] = max(1, new[0])
        before = max(1, 2000 * 8 * 128 * 64 // (count * kv_heads * d * 8))
        return dict(op=op, lengths=",".join(str(n + rng.randint(0, min(before, 2000))) for n in new), new=",".join(map(str, new)), pool=count + rng.choice([0, 0, 5]),
                    heads=heads, kv_heads=kv_heads, d=d, sections=_sections(rng, d), pairs=rng.random() < 0.5, dtype=dtype, cache=cache, page=page, layers=rng.choice([1, 2]))
    if op == "attention":
        count = _log_int(rng, 1, 200)
        longest = max(1, min(131072, 64 * 2500 * 8 * 128 // (count * kv_heads * d)))
        first = _log_int(rng, 1, longest)
        lengths = [first] + [rng.choice([0, 1, rng.randint(1, first), rng.randint(1, first), first]) for _ in range(count - 1)]
        return dict(op=op, lengths=",".join(map(str, lengths)), pool=count + rng.choice([0, 0, 5]), heads=heads, kv_heads=kv_heads, d=d, page=page,
                    window=rng.choice([0, 0, 0, _log_int(rng, 1, 4096)]), dtype=dtype, cache=cache, layers=rng.choice([1, 2]) if count * first * kv_heads * d < 1 << 27 else 1)
    layers = rng.choice([1, 2, 4, 16])
    if op == "fork":
        count = rng.choice([1, 2, 3, 8])
        longest = max(1, min(8192, (1 << 27) // (layers * count * kv_heads * d)))
        parents = [_log_int(rng, 1, longest) for _ in range(count)]
        children = rng.choice([1, 2, 3, 6])
        return dict(op=op, parents=",".join(map(str, parents)), children=children, pool=count * (children + 1) + rng.choice([0, 0, 7]), kv_heads=kv_heads, d=d, page=page,
                    grow=rng.choice([0, 1, 5, 60]), cache=cache, layers=layers)
    return dict(op=op, pages=_log_int(rng, 9, max(9, min(20000, (1 << 28) // (layers * kv_heads * d * page)))), live=rng.choice([0.1, 0.5, 0.6, 0.9]), pool=_log_int(rng, 1, 60),
                kv_heads=kv_heads, d=d, page=page, cache=cache, layers=layers)


# ------------------------------------------------------------------------------------------ inputs
def _ints(text):
    return [int(t) for t in text.split(",")]


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _attended(case):
    n = _ints(case["lengths"])
    return [min(t, case["window"]) if case["window"] else t for t in n]


def _frequencies(sections):
    """Angles of a step, for each pair: one row of them over all axes."""
    pairs = sum(sections)
    return 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device=DEV) / pairs)


def _pages(case, gen, held, spare):
    """A cache whose slot i holds held[i] tokens on pages in no order: (k, v, table, lengths, refs, scales of k, scales of v)."""
    page, layers, Hk, d = case["page"], case["layers"], case["kv_heads"], case["d"]
    need = [-(-n // page) for n in held]
    count = sum(need) + spare
    width = max(max(need), 1) + -(-case.get("grow", 0) // page) + 1
    order = torch.randperm(count, generator=gen, device=DEV).to(torch.int32)
    used, first = torch.tensor(need, device=DEV), torch.tensor([sum(need[:i]) for i in range(len(need))], device=DEV)
    at = torch.arange(width, device=DEV)
    there = at < used[:, None]
    table = torch.where(there, order[torch.where(there, first[:, None] + at, 0)], -1).to(torch.int32)
    refs = torch.zeros(count, dtype=torch.int32, device=DEV)
    refs[order[:sum(need)].long()] = 1
    k, v = (torch.randn(layers, count, page, Hk, d, generator=gen, device=DEV, dtype=torch.bfloat16).to(TYPES[case["cache"]]) for _ in range(2))
    ks = vs = None
    if case["cache"] == "e4m3":
        ks, vs = (torch.rand(layers, Hk, generator=gen, device=DEV) * 0.02 + 0.02 for _ in range(2))
        k, v = ((t.float() * 16).to(E4M3) for t in (k, v))    # (codes as they are used: numbers of up to 60 or so)
    return k, v, table, _int32(held), refs, ks, vs


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, dtype):
        return torch.randn(*shape, generator=gen, device=DEV).to(TYPES[dtype])

    if case["op"] == "rotary":
        rows, H, Hk, d, sections = case["rows"], case["heads"], case["kv_heads"], case["d"], _ints(case["sections"])
        side = max(1, math.isqrt(rows))
        row = torch.arange(rows, device=DEV)
        positions = torch.stack((row // (side * side) + 7, row // side % side, row % side), 1)[:, :len(sections)]
        if case["fractions"]:
            positions = positions + torch.rand(rows, len(sections), generator=gen, device=DEV)
        else:
            positions = (positions + torch.randint(0, 100000, (1,), generator=gen, device=DEV)).to(torch.int32)
        qkv = normal(rows, (H + 2 * Hk) * d, dtype=case["dtype"])
        q, k = qkv[:, :H * d], qkv[:, H * d:(H + Hk) * d]
        if not case["fused"]:
            q, k = q.contiguous(), k.contiguous()
        return dict(case, q=q, k=k, positions=positions.contiguous(), sections=tuple(sections), frequencies=_frequencies(sections))
    if case["op"] in ("append", "attention"):
        H, Hk, d, lengths = case["heads"], case["kv_heads"], case["d"], _ints(case["lengths"])
        slots = torch.randperm(case["pool"], generator=gen, device=DEV)[:len(lengths)].tolist()
        held = [0] * case["pool"]
        for s, n in zip(slots, lengths):
            held[s] = n
        k, v, table, held, refs, ks, vs = _pages(case, gen, held, 3)
        s = dict(case, k_pages=k, v_pages=v, table=table, held=held, refs=refs, k_scale=ks, v_scale=vs, layer=case["layers"] - 1)
        if case["op"] == "attention":
            return dict(s, q=normal(len(lengths), H * d, dtype=case["dtype"]), slots=_int32(slots))
        sections, new = _ints(case["sections"]), _ints(case["new"])
        rows = sum(new)
        qkv = normal(rows, (H + 2 * Hk) * d, dtype=case["dtype"])
        places = [n - m + i for n, m in zip(lengths, new) for i in range(m)]
        positions = torch.randint(0, 200000, (rows, len(sections)), generator=gen, device=DEV).to(torch.int32)
        return dict(s, q=qkv[:, :H * d], k=qkv[:, H * d:(H + Hk) * d], v=qkv[:, (H + Hk) * d:], sections=tuple(sections), frequencies=_frequencies(sections),
                    positions=positions, slots=_int32([t for t, m in zip(slots, new) for _ in range(m)]), places=_int32(places))
    if case["op"] == "fork":
        parents, pool, children = _ints(case["parents"]), case["pool"], case["children"]
        slots = torch.randperm(pool, generator=gen, device=DEV).tolist()
        held, parent, counts = [0] * pool, list(range(pool)), [0] * pool
        for i, n in enumerate(parents):
            held[slots[i]] = n
        for i in range(len(parents) * children):   # each held something of its own before
            child = slots[len(parents) + i]
            held[child] = parents[i % len(parents)] // 2 if i % 3 else 0
            parent[child], counts[child] = slots[i % len(parents)], case["grow"] * (i % 4) // 3
        for child in slots[len(parents) * (children + 1):]:   # and these are done
            held[child], parent[child] = 5, -1
        spare = sum(-(-counts[s] // case["page"]) + 1 for s in range(pool)) + 2
        k, v, table, held, refs, _, _ = _pages(case, gen, held, spare)
        return dict(case, k_pages=k, v_pages=v, table=table, held=held, refs=refs, parent=_int32(parent), counts=_int32(counts))
    pages, pool, page = case["pages"], case["pool"], case["page"]
    live = max(1, int(pages * case["live"]))
    held = [0] * pool
    for i in range(live):
        held[i % pool if i < pool else (i * 7 + i // 5) % pool] += page
    held = [max(0, n - i % page) for i, n in enumerate(held)]
    used = sum(-(-n // page) for n in held)
    k, v, table, held, refs, _, _ = _pages(case, gen, held, pages - used)
    return dict(case, k_pages=k, v_pages=v, table=table, held=held, refs=refs, table0=table.clone(), refs0=refs.clone())


# ------------------------------------------------------------------------------------------ the plain forms
def _turned(t, heads, s):
    """Rows [rows, heads * d] turned by their positions, in 32 bits; the angles in 64."""
    rows, d, n = t.shape[0], s["d"], sum(s["sections"])
    axis = torch.repeat_interleave(torch.arange(len(s["sections"]), device=DEV), torch.tensor(s["sections"], device=DEV), output_size=n)
    angle = s["positions"].double()[:, axis] * s["frequencies"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = t.float().view(rows, heads, d)
    turn = x[..., :2 * n]
    a, b = (turn[..., 0::2], turn[..., 1::2]) if s["pairs"] else (turn[..., :n], turn[..., n:])
    a, b = a * cos - b * sin, b * cos + a * sin
    turn = torch.stack((a, b), -1).flatten(-2) if s["pairs"] else torch.cat((a, b), -1)
    return torch.cat((turn, x[..., 2 * n:]), -1)


def _plain_rotary(s):
    return [_turned(s[n], s[h], s).to(s[n].dtype).flatten(1) for n, h in (("q", "heads"), ("k", "kv_heads"))]


def _plain_append(s):
    page = s["page"]
    q = _turned(s["q"], s["heads"], s).to(s["q"].dtype).flatten(1)
    k = _turned(s["k"], s["kv_heads"], s)
    v = s["v"].float().view(k.shape)
    e = s["table"][s["slots"].long(), s["places"].long() // page].long()
    at = s["places"].long() % page
    for pool, rows, scale in ((s["k_pages"], k, s["k_scale"]), (s["v_pages"], v, s["v_scale"])):
        if scale is not None:
            codes = (rows / scale[s["layer"]][:, None]).clamp(-448, 448).to(E4M3)
            pool.view(torch.uint8)[s["layer"]][e, at] = codes.view(torch.uint8)
        else:
            pool[s["layer"]][e, at] = rows.to(pool.dtype)
    return [q, s["k_pages"], s["v_pages"]]


def _plain_attention(s):
    H, Hk, d, page, layer = s["heads"], s["kv_heads"], s["d"], s["page"], s["layer"]
    n = s["held"][s["slots"].long()].long()
    low = (n - s["window"]).clamp(min=0) if s["window"] else torch.zeros_like(n)
    table = s["table"][s["slots"].long()].clamp(min=0).long()
    t = torch.arange(table.shape[1] * page, device=DEV)
    inside = (t >= low[:, None]) & (t < n[:, None])

    def taken(pool, scale):
        x = pool[layer].view(torch.uint8)[table].view(pool.dtype) if scale is not None else pool[layer][table]
        x = x.float().view(len(n), -1, Hk, d).transpose(1, 2)
        return x if scale is None else x * scale[layer][:, None, None]

    q = s["q"].float().view(-1, Hk, H // Hk, d) * d ** -0.5
    x = taken(s["k_pages"], s["k_scale"]).contiguous() @ q.transpose(-1, -2).contiguous()     # [rows, Hk, tokens, H / Hk]
    x = x.masked_fill(~inside[:, None, :, None], -math.inf)
    p = torch.exp(x - x.amax(2, keepdim=True).clamp(min=-3e38))
    total = p.sum(2)[..., None]
    o = p.transpose(-1, -2).contiguous() @ taken(s["v_pages"], s["v_scale"]).contiguous()
    return torch.where(total > 0, o / total, 0).to(s["q"].dtype).flatten(1)


def _lowest_free(refs, wanted):
    """The lowest free page for each place that wants one, in order; -1 where there is none left."""
    order = torch.argsort((refs != 0).to(torch.int32), stable=True)
    rank = torch.cumsum(wanted.flatten().long(), 0).view(wanted.shape) - 1
    got = wanted & (rank < (refs == 0).sum())
    return torch.where(got, order[rank.clamp(0, refs.numel() - 1)], -1)


def _plain_fork(s):
    page, table, refs, held, parent = s["page"], s["table"], s["refs"], s["held"], s["parent"].long()
    slots, width = table.shape
    me, at = torch.arange(slots, device=DEV), torch.arange(width, device=DEV)
    stays = parent == me
    takes = ~stays & (parent >= 0) & (parent < slots)
    source = torch.where(takes, parent, 0)
    new = torch.where(stays, held, torch.where(takes, held[source], 0))
    full, part = new // page, new % page
    # the lowest taker of a slot that gives its pages up has the page not yet full as it is
    first = torch.full((slots + 1,), slots, device=DEV).scatter_reduce(0, torch.where(takes, parent, slots), me, "amin")
    heir = takes & ~stays[source] & (first[source] == me)
    copies = takes & ~heir & (part > 0)
    taken = table[source]
    kept = takes[:, None] & ((at < full[:, None]) | (heir & (part > 0))[:, None] & (at == full[:, None]))
    left = ~stays[:, None] & (at < (-(-held // page))[:, None])
    count = torch.zeros(refs.numel() + 1, dtype=torch.int32, device=DEV)
    count.index_add_(0, torch.where(kept, taken, refs.numel()).flatten().long(), torch.ones_like(taken).flatten())
    count.index_add_(0, torch.where(left, table, refs.numel()).flatten().long(), -torch.ones_like(taken).flatten())
    refs += count[:-1]
    fresh = _lowest_free(refs, copies)
    row = torch.where(kept, taken, -1)
    row = torch.where(copies[:, None] & (at == full[:, None]), fresh[:, None].to(torch.int32), row)
    table.copy_(torch.where(stays[:, None], table, row))
    copied = copies.nonzero()[:, 0]
    src, dst = taken[copied, full[copied].long()].long(), fresh[copied]
    refs[dst] = 1
    some = (torch.arange(page, device=DEV) < part[copied, None])[:, :, None, None]
    for pool in (s["k_pages"], s["v_pages"]):
        raw = pool.view(torch.uint8) if pool.dtype == E4M3 else pool
        raw[:, dst] = torch.where(some, raw[:, src], raw[:, dst])
    # and what they are going to say
    longer = new + s["counts"]
    wanted = (at >= (-(-new // page))[:, None]) & (at < (-(-longer // page))[:, None])
    fresh = _lowest_free(refs, wanted)
    table.copy_(torch.where(wanted, fresh.to(torch.int32), table))
    refs.index_add_(0, fresh[wanted], torch.ones_like(fresh[wanted], dtype=torch.int32))
    held.copy_(longer)
    return [s["k_pages"], s["v_pages"], table, held, refs]


def _plain_compact(s):
    table, refs = s["table"], s["refs"]
    live = refs > 0
    n = live.sum()
    number = torch.arange(refs.numel(), device=DEV)
    moving, hole = (live & (number >= n)).nonzero()[:, 0], (~live & (number < n)).nonzero()[:, 0]
    to = number.clone()
    to[moving] = hole
    refs[hole] = refs[moving]
    refs[moving] = 0
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), table))
    for pool in (s["k_pages"], s["v_pages"]):
        raw = pool.view(torch.uint8) if pool.dtype == E4M3 else pool
        raw[:, hole] = raw[:, moving]
    return [s["k_pages"], s["v_pages"], table, refs, n.to(torch.int32).view(1)]


def run(state):
    s = state
    if s["op"] == "compact":   # the pages as they lay before the last pass
        s["table"].copy_(s["table0"])
        s["refs"].copy_(s["refs0"])
    if own:
        from katz_amd import ops

        if s["op"] == "rotary":
            return list(ops.rotary(s["q"], s["k"], s["heads"], s["positions"], s["frequencies"], s["sections"], kv_heads=s["kv_heads"], pairs=s["pairs"]))
        cache = ops.PagedCache(s["k_pages"], s["v_pages"], s["table"], s["held"], s["refs"], s.get("k_scale"), s.get("v_scale"))
        if s["op"] == "append":
            q = ops.cache_append(s["q"], s["k"], s["v"], cache, s["heads"], s["positions"], s["frequencies"], s["sections"], layer=s["layer"], slots=s["slots"],
                                 places=s["places"], pairs=s["pairs"])
            return [q, s["k_pages"], s["v_pages"]]
        if s["op"] == "attention":
            return ops.paged_attention(s["q"], cache, s["heads"], layer=s["layer"], slots=s["slots"], window=s["window"])
        if s["op"] == "fork":
            ops.cache_reorder(cache, s["parent"])
            ops.cache_extend(cache, s["counts"])
            return [s["k_pages"], s["v_pages"], s["table"], s["held"], s["refs"]]
        n = ops.cache_compact(cache)
        return [s["k_pages"], s["v_pages"], s["table"], s["refs"], n]
    return {"rotary": _plain_rotary, "append": _plain_append, "attention": _plain_attention, "fork": _plain_fork, "compact": _plain_compact}[s["op"]](s)


# ------------------------------------------------------------------------------------------ the definitions in 64 bits
def _exact_turned(t, heads, s):
    x = t.double().reshape(t.shape[0], heads, s["d"]).clone()
    n, j = sum(s["sections"]), 0
    for axis, count in enumerate(s["sections"]):
        for _ in range(count):
            a, b = (2 * j, 2 * j + 1) if s["pairs"] else (j, j + n)
            z = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), s["positions"][:, axis].double() * float(s["frequencies"][j]))
            y = torch.complex(x[:, :, a], x[:, :, b]) * z[:, None]
            x[:, :, a], x[:, :, b] = y.real, y.imag
            j += 1
    return x


def _moved(pool, moves):
    """The pool in 64 bits after (from, to, tokens) in turn, all read first."""
    out = pool.double()
    for src, dst, tokens in moves:
        out[:, dst, :tokens] = pool[:, src, :tokens].double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "rotary":
        return [_exact_turned(s["q"], case["heads"], s).flatten(1), _exact_turned(s["k"], case["kv_heads"], s).flatten(1)]
    page, d = case["page"], case["d"]
    if case["op"] == "append":
        k, v = _exact_turned(s["k"], case["kv_heads"], s), s["v"].to(f).reshape(-1, case["kv_heads"], d)
        pools = []
        table, slots, places = s["table"].tolist(), s["slots"].tolist(), s["places"].tolist()
        e = torch.tensor([table[a][b // page] for a, b in zip(slots, places)], device=DEV)
        at = torch.tensor([b % page for b in places], device=DEV)
        for pool, rows, scale in ((s["k_pages"], k, s["k_scale"]), (s["v_pages"], v, s["v_scale"])):
            if scale is not None:
                rows = (rows / scale[s["layer"]].to(f)[:, None]).clamp(-448, 448).to(E4M3).to(f)
            out = pool.to(f)
            out[s["layer"]].index_put_((e, at), rows)
            pools.append(out)
        return [_exact_turned(s["q"], case["heads"], s).flatten(1)] + pools
    if case["op"] == "attention":
        H, Hk, layer = case["heads"], case["kv_heads"], s["layer"]
        outs = []
        for r, (slot, n) in enumerate(zip(s["slots"].tolist(), _ints(case["lengths"]))):
            low = max(0, n - case["window"]) if case["window"] else 0
            if n == low:
                outs.append(torch.zeros(H, d, dtype=f, device=DEV))
                continue
            t = torch.arange(low, n, device=DEV)
            e = s["table"][slot, t // page].long()
            k, v = (p[layer].view(torch.uint8)[e, t % page].view(E4M3).to(f) if z is not None else p[layer][e, t % page].to(f)
                    for p, z in ((s["k_pages"], s["k_scale"]), (s["v_pages"], s["v_scale"])))
            if s["k_scale"] is not None:
                k, v = k * s["k_scale"][layer].to(f)[:, None], v * s["v_scale"][layer].to(f)[:, None]
            q = s["q"][r].to(f).view(Hk, H // Hk, d)
            for h in range(Hk):
                x = (k[:, h].contiguous() @ q[h].t().contiguous()) / math.sqrt(d)
                p = torch.softmax(x, 0)
                outs.append(p.t().contiguous() @ v[:, h].contiguous())
        return torch.cat([o.reshape(-1, d) for o in outs]).view(len(s["slots"]), H * d).contiguous()
    table, held, refs = s["table"].tolist(), s["held"].tolist(), s["refs"].tolist()
    moves = []
    if case["op"] == "fork":
        parent, counts = s["parent"].tolist(), s["counts"].tolist()
        before = [list(r) for r in table]
        lengths, given = list(held), set()
        pools = len(table)
        for me in range(pools):
            if parent[me] != me:
                for e in before[me][:-(-held[me] // page)]:
                    refs[e] -= 1
        late = []
        for me in range(pools):
            p = parent[me]
            if p == me:
                continue
            table[me] = [-1] * len(before[me])
            lengths[me] = 0
            if 0 <= p < pools:
                lengths[me] = held[p]
                whole, part = divmod(held[p], page)
                for i in range(whole):
                    table[me][i] = before[p][i]
                    refs[before[p][i]] += 1
                if part and parent[p] != p and p not in given:
                    table[me][whole] = before[p][whole]
                    refs[before[p][whole]] += 1
                elif part:
                    late.append((me, whole, before[p][whole], part))
                given.add(p)
        free = [e for e, n in enumerate(refs) if n == 0]
        for me, whole, src, part in late:
            table[me][whole] = free.pop(0)
            refs[table[me][whole]] = 1
            moves.append((src, table[me][whole], part))
        for me in range(pools):
            for i in range(-(-lengths[me] // page), -(-(lengths[me] + counts[me]) // page)):
                table[me][i] = free.pop(0)
                refs[table[me][i]] = 1
            lengths[me] += counts[me]
        return [_moved(s["k_pages"], moves), _moved(s["v_pages"], moves), _int32(table), _int32(lengths), _int32(refs)]
    live = [e for e, n in enumerate(refs) if n > 0]
    n = len(live)
    to = dict(zip([e for e in live if e >= n], [e for e in range(n) if refs[e] == 0]))
    for src, dst in to.items():
        refs[dst], refs[src] = refs[src], 0
        moves.append((src, dst, page))
    return [_moved(s["k_pages"], moves), _moved(s["v_pages"], moves), _int32([[to.get(e, e) for e in r] for r in table]), _int32(refs), _int32([n])]


def work(case):
    Hk, d = case["kv_heads"], case["d"]
    if case["op"] == "rotary":
        cells = case["rows"] * (case["heads"] + Hk) * d
        return {"bytes": 2.0 * cells * SIZE[case["dtype"]] + 4 * case["rows"] * len(_ints(case["sections"])), "flops": 3.0 * cells}
    token = Hk * d * SIZE[case["cache"]]
    if case["op"] == "append":   # q read and written, k and v read in the rows' type and written in the cache's
        rows = sum(_ints(case["new"]))
        return {"bytes": rows * (2 * SIZE[case["dtype"]] * (case["heads"] + Hk) * d + 2 * token + 12), "flops": 3.0 * rows * (case["heads"] + Hk) * d}
    if case["op"] == "attention":
        tokens, rows = sum(_attended(case)), len(_ints(case["lengths"]))
        return {"bytes": 2.0 * tokens * token + 2 * SIZE[case["dtype"]] * rows * case["heads"] * d + 4 * tokens / case["page"], "flops": 4.0 * tokens * case["heads"] * d}
    if case["op"] == "fork":     # the pages not yet full read and written once a child, tables and counts once
        parents, page = _ints(case["parents"]), case["page"]
        copied = case["children"] * sum(n % page for n in parents)
        entries = sum(-(-n // page) for n in parents) * (case["children"] + 1)
        return {"bytes": 4.0 * case["layers"] * copied * token + 8 * entries, "flops": 0.0}
    used = max(1, int(case["pages"] * case["live"]))
    return {"bytes": 4.0 * case["layers"] * used * (1 - used / case["pages"]) * case["page"] * token + 8 * case["pages"], "flops": 0.0}
