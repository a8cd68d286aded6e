"""Attention over a paged cache as a model runs it: a block of norms, projections with weights in 4 bits, rotary positions, the cache, a gated feed-forward;
over prompts, token by token, forked, moved together, captured, and on other streams."""
import math

import pytest
import torch

from test_gpu_token_block import BF, DEV, F64, HALF, close, linear

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
D, H, HK, DK, FF, LAYERS, SECTIONS = 256, 4, 2, 64, 512, 2, (8, 12, 12)


def int32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Model:
    """Rows h [rows, D] -> h: LAYERS blocks of attention over the cache and a feed-forward."""

    def __init__(self, seed=0):
        from katz_amd import ops

        g = torch.Generator().manual_seed(seed)
        vec = lambda: (torch.randn(D, generator=g) * 0.1 + 1).to(DEV, BF)       # noqa: E731
        self.layers = [(linear(g, (H + 2 * HK) * DK, D), linear(g, D, H * DK, zeros=True, group=32), linear(g, 2 * FF, D, group=128), linear(g, D, FF), vec(), vec())
                       for _ in range(LAYERS)]
        self.frequencies = ops.rotary_frequencies(sum(SECTIONS), device=DEV)

    def __call__(self, h, cache, positions, slots=None, places=None, lengths=None, attended=None):
        from katz_amd import ops

        for i, (qkv, out, up, down, w0, w1) in enumerate(self.layers):
            _, u = ops.block_norm(None, h, pre_weight=w0)
            q, k, v = qkv(u).split([H * DK, HK * DK, HK * DK], -1)
            q = ops.cache_append(q, k, v, cache, H, positions, self.frequencies, SECTIONS, layer=i, slots=slots, places=places)
            o = ops.paged_attention(q, cache, H, layer=i, slots=slots, lengths=lengths)
            h, u = ops.block_norm(out(o), h, pre_weight=w1)
            h, _ = ops.block_norm(down(ops.geglu(up(u))), h, pre=False)
        return h


def reference(model, h, dtype, scales):
    """The same over a whole sequence [T, D] in 64 bits, rounded where the kernels store."""
    from katz_amd import ops

    r = lambda t: t.to(BF).to(F64)                       # noqa: E731
    c = lambda t: t.detach().cpu().to(F64)               # noqa: E731
    T = h.shape[0]
    lin = lambda layer, x: r(x @ c(ops.dequantize_w4(layer.packed_weight(), torch.float32)).t() + c(layer.bias))      # noqa: E731
    norm = lambda t, w: t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * c(w)       # noqa: E731
    angle = torch.arange(T, dtype=F64)[:, None] * model.frequencies.cpu()                  # (text: one position on all axes)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    causal = torch.arange(T)[:, None] >= torch.arange(T)

    def turn(x, heads):
        a, b = x.view(T, heads, DK).chunk(2, -1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    for i, (qkv, out, up, down, w0, w1) in enumerate(model.layers):
        q, k, v = lin(qkv, r(norm(h, w0))).split([H * DK, HK * DK, HK * DK], -1)
        q, k, v = r(turn(q, H)), turn(k, HK), v.view(T, HK, DK)
        if dtype is E4M3:
            s = [t[i].cpu().to(F64)[:, None] for t in scales]
            k, v = ((t / z).to(torch.float32).to(E4M3).to(F64) * z for t, z in zip((k, v), s))
        else:
            k, v = r(k), r(v)
        k, v = (t.repeat_interleave(H // HK, 1).transpose(0, 1) for t in (k, v))
        p = torch.softmax((q.transpose(0, 1) @ k.transpose(1, 2) * DK ** -0.5).masked_fill(~causal, -math.inf), -1)
        o = r((p @ v).transpose(0, 1).reshape(T, H * DK))
        h1 = h + lin(out, o)
        u, h = r(norm(h1, w1)), r(h1)
        a, b = lin(up, u).chunk(2, -1)
        h = r(h + lin(down, r(a * 0.5 * b * (1 + torch.erf(b / math.sqrt(2))))))
    return h


def new_cache(dtype, slots=6, pages=40, page=16, width=8):
    from katz_amd import ops

    scales = [torch.full((LAYERS, HK), z, device=DEV) for z in (0.03, 0.04)] if dtype is E4M3 else [None, None]
    return ops.PagedCache.empty(LAYERS, pages, page, HK, DK, slots, width, dtype, DEV, *scales)


def prompt_rows(lengths, slots):
    s = [s for s, n in zip(slots, lengths) for _ in range(n)]
    t = [i for n in lengths for i in range(n)]
    return dict(slots=int32(s), places=int32(t), lengths=int32([i + 1 for i in t])), int32([[i] * 3 for i in t])


@pytest.mark.parametrize("dtype", [BF, E4M3])
def test_prompts_tokens_forks_and_moves(dtype):
    from katz_amd import ops

    model, cache = Model(), new_cache(dtype)
    g = torch.Generator().manual_seed(3)
    slots, lengths, more = [4, 1], [37, 16], 20
    texts = {s: torch.randn(n + more, D, generator=g).to(BF) for s, n in zip(slots, lengths)}
    texts[0] = torch.cat((texts[4][:lengths[0]], torch.randn(more, D, generator=g).to(BF)))    # goes on from slot 4's prompt with tokens of its own
    counts = [0] * 6
    for s, n in zip(slots, lengths):
        counts[s] = n
    assert ops.cache_extend(cache, int32(counts)).item() == 0
    on, positions = prompt_rows(lengths, slots)
    h = torch.cat([texts[s][:n] for s, n in zip(slots, lengths)]).to(DEV)
    out = model(h, cache, positions, **on).split(lengths)
    got = {s: [o] for s, o in zip(slots, out)}
    assert ops.cache_reorder(cache, int32([4, 1, 2, 3, 4, 5])).item() == 0
    assert cache.table[0, :2].tolist() == cache.table[4, :2].tolist() and cache.table[0, 2] != cache.table[4, 2]
    got[0] = [got[4][0]]
    live, start = [0, 1, 4], {0: 37, 1: 16, 4: 37}
    for i in range(more):
        assert ops.cache_extend(cache, int32([int(s in live) for s in range(6)])).item() == 0
        if i == 7:
            ops.cache_compact(cache)
        if i == 9:                                       # slots 0 and 4 change places
            assert ops.cache_reorder(cache, int32([4, 1, 2, 3, 0, 5])).item() == 0
            got[0], got[4], texts[0], texts[4] = got[4], got[0], texts[4], texts[0]
        h = torch.stack([texts[s][start[s] + i] for s in live] + [torch.zeros(D, dtype=BF)]).to(DEV)        # and a row of no sequence
        places = cache.lengths[live] - 1
        positions = torch.cat((places, places[:1]))[:, None].repeat(1, 3).contiguous()
        o = model(h, cache, positions, slots=int32(live + [-1]), places=torch.cat((places, places[:1])))
        for s, row in zip(live, o):
            got[s].append(row[None])
    assert cache.lengths.tolist() == [57, 36, 0, 0, 57, 0]
    for s in live:
        close(torch.cat(got[s]), reference(model, texts[s].to(F64), dtype, (cache.k_scale, cache.v_scale)), f"slot {s}")


def test_captured_tokens_grow_their_sequences_at_every_replay():
    from katz_amd import ops

    model, slots, n = Model(1), 4, 30
    g = torch.Generator().manual_seed(4)
    prompts = [5, 16, 0, 31]
    tokens = [torch.randn(slots, D, generator=g).to(DEV, BF) for _ in range(n)]
    counts = [int32([1, 1, int(i > 9), int(i < 20)]) for i in range(n)]          # a slot that joins, one that ends

    def filled():
        cache = new_cache(BF, slots, 24, 16, 6)
        ops.cache_extend(cache, int32(prompts))
        on, positions = prompt_rows(prompts, range(slots))
        h = torch.randn(sum(prompts), D, generator=torch.Generator().manual_seed(5)).to(DEV, BF)
        model(h, cache, positions, **on)
        return cache

    def step(cache, h, count, where):
        ops.cache_extend(cache, count)
        positions = (cache.lengths - 1)[:, None].repeat(1, 3).contiguous()
        where.copy_(torch.where(count > 0, torch.arange(slots, device=DEV, dtype=torch.int32), -1))
        return model(h, cache, positions, slots=where, places=(cache.lengths - 1))

    eager, want, where = filled(), [], torch.zeros(slots, dtype=torch.int32, device=DEV)
    for h, c in zip(tokens, counts):
        want.append(step(eager, h, c, where).clone())
    runs = []
    for _ in range(2):                                   # two graphs, each with a cache and buffers of its own, replayed in turn
        cache, h, c, w = filled(), torch.zeros_like(tokens[0]), torch.zeros_like(counts[0]), torch.zeros_like(where)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(cache, h, c, w)                         # (no slot grows)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(cache, h, c, w)
        runs.append((graph, cache, h, c, out))
    other = filled()
    for i in range(n):
        for graph, cache, h, c, out in runs:
            h.copy_(tokens[i])
            c.copy_(counts[i])
            graph.replay()
            ops.cache_compact(other)                     # eager work between the replays
            ops.paged_attention(tokens[0], other, H)
            torch.cuda.synchronize()
            rows = counts[i] > 0
            assert torch.equal(out[rows], want[i][rows]), f"replay {i}"
    for _, cache, *_ in runs:
        assert torch.equal(cache.table, eager.table) and torch.equal(cache.lengths, eager.lengths) and torch.equal(cache.refs, eager.refs)
        assert cache.lengths.tolist() == [35, 46, 20, 51]


def test_captured_beams_change_places():
    from katz_amd import ops

    def filled():
        cache = new_cache(BF, 4, 20, 16, 5)
        ops.cache_extend(cache, int32([20, 33, 16, 7]))
        cache.k.normal_(generator=torch.Generator(DEV).manual_seed(1))
        cache.v.normal_(generator=torch.Generator(DEV).manual_seed(2))
        return cache

    moves = [[1, 1, 0, 3], [0, 0, 0, 0], [3, 2, 1, 0], [0, -1, 2, 2], [0, 0, 2, 3]]
    eager, cache, parents, counts = filled(), filled(), int32([0, 1, 2, 3]), int32([0, 0, 0, 0])
    graph = torch.cuda.CUDAGraph()
    ops.cache_reorder(cache, parents)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        lost = ops.cache_reorder(cache, parents)
        ops.cache_extend(cache, counts)
        used = ops.cache_compact(cache)
    for m in moves:
        ops.cache_reorder(eager, int32(m))
        ops.cache_extend(eager, int32([1, 0, 2, 16]))
        n = ops.cache_compact(eager)
        parents.copy_(int32(m))
        counts.copy_(int32([1, 0, 2, 16]))
        graph.replay()
        torch.cuda.synchronize()
        assert lost.item() == 0 and used.item() == n.item()
        for a, b in zip((cache.table, cache.lengths, cache.refs, cache.k, cache.v), (eager.table, eager.lengths, eager.refs, eager.k, eager.v)):
            assert torch.equal(a, b), m


def test_caches_on_two_streams_at_once():
    from katz_amd import ops

    g = torch.Generator().manual_seed(6)
    streams = [torch.cuda.Stream() for _ in range(2)]
    caches = [new_cache(BF, 8, 400, 16, 40) for _ in range(2)]
    rows = [torch.randn(8, (H + 2 * HK) * DK, generator=g).to(DEV, BF) for _ in range(2)]
    for cache in caches:
        ops.cache_extend(cache, int32([600, 1, 77, 300, 0, 16, 450, 33]))
        cache.k.normal_(generator=torch.Generator(DEV).manual_seed(3))
        cache.v.normal_(generator=torch.Generator(DEV).manual_seed(4))
    torch.cuda.synchronize()

    def steps(cache, x):
        out = []
        for i in range(6):
            ops.cache_extend(cache, int32([1] * 8))
            q = ops.cache_append(x[:, :H * DK], x[:, H * DK:(H + HK) * DK], x[:, (H + HK) * DK:], cache, H)
            out.append(ops.paged_attention(q, cache, H))
            if i == 3:
                ops.cache_reorder(cache, int32([0, 0, 2, 3, 3, 5, 6, 7]))
        return out

    got = []
    for s, cache, x in zip(streams, caches, rows):
        with torch.cuda.stream(s):
            got.append(steps(cache, x))
    torch.cuda.synchronize()
    for x, out in zip(rows, got):
        cache = new_cache(BF, 8, 400, 16, 40)
        ops.cache_extend(cache, int32([600, 1, 77, 300, 0, 16, 450, 33]))
        cache.k.normal_(generator=torch.Generator(DEV).manual_seed(3))
        cache.v.normal_(generator=torch.Generator(DEV).manual_seed(4))
        assert all(torch.equal(a, b) for a, b in zip(steps(cache, x), out))
