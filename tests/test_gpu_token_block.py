"""The operators of a block that answers token by token, together as a model runs them: norm, projections with weights in 4 bits and adapters,
linear attention, gate and residual, a gated feed-forward; over a prompt, token by token, captured, and on other streams."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F64 = torch.bfloat16, torch.float64
HALF = torch.finfo(BF).eps / 2
DEV = "cuda:0"
D, H, HK, DK, FF = 256, 4, 2, 64, 512


def linear(g, n, k, rank=0, zeros=False, group=64):
    from katz_amd.layers import LoRALinearW4

    src = torch.nn.Linear(k, n).to(BF)
    with torch.no_grad():
        src.weight.copy_(torch.randn(n, k, generator=g) * k ** -0.5)
        src.bias.copy_(torch.randn(n, generator=g) * 0.1)
    layer = LoRALinearW4.from_linear(src.to(DEV), group, zeros)
    if rank:
        layer.add_adapter("a", (torch.randn(rank, k, generator=g) * k ** -0.5).to(BF), (torch.randn(n, rank, generator=g) * 0.1).to(BF), weight=0.7)
        layer.set_active(["a"])
    return layer


class Block:
    """h -> h: attention and feed-forward, norms before and after each, a gate a channel."""

    def __init__(self, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.qkv = linear(g, (H + 2 * HK) * DK, D, rank=32)
        self.out = linear(g, D, H * DK, zeros=True, group=32)
        self.up, self.down = linear(g, 2 * FF, D, rank=16, group=128), linear(g, D, FF, zeros=True)
        vec = lambda std, mean: (torch.randn(D, generator=g) * std + mean).to(DEV, BF)      # noqa: E731
        self.w = [vec(0.1, 1.0) for _ in range(5)]
        self.gates = [vec(0.3, 0.5) for _ in range(2)]
        self.log_decay = torch.tensor([-0.5, -0.05, -0.002, 0.0], device=DEV)

    def __call__(self, h, state, ops, step=False, attend=None):
        """h [B,T,D] (a prompt) or [B,D] (one token); the state is advanced in place."""
        _, u = ops.block_norm(None, h, pre_weight=self.w[0])
        qkv = self.qkv(u)
        q, k, v = qkv.split([H * DK, HK * DK, HK * DK], -1)
        o, _ = (ops.linear_attention_step if step else ops.linear_attention)(q, k, v, H, self.log_decay, state=state, kv_heads=HK)
        h, u = ops.block_norm(self.out(o), h, post=True, post_weight=self.w[1], gate=self.gates[0], pre_weight=self.w[2])
        y = self.down(ops.geglu(self.up(u)))
        return ops.block_norm(y, h, post=True, post_weight=self.w[3], gate=self.gates[1], residual_scale=0.9, pre_weight=self.w[4])


def reference(block, h, state):
    """The same in 64 bits, rounded to bf16 where the kernels store: one sequence [T, D]; (h, u, state)."""
    r = lambda t: t.to(BF).to(F64)                       # noqa: E731
    c = lambda t: t.detach().cpu().to(F64)               # noqa: E731

    def lin(layer, x):
        from katz_amd import ops

        y = x @ c(ops.dequantize_w4(layer.packed_weight(), torch.float32)).t() + c(layer.bias)
        p = layer._packed
        return r(y if p is None else y + ((x @ c(p.a_cat).t()) * c(p.col_scale)) @ c(p.b_cat).t())

    def norm(t, w):
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * c(w)

    u = r(norm(h, block.w[0]))
    q, k, v = lin(block.qkv, u).split([H * DK, HK * DK, HK * DK], -1)
    d, S, o = torch.exp(c(block.log_decay))[:, None, None], state.clone(), []
    for t in range(h.shape[0]):
        kt, vt = (x[t].view(HK, DK).repeat_interleave(H // HK, 0) for x in (k, v))
        S = d * S + kt[:, :, None] * vt[:, None, :]
        o.append(((q[t].view(H, 1, DK) @ S)[:, 0] * DK ** -0.5).flatten())
    o = r(torch.stack(o))
    h1 = h + norm(lin(block.out, o), block.w[1]) * c(block.gates[0])
    u = r(norm(h1, block.w[2]))                           # (normed before the sum is rounded)
    h1 = r(h1)
    a, b = lin(block.up, u).chunk(2, -1)
    y = lin(block.down, r(a * 0.5 * b * (1 + torch.erf(b / math.sqrt(2)))))
    h2 = 0.9 * h1 + norm(y, block.w[3]) * c(block.gates[1])
    return r(h2), r(norm(h2, block.w[4])), S


def close(got, ref, what):
    """Norm of the difference over the norm.  The reference rounds where the kernels do, so what remains is sums in 32 bits and the few values that they
    carry over a border between two bf16 numbers, a step each: less than if every last value had been rounded twice, 2 * HALF."""
    got, ref = got.detach().cpu().to(F64), ref.to(F64)
    off = ((got - ref).norm() / ref.norm()).item()
    assert off <= 2 * HALF, f"{what}: {off:.2e}"


@pytest.mark.parametrize("T", [1, 70])
def test_a_block_over_a_prompt_and_then_token_by_token(T):
    from katz_amd import ops

    block, B, more = Block(), 2, 5
    g = torch.Generator().manual_seed(T)
    h = torch.randn(B, T + more, D, generator=g).to(BF)
    state = torch.randn(B, H, DK, DK, generator=g)
    sd = state.to(DEV)
    got, u = block(h[:, :T].contiguous().to(DEV), sd, ops)
    steps = [block(h[:, T + i].contiguous().to(DEV), sd, ops, step=True) for i in range(more)]
    got, u = torch.cat([got] + [s[0][:, None] for s in steps], 1), torch.cat([u] + [s[1][:, None] for s in steps], 1)
    for b in range(B):
        rh, ru, rs = reference(block, h[b].to(F64), state[b].to(F64))
        close(got[b], rh, "h")
        close(u[b], ru, "u")
        close(sd[b], rs, "state")


def test_a_captured_token_advances_its_state_at_every_replay():
    from katz_amd import ops

    block, B = Block(1), 3
    g = torch.Generator().manual_seed(9)
    tokens = [torch.randn(B, D, generator=g).to(DEV, BF) for _ in range(6)]
    state = torch.randn(B, H, DK, DK, generator=g).to(DEV)
    eager, want = state.clone(), []
    for t in tokens:
        want.append([x.clone() for x in block(t, eager, ops, step=True)])
    # two graphs, each with buffers and a state of its own, replayed in turn
    runs = []
    for _ in range(2):
        x, s = torch.zeros_like(tokens[0]), state.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block(x, s.clone(), ops, step=True)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block(x, s, ops, step=True)
        runs.append((graph, x, s, out))
    for i, t in enumerate(tokens):
        for graph, x, s, out in runs:
            x.copy_(t)
            graph.replay()
            block(tokens[0], state.clone(), ops, step=True)          # eager work between the replays
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[i][0]) and torch.equal(out[1], want[i][1]), f"replay {i}"
    assert all(torch.equal(s, eager) for _, _, s, _ in runs)


def test_a_captured_prompt_replays_the_same():
    from katz_amd import ops

    block = Block(2)
    g = torch.Generator().manual_seed(4)
    B, T = 1, 520                                                    # several segments
    h = torch.randn(B, T, D, generator=g).to(DEV, BF)
    zero = torch.zeros(B, H, DK, DK, device=DEV)
    want = block(h, zero.clone(), ops)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(h, zero.clone(), ops)
    torch.cuda.current_stream().wait_stream(side)
    x, s = torch.zeros_like(h), zero.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(x, s, ops)
    for i in range(3):
        x.copy_(h if i != 1 else -h)
        s.zero_()
        graph.replay()
        other = block(h.flip(1).contiguous(), zero.clone(), ops)
        torch.cuda.synchronize()
        ref = want if i != 1 else block((-h).contiguous(), zero.clone(), ops)
        assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1]), f"replay {i}"
        assert not torch.equal(other[0], out[0])


def test_blocks_on_two_streams_at_once():
    from katz_amd import ops

    blocks = [Block(3), Block(4)]
    g = torch.Generator().manual_seed(5)
    hs = [torch.randn(2, 300, D, generator=g).to(DEV, BF) for _ in blocks]
    zero = torch.zeros(2, H, DK, DK, device=DEV)
    want = [b(h, zero.clone(), ops)[0] for b, h in zip(blocks, hs)]
    streams = [torch.cuda.Stream() for _ in blocks]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(blocks[i](hs[i], zero.clone(), ops)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(t, want[i]) for i in range(2) for t in got[i])


def test_layer_with_adapters_follows_scales_and_fuses():
    from katz_amd import ops

    g = torch.Generator().manual_seed(6)
    layer = linear(g, 96, 128)
    x = torch.randn(5, 128, generator=g).to(DEV, BF)
    base = layer(x)
    ads = {n: ((torch.randn(r, 128, generator=g) * 0.1).to(BF), (torch.randn(96, r, generator=g) * 0.1).to(BF)) for n, r in (("a", 16), ("b", 80), ("c", 70))}
    for n, (down, up) in ads.items():
        layer.add_adapter(n, down, up, alpha=8.0)
    assert torch.equal(layer(x), base)                               # not active yet
    w = ops.dequantize_w4(layer.packed_weight(), torch.float32).cpu().to(F64)

    def want(scales):
        y = x.cpu().to(F64) @ w.t() + layer.bias.detach().cpu().to(F64)
        for n, s in scales.items():
            down, up = (t.to(F64) for t in ads[n])
            y = y + s * 8.0 / down.shape[0] * (x.cpu().to(F64) @ down.t()) @ up.t()
        return y

    layer.set_active(["a", "b"], [0.5, 1.0])
    close(layer(x), want({"a": 0.5, "b": 1.0}), "two adapters")
    pack = layer._packed
    layer.set_active(["a", "b"], [1.5, 0.25])
    assert layer._packed is pack                                     # the same buffers, other scales
    close(layer(x), want({"a": 1.5, "b": 0.25}), "other scales")
    layer.set_global_scale(0.5)
    close(layer(x), want({"a": 0.75, "b": 0.125}), "global scale")
    layer.set_global_scale(1.0)
    layer.set_active(["a", "b", "c"], [1.0, 1.0, 1.0])               # 166 rank columns: beyond one launch
    assert layer._packed.overflow
    close(layer(x), want({"a": 1.0, "b": 1.0, "c": 1.0}), "three adapters")
    layer.set_active(["a"], [1.0])
    at = layer.weight_q.data_ptr()
    layer.fuse(0.5)
    assert layer._packed is None and layer.weight_q.data_ptr() == at
    merged = (w + 0.25 * ads["a"][1].to(F64) @ ads["a"][0].to(F64)).float()
    again = ops.quantize_w4(merged.to(DEV), 64)
    codes = lambda q: torch.stack((q & 15, q >> 4)).int()            # noqa: E731
    assert (codes(layer.weight_q) - codes(again.q)).abs().max() <= 1                    # (sums of the products in another order)
    with pytest.raises(ValueError):
        layer.add_adapter("bad", ads["a"][0][:, :64], ads["a"][1])
    saved = layer.state_dict()
    from katz_amd.layers import LoRALinearW4
    other = LoRALinearW4(128, 96, device=DEV)
    other.load_state_dict(saved)
    assert torch.equal(other(x), layer(x))


def test_layer_with_adapters_converts_and_keeps_its_own_weights():
    """A layer of another type keeps the scales that its codes were chosen against; a LoRALinear that one was made from keeps its adapters' weights."""
    from katz_amd.layers import LoRALinear, LoRALinearW4

    g = torch.Generator().manual_seed(7)
    src = LoRALinear(128, 96, bias=True, device=DEV, dtype=BF)
    src.weight.data.copy_(torch.randn(96, 128, generator=g) * 0.05)
    src.bias.data.copy_(torch.randn(96, generator=g))
    src.add_adapter("a", (torch.randn(16, 128, generator=g) * 0.1).to(BF), (torch.randn(96, 16, generator=g) * 0.1).to(BF), weight=0.5)
    src.set_active(["a"])
    layer = LoRALinearW4.from_linear(src)
    layer.set_active(["a"], [1.0])
    assert src.adapters["a"].weight == 0.5 and layer.adapters["a"].weight == 1.0
    x = torch.randn(5, 128, generator=g).to(DEV, BF)
    y, scale = layer(x), layer.weight_scale.clone()
    layer.to(torch.float16)
    assert layer.dtype is torch.float16 and layer.weight_scale.dtype is BF and torch.equal(layer.weight_scale, scale)
    close(layer(x.half()), y.cpu().to(F64), "in fp16")
    layer.to(BF)
    assert torch.equal(layer(x), y)
    with pytest.raises(TypeError):
        layer.float()
    assert torch.equal(layer(x), y)
    assert torch.equal(layer.cpu().to(DEV)(x), y)


def test_names_that_were_fused_are_free_for_other_adapters():
    """A merged adapter is part of the weights: one that is added under its name, or the same one over weights that are loaded anew, applies."""
    from katz_amd import ops

    g = torch.Generator().manual_seed(8)
    layer = linear(g, 96, 128)
    x = torch.randn(5, 128, generator=g).to(DEV, BF)
    ads = [((torch.randn(16, 128, generator=g) * 0.1).to(BF), (torch.randn(96, 16, generator=g) * 0.1).to(BF)) for _ in range(2)]
    saved = {k: v.clone() for k, v in layer.state_dict().items()}

    def want(down, up):
        w = ops.dequantize_w4(layer.packed_weight(), torch.float32).cpu().to(F64)
        xd = x.cpu().to(F64)
        return xd @ w.t() + layer.bias.detach().cpu().to(F64) + (xd @ down.to(F64).t()) @ up.to(F64).t()

    def fused_first():
        layer.load_state_dict(saved)
        for n in list(layer.adapters):
            layer.delete_adapter(n)
        layer.add_adapter("a", *ads[0])
        layer.set_active(["a"])
        layer.fuse()
        layer.set_active(["a"])
        assert layer._packed is None                                 # (merged: not applied twice)

    fused_first()                                                    # deleted, and another one under its name
    layer.delete_adapter("a")
    layer.add_adapter("a", *ads[1])
    layer.set_active(["a"])
    close(layer(x), want(*ads[1]), "deleted and added")
    fused_first()                                                    # replaced while its name is active
    layer.add_adapter("a", *ads[1])
    close(layer(x), want(*ads[1]), "replaced")
    before = layer.weight_q.clone()
    layer.fuse()
    assert layer._packed is None and not torch.equal(layer.weight_q, before)
    fused_first()                                                    # the weights from before it was merged
    layer.load_state_dict(saved)
    close(layer(x), want(*ads[0]), "loaded anew")


@pytest.mark.parametrize("M", [1, 5, 40, 700])
@pytest.mark.parametrize("dtype,N,K,ranks", [(torch.float16, 96, 128, (64, 64, 16)), (BF, 1283, 2050, (96, 80)), (torch.float16, 4103, 70, (200,)), (BF, 4100, 640, (128, 128, 128, 5))])
def test_layer_with_more_rank_columns_than_one_pack(M, dtype, N, K, ranks):
    """Any type and size that the layer has, in one launch: no rounding between the packs."""
    from katz_amd import ops
    from katz_amd.layers import LoRALinearW4

    g = torch.Generator().manual_seed(M + N)
    layer = LoRALinearW4(K, N, group=32, zeros=True, device=DEV, dtype=dtype)
    layer._assign(ops.quantize_w4((torch.randn(N, K, generator=g) * K ** -0.5).to(DEV), 32, True))
    layer.bias.data.copy_(torch.randn(N, generator=g))
    x, res = (torch.randn(M, n, generator=g).to(dtype) for n in (K, N))
    xd = x.to(F64)
    w = ops.dequantize_w4(layer.packed_weight(), torch.float32).cpu().to(F64)
    parts = [xd @ w.t(), layer.bias.detach().cpu().to(F64), res.to(F64)]
    mag = [48 * 2 * xd.abs() @ w.abs().amax(1, keepdim=True).expand(N, K).t(), parts[1].abs(), parts[2].abs()]       # (codes are carried in numbers of 63 at most: 9 values' steps each)
    names = [f"a{i}" for i in range(len(ranks))]
    for i, (n, r) in enumerate(zip(names, ranks)):
        down, up = (torch.randn(r, K, generator=g) * K ** -0.5).to(dtype), (torch.randn(N, r, generator=g) * 0.1).to(dtype)
        layer.add_adapter(n, down, up, alpha=r * (i + 1) / 4)
        parts.append((i + 1) / 4 * (xd @ down.to(F64).t()) @ up.to(F64).t())
        mag.append((i + 1) / 4 * (xd.abs() @ down.to(F64).abs().t()) @ up.to(F64).abs().t())
    layer.set_active(names)
    assert layer._packed.wide
    # 64 roundings in 32 bits of a term at most: groups and waves, a rank's product and its sum
    half = torch.finfo(dtype).eps / 2
    for scale in (1.0, 0.5):
        layer.set_global_scale(scale)
        ref, slop = sum(parts[:3]) + scale * sum(parts[3:]), 64 * 2.0 ** -24 * (sum(mag[:3]) + scale * sum(mag[3:]))
        y = layer(x.to(DEV), residual=res.to(DEV)).cpu().to(F64)
        assert ((y - ref).abs() <= half * ref.abs() + slop).all()
    before, operands = layer(x.to(DEV)), layer._operands
    layer.set_global_scale(1.0)
    assert all(a is b for a, b in zip(layer._operands, operands)) or layer._operands[2].data_ptr() == operands[2].data_ptr()   # a captured graph stays valid
    assert not torch.equal(layer(x.to(DEV)), before)


@pytest.mark.parametrize("M,dtype", [(3, BF), (700, torch.float16)])
def test_a_captured_layer_of_many_rank_columns_follows_its_scales(M, dtype):
    """Packs that lie side by side are written to in place: replays take the scales that are set between them, beside eager calls on another stream."""
    from katz_amd import ops
    from katz_amd.layers import LoRALinearW4

    g = torch.Generator().manual_seed(M)
    layer = LoRALinearW4(200, 4100, device=DEV, dtype=dtype)
    layer._assign(ops.quantize_w4((torch.randn(4100, 200, generator=g) * 0.1).to(DEV), 64))
    for n, r in (("a", 100), ("b", 60), ("c", 9)):
        layer.add_adapter(n, (torch.randn(r, 200, generator=g) * 0.1).to(dtype), (torch.randn(4100, r, generator=g) * 0.1).to(dtype))
    layer.set_active(["a", "b", "c"], [1.0, 0.5, 2.0])
    x, other = (torch.randn(M, 200, generator=g).to(DEV, dtype) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x)
    torch.cuda.current_stream().wait_stream(side)
    graph, held = torch.cuda.CUDAGraph(), torch.zeros_like(x)
    with torch.cuda.graph(graph):
        y = layer(held)
    seen = []
    for weights in ([1.0, 0.5, 2.0], [0.0, 0.0, 1.0], [2.0, 1.0, 0.0], [1.0, 0.5, 2.0]):
        layer.set_active(["a", "b", "c"], weights)
        held.copy_(x)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            beside = layer(other)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, layer(x)) and torch.equal(beside, layer(other))
        seen.append(y.clone())
    assert torch.equal(seen[0], seen[3]) and not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])
