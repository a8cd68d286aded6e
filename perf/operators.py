"""The operators of a block that answers token by token, as cases that can be timed and whose outputs can be compared.

Five operators: weights quantised to 4 bits by groups, linears with such weights (with or without low-rank adapters), the
norms before and after a block with the gate and the residual between them, linear attention with a decay for each head
over whole prompts, and its form for single tokens.  Widths are those of SDXL's text side and transformer blocks
(640, 1280, 2048, 5120, 10240; 77 tokens a prompt; heads of 64) or generic ones.  Weights are random at the spread of the usual
initialisers, activations ~ N(0, 1), adapters ~ N(0, 0.02).
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
BF = torch.bfloat16
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CHUNK = 64   # tokens a block of the plain linear attention


def listed():
    return [
        # An adapter was merged into one attention projection, whose 4-bit form is made anew.
        dict(name="quantize_1280x1280", op="quantize", n=1280, k=1280, group=64, zeros=False),
        # The largest weight that is loaded in 16 bits and kept in 4, with zero points.
        dict(name="quantize_16384x8192_zeros", op="quantize", n=16384, k=8192, group=128, zeros=True),
        # The second linear of the time embedding of a guidance pair: the smallest call.
        dict(name="linear_2_rows_1280x1280", op="linear", rows=2, n=1280, k=1280, group=64, zeros=False, rank=0, bias=True,
             residual=False, dtype="bf16"),
        # One token through the largest weight, with an adapter of rank 64 beside it: the bytes of the weights bound it.
        dict(name="linear_1_row_16384x8192_rank64", op="linear", rows=1, n=16384, k=8192, group=128, zeros=True, rank=64, bias=False,
             residual=False, dtype="bf16"),
        # A few requests' tokens, no size a multiple of any tile, small groups, a residual.
        dict(name="linear_13_rows_1283x2050", op="linear", rows=13, n=1283, k=2050, group=32, zeros=True, rank=32, bias=True,
             residual=True, dtype="bf16"),
        # Eight prompts of 77 tokens through a feed-forward projection with two adapters (64 + 32).
        dict(name="linear_616_rows_10240x1280_rank96", op="linear", rows=616, n=10240, k=1280, group=64, zeros=False, rank=96, bias=True,
             residual=False, dtype="bf16"),
        # The end of a block and the beginning of the next for one token.
        dict(name="norm_1_row_1280", op="norm", batch=1, tokens=1, width=1280, kind="rms", post=True, pre=True, gate="channel",
             affine_bias=False, dtype="bf16", stream="bf16", residual_scale=1.0),
        # The same over the image tokens of a guidance pair at 832 x 1216, a gate for each image, a stream in 32 bits.
        dict(name="norm_2x3952_1280_stream32", op="norm", batch=2, tokens=3952, width=1280, kind="layer", post=True, pre=True,
             gate="sequence", affine_bias=True, dtype="bf16", stream="fp32", residual_scale=0.7),
        # The prompts of a guidance pair: two sequences of 77 tokens.
        dict(name="prompt_2x77_20_heads", op="prompt", lengths="77,77", packed=False, heads=20, kv_heads=20, dk=64, dv=64, state=False),
        # Requests of mixed lengths packed behind one another, each going on from its state; an empty one among them.
        dict(name="prompt_packed_16_heads_128", op="prompt", lengths="4096,77,0,1023,8192,1,640,2355", packed=True, heads=16, kv_heads=8,
             dk=128, dv=128, state=True),
        # One token of a guidance pair.
        dict(name="token_2_20_heads", op="token", batch=2, heads=20, kv_heads=20, dk=64, dv=64, slots=0),
        # One token each of 64 requests, whose states lie in a pool of 96.
        dict(name="token_64_32_heads_128", op="token", batch=64, heads=32, kv_heads=8, dk=128, dv=128, slots=96),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "norm", "prompt", "token"])
    if op == "quantize":
        n = _log_int(rng, 16, 16384)
        return dict(op=op, n=n, k=_log_int(rng, 33, min(8192 * 16384 // n, 16384)), group=rng.choice([32, 64, 128]),
                    zeros=rng.random() < 0.5)
    if op == "linear":
        n = _log_int(rng, 16, 16384)
        k = _log_int(rng, 64, 8192)
        if rng.random() < 0.7:
            n, k = -(-n // 8) * 8, -(-k // 64) * 64
        rows = _log_int(rng, 1, max(1, min(616, 616 * 10240 * 1280 // (n * k))))
        return dict(op=op, rows=rows, n=n, k=k, group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.5,
                    rank=rng.choice([0, 0, 32, 64, 96, 128]), bias=rng.random() < 0.5, residual=rng.random() < 0.4,
                    dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if op == "norm":
        width = _log_int(rng, 64, 8192)
        if rng.random() < 0.7:
            width = -(-width // 8) * 8
        batch = rng.choice([1, 2, 3, 8])
        tokens = _log_int(rng, 1, max(1, 2 * 3952 * 1280 // (batch * width)))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return dict(op=op, batch=batch, tokens=tokens, width=width, kind=rng.choice(["rms", "layer"]), post=rng.random() < 0.7,
                    pre=rng.random() < 0.9, gate=rng.choice(["none", "channel", "sequence", "full"]), affine_bias=rng.random() < 0.5,
                    dtype=dtype, stream=rng.choice([dtype, "fp32"]), residual_scale=rng.choice([1.0, 0.5, 1.3]))
    kv_heads = rng.choice([1, 2, 4, 5, 8, 10])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    dk, dv = rng.choice([64, 64, 128]), rng.choice([64, 64, 128])
    if op == "prompt":
        count = rng.choice([1, 1, 2, 3, 5, 9])
        longest = max(1, 16384 * 16 * 256 // (count * heads * (dk + dv)))
        packed = rng.random() < 0.5
        first = _log_int(rng, 1, min(longest, 8192))
        lengths = [first] + [rng.choice([0, 1, rng.randint(1, first), first]) if packed else first for _ in range(count - 1)]
        return dict(op=op, lengths=",".join(map(str, lengths)), packed=packed, heads=heads, kv_heads=kv_heads, dk=dk, dv=dv,
                    state=rng.random() < 0.5)
    batch = _log_int(rng, 1, max(1, min(256, 64 * 32 * 128 * 128 // (heads * dk * dv))))
    return dict(op=op, batch=batch, heads=heads, kv_heads=kv_heads, dk=dk, dv=dv, slots=rng.choice([0, batch + rng.randint(0, 40)]))


# ------------------------------------------------------------------------------------------ inputs
def _decays(heads):
    """log of the decay a token for each head: half-lives from a few tokens to thousands."""
    return -torch.exp2(-8.0 * torch.arange(1, heads + 1, device=DEV, dtype=torch.float64) / heads).float()


def _lengths(case):
    return [int(t) for t in case["lengths"].split(",")]


def _groups(case):
    return -(-case["k"] // case["group"])


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0, dtype=BF):
        return (torch.randn(*shape, generator=gen, device=DEV) * std).to(dtype)

    if case["op"] == "quantize":
        return dict(case, weight=normal(case["n"], case["k"], std=case["k"] ** -0.5))
    if case["op"] == "linear":
        n, k, dt, groups = case["n"], case["k"], TYPES[case["dtype"]], _groups(case)
        # a row of codes: two to a byte, the even one in the low half, filled up to a multiple of 32 of them;
        # a row of scales (and zero points): filled up to a multiple of 4
        spread = torch.randn(n, -(-k // 32) * 32, generator=gen, device=DEV).mul_(2.6).round_().add_(8).clamp_(0, 15).to(torch.uint8)
        spread[:, k:] = 0
        codes = spread[:, 0::2] | (spread[:, 1::2] << 4)
        scale = torch.zeros(n, -(-groups // 4) * 4, dtype=BF, device=DEV)
        scale[:, :groups] = (torch.rand(n, groups, generator=gen, device=DEV) + 0.5) * (k ** -0.5 / 2.6)
        zero = None
        if case["zeros"]:
            zero = torch.zeros_like(scale, dtype=torch.uint8)
            zero[:, :groups] = torch.randint(5, 12, (n, groups), generator=gen, device=DEV).to(torch.uint8)
        s = dict(case, x=normal(case["rows"], k, dtype=dt), codes=codes, scale=scale, zero=zero, b=None, res=None, a_cat=None, b_cat=None,
                 col_scale=None)
        if case["bias"]:
            s["b"] = normal(n, std=0.1, dtype=dt)
        if case["residual"]:
            s["res"] = normal(case["rows"], n, dtype=dt)
        if case["rank"]:
            s["a_cat"], s["b_cat"] = normal(case["rank"], k, std=0.02, dtype=dt), normal(n, case["rank"], std=0.02, dtype=dt)
            s["col_scale"] = torch.rand(case["rank"], generator=gen, device=DEV) + 0.5
        return s
    if case["op"] == "norm":
        B, T, D, dt = case["batch"], case["tokens"], case["width"], TYPES[case["dtype"]]
        shape = {"none": None, "channel": (D,), "sequence": (B, D), "full": (B, T, D)}[case["gate"]]
        s = dict(case, y=normal(B, T, D, std=2.0, dtype=dt), h=normal(B, T, D, dtype=TYPES[case["stream"]]),
                 g=None if shape is None else normal(*shape, std=0.5, dtype=dt))
        for side in ("post", "pre"):
            s[side + "_w"] = (normal(D, std=0.1, dtype=torch.float32) + 1).to(dt) if case[side] else None
            s[side + "_b"] = normal(D, std=0.1, dtype=dt) if case[side] and case["affine_bias"] else None
        return s
    H, Hk, dk, dv = case["heads"], case["kv_heads"], case["dk"], case["dv"]
    if case["op"] == "prompt":
        lengths = _lengths(case)
        lead = (sum(lengths) + 3,) if case["packed"] else (len(lengths), lengths[0])   # three rows behind the last packed sequence
        s = dict(case, longest=max(lengths), q=normal(*lead, H * dk), k=normal(*lead, Hk * dk), v=normal(*lead, Hk * dv), log_decay=_decays(H),
                 starts=None, s0=None, out=torch.zeros(*lead, H * dv, dtype=BF, device=DEV),
                 s1=torch.zeros(len(lengths), H, dk, dv, device=DEV))
        if case["packed"]:
            s["starts"] = torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device=DEV)
        if case["state"]:
            s["s0"] = normal(len(lengths), H, dk, dv, std=3.0, dtype=torch.float32)
        return s
    B = case["batch"]
    pool = case["slots"] or B
    slots = torch.randperm(pool, generator=gen, device=DEV)[:B].to(torch.int32) if case["slots"] else None
    return dict(case, q=normal(B, H * dk), k=normal(B, Hk * dk), v=normal(B, Hk * dv), log_decay=_decays(H), slot=slots,
                s0=normal(pool, H, dk, dv, std=3.0, dtype=torch.float32), s1=torch.zeros(pool, H, dk, dv, device=DEV))


# ------------------------------------------------------------------------------------------ the plain forms
def _plain_quantize(s):
    n, k, G, groups = s["n"], s["k"], s["group"], _groups(s)
    w = torch.nn.functional.pad(s["weight"].float(), (0, groups * G - k)).view(n, groups, G)
    if s["zeros"]:
        low, high = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        scale = ((high - low) / torch.full_like(high, 15)).to(BF)
    else:
        high = w.abs().amax(-1)
        scale = (high / torch.full_like(high, 7)).to(BF)
    step = scale.float()
    some = step > 0
    zero = torch.where(some, (-low / step).round(), 0).clamp(0, 15) if s["zeros"] else torch.full_like(step, 8)
    code = (torch.where(some[..., None], (w / step[..., None]).round(), 0) + zero[..., None]).clamp(0, 15)
    values = ((code - zero[..., None]) * step[..., None]).view(n, groups * G)[:, :k].to(BF)
    return [values, scale] + ([zero.to(torch.uint8)] if s["zeros"] else [])


def _plain_linear(s):
    n, k, G, groups = s["n"], s["k"], s["group"], _groups(s)
    code = torch.stack((s["codes"] & 15, s["codes"] >> 4), -1).view(n, -1)[:, :k]
    code = torch.nn.functional.pad(code, (0, groups * G - k)).view(n, groups, G).float()
    zero = 8.0 if s["zero"] is None else s["zero"][:, :groups, None].float()
    w = ((code - zero) * s["scale"][:, :groups, None].float()).view(n, groups * G)[:, :k]
    x = s["x"].float()
    y = x @ w.t()
    if s["rank"]:
        y += ((x @ s["a_cat"].float().t()) * s["col_scale"]) @ s["b_cat"].float().t()
    if s["b"] is not None:
        y += s["b"].float()
    if s["res"] is not None:
        y += s["res"].float()
    return y.to(s["x"].dtype)


def _plain_normed(t, kind, weight, bias, eps):
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps) * weight.float()
    return t if bias is None else t + bias.float()


def _plain_norm(s):
    y, h = s["y"].float(), s["h"].float()
    if s["post"]:
        y = _plain_normed(y, s["kind"], s["post_w"], s["post_b"], 1e-6)
    if s["g"] is not None:
        g = s["g"].float()
        y = y * (g[:, None] if s["gate"] == "sequence" else g)
    h = s["residual_scale"] * h + y
    return [h.to(s["h"].dtype)] + ([_plain_normed(h, s["kind"], s["pre_w"], s["pre_b"], 1e-6).to(s["y"].dtype)] if s["pre"] else [])


def _plain_prompt(s):
    H, Hk, dk, dv, longest = s["heads"], s["kv_heads"], s["dk"], s["dv"], s["longest"]
    if s["packed"]:   # the sequences side by side, filled up with zeros
        length = s["starts"][1:] - s["starts"][:-1]
        at = torch.arange(longest, device=DEV)
        there = at < length[:, None]
        row = torch.where(there, s["starts"][:-1, None] + at, 0).long()
        q, k, v = (s[n].float()[row] * there[..., None] for n in ("q", "k", "v"))
    else:
        length = torch.full((s["q"].shape[0],), longest, device=DEV)
        q, k, v = (s[n].float() for n in ("q", "k", "v"))
    B, n, full = q.shape[0], -(-longest // CHUNK), -(-longest // CHUNK) * CHUNK

    def heads(t, count):
        t = torch.nn.functional.pad(t, (0, 0, 0, full - longest)).view(B, full, count, -1).transpose(1, 2)
        return t.repeat_interleave(H // count, 1).reshape(B, H, n, CHUNK, -1)

    q, k, v = heads(q, H) * dk ** -0.5, heads(k, Hk), heads(v, Hk)
    g = s["log_decay"]
    i = torch.arange(CHUNK, device=DEV)
    between = torch.where(i[:, None] >= i, torch.exp(g[:, None, None] * (i[:, None] - i).clamp(min=0)), 0)
    out = (q @ k.transpose(-1, -2).contiguous() * between[:, None]) @ v
    gain = (k * torch.exp(g[:, None] * (CHUNK - 1 - i))[:, None, :, None]).transpose(-1, -2).contiguous() @ v
    c = torch.arange(n, device=DEV)
    carry = torch.where(c[:, None] > c, torch.exp(g[:, None, None] * CHUNK * (c[:, None] - 1 - c).clamp(min=0)), 0)
    before = (carry @ gain.view(B, H, n, dk * dv)).view(B, H, n, dk, dv)
    if s["s0"] is not None:
        before = before + torch.exp(g[:, None] * CHUNK * c)[:, :, None, None] * s["s0"][:, :, None]
    out = out + (q * torch.exp(g[:, None] * (i + 1))[:, None, :, None]) @ before
    out = out.view(B, H, full, dv)[:, :, :longest].transpose(1, 2).reshape(B, longest, H * dv).to(BF)
    if s["packed"]:
        whole = torch.zeros_like(s["out"])
        whole[row[there]] = out[there]
        out = whole
    left = length[:, None] - 1 - torch.arange(full, device=DEV)   # tokens from each to the end of its sequence
    weight = torch.where(left[:, None] >= 0, torch.exp(g[:, None] * left[:, None].clamp(min=0)), 0)
    state = (k.view(B, H, full, dk) * weight[..., None]).transpose(-1, -2).contiguous() @ v.view(B, H, full, dv)
    if s["s0"] is not None:
        state = state + torch.exp(g * length[:, None])[..., None, None] * s["s0"]
    return [out, state]


def _plain_token(s):
    B, H, Hk, dk, dv = s["batch"], s["heads"], s["kv_heads"], s["dk"], s["dv"]
    q = s["q"].float().view(B, H, dk) * dk ** -0.5
    k = s["k"].float().view(B, Hk, dk).repeat_interleave(H // Hk, 1)
    v = s["v"].float().view(B, Hk, dv).repeat_interleave(H // Hk, 1)
    old = s["s0"] if s["slot"] is None else s["s0"][s["slot"].long()]
    new = torch.exp(s["log_decay"])[:, None, None] * old + k[..., None] * v[..., None, :]
    out = (q[..., None] * new).sum(-2).reshape(B, H * dv).to(BF)
    if s["slot"] is not None:
        pool = torch.zeros_like(s["s1"])
        pool[s["slot"].long()] = new
        new = pool
    return [out, new]


def run(state):
    s = state
    if own:
        from katz_amd import ops

        if s["op"] == "quantize":
            w = ops.quantize_w4(s["weight"], s["group"], zeros=s["zeros"])
            return [ops.dequantize_w4(w), w.scale[:, :w.groups]] + ([w.zero[:, :w.groups]] if s["zeros"] else [])
        if s["op"] == "linear":
            w = ops.W4Weight(s["codes"], s["scale"], s["zero"], s["k"], s["group"])
            return ops.w4_linear(s["x"], w, s["b"], s["a_cat"], s["b_cat"], s["col_scale"], residual=s["res"])
        if s["op"] == "norm":
            h, u = ops.block_norm(s["y"], s["h"], post=s["post"], post_weight=s["post_w"], post_bias=s["post_b"], gate=s["g"],
                                  residual_scale=s["residual_scale"], pre=s["pre"], pre_weight=s["pre_w"], pre_bias=s["pre_b"],
                                  kind=s["kind"], eps=1e-6)
            return [h, u] if s["pre"] else [h]
        if s["op"] == "prompt":
            return list(ops.linear_attention(s["q"], s["k"], s["v"], s["heads"], s["log_decay"], kv_heads=s["kv_heads"], state=s["s0"],
                                             state_out=s["s1"], seg_start=s["starts"], max_seg_rows=s["longest"], out=s["out"]))
        return list(ops.linear_attention_step(s["q"], s["k"], s["v"], s["heads"], s["log_decay"], s["s0"], kv_heads=s["kv_heads"],
                                              state_out=s["s1"], slots=s["slot"]))
    return {"quantize": _plain_quantize, "linear": _plain_linear, "norm": _plain_norm, "prompt": _plain_prompt,
            "token": _plain_token}[s["op"]](s)


# ------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "quantize":
        G, groups = case["group"], _groups(case)
        values, scales, zeros = [], [], []
        for rows in s["weight"].split(2048):
            w = torch.zeros(rows.shape[0], groups * G, dtype=f, device=DEV)
            w[:, :case["k"]] = rows
            w = w.view(-1, groups, G)
            top, bottom = w.max(-1)[0], w.min(-1)[0]
            span = torch.clamp(top, min=0) - torch.clamp(bottom, max=0) if case["zeros"] else torch.maximum(top, -bottom)
            scale = (span / (15 if case["zeros"] else 7)).to(BF).to(f)
            zero = torch.round(-torch.clamp(bottom, max=0) / scale) if case["zeros"] else torch.full_like(scale, 8)
            code = torch.clamp(torch.round(w / scale[..., None]) + zero[..., None], 0, 15)
            values.append(((code - zero[..., None]) * scale[..., None]).flatten(1)[:, :case["k"]])
            scales.append(scale)
            zeros.append(zero.to(torch.uint8))
        return [torch.cat(values), torch.cat(scales)] + ([torch.cat(zeros)] if case["zeros"] else [])
    if case["op"] == "linear":
        x = s["x"].to(f)
        parts = []
        for r in range(0, case["n"], 2048):
            codes = s["codes"][r:r + 2048]
            w = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=f, device=DEV)
            w[:, 0::2], w[:, 1::2] = codes % 16, codes // 16
            column = torch.arange(case["k"], device=DEV) // case["group"]
            zero = 8 if s["zero"] is None else s["zero"][r:r + 2048, column].to(f)
            parts.append(x @ ((w[:, :case["k"]] - zero) * s["scale"][r:r + 2048, column].to(f)).t().contiguous())
        y = torch.cat(parts, 1)
        if case["rank"]:
            y = y + ((x @ s["a_cat"].to(f).t().contiguous()) * s["col_scale"].to(f)) @ s["b_cat"].to(f).t().contiguous()
        for extra in ("b", "res"):
            if s[extra] is not None:
                y = y + s[extra].to(f)
        return y
    if case["op"] == "norm":
        def normed(t, side):
            m = t.mean(-1, keepdim=True) if case["kind"] == "layer" else torch.zeros_like(t[..., :1])
            t = (t - m) / torch.sqrt(((t - m) ** 2).mean(-1, keepdim=True) + 1e-6) * s[side + "_w"].to(f)
            return t if s[side + "_b"] is None else t + s[side + "_b"].to(f)

        y, h = s["y"].to(f), s["h"].to(f)
        y = normed(y, "post") if case["post"] else y
        if case["gate"] != "none":
            y = y * (s["g"].to(f).unsqueeze(1) if case["gate"] == "sequence" else s["g"].to(f))
        h = h * case["residual_scale"] + y
        return [h, normed(h, "pre")] if case["pre"] else [h]
    H, Hk, dk, dv = case["heads"], case["kv_heads"], case["dk"], case["dv"]
    decay = torch.exp(s["log_decay"].to(f))[:, None, None]
    share = torch.arange(H, device=DEV) // (H // Hk)
    if case["op"] == "prompt":
        lengths = _lengths(case)
        q, k, v = (s[n].reshape(-1, c, d) for n, c, d in (("q", H, dk), ("k", Hk, dk), ("v", Hk, dv)))
        first = torch.tensor([sum(lengths[:i]) for i in range(len(lengths))], device=DEV)
        S = torch.zeros(len(lengths), H, dk, dv, dtype=f, device=DEV) if s["s0"] is None else s["s0"].to(f)
        out = torch.zeros(q.shape[0], H, dv, dtype=f, device=DEV)
        for t in range(max(lengths)):
            here = torch.tensor([b for b, n in enumerate(lengths) if n > t])
            if t == 0 or here.numel() != live.numel():
                live = here
                on = here.to(DEV)
            row = first[on] + t
            new = decay * S[on] + k[row][:, share].to(f)[..., None] * v[row][:, share].to(f)[..., None, :]
            S[on] = new
            out[row] = (q[row].to(f)[..., None, :] @ new)[..., 0, :] * dk ** -0.5
        return [out.view(s["out"].shape), S]
    old = s["s0"].to(f) if s["slot"] is None else s["s0"][s["slot"].long()].to(f)
    q, k, v = (s[n].to(f).view(case["batch"], -1, d) for n, d in (("q", dk), ("k", dk), ("v", dv)))
    new = decay * old + torch.einsum("bhi,bhj->bhij", k[:, share], v[:, share])
    out = torch.einsum("bhi,bhij->bhj", q, new) * dk ** -0.5
    if s["slot"] is not None:
        pool = torch.zeros(s["s0"].shape, dtype=f, device=DEV)
        pool[s["slot"].long()] = new
        new = pool
    return [out.flatten(1), new]


def work(case):
    if case["op"] == "quantize":   # the weights read, the codes and the values that they stand for written
        cells, marks = case["n"] * case["k"], case["n"] * _groups(case) * (3 if case["zeros"] else 2)
        return {"bytes": 4.5 * cells + marks, "flops": 4.0 * cells}
    if case["op"] == "linear":
        M, n, k, r = case["rows"], case["n"], case["k"], case["rank"]
        nbytes = n * k / 2 + n * _groups(case) * (3 if case["zeros"] else 2) + 2 * M * (k + n) + 2 * r * (k + n) + 4 * r
        nbytes += (2 * n if case["bias"] else 0) + (2 * M * n if case["residual"] else 0)
        return {"bytes": nbytes, "flops": 2.0 * M * n * k + 2.0 * M * r * (k + n)}
    if case["op"] == "norm":
        size = {"bf16": 2, "fp16": 2, "fp32": 4}
        e, cells = size[case["dtype"]], case["batch"] * case["tokens"] * case["width"]
        gate = {"none": 0, "channel": case["width"], "sequence": case["batch"] * case["width"], "full": cells}[case["gate"]]
        return {"bytes": cells * (e + 2 * size[case["stream"]] + (e if case["pre"] else 0)) + e * gate, "flops": 12.0 * cells}
    H, Hk, dk, dv = case["heads"], case["kv_heads"], case["dk"], case["dv"]
    if case["op"] == "prompt":
        lengths = _lengths(case)
        rows = sum(lengths)
        return {"bytes": 2 * rows * (H * (dk + dv) + Hk * (dk + dv)) + 4 * len(lengths) * H * dk * dv * (2 if case["state"] else 1),
                "flops": rows * H * 4.0 * dk * dv}
    B = case["batch"]
    return {"bytes": 2 * B * (H * (dk + dv) + Hk * (dk + dv)) + 8 * B * H * dk * dv, "flops": B * H * 5.0 * dk * dv}
