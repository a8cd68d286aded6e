"""The operators of a block that answers token by token (norms around a block, weights in 4 bits, linear attention) against
plain implementations in 64 bits.

Tolerances.  A result that is rounded once is off by at most half a step of its type, finfo(t).eps / 2 relative to the value (HALF).  What 32-bit sums
add is bounded by the number of roundings a term passes times 2^-24 times the sum of the magnitudes that are added up, which the references
return beside the result; the numbers are derived at each test.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP16, FP32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
HALF = {t: torch.finfo(t).eps / 2 for t in (BF, FP16, FP32)}
DEV = "cuda:0"


def say(*a):
    print(*a, flush=True)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, std=1.0, dtype=BF):
    return (torch.randn(*shape, generator=g) * std).to(dtype)


def on(t):
    return None if t is None else t.to(DEV)


def assert_within(got, ref, bound, what):
    """|got - ref| <= bound elementwise (all on the CPU, 64 bits); NaN and infinities have to be where the reference has them."""
    got, ref = got.detach().to("cpu", F64), ref.to(F64)
    assert got.shape == ref.shape, f"{what}: {tuple(got.shape)} for {tuple(ref.shape)}"
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN in other places"
    assert torch.equal(got[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)]), f"{what}: infinities"
    over = ((got - ref).abs() - bound)[fine]
    assert over.numel() == 0 or over.max() <= 0, f"{what}: off by {(got - ref)[fine].abs().max():.3e}, {over.max():.3e} more than allowed"


# ------------------------------------------------------------------------------------------------ the norms around a block
def normed(t, kind, w, b, eps):
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    n = t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)
    n = n if w is None else n * w.to(F64)
    return n if b is None else n + b.to(F64)


def normed_magnitude(t, mag, kind, w, b, eps):
    """What the roundings of a norm of t are relative to, for an element: t's own terms `mag`, and for a layer norm those of the mean that is taken off
    (t - mean is off by 2^-24 of both however small it is), times what the norm multiplies with; the result itself; the bias."""
    c = t - t.mean(-1, keepdim=True) if kind == "layer" else t
    up = (mag + mag.mean(-1, keepdim=True)) / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    up = up if w is None else up * w.to(F64).abs()
    return up + normed(t, kind, w, b, eps).abs() + (0 if b is None else b.to(F64).abs())


def norm_reference(y, h, post, pw, pb, gate, rho, pre, qw, qb, kind, eps):
    """(h', magnitude of its terms, u, magnitude of u's terms)."""
    h = h.to(F64)
    if y is None:
        s, mag = h, h.abs()
    else:
        y = y.to(F64)
        n, a = (normed(y, kind, pw, pb, eps), normed_magnitude(y, y.abs(), kind, pw, pb, eps)) if post else (y, y.abs())
        if gate is not None:
            g = gate.to(F64)
            g = g[:, None] if gate.dim() == 2 and h.dim() == 3 and gate.shape != h.shape else g
            n, a = n * g, a * g.abs()
        s, mag = rho * h + n, (rho * h).abs() + a
    if not pre:
        return s, mag, None, None
    return s, mag, normed(s, kind, qw, qb, eps), normed_magnitude(s, mag, kind, qw, qb, eps)


# roundings in 32 bits that an element passes: a sum over at most 32768 elements held by 64 .. 1024 threads (32 in a chain at most, 10 in
# the tree), root, quotient, products: fewer than 64
NORM_SLOP = 64 * 2.0 ** -24

NORM_CASES = [
    # shape, kind, type, stream, post, pre, gate, affine, rho
    ((1, 1, 1280), "rms", BF, BF, True, True, "channel", "w", 1.0),
    ((2, 77, 640), "layer", BF, FP32, True, True, "sequence", "wb", 0.7),
    ((3, 5, 2050), "rms", BF, BF, True, True, "full", "w", -1.5),
    ((2, 3, 1), "layer", FP32, FP32, True, True, "none", "wb", 1.0),       # one element: zero variance
    ((2, 7, 33), "rms", FP16, FP16, False, True, "channel", "", 1.0),
    ((1, 9, 4097), "layer", FP16, FP32, True, False, "none", "w", 1.0),
    ((2, 2, 8192), "rms", FP32, FP32, True, True, "sequence", "wb", 0.5),
    ((1, 3, 9000), "layer", BF, FP32, True, True, "channel", "wb", 1.0),
    ((1, 2, 32768), "rms", BF, BF, True, True, "channel", "w", 1.0),
    ((1, 2, 20011), "layer", FP32, FP32, True, True, "full", "w", 1.0),
    ((515, 1000), "layer", BF, BF, True, True, "full", "wb", 1.0),
    ((5, 1, 512), "rms", BF, FP32, False, False, "sequence", "", 0.0),
    ((64,), "rms", BF, BF, True, True, "channel", "w", 1.0),
    ((4100, 1280), "layer", BF, FP32, True, True, "channel", "w", 1.0),     # a wave a row, stored past the caches
    ((4097, 1999), "rms", FP16, FP16, True, True, "none", "wb", 1.0),
    ((4096, 1400), "rms", BF, BF, True, False, "channel", "", 0.5),
]


@pytest.mark.parametrize("case", NORM_CASES, ids=lambda c: "x".join(map(str, c[0])) + f"-{c[1]}-{c[6]}")
def test_block_norm(case):
    from katz_amd import ops

    shape, kind, dt, st, post, pre, gate, affine, rho = case
    say("block_norm", case)
    g, D = gen(len(shape) * 1000 + shape[-1]), shape[-1]
    y, h = randn(g, *shape, std=2.0, dtype=dt) + 0.5, randn(g, *shape, dtype=st)
    gs = {"none": None, "channel": (D,), "sequence": (shape[0], D), "full": shape}[gate]
    gt = None if gs is None else randn(g, *gs, dtype=dt)
    pw, qw = (randn(g, D, dtype=dt) if "w" in affine else None for _ in range(2))
    pb, qb = (randn(g, D, dtype=dt) if "b" in affine else None for _ in range(2))
    if not post:
        pw = pb = None
    if not pre:
        qw = qb = None
    rh, mh, ru, mu = norm_reference(y, h, post, pw, pb, gt, rho, pre, qw, qb, kind, 1e-6)
    args = dict(post=post, post_weight=on(pw), post_bias=on(pb), gate=on(gt), residual_scale=rho, pre=pre, pre_weight=on(qw), pre_bias=on(qb), kind=kind)
    gh, gu = ops.block_norm(on(y), on(h), **args)
    assert gh.dtype == st and (gu is None) == (not pre)
    assert_within(gh, rh, HALF[st] * rh.abs() + NORM_SLOP * mh, "h'")
    if pre:
        assert gu.dtype == dt
        assert_within(gu, ru, HALF[dt] * ru.abs() + NORM_SLOP * mu, "u")
    # in place: the stream over itself, u over y
    y2, h2 = on(y), on(h)
    ops.block_norm(y2, h2, h_out=h2, out=y2 if pre else None, **args)
    assert torch.equal(h2, gh) and (not pre or torch.equal(y2, gu))


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("D", [24, 1280, 1283])
def test_block_norm_before_the_first_block(kind, D):
    from katz_amd import ops

    g = gen(D)
    h, w = randn(g, 3, 11, D, dtype=BF), randn(g, D)
    same, u = ops.block_norm(None, (hd := on(h)), pre_weight=on(w), kind=kind)
    assert same is hd and torch.equal(hd.cpu(), h)
    _, _, ru, mu = norm_reference(None, h, False, None, None, None, 1.0, True, w, None, kind, 1e-6)
    assert_within(u, ru, HALF[BF] * ru.abs() + NORM_SLOP * mu, "u")


def test_block_norm_of_unaligned_views_and_of_rows_that_are_no_numbers():
    from katz_amd import ops

    g = gen(3)
    flat = randn(g, 4 * 640 + 1)
    h, y = flat[1:].view(4, 640), randn(g, 4, 640)          # rows 2 bytes off every 16-byte border
    y[1, 5], y[2, 7] = float("inf"), float("nan")
    big = on(flat)
    gh, gu = ops.block_norm(on(y), big[1:].view(4, 640), post=True)
    rh, mh, ru, mu = norm_reference(y, h, True, None, None, None, 1.0, True, None, None, "rms", 1e-6)
    for r in (0, 3):
        assert_within(gh[r], rh[r], HALF[BF] * rh[r].abs() + NORM_SLOP * mh[r], "h'")
        assert_within(gu[r], ru[r], HALF[BF] * ru[r].abs() + NORM_SLOP * mu[r], "u")
    # a row with an infinity: that element is inf / inf, no number, and with it the next norm's row; the row's others keep the stream
    assert torch.isnan(gh[1, 5]) and torch.isnan(gu[1]).all() and torch.equal(gh[1, :5].cpu(), h[1, :5])
    assert torch.isnan(gh[2]).all() and torch.isnan(gu[2]).all()


# ------------------------------------------------------------------------------------------------ weights in 4 bits
def quantized(w, group, zeros):
    """(codes, scales, zero points) [N, K], [N, groups], [N, groups] by the formulas."""
    N, K = w.shape
    groups = -(-K // group)
    p = torch.zeros(N, groups * group, dtype=F64)
    p[:, :K] = w.to(F64)
    p = p.view(N, groups, group)
    if zeros:
        lo, hi = p.amin(-1).clamp(max=0), p.amax(-1).clamp(min=0)
        s = ((hi - lo).float() / torch.full_like(hi.float(), 15)).to(BF)
    else:
        s = (p.abs().amax(-1).float() / torch.full((N, groups), 7.0)).to(BF)
    step = s.to(F64)
    ok = step > 0
    z = torch.where(ok, (-lo / step).round().nan_to_num(0), 0.0).clamp(0, 15) if zeros else torch.full_like(step, 8)
    q = (torch.where(ok[..., None], (p / step[..., None]).round().nan_to_num(0, 0, 0), 0.0) + z[..., None]).clamp(0, 15)
    return q.view(N, -1)[:, :K].to(torch.uint8), s, z.to(torch.uint8)


def unpacked(w4):
    q = w4.q.cpu()
    return torch.stack((q & 15, q >> 4), -1).view(q.shape[0], -1)[:, :w4.in_features]


def values(codes, s, z, group):
    at = torch.arange(codes.shape[1]) // group
    return (codes.to(F64) - z.to(F64)[:, at]) * s.to(F64)[:, at]


def packed(codes, s, z, group, zeros):
    from katz_amd import ops

    N, K = codes.shape
    full = torch.zeros(N, -(-K // 32) * 32, dtype=torch.uint8)
    full[:, :K] = codes
    pad = -s.shape[1] % 4
    return ops.W4Weight(on(full[:, 0::2] | (full[:, 1::2] << 4)), on(torch.nn.functional.pad(s, (0, pad))),
                        on(torch.nn.functional.pad(z, (0, pad))) if zeros else None, K, group)


@pytest.mark.parametrize("dtype", [BF, FP16, FP32])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("N,K,group", [(1, 1, 32), (3, 31, 32), (5, 64, 64), (7, 65, 64), (16, 129, 128), (33, 1280, 64), (9, 2050, 32),
                                       (130, 96, 128), (2, 4095, 128)])
def test_quantize_w4(N, K, group, zeros, dtype):
    from katz_amd import ops

    say("quantize_w4", N, K, group, zeros, dtype)
    g = gen(N * 7 + K)
    w = randn(g, N, K, std=0.05, dtype=BF).to(dtype)        # 8 bits: quotients stay clear of halves in any precision, so codes are equal
    if N > 2:
        w[1] = 0                                            # a row of zeros
        w[2] = w[2].abs() + 0.01                            # all of one sign
    codes, s, z = quantized(w, group, zeros)
    got = ops.quantize_w4(on(w), group, zeros=zeros)
    assert torch.equal(got.scale[:, :got.groups].cpu(), s) and not got.scale[:, got.groups:].any()
    assert torch.equal(unpacked(got), codes)
    if zeros:
        assert torch.equal(got.zero[:, :got.groups].cpu(), z) and not got.zero[:, got.groups:].any()
    filled = torch.stack((got.q.cpu() & 15, got.q.cpu() >> 4), -1).view(N, -1)[:, K:]
    assert not filled.any()
    for out in (BF, FP16, FP32):
        v = values(codes, s, z, group)
        assert torch.equal(ops.dequantize_w4(got, out).cpu(), v.float().to(out))     # a product of 8 and 5 bits, rounded once
    if dtype == BF:    # a value is half a step off at most, and what the rounded scale cannot reach (7 of its halves of 2^-8, 15 with zero points)
        step = s.to(F64)[:, torch.arange(K) // group]
        assert ((values(codes, s, z, group) - w.to(F64)).abs() <= step * (1 + 15 * 2.0 ** -8)).all()


def test_quantize_w4_of_groups_that_are_no_numbers():
    from katz_amd import ops

    w = randn(gen(5), 4, 128, dtype=BF)
    w[0, 3], w[1, 70], w[2, 100] = float("nan"), float("inf"), -float("inf")
    for zeros in (False, True):
        got = ops.quantize_w4(on(w), 64, zeros=zeros)
        s = got.scale[:, :2].float().cpu()
        assert torch.isnan(s[0, 0]) and torch.isinf(s[1, 1]) and torch.isinf(s[2, 1])
        assert torch.isfinite(s[[0, 1, 2, 3, 3], [1, 0, 0, 0, 1]]).all()
        v = ops.dequantize_w4(got)
        assert torch.isnan(v[0, :64]).all() and torch.isnan(v[1, 64:]).any() and torch.isfinite(v[3]).all() and torch.isfinite(v[0, 64:]).all()


def linear_reference(x, codes, s, z, group, bias, a, b, c, res):
    """(y, what its 32-bit sums add up in magnitude: products with the numbers P + code and P + zero that the kernel multiplies)."""
    P = 128 if x.dtype == BF else 1024
    x, v = x.to(F64), values(codes, s, z, group)
    at = torch.arange(codes.shape[1]) // group
    y = x @ v.t()
    mag = x.abs() @ (s.to(F64).abs()[:, at] * 2 * (P + 15)).t()
    if a is not None:
        t = (x @ a.to(F64).t()) * c.to(F64)
        y = y + t @ b.to(F64).t()
        # the rank-R product may be multiplied in two pieces of the type: 2^-16 of it for bf16
        mag = mag + 2.0 ** 6 * ((x.abs() @ a.to(F64).abs().t()) * c.to(F64).abs()) @ b.to(F64).abs().t()
    for e in (bias, res):
        if e is not None:
            y, mag = y + e.to(F64), mag + e.to(F64).abs()
    return y, mag


# roundings a product passes: the tree of 32 and up to 8 steps of the matrix unit in a group, one product with the scale, then the chain of groups of one
# wave (at most 32 here) and of 8 waves, bias and residual
LINEAR_SLOP = 64 * 2.0 ** -24

LINEAR_CASES = [
    # M, N, K, group, zeros, R, bias, residual, type
    (1, 16, 64, 64, False, 0, False, False, BF),
    (1, 1, 1, 32, True, 0, True, True, BF),
    (2, 1280, 1280, 64, False, 0, True, False, BF),
    (1, 520, 2048, 128, True, 64, False, False, BF),
    (13, 259, 2050, 32, True, 32, True, True, BF),
    (16, 33, 129, 128, False, 96, False, True, BF),
    (17, 48, 255, 64, True, 0, False, False, FP16),
    (31, 100, 1000, 32, False, 128, True, True, FP16),
    (40, 17, 4097, 128, True, 32, False, False, BF),
    (64, 128, 512, 64, False, 64, True, False, BF),
    (65, 130, 640, 64, True, 96, True, True, BF),
    (77, 320, 768, 128, False, 0, False, False, FP16),
    (154, 640, 2048, 64, False, 96, True, False, BF),
    (300, 257, 333, 32, True, 32, True, True, BF),
    (129, 512, 1280, 128, True, 128, False, True, FP16),
    (616, 384, 1280, 64, False, 96, True, False, BF),
    (3, 5000, 1001, 64, True, 32, True, False, BF),        # rows of x on odd addresses, 313 tiles of columns
    (4, 8200, 3001, 32, False, 0, False, True, FP16),
    (9, 9000, 640, 128, True, 64, False, False, BF),
    (16, 6001, 385, 32, True, 0, True, False, BF),
    (2, 40, 20000, 128, True, 128, False, False, FP16),    # many blocks to a wave
    (30, 8300, 514, 64, True, 32, False, True, BF),
    (20, 5000, 1536, 128, False, 0, True, False, FP16),
    # few rows whose rank products begin in the same launch
    (16, 200, 1279, 64, False, 64, False, True, BF),
    (6, 700, 33, 32, True, 32, True, False, FP16),
    (1, 64, 1280, 64, False, 64, False, False, BF),
    (4, 8400, 1000, 128, True, 64, True, False, FP16),
    (12, 5000, 31, 32, False, 64, False, True, BF),
    (16, 9000, 640, 64, True, 32, False, False, FP16),
    (3, 40, 2560, 128, False, 32, True, True, BF),
    # many rows
    (130, 8200, 200, 64, False, 32, True, True, BF),
    (1100, 2050, 385, 32, True, 96, True, True, FP16),
    (1030, 1800, 1280, 128, True, 128, False, False, BF),
    (616, 4000, 640, 64, False, 0, True, False, BF),
    (200, 8209, 130, 128, False, 64, False, True, BF),
    (70, 16500, 64, 64, True, 0, True, False, FP16),
    (513, 3330, 1000, 32, False, 64, True, True, BF),
    (700, 4100, 1000, 32, False, 64, True, True, BF),
    (800, 5000, 1280, 128, True, 128, False, False, BF),
    (200, 1000, 96, 32, False, 0, False, True, BF),
]


@pytest.mark.parametrize("case", LINEAR_CASES, ids=lambda c: f"M{c[0]}N{c[1]}K{c[2]}g{c[3]}z{int(c[4])}r{c[5]}")
def test_w4_linear(case):
    from katz_amd import ops

    M, N, K, group, zeros, R, bias, residual, dt = case
    say("w4_linear", case)
    g = gen(M * 31 + N + K)
    groups = -(-K // group)
    codes = torch.randint(0, 16, (N, K), generator=g).to(torch.uint8)
    s = ((torch.rand(N, groups, generator=g) + 0.5) * K ** -0.5 / 4).to(BF)
    z = torch.randint(0, 16, (N, groups), generator=g).to(torch.uint8) if zeros else torch.full((N, groups), 8, dtype=torch.uint8)
    x = randn(g, M, K, dtype=dt)
    b = randn(g, N, dtype=dt) if bias else None
    res = randn(g, M, N, dtype=dt) if residual else None
    A = B = c = None
    if R:
        A, B, c = randn(g, R, K, std=0.05, dtype=dt), randn(g, N, R, std=0.05, dtype=dt), torch.rand(R, generator=g) + 0.5
    ref, mag = linear_reference(x, codes, s, z, group, b, A, B, c, res)
    w = packed(codes, s, z, group, zeros)
    y = ops.w4_linear(on(x), w, on(b), on(A), on(B), on(c), residual=on(res))
    assert y.dtype == dt
    assert_within(y, ref, HALF[dt] * ref.abs() + LINEAR_SLOP * mag, "y")
    # roundings to the type are spread over half a step; sums in 32 bits are far below
    assert y.numel() < 256 or (y.cpu().to(F64) - ref).norm() <= HALF[dt] * ref.norm()
    again = ops.w4_linear(on(x), w, on(b), on(A), on(B), on(c), residual=on(res), out=torch.full_like(y, float("nan")))
    assert torch.equal(again, y)
    # in place of its residual
    if res is not None:
        buf = on(res)
        assert torch.equal(ops.w4_linear(on(x), w, on(b), on(A), on(B), on(c), residual=buf, out=buf), y)


@pytest.mark.parametrize("M,R", [(3, 32), (16, 64), (5, 96), (40, 64)])
def test_w4_linear_of_operands_at_any_address(M, R):
    from katz_amd import ops

    g = gen(18)
    w = ops.quantize_w4(on(randn(g, 100, 640, std=0.05)), 64)
    x, A, B, c = randn(g, M, 640), randn(g, R, 640, std=0.05), randn(g, 100, R, std=0.05), torch.rand(R, generator=g)

    def moved(t, by):                                       # a contiguous copy `by` elements behind an allocation's start
        return torch.cat([torch.zeros(by, dtype=t.dtype), t.flatten()]).to(DEV)[by:].view(t.shape)

    y = ops.w4_linear(on(x), w, None, on(A), on(B), on(c))
    for dx, da, db in ((1, 0, 0), (0, 1, 1), (0, 3, 2), (5, 2, 0)):
        got = ops.w4_linear(moved(x, dx), w, None, moved(A, da), moved(B, db), on(c))
        bound = 2 * HALF[BF] * y.cpu().to(F64).abs() + LINEAR_SLOP * 64          # (blocks on other paths: sums in another order, magnitudes below 64)
        assert_within(got, y.cpu().to(F64), bound, f"moved by {dx}, {da}, {db}")


def test_w4_linear_reads_only_its_rows():
    """x, codes, scales and outputs lie in larger buffers of NaN and of marks: nothing outside is used or written."""
    from katz_amd import ops

    for M, N, K in ((3, 24, 100), (70, 40, 1000)):
        g = gen(M)
        w = ops.quantize_w4(on(randn(g, N, K, std=0.1)), 64, zeros=True)
        x = randn(g, M, K)
        want = ops.w4_linear(on(x), w)
        xs = torch.full((M * K + 2 * K,), float("nan"), dtype=BF, device=DEV)
        xs[K + 1:K + 1 + M * K] = on(x).flatten()
        ys = torch.full((M * N + 2 * N,), 7.0, dtype=BF, device=DEV)
        ops.w4_linear(xs[K + 1:K + 1 + M * K].view(M, K), w, out=ys[N + 1:N + 1 + M * N].view(M, N))
        assert torch.equal(ys[N + 1:N + 1 + M * N].view(M, N), want)
        assert (ys[:N + 1] == 7).all() and (ys[N + 1 + M * N:] == 7).all()


def test_w4_linear_does_not_use_what_rows_are_filled_up_with():
    """Behind the last code, scale and zero point of a row there may be anything."""
    from katz_amd import ops

    for M, N, K, group in ((2, 40, 300, 64), (20, 33, 650, 32), (700, 4100, 200, 128)):
        g = gen(K)
        w = ops.quantize_w4(on(randn(g, N, K, std=0.1)), group, zeros=True)
        x = on(randn(g, M, K))
        want, values_ = ops.w4_linear(x, w), ops.dequantize_w4(w)
        q, s, z = w.q.clone(), w.scale.clone(), w.zero.clone()
        q.view(N, -1)[:, (K + 1) // 2:] = 0xFF
        s[:, w.groups:], z[:, w.groups:] = float("nan"), 255
        other = ops.W4Weight(q, s, z, K, group)
        assert torch.equal(ops.w4_linear(x, other), want) and torch.equal(ops.dequantize_w4(other), values_)


def test_w4_linear_of_rows_that_are_no_numbers():
    from katz_amd import ops

    g = gen(8)
    w = ops.quantize_w4(on(randn(g, 64, 256, std=0.1)), 64)
    x = randn(g, 20, 256)
    clean = ops.w4_linear(on(x), w)
    x[3, 9], x[17, 200] = float("nan"), float("inf")
    y = ops.w4_linear(on(x), w)
    assert torch.isnan(y[3]).all() and torch.isnan(y[17]).all()
    keep = [i for i in range(20) if i not in (3, 17)]
    assert torch.equal(y[keep], clean[keep])
    w.scale[5, 1] = float("nan")
    y = ops.w4_linear(on(torch.ones(2, 256, dtype=BF)), w)
    assert torch.isnan(y[:, 5]).all() and torch.isfinite(y[:, :5]).all() and torch.isfinite(y[:, 6:]).all()


# ------------------------------------------------------------------------------------------------ linear attention
def attention_reference(q, k, v, H, Hk, g, scale, s0):
    """One sequence, [T, H * dk] ..: (o, magnitude, state, magnitude) by the recurrence."""
    T = q.shape[0]
    dk, dv = q.shape[1] // H, v.shape[1] // Hk
    q, k, v = q.to(F64).view(T, H, dk), k.to(F64).view(T, Hk, dk), v.to(F64).view(T, Hk, dv)
    k, v = k.repeat_interleave(H // Hk, 1), v.repeat_interleave(H // Hk, 1)
    d = torch.exp(g.to(F64))[:, None, None]
    S = torch.zeros(H, dk, dv, dtype=F64) if s0 is None else s0.to(F64)
    A = S.abs()
    o, m = torch.zeros(T, H, dv, dtype=F64), torch.zeros(T, H, dv, dtype=F64)
    for t in range(T):
        S = d * S + k[t][:, :, None] * v[t][:, None, :]
        A = d * A + (k[t][:, :, None] * v[t][:, None, :]).abs()
        o[t] = scale * (q[t][:, None, :] @ S)[:, 0]
        m[t] = abs(scale) * (q[t].abs()[:, None, :] @ A)[:, 0]
    return o.view(T, H * dv), m.view(T, H * dv), S, A


# scores and states as two pieces of 8 bits leave 2^-17 of a term, sums and powers in 32 bits far less
OUT_SLOP = 2.0 ** -16
# three pieces leave 2^-25; a term passes a product, the powers exp(g n) (|g n| 2^-24 of them, and they vanish where that is much) and one product and one sum
# a block: below 32 roundings for the blocks of these tests
STATE_SLOP = 2.0 ** -19

ATTENTION_CASES = [
    # lengths, packed, H, Hk, dk, dv, state
    ((1,), False, 1, 1, 64, 64, False),
    ((1, 1, 1), False, 4, 2, 128, 64, True),
    ((77, 77), False, 5, 5, 64, 64, False),
    ((64,), False, 3, 1, 64, 128, True),
    ((65,), False, 2, 2, 128, 128, True),
    ((128, 128), False, 2, 1, 64, 64, False),
    ((515,), False, 1, 1, 64, 64, True),
    ((300, 1, 0, 64, 129, 0), True, 4, 2, 64, 64, True),
    ((0, 5), True, 2, 2, 128, 192, False),
    ((0,), True, 1, 1, 64, 64, True),
    ((700, 63), True, 2, 1, 128, 64, True),
    ((16,) * 9, True, 40, 10, 64, 64, True),       # enough heads that no sequence is cut
    ((200,) * 3, False, 40, 10, 64, 576, False),
    ((700, 0, 63, 1, 0, 1290, 64, 128, 5), True, 2, 1, 64, 64, True),      # cut wherever sequences end
    ((0, 64, 700, 0), True, 2, 2, 128, 128, False),
    ((1100, 1100), False, 3, 1, 64, 192, True),
    ((2600,) + (10, 0, 3) * 101, True, 1, 1, 64, 64, True),                # more sequences than a workgroup has threads
]


@pytest.mark.parametrize("case", ATTENTION_CASES, ids=lambda c: f"{'-'.join(map(str, c[0][:9]))}-H{c[2]}of{c[3]}-{c[4]}x{c[5]}-{'packed' if c[1] else 'dense'}")
def test_linear_attention(case):
    from katz_amd import ops

    lengths, pack, H, Hk, dk, dv, state = case
    say("linear_attention", case)
    r = gen(sum(lengths) + H)
    B, rows = len(lengths), sum(lengths) + 5
    q, k, v = randn(r, rows, H * dk), randn(r, rows, Hk * dk), randn(r, rows, Hk * dv)
    g = -torch.exp2(torch.linspace(-8, 0, H)) if H > 1 else torch.tensor([-0.02])
    if H > 2:
        g[0], g[1] = 0.0, float("-inf")                    # no decay at all, and no memory
    s0 = torch.randn(B, H, dk, dv, generator=r) if state else None
    start = [sum(lengths[:i]) + 2 for i in range(B + 1)]   # two rows before the first sequence, three behind the last
    mark = torch.full((rows, H * dv), 9.0, dtype=BF)
    sd = on(s0)
    if pack:
        got, S = ops.linear_attention(on(q), on(k), on(v), H, on(g), kv_heads=Hk, state=sd, seg_start=torch.tensor(start, dtype=torch.int32, device=DEV),
                                      max_seg_rows=max(max(lengths), 1), out=on(mark))
        got = got.cpu()
        inside = torch.zeros(rows, dtype=torch.bool)
        inside[start[0]:start[-1]] = True
        assert (got[~inside] == 9).all()
    else:
        T = lengths[0]
        cut = [t[2:2 + B * T].reshape(B, T, -1) for t in (q, k, v)]
        got, S = ops.linear_attention(*map(on, cut), H, on(g), kv_heads=Hk, state=sd)
        got = torch.cat([mark[:2], got.cpu().reshape(B * T, -1)])
    assert S.dtype == FP32 and (sd is None or S is sd)
    for b, n in enumerate(lengths):
        at = slice(start[b], start[b] + n)
        o, m, rs, ms = attention_reference(q[at], k[at], v[at], H, Hk, g, dk ** -0.5, None if s0 is None else s0[b])
        assert_within(got[at], o, HALF[BF] * o.abs() + OUT_SLOP * m, f"o of sequence {b}")
        assert_within(S[b], rs, HALF[FP32] * rs.abs() + STATE_SLOP * ms, f"state of sequence {b}")


@pytest.mark.parametrize("B,H,Hk,dk,dv,pool", [(1, 1, 1, 64, 64, 0), (3, 8, 2, 128, 128, 0), (5, 4, 4, 64, 192, 9), (2, 20, 20, 64, 64, 0)])
def test_linear_attention_step(B, H, Hk, dk, dv, pool):
    from katz_amd import ops

    say("step", B, H, Hk, dk, dv, pool)
    r = gen(B + H)
    q, k, v = randn(r, B, H * dk), randn(r, B, Hk * dk), randn(r, B, Hk * dv)
    g = -torch.rand(H, generator=r)
    s0 = torch.randn(pool or B, H, dk, dv, generator=r)
    slots = torch.randperm(pool, generator=r)[:B].to(torch.int32) if pool else None
    if pool:
        slots[1], slots[3] = -1, pool                      # rows that are left out
    mark = torch.full((B, H * dv), 9.0, dtype=BF, device=DEV)
    sd = on(s0)
    got, S = ops.linear_attention_step(on(q), on(k), on(v), H, on(g), sd, kv_heads=Hk, slots=on(slots), out=mark)
    assert S is sd and got is mark
    seen = set()
    for b in range(B):
        at = b if slots is None else int(slots[b])
        if at < 0 or at >= (pool or B):
            assert (got[b] == 9).all()
            continue
        seen.add(at)
        o, m, rs, ms = attention_reference(q[b:b + 1], k[b:b + 1], v[b:b + 1], H, Hk, g, dk ** -0.5, s0[at])
        assert_within(got[b:b + 1], o, HALF[BF] * o.abs() + OUT_SLOP * m, "o")
        assert_within(S[at], rs, HALF[FP32] * rs.abs() + STATE_SLOP * ms, "state")
    for at in range(pool or B):
        assert at in seen or torch.equal(S[at].cpu(), s0[at])
    if pool:                                               # rows of a new output that are left out are zero
        new, _ = ops.linear_attention_step(on(q), on(k), on(v), H, on(g), on(s0), kv_heads=Hk, slots=on(slots))
        assert not new[1].any() and not new[3].any() and torch.equal(new[[0, 2, 4]], got[[0, 2, 4]])
    # into another pool: the first one stays
    other, keep = torch.full_like(sd, 5.0), sd.clone()
    ops.linear_attention_step(on(q), on(k), on(v), H, on(g), sd, kv_heads=Hk, slots=on(slots), state_out=other)
    assert torch.equal(sd, keep) and all((other[at] == 5).all() for at in range(pool or B) if at not in seen)


def test_linear_attention_takes_views_and_slots():
    """q, k and v as columns of one projection, outputs as columns of a wider tensor, sequences in slots of a pool."""
    from katz_amd import ops

    r = gen(11)
    B, T, H, d = 2, 150, 2, 64
    qkv = randn(r, B, T, 3 * H * d)
    g = torch.tensor([-0.3, -0.01])
    pool = torch.randn(4, H, d, d, generator=r)
    wide = torch.full((B, T, 2 * H * d), 9.0, dtype=BF, device=DEV)
    dq = on(qkv)
    pd = on(pool)
    o, S = ops.linear_attention(*dq.split(H * d, -1), H, on(g), scale=0.25, state=pd, slots=torch.tensor([3, 0], dtype=torch.int32, device=DEV),
                                out=wide[..., H * d:])
    assert (wide[..., :H * d] == 9).all() and torch.equal(S[1:3].cpu(), pool[1:3])
    for b, at in ((0, 3), (1, 0)):
        ro, m, rs, ms = attention_reference(*[t[b] for t in qkv.split(H * d, -1)], H, H, g, 0.25, pool[at])
        assert_within(o[b], ro, HALF[BF] * ro.abs() + OUT_SLOP * m, "o")
        assert_within(S[at], rs, HALF[FP32] * rs.abs() + STATE_SLOP * ms, "state")


def test_linear_attention_tables_outside_the_tensors_stay_inside():
    """Row tables that are no row tables (descending, negative, past the end) are cut to the rows there are."""
    from katz_amd import ops

    r = gen(12)
    rows, H, d = 100, 2, 64
    q, k, v = (on(randn(r, rows, H * d)) for _ in range(3))
    g = on(torch.tensor([-0.1, -0.2]))
    mark = torch.full((rows, H * d), 9.0, dtype=BF, device=DEV)
    table = torch.tensor([-5, 30, 20, 1 << 30], dtype=torch.int32, device=DEV)      # rows 0..30, none, 20..100
    o, S = ops.linear_attention(q, k, v, H, g, seg_start=table, max_seg_rows=80, out=mark)
    good = torch.tensor([0, 30], dtype=torch.int32, device=DEV)
    _, first = ops.linear_attention(q, k, v, H, g, seg_start=good, max_seg_rows=80)
    assert torch.equal(S[0], first[0]) and not S[1].any()
    lone = torch.tensor([20, 100], dtype=torch.int32, device=DEV)
    ol, last = ops.linear_attention(q, k, v, H, g, seg_start=lone, max_seg_rows=80)
    assert torch.equal(S[2], last[0]) and torch.equal(o[30:], ol[30:])


def test_linear_attention_does_not_read_rows_of_no_sequence():
    from katz_amd import ops

    r = gen(13)
    H, d, start = 2, 64, [3, 40, 40, 170]
    q, k, v = (on(randn(r, 180, H * d)) for _ in range(3))
    g = on(torch.tensor([-0.1, 0.0]))
    table = torch.tensor(start, dtype=torch.int32, device=DEV)
    o, S = ops.linear_attention(q, k, v, H, g, seg_start=table, max_seg_rows=130)
    assert not o[:3].any() and not o[170:].any()                       # a new output's rows of no sequence are zero
    for t in (q, k, v):
        t[:3] = t[170:] = float("nan")
    o2, S2 = ops.linear_attention(q, k, v, H, g, seg_start=table, max_seg_rows=130)
    assert torch.equal(o, o2) and torch.equal(S, S2) and torch.isfinite(S).all()


def test_empty_calls():
    from katz_amd import ops

    e = lambda *s, dtype=BF: torch.empty(*s, dtype=dtype, device=DEV)       # noqa: E731
    g = torch.zeros(2, device=DEV)
    o, S = ops.linear_attention(e(0, 5, 128), e(0, 5, 128), e(0, 5, 128), 2, g)
    assert o.shape == (0, 5, 128) and S.shape == (0, 2, 64, 64)
    o, S = ops.linear_attention(e(3, 0, 128), e(3, 0, 128), e(3, 0, 128), 2, g)
    assert o.shape == (3, 0, 128) and not S.any()
    o, S = ops.linear_attention_step(e(0, 128), e(0, 128), e(0, 128), 2, g, e(0, 2, 64, 64, dtype=FP32))
    assert o.shape == (0, 128)
    w = ops.quantize_w4(on(randn(gen(1), 8, 32)), 32)
    assert ops.w4_linear(e(0, 32), w).shape == (0, 8)
    h, u = ops.block_norm(e(0, 64), e(0, 64))
    assert h.shape == u.shape == (0, 64)


@pytest.mark.parametrize("T,H,dk,dv", [(200, 2, 64, 64), (200, 1, 128, 128), (1500, 1, 64, 128), (1500, 1, 128, 64)])
def test_linear_attention_does_not_depend_on_later_tokens(T, H, dk, dv):
    """What is no number in the keys or values of a token leaves the outputs of the tokens before it as they were; in a value it is seen in its column from
    there on."""
    from katz_amd import ops

    r = gen(14)
    q, k, v = randn(r, 1, T, H * dk), randn(r, 1, T, H * dk), randn(r, 1, T, H * dv)
    g = on(torch.tensor([-0.02, -0.3][:H]))
    clean, _ = ops.linear_attention(on(q), on(k), on(v), H, g)
    for at, col, bad in ((T - 130, 5, float("nan")), (T - 97, dv - 1, float("inf")), (T - 1, 17, float("-inf")), (0, 0, float("nan"))):
        v2 = v.clone()
        v2[0, at, col] = bad
        o, S = ops.linear_attention(on(q), on(k), on(v2), H, g)
        others = [c for c in range(H * dv) if c != col]
        assert torch.equal(o[:, :at], clean[:, :at]) and torch.equal(o[..., others], clean[..., others])
        assert not torch.isfinite(o[:, at:, col]).any() and not torch.isfinite(S[0, 0, :, col]).any()
    for at in (T - 130, T - 97, T - 1):
        k2 = k.clone()
        k2[0, at, :dk] = float("nan")
        o, _ = ops.linear_attention(on(q), on(k2), on(v), H, g)
        assert torch.equal(o[:, :at], clean[:, :at]) and torch.isnan(o[:, at:, :dv]).all()


def test_sequences_without_tokens_leave_pools_as_they_are():
    from katz_amd import ops

    e = lambda *s: torch.empty(*s, dtype=BF, device=DEV)                    # noqa: E731
    g = torch.zeros(2, device=DEV)
    r = gen(15)
    pool, other = (on(torch.randn(4, 2, 64, 64, generator=r)) for _ in range(2))
    keep = other.clone()
    slots = torch.tensor([2, -1, 9], dtype=torch.int32, device=DEV)
    ops.linear_attention(e(3, 0, 128), e(3, 0, 128), e(3, 0, 128), 2, g, state=pool, state_out=other, slots=slots)
    assert torch.equal(other[2], pool[2]) and torch.equal(other[[0, 1, 3]], keep[[0, 1, 3]])
    ops.linear_attention(e(3, 0, 128), e(3, 0, 128), e(3, 0, 128), 2, g, state_out=other, slots=slots)
    assert not other[2].any() and torch.equal(other[[0, 1, 3]], keep[[0, 1, 3]])
    ops.linear_attention(e(0, 4, 128), e(0, 4, 128), e(0, 4, 128), 2, g, state_out=other, slots=slots[:0])
    assert not other[2].any() and torch.equal(other[[0, 1, 3]], keep[[0, 1, 3]])


@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_w4_linear_of_rows_of_larger_weights(group, zeros):
    """Rows first .. last of a weight are a weight: a part of a linear's outputs."""
    from katz_amd import ops

    r = gen(16)
    w = ops.quantize_w4(on(randn(r, 71, 320, std=0.1)), group, zeros)
    for M in (3, 40):
        x = on(randn(r, M, 320))
        y = ops.w4_linear(x, w)
        for a, b in ((1, 71), (3, 20), (70, 71)):
            part = ops.W4Weight(w.q[a:b], w.scale[a:b], None if w.zero is None else w.zero[a:b], 320, group)
            assert torch.equal(ops.w4_linear(x, part), y[:, a:b])
            assert torch.equal(ops.dequantize_w4(part), ops.dequantize_w4(w)[a:b])


def test_linear_attention_of_cut_sequences_with_slots():
    """Sequences that are cut, of a pool, into another one or the same: slots that are named hold the states behind the last tokens (those of sequences without
    tokens as they were), the others stay; sequences without a slot are left out."""
    from katz_amd import ops

    r = gen(17)
    H, d, lengths, slots = 2, 64, (900, 77, 0, 640, 0, 200), (3, -1, 5, 0, 9, 6)
    start = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    q, k, v = (randn(r, start[-1], H * d) for _ in range(3))
    g = torch.tensor([-0.3, -0.004])
    pool = torch.randn(7, H, d, d, generator=r)
    args = dict(seg_start=torch.tensor(start, dtype=torch.int32, device=DEV), max_seg_rows=900, slots=torch.tensor(slots, dtype=torch.int32, device=DEV))
    src, dst = on(pool), torch.full((7, H, d, d), 8.0, device=DEV)
    o, S = ops.linear_attention(on(q), on(k), on(v), H, on(g), state=src, state_out=dst, **args)
    assert S is dst and torch.equal(src.cpu(), pool)
    o2, S2 = ops.linear_attention(on(q), on(k), on(v), H, on(g), state=src, **args)
    assert S2 is src and torch.equal(o, o2)
    for b, (n, at) in enumerate(zip(lengths, slots)):
        rows = slice(start[b], start[b] + n)
        if not 0 <= at < 7:
            assert not o[rows].any()
            continue
        ro, m, rs, ms = attention_reference(*[t[rows] for t in (q, k, v)], H, H, g, d ** -0.5, pool[at])
        assert_within(o[rows], ro, HALF[BF] * ro.abs() + OUT_SLOP * m, f"o of sequence {b}")
        for got in (S, S2):
            assert_within(got[at], rs, HALF[FP32] * rs.abs() + STATE_SLOP * ms, f"state of sequence {b}")
    others = [i for i in range(7) if i not in slots]
    assert (dst[others] == 8).all() and torch.equal(src[others].cpu(), pool[others])


def test_w4_linear_with_and_without_adapters_in_turn():
    """One kernel with more and with less LDS."""
    from katz_amd import ops

    g = gen(20)
    for N, K in ((9000, 640), (5000, 512), (100, 640)):
        w = ops.quantize_w4(on(randn(g, N, K, std=0.05)), 128, True)
        A, B, c = on(randn(g, 64, K, std=0.05)), on(randn(g, N, 64, std=0.05)), on(torch.rand(64, generator=g))
        for M in (2, 9):
            x = on(randn(g, M, K))
            plain = ops.w4_linear(x, w)
            none = ops.w4_linear(x, w, None, A, B, torch.zeros_like(c))
            some = ops.w4_linear(x, w, None, A, B, c)
            assert torch.equal(plain, none) and not torch.equal(plain, some) and torch.equal(ops.w4_linear(x, w), plain)


def test_a_captured_packed_prompt_takes_other_lengths():
    """A graph of one packed call with its table and slots in buffers: other lengths, sequences without tokens or without a slot at every replay."""
    from katz_amd import ops

    r = gen(19)
    rows, B, H, d = 1500, 4, 2, 64
    q, k, v = (on(randn(r, rows, H * d)) for _ in range(3))
    g = on(torch.tensor([-0.2, -0.003]))
    pool = on(torch.randn(5, H, d, d, generator=r))
    table, slots = torch.zeros(B + 1, dtype=torch.int32, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV)
    state, out = pool.clone(), torch.zeros(rows, H * d, dtype=BF, device=DEV)
    call = lambda s, o: ops.linear_attention(q, k, v, H, g, state=s, slots=slots, seg_start=table, max_seg_rows=rows, out=o)      # noqa: E731
    slots.copy_(torch.arange(B, dtype=torch.int32))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(state, out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(state, out)
    for starts, places in (((0, 1500, 1500, 1500, 1500), (0, 1, 2, 3)), ((0, 10, 700, 700, 1400), (4, 0, -1, 2)), ((5, 5, 5, 5, 6), (0, 1, 2, 3)),
                           ((0, 400, 800, 1200, 1499), (3, -1, 1, 7)), ((0, 1500, 1500, 1500, 1500), (1, 0, 2, 3))):
        table.copy_(torch.tensor(starts, dtype=torch.int32))
        slots.copy_(torch.tensor(places, dtype=torch.int32))
        state.copy_(pool)
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        s2, o2 = pool.clone(), torch.full_like(out, 3.0)
        call(s2, o2)
        assert torch.equal(out, o2) and torch.equal(state, s2), (starts, places)


@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 64), (128, 128)])
@pytest.mark.parametrize("T", [2, 64, 65, 130, 1500])
def test_linear_attention_multiplies_scores_states_and_values_of_24_bits(T, dk, dv):
    """Terms that cancel but for their last 8 of 24 bits: every sum and product below is a number of 24 bits, so the result is the difference itself, rounded once."""
    from katz_amd import ops

    say("24 bits", T, dk, dv)
    a = 171 / 128                                          # eight bits; three of them, 2^-8 apart, are 24 without a gap
    far = torch.zeros(1, device=DEV)                       # no decay, and a scale of 1: nothing else is rounded
    want = a * 2.0 ** -16
    # two scores of the last token, a (1 + 2^-8 + 2^-16) and a (1 + 2^-8), with values 1 and -1
    q, k, v = (torch.zeros(1, T, w, dtype=BF) for w in (dk, dk, dv))
    first = max(0, T - 2 - (T - 1) % 64 // 2)              # (in the last block, with the other one where it has two)
    q[0, -1, :3] = torch.tensor([1.0, 2.0 ** -8, 2.0 ** -16])
    k[0, first, :3], k[0, -1, :2] = a, a
    v[0, first, 3], v[0, -1, 3] = 1.0, -1.0
    if first // 64 == (T - 1) // 64:
        o, _ = ops.linear_attention(on(q), on(k), on(v), 1, far, scale=1.0)
        assert o[0, -1, 3].item() == torch.tensor(want).to(BF).item()
        assert not o[0, -1, :3].any() and not o[0, :-1, :3].any()
    # a state of two such rows, which the last token's query takes off one another
    s0 = torch.zeros(1, 1, dk, dv)
    s0[0, 0, 5, 7], s0[0, 0, 40, 7] = a * (1 + 2.0 ** -8 + 2.0 ** -16), a * (1 + 2.0 ** -8)
    q, k, v = (torch.zeros(1, T, w, dtype=BF) for w in (dk, dk, dv))
    q[0, -1, 5], q[0, -1, 40] = 1.0, -1.0
    o, S = ops.linear_attention(on(q), on(k), on(v), 1, far, scale=1.0, state=on(s0))
    assert o[0, -1, 7].item() == torch.tensor(want).to(BF).item() and torch.equal(S.cpu(), s0)


def test_linear_attention_of_cut_sequences_adds_decayed_values_of_24_bits():
    """In a chunk where no sequence ends, too: a decayed value of 24 bits, less what a later block's query sees of it in 16."""
    from katz_amd import ops

    T, d, end = 16384, 64, 134                             # (the third block of one sequence, far from its end)
    say("24 bits of decayed values")
    g = torch.tensor([-0.6931471805599453 / 64])           # half a block on
    lam = torch.exp(g.to(F64))
    w = lam ** (63 - torch.arange(64, dtype=F64))          # what the values of the first block are multiplied with
    rest = w - w.to(BF).to(F64)
    rest = (rest - rest.to(BF).to(F64)).abs() / w
    at = int(rest.argmax())                                # where two pieces of 8 bits would leave the most
    assert rest[at] > 2.0 ** -17.5
    q, k, v = (torch.zeros(1, T, d, dtype=BF) for _ in range(3))
    k[0, at, 9], v[0, at, 11], q[0, end, 9] = 1.0, 1.0, 1.0
    first = left = (lam ** (end - at)).item()
    for t in (end - 6, end - 4, end - 2):                  # three tokens of the query's block take it away but for its last bits
        power = (lam ** (end - t)).item()
        v[0, t, 11], k[0, t, 9] = left / power, -1.0
        left -= v[0, t, 11].item() * power
    o, _ = ops.linear_attention(on(q), on(k), on(v), 1, on(g), scale=1.0)
    # Of a term: three powers, of 2^-23 and of 2^-24 for their arguments below 1.5, four products, three sums, two times three pieces that leave 2^-25: 18 times
    # 2^-24 at most; of the second and third later token 2^-8 and less of that
    slop = 18 * 2.0 ** -24 * 2.02 * first
    assert abs(o[0, end, 11].item() - left) <= slop + HALF[BF] * abs(left), (o[0, end, 11].item(), left, slop, rest[at].item() * first)


@pytest.mark.parametrize("dtype", [BF, FP16])
@pytest.mark.parametrize("M,N,R", [(1, 48, 32), (20, 40, 96), (700, 4100, 32), (700, 4100, 64), (1030, 4608, 128)])
def test_w4_linear_keeps_rank_products_in_32_bits(M, N, R, dtype):
    """Two ranks whose products cancel but for the last 8 of 24 bits, over weights that are zero, for few rows and for many."""
    from katz_amd import ops

    say("rank products", M, N, R, dtype)
    K, a, b = 64, 171 / 128, 171 / 128 + (2.0 ** -10 if dtype is FP16 else 0)     # 8 bits, and 11 of them
    w = ops.W4Weight(torch.full((N, K // 2), 0x88, dtype=torch.uint8, device=DEV), torch.zeros(N, 4, dtype=BF, device=DEV), None, K, 64)
    x, A, B, c = torch.zeros(M, K, dtype=dtype), torch.zeros(R, K, dtype=dtype), torch.zeros(N, R, dtype=dtype), torch.zeros(R)
    x[:, 3], A[2, 3], A[R - 1, 3], B[:, 2], B[:, R - 1] = 1.0, 1.0, 1.0, b, -b
    c[2], c[R - 1] = a * (1 + 2.0 ** -8 + 2.0 ** -16), a * (1 + 2.0 ** -8)
    y = ops.w4_linear(on(x), w, None, on(A), on(B), on(c))
    want = a * 2.0 ** -16 * b
    # products of 24 and 11 bits and their sums: fewer than 8 roundings of 2^-24 of the terms (none where B has 8 bits: sums of 32 at most, of which the upper 24
    # cancel), then the type's, which is that of the numbers below the normal ones in fp16
    bound = 8 * 2.0 ** -24 * 2 * a * b + max(HALF[dtype] * want, 2.0 ** -25 if dtype is FP16 else 0)
    assert (y.cpu().to(F64) - want).abs().max() <= bound, ((y.cpu().to(F64) - want).abs().max().item(), bound, want)


@pytest.mark.parametrize("dtype", [BF, FP16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,N,K,group", [(2, 1280, 1280, 64), (16, 320, 4096, 128), (30, 640, 1024, 32), (616, 2000, 1280, 64), (616, 2000, 2048, 128)])
def test_w4_linear_of_activations_with_a_mean(M, N, K, group, zeros, dtype):
    """Sums of products with codes lose nothing to what the codes are carried in, also where x does not average out."""
    from katz_amd import ops

    say("activations with a mean", M, N, K, group, zeros, dtype)
    g = gen(M + K)
    groups = K // group
    codes = (torch.randn(N, K, generator=g) * 2.6 + 8).round().clamp(0, 15).to(torch.uint8)       # (weights without a mean)
    s = ((torch.rand(N, groups, generator=g) + 0.5) * K ** -0.5 / 4).to(BF)
    z = torch.randint(7, 10, (N, groups), generator=g).to(torch.uint8) if zeros else torch.full((N, groups), 8, dtype=torch.uint8)
    x = (torch.randn(M, K, generator=g) + 3).to(dtype)
    y = ops.w4_linear(on(x), packed(codes, s, z, group, zeros)).cpu().to(F64)
    v = values(codes, s, z, group)
    ref = x.to(F64) @ v.t()
    # The sums are of products with numbers of 31 at most (48 + 15 and 48 with zero points and many rows), codes and what is taken off them: a group's 2 * 4 steps of
    # the matrix unit with a tree of 32 in each (below 16 roundings in a row), a product, and the chains of groups and of waves, whose terms are the groups' results
    carried = (63 if zeros and M > 32 else 31) * 2.0
    mag = x.to(F64).abs() @ (s.to(F64).abs()[:, torch.arange(K) // group] * carried).t()
    slop = 16 * 2.0 ** -24 * mag + (K // group + 16) * 2.0 ** -24 * (x.to(F64).abs() @ v.abs().t())
    over = (y - ref).abs() - HALF[dtype] * ref.abs() - slop
    assert over.max() <= 0, over.max().item()
    # their errors are of either sign: all of them together are far below the type's rounding
    nearest = ref.to(dtype).to(F64)
    assert (y - ref).norm() <= 1.02 * (nearest - ref).norm(), ((y - ref).norm() / (nearest - ref).norm()).item()


@pytest.mark.parametrize("M,N", [(2, 40), (20, 40), (700, 4100)])
def test_zero_points_are_their_lower_four_bits(M, N):
    """For the values as for the linear, whatever the upper bits of their bytes hold."""
    from katz_amd import ops

    r = gen(21)
    w = ops.quantize_w4(on(randn(r, N, 200, std=0.1)), 64, zeros=True)
    x = on(randn(r, M, 200))
    other = ops.W4Weight(w.q, w.scale, w.zero | 0xB0, 200, 64)
    assert torch.equal(ops.dequantize_w4(other), ops.dequantize_w4(w)) and torch.equal(ops.w4_linear(x, other), ops.w4_linear(x, w))
