"""Attention over a paged cache where a type, a size or a number is at its edge, against plain implementations in 64 bits (tolerances as in test_gpu_paged_cache)."""
import pytest
import torch

from test_gpu_paged_cache import BF, DEV, E4M3, F64, FP16, FP32, HALF, TINY, U, Model, Pages, assert_within, attention_reference, gen, int32, randn, raw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, FP16])
def test_weights_stay_finite_where_scores_have_steps_of_16(dtype):
    """Scores of 2 * 10^8 in binary digits, each 128 tokens a step or two of 16 above the ones before: weights are those of a maximum that has seen them."""
    from katz_amd import ops

    n, d = 512, 64
    pages = Pages(46, [n], 16, 1, d, dtype, width=32)
    k = torch.zeros(n, d)
    k[:, 0], k[:, 1] = 32768, torch.arange(n) // 128 * 2.0 ** -8
    for t in range(n):
        pages.k[0, pages.table[0, t // 16], t % 16, 0] = k[t].to(dtype)
    pages.dev.k.copy_(pages.k)
    q = torch.zeros(1, d, dtype=dtype)
    q[0, :2] = 1
    got = ops.paged_attention(q.to(DEV), pages.dev, 1, scale=4096.0)
    assert torch.isfinite(got).all() and got.abs().max() <= pages.v[torch.isfinite(pages.v)].abs().max()


@pytest.mark.parametrize("dtype,cache", [(FP16, FP16), (FP16, E4M3), (BF, BF), (BF, E4M3)])
@pytest.mark.parametrize("gap", [10.0, 13.0, 15.0, 16.5, 19.0, 24.0])
@pytest.mark.parametrize("n,heads,kv,d", [(33, 1, 1, 64), (600, 4, 2, 80), (5000, 6, 1, 128), (300, 2, 2, 256)])
def test_weights_far_below_the_largest_count(dtype, cache, gap, n, heads, kv, d):
    """One token far above the rest has values of zero: what comes out are the weights of the rest, e^-gap of its own and about, each to its own last bits."""
    from katz_amd import ops

    g = gen(n + d)
    pages = Pages(40, [n], 16, kv, d, cache)
    k, v = torch.randn(n, kv, d, generator=g) * 0.25, (torch.randn(n, kv, d, generator=g).abs() * 100 + 50).clamp(max=440)
    k[:, :, 0], v[n // 3] = 0, 0
    k[n // 3], k[n // 3, :, 0] = 0, gap
    large = 64.0 if gap > 20 else 1.0                    # (so that fp16 shows them)
    for pool, x, scale in ((pages.k, k, pages.ks), (pages.v, v, pages.vs)):
        if scale is not None:
            scale[:] = 2.0 ** -4 if pool is pages.k else large
            x = x / scale[0, 0] if pool is pages.k else x
        elif pool is pages.v:
            x = x * large
        for t in range(n):
            pool[0, pages.table[0, t // 16], t % 16] = x[t].to(cache)
    for to, x in ((pages.dev.k, pages.k), (pages.dev.v, pages.v), (pages.dev.k_scale, pages.ks), (pages.dev.v_scale, pages.vs)):
        if x is not None:
            to.copy_(x)
    q = randn(g, 1, heads, d, dtype=FP32, std=d ** -0.5)
    q[..., 0] = 1
    q = q.view(1, heads * d).to(dtype)
    ref, off = attention_reference(q, pages, heads, [0], [n], scale=1.0)
    got = ops.paged_attention(q.to(DEV), pages.dev, heads, scale=1.0)
    assert_within(got.view(1, heads, d), ref, HALF[dtype] * ref.abs() + off + TINY[dtype], "weights far below the largest")


@pytest.mark.parametrize("dtype", [BF, FP16])
@pytest.mark.parametrize("n,d", [(40, 64), (700, 128), (2500, 256)])
def test_equal_weights_far_below_the_largest_have_no_error_in_common(dtype, n, d):
    """As above with the rest of the tokens alike: what their weights lack is lacking from the whole output.  Weights of 2^-12 .. 2^-35; the values are as large as
    fp16 has them.  Scores are one product of two exact numbers: off by the roundings of the factor, the product and the difference, 4 * 2^-24 of themselves, and the exponential's 2^-22; the
    sums as in the reference."""
    from katz_amd import ops

    g = gen(n)
    gaps = [8.0 + 0.37 * i for i in range(44)]
    pages = Pages(49, [n], 16, 1, d, dtype)
    v = (torch.rand(n, d, generator=g) + 1) * 20000
    v[5] = 0
    for t in range(n):
        e, at = pages.table[0, t // 16], t % 16
        pages.k[0, e, at, 0], pages.v[0, e, at, 0] = 0, v[t].to(dtype)
    pages.k[0, pages.table[0, 0], 5, 0, 0] = 1
    pages.dev.k.copy_(pages.k)
    pages.dev.v.copy_(pages.v)
    q = torch.zeros(len(gaps), d, dtype=dtype)
    q[:, 0] = torch.tensor(gaps).to(dtype)               # (the score of the fifth; the others have 0)
    slots = torch.zeros(len(gaps), dtype=torch.int32)
    ref, _ = attention_reference(q, pages, 1, slots, [n] * len(gaps), scale=1.0)
    got = ops.paged_attention(q.to(DEV), pages.dev, 1, slots=slots.to(DEV), scale=1.0)
    slack = 2 * (4 * U * max(gaps) + 2.0 ** -22) + 2 * (n / 4 + 64) * U
    half = torch.exp2(torch.floor(torch.log2(ref * (1 + slack)))) * HALF[dtype]          # (of the value's own step)
    assert_within(got.view(-1, 1, d), ref, half.clamp(min=TINY[dtype]) + slack * ref, "equal weights")


@pytest.mark.parametrize("dtype", [BF, FP16])
@pytest.mark.parametrize("d,turn", [(128, 32), (40, 12), (72, 0)])
def test_codes_are_those_of_the_quotient_in_32_bits(dtype, d, turn):
    """Scales as calibration makes them (the largest number / 448): multiples of sevenths lie on borders between codes, or a rounding of the scale beside them, and one quotient in a
    thousand goes to a border in 32 bits.  Values, dimensions beyond the pairs and keys at place 0, which turn by nothing: what (x.float() / scale).to(float8) gives."""
    from katz_amd import ops

    g, rows, kv, layers = gen(50 + d), 500, 6, 2
    x = randn(g, rows, (2 + 2) * kv * d, dtype=dtype, std=2.0)
    x[:, ::7] = (torch.randint(-200, 200, x[:, ::7].shape, generator=g) * 2.0 ** -6).to(dtype)
    x[0, 2 * kv * d::kv * d // 2], x[1, 2 * kv * d + 1::kv * d // 2] = float("inf"), -float("inf")
    most = (torch.randint(1, 64, (2, layers, kv), generator=g) * 2.0 ** -4).float()
    scales = [(m / 448).to(DEV) for m in most]
    k, v = (torch.zeros(layers, 63, 8, kv, d, device=DEV).to(E4M3) for _ in range(2))
    cache = ops.PagedCache(k, v, int32([list(range(63))]), int32([rows]), None, *scales)
    dev = x.to(DEV)
    freq = ops.rotary_frequencies(turn, device=DEV) if turn else None
    ops.cache_append(dev[:, :2 * kv * d], dev[:, 2 * kv * d:3 * kv * d], dev[:, 3 * kv * d:], cache, 2 * kv, torch.zeros(rows, 1, dtype=torch.int32, device=DEV) if turn else None, freq,
                     layer=1, slots=int32([0] * rows), places=int32(list(range(rows))))
    for pool, at, scale in ((cache.k, 2, scales[0]), (cache.v, 3, scales[1])):
        y = x[:, at * kv * d:(at + 1) * kv * d].to(F64).view(rows, kv, d)
        if at == 2:                                      # cosine 1, sine 0: an infinity leaves its pair's other half no number
            y[..., :turn], y[..., turn:2 * turn] = y[..., :turn] - 0 * y[..., turn:2 * turn], y[..., turn:2 * turn] + 0 * y[..., :turn]
        want = (y.float() / scale[1].cpu()[:, None]).clamp(-448, 448).to(E4M3)
        got = pool[1].cpu().view(-1, kv, d)[:rows]
        bad = (raw(got) != raw(want)) & ~torch.isnan(want.float())
        assert not bad.any() and torch.equal(torch.isnan(got.float()), torch.isnan(want.float())), f"{bad.sum()} of {got.numel()} codes"


@pytest.mark.parametrize("page,width,counts", [(1, 4, [2 ** 31 - 1] * 3), (1, 4, [2 ** 31 - 1, 5, 0]), (2, 3, [2 ** 31 - 1] * 4), (1, 1, [2 ** 31 - 1] * 1500), (16, 2, [2 ** 31 - 1, 1 << 30, 7])])
def test_pages_that_are_missing_are_counted_as_far_as_32_bits_go(page, width, counts):
    from katz_amd import ops

    slots = len(counts)
    cache = ops.PagedCache.empty(1, 9, page, 1, 8, slots, width, BF, DEV)
    got = ops.cache_extend(cache, int32(counts)).item()
    wanted = sum(-(-n // page) for n in counts)
    assert got == min(wanted - min(9, sum(min(-(-n // page), width) for n in counts)), 2 ** 31 - 1)
    assert cache.lengths.tolist() == [min(n, width * page) for n in counts]


def test_calls_without_rows_in_any_shape():
    from katz_amd import ops

    pages = Pages(45, [5], 16, 2, 64)
    freq = ops.rotary_frequencies(32, device=DEV)
    for shape in ((2, 0), (0, 3), (3, 0, 2), (3, 2, 0), (1, 0)):
        none = torch.zeros(*shape, 4 * 64, dtype=BF, device=DEV)
        q, k = ops.rotary(none, none[..., :128], 4, int32([]).view(0, 1), freq, kv_heads=2)
        assert q.shape == none.shape and k.shape == (*shape, 128)
        assert ops.cache_append(none, none[..., :128], none[..., :128], pages.dev, 4).shape == none.shape
        assert ops.paged_attention(none, pages.dev, 4).shape == none.shape


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("positions", ["near", "far", "fractions"])
def test_sine_and_cosine_of_32_bits_are_those_of_the_whole_angle(positions, pairs):
    """(1, 0) turned is the angle's cosine and sine themselves: a step of theirs (2^-24) and the rounding of what the angle's last bits add to them (2^-25)."""
    from katz_amd import ops

    g, rows, n = gen(61), 4000, 64
    pos = {"near": torch.arange(rows, dtype=torch.int32), "far": torch.randint(0, 1 << 24, (rows,), generator=g, dtype=torch.int32), "fractions": torch.rand(rows, generator=g) * 500}[positions]
    freq = ops.rotary_frequencies(n, device=DEV)
    x = torch.zeros(rows, n, 2) if pairs else torch.zeros(rows, 2, n)
    (x[..., 0] if pairs else x[:, 0])[:] = 1
    got, _ = ops.rotary(x.view(rows, 2 * n).to(DEV), x.view(rows, 2 * n).to(DEV), 1, pos[:, None].to(DEV), freq, pairs=pairs)
    got = got.cpu().view_as(x)
    c, s = (got[..., 0], got[..., 1]) if pairs else (got[:, 0], got[:, 1])
    angle = pos.to(F64)[:, None] * freq.cpu()
    far = 2.0 ** 24 * 2.0 ** -52                         # (an angle of up to 2^24 in 64 bits, in the reference and there)
    assert_within(c, angle.cos(), torch.full_like(angle, 1.5 * U + far), "cosine")
    assert_within(s, angle.sin(), torch.full_like(angle, 1.5 * U + far), "sine")
    assert (c[0] == 1).all() and (s[0] == 0).all() or positions != "near"


def test_scores_that_are_infinite():
    """All scores of a row minus infinity: nothing to attend to.  One that is plus infinity: no number."""
    from katz_amd import ops

    for dtype in (BF, FP16):
        pages = Pages(43, [200, 700, 40], 16, 1, 64, dtype)
        q = randn(gen(44), 3, 2 * 64, dtype=dtype)
        q[:, 3] = 1.0                                    # (of the first head)
        q[:, 64 + 3] = 0.0
        for s, n in enumerate([200, 700, 40]):
            for t in range(n):
                pages.k[0, pages.table[s, t // 16], t % 16, 0, 3] = -float("inf") if s < 2 else 0.5
        pages.k[0, pages.table[2, 1], 3, 0, 3] = float("inf")
        pages.dev.k.copy_(pages.k)
        got = ops.paged_attention(q.to(DEV), pages.dev, 2).view(3, 2, 64)
        assert (got[:2, 0] == 0).all() and torch.isnan(got[:2, 1]).all() and torch.isnan(got[2]).all()       # (0 times infinity is no number either)


LONG = [  # lengths, heads, kv, d, page, type, cache: more than 16 query heads on a key head, and heads that no kernel has the size of, where sequences are cut
    ([2000, 0, 900], 40, 2, 64, 16, BF, BF),
    ([2000, 0, 900], 34, 2, 72, 12, FP16, FP16),
    ([20000], 33, 1, 80, 24, FP16, E4M3),
    ([9000], 17, 1, 40, 5, BF, BF),
    ([30, 12000], 48, 1, 256, 32, BF, BF),
    ([6000, 1], 20, 1, 200, 16, BF, E4M3),
    ([700] * 9, 32, 1, 128, 16, FP16, FP16),
    ([9000], 7, 1, 96, 64, FP16, FP16),
]


@pytest.mark.parametrize("window", [0, 1000])
@pytest.mark.parametrize("case", LONG, ids=lambda c: f"{'-'.join(map(str, c[0][:3]))}-H{c[1]}of{c[2]}-{c[3]}-p{c[4]}-{str(c[5])[6:]}-{str(c[6])[6:]}")
def test_many_query_heads_on_a_key_head_over_long_sequences(case, window):
    from katz_amd import ops

    lengths, heads, kv, d, page, dtype, cache = case
    pages = Pages(41, lengths, page, kv, d, cache)
    q = randn(gen(42), len(lengths), heads * d, dtype=dtype)
    ref, off = attention_reference(q, pages, heads, range(len(lengths)), pages.held, window=window)
    got = ops.paged_attention(q.to(DEV), pages.dev, heads, window=window)
    assert_within(got.view(-1, heads, d), ref, HALF[dtype] * ref.abs() + off + TINY[dtype], "long")
    assert torch.equal(got, ops.paged_attention(q.to(DEV), pages.dev, heads, window=window))


def test_entries_and_lengths_outside_the_cache_change_nothing_else():
    """Entries that are no pages and lengths that no table holds, through every call: table, lengths, refs and the bits of the pages are those of the model."""
    from katz_amd import ops

    pages = Pages(22, [40, 40, 8, 61], 16, 2, 64, spare=3)
    big, most = 2 ** 31 - 1, pages.table.shape[1] * 16
    pages.table[0] = torch.tensor([big, -7, int(pages.table[0, 2]), -1, -1], dtype=torch.int32)
    pages.table[1, 2] = 999                              # the page not yet full of a sequence that is taken over
    pages.table[3, 1] = pages.refs.numel()
    lengths = torch.tensor([big, 40, -9, 61], dtype=torch.int32)
    pages.dev.table.copy_(pages.table)
    pages.dev.lengths.copy_(lengths)
    pages.held = lengths
    model = Model(pages)
    clamped = [min(max(n, 0), most) for n in model.held]

    def same(what):
        c = pages.dev
        assert c.table.tolist() == model.table and c.lengths.tolist() == model.held and c.refs.tolist() == model.refs, what
        assert torch.equal(raw(c.k), model.k) and torch.equal(raw(c.v), model.v), f"{what}: pages"

    counts = [5, 0, 100, -1]
    kept = [n for n, m in zip(model.held, counts)]
    model.held = clamped
    want = model.extend(counts)
    model.held = [n if m > 0 else k for n, m, k in zip(model.held, counts, kept)]        # (a slot that gets nothing keeps what it says)
    assert ops.cache_extend(pages.dev, int32(counts)).item() == want
    same("extended")
    assert model.compact() == ops.cache_compact(pages.dev).item()
    same("moved together")
    for parents in ([1, 1, 0, 3], [3, 9, 3, -1], [0, 0, 0, 0]):
        assert model.reorder(parents) == ops.cache_reorder(pages.dev, int32(parents)).item()
        same(f"reordered {parents}")
    assert model.compact() == ops.cache_compact(pages.dev).item()
    same("moved together again")


def test_a_long_sequence_among_many_rows():
    """Parts of one sequence by the hundred where the rows are too many for the join that goes by parts."""
    from katz_amd import ops

    rows, longest, d = 60, 20000, 64
    lengths = [0] * rows
    lengths[17], lengths[59] = longest, 130
    pages = Pages(47, lengths, 64, 1, d, spare=1)
    q = randn(gen(48), rows, 2 * d)
    ref, off = attention_reference(q, pages, 2, range(rows), pages.held)
    got = ops.paged_attention(q.to(DEV), pages.dev, 2)
    assert_within(got.view(rows, 2, d), ref, HALF[BF] * ref.abs() + off, "one long")
