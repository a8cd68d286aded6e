"""Attention over a paged cache (rotary positions, appends, single tokens, what keeps the pages) against plain implementations in 64 bits.

Tolerances.  A result that is rounded once is off by at most half a step of its type, finfo(t).eps / 2 relative to the value (HALF); what 32-bit
arithmetic adds is bounded by the roundings a term passes times 2^-24 times the magnitudes that are added up, derived at each reference.  Rows of the caches that no
token lies in, pages that nobody holds and rows behind an end are NaN, unless a test says otherwise.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP16, FP32, F64, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float64, torch.float8_e4m3fn
HALF = {t: torch.finfo(t).eps / 2 for t in (BF, FP16, FP32)}
TINY = {BF: 0.0, FP16: 2.0 ** -25, FP32: 0.0}       # half a step of fp16's smallest numbers
DEV = "cuda:0"
NAN = float("nan")
U = 2.0 ** -24


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=BF, std=1.0):
    return (torch.randn(*shape, generator=g) * std).to(dtype)


def raw(t):
    """Its bits, to be compared where there are NaN."""
    return t.detach().cpu().contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def assert_within(got, ref, bound, what):
    got, ref = got.detach().to("cpu", F64), ref.to(F64)
    assert got.shape == ref.shape, f"{what}: {tuple(got.shape)} for {tuple(ref.shape)}"
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN in other places"
    fine = torch.isfinite(ref)
    assert torch.equal(got[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)]), f"{what}: infinities"
    over = ((got - ref).abs() - bound)[fine]
    assert over.numel() == 0 or over.max() <= 0, f"{what}: off by {(got - ref)[fine].abs().max():.3e}, {over.max():.3e} more than allowed"


# ------------------------------------------------------------------------------------------------ rotary positions
def turned(x, heads, positions, freq, sections, pairs):
    """(rows of x turned, what roundings are relative to), [rows, heads, d] in 64 bits.  Sine and cosine are those of an angle that is off by pi 2^-24 (turns
    rounded to 32 bits) and off by two steps themselves; product and sum add two roundings: under 9 * 2^-24 * (|a| + |b|) in all."""
    x = x.to(F64).reshape(-1, heads, x.shape[-1] // heads).clone()
    mag, n = torch.zeros_like(x), sum(sections)
    axis = [a for a, m in enumerate(sections) for _ in range(m)]
    for j in range(n):
        i, k = (2 * j, 2 * j + 1) if pairs else (j, j + n)
        angle = positions[:, axis[j]].to(F64) * float(freq[j])
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        a, b = x[..., i].clone(), x[..., k].clone()
        x[..., i], x[..., k] = a * c - b * s, b * c + a * s
        mag[..., i] = mag[..., k] = a.abs() + b.abs()
    return x, 9 * U * mag


@pytest.mark.parametrize("dtype", [BF, FP16, FP32])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("rows,heads,kv,d,sections", [(1, 1, 1, 8, (4,)), (2, 20, 20, 64, (8, 12, 12)), (77, 4, 2, 80, (16, 8)), (5, 3, 1, 128, (16, 24, 24)), (33, 6, 2, 70, (3, 5, 2, 7)),
                                                      (4100, 5, 1, 64, (32,)), (3, 2, 1, 256, (0, 64, 0)), (9, 2, 2, 33, (0,)), (2, 1, 1, 1024, (512,)), (2, 1, 1, 2, (1,))])
def test_rotary(rows, heads, kv, d, sections, pairs, dtype):
    from katz_amd import ops

    g = gen(rows + d)
    q, k = randn(g, rows, heads * d, dtype=dtype), randn(g, rows, kv * d, dtype=dtype)
    pos = torch.randint(0, 100000, (rows, len(sections)), generator=g, dtype=torch.int32)
    freq = ops.rotary_frequencies(sum(sections), device=DEV)
    got = ops.rotary(q.to(DEV), k.to(DEV), heads, pos.to(DEV), freq, sections, kv_heads=kv, pairs=pairs)
    for t, h, out in ((q, heads, got[0]), (k, kv, got[1])):
        ref, more = turned(t, h, pos, freq.cpu(), sections, pairs)
        assert out.dtype is dtype
        assert_within(out.view(rows, h, d), ref, HALF[dtype] * ref.abs() + more + TINY[dtype], "rotary")


@pytest.mark.parametrize("d,sections", [(64, (8, 12, 12)), (72, (9, 11))])
def test_rotary_of_views_in_place_and_by_other_positions(d, sections):
    from katz_amd import ops

    g, heads, kv, B, T = gen(3), 4, 2, 3, 10
    qkv = randn(g, B, T, (heads + 2 * kv) * d)
    freq = ops.rotary_frequencies(sum(sections), 500.0, sections, DEV)
    assert freq.dtype is F64 and freq.shape == (sum(sections),) and float(freq[sections[0]]) == 1.0
    dev = qkv.to(DEV)
    q, k = dev[..., :heads * d], dev[..., heads * d:(heads + kv) * d]
    for pos, f in ((torch.randint(0, 1 << 40, (B * T, len(sections)), generator=g), freq), (torch.rand(B * T, len(sections), generator=g) * 1000, freq.float()),
                   (torch.randint(-500, 500, (B, T, len(sections)), generator=g, dtype=torch.int32), freq)):
        out = torch.full((B, T, heads * d + 8), 7.0, dtype=BF, device=DEV)
        got, got_k = ops.rotary(q, k, heads, pos.to(DEV), f, sections, kv_heads=kv, out=out[..., :heads * d])
        p = pos.reshape(B * T, -1).to(F64)
        ref, more = turned(qkv[..., :heads * d].reshape(B * T, -1), heads, p, f.cpu(), sections, False)
        # a position of 2^40 times a frequency that 64 bits hold to 2^-53 leaves the angle 2^-12 off (twice: here and in the reference)
        more = more + (p.abs().max() * 2.0 ** -51) * 2 * torch.ones_like(more) * qkv.to(F64).abs().max()
        assert_within(got.reshape(B * T, heads, d), ref, HALF[BF] * ref.abs() + more, "views")
        assert (out[..., heads * d:] == 7).all()
        ref, m = turned(qkv[..., heads * d:(heads + kv) * d].reshape(B * T, -1), kv, p, f.cpu(), sections, False)
        assert_within(got_k.reshape(B * T, kv, d), ref, HALF[BF] * ref.abs() + m + more[0, 0, 0], "views")
    apart = ops.rotary(q, k, heads, pos.to(DEV), freq, sections, kv_heads=kv, pairs=True)
    rest = dev[..., (heads + kv) * d:].clone()
    same = ops.rotary(q, k, heads, pos.to(DEV), freq, sections, kv_heads=kv, pairs=True, out=q, k_out=k)
    assert same[0] is q and torch.equal(q, apart[0]) and torch.equal(k, apart[1]) and torch.equal(dev[..., (heads + kv) * d:], rest)
    odd = torch.zeros(T * heads * d + 1, dtype=BF, device=DEV)[1:].view(T, heads * d)          # two bytes off any alignment
    odd.copy_(apart[0][0])
    got = ops.rotary(odd, odd.clone(), heads, pos[0].to(DEV), freq, sections)
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], ops.rotary(odd.clone(), odd.clone(), heads, pos[0].to(DEV), freq, sections)[0])


def test_rotary_of_numbers_that_are_none_stays_in_their_pairs():
    from katz_amd import ops

    x = torch.ones(4, 64, device=DEV)
    x[1, 3], x[2, 40] = NAN, float("inf")
    pos = torch.tensor([[0], [5], [7], [2 ** 31 - 1]], dtype=torch.int32, device=DEV)
    y, _ = ops.rotary(x, x, 1, pos, ops.rotary_frequencies(32, device=DEV))
    bad = ~torch.isfinite(y.cpu())
    assert bad.nonzero().tolist() == [[1, 3], [1, 35], [2, 8], [2, 40]]
    assert torch.equal(y[0], x[0])                       # position 0 turns nothing


# ------------------------------------------------------------------------------------------------ caches
class Pages:
    """A cache on the CPU as the tests know it, and on the GPU."""

    def __init__(self, seed, held, page, kv, d, dtype=BF, layers=1, spare=2, width=None, fill=NAN, heads_first=False):
        from katz_amd import ops

        g = gen(seed)
        need = [-(-n // page) for n in held]
        count = sum(need) + spare
        width = width or max(need + [1]) + 1
        order = torch.randperm(count, generator=g).tolist()
        self.table = torch.full((len(held), width), -1, dtype=torch.int32)
        self.refs = torch.zeros(count, dtype=torch.int32)
        self.held = torch.tensor(held, dtype=torch.int32)
        self.page = page
        k, v = (torch.full((layers, count, page, kv, d), fill, dtype=FP32) for _ in range(2))
        for s, n in enumerate(held):
            for i in range(need[s]):
                e = order.pop()
                self.table[s, i], self.refs[e] = e, 1
                m = min(page, n - i * page)
                for t in (k, v):
                    t[:, e, :m] = torch.randn(layers, m, kv, d, generator=g)
        self.ks = self.vs = None
        if dtype is E4M3:
            self.ks, self.vs = (torch.rand(layers, kv, generator=g) * 0.02 + 0.02 for _ in range(2))
            k, v = k * 16, v * 16
        self.k, self.v = k.to(dtype), v.to(dtype)
        up = lambda t: t if t is None else t.to(DEV)      # noqa: E731
        place = (lambda t: up(t).permute(0, 1, 3, 2, 4).contiguous().permute(0, 1, 3, 2, 4)) if heads_first else up
        self.dev = ops.PagedCache(place(self.k), place(self.v), up(self.table), up(self.held), up(self.refs), up(self.ks), up(self.vs))

    def tokens(self, slot, n, layer, which):
        """[n, kv, d] in 64 bits; a token without a page is None's: rows of NaN, listed in the second."""
        pool, scale = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        t = torch.arange(n)
        e = self.table[slot, t // self.page].long()
        there = (e >= 0) & (e < pool.shape[1])
        x = pool[layer].to(F64)[torch.where(there, e, 0), t % self.page]
        return (x if scale is None else x * scale[layer].to(F64)[:, None]), there


def attention_reference(q, pages, heads, slots, lengths, layer=0, window=0, scale=None):
    """([rows, heads, d] in 64 bits, how far 32 bits may be off).  A score sums d products that are exact (d roundings, the factors' three more), so with
    E = (d + 4) 2^-24 scale max_t sum |q k| + (2^-24 max |x| + 2^-22 for the subtraction and the exponential) every weight is off by a factor e^(+-E), numerator and denominator;
    the sums over n tokens are four of n / 4 and their join: n / 4 + 64 roundings each.  Both relative to sum p |v| / sum p."""
    kv, d = pages.k.shape[3], pages.k.shape[4]
    scale = d ** -0.5 if scale is None else scale
    out, off = torch.zeros(q.shape[0], heads, d, dtype=F64), torch.zeros(q.shape[0], heads, d, dtype=F64)
    for r in range(q.shape[0]):
        n = max(0, min(int(lengths[r]), pages.table.shape[1] * pages.page))
        k, there = pages.tokens(int(slots[r]), n, layer, "k")
        v, _ = pages.tokens(int(slots[r]), n, layer, "v")
        low = max(0, n - window) if window else 0
        there[:low] = False
        k, v = k[there], v[there]
        if not len(k):
            continue
        for h in range(heads):
            one, key, value = q[r].to(F64).view(heads, d)[h], k[:, h // (heads // kv)], v[:, h // (heads // kv)]
            x = key @ one * scale
            p = torch.exp(x - x.max())
            out[r, h] = (p[:, None] * value).sum(0) / p.sum()
            E = (d + 4) * U * abs(scale) * (key.abs() @ one.abs()).max() + U * x.abs().max() * 4 + 2.0 ** -22
            off[r, h] = ((p[:, None] * value.abs()).sum(0) / p.sum()) * (2 * E + 2 * (n / 4 + 64) * U)
    return out, off


ATTENTION_CASES = [  # lengths, heads, kv, d, page, type, cache, window
    ([1], 1, 1, 8, 1, BF, BF, 0),
    ([77, 77], 20, 20, 64, 16, BF, BF, 0),
    ([0, 1, 31, 32, 33, 127, 128, 129, 500], 8, 2, 128, 16, BF, BF, 0),
    ([0, 1, 31, 32, 33, 127, 128, 129, 500], 8, 2, 128, 16, FP16, FP16, 0),
    ([300, 5], 6, 3, 80, 24, BF, BF, 0),
    ([1000, 0, 260], 5, 1, 40, 7, FP16, FP16, 0),
    ([700, 300], 16, 1, 256, 32, BF, BF, 0),
    ([200], 4, 2, 200, 8, FP16, FP16, 0),
    ([150, 40], 40, 2, 64, 100, BF, BF, 0),            # twenty query heads a key head: two units
    ([333], 33, 1, 96, 12, FP16, FP16, 0),
    ([5000, 1, 999, 1000, 1001, 0, 24], 15, 3, 80, 24, BF, E4M3, 1000),
    ([640, 77, 129], 8, 8, 64, 32, FP16, E4M3, 0),
    ([900], 4, 4, 256, 5, BF, E4M3, 0),
    ([260, 131], 4, 1, 128, 16, BF, BF, 1),
    ([260, 131, 8], 4, 1, 128, 16, FP16, FP16, 130),
    ([6000], 2, 1, 128, 64, BF, BF, 0),                # a row on many workgroups
    ([3000, 2, 2500], 3, 1, 64, 3, BF, BF, 0),
]


@pytest.mark.parametrize("case", ATTENTION_CASES, ids=lambda c: f"{'-'.join(map(str, c[0]))}-H{c[1]}of{c[2]}-{c[3]}-p{c[4]}-{str(c[5])[6:]}-{str(c[6])[6:]}-w{c[7]}")
@pytest.mark.parametrize("named", [False, True])
def test_paged_attention(case, named):
    from katz_amd import ops

    lengths, heads, kv, d, page, dtype, cache, window = case
    g = gen(len(lengths) + d + page)
    layers, layer = (3, 1) if named else (1, 0)
    pool = [0, *lengths, 3] if named else lengths
    pages = Pages(5, pool, page, kv, d, cache, layers, heads_first=named)
    slots = torch.arange(len(lengths)).flip(0) + 1 if named else torch.arange(len(lengths))
    n = pages.held[slots]
    wide = randn(g, len(lengths), heads * d + 8, dtype=dtype)
    q = wide[:, 8:] if named else wide[:, 8:].contiguous()
    on = dict(slots=slots.int().to(DEV), layer=layer) if named else {}
    ref, off = attention_reference(q, pages, heads, slots, n, layer, window)
    q_dev = wide.to(DEV)[:, 8:] if named else q.to(DEV)
    got = ops.paged_attention(q_dev, pages.dev, heads, window=window, **on)
    assert got.dtype is dtype
    assert_within(got.view(-1, heads, d), ref, HALF[dtype] * ref.abs() + off + TINY[dtype], "attention")
    assert torch.equal(got, ops.paged_attention(q_dev, pages.dev, heads, window=window, **on))


def test_paged_attention_of_rows_at_any_address_and_given_outputs():
    from katz_amd import ops

    g, heads, d = gen(8), 4, 64
    pages = Pages(6, [130, 0, 300], 16, 2, d)
    q = randn(g, 3, heads * d)
    flat = torch.zeros(3 * heads * d + 1, dtype=BF, device=DEV)
    odd = flat[1:].view(3, heads * d)
    odd.copy_(q)
    want = ops.paged_attention(q.to(DEV), pages.dev, heads)
    assert torch.equal(ops.paged_attention(odd, pages.dev, heads), want)
    slots = torch.tensor([2, -1, 0], dtype=torch.int32, device=DEV)
    out = torch.full((3, heads * d + 3), 9.0, dtype=BF, device=DEV)
    got = ops.paged_attention(q.to(DEV), pages.dev, heads, slots=slots, out=out[:, 1:-2])
    new = ops.paged_attention(q.to(DEV), pages.dev, heads, slots=slots)
    assert (out[:, 0] == 9).all() and (out[:, -2:] == 9).all() and (got[1] == 9).all() and (new[1] == 0).all()
    assert torch.equal(got[0], new[0]) and torch.equal(got[2], new[2])
    assert (want[1] == 0).all()                          # an empty sequence: nothing to attend to
    scaled = ops.paged_attention(q.to(DEV), pages.dev, heads, scale=-0.3)
    ref, off = attention_reference(q, pages, heads, range(3), pages.held, scale=-0.3)
    assert_within(scaled.view(3, heads, d), ref, HALF[BF] * ref.abs() + off, "a negative scale")


@pytest.mark.parametrize("page", [16, 24, 5])
@pytest.mark.parametrize("dtype", [BF, E4M3])
def test_tables_and_lengths_outside_the_cache_stay_inside(page, dtype):
    from katz_amd import ops

    heads, d = 4, 64
    pages = Pages(9, [400, 300, 200, 100, 50], page, 2, d, dtype)
    t = pages.table
    t[0, 1], t[0, 3], t[1, 0], t[2, 2] = -1, 1 << 30, pages.k.shape[1], -(1 << 31)
    t[3] = -1                                            # a sequence without any page
    pages.dev.table.copy_(t)
    g = gen(10)
    q = randn(g, 5, heads * d)
    ref, off = attention_reference(q, pages, heads, range(5), pages.held)
    got = ops.paged_attention(q.to(DEV), pages.dev, heads)
    assert_within(got.view(5, heads, d), ref, HALF[BF] * ref.abs() + off, "holes in the table")
    assert (got[3] == 0).all()
    n = torch.tensor([1 << 30, -5, 2 ** 31 - 1, 7, -(2 ** 31)], dtype=torch.int32)
    long = Pages(11, [page * 20] * 5, page, 2, d, dtype, width=20)
    ref, off = attention_reference(q, long, heads, range(5), n.clamp(0, page * 20))
    got = ops.paged_attention(q.to(DEV), long.dev, heads, lengths=n.to(DEV))
    assert_within(got.view(5, heads, d), ref, HALF[BF] * ref.abs() + off, "lengths")
    slots = torch.tensor([5, 1 << 30, -(1 << 31), 2, -1], dtype=torch.int32, device=DEV)
    got = ops.paged_attention(q.to(DEV), long.dev, heads, slots=slots)
    assert (got[[0, 1, 2, 4]] == 0).all() and torch.isfinite(got).all() and (got[3] != 0).any()


def test_rows_of_one_sequence_are_a_prompt():
    from katz_amd import ops

    heads, d, T = 6, 64, 150
    pages = Pages(12, [T, 9], 16, 2, d, width=30)
    q = randn(gen(13), T, heads * d)
    n = torch.arange(1, T + 1, dtype=torch.int32)
    slots = torch.zeros(T, dtype=torch.int32)
    ref, off = attention_reference(q, pages, heads, slots, n)
    got = ops.paged_attention(q.to(DEV), pages.dev, heads, slots=slots.to(DEV), lengths=n.to(DEV))
    assert_within(got.view(T, heads, d), ref, HALF[BF] * ref.abs() + off, "a prompt")


@pytest.mark.parametrize("dtype", [BF, FP16])
@pytest.mark.parametrize("n", [2, 200, 4000])
def test_weights_are_multiplied_in_24_bits(dtype, n):
    """Half of the values are 1 and half -1, the weights 1 and 1 - 2^-10: in a type of 16 bits all but a bit of the result is gone."""
    from katz_amd import ops

    d = 64
    pages = Pages(14, [n], 16, 1, d, dtype)
    step = -math.log1p(-2.0 ** -10)
    first = torch.arange(n) < n // 2
    q = torch.zeros(1, d, dtype=dtype)
    q[0, 0] = 1.0
    for t in range(n):
        e, at = pages.table[0, t // 16], t % 16
        pages.k[0, e, at] = 0
        pages.k[0, e, at, 0, 0] = 0.0 if first[t] else -1.0
        pages.v[0, e, at] = 1.0 if first[t] else -1.0
    pages.dev.k.copy_(pages.k)
    pages.dev.v.copy_(pages.v)
    ref, _ = attention_reference(q, pages, 1, [0], [n], scale=step)
    got = ops.paged_attention(q.to(DEV), pages.dev, 1, scale=step)
    # the score is one product (rounded with the scale, three times: 3 * 2^-24 * 2^-10), the exponential 2^-23 off, sums of n / 4 + 64 roundings of up to their own size
    bound = HALF[dtype] * ref.abs() + 4 * U + 2 * (n / 4 + 64) * U
    assert ref.abs().min() > 2.0 ** -12
    assert_within(got.view(1, 1, d), ref, bound, "weights")
    assert ((got.double().cpu() - ref.view(1, d)).abs() < 2.0 ** -14).all()


def test_scores_far_apart_and_values_that_are_no_numbers():
    from katz_amd import ops

    heads, d, n = 2, 64, 300
    pages = Pages(15, [n, n, n], 16, 1, d, fill=float("inf"))
    for t in range(n):
        pages.k[0, pages.table[0, t // 16], t % 16] *= 1e4          # scores of +-1e5: all but one weight is gone
    pages.k[0, pages.table[1, 3], 5, 0, 7] = NAN
    pages.v[0, pages.table[2, 3], 5, 0, 7] = NAN
    pages.dev.k.copy_(pages.k)
    pages.dev.v.copy_(pages.v)
    q = randn(gen(16), 3, heads * d)
    got = ops.paged_attention(q.to(DEV), pages.dev, heads).view(3, heads, d).cpu()
    ref, off = attention_reference(q, pages, heads, range(3), [n] * 3)
    assert_within(got[0], ref[0], HALF[BF] * ref[0].abs() + off[0], "far apart")
    assert torch.isnan(got[1]).all()                     # a score that is no number
    assert torch.isnan(got[2][:, 7]).all() and torch.isfinite(got[2][:, [i for i in range(d) if i != 7]]).all()
    # and none of it reaches rows that do not attend to it
    n = torch.tensor([50, 53, 53], dtype=torch.int32)
    got = ops.paged_attention(q.to(DEV), pages.dev, heads, lengths=n.to(DEV)).view(3, heads, d)
    ref, off = attention_reference(q, pages, heads, range(3), n)
    assert_within(got, ref, HALF[BF] * ref.abs() + off, "before it")
    got = ops.paged_attention(q.to(DEV), pages.dev, heads, window=300 - 54).view(3, heads, d)
    ref, off = attention_reference(q, pages, heads, range(3), [300] * 3, window=300 - 54)
    assert_within(got, ref, HALF[BF] * ref.abs() + off, "behind it")


# ------------------------------------------------------------------------------------------------ appends
def nearest(x, more, dtype, scale):
    """(the value an exact x is held as, how far off it may be)."""
    if dtype is E4M3:
        c = x if scale is None else x / scale.to(F64)[:, None]
        r = (more if scale is None else more / scale.to(F64)[:, None]) + 2 * U * c.abs()
        c = c.clamp(-448, 448)
        return c, c.abs() * 2.0 ** -4 + 2.0 ** -10 + r * (1 + 2.0 ** -4)
    return x, HALF[dtype] * x.abs() + more + TINY[dtype]


@pytest.mark.parametrize("dtype,cache,page,kv,d,sections,pairs", [(BF, BF, 16, 2, 64, (32,), False), (FP16, FP16, 24, 1, 80, (24,), False), (BF, E4M3, 32, 4, 128, (16, 24, 24), True),
                                                                  (FP16, E4M3, 5, 2, 40, (7, 6), False), (BF, BF, 7, 3, 72, (9, 9, 9), True), (FP16, E4M3, 16, 1, 256, (), False)])
def test_cache_append(dtype, cache, page, kv, d, sections, pairs):
    from katz_amd import ops

    heads, layers, layer = 2 * kv, 2, 1
    held = [page * 2 + 3, 0, 1, 200, page]
    new = [page + 2, 0, 1, 150, 1]
    pages = Pages(17, held, page, kv, d, cache, layers, fill=3.0, heads_first=pairs)
    g = gen(18)
    slots = torch.tensor([s for s, m in enumerate(new) for _ in range(m)], dtype=torch.int32)
    places = torch.tensor([held[s] - m + i for s, m in enumerate(new) for i in range(m)], dtype=torch.int32)
    order = torch.randperm(len(slots), generator=g)
    slots, places = slots[order], places[order]
    rows = len(slots) + 4
    # rows that are left out: no slot, no such slot, a place behind the end, one before the beginning
    slots = torch.cat((slots, torch.tensor([-1, 99, 0, 3], dtype=torch.int32)))
    places = torch.cat((places, torch.tensor([0, 0, held[0], -1], dtype=torch.int32)))
    pos = torch.randint(0, 5000, (rows, max(1, len(sections))), generator=g, dtype=torch.int32)
    qkv = randn(g, rows, (heads + 2 * kv) * d, dtype=dtype)
    if cache is E4M3:
        qkv[0, heads * d] = 60000.0                      # past the largest code
    dev = qkv.to(DEV)
    freq = ops.rotary_frequencies(sum(sections), device=DEV) if sections else None
    q_out = torch.full((rows, heads * d), 5.0, dtype=dtype, device=DEV)
    before = raw(pages.dev.k), raw(pages.dev.v)
    args = dev[:, :heads * d], dev[:, heads * d:(heads + kv) * d], dev[:, (heads + kv) * d:]
    on = dict(layer=layer, slots=slots.to(DEV), places=places.to(DEV), pairs=pairs)
    got = ops.cache_append(*args, pages.dev, heads, pos.to(DEV) if sections else None, freq, sections or None, out=q_out, **on)
    ref, more = turned(qkv[:, :heads * d], heads, pos, [] if freq is None else freq.cpu(), sections or (0,), pairs)
    assert_within(got.view(rows, heads, d)[:-4], ref[:-4], (HALF[dtype] * ref.abs() + more + TINY[dtype])[:-4], "q")
    assert (got[-4:] == 5).all()
    at = pages.table[slots[:-4].long(), places[:-4].long() // page].long(), places[:-4].long() % page
    k, more = turned(qkv[:-4, heads * d:(heads + kv) * d], kv, pos[:-4], [] if freq is None else freq.cpu(), sections or (0,), pairs)
    v = qkv[:-4, (heads + kv) * d:].to(F64).view(-1, kv, d)
    for pool, old, x, r, scale, name in ((pages.dev.k, before[0], k, more, pages.ks, "k"), (pages.dev.v, before[1], v, torch.zeros_like(v), pages.vs, "v")):
        want, bound = nearest(x, r, cache, None if scale is None else scale[layer])
        assert_within(pool[layer].cpu().to(F64)[at], want, bound, name)
        now = raw(pool)
        now[layer][at] = old[layer][at]
        assert torch.equal(now, old), f"{name}: other places were written"
    again = ops.cache_append(*args, pages.dev, heads, pos.to(DEV) if sections else None, freq, sections or None, **on)
    assert torch.equal(again[:-4], got[:-4]) and (again[-4:] == 0).all()


def test_cache_append_of_the_last_token_of_every_slot():
    from katz_amd import ops

    heads, kv, d, page = 4, 2, 64, 16
    held = [33, 0, 16, 1]
    pages = Pages(19, held, page, kv, d, fill=1.0)
    pages.table[2, 0] = pages.k.shape[1]                 # a sequence whose page is none: its token is dropped
    pages.dev.table.copy_(pages.table)
    g = gen(20)
    q, k, v = (randn(g, 4, h * d) for h in (heads, kv, kv))
    freq = ops.rotary_frequencies(32, device=DEV)
    before = pages.dev.k.clone()
    got = ops.cache_append(q.to(DEV), k.to(DEV), v.to(DEV), pages.dev, heads, frequencies=freq)
    pos = torch.tensor([[32], [0], [15], [0]])
    ref, more = turned(q, heads, pos, freq.cpu(), (32,), False)
    keep = [0, 2, 3]
    assert_within(got.view(4, heads, d)[keep], ref[keep], (HALF[BF] * ref.abs() + more)[keep], "q")
    assert (got[1] == 0).all()
    ref, more = turned(k, kv, pos, freq.cpu(), (32,), False)
    for s, t in ((0, 32), (3, 0)):
        e = int(pages.table[s, t // page])
        assert_within(pages.dev.k[0, e, t % page], ref[s], HALF[BF] * ref[s].abs() + more[s], "k")
        assert torch.equal(pages.dev.v[0, e, t % page].cpu().view(-1), v[s])
        before[0, e, t % page] = pages.dev.k[0, e, t % page]
    assert torch.equal(before, pages.dev.k)


# ------------------------------------------------------------------------------------------------ the pages of a cache
class Model:
    """What the calls that keep a cache's pages are to do, page by page."""

    def __init__(self, pages):
        self.p, self.page = pages, pages.page
        self.table, self.held, self.refs = pages.table.tolist(), pages.held.tolist(), pages.refs.tolist()
        self.k, self.v = raw(pages.k).clone(), raw(pages.v).clone()
        self.width = len(self.table[0])

    def take(self):
        e = self.refs.index(0) if 0 in self.refs else -1
        if e >= 0:
            self.refs[e] = 1
        return e

    def extend(self, counts):
        missing = 0
        for s, more in enumerate(counts):
            n = self.held[s]
            if more <= 0:
                continue
            new = min(n + more, self.width * self.page)
            missing += max(0, -(-(n + more) // self.page) - self.width)
            for i in range(-(-n // self.page), -(-new // self.page)):
                self.table[s][i] = self.take()
                missing += self.table[s][i] < 0
            self.held[s] = new
        return missing

    def reorder(self, parents):
        slots, rows, held = len(parents), [list(r) for r in self.table], list(self.held)
        changed = [s for s in range(slots) if parents[s] != s]
        for s in changed:
            for e in rows[s][:-(-held[s] // self.page)]:
                if 0 <= e < len(self.refs):
                    self.refs[e] -= 1
        late, given = [], set()
        for s in changed:
            p = parents[s]
            self.table[s], self.held[s] = [-1] * self.width, 0
            if not 0 <= p < slots:
                continue
            self.held[s] = held[p]
            full, part = divmod(held[p], self.page)
            whole = full
            if part and parents[p] != p and p not in given:
                whole += 1
            elif part:
                late.append((s, full, rows[p][full], part))
            given.add(p)
            for i in range(whole):
                e = self.table[s][i] = rows[p][i]
                if 0 <= e < len(self.refs):
                    self.refs[e] += 1
        missing = 0
        for s, i, src, part in late:
            if not 0 <= src < len(self.refs):
                continue
            e = self.table[s][i] = self.take()
            missing += e < 0
            if e >= 0:
                for pool in (self.k, self.v):
                    pool[:, e, :part] = pool[:, src, :part]
        return missing

    def compact(self):
        live = [e for e, n in enumerate(self.refs) if n > 0]
        to = dict(zip([e for e in live if e >= len(live)], [e for e in range(len(live)) if self.refs[e] == 0]))
        for src, dst in to.items():
            self.refs[dst], self.refs[src] = self.refs[src], 0
            for pool in (self.k, self.v):
                pool[:, dst] = pool[:, src]
        self.table = [[to.get(e, e) for e in r] for r in self.table]
        return len(live)

    def same(self, what):
        c = self.p.dev
        assert c.table.tolist() == self.table, f"{what}: table"
        assert c.lengths.tolist() == self.held, f"{what}: lengths"
        assert c.refs.tolist() == self.refs, f"{what}: refs"
        assert torch.equal(raw(c.k), self.k) and torch.equal(raw(c.v), self.v), f"{what}: pages"
        counted = [0] * len(self.refs)
        for r, n in zip(self.table, self.held):
            for e in r[:-(-n // self.page)]:
                if e >= 0:
                    counted[e] += 1
        assert counted == self.refs, f"{what}: refs are not how many hold a page"


def int32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("seed,slots,page,kv,d,dtype,layers,spare,heads_first", [
    (0, 4, 16, 2, 64, BF, 2, 6, False), (1, 9, 5, 1, 40, FP16, 1, 3, False), (2, 30, 8, 3, 72, E4M3, 3, 40, True), (3, 1, 1, 1, 8, BF, 1, 1, False), (4, 70, 32, 1, 128, BF, 1, 30, True),
    (5, 12, 24, 2, 24, E4M3, 2, 0, False), (6, 3, 64, 20, 64, BF, 2, 5, False), (7, 300, 2, 1, 8, FP16, 1, 200, False)])
def test_pages_through_many_calls(seed, slots, page, kv, d, dtype, layers, spare, heads_first):
    import random

    from katz_amd import ops

    rng = random.Random(seed)
    held = [rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, 5 * page)]) for _ in range(slots)]
    pages = Pages(seed, held, page, kv, d, dtype, layers, spare, width=7, heads_first=heads_first)
    model = Model(pages)
    for call in range(8):
        kind = ["reorder", "extend", "compact"][call % 3] if call < 6 else rng.choice(["reorder", "extend"])
        if kind == "reorder":
            parents = [rng.choice([s, s, rng.randrange(slots), rng.randrange(slots), -1, slots, -(2 ** 31)]) for s in range(slots)]
            if call == 0:
                parents = [(s + 1) % slots for s in range(slots)]        # every page not yet full changes hands
            elif call == 3:
                parents = [slots // 2] * slots                           # all from one
            want, got = model.reorder(parents), ops.cache_reorder(pages.dev, int32(parents))
        elif kind == "extend":
            counts = [rng.choice([0, 0, 1, page, -3, rng.randint(0, 9 * page)]) for _ in range(slots)]
            want, got = model.extend(counts), ops.cache_extend(pages.dev, int32(counts))
        else:
            want, got = model.compact(), ops.cache_compact(pages.dev)
        assert got.tolist() == [want], (call, kind)
        model.same(f"call {call}, {kind}")


def test_beams_that_change_places_copy_nothing():
    from katz_amd import ops

    pages = Pages(21, [37, 50, 3, 16], 16, 1, 64, spare=0)
    model = Model(pages)
    parents = [1, 0, 3, 2]                               # no page is free, and none is wanted
    assert model.reorder(parents) == 0 and ops.cache_reorder(pages.dev, int32(parents)).tolist() == [0]
    model.same("a swap")
    parents = [0, 0, 2, 0]                               # slot 1's four pages are free then: two are wanted
    assert model.reorder(parents) == 0 and ops.cache_reorder(pages.dev, int32(parents)).tolist() == [0]
    model.same("a fork")


def test_tables_of_pages_that_are_none_stay_inside():
    from katz_amd import ops

    pages = Pages(22, [40, 40, 8], 16, 2, 64, spare=3)
    big = 2 ** 31 - 1
    pages.table[0] = torch.tensor([big, -7, int(pages.table[0, 2]), -1], dtype=torch.int32)
    pages.table[1, 2] = 999                              # the page not yet full of a sequence that is taken over
    pages.dev.table.copy_(pages.table)
    pages.dev.lengths.copy_(torch.tensor([big, 40, -9], dtype=torch.int32))
    k = raw(pages.dev.k)
    ops.cache_extend(pages.dev, int32([5, 0, big]))
    ops.cache_reorder(pages.dev, int32([1, 1, 0]))
    n = ops.cache_compact(pages.dev)
    assert 0 <= n.item() <= pages.refs.numel()
    assert pages.dev.lengths[0].item() == 40 and pages.dev.table[0, 2].item() == -1
    assert raw(pages.dev.k).shape == k.shape


def test_pages_past_32_bits():
    """Pages whose addresses are more than 2^32 bytes and 2^31 elements behind the first."""
    from katz_amd import ops

    page, kv, d, pages = 64, 8, 128, 36000               # 4.7 GB each of keys and values
    k, v = (torch.empty(1, pages, page, kv, d, dtype=BF, device=DEV) for _ in range(2))
    table = torch.full((2, 4), -1, dtype=torch.int32, device=DEV)
    cache = ops.PagedCache(k, v, table, int32([0, 0]), torch.ones(pages, dtype=torch.int32, device=DEV))
    cache.refs[pages - 5:] = 0
    assert ops.cache_extend(cache, int32([150, 70])).tolist() == [0]
    assert table.tolist() == [[pages - 5, pages - 4, pages - 3, -1], [pages - 2, pages - 1, -1, -1]]
    g, heads = gen(23), 16
    rows = 150
    x = randn(g, rows, (heads + 2 * kv) * d)
    dev = x.to(DEV)
    slots, places = torch.zeros(rows, dtype=torch.int32, device=DEV), torch.arange(rows, dtype=torch.int32, device=DEV)
    q = ops.cache_append(dev[:, :heads * d], dev[:, heads * d:(heads + kv) * d], dev[:, (heads + kv) * d:], cache, heads, slots=slots, places=places)
    assert torch.equal(q.cpu(), x[:, :heads * d])
    got = ops.paged_attention(q[-1:], cache, heads, lengths=int32([150]))

    near = Pages.__new__(Pages)
    near.page, near.ks, near.vs, near.table = page, None, None, torch.tensor([[0, 1, 2]])
    near.k, near.v = (torch.nn.functional.pad(x[:, a:a + kv * d], (0, 0, 0, 42)).view(1, 3, page, kv, d) for a in (heads * d, (heads + kv) * d))
    ref, off = attention_reference(x[-1:, :heads * d], near, heads, [0], [150])
    assert_within(got.view(1, heads, d), ref, HALF[BF] * ref.abs() + off, "far pages")
    cache.refs[:40] = 0
    assert ops.cache_reorder(cache, int32([0, 0])).tolist() == [0]
    assert table[1].tolist() == [pages - 5, pages - 4, 0, -1] and torch.equal(k[0, 0, :22], k[0, pages - 3, :22])
    n = ops.cache_compact(cache)
    assert n.item() == pages - 41                        # (39 of the first and the two that slot 1 gave up are free)
    got2 = ops.paged_attention(q[-1:], cache, heads, lengths=int32([150]))
    assert torch.equal(got, got2) and table.max().item() < 36000 - 41


def test_calls_without_rows():
    from katz_amd import ops

    pages = Pages(24, [5], 16, 2, 64)
    none = torch.zeros(0, 4 * 64, dtype=BF, device=DEV)
    assert ops.paged_attention(none, pages.dev, 4).shape == (0, 256)
    assert ops.cache_append(none, none[:, :128], none[:, :128], pages.dev, 4).shape == (0, 256)
    assert ops.rotary(none, none[:, :128], 4, int32([]).view(0, 1), ops.rotary_frequencies(32, device=DEV), kv_heads=2)[1].shape == (0, 128)


@pytest.mark.parametrize("rows,longest,kv,d", [(40, 20000, 1, 64), (3, 20000, 2, 64), (9, 9000, 1, 128)])
def test_long_sequences_among_short_ones(rows, longest, kv, d):
    """More parts of one sequence than a wave has lanes (the workgroups are dealt to few rows), and many of several."""
    from katz_amd import ops

    lengths = [0] * rows
    lengths[rows // 2] = longest
    if rows < 10:
        lengths[0], lengths[-1] = 700, longest // 2
    pages = Pages(25, lengths, 64, kv, d, spare=1)
    q = randn(gen(26), rows, 2 * kv * d)
    ref, off = attention_reference(q, pages, 2 * kv, range(rows), pages.held)
    got = ops.paged_attention(q.to(DEV), pages.dev, 2 * kv)
    assert_within(got.view(rows, 2 * kv, d), ref, HALF[BF] * ref.abs() + off, "long among short")


def test_rows_by_the_hundred():
    """More rows than a workgroup has threads."""
    from katz_amd import ops

    rows, heads, d = 700, 2, 64
    lengths = [(i * 37) % 90 if i % 5 else 0 for i in range(rows)]
    pages = Pages(27, lengths, 16, 1, d, width=10)
    q = randn(gen(28), rows, heads * d)
    slots = torch.arange(rows, dtype=torch.int32)
    slots[::50] = -1
    ref, off = attention_reference(q, pages, heads, slots.clamp(min=0), torch.where(slots < 0, 0, pages.held[slots.clamp(min=0).long()]))
    got = ops.paged_attention(q.to(DEV), pages.dev, heads, slots=slots.to(DEV))
    assert_within(got.view(rows, heads, d), ref, HALF[BF] * ref.abs() + off, "rows")


@pytest.mark.parametrize("dtype", [BF, FP16])
def test_codes_are_the_nearest_ones(dtype):
    """Every number of 16 bits, written as an 8-bit code: the nearest, halves to even, at most 448, as torch rounds."""
    from katz_amd import ops

    every = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dtype)
    x = every.view(256, 256).to(DEV)
    cache = ops.PagedCache.empty(1, 16, 16, 1, 256, 1, 16, E4M3, DEV)
    ops.cache_extend(cache, int32([256]))
    rows = dict(slots=int32([0] * 256), places=int32(list(range(256))))
    ops.cache_append(x, x, x, cache, 1, **rows)
    want = every.float().clamp(-448, 448).to(E4M3)
    order = cache.table[0].long().cpu()
    for pool in (cache.k, cache.v):
        got = pool[0].cpu().view(torch.uint8)[order].view(-1)
        nan = torch.isnan(every)
        assert torch.equal(got[~nan], want.view(torch.uint8)[~nan]) and (got[nan] & 127 == 127).all()


def test_axes_of_one_element_have_any_stride():
    from katz_amd import ops

    g = gen(29)
    base = torch.zeros(3, 1, 16, 1, 72, dtype=BF, device=DEV)[:, :, :, :, :64]
    k, v = (base.as_strided((1, 1, 16, 1, 64), (5, 3, 72, 1 << 33, 1), o) for o in (0, 72 * 16))
    k[0, 0, :9, 0], v[0, 0, :9, 0] = randn(g, 9, 64).to(DEV), randn(g, 9, 64).to(DEV)
    cache = ops.PagedCache(k, v, int32([[0, -1]]), int32([9]), int32([1]))
    pages = Pages.__new__(Pages)
    pages.page, pages.ks, pages.vs, pages.table, pages.k, pages.v = 16, None, None, cache.table.cpu(), k.cpu(), v.cpu()
    q = randn(g, 1, 128)
    ref, off = attention_reference(q, pages, 2, [0], [9])
    assert_within(ops.paged_attention(q.to(DEV), cache, 2).view(1, 2, 64), ref, HALF[BF] * ref.abs() + off, "one page")
    assert ops.cache_reorder(cache, int32([0])).item() == 0 and ops.cache_compact(cache).item() == 1


@pytest.mark.parametrize("dtype", [BF, FP16])
@pytest.mark.parametrize("n", [2, 64, 1500])
def test_weights_that_no_type_of_16_bits_holds(dtype, n):
    """As above, weights 1 and exp(-0.00137), which is 2^-12 off in 11 bits: a fifth of the result."""
    from katz_amd import ops

    d, step = 64, 0.00137
    pages = Pages(30, [n], 16, 1, d, dtype)
    first = torch.arange(n) < n // 2
    for t in range(n):
        e, at = pages.table[0, t // 16], t % 16
        pages.k[0, e, at] = 0
        pages.k[0, e, at, 0, 0] = 0.0 if first[t] else -1.0
        pages.v[0, e, at] = 1.0 if first[t] else -1.0
    pages.dev.k.copy_(pages.k)
    pages.dev.v.copy_(pages.v)
    q = torch.zeros(1, d, dtype=dtype)
    q[0, 0] = 1.0
    ref, _ = attention_reference(q, pages, 1, [0], [n], scale=step)
    got = ops.paged_attention(q.to(DEV), pages.dev, 1, scale=step)
    assert_within(got.view(1, 1, d), ref, HALF[dtype] * ref.abs() + 4 * U + 2 * (n / 4 + 64) * U, "weights")


def test_the_smallest_numbers_of_fp16():
    """Keys, queries and values below fp16's normal numbers are numbers: none is taken as zero."""
    from katz_amd import ops

    g, heads, d, n = gen(31), 4, 64, 200
    pages = Pages(32, [n, n], 16, 2, d, FP16)
    pages.v[:] = pages.v * 2.0 ** -18
    pages.k[:] = torch.where(torch.arange(d) < 32, pages.k * 2.0 ** -16, pages.k)
    pages.dev.k.copy_(pages.k)
    pages.dev.v.copy_(pages.v)
    q = randn(g, 2, heads * d, dtype=FP16).view(2, heads, d)
    q[..., 32:] = q[..., 32:] * 2.0 ** -17
    q = q.reshape(2, heads * d)
    # (scores of 2^-13 or so, scaled up to some ones: a subnormal key or query taken as zero would change them all)
    ref, off = attention_reference(q, pages, heads, range(2), [n] * 2, scale=2.0 ** 13)
    got = ops.paged_attention(q.to(DEV), pages.dev, heads, scale=2.0 ** 13)
    assert_within(got.view(2, heads, d), ref, HALF[FP16] * ref.abs() + off + TINY[FP16], "small numbers")
    big, more = attention_reference(q, pages, heads, range(2), [n] * 2, scale=2.0 ** 13)
    assert (big.abs().max() > 2.0 ** -20) and (got.abs().max().item() > 0)


@pytest.mark.parametrize("slots,page,longest,spare,shift", [(1500, 2, 9, 900, 0), (3, 1, 6500, 9000, 0), (40, 1, 300, 5000, 1)])
def test_slots_and_pages_by_the_thousand(slots, page, longest, spare, shift):
    """More slots than the workgroup that deals pages out has threads, more pages than it looks at in one go, counts at an address of four bytes."""
    import random

    from katz_amd import ops

    rng = random.Random(slots)
    held = [rng.choice([0, rng.randint(0, longest)]) for _ in range(slots)]
    held[0] = longest
    pages = Pages(33, held, page, 1, 8, BF, 1, spare, width=longest // page + 40)
    if shift:
        c = pages.dev
        refs = torch.zeros(c.refs.numel() + 1, dtype=torch.int32, device=DEV)[1:]
        refs.copy_(c.refs)
        pages.dev = ops.PagedCache(c.k, c.v, c.table, c.lengths, refs)
    model = Model(pages)
    for call in range(4):
        counts = [rng.choice([0, 1, 2, rng.randint(0, 12), -5]) for _ in range(slots)]
        counts[-1] = 33 * page
        assert ops.cache_extend(pages.dev, int32(counts)).tolist() == [model.extend(counts)]
        model.same(f"extended, {call}")
        parents = [rng.choice([s, s, s, rng.randrange(slots), -1]) for s in range(slots)]
        assert ops.cache_reorder(pages.dev, int32(parents)).tolist() == [model.reorder(parents)]
        model.same(f"reordered, {call}")
        if call != 1:
            assert ops.cache_compact(pages.dev).tolist() == [model.compact()]
            model.same(f"moved together, {call}")


def test_rotary_of_more_than_the_caches_hold():
    from katz_amd import ops

    g = torch.Generator(DEV).manual_seed(34)
    rows, heads, kv, d = 70000, 6, 2, 64
    q, k = (torch.randn(rows, h * d, generator=g, device=DEV, dtype=FP32) for h in (heads, kv))
    pos, freq = torch.arange(rows, dtype=torch.int32, device=DEV)[:, None], ops.rotary_frequencies(32, device=DEV)
    for pairs in (False, True):
        got = ops.rotary(q, k, heads, pos, freq, kv_heads=kv, pairs=pairs)
        for lo in range(0, rows, 10000):                 # the same as in parts that the caches hold
            part = ops.rotary(q[lo:lo + 10000], k[lo:lo + 10000], heads, pos[lo:lo + 10000], freq, kv_heads=kv, pairs=pairs)
            assert torch.equal(got[0][lo:lo + 10000], part[0]) and torch.equal(got[1][lo:lo + 10000], part[1])


@pytest.mark.parametrize("window", [1, 127, 128, 129, 300, 2 ** 30, 2 ** 30 + 1, 2 ** 62])
@pytest.mark.parametrize("longest", [300, 2000])
def test_windows_of_every_size(window, longest):
    from katz_amd import ops

    heads, d = 4, 64
    pages = Pages(35, [longest, 128, 0, longest - 1, 129], 16, 2, d)
    q = randn(gen(36), 5, heads * d)
    ref, off = attention_reference(q, pages, heads, range(5), pages.held, window=min(window, longest))
    got = ops.paged_attention(q.to(DEV), pages.dev, heads, window=window)
    assert_within(got.view(5, heads, d), ref, HALF[BF] * ref.abs() + off, "a window")


@pytest.mark.parametrize("pairs", [False, True])
def test_turned_keys_become_the_codes_that_64_bits_give(pairs):
    """Three hundred thousand keys: in 32 bits (2^-23 off, codes 2^-3 apart) about one in a million would go to the wrong side of a border, in 64 (angles of 2 * 10^5 are 2^-33
    off) one in ten thousand millions."""
    from katz_amd import ops

    g, rows, kv, d, page = gen(37), 600, 4, 128, 32
    scale = torch.rand(1, kv, generator=g) * 0.01 + 0.01
    cache = ops.PagedCache.empty(1, 20, page, kv, d, 1, 20, E4M3, DEV, scale.to(DEV))
    ops.cache_extend(cache, int32([rows]))
    x = randn(g, rows, 2 * kv * d)
    pos = torch.randint(0, 200000, (rows, 1), generator=g, dtype=torch.int32)
    freq = ops.rotary_frequencies(d // 2, device=DEV)
    k = x[:, :kv * d].contiguous()
    for _ in range(2):
        ops.cache_append(x.to(DEV), k.to(DEV), x[:, kv * d:].to(DEV), cache, 2 * kv, pos.to(DEV), freq, slots=int32([0] * rows), places=int32(list(range(rows))), pairs=pairs)
        ref, _ = turned(k, kv, pos, freq.cpu(), (d // 2,), pairs)
        want = (ref / scale[0].to(F64)[:, None]).float().clamp(-448, 448).to(E4M3)
        got = cache.k[0].cpu().view(torch.uint8)[cache.table[0].long().cpu()].view(-1, kv, d)[:rows]
        assert torch.equal(got, want.view(torch.uint8))
        k = (k.float() * 1.0009765625).to(BF)
