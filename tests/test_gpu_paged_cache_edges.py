"""Attention over a paged cache where a type, a size or a number is at its edge, against plain implementations in 64 bits (tolerances as in test_gpu_paged_cache)."""
import math

import pytest
import torch

from test_gpu_paged_cache import BF, DEV, E4M3, F64, FP16, FP32, HALF, TINY, U, Model, Pages, assert_within, attention_reference, gen, int32, randn, raw, turned

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
