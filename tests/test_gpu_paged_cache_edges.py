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
