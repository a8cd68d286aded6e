"""What a paged cache and its calls take and refuse at their edges, without a GPU."""
import copy
import pickle
import struct

import pytest
import torch

from test_paged_cache_refusals import cache, lib, parts  # noqa: F401


@pytest.mark.parametrize("which", range(8))
def test_strides_below_zero_are_refused(lib, which):  # noqa: F811
    strides = [18432, 2048, 128, 64] * 2
    strides[which] = -strides[which]
    c = cache(strides=tuple(strides))
    assert lib.kh_paged_attention(16, 16, c, 0, 16, None, 16, 2, 4, 256, 256, 0, 0.1, 0, 0, None) == -1
    assert lib.kh_cache_extend(c, 16, 16, 16, None) == -1 and lib.kh_cache_reorder(c, 16, 16, 16, None) == -1 and lib.kh_cache_compact(c, 16, 16, None) == -1
    ends = struct.pack("4q", 8, 8, 8, 8)
    assert lib.kh_rotary(16, 16, 16, 16, None, 16, 0, 16, ends, 1, c, 0, 16, None, 2, 4, 2, 64, 256, 128, 128, 256, 0, 0, 0, None) == -1


def test_rows_of_empty_tensors():
    from katz_amd.ops import _token_rows

    for shape in ((0, 8), (0, 3, 8), (2, 0, 8), (3, 0, 2, 8), (3, 2, 0, 8), (1, 0, 8)):
        assert _token_rows(torch.zeros(shape), 8, "q")[0] == 0, shape
        assert _token_rows(torch.zeros(*shape[:-1], 12)[..., 2:10], 8, "q")[0] == 0, shape
    assert _token_rows(torch.zeros(2, 3, 12)[..., :8], 8, "q") == (6, 12) and _token_rows(torch.zeros(2, 1, 12)[..., :8], 8, "q") == (2, 12)
    for bad in (torch.zeros(2, 4, 8)[:, :2], torch.zeros(2, 0, 9), torch.zeros(0, 4, 16)[..., ::2], torch.zeros(8)):
        with pytest.raises(ValueError):
            _token_rows(bad, 8, "q")
