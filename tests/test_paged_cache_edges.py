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


def describes(c):
    """Whether the description that the library gets is that of the tensors the cache has."""
    from katz_amd.ops import PagedCache

    return c.desc == PagedCache(c.k, c.v, c.table, c.lengths, c.refs, c.k_scale, c.v_scale).desc and (c.layers, c.pages, c.page, c.kv_heads, c.d) == tuple(c.k.shape) and (c.slots, c.width) == tuple(c.table.shape)


def test_a_cache_follows_the_tensors_that_it_is_given():
    from katz_amd.ops import PagedCache

    c = PagedCache(**parts())
    lengths = c.lengths
    c.lengths = c.lengths + 1
    assert c.lengths is not lengths and describes(c)
    c.lengths += 1
    assert c.lengths.tolist() == [2] * 4 and describes(c)
    c.k, c.v, c.refs = torch.ones_like(c.k), torch.ones_like(c.v), None
    assert c.refs is None and describes(c)
    c.table = torch.zeros(4, 9, dtype=torch.int32)       # wider rows of the same slots
    assert c.width == 9 and describes(c)
    eight = PagedCache(**parts(dtype=torch.float8_e4m3fn))
    eight.k_scale = torch.ones(2, 2)
    assert describes(eight)
    eight.k_scale = None
    assert describes(eight)


def test_a_cache_refuses_tensors_that_do_not_fit_and_stays_as_it_was():
    from katz_amd.ops import PagedCache

    c = PagedCache(**parts())
    before = c.desc
    for name, bad, kind in (("lengths", torch.zeros(5, dtype=torch.int32), ValueError), ("table", torch.zeros(3, 5, dtype=torch.int32), ValueError), ("k", c.k[:, :8], ValueError),
                            ("v", c.v.half(), TypeError), ("refs", c.refs.long(), TypeError), ("k_scale", torch.ones(2, 2), ValueError)):
        old = getattr(c, name)
        with pytest.raises(kind):
            setattr(c, name, bad)
        assert getattr(c, name) is old and c.desc == before
    for name in ("layers", "pages", "page", "kv_heads", "d", "slots", "width", "desc", "other"):
        with pytest.raises(AttributeError):
            setattr(c, name, 1)
    assert describes(c)


def test_copies_of_a_cache_describe_themselves():
    from katz_amd.ops import PagedCache

    c = PagedCache(**parts())
    c.lengths[1] = 7
    for other in (copy.deepcopy(c), pickle.loads(pickle.dumps(c))):
        assert other.lengths.tolist() == [0, 7, 0, 0] and other.lengths.data_ptr() != c.lengths.data_ptr() and describes(other)
    same = copy.copy(c)
    assert same.k is c.k and describes(same)


def test_sections_are_whole_numbers_of_any_kind():
    from katz_amd.ops import _section_ends

    want = struct.pack("4q", 9, 21, 21, 21), 2, 21
    for sections in ((9.0, 12.0), (9, 12), (torch.tensor(9), 12)):
        assert _section_ends(sections) == want
    for bad in ((9.5, 12), (-1, 4), (), (1, 1, 1, 1, 1), (float("nan"),)):
        with pytest.raises(ValueError):
            _section_ends(bad)


@pytest.mark.parametrize("heads", [0, -4])
def test_heads_that_are_none_are_refused(lib, heads):  # noqa: F811
    from katz_amd import ops

    c = ops.PagedCache(**parts())
    none, k = torch.zeros(4, 0, dtype=torch.bfloat16), torch.zeros(4, 128, dtype=torch.bfloat16)
    for call in (lambda: ops.cache_append(none, k, k, c, heads), lambda: ops.paged_attention(none, c, heads)):
        with pytest.raises(ValueError):
            call()
