"""What the operators on a paged cache refuse, without a GPU: the C entry points before any device call, the tensor functions by type, shape and place."""
import struct

import pytest
import torch

BF = torch.bfloat16


@pytest.fixture
def lib():
    from katz_amd import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("libkatz_hip.so not built")
    return _lib.load()


def cache(k=16, v=16, table=16, lengths=16, refs=16, ks=0, vs=0, layers=2, pages=9, page=16, kv=2, d=64, slots=4, width=5, kind=0, strides=(18432, 2048, 128, 64) * 2):
    return struct.pack("23q", k, v, table, lengths, refs, ks, vs, layers, pages, page, kv, d, slots, width, kind, *strides)


BAD_CACHES = [
    (-1, dict(k=0)), (-1, dict(v=0)), (-1, dict(table=0)), (-1, dict(lengths=0)), (-1, dict(layers=0)), (-1, dict(pages=0)), (-1, dict(page=0)), (-1, dict(kv=0)),
    (-1, dict(slots=0)), (-1, dict(width=-1)), (-1, dict(kind=2)), (-1, dict(kind=4)), (-1, dict(ks=16)), (-2, dict(d=60)), (-2, dict(d=264)), (-3, dict(k=8)),
    (-3, dict(kind=3, v=4)), (-3, dict(table=2)), (-3, dict(strides=(18432, 2048, 128, 68) * 2)), (-4, dict(pages=1 << 31)), (-4, dict(width=1 << 27)), (-4, dict(slots=1 << 21))]


@pytest.mark.parametrize("code,bad", BAD_CACHES, ids=lambda x: str(x))
def test_caches_that_are_refused(lib, code, bad):
    c = cache(**bad)
    assert lib.kh_paged_attention(16, 16, c, 0, 16, None, 16, 2, 4, 256, 256, 0, 0.1, 0, 0, None) == code
    assert lib.kh_cache_extend(c, 16, 16, 16, None) == code and lib.kh_cache_reorder(c, 16, 16, 16, None) == code and lib.kh_cache_compact(c, 16, 16, None) == code
    ends = struct.pack("4q", 8, 8, 8, 8)
    d, kv = bad.get("d", 64), bad.get("kv", 2)
    assert lib.kh_rotary(16, 16, 16, 16, None, 16, 0, 16, ends, 1, c, 0, 16, None, 2, 4, max(kv, 1), d, 1 << 12, 1 << 12, 1 << 12, 1 << 12, 0, 0, 0, None) == code


def test_rotary_entry_point(lib):
    def call(q=16, k=16, v=None, qo=16, ko=16, pos=16, pt=0, freq=16, ends=(8, 20, 32), c=None, layer=0, slots=None, places=None, rows=2, H=4, Hk=2, d=64, ldq=256, ldk=128,
             ldv=0, ldqo=256, ldko=128, flags=0, t=0):
        e = struct.pack("4q", *(tuple(ends) + (32,) * 4)[:4])
        return lib.kh_rotary(q, k, v, qo, ko, pos, pt, freq, e, len(ends), c, layer, slots, places, rows, H, Hk, d, ldq, ldk, ldv, ldqo, ldko, flags, t, None)

    assert call(q=None) == -1 and call(k=None) == -1 and call(qo=None) == -1 and call(ko=None) == -1 and call(pos=None) == -1 and call(freq=None) == -1
    assert call(rows=0) == -1 and call(H=0) == -1 and call(Hk=0) == -1 and call(d=0) == -1 and call(d=62) == -1 and call(t=3) == -1 and call(pt=3) == -1 and call(flags=8) == -1
    assert call(ends=(8, 4, 32)) == -1 and call(ends=(-1,)) == -1 and call(ends=()) == -1 and call(slots=16) == -1 and call(places=16) == -1
    assert call(ldq=255) == -1 and call(ldk=100) == -1 and call(ldqo=8) == -1 and call(ldko=8) == -1
    assert call(q=17) == -3 and call(q=18, t=2) == -3 and call(pos=18) == -3 and call(pos=20, pt=1) == -3 and call(freq=20) == -3 and call(ko=17) == -3
    assert call(d=1026, ldq=1 << 13, ldk=1 << 13, ldqo=1 << 13, ldko=1 << 13) == -2 and call(rows=1 << 31) == -4
    assert call(rows=1 << 30) == -4 and call(rows=1 << 24, d=1024, ends=(512,), ldq=1 << 12, ldk=1 << 11, ldqo=1 << 12, ldko=1 << 11) == -4    # more than 2^32 threads
    assert call(H=1 << 19, ldq=1 << 25, ldqo=1 << 25) == -4
    held = cache()
    into = dict(c=held, v=16, ldv=128, ko=None, ldko=0)
    assert call(**{**into, "v": None}) == -1 and call(**into, layer=2) == -1 and call(**into, layer=-1) == -1 and call(**into, rows=5) == -1 and call(**{**into, "ldv": 64}) == -1
    assert call(**into, Hk=1) == -1 and call(**into, d=72, ldq=1 << 10, ldk=1 << 10, ldqo=1 << 10) == -1
    assert call(**into, t=1) == -2 and call(**into, t=2) == -2 and call(**{**into, "c": cache(kind=3)}, t=2) == -2
    assert call(**into, slots=18) == -3 and call(**into, places=17) == -3 and call(**{**into, "v": 17}) == -3


def test_attention_entry_point(lib):
    def call(q=16, o=16, c=None, layer=0, slots=None, lengths=None, ws=16, rows=2, H=4, ldq=256, ldo=256, window=0, flags=0, t=0):
        return lib.kh_paged_attention(q, o, c or cache(), layer, slots, lengths, ws, rows, H, ldq, ldo, window, 0.1, flags, t, None)

    assert call(q=None) == -1 and call(o=None) == -1 and call(rows=0) == -1 and call(rows=5) == -1 and call(H=3) == -1 and call(H=0) == -1
    assert call(layer=2) == -1 and call(layer=-1) == -1 and call(ldq=128) == -1 and call(ldo=128) == -1 and call(window=-1) == -1 and call(flags=2) == -1 and call(t=2) == -1
    assert call(t=1) == -2 and call(c=cache(kind=1)) == -2
    assert call(q=17) == -3 and call(ws=8) == -3 and call(slots=18) == -3 and call(lengths=17) == -3
    assert call(rows=1 << 25, slots=16) == -4 and call(H=1 << 17, ldq=1 << 24, ldo=1 << 24) == -4
    assert lib.kh_paged_attention(16, 16, None, 0, None, None, 16, 2, 4, 256, 256, 0, 0.1, 0, 0, None) == -1
    size = lib.kh_paged_attention_workspace_bytes
    assert size(0, 4, 2, 64, 80) == -1 and size(2, 3, 2, 64, 80) == -1 and size(2, 4, 0, 64, 80) == -1 and size(2, 4, 2, 64, 0) == -1 and size(2, 4, 2, 60, 80) == -2 and size(2, 4, 2, 264, 80) == -2
    assert call(ws=None, c=cache(width=40)) == -1               # sequences of more than four tiles may be cut: there are parts to be joined
    assert size(1 << 25, 4, 2, 64, 80) == -4 and size(2, 4, 2, 64, 1 << 31) == -4 and size(1 << 20, 1 << 10, 1 << 10, 64, 1 << 20) == -4
    assert size(1, 1, 1, 8, 1) == 0 and size(64, 4, 2, 64, 512) == 0 and size(1, 1, 1, 8, 513) > 0
    assert size(1, 8, 1, 128, 1 << 20) < 1 << 25                # a workgroup's parts, however long the cache


def test_entry_points_of_the_pages(lib):
    for call in (lambda c=cache(), a=16, t=16, w=16: lib.kh_cache_extend(c, a, t, w, None), lambda c=cache(), a=16, t=16, w=16: lib.kh_cache_reorder(c, a, t, w, None)):
        assert call(a=None) == -1 and call(t=None) == -1 and call(w=None) == -1 and call(c=cache(refs=0)) == -1 and call(c=None) == -1
        assert call(a=18) == -3 and call(t=17) == -3 and call(w=8) == -3
    assert lib.kh_cache_compact(cache(), None, 16, None) == -1 and lib.kh_cache_compact(cache(), 16, None, None) == -1 and lib.kh_cache_compact(cache(refs=0), 16, 16, None) == -1
    assert lib.kh_cache_compact(cache(), 18, 16, None) == -3 and lib.kh_cache_compact(cache(), 16, 24, None) == -3
    assert lib.kh_cache_reorder(cache(slots=65537), 16, 16, 16, None) == -4
    size = lib.kh_cache_workspace_bytes
    assert size(0, 1, 1) == -1 and size(1, 0, 1) == -1 and size(1, 1, 0) == -1 and size(1 << 21, 1, 1) == -4 and size(1 << 16, 1 << 15, 9) == -4 and size(1, 1, 1) > 0
    slots, width, pages = 5, 7, 11                              # rows, three numbers and a copy a slot, three numbers and a copy a page, a count
    assert size(slots, width, pages) >= 4 * (slots * width + 6 * slots + 3 * pages + 3 * pages + 1)


def parts(layers=2, pages=9, page=16, kv=2, d=64, slots=4, width=5, dtype=BF, device="cpu"):
    z = lambda *s, dtype: torch.zeros(*s, dtype=dtype, device=device)       # noqa: E731
    return dict(k=z(layers, pages, page, kv, d, dtype=dtype), v=z(layers, pages, page, kv, d, dtype=dtype), table=z(slots, width, dtype=torch.int32),
                lengths=z(slots, dtype=torch.int32), refs=z(pages, dtype=torch.int32))


def test_a_cache_checks_its_parts():
    from katz_amd.ops import PagedCache

    good = parts()
    c = PagedCache(**good)
    assert (c.layers, c.pages, c.page, c.kv_heads, c.d, c.slots, c.width) == (2, 9, 16, 2, 64, 4, 5) and len(c.desc) == 23 * 8
    assert PagedCache(good["k"], good["v"], good["table"], good["lengths"]).refs is None
    s = torch.ones(2, 2)
    eight = parts(dtype=torch.float8_e4m3fn)
    assert PagedCache(**eight, k_scale=s).k_scale is s
    k, i = good["k"], torch.int32
    for bad in (dict(k=k[0]), dict(v=good["v"][:, :, :8]), dict(k=k[:0], v=k[:0]), dict(k=k.transpose(3, 4), v=k.transpose(3, 4)), dict(k=k[..., :60], v=k[..., :60]),
                dict(table=good["table"][0]), dict(table=good["table"][:, :3]), dict(lengths=good["lengths"][:3]), dict(refs=good["refs"][:8]), dict(k_scale=s), dict(v_scale=s),
                dict(table=torch.zeros(4, 0, dtype=i))):
        with pytest.raises(ValueError):
            PagedCache(**{**good, **bad})
    for bad in (dict(k=k.float(), v=k.float()), dict(v=k.half()), dict(table=good["table"].long()), dict(lengths=good["lengths"].float()), dict(refs=good["refs"].short())):
        with pytest.raises(TypeError):
            PagedCache(**{**good, **bad})
    with pytest.raises(ValueError):
        PagedCache(**eight, k_scale=s[:1])
    with pytest.raises(TypeError):
        PagedCache(**eight, v_scale=s.double())


def test_frequencies():
    from katz_amd.ops import rotary_frequencies

    f = rotary_frequencies(4, 16.0, device="cpu")
    assert f.dtype is torch.float64 and f.tolist() == [1.0, 0.5, 0.25, 0.125]
    assert rotary_frequencies(5, 16.0, (2, 0, 3), device="cpu").tolist() == pytest.approx([1.0, 0.25, 1.0, 16 ** (-1 / 3), 16 ** (-2 / 3)], rel=1e-15)
    assert rotary_frequencies(0, device="cpu").numel() == 0
    with pytest.raises(ValueError):
        rotary_frequencies(4, sections=(2, 3), device="cpu")


def test_tensor_functions_refuse_what_is_not_on_the_gpu(lib):
    from katz_amd import ops
    from katz_amd._lib import KatzHipError

    c = ops.PagedCache(**parts())
    x, i = torch.zeros(4, 256, dtype=BF), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: ops.rotary(x, x, 4, i, torch.zeros(32)), lambda: ops.cache_append(x, x[:, :128], x[:, :128], c, 4), lambda: ops.paged_attention(x, c, 4),
                 lambda: ops.cache_extend(c, i), lambda: ops.cache_reorder(c, i), lambda: ops.cache_compact(c)):
        with pytest.raises(KatzHipError):
            call()


@pytest.mark.gpu
def test_tensor_functions_refuse_shapes_and_types():
    from katz_amd import ops
    from katz_amd._lib import KatzHipError

    dev = "cuda:0"
    t = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device=dev)      # noqa: E731
    c, eight = ops.PagedCache(**parts(device=dev)), ops.PagedCache(**parts(device=dev, dtype=torch.float8_e4m3fn))
    bare = ops.PagedCache(**{**parts(device=dev), "refs": None})
    i32 = torch.int32
    q, k, f = t(4, 256), t(4, 128), t(32, dtype=torch.float64)
    pos = t(4, dtype=i32)
    bad = [
        (ValueError, lambda: ops.rotary(q, k, 3, pos, f)), (ValueError, lambda: ops.rotary(q, k, 4, pos, f)), (ValueError, lambda: ops.rotary(q, t(3, 256), 4, pos, f)),
        (TypeError, lambda: ops.rotary(q, q.half(), 4, pos, f)), (TypeError, lambda: ops.rotary(q.double(), q.double(), 4, pos, f)), (TypeError, lambda: ops.rotary(q, q, 4, pos.short(), f)),
        (TypeError, lambda: ops.rotary(q, q, 4, pos, f.half())), (ValueError, lambda: ops.rotary(q, q, 4, pos, f, (8, 8))), (ValueError, lambda: ops.rotary(q, q, 4, pos[:3], f)),
        (ValueError, lambda: ops.rotary(q, q, 4, t(4, 4, dtype=i32)[:, :1], f)), (ValueError, lambda: ops.rotary(q, q, 4, pos, t(33, dtype=torch.float64))),
        (ValueError, lambda: ops.rotary(q, q, 4, t(4, 5, dtype=i32), t(5), (1, 1, 1, 1, 1))), (ValueError, lambda: ops.rotary(q, q, 4, pos, f, (-1, 33))),
        (ValueError, lambda: ops.rotary(q, q, 4, pos, f, out=t(4, 255))), (TypeError, lambda: ops.rotary(q, q, 4, pos, f, out=t(4, 256, dtype=torch.float16))),
        (ValueError, lambda: ops.rotary(t(256, 4).t(), q, 4, pos, f)), (KatzHipError, lambda: ops.rotary(q, q, 4, pos.cpu(), f)),
        (ValueError, lambda: ops.rotary(t(2, 3, 256)[:, :2], t(2, 2, 256), 4, t(4, dtype=i32), f)),
        (ValueError, lambda: ops.cache_append(q, k, k, c, 4, layer=2)), (ValueError, lambda: ops.cache_append(q, q, k, c, 4)), (ValueError, lambda: ops.cache_append(q, k, k[:3], c, 4)),
        (TypeError, lambda: ops.cache_append(q.half(), k.half(), k.half(), c, 4)), (TypeError, lambda: ops.cache_append(q.float(), k.float(), k.float(), eight, 4)),
        (TypeError, lambda: ops.cache_append(q, k, k.half(), c, 4)), (TypeError, lambda: ops.cache_append(q, k, k, c, 4, slots=pos.long())), (ValueError, lambda: ops.cache_append(q, k, k, c, 4, slots=pos[:3])),
        (ValueError, lambda: ops.cache_append(q, k, k, c, 4, places=pos[:3])), (ValueError, lambda: ops.cache_append(t(5, 256), t(5, 128), t(5, 128), c, 4)),
        (ValueError, lambda: ops.cache_append(q, k, k, c, 8)), (ValueError, lambda: ops.cache_append(q, k, k, c, 4, sections=(32,))),
        (KatzHipError, lambda: ops.cache_append(q, k, k, c, 4, slots=pos.cpu())),
        (ValueError, lambda: ops.paged_attention(q, c, 5)), (ValueError, lambda: ops.paged_attention(q, c, 6)), (ValueError, lambda: ops.paged_attention(q, c, 4, layer=-1)),
        (ValueError, lambda: ops.paged_attention(q, c, 4, window=-1)), (TypeError, lambda: ops.paged_attention(q.half(), c, 4)), (TypeError, lambda: ops.paged_attention(q.float(), eight, 4)),
        (ValueError, lambda: ops.paged_attention(t(5, 256), c, 4)), (ValueError, lambda: ops.paged_attention(q, c, 4, out=t(3, 256))), (TypeError, lambda: ops.paged_attention(q, c, 4, out=q.half())),
        (TypeError, lambda: ops.paged_attention(q, c, 4, lengths=pos.long())), (ValueError, lambda: ops.paged_attention(q, c, 4, lengths=pos[:2])), (KatzHipError, lambda: ops.paged_attention(q, c, 4, slots=pos.cpu())),
        (ValueError, lambda: ops.cache_extend(c, pos[:3])), (TypeError, lambda: ops.cache_reorder(c, pos.long())), (ValueError, lambda: ops.cache_compact(bare)), (ValueError, lambda: ops.cache_extend(bare, pos)),
        (KatzHipError, lambda: ops.cache_extend(c, pos.cpu())),
    ]
    for n, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            print("call", n)
