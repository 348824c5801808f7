"""CPU tests of what the paged entry points refuse. Arguments are checked before anything of the context is used, so that a
block of zeros stands for it."""
import ctypes as C

import pytest

from fast_llm_b200 import build, capi

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lib():
    build.build()
    return capi.load()


CTX = C.create_string_buffer(4096)
P = C.c_void_p(1 << 20)        # never followed
ODD = C.c_void_p((1 << 20) + 2)


def cache(k=P, v=P, n_pages=10, page=16, n_kv=2, dim=64):
    from fast_llm_b200.paged import PagedCacheP
    return PagedCacheP(k, v, n_pages, page, n_kv, dim)


def call(lib, name, args):
    from fast_llm_b200 import paged
    return paged._entry(lib, name)(*args)


PLAN = dict(ctx=CTX, held=P, past=P, new=P, n_seq=3, page=16, table=P, blocks=4, free=P, n_pages=10, fin=P, fout=P, start=P, length=P, pos=P, slot=P, tok=8)
APPEND = dict(ctx=CTX, cache=cache(), act=0, q=P, n_q=4, qs=256, k=P, v=P, ks=128, pos=P, slot=P, n=5, rot=64, base=10000.0, out=P, os=256)
ATTN = dict(ctx=CTX, cache=cache(), act=0, q=P, n_q=4, qs=256, table=P, blocks=4, start=P, length=P, n_seq=2, n=5, most=3, scale=0.1, out=P, os=256, lse=None)


@pytest.mark.parametrize("change", [dict(ctx=None), dict(held=None), dict(past=None), dict(new=None), dict(table=None), dict(free=None), dict(fin=None), dict(fout=None), dict(start=None),
                                    dict(length=None), dict(pos=None), dict(slot=None), dict(n_seq=0), dict(n_seq=4097), dict(page=8), dict(page=24), dict(page=512), dict(blocks=0),
                                    dict(blocks=1 << 27), dict(n_pages=0), dict(n_pages=1 << 27), dict(tok=1 << 31), dict(held=ODD), dict(slot=ODD)])
def test_plan_refuses(lib, change):
    assert call(lib, "fl_b200_paged_plan", dict(PLAN, **change).values()) == 1
    assert b"paged_plan" in lib.fl_b200_last_error()


@pytest.mark.parametrize("change", [dict(ctx=None), dict(cache=None), dict(cache=cache(k=None)), dict(cache=cache(dim=96)), dict(cache=cache(page=48)), dict(cache=cache(n_kv=0)),
                                    dict(cache=cache(n_pages=0)), dict(cache=cache(n_pages=1 << 26)), dict(cache=cache(v=ODD)), dict(act=2), dict(q=None), dict(q=ODD), dict(qs=252), dict(qs=258),
                                    dict(out=None), dict(os=128), dict(k=None), dict(v=None), dict(ks=64), dict(pos=None), dict(slot=None), dict(n=0), dict(rot=66), dict(rot=3),
                                    dict(base=0.0), dict(base=float("nan")), dict(act=1, qs=260), dict(out=P, os=512)])
def test_append_refuses(lib, change):
    assert call(lib, "fl_b200_paged_append", dict(APPEND, **change).values()) == 1
    assert b"paged_append" in lib.fl_b200_last_error()


@pytest.mark.parametrize("change", [dict(ctx=None), dict(cache=None), dict(cache=cache(dim=32)), dict(act=-1), dict(q=None), dict(out=None), dict(table=None), dict(start=None), dict(length=None),
                                    dict(n_q=0), dict(n_q=3), dict(n_q=260, qs=16640, os=16640), dict(qs=128), dict(os=254), dict(blocks=0), dict(blocks=1 << 28), dict(n_seq=0),
                                    dict(n_seq=5000), dict(n=0), dict(n=1 << 30), dict(most=0), dict(most=6), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(table=ODD),
                                    dict(lse=C.c_void_p((1 << 20) + 4))])
def test_attn_refuses(lib, change):
    assert call(lib, "fl_b200_paged_attn", dict(ATTN, **change).values()) == 1
    assert b"paged_attn" in lib.fl_b200_last_error()


def test_python_checks():
    from fast_llm_b200 import paged

    class Ctx:
        device = 0
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):          # not on the device
        paged._ints(0, "pos", i, 4)
    with pytest.raises(ValueError):
        paged._rows(0, "q", torch.zeros(3, 64), torch.float32, 3, 64)
    with pytest.raises(ValueError):
        paged.PagedCache(Ctx, torch.zeros(8).half(), torch.zeros(8).half(), 1, 16, 1, 64)


def test_rows_of_bad_pages_stay_outside_the_pool():
    """The copy's coordinate of a page: inside the pool for pages inside it, its end (where copies bring zeros) for any other,
    whatever 32 bits the table holds; no product passes 32 bits."""
    for n_pages, n_kv, shift in ((10, 2, 4), ((1 << 31) // (8 * 16) - 1, 8, 4), ((1 << 31) // 256 - 1, 1, 8)):
        groups = (1 << shift) >> 3
        outside = n_pages * n_kv * groups
        assert outside < 1 << 31
        for page in (0, 1, n_pages - 1, n_pages, 1 << 30, -1, -(1 << 31), (1 << 31) - 1):
            u = page & 0xFFFFFFFF
            for hkv in (0, n_kv - 1):
                for row in (0, (1 << shift) - 8):
                    at = (u * n_kv + hkv) * groups + (row >> 3) if u < n_pages else outside
                    assert at <= outside and (at < outside) == (0 <= page < n_pages)


@pytest.mark.parametrize("page", [16, 64, 128, 256])
def test_attn_refuses_tables_whose_last_tile_ends_past_31_bits(lib, page):
    change = dict(cache=cache(page=page), blocks=((1 << 31) - 256) // page + 1)
    assert call(lib, "fl_b200_paged_attn", dict(ATTN, **change).values()) == 1
    assert b"blocks" in lib.fl_b200_last_error()


def test_python_sizes_past_32_bits():
    """ctypes cuts what does not fit: a stride of 2^32 + 128 would become one of 128."""
    from fast_llm_b200 import paged

    class Ctx:
        device, lib, _h = -1, None, None          # -1: where tensors without storage are
    meta = lambda *shape: torch.empty(shape, dtype=torch.float16, device="meta")   # noqa: E731
    wide = torch.empty_strided((2, 128), ((1 << 32) + 128, 1), dtype=torch.float32, device="meta")
    with pytest.raises(ValueError, match="stride"):
        paged._rows(-1, "q", wide, torch.float32, 2, 128)
    with pytest.raises(ValueError, match="n_pages"):
        paged.PagedCache(Ctx, meta(64, 128), meta(64, 128), -4, -16, 1, 128)
    cache = paged.PagedCache(Ctx, meta(64, 128), meta(64, 128), 4, 16, 1, 128)
    ints = lambda *shape: torch.empty(shape, dtype=torch.int32, device="meta")     # noqa: E731
    q = meta(2, 128)
    for most in ((1 << 32) + 1, -1):
        with pytest.raises(ValueError, match="max_new"):
            cache.attn(q, ints(1, 4), ints(2), ints(1), most, 0.1, q)
    with pytest.raises(ValueError, match="n_rot"):
        cache.append(q, q, q, ints(2), ints(2), q, freq_base=1e4, n_rot=(1 << 32) + 64)
    with pytest.raises(ValueError, match="page_size"):
        paged.plan(Ctx, ints(1), ints(1), ints(1), ints(1, 4), ints(4), ints(1), ints(1), ints(2), ints(1), ints(3), ints(3), page_size=(1 << 32) + 16)
    with pytest.raises(ValueError, match="q_out"):
        cache.append(q, q, q, ints(2), ints(2), None, freq_base=1e4)
