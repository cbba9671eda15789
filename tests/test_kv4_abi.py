"""What the cache's entry points refuse, before they touch a device."""
import ctypes

import pytest


def cache(tb, data=4096, pages=8, page=16, heads=2, dim=64, ks=1.0, vs=1.0, stride=0):
    return tb.KV4Cache(data, pages, page, heads, dim, ks, vs, stride)


def rows(tb, cu=4096, lens=4096, table=4096, batch=2, width=4, n=8):
    return tb.KV4Rows(cu, lens, table, batch, width, n)


def append(tb, c, r, fmt=0, k=4096, ks=0, v=4096, vs=0):
    return tb.lib().tb_kv4_append(c, r, fmt, k, ks, v, vs, None)


def read(tb, c, r, fmt=0, k=4096, ks=0, v=4096, vs=0):
    return tb.lib().tb_kv4_read(c, r, fmt, k, ks, v, vs, None)


def attention(tb, c, r, fmt=0, q=4096, qs=0, out=4096, os=0, lse=None, heads=4, max_rows=1, max_len=64, scale=0.125,
              window=0, sinks=0, ws=None, ws_bytes=0):
    return tb.lib().tb_kv4_attention(c, r, fmt, q, qs, out, os, lse, heads, max_rows, max_len, scale, window, sinks,
                                     ws, ws_bytes, None)


ALL = [append, read, attention]


@pytest.mark.parametrize("f", ALL)
def test_cache_is_checked(tb, f):
    S = tb.Status
    null = ctypes.POINTER(tb.KV4Cache)()
    assert f(tb, null, rows(tb)) == S.INVALID_ARGUMENT
    for page in (0, -16, 8, 24, 48, 2048):
        assert f(tb, cache(tb, page=page), rows(tb)) == S.SHAPE
    for dim in (0, -64, 8, 72, 272):
        assert f(tb, cache(tb, dim=dim), rows(tb)) == S.SHAPE
    assert f(tb, cache(tb, heads=0), rows(tb)) == S.SHAPE
    assert f(tb, cache(tb, pages=-1), rows(tb)) == S.SHAPE
    need = tb.kv4_page_bytes(16, 2, 64)
    assert f(tb, cache(tb, stride=need - 16), rows(tb)) == S.SHAPE
    assert f(tb, cache(tb, stride=need + 8), rows(tb)) == S.ALIGNMENT
    assert f(tb, cache(tb, data=4104), rows(tb)) == S.ALIGNMENT
    assert f(tb, cache(tb, data=0), rows(tb)) == S.INVALID_ARGUMENT
    for bad in (0.0, -1.0, float("inf"), float("nan"), 1e-38, 1e35):
        assert f(tb, cache(tb, ks=bad), rows(tb)) == S.INVALID_ARGUMENT
        assert f(tb, cache(tb, vs=bad), rows(tb)) == S.INVALID_ARGUMENT


@pytest.mark.parametrize("f", ALL)
def test_rows_are_checked(tb, f):
    S = tb.Status
    assert f(tb, cache(tb), ctypes.POINTER(tb.KV4Rows)()) == S.INVALID_ARGUMENT
    for kw in (dict(batch=-1), dict(width=-1), dict(n=-1), dict(width=1 << 28)):
        assert f(tb, cache(tb), rows(tb, **kw)) == S.SHAPE
    for kw in (dict(cu=0), dict(lens=0), dict(table=0)):
        assert f(tb, cache(tb), rows(tb, **kw)) == S.INVALID_ARGUMENT
    for fmt in (1, 2, 3, 4, 6, 7, 99, -1):
        assert f(tb, cache(tb), rows(tb), fmt=fmt) == S.INVALID_ARGUMENT


@pytest.mark.parametrize("f", [append, read])
def test_copies_are_checked(tb, f):
    S = tb.Status
    c, r = cache(tb), rows(tb)
    assert f(tb, c, r, ks=127) == S.SHAPE and f(tb, c, r, vs=120) == S.SHAPE and f(tb, c, r, ks=-128) == S.SHAPE
    assert f(tb, c, r, ks=129) == S.ALIGNMENT and f(tb, c, r, vs=132) == S.ALIGNMENT
    assert f(tb, c, r, k=0) == S.INVALID_ARGUMENT and f(tb, c, r, v=0) == S.INVALID_ARGUMENT
    assert f(tb, c, r, k=4104) == S.ALIGNMENT and f(tb, c, r, v=4098) == S.ALIGNMENT
    # nothing to do
    assert f(tb, c, rows(tb, batch=0), k=0, v=0) == S.OK
    assert f(tb, c, rows(tb, n=0), k=0, v=0) == S.OK


def test_attention_is_checked(tb):
    S = tb.Status
    c, r = cache(tb), rows(tb)
    for dim in (16, 80, 96, 256):
        assert attention(tb, cache(tb, dim=dim), r) == S.SHAPE
    for heads in (0, -2, 1, 3):
        assert attention(tb, c, r, heads=heads) == S.SHAPE
    assert attention(tb, c, r, max_rows=-1) == S.SHAPE and attention(tb, c, r, max_len=-1) == S.SHAPE
    assert attention(tb, c, r, window=-1) == S.INVALID_ARGUMENT
    assert attention(tb, c, r, sinks=-1) == S.INVALID_ARGUMENT
    for scale in (float("inf"), float("nan")):
        assert attention(tb, c, r, scale=scale) == S.INVALID_ARGUMENT
    assert attention(tb, c, r, qs=248) == S.SHAPE and attention(tb, c, r, os=260) == S.ALIGNMENT
    assert attention(tb, c, r, q=0) == S.INVALID_ARGUMENT and attention(tb, c, r, out=0) == S.INVALID_ARGUMENT
    assert attention(tb, c, r, q=4104) == S.ALIGNMENT and attention(tb, c, r, out=4104) == S.ALIGNMENT
    assert attention(tb, c, rows(tb, n=1 << 30)) == S.SHAPE
    assert attention(tb, c, rows(tb, batch=0), q=0, out=0) == S.OK
    assert attention(tb, c, rows(tb, n=0), q=0, out=0) == S.OK
    assert attention(tb, c, r, max_rows=0, q=0, out=0) == S.OK


def test_helpers(tb):
    assert tb.kv4_page_bytes(16, 8, 128) == 16 * 8 * 144
    assert tb.kv4_page_bytes(64, 1, 80) == 64 * 90
    assert tb.kv4_page_bytes(0, 1, 64) == 0
    # a bad description needs no workspace: the call itself says what is wrong
    assert tb.kv4_attention_workspace(cache(tb, dim=80), rows(tb), 4, 1, 5000) == 0
    with pytest.raises(tb.TBError) as e:
        tb.kv4_read(cache(tb, page=20), rows(tb), tb.Format.F16, 4096, 4096, stream=0)
    assert e.value.status == tb.Status.SHAPE and "page_size" in str(e.value)
