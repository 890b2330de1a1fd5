"""Argument checks of the RMS norm and of the paged cache's operators: every refusal comes from the
host, before a device is touched.  CPU only."""
import ctypes as C

import pytest

from lightship_b200 import _lib

PTR = 1 << 20  # an aligned address that no check reads


def _cache(**kw):
    d = dict(k=PTR, v=PTR, dtype=_lib.DTYPE_F16, page_size=16, kv_heads=2, head_dim=64, num_pages=10,
             page_stride=16 * 128, token_stride=128, head_stride=64, page_table=PTR, table_stride=4, kv_lens=PTR,
             max_pages=4, batch=3)
    d.update(kw)
    return _lib.lsc_paged_kv(*[d[n] for n, _ in _lib.lsc_paged_kv._fields_])


def _append(cache, k=PTR, v=PTR, tokens=5, ts=128, hs=64, off=PTR):
    return _lib.lib().lsc_kv_cache_append(C.byref(cache), k, v, tokens, ts, hs, off, None)


def _prefill(cache, q=PTR, tokens=5, heads=4, ts=256, hs=64, off=PTR, alpha=0.125, window=0, sinks=0, out=PTR, i8=None,
             s=1.0, rnd=0):
    return _lib.lib().lsc_paged_attention_prefill(C.byref(cache), q, tokens, heads, ts, hs, off, alpha, window, sinks,
                                                  out, i8, s, rnd, None)


def _decode(cache, q=PTR, heads=4, ts=256, hs=64, alpha=0.125, window=0, sinks=0, out=PTR, i8=None, s=1.0, rnd=0,
            ws=PTR, ws_bytes=1 << 40):
    return _lib.lib().lsc_paged_attention_decode(C.byref(cache), q, heads, ts, hs, alpha, window, sinks, out, i8, s,
                                                 rnd, ws, ws_bytes, None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=_lib.DTYPE_F32), _lib.ERROR_UNSUPPORTED_DATATYPE),
    (dict(page_size=4), _lib.ERROR_INVALID_ARGUMENT), (dict(page_size=24), _lib.ERROR_INVALID_ARGUMENT),
    (dict(page_size=512), _lib.ERROR_INVALID_ARGUMENT), (dict(head_dim=96), _lib.ERROR_INVALID_ARGUMENT),
    (dict(kv_heads=0), _lib.ERROR_INVALID_ARGUMENT), (dict(batch=-1), _lib.ERROR_INVALID_ARGUMENT),
    (dict(batch=65536), _lib.ERROR_INVALID_ARGUMENT), (dict(max_pages=-1), _lib.ERROR_INVALID_ARGUMENT),
    (dict(max_pages=1 << 27, table_stride=1 << 27), _lib.ERROR_INVALID_ARGUMENT),
    (dict(kv_lens=None), _lib.ERROR_INVALID_ARGUMENT), (dict(page_table=None), _lib.ERROR_INVALID_ARGUMENT),
    (dict(kv_lens=PTR + 2), _lib.ERROR_INVALID_ARGUMENT), (dict(page_table=PTR + 1), _lib.ERROR_INVALID_ARGUMENT),
    (dict(num_pages=0), _lib.ERROR_INVALID_ARGUMENT), (dict(table_stride=3), _lib.ERROR_INVALID_ARGUMENT), (dict(k=None), _lib.ERROR_INVALID_ARGUMENT),
    (dict(v=PTR + 8), _lib.ERROR_INVALID_ARGUMENT), (dict(token_stride=132), _lib.ERROR_INVALID_ARGUMENT),
    (dict(head_stride=32), _lib.ERROR_INVALID_ARGUMENT), (dict(page_stride=-8), _lib.ERROR_INVALID_ARGUMENT),
])
def test_cache_description_refused(change, code):
    cache = _cache(**change)
    assert _append(cache) == code
    assert "kv_cache_append" in _lib.last_error()
    assert _prefill(cache) == code
    assert "paged_attention_prefill" in _lib.last_error()
    assert _decode(cache) == code
    assert "paged_attention_decode" in _lib.last_error()


def test_no_cache_refused():
    lib = _lib.lib()
    assert lib.lsc_kv_cache_append(None, PTR, PTR, 1, 128, 64, PTR, None) == _lib.ERROR_INVALID_ARGUMENT
    assert lib.lsc_paged_attention_prefill(None, PTR, 1, 4, 256, 64, PTR, 1.0, 0, 0, PTR, None, 1.0, 0,
                                           None) == _lib.ERROR_INVALID_ARGUMENT
    assert lib.lsc_paged_attention_decode(None, PTR, 4, 256, 64, 1.0, 0, 0, PTR, None, 1.0, 0, PTR, 1 << 40,
                                          None) == _lib.ERROR_INVALID_ARGUMENT
    assert lib.lsc_paged_attention_decode_workspace_size(None, 4) == 0


@pytest.mark.parametrize("kw", [dict(tokens=-1), dict(k=None), dict(v=None), dict(off=None), dict(k=PTR + 2),
                                dict(ts=130), dict(hs=4), dict(ts=-128),
                                dict(off=PTR + 2), dict(tokens=(1 << 30) + 1)])
def test_append_refusals(kw):
    assert _append(_cache(), **kw) == _lib.ERROR_INVALID_ARGUMENT


BOTH = [dict(heads=3), dict(heads=0), dict(alpha=0.0), dict(alpha=-1.0), dict(alpha=float("nan")),
        dict(alpha=float("inf")), dict(window=-1), dict(sinks=-1), dict(rnd=2), dict(ts=257), dict(hs=-8),
        dict(q=None), dict(out=None), dict(q=PTR + 8), dict(out=PTR + 2), dict(i8=PTR + 4), dict(i8=PTR, s=0.0),
        dict(i8=PTR, s=float("nan"))]


@pytest.mark.parametrize("kw", BOTH + [dict(off=None), dict(off=PTR + 1), dict(tokens=-1),
                                       dict(tokens=(1 << 30) + 1)])
def test_prefill_refusals(kw):
    assert _prefill(_cache(), **kw) == _lib.ERROR_INVALID_ARGUMENT


@pytest.mark.parametrize("kw", BOTH)
def test_decode_refusals(kw):
    assert _decode(_cache(), **kw) == _lib.ERROR_INVALID_ARGUMENT


@pytest.mark.parametrize("kw", [dict(ws=None), dict(ws=PTR + 8), dict(ws_bytes=0), dict(ws_bytes=1 << 20)])
def test_decode_workspace_refusals(kw):
    """A cache whose sequences can be cut needs a workspace; a short one needs none."""
    long = _cache(max_pages=1000, table_stride=1000)
    need = _lib.lib().lsc_paged_attention_decode_workspace_size(C.byref(long), 4)
    assert need > 1 << 20
    assert _decode(long, **kw) == _lib.ERROR_INVALID_ARGUMENT
    assert "workspace" in _lib.last_error()
    assert _lib.lib().lsc_paged_attention_decode_workspace_size(C.byref(_cache()), 4) == 0


def test_empty_calls_succeed_without_a_device():
    assert _append(_cache(), tokens=0, k=None, v=None, off=None) == _lib.SUCCESS
    assert _append(_cache(batch=0, kv_lens=None, page_table=None)) == _lib.SUCCESS
    assert _prefill(_cache(), tokens=0, q=None, out=None, off=None) == _lib.SUCCESS
    assert _prefill(_cache(batch=0)) == _lib.SUCCESS
    assert _decode(_cache(batch=0), q=None, out=None, ws=None) == _lib.SUCCESS
    assert _rms(rows=0, x=None, out=None) == _lib.SUCCESS
    assert _rms(d=0, x=None, out=None) == _lib.SUCCESS


def _rms(x=PTR, xt=_lib.DTYPE_F16, xs=64, r=None, rt=_lib.DTYPE_F16, rs=64, rows=4, d=64, g=PTR, eps=1e-5, sm=None,
         ss=64, out=PTR + 4096, os=64, q=None, qs=64, s=0.0, scales=None, rnd=0):
    return _lib.lib().lsc_rmsnorm(x, xt, xs, r, rt, rs, rows, d, g, eps, sm, ss, out, os, q, qs, s, scales, rnd, None)


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), 2), (dict(d=-1), 2), (dict(xt=3), _lib.ERROR_UNSUPPORTED_DATATYPE),
    (dict(r=PTR, rt=_lib.DTYPE_BF16), _lib.ERROR_UNSUPPORTED_DATATYPE),
    (dict(xt=_lib.DTYPE_F32, r=PTR, rt=_lib.DTYPE_F16), _lib.ERROR_UNSUPPORTED_DATATYPE),
    (dict(sm=PTR), 2), (dict(eps=-1.0), 2), (dict(eps=float("nan")), 2), (dict(eps=float("inf")), 2), (dict(rnd=3), 2),
    (dict(scales=PTR), 2), (dict(x=None), 2), (dict(out=None), 2), (dict(q=PTR), 2), (dict(q=PTR, s=-1.0), 2),
    (dict(xs=63), 2), (dict(os=8), 2), (dict(q=PTR, qs=1, s=1.0), 2), (dict(r=PTR, rs=60), 2),
    (dict(r=PTR, sm=PTR, ss=60), 2), (dict(r=PTR, sm=PTR + 4096), 2), (dict(x=PTR + 1), 2), (dict(g=PTR + 2), 2),
    (dict(q=PTR, scales=PTR + 2), 2)])
def test_rmsnorm_refusals(kw, code):
    assert _rms(**kw) == code
    assert "rmsnorm" in _lib.last_error()
