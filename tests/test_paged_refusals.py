"""CPU: the paged-cache operators refuse bad arguments before anything is launched, and plan their
workspace from the arguments alone."""
import ctypes as C

import pytest

import gsvk


def _kv(**kw):
    a = dict(k=4096, v=8192, type=1, n_kv=2, hd=64, page_size=16, n_pages=10, page_stride=0, table=64, table_stride=4,
             table_cols=4, B=2, seq_start=64, kv_len=64)
    a.update(kw)
    return gsvk.PagedKVArgs(*[a[n] for n, _ in gsvk.PagedKVArgs._fields_])


def _append(kv=None, q=4096, k=4096, v=4096, x_type=1, tokens=3, nh=4, qs=256, ks=128, vs=128, rope=None, q_out=8192):
    return gsvk.lib().gsvk_op_paged_append(kv if kv is None else C.byref(kv), q, k, v, x_type, tokens, nh, qs, ks, vs,
                                           None if rope is None else C.byref(rope), q_out, None, None)


def _attn(kv=None, q=4096, tokens=3, nh=4, qs=256, max_new=2, max_keys=64, scale=0.1, window=0, out=4096, out_type=1,
          os_=256, ws=None, ws_bytes=0):
    return gsvk.lib().gsvk_op_attn_paged(kv if kv is None else C.byref(kv), q, tokens, nh, qs, max_new, max_keys, scale,
                                         window, None, out, out_type, os_, None, ws, ws_bytes, None)


BAD_KV = [dict(type=0), dict(type=8), dict(hd=48), dict(hd=256), dict(page_size=8), dict(page_size=48),
          dict(page_size=65536), dict(n_kv=0), dict(B=-1), dict(B=65536), dict(n_pages=0), dict(page_stride=2047),
          dict(page_stride=2052), dict(table_cols=0), dict(table_stride=3), dict(k=None), dict(v=None),
          dict(table=None), dict(seq_start=None), dict(kv_len=None), dict(k=4104), dict(v=8194)]


@pytest.mark.parametrize("bad", BAD_KV, ids=lambda d: "-".join(f"{k}={v}" for k, v in d.items()))
def test_bad_caches_are_refused(bad):
    for call, name in ((_append, "paged_append"), (_attn, "attn_paged")):
        assert call(_kv(**bad)) == 1
        assert name in gsvk.last_error()


def test_missing_cache_is_refused():
    assert _append(None) == 1 and _attn(None) == 1


@pytest.mark.parametrize("bad", [
    dict(x_type=30), dict(x_type=8), dict(tokens=-1), dict(tokens=2 ** 31), dict(nh=-1), dict(nh=0), dict(q=None),
    dict(q_out=None), dict(k=None), dict(v=None), dict(qs=255), dict(qs=260), dict(ks=100), dict(vs=132),
    dict(q=4100), dict(k=4104), dict(v=4098), dict(q_out=8194), dict(q=8192, qs=512), dict(q=8192, x_type=0),
], ids=lambda d: "-".join(f"{k}={v}" for k, v in d.items()))
def test_append_refuses(bad):
    assert _append(_kv(), **bad) == 1, bad
    assert "paged_append" in gsvk.last_error()


@pytest.mark.parametrize("bad", [dict(cos=None), dict(sin=None), dict(rows=0), dict(rot=8), dict(rot=40), dict(rot=80),
                                 dict(cos=4100)], ids=lambda d: "-".join(f"{k}={v}" for k, v in d.items()))
def test_append_refuses_rotations(bad):
    a = dict(cos=4096, sin=4096, rows=100, rot=64, pairs=0, pos=None)
    a.update(bad)
    assert _append(_kv(), rope=gsvk.RopeArgs(*[a[n] for n, _ in gsvk.RopeArgs._fields_])) == 1
    assert "paged_append" in gsvk.last_error()


@pytest.mark.parametrize("bad", [
    dict(nh=0), dict(nh=3), dict(nh=65536), dict(tokens=-1), dict(out_type=30), dict(out_type=8), dict(scale=0.0),
    dict(scale=-0.1), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=3e38), dict(window=-1),
    dict(max_new=-1), dict(max_keys=-1), dict(q=None), dict(out=None), dict(qs=255), dict(qs=260), dict(os_=250),
    dict(os_=260), dict(q=4104), dict(out=4100),
], ids=lambda d: "-".join(f"{k}={v}" for k, v in d.items()))
def test_attn_refuses(bad):
    assert _attn(_kv(), **bad) == 1, bad
    assert "attn_paged" in gsvk.last_error()


def test_nothing_to_do_is_no_error():
    """No tokens or no sequences: nothing is launched (there is no device here)."""
    assert _append(_kv(), tokens=0) == 0 and _append(_kv(B=0)) == 0
    assert _attn(_kv(), tokens=0) == 0 and _attn(_kv(B=0)) == 0 and _attn(_kv(), max_new=0) == 0


def test_empty_arrays_may_be_null():
    """An empty tensor has no address: a step without rows passes through."""
    assert _append(_kv(), tokens=0, q=None, k=None, v=None, q_out=None) == 0
    assert _attn(_kv(), tokens=0, q=None, out=None) == 0


def _ws(kv, tokens, nh, max_new, max_keys):
    return gsvk.lib().gsvk_attn_paged_workspace_bytes(C.byref(kv), tokens, nh, max_new, max_keys, 0)


def test_more_work_than_a_launch_holds_is_refused():
    """2^32 threads or more: said before the launch."""
    assert _append(_kv(n_kv=16, hd=128), tokens=2 ** 25, nh=64, qs=8192, ks=2048, vs=2048) == 1
    assert "too many" in gsvk.last_error()
    assert _attn(_kv(n_kv=8, hd=64, B=65535), tokens=2 ** 24, nh=64, qs=4096, os_=4096, max_new=8192, max_keys=8192) == 1
    assert "too many" in gsvk.last_error()


def test_workspace_is_asked_for():
    """One long sequence is split over its keys: a call without the workspace it needs is refused; one
    short sequence needs none."""
    kv = _kv(table_stride=10000, table_cols=10000, n_pages=10000, B=1)
    need = _ws(kv, 1, 4, 1, 100000)
    assert need > 0
    assert _attn(kv, tokens=1, max_new=1, max_keys=100000) == 1
    assert "workspace" in gsvk.last_error()
    assert _attn(kv, tokens=1, max_new=1, max_keys=100000, ws=4096, ws_bytes=need - 1) == 1
    assert _attn(kv, tokens=1, max_new=1, max_keys=100000, ws=4104, ws_bytes=need) == 1
    assert _ws(kv, 1, 4, 1, 16) == 0
    assert _ws(_kv(hd=48), 1, 4, 1, 100000) == 0      # (arguments that the call itself refuses)
    assert gsvk.lib().gsvk_attn_paged_workspace_bytes(None, 1, 4, 1, 100000, 0) == 0
