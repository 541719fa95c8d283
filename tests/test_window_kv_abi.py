"""What window attention and the key/value cache refuse, and calls without work; no GPU:
each check precedes the first device call."""
from __future__ import annotations

import ctypes

import pytest

import kvops as K
import lmops as M


@pytest.fixture(scope="module")
def L():
    return K.lib()


X = 4096  # an address that is never read


def window(L, B=1, H=2, Hkv=1, T=4, d=64, window=2, sinks=0, st=None, p=X, bwd=False, ws=(X, 1 << 40)):
    s = (ctypes.c_int64 * 24)(*(st or [H * T * d, T * d, d] * 8))
    if bwd:
        return L.aar_window_attn_bwd_f32(*[p] * 9, B, H, Hkv, T, d, s, window, sinks, 1.0, *ws, None)
    return L.aar_window_attn_fwd_f32(*[p] * 5, B, H, Hkv, T, d, s, window, sinks, 1.0, None, 0, None)


@pytest.mark.parametrize("bwd", [False, True])
def test_window_refusals(L, bwd):
    for bad in ({"B": -1}, {"H": -1}, {"Hkv": 0}, {"T": -1}, {"d": 0}, {"d": 129}, {"H": 3, "Hkv": 2}, {"window": 0},
                {"window": -5}, {"sinks": -1}, {"p": None}):
        assert window(L, bwd=bwd, **bad) == M.EINVAL, bad
    for bad in ({"T": (1 << 24) + 1}, {"B": (1 << 20) + 1}, {"H": 1 << 21, "Hkv": 1}, {"B": 1 << 19, "H": 32, "Hkv": 32},
                {"st": [512, 256, 63] * 8}, {"st": [512, 256, -64] * 8}, {"st": [512, 256, 0] * 8},
                {"st": [512, 256, (1 << 23) + 4] * 8}):
        assert window(L, bwd=bwd, **bad) == M.EUNSUPPORTED, bad
    for none in ({"B": 0}, {"T": 0}, {"H": 0, "Hkv": 0}):
        assert window(L, bwd=bwd, p=None, **none) == 0, none


def test_window_workspace(L):
    assert window(L, bwd=True, ws=(None, 0)) == M.EWORKSPACE
    need = L.aar_window_attn_bwd_workspace_bytes(1, 2, 1, 4, 64, 2, 0)
    assert need >= 4 * 2 * 4
    assert window(L, bwd=True, ws=(X, need - 1)) == M.EWORKSPACE
    assert window(L, bwd=True, ws=(X + 4, need)) == M.EWORKSPACE
    assert L.aar_window_attn_bwd_workspace_bytes(1, 2, 1, 4, 64, 0, 0) == 0
    # a forward of a text that LDS holds needs none
    assert L.aar_window_attn_fwd_workspace_bytes(1, 2, 1, 256, 64, 2, 0) == 0
    assert L.aar_window_attn_fwd_workspace_bytes(1, 2, 1, 257, 64, 2, 0) > 0
    assert window(L, T=300) == M.EWORKSPACE
    # sinks of any number: a few hundred parts at most
    for sinks in (1, 100, 5000, 1 << 40):
        assert L.aar_window_attn_bwd_workspace_bytes(1, 1, 1, 1 << 20, 64, 16, sinks) < 1 << 31


def cache(**kw):
    f = {"pages": X, "scales": X, "open": X, "table": X, "sequences": 2, "table_width": 4, "n_pages": 8, "kv_heads": 2,
         "page": 64, "d": 64}
    f.update(kw)
    return K.Cache(*(f[n] for n, _ in K.Cache._fields_))


def calls(L, c, p=X, T=1, H=4, window=1, sinks=0):
    st = (ctypes.c_int64 * 6)(*[512, 64, 64] * 2) if p else None
    r = ctypes.byref(c) if c is not None else None
    return (L.aar_kv_cache_append_f32(r, p, p, st, p, None, T, None, None),
            L.aar_kv_cache_read_f32(r, None, p, p, p, st, T, None, None),
            L.aar_kv_cache_attn_f32(r, p, p, st, p, None, H, T, window, sinks, 1.0, None, 0, None, None))


def test_cache_refusals(L):
    assert calls(L, None) == (M.EINVAL,) * 3
    for bad in ({"sequences": -1}, {"table_width": -1}, {"n_pages": -1}, {"kv_heads": 0}, {"d": 0}, {"d": 129},
                {"page": 16}, {"page": 96}, {"page": 0}, {"page": 256}, {"page": -64}):
        assert calls(L, cache(**bad)) == (M.EINVAL,) * 3, bad
    for bad in ({"table_width": (1 << 24) + 1}, {"kv_heads": (1 << 16) + 1}, {"sequences": (1 << 22) + 1},
                {"sequences": 1 << 21, "kv_heads": 4}, {"n_pages": 1 << 41}):
        assert calls(L, cache(**bad)) == (M.EUNSUPPORTED,) * 3, bad
    for bad in ({"pages": X + 8}, {"pages": None}, {"scales": None}, {"table": None}):
        assert calls(L, cache(**bad)) == (M.EINVAL,) * 3, bad
    assert calls(L, cache(open=None))[0] == M.EINVAL
    assert calls(L, cache(), p=None) == (M.EINVAL,) * 3
    assert calls(L, cache(), T=-1) == (M.EINVAL,) * 3
    assert calls(L, cache(), T=(1 << 30) + 1) == (M.EUNSUPPORTED,) * 3
    for bad in ({"H": 3}, {"H": 0}, {"window": 0}, {"sinks": -1}):
        assert calls(L, cache(sequences=0), **bad)[2] == M.EINVAL, bad
    for bad in ({"T": 1 << 24, "H": 4}, {"H": 1 << 25}):
        assert calls(L, cache(), **bad)[2] == M.EUNSUPPORTED, bad
    # no sequences, or no tokens
    assert calls(L, cache(sequences=0), p=None) == (0, 0, 0)
    assert calls(L, cache(), p=None, T=0) == (0, 0, 0)


def test_page_bytes(L):
    assert L.aar_kv_cache_page_bytes(2, 64, 64) == 2 * 2 * 64 * 64
    assert L.aar_kv_cache_page_bytes(3, 32, 30) == 3 * 2 * 32 * 32
    assert L.aar_kv_cache_page_bytes(1, 128, 1) == 2 * 128 * 16
    for bad in ((0, 64, 64), (1, 16, 64), (1, 64, 0), (1, 64, 129)):
        assert L.aar_kv_cache_page_bytes(*bad) == 0
