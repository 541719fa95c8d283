"""CPU checks of the encoder-reading decoder's operators: what their entry points
refuse before any launch, workspace sizes, and the host layer's argument checks."""
from __future__ import annotations

import numpy as np
import pytest

import lmops as M

X = 4096  # a pointer that is never dereferenced: every call below returns before any device work


@pytest.fixture(scope="module")
def L():
    return M.lib()


def st(n):
    return (M.I64 * n)(*([64] * n))


def test_cross_attention_refusals(L):
    def fwd(B=1, H=4, Hkv=2, Tq=3, Tk=5, d=64, q=X, k=X, v=X, o=X, lse=X, strides=st(12), ws=None, nb=0):
        return L.aar_cross_attn_fwd_f32(q, k, v, None, o, lse, B, H, Hkv, Tq, Tk, d, strides, 1.0, ws, nb, None)

    for bad in ({"B": -1}, {"H": -4}, {"Hkv": -2}, {"Tq": -1}, {"Tk": -1}, {"d": 0}, {"d": 129}, {"Hkv": 3}, {"Hkv": 0},
                {"H": 0}, {"q": None}, {"k": None}, {"v": None}, {"o": None}, {"lse": None}, {"strides": None}):
        assert fwd(**bad) == M.EINVAL, bad
    for big in ({"B": 1 << 25}, {"Tq": 1 << 25}, {"Tk": 1 << 25}, {"B": 1 << 20, "H": 64, "Hkv": 64},
                {"Tq": 1 << 24, "H": 64, "Hkv": 1}):
        assert fwd(**big) == M.EUNSUPPORTED, big
    assert fwd(B=0) == 0 and fwd(Tq=0, q=None, o=None, lse=None) == 0 and fwd(H=0, Hkv=0) == 0
    # few rows against many keys: the key range is split, and the parts need their room
    nb = L.aar_cross_attn_fwd_workspace_bytes(1, 4, 2, 1, 4096, 64)
    assert nb > 0 and nb % 4 == 0
    assert fwd(Tq=1, Tk=4096) == M.EWORKSPACE and fwd(Tq=1, Tk=4096, ws=X, nb=nb - 1) == M.EWORKSPACE
    assert fwd(Tq=1, Tk=4096, ws=X + 4, nb=nb) == M.EWORKSPACE
    assert L.aar_cross_attn_fwd_workspace_bytes(64, 6, 6, 256, 577, 64) == 0
    assert L.aar_cross_attn_fwd_workspace_bytes(1, 4, 3, 1, 4096, 64) == 0

    def bwd(B=1, H=4, Hkv=2, Tq=3, Tk=5, d=64, ptrs=(X,) * 9, strides=st(24), ws=X, nb=1 << 40):
        q, k, v, o, lse, do, dq, dk, dv = ptrs
        return L.aar_cross_attn_bwd_f32(q, k, v, None, o, lse, do, dq, dk, dv, B, H, Hkv, Tq, Tk, d, strides, 1.0, ws, nb,
                                        None)

    for bad in ({"B": -1}, {"d": 129}, {"Hkv": 3}, {"strides": None}, {"H": 0}):
        assert bwd(**bad) == M.EINVAL, bad
    for i in range(9):
        assert bwd(ptrs=(X,) * i + (None,) + (X,) * (8 - i)) == M.EINVAL, i
    assert bwd(ws=None) == M.EWORKSPACE and bwd(nb=3 * 4 * 4 - 1) == M.EWORKSPACE
    assert L.aar_cross_attn_bwd_workspace_bytes(1, 4, 2, 3, 5, 64) >= 3 * 4 * 4
    assert bwd(B=0) == 0 and bwd(Tq=0, Tk=0, ptrs=(None,) * 9) == 0


def test_qk_norm_rope_refusals(L):
    def fwd(x=X, xr=256, wq=X, wk=X, pos=X, n=4, y=X + 65536, yr=256, rows=4, hq=2, hk=2, d=64, r=64, base=1e4, eps=1e-6):
        return L.aar_qk_norm_rope_fwd_f32(x, xr, wq, wk, pos, n, y, yr, rows, hq, hk, d, r, base, eps, None)

    def bwd(gy=X, gr=256, x=X, xr=256, wq=X, wk=X, pos=X, n=4, dx=X + 65536, dr=256, dwq=X, dwk=X, rows=4, hq=2, hk=2, d=64,
            r=64, base=1e4, eps=1e-6, ws=X, nb=1 << 30):
        return L.aar_qk_norm_rope_bwd_f32(gy, gr, x, xr, wq, wk, pos, n, dx, dr, dwq, dwk, rows, hq, hk, d, r, base, eps, ws,
                                          nb, None)

    inf, nan = float("inf"), float("nan")
    for call in (fwd, bwd):
        for bad in ({"rows": -1}, {"hq": -1}, {"hk": -1}, {"d": 1}, {"d": 0}, {"r": 63}, {"r": 66}, {"r": -2}, {"base": 0.0},
                    {"base": -1.0}, {"base": inf}, {"base": nan}, {"eps": -1.0}, {"eps": nan}, {"eps": inf}, {"n": 3},
                    {"n": 0}, {"pos": None}, {"x": None}, {"wq": None}, {"wk": None}, {"xr": 255}):
            assert call(**bad) == M.EINVAL, bad
        assert call(d=258, r=258) == M.EUNSUPPORTED and call(rows=1 << 41, n=1) == M.EUNSUPPORTED
    assert fwd(y=None) == M.EINVAL and fwd(yr=255) == M.EINVAL and fwd(y=X, yr=512) == M.EINVAL
    assert fwd(rows=0) == 0 and fwd(hq=0, hk=0) == 0
    for bad in ({"gy": None}, {"dx": None}, {"dwq": None}, {"dwk": None}, {"gr": 255}, {"dr": 255}, {"dx": X, "dr": 512}):
        assert bwd(**bad) == M.EINVAL, bad
    nb = L.aar_qk_norm_rope_bwd_workspace_bytes(4, 2, 2, 64)
    assert nb > 0 and bwd(ws=None) == M.EWORKSPACE and bwd(nb=nb - 1) == M.EWORKSPACE
    assert L.aar_qk_norm_rope_bwd_workspace_bytes(0, 2, 2, 64) == 0 and L.aar_qk_norm_rope_bwd_workspace_bytes(4, 2, 2, 300) == 0


def test_embedding_refusals(L):
    def fwd(w=X, ids=X, out=X, n=4, vocab=8, dim=4):
        return L.aar_embedding_scaled_fwd_f32(w, ids, out, n, vocab, dim, 1.0, None, None)

    def bwd(g=X, ids=X, dw=X, n=4, vocab=8, dim=4, ws=X, nb=1 << 40):
        return L.aar_embedding_sorted_bwd_f32(g, ids, dw, n, vocab, dim, 1.0, ws, nb, None)

    for bad in ({"n": -1}, {"vocab": -1}, {"dim": -1}, {"w": None}, {"ids": None}, {"out": None}):
        assert fwd(**bad) == M.EINVAL, bad
    for bad in ({"n": -1}, {"vocab": -1}, {"dim": -1}, {"g": None}, {"ids": None}, {"dw": None}):
        assert bwd(**bad) == M.EINVAL, bad
    assert fwd(n=0) == 0 and fwd(dim=0) == 0 and bwd(vocab=0) == 0 and bwd(dim=0) == 0
    assert fwd(n=1 << 40) == M.EUNSUPPORTED
    for big in ({"n": 1 << 31}, {"vocab": 1 << 31}, {"dim": 1 << 31}):
        assert bwd(**big) == M.EUNSUPPORTED
    nb = L.aar_embedding_sorted_bwd_workspace_bytes(4, 8, 4)
    assert nb > 0 and bwd(ws=None) == M.EWORKSPACE and bwd(nb=nb - 1) == M.EWORKSPACE and bwd(ws=X + 8) == M.EWORKSPACE
    assert L.aar_embedding_sorted_bwd_workspace_bytes(0, 8, 4) == 0


def test_distill_refusals(L):
    def fwd(z=X, t=X, ids=X, loss=X, stats=X, n=4, vocab=8, top=2, tau=1.0, ws=X, nb=16):
        return L.aar_distill_fwd_f32(z, t, ids, loss, stats, n, vocab, top, tau, None, ws, nb, None)

    def bwd(grad=X, z=X, t=X, ids=X, stats=X, dz=X, n=4, vocab=8, top=2, tau=1.0):
        return L.aar_distill_bwd_f32(grad, z, t, ids, stats, dz, n, vocab, top, tau, None)

    for call in (fwd, bwd):
        for bad in ({"n": -1}, {"vocab": 0}, {"top": 0}, {"tau": 0.0}, {"tau": -1.0}, {"tau": float("nan")},
                    {"tau": float("inf")}, {"z": None}, {"t": None}, {"ids": None}, {"stats": None}):
            assert call(**bad) == M.EINVAL, bad
        assert call(top=1025) == M.EUNSUPPORTED and call(vocab=1 << 31) == M.EUNSUPPORTED and call(n=1 << 40) == M.EUNSUPPORTED
    assert fwd(loss=None) == M.EINVAL and bwd(grad=None) == M.EINVAL and bwd(dz=None) == M.EINVAL
    assert fwd(ws=None) == M.EWORKSPACE and fwd(nb=15) == M.EWORKSPACE and bwd(n=0) == 0
    assert L.aar_distill_workspace_bytes(4) == 16 and L.aar_distill_workspace_bytes(-1) == 0


def test_host_checks(ag):
    f = lambda *s: ag.from_numpy(np.zeros(s, np.float32))  # noqa: E731
    i = lambda *s: ag.from_numpy(np.zeros(s, np.int64))  # noqa: E731
    q, k = f(2, 4, 3, 8), f(2, 2, 5, 8)
    for args, msg in (((f(2, 3, 8), k, k), "4D"), ((q, k, f(2, 2, 6, 8)), "share shape"), ((q, f(3, 2, 5, 8), f(3, 2, 5, 8)), "batch"),
                      ((q, f(2, 2, 5, 4), f(2, 2, 5, 4)), "head dim"), ((q, f(2, 3, 5, 8), f(2, 3, 5, 8)), "multiple"),
                      ((f(2, 4, 3, 136), f(2, 2, 5, 136), f(2, 2, 5, 136)), "d_head"), ((i(2, 4, 3, 8), k, k), "only Fp32"),
                      ((q, k, k, f(2)), "Int64"), ((q, k, k, i(3)), "1D"), ((q, k, k, i(2, 1)), "1D")):
        with pytest.raises(ValueError, match=msg):
            ag.cross_attention(*args)
    packed = ag._core._cross_attention_packed
    for args, msg in (((f(2, 3, 32), f(2, 5, 30), 4, 2), "last dims"), ((f(2, 3, 32), f(3, 5, 32), 4, 2), "need q"),
                      ((f(2, 3, 32), f(2, 5, 32), 4, 3), "multiple"), ((f(2, 3, 30), f(2, 5, 32), 4, 2), "last dims"),
                      ((f(2, 3, 32), f(2, 5, 32), 0, 0), "multiple")):
        with pytest.raises(ValueError, match=msg):
            packed(*args)
    x, w, p = f(2, 3, 32), f(8), i(3)
    for args, msg in (((x, w, w, p, 3, 2), "heads"), ((x, w, w, p, -1, 5), "negative"), ((x, f(9), w, p, 2, 2), "weights"),
                      ((x, w, w, p, 2, 2, 7), "rotary_dim"), ((x, w, w, p, 2, 2, 10), "rotary_dim"), ((x, w, w, None, 2, 2), "positions"),
                      ((x, w, w, i(4), 2, 2), "positions"), ((x, w, w, f(3), 2, 2), "Int64"), ((x, w, w, p, 2, 2, 8, -1.0), "base"),
                      ((x, w, w, p, 2, 2, 8, 1e4, -1.0), "eps"), ((f(2, 3, 4), f(1), f(1), p, 2, 2), "d_head")):
        with pytest.raises(ValueError, match=msg):
            ag.qk_norm_rope(*args)
    for args, msg in (((f(4), i(2), 1.0), "2D"), ((f(4, 2), f(2), 1.0), "Int64"), ((i(4, 2), i(2), 1.0), "Fp32")):
        with pytest.raises(ValueError, match=msg):
            ag.embedding_scaled(*args)
    for args, msg in (((f(4), f(4, 2), i(4, 2)), "2D"), ((f(4, 9), f(3, 2), i(3, 2)), r"\(N, K\)"), ((f(4, 9), f(4, 3), i(4, 2)), r"\(N, K\)"),
                      ((f(4, 9), f(4, 2), f(4, 2)), "Int64"), ((f(4, 9), f(4, 2), i(4, 2), 0.0), "temperature"),
                      ((f(4, 9), f(4, 0), i(4, 0)), "K must"), ((f(4, 0), f(4, 2), i(4, 2)), "vocabulary")):
        with pytest.raises(ValueError, match=msg):
            ag.distill_loss(*args)
    # well-formed calls on host tensors: this build computes on the GPU only
    for call in (lambda: ag.cross_attention(q, k, k, i(2)), lambda: packed(f(2, 3, 32), f(2, 5, 32), 4, 2),
                 lambda: ag.qk_norm_rope(x, w, w, p, 2, 2), lambda: ag.qk_norm_rope(x, w, w, None, 2, 2, 0),
                 lambda: ag._core._flash_attention_qkv_rope(f(2, 3, 48), w, w, p, 2, True),
                 lambda: ag.embedding_scaled(f(4, 2), i(2), 1.0), lambda: ag.distill_loss(f(4, 9), f(4, 2), i(4, 2))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_modules(ag):
    nn = ag.nn
    rng = lambda: np.random.default_rng(1)  # noqa: E731
    m = nn.CrossAttention(96, 6, d_context=40, n_kv_heads=2, rng=rng())
    assert [p.tensor.shape for p in m.parameters()] == [[96, 96], [96], [64, 40], [64], [96, 96], [96]]
    for bad in (dict(d_model=95, n_heads=6), dict(d_model=96, n_heads=6, n_kv_heads=4), dict(d_model=96, n_heads=6, n_kv_heads=0)):
        with pytest.raises(ValueError):
            nn.CrossAttention(**bad)
    # without norms the attention draws, holds and checks what it did
    a, b = nn.MultiHeadAttention(64, 4, rng=rng()), nn.MultiHeadAttention(64, 4, rng=rng(), qk_norm=True)
    pa, pb = list(a.parameters()), list(b.parameters())
    assert len(pa) == 4 and len(pb) == 6
    for x, y in zip(pa, pb[2:]):
        np.testing.assert_array_equal(ag.to_numpy(x.tensor), ag.to_numpy(y.tensor))
    f = lambda *s: ag.from_numpy(np.zeros(s, np.float32))  # noqa: E731
    with pytest.raises(RuntimeError, match="GPU only"):
        b(f(2, 3, 64))
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            nn.DistillationLoss(bad)
    e, s = nn.Embedding(9, 4, rng=rng()), nn.Embedding(9, 4, rng=rng(), scale=2.0)
    np.testing.assert_array_equal(ag.to_numpy(e.weight.tensor), ag.to_numpy(s.weight.tensor))
