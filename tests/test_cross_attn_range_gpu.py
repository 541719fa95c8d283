"""Cross attention's magnitudes: operands that are large or small together, rows of
any size with small columns, and terms far below a row's largest."""
from __future__ import annotations

import math

import pytest
import torch

import lmops as M
from test_cross_attn_gpu import rand, run

pytestmark = pytest.mark.gpu

NAMES = ("o", "lse", "dq", "dk", "dv")


@pytest.fixture(scope="module")
def L(gpu):
    return M.lib()


def hide(q, k, keys, score, unit=1.0):
    """Column 0 gives `keys` a score of about `score`, the others none."""
    q[..., 0] = 8.0 * unit
    k[..., 0] = 0.0
    k[:, :, keys, 0] = score / (8.0 * q.shape[-1] ** -0.5) / unit


@pytest.mark.parametrize("d", [64, 128, 30])
@pytest.mark.parametrize("Hkv", [2, 1])
def test_keys_without_weight_beside_large_operands(L, d, Hkv):
    """P = 0 for a wave's 32 keys whose values are large, as Q and dO are: dP - D is
    finite, its product with Q's magnitude is not, and dK is 0."""
    big = 2.0 ** 45
    q, do = rand(1, 1, 2, 50, d) * big, rand(2, 1, 2, 50, d) * 2.0 ** 50
    k, v = rand(3, 1, Hkv, 100, d) / big, rand(4, 1, Hkv, 100, d)
    keys = slice(32, 64)
    hide(q, k, keys, -200.0, big)
    v[:, :, keys] *= 2.0 ** 50
    got, ref, mass = run(L, q, k, v, None, do), M.cross_exact(q, k, v, None, do), M.cross_mass(q, k, v, None, do)
    assert (got[3][:, :, keys] == 0).all() and (got[4][:, :, keys] == 0).all()
    for name, a, b in zip(NAMES, got, ref):
        # scores up to 6 beside the 200 that the first column adds
        M.near(a, b, M.attn_tol(d, 100, 206.0) * (2 if name[0] == "d" else 1), name, mass.get(name))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("e", [-50, -58, -62, -90])
def test_small_columns_of_small_rows(L, d, e):
    """Rows of magnitude 2^e whose columns but the first are 2^-20 of it: each is held to
    2^-38 of the row's largest element, as rows of ordinary size are."""
    f, small = 2.0 ** e, 2.0 ** -20
    q, do = rand(1, 1, 2, 50, d), rand(2, 1, 2, 50, d)
    k, v = rand(3, 1, 2, 70, d), rand(4, 1, 2, 70, d)
    tol = M.attn_tol(d, 70)

    def columns(got, ref, weight, x, what):
        # off by 2^-38 of x's largest a term, and by the sums' roundings, times the terms' weights
        bound = weight * (2.0 ** -38 * x.abs().max().item() + 8 * tol * x[..., 1:].abs().max().item())
        assert (got.double().cpu() - ref)[..., 1:].abs().max().item() <= bound, what

    def shrink(x):
        x = x * f
        x[..., 1:] *= small
        return x

    # O = P V: weights of a row add up to 1
    x = shrink(v)
    columns(run(L, q, k, x, None)[0], M.cross_exact(q, k, x)[0], 1.0, x, "o")
    # dV = P^T dO: weights of a key add up to less than the number of rows
    x = shrink(do)
    columns(run(L, q, k, v, None, x)[4], M.cross_exact(q, k, v, None, x)[4], 50.0, x, "dv")
    # dQ = scale dS K; sum_j |dS_ij| <= 2 max |dO . v|
    ds = 2 * (do @ v.transpose(2, 3)).abs().max().item() * d ** -0.5
    x = shrink(k)
    columns(run(L, q, x, v, None, do)[2], M.cross_exact(q, x, v, None, do)[2], ds, x, "dq")
    # dK = scale dS^T Q
    x = shrink(q)
    columns(run(L, x, k, v, None, do)[3], M.cross_exact(x, k, v, None, do)[3], 50 * ds, x, "dk")


@pytest.mark.parametrize("d", [64, 128, 30])
@pytest.mark.parametrize("score", [-60.0, -70.0, -78.0])
def test_keys_of_tiny_weight(L, d, score):
    """Keys that every row gives a weight of 2^-91 to 2^-120: their gradients, as small,
    keep their digits."""
    q, do = rand(1, 1, 2, 50, d), rand(2, 1, 2, 50, d)
    k, v = rand(3, 1, 2, 100, d) * 0.25, rand(4, 1, 2, 100, d)
    keys = slice(32, 64)
    hide(q, k, keys, score)
    _, _, _, dk, dv = run(L, q, k, v, None, do)
    _, _, _, rk, rv = M.cross_exact(q, k, v, None, do)
    s = (q.double().cpu() @ k.double().cpu().transpose(2, 3)) * d ** -0.5
    p = torch.softmax(s, -1)
    # a weight is off by its score's roundings, a gradient by that of its terms' magnitudes
    tol = M.attn_tol(d, 100, 90.0)
    assert 2.0 ** -126 < p[..., keys].min() and p[..., keys].max() < 2.0 ** -70
    mass = {"dv": p.transpose(2, 3) @ do.double().cpu().abs(), "dk": M.cross_mass(q, k, v, None, do)["dk"]}
    for name, g, r in (("dv", dv, rv), ("dk", dk, rk)):
        err = (g.double().cpu() - r).abs()[:, :, keys]
        # results below 2^-126 are whole steps of 2^-149, as the weights' exponentials end at 2^-126
        bound = 2 * tol * mass[name][:, :, keys] + 50 * 2.0 ** -149
        assert (err <= bound).all(), (name, (err / bound).max().item())
