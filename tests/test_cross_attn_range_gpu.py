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
