"""Cross attention (aar_cross_attn_*, ag.cross_attention, nn.CrossAttention) on
the GPU against its definition in 64 bits: lengths from none to long, odd sizes,
padded contexts (rows without keys, garbage behind the lengths), shared heads,
strided and unaligned operands, other streams and captured graphs."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import lmops as M
from devutil import dev, host

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L(gpu):
    return M.lib()


def rand(seed, *shape, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).cuda()


def run(L, q, k, v, lens, do=None, scale=None):
    B, H, Tq, d = q.shape
    o, lse = torch.full_like(q, 7.0, memory_format=torch.contiguous_format), torch.full((B, H, Tq), 7.0, device="cuda")
    M.cross_fwd(L, q, k, v, lens, o, lse, scale)
    if do is None:
        return o, lse
    dq, dk, dv = (torch.full(t.shape, 7.0, device="cuda") for t in (q, k, v))
    M.cross_bwd(L, q, k, v, lens, o, lse, do, dq, dk, dv, scale)
    return o, lse, dq, dk, dv


def check(L, q, k, v, lens, do, scale=None, smax=6.0):
    got = run(L, q, k, v, lens, do, scale)
    ref = M.cross_exact(q, k, v, lens, do, scale)
    tol = M.attn_tol(q.shape[-1], max(k.shape[2], q.shape[2] * q.shape[1] // k.shape[1]), smax)
    mass = M.cross_mass(q, k, v, lens, do, scale)
    for name, g, r in zip(("o", "lse", "dq", "dk", "dv"), got, ref):
        # dS is a difference of two sums of their own: twice the roundings
        M.near(g, r, tol * (2 if name[0] == "d" else 1), name, mass.get(name))


# B, H, Hkv, Tq, Tk, d
SHAPES = [
    (1, 1, 1, 1, 1, 64), (2, 3, 3, 1, 5, 64), (3, 2, 2, 1, 300, 64), (2, 4, 1, 1, 777, 128), (1, 8, 1, 1, 65, 32),
    (2, 6, 2, 2, 129, 40), (1, 2, 2, 7, 1000, 64), (1, 2, 2, 8, 31, 30), (2, 3, 3, 9, 33, 64), (1, 5, 5, 31, 64, 128),
    (2, 2, 2, 32, 32, 64), (1, 3, 3, 33, 31, 96), (2, 4, 2, 100, 65, 64), (1, 2, 1, 129, 200, 36), (1, 1, 1, 300, 1, 64),
    (1, 2, 2, 257, 577, 64), (2, 8, 4, 65, 300, 128), (1, 3, 3, 50, 70, 1), (1, 2, 2, 40, 90, 3), (1, 2, 2, 64, 2049, 64),
    (4, 12, 12, 130, 260, 64), (1, 1, 1, 2000, 40, 64), (1, 1, 1, 1, 8192, 64), (16, 16, 16, 140, 140, 64),
    (2, 2, 2, 3, 150, 30), (2, 4, 2, 2, 65, 64), (1, 1, 1, 4, 2100, 96), (3, 3, 3, 4, 1, 128), (2, 2, 2, 5, 500, 64),
    (1, 3, 3, 8, 1030, 128), (2, 6, 2, 3, 70, 30), (1, 1, 1, 9, 300, 32), (2, 4, 2, 70, 130, 32),
    (1, 2, 2, 40, 90, 4), (1, 3, 3, 2000, 33, 16), (1, 1, 1, 40, 3000, 32),
]


@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_definition(L, shape):
    B, H, Hkv, Tq, Tk, d = shape
    q, do = rand(1, B, H, Tq, d), rand(2, B, H, Tq, d)
    k, v = rand(3, B, Hkv, Tk, d), rand(4, B, Hkv, Tk, d)
    check(L, q, k, v, None, do)


@pytest.mark.parametrize("shape", [(5, 2, 2, 1, 200, 64), (5, 4, 2, 3, 100, 128), (5, 2, 2, 40, 200, 64),
                                   (5, 4, 2, 2, 100, 128), (5, 2, 2, 3, 700, 30),
                                   (5, 4, 1, 70, 333, 36), (5, 3, 3, 200, 130, 30), (5, 2, 2, 33, 900, 64)])
def test_padded_contexts(L, shape):
    """Lengths none, one, a tile's border, some and all; what stands behind them is
    never read: infinities and NaN there change nothing."""
    B, H, Hkv, Tq, Tk, d = shape
    q, do = rand(1, B, H, Tq, d), rand(2, B, H, Tq, d)
    k, v = rand(3, B, Hkv, Tk, d), rand(4, B, Hkv, Tk, d)
    lens = torch.tensor([0, 1, 32, Tk // 2 + 1, Tk], device="cuda")
    check(L, q, k, v, lens, do)
    clean = run(L, q, k, v, lens, do)
    for b in range(B):
        n = int(lens[b])
        k[b, :, n:] = math.nan
        v[b, :, n:] = math.inf
    dirty = run(L, q, k, v, lens, do)
    for a, b in zip(clean, dirty):
        assert torch.equal(a, b)
    o, lse, dq, dk, dv = dirty
    assert (o[0] == 0).all() and (lse[0] == -math.inf).all() and (dq[0] == 0).all()
    for b in range(B):
        assert (dk[b, :, int(lens[b]):] == 0).all() and (dv[b, :, int(lens[b]):] == 0).all()
    # lengths outside [0, Tk] count as its ends
    odd = torch.tensor([-5, 1, 32, Tk // 2 + 1, Tk + 1000], device="cuda")
    for a, b in zip(dirty, run(L, q, k, v, odd, do)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("Tq", [1, 5, 40])
def test_no_keys_and_no_queries(L, Tq):
    q, do = rand(1, 2, 4, Tq, 64), rand(2, 2, 4, Tq, 64)
    k = torch.empty(2, 2, 0, 64, device="cuda")
    o, lse, dq, dk, dv = run(L, q, k, k, None, do)
    assert (o == 0).all() and (lse == -math.inf).all() and (dq == 0).all() and dk.numel() == 0
    k = rand(3, 2, 2, 50, 64)
    none = torch.empty(2, 4, 0, 64, device="cuda")
    o, lse, dq, dk, dv = run(L, none, k, k, None, none)
    assert (dk == 0).all() and (dv == 0).all()


@pytest.mark.parametrize("Tq", [1, 6, 90])
@pytest.mark.parametrize("d", [64, 128, 36])
def test_strided_operands(L, Tq, d):
    """Packed projections, rows and heads in other orders, unaligned bases."""
    B, H, Hkv, Tk = 2, 4, 2, 150
    qp, kv = rand(1, B, Tq, H, d), rand(2, B, Tk, 2, Hkv, d)
    do = rand(3, B, Tq, H, d)
    q, k, v = qp.permute(0, 2, 1, 3), kv[:, :, 0].permute(0, 2, 1, 3), kv[:, :, 1].permute(0, 2, 1, 3)
    ref = M.cross_exact(q, k, v, None, do.permute(0, 2, 1, 3))
    tol = 2 * M.attn_tol(d, Tk)
    dense = run(L, q.contiguous(), k.contiguous(), v.contiguous(), None, do.permute(0, 2, 1, 3).contiguous())
    for offset in (0, 1):  # unaligned by one float: the element-wise path
        def at(t):
            buf = torch.empty(t.numel() + 8, device="cuda")
            got = torch.as_strided(buf, t.shape, t.stride(), offset)
            got.copy_(t)
            return got
        q1, do1 = at(qp).permute(0, 2, 1, 3), at(do).permute(0, 2, 1, 3)
        kv1 = at(kv)
        k1, v1 = kv1[:, :, 0].permute(0, 2, 1, 3), kv1[:, :, 1].permute(0, 2, 1, 3)
        o, dq = at(torch.zeros_like(qp)).permute(0, 2, 1, 3), at(torch.zeros_like(qp)).permute(0, 2, 1, 3)
        dkv = at(torch.zeros_like(kv))
        dk, dv = dkv[:, :, 0].permute(0, 2, 1, 3), dkv[:, :, 1].permute(0, 2, 1, 3)
        lse = torch.empty(B, H, Tq, device="cuda")
        M.cross_fwd(L, q1, k1, v1, None, o, lse)
        M.cross_bwd(L, q1, k1, v1, None, o, lse, do1, dq, dk, dv)
        for name, g, r, x in zip(("o", "lse", "dq", "dk", "dv"), (o, lse, dq, dk, dv), ref, dense):
            M.near(g, r, tol, name)
            if offset == 0:
                assert torch.equal(g, x), name


@pytest.mark.parametrize("d", [64, 30])
def test_broadcast_operands(L, d):
    """Expanded keys, values and queries: strides of zero."""
    q = rand(1, 1, 1, 40, d).expand(2, 4, 40, d)
    k, v = rand(2, 2, 2, 1, d).expand(2, 2, 70, d), rand(3, 1, 1, 70, d).expand(2, 2, 70, d)
    do = rand(4, 2, 4, 1, d).expand(2, 4, 40, d)
    lens = torch.tensor([70, 33], device="cuda")
    check(L, q, k, v, lens, do)
    x = v.contiguous()
    x[1, :, 33:] = math.inf
    x[0, 0, 5, 3] = math.inf  # an infinite value, and expanded keys behind the length
    o, lse = run(L, q, k, x, lens)
    ro, _ = M.cross_exact(q, k, x, lens)
    M.near(o, ro, M.attn_tol(d, 70), "o")


@pytest.mark.parametrize("Tq", [1, 40])
def test_far_rows(L, Tq):
    """Rows and heads whose offsets pass 31 and 32 bits: a cache of 2^32 elements, heads of
    a group 2^29 apart, rows 2^24 apart."""
    H, Tk, d = 2, 70000, 64
    rows = torch.empty(Tk * 65536, device="cuda").view(Tk, 65536)  # 2^32 elements and more
    k, v = (torch.as_strided(rows, (1, 1, Tk, d), (0, 0, 65536, 1), at) for at in (0, 64))
    k.copy_(rand(2, 1, 1, Tk, d))
    v.copy_(rand(3, 1, 1, Tk, d))
    q, do = rand(1, 1, H, Tq, d), rand(4, 1, H, Tq, d)
    check(L, q, k, v, None, do)
    del k, v
    flat = rows.view(-1)
    k, v = rand(2, 1, 1, 90, d), rand(3, 1, 1, 90, d)
    for sh, st in ((2 ** 29, d), (d, 2 ** 24)):
        qf = torch.as_strided(flat, (1, H, Tq, d), (0, sh, st, 1))
        qf.copy_(q)
        check(L, qf, k, v, None, do)
    kf = torch.as_strided(flat, (1, 1, 90, d), (0, 0, 2 ** 24, 1))
    kf.copy_(k)
    check(L, q, kf, v, None, do)


@pytest.mark.parametrize("Tq", [1, 50])
def test_extreme_scores(L, Tq):
    """Scores of +-1000 (one key takes all), all keys equal, a negative scale, and
    keys of -inf that leave a row nothing."""
    q, k, v = rand(1, 1, 2, Tq, 64), rand(2, 1, 2, 100, 64), rand(3, 1, 2, 100, 64)
    o, lse = run(L, q, k, v, None, scale=100.0)
    ro, rl = M.cross_exact(q, k, v, None, scale=100.0)
    M.near(lse, rl, M.attn_tol(64, 100, 1.0), "lse")  # of the size of its scores
    # P moves by the scores' own rounding: sqrt(64) half steps of scores up to 6 * 8 * 100
    M.near(o, ro, M.attn_tol(64, 100, 4800.0), "o")
    check(L, q, torch.zeros_like(k), v, None, rand(4, 1, 2, Tq, 64))
    check(L, q, k, v, None, rand(4, 1, 2, Tq, 64), scale=-0.125)
    # queries with a positive first column against keys of -inf there: every score is -inf
    q[..., 0] = q[..., 0].abs() + 1
    k[..., 0] = -math.inf
    o, lse = run(L, q, k, v, None)
    assert (o == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("d", [64, 128, 30])
@pytest.mark.parametrize("Tq,Tk", [(1, 70), (40, 130), (290, 33)])
def test_powers_of_two(L, d, Tq, Tk):
    """Powers of two go through every product and sum unrounded, whatever form the
    operands take inside: rows of dO of magnitudes 2^-40 to 2^40 give dQ's rows times
    the same, V's gives O and dQ, K's against Q's nothing but the gradients'."""
    q, do = rand(1, 2, 4, Tq, d), rand(2, 2, 4, Tq, d)
    k, v = rand(3, 2, 2, Tk, d), rand(4, 2, 2, Tk, d)
    lens = torch.tensor([Tk, Tk // 2], device="cuda")
    o, lse, dq, dk, dv = run(L, q, k, v, lens, do)
    f = torch.exp2(torch.randint(-40, 41, (2, 4, Tq, 1), generator=torch.Generator().manual_seed(5)).float()).cuda()
    assert torch.equal(run(L, q, k, v, lens, do * f)[2], dq * f)
    for e in (-40, 40):
        g = run(L, q, k, v * 2.0 ** e, lens, do)
        for a, b in zip(g, (o * 2.0 ** e, lse, dq * 2.0 ** e, dk * 2.0 ** e, dv)):
            assert torch.equal(a, b)
        g = run(L, q * 2.0 ** -e, k * 2.0 ** e, v, lens, do)
        for a, b in zip(g, (o, lse, dq * 2.0 ** e, dk * 2.0 ** -e, dv)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("e", [-75, 62])
@pytest.mark.parametrize("d", [64, 128])
def test_very_small_and_very_large(L, d, e):
    """Operands (all of one, or one row of it) whose magnitudes two fp16 parts do not hold."""
    q, do = rand(1, 2, 2, 50, d), rand(2, 2, 2, 50, d)
    k, v = rand(3, 2, 2, 100, d), rand(4, 2, 2, 100, d)
    f, tol = 2.0 ** e, M.attn_tol(d, 100)
    ref = M.cross_exact(q, k, v, None, do)
    mass = M.cross_mass(q, k, v, None, do)
    names = ("o", "lse", "dq", "dk", "dv")

    def same(got, scales):
        for name, g, r, s in zip(names, got, ref, scales):
            M.near(g.double() / s, r, tol * (2 if name[0] == "d" else 1), name, mass.get(name))

    same(run(L, q, k, v * f, None, do), (f, 1, f, f, 1))
    same(run(L, q, k, v, None, do * f), (1, 1, f, f, f))
    same(run(L, q / f, k * f, v, None, do), (1, 1, f, 1 / f, 1))
    # one row alone
    x = v.clone()
    x[0, 1, 33] *= f
    got, r = run(L, q, k, x, None, do), M.cross_exact(q, k, x, None, do)
    w = M.cross_mass(q, k, x, None, do)
    for name, a, b in zip(names, got, r):
        M.near(a, b, tol * (2 if name[0] == "d" else 1), name, w.get(name))


@pytest.mark.parametrize("d", [64, 128])
def test_an_outlier_that_no_row_attends_to(L, d):
    """A value 2^40 times the others' behind a score of -100, a value of zeros that takes most of
    the weight, and values of 2^-30: the others keep their digits."""
    q, do = rand(1, 1, 2, 70, d), rand(2, 1, 2, 70, d)
    k, v = rand(3, 1, 2, 90, d), rand(4, 1, 2, 90, d)
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    k[:, :, 10, 0] = -100.0 / (8.0 * d ** -0.5)
    v[:, :, 10] *= 2.0 ** 40
    o, lse = run(L, q, k, v, None)
    ro, rl = M.cross_exact(q, k, v)
    M.near(o, ro, M.attn_tol(d, 90, 100.0), "o")
    v[:, :, 10] *= 2.0 ** -40
    k[:, :, 10, 0] = 12.0 / (8.0 * d ** -0.5)
    v[:, :, 10] = 0.0
    v[:, :, 40] *= 2.0 ** -30
    got, ref, w = run(L, q, k, v, None, do), M.cross_exact(q, k, v, None, do), M.cross_mass(q, k, v, None, do)
    for name, a, b in zip(("o", "lse", "dq", "dk", "dv"), got, ref):
        M.near(a, b, M.attn_tol(d, 90, 16.0) * (2 if name[0] == "d" else 1), name, w.get(name))


@pytest.mark.parametrize("d", [64, 128])
def test_small_columns_of_large_rows(L, d):
    """Elements 2^-28 of their row's largest: in two fp16 parts under the row's scale they
    are subnormal, held to 2^-38 of the largest; each product with them is off by
    that times its weight, beside the roundings of the sums."""
    q, do = rand(1, 1, 2, 50, d), rand(2, 1, 2, 50, d)
    k, v = rand(3, 1, 2, 70, d), rand(4, 1, 2, 70, d)
    small = 2.0 ** -28
    v[..., 1:] *= small
    o, lse = run(L, q, k, v, None)
    ro, _ = M.cross_exact(q, k, v)
    top = v.abs().max().item()
    bound = 2.0 ** -38 * top + 4 * M.attn_tol(d, 70) * v[..., 1:].abs().max().item()
    assert (o.double().cpu() - ro)[..., 1:].abs().max().item() <= bound
    # K's small columns in dQ = scale dS K, with sum_j |dS_ij| <= 2 max|dO . v|
    v = rand(4, 1, 2, 70, d)
    k[..., 1:] *= small
    q[..., 1:] *= 2.0
    _, _, dq, _, _ = run(L, q, k, v, None, do)
    rq = M.cross_exact(q, k, v, None, do)[2]
    ds = 2 * (do @ v.transpose(2, 3)).abs().max().item() * d ** -0.5
    bound = ds * (2.0 ** -38 * k.abs().max().item() + 8 * M.attn_tol(d, 70) * k[..., 1:].abs().max().item())
    assert (dq.double().cpu() - rq)[..., 1:].abs().max().item() <= bound


@pytest.mark.parametrize("d", [64, 128, 30])
def test_infinities_and_nan(L, d):
    """Where keys, values or gradients hold them, as fp32 arithmetic has it."""
    q, do = rand(1, 2, 2, 40, d), rand(2, 2, 2, 40, d)
    k, v = rand(3, 2, 2, 80, d), rand(4, 2, 2, 80, d)
    tol = M.attn_tol(d, 80)
    for bad in (math.inf, -math.inf, math.nan):
        x = v.clone()
        x[0, 1, 35, 3] = bad
        o, lse = run(L, q, k, x, None)
        ro, rl = M.cross_exact(q, k, x)
        M.near(o, ro, tol, "o")
        M.near(lse, rl, tol, "lse", M.cross_mass(q, k, v, None, do)["lse"])
        g = do.clone()
        g[1, 0, 7, 2] = bad
        o, lse, dq, dk, dv = run(L, q, k, v, None, g)
        clean = run(L, q, k, v, None, do)
        # dP - D is inf - inf for the keys whose value has D's sign there, inf for the others
        assert torch.isnan(dq[1, 0, 7]).all() and not torch.isfinite(dk[1, 0]).any()
        assert not torch.isfinite(dv[1, 0, :, 2]).any()
        other = torch.ones_like(dq, dtype=torch.bool)
        other[1, 0] = False
        assert torch.equal(dq[other], clean[2][other]) and torch.isfinite(dq[1, 0, 8:]).all()


def test_gradients_against_differences(L):
    """d/dh of sum(do * O) along random directions, from forwards alone, in steps
    whose own error is of order h^2."""
    q, k, v = rand(1, 1, 4, 5, 64), rand(2, 1, 2, 60, 64), rand(3, 1, 2, 60, 64)
    do = rand(4, 1, 4, 5, 64)
    lens = torch.tensor([47], device="cuda")
    _, _, dq, dk, dv = run(L, q, k, v, lens, do)
    h = 2.0 ** -6
    for i, (x, g) in enumerate(((q, dq), (k, dk), (v, dv))):
        w = rand(10 + i, *x.shape)
        args = [q, k, v]
        vals = []
        for s in (h, -h):
            args[i] = x + s * w
            vals.append((run(L, *args, lens)[0].double() * do.double()).sum().item())
        want = (g.double() * w.double()).sum().item()
        # third derivative about |w|^3 ~ 1 per score; outputs' roundings over 2 h
        bound = (h * h + M.attn_tol(64, 60) / h) * (do.norm() * w.norm()).item() / 4
        assert abs((vals[0] - vals[1]) / (2 * h) - want) <= bound


def test_reproducible_and_on_other_streams(L):
    q, k, v, do = rand(1, 3, 4, 70, 64), rand(2, 3, 2, 500, 64), rand(3, 3, 2, 500, 64), rand(4, 3, 4, 70, 64)
    lens = torch.tensor([500, 3, 77], device="cuda")
    first = run(L, q, k, v, lens, do)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run(L, q, k, v, lens, do)
    side.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)


@pytest.mark.parametrize("Tq", [1, 40])
def test_captured_graph(L, Tq):
    """A captured forward and backward replayed with new inputs, with eager work
    between the replays."""
    q, k, v, do = rand(1, 2, 4, Tq, 64), rand(2, 2, 2, 600, 64), rand(3, 2, 2, 600, 64), rand(4, 2, 4, Tq, 64)
    lens = torch.tensor([600, 30], device="cuda")
    o, lse = torch.empty_like(q), torch.empty(2, 4, Tq, device="cuda")
    dq, dk, dv = (torch.empty_like(t) for t in (q, k, v))
    dims = (2, 4, 2, Tq, 600, 64)
    wf, wb = M.scratch(L.aar_cross_attn_fwd_workspace_bytes(*dims)), M.scratch(L.aar_cross_attn_bwd_workspace_bytes(*dims))

    def both():
        M.cross_fwd(L, q, k, v, lens, o, lse, ws=wf)
        M.cross_bwd(L, q, k, v, lens, o, lse, do, dq, dk, dv, ws=wb)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for i in range(3):
        for j, t in enumerate((q, k, v, do)):
            t.copy_(rand(20 + 4 * i + j, *t.shape))
        lens.copy_(torch.tensor([600 - 100 * i, 31 * i]))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (o, lse, dq, dk, dv)]
        for a, b in zip(got, run(L, q, k, v, lens, do)):
            assert torch.equal(a, b)


def test_ops_and_module(gpu):
    """ag.cross_attention on views, and nn.CrossAttention whole, projected once for
    single tokens, and with the context's gradient."""
    rng = np.random.default_rng(5)
    B, Tq, Tk, D, C, H, Hkv = 3, 9, 40, 96, 56, 6, 2
    d = D // H
    lens = np.array([40, 0, 17], np.int64)
    tl = gpu.from_numpy(lens).to(gpu.Device.CUDA)
    x, ctx = rng.standard_normal((B, Tq, D)).astype(np.float32), rng.standard_normal((B, Tk, C)).astype(np.float32)
    gy = rng.standard_normal((B, Tq, D)).astype(np.float32)
    m = gpu.nn.CrossAttention(D, H, d_context=C, n_kv_heads=Hkv, rng=rng).to(gpu.Device.CUDA)
    tx, tc = dev(gpu, x, True), dev(gpu, ctx, True)
    y = m(tx, tc, tl)
    y.backward(dev(gpu, gy))
    w = [torch.from_numpy(host(gpu, p.tensor)).double().requires_grad_() for p in m.parameters()]
    X, Cx = (torch.from_numpy(t).double().requires_grad_() for t in (x, ctx))
    q = (X @ w[0].t() + w[1]).view(B, Tq, H, d).transpose(1, 2)
    kv = (Cx @ w[2].t() + w[3]).view(B, Tk, 2, Hkv, d)
    k, v = (kv[:, :, i].transpose(1, 2).repeat_interleave(H // Hkv, 1) for i in (0, 1))
    seen = torch.arange(Tk) < torch.from_numpy(lens).view(B, 1, 1, 1)
    s = (q @ k.transpose(2, 3) / math.sqrt(d)).masked_fill(~seen, -1e300)
    p = torch.softmax(s, -1) * seen
    ref = (p @ v).transpose(1, 2).reshape(B, Tq, D) @ w[4].t() + w[5]
    ref.backward(torch.from_numpy(gy).double())
    # products of up to 96 terms on both sides of the attention
    tol = 4 * M.attn_tol(96, 40)
    M.near(host(gpu, y), ref, tol, "y")
    M.near(host(gpu, tx.grad), X.grad, tol, "dx")
    M.near(host(gpu, tc.grad), Cx.grad, tol, "dcontext")
    for i, (a, b) in enumerate(zip(m.parameters(), w)):
        M.near(host(gpu, a.tensor.grad), b.grad, tol, f"parameter {i}")
    kvp = m.project_context(dev(gpu, ctx))
    for t in range(Tq):
        one = m.attend(dev(gpu, x[:, t:t + 1]), kvp, tl)
        M.near(host(gpu, one)[:, 0], ref.detach()[:, t], tol, f"token {t}")
    # the op itself over transposed views
    tq, tk = dev(gpu, rng.standard_normal((B, Tq, H, d)), True), dev(gpu, rng.standard_normal((B, Tk, Hkv, d)), True)
    tv = dev(gpu, rng.standard_normal((B, Tk, Hkv, d)), True)
    o = gpu.cross_attention(*(gpu.transpose(t, 1, 2) for t in (tq, tk, tv)), tl)
    g = rng.standard_normal((B, H, Tq, d)).astype(np.float32)
    o.backward(dev(gpu, g))
    hq, hk, hv = (torch.from_numpy(host(gpu, t)).transpose(1, 2) for t in (tq, tk, tv))
    ro, _, dq, dk, dv = M.cross_exact(hq, hk, hv, torch.from_numpy(lens), torch.from_numpy(g))
    for name, a, b in (("o", host(gpu, o), ro), ("dq", host(gpu, tq.grad), dq.transpose(1, 2)),
                       ("dk", host(gpu, tk.grad), dk.transpose(1, 2)), ("dv", host(gpu, tv.grad), dv.transpose(1, 2))):
        M.near(a, b, 2 * M.attn_tol(d, Tk), name)
