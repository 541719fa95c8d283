"""Window attention with sinks (aar_window_attn_*) on the GPU against its definition in
64 bits: windows from one token to all, sinks from none to all, lengths from one token
to long ones, shared heads, strided and unaligned operands, values of every magnitude,
infinities and NaN that are hidden, other streams and captured graphs."""
from __future__ import annotations

import math

import pytest
import torch

import kvops as K
import lmops as M

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L(gpu):
    return K.lib()


def rand(seed, *shape, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).cuda()


def inputs(B, H, Hkv, T, d):
    return rand(1, B, H, T, d), rand(2, B, Hkv, T, d), rand(3, B, Hkv, T, d), rand(4, B, H, T, d)


NAMES = ("o", "lse", "dq", "dk", "dv")


def check(L, q, k, v, do, window, sinks, scale=None):
    got = K.window_run(L, q, k, v, do, window, sinks, scale)
    ref, mass = K.window_exact(q, k, v, do, window, sinks, scale)
    T, d = q.shape[2:]
    # a key's sums have a term for each query of each head that sees it
    n = T * q.shape[1] // k.shape[1] if min(sinks, T) else min(T, window) * q.shape[1] // k.shape[1]
    tol = M.attn_tol(d, max(n, min(T, window + sinks)))
    for name, g, r in zip(NAMES, got, ref):
        M.near(g, r, tol * (2 if name[0] == "d" else 1), name, mass.get(name))
    return got


# B, H, Hkv, T, d, window, sinks
SHAPES = [
    (1, 1, 1, 1, 64, 1, 0), (2, 3, 3, 1, 40, 5, 2), (1, 2, 1, 2, 64, 1, 1), (2, 2, 2, 31, 64, 8, 0),
    (1, 2, 2, 32, 128, 32, 1), (2, 4, 2, 33, 64, 16, 4), (1, 3, 3, 64, 30, 33, 0), (1, 2, 2, 65, 64, 64, 2),
    (2, 6, 2, 127, 96, 31, 3), (1, 2, 2, 128, 64, 1, 0), (1, 2, 2, 128, 64, 1, 1), (2, 2, 2, 129, 64, 128, 4),
    (1, 4, 1, 200, 128, 64, 2), (1, 2, 2, 256, 64, 1 << 40, 0), (1, 2, 2, 257, 64, 255, 5), (1, 1, 1, 300, 1, 50, 2),
    (1, 2, 2, 300, 3, 100, 70), (1, 3, 3, 333, 36, 40, 400), (2, 8, 4, 500, 64, 100, 4), (1, 2, 2, 777, 32, 300, 33),
    (1, 8, 1, 640, 64, 129, 1), (1, 2, 2, 1000, 128, 200, 130), (1, 1, 1, 2049, 64, 500, 4), (1, 4, 2, 1500, 64, 32, 3),
    (1, 2, 1, 3000, 64, 40, 200), (3, 2, 2, 160, 128, 33, 31), (1, 1, 1, 4097, 64, 7, 1), (16, 12, 12, 130, 64, 65, 4),
]


@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_definition(L, shape):
    B, H, Hkv, T, d, window, sinks = shape
    check(L, *inputs(B, H, Hkv, T, d), window, sinks)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scales(L, scale):
    q, k, v, do = inputs(1, 2, 2, 150, 64)
    check(L, q * 0.3, k * 0.3, v, do, 40, 3, scale)


def test_a_window_of_everything_is_causal_attention(L):
    q, k, v, do = inputs(2, 3, 3, 300, 64)
    got = K.window_run(L, q, k, v, do, 300, 0)
    for a, b in zip(got, K.window_run(L, q, k, v, do, 1 << 62, 9)):
        assert torch.equal(a, b)
    # and one token's window its own value
    o, lse, dq, dk, dv = K.window_run(L, q, k, v, do, 1, 0)
    M.near(o, v, 2 * M.U + 2.0 ** -22, "o")
    # P = 2^(s - lse) there: lse, its product with log2(e) and the difference's operands are
    # each rounded, half a step of at most |lse| log2(e) <= 1.5 |lse|, and 2^x moves by less than x
    M.near(dv, do, 2 * M.U + 2.0 ** -22 + 3 * M.U * 1.5 * lse.abs().max().item(), "dv")


@pytest.mark.parametrize("d", [64, 128, 36])
@pytest.mark.parametrize("offset", [0, 1])
def test_strided_operands(L, d, offset):
    """A packed projection's views, outputs in [B, T, H, d] order, unaligned bases."""
    B, H, Hkv, T = 2, 4, 2, 170
    q, k, v, do = inputs(B, H, Hkv, T, d)
    ref, mass = K.window_exact(q, k, v, do, 50, 3)

    def rows(*shape):
        n = math.prod(shape)
        return torch.full((n + 4,), 3.0, device="cuda")[offset : offset + n].view(shape)

    packed, gpacked = rows(B, T, H + 2 * Hkv, d), rows(B, T, H + 2 * Hkv, d)
    views = lambda t: (t[:, :, :H].transpose(1, 2), t[:, :, H : H + Hkv].transpose(1, 2),  # noqa: E731
                       t[:, :, H + Hkv :].transpose(1, 2))
    for dst, src in zip(views(packed), (q, k, v)):
        dst.copy_(src)
    o, lse, dout = rows(B, T, H, d), torch.empty(B, H, T, device="cuda"), rows(B, T, H, d)
    dout.transpose(1, 2).copy_(do)
    K.window_fwd(L, *views(packed), o.transpose(1, 2), lse, 50, 3)
    K.window_bwd(L, *views(packed), o.transpose(1, 2), lse, dout.transpose(1, 2), *views(gpacked), 50, 3)
    tol = M.attn_tol(d, 2 * T)
    for name, g, r in zip(NAMES, (o.transpose(1, 2), lse, *views(gpacked)), ref):
        M.near(g, r, tol * (2 if name[0] == "d" else 1), name, mass.get(name))


def test_broadcast_operands(L):
    """Batches and heads that share memory (strides of 0), gradients of their own."""
    q, k, v, do = inputs(1, 1, 1, 90, 64)
    q, do = q.expand(2, 4, 90, 64), do.expand(2, 4, 90, 64)
    k, v = k.expand(2, 2, 90, 64), v.expand(2, 2, 90, 64)
    check(L, q, k, v, do, 20, 2)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("which", ["q", "k", "v", "do"])
@pytest.mark.parametrize("power", [-140, -105, -60, 50, 62])
def test_rows_of_any_magnitude(L, which, power, d):
    """One row in every eight scaled by 2^power, the scores kept small: held in parts or
    done again with the fp32 instruction."""
    q, k, v, do = inputs(1, 2, 2, 100, d)
    x = {"q": q, "k": k, "v": v, "do": do}
    if which in "qk":
        other = "k" if which == "q" else "q"
        x[other] *= 2.0 ** -min(100, max(0, power))
    x[which][:, :, ::8] *= 2.0 ** power
    got = K.window_run(L, q, k, v, do, 30, 2)
    ref, mass = K.window_exact(q, k, v, do, 30, 2)
    tol = M.attn_tol(d, 100)
    for name, g, r in zip(NAMES, got, ref):
        # rows apart: the large ones' errors are not the small ones'; half a step of 2^-149 a term of a sum
        w = mass.get(name, r)
        top = w.double().abs().amax(-1, keepdim=True) if w.dim() == 4 else w.double().abs()
        off = (g.double() - r).abs()
        assert (off <= 16 * tol * top + 100 * 2.0 ** -149).all(), (name, (off / (top + 1e-300)).max().item())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("T", [100, 600])
@pytest.mark.parametrize("spread", [8, 30])
def test_rows_of_mixed_magnitude(L, T, spread, d):
    """Values and gradients whose rows lie up to 2^(2 spread) apart inside a tile: on both
    sides of what a tile's parts hold."""
    q, k, v, do = inputs(1, 4, 2, T, d)
    power = torch.randint(-spread, spread + 1, (2, T), generator=torch.Generator().manual_seed(spread)).cuda()
    v *= (2.0 ** power[0].double()).float()[:, None]
    do *= (2.0 ** power[1].double()).float()[:, None]
    got = K.window_run(L, q, k, v, do, 70, 2)
    ref, mass = K.window_exact(q, k, v, do, 70, 2)
    # each result's terms without their signs: cancelled or not, they are rounded
    mass["o"] = K.window_exact(q, k, v.abs(), None, 70, 2)[0][0]
    p = torch.matmul(q.double(), k.double().repeat_interleave(2, 1).transpose(2, 3).contiguous()) * d ** -0.5
    p = torch.softmax(p.masked_fill(~K.window_mask(T, 70, 2).cuda(), -math.inf), -1)
    mass["dv"] = torch.matmul(p.transpose(2, 3).contiguous(), do.double().abs()).view(1, 2, 2, T, d).sum(2)
    tol = M.attn_tol(d, T)
    for name, g, r in zip(NAMES, got, ref):
        w = mass[name].amax(-1, keepdim=True) if r.dim() == 4 else mass[name]
        off = (g.double() - r).abs()
        assert (off <= 8 * tol * w).all(), (name, (off / w).max().item(), tol)


@pytest.mark.parametrize("d", [64, 128, 36])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_finite_stays_where_it_is_seen(L, d, bad):
    """A key, value, query or gradient with a NaN or an infinity changes no row that
    does not see it."""
    T, window, sinks = 200, 40, 2
    q, k, v, do = inputs(1, 2, 2, T, d)
    sees = K.window_mask(T, window, sinks).cuda()
    clean = K.window_run(L, q, k, v, do, window, sinks)
    at = 77
    for which in range(4):
        x = [t.clone() for t in (q, k, v, do)]
        x[which][0, 1, at, d // 2] = bad
        o, lse, dq, dk, dv = K.window_run(L, *x, window, sinks)
        rows = sees[:, at] if which in (1, 2) else torch.arange(T, device="cuda") == at  # queries that have it
        tainted = (sees[rows].any(0))  # keys that one of these sees
        for head in (0, 1):
            for name, g, c in (("o", o, clean[0]), ("dq", dq, clean[2])):
                fine = ~rows if head == 1 else torch.ones_like(rows)
                M.near(g[0, head][fine], c[0, head][fine], M.attn_tol(d, T), name)
            for name, g, c in (("dk", dk, clean[3]), ("dv", dv, clean[4])):
                fine = ~tainted if head == 1 else torch.ones_like(tainted)
                M.near(g[0, head][fine], c[0, head][fine], 2 * M.attn_tol(d, T), name)
        if which == 2:
            assert not torch.isfinite(o[0, 1, :, d // 2][rows]).any()
            assert torch.isfinite(o[0, 1, :, : d // 2]).all()
        if which == 3:
            assert torch.isfinite(o).all() and not torch.isfinite(dq[0, 1, at]).all()


def test_gradients_by_differences(L):
    """Central differences of a weighted sum of O, in fp32 along random directions."""
    q, k, v, do = inputs(1, 4, 2, 70, 64)
    o, lse, dq, dk, dv = K.window_run(L, q, k, v, do, 20, 3)
    for i, (x, g) in enumerate(((q, dq), (k, dk), (v, dv))):
        u = rand(10 + i, *x.shape)
        h = 1e-2
        sums = []
        for s in (h, -h):
            args = [q, k, v]
            args[i] = x + s * u
            sums.append((K.window_run(L, *args, None, 20, 3)[0].double() * do.double()).sum())
        by = ((sums[0] - sums[1]) / (2 * h)).item()
        # the third derivative's part, h^2 / 6 of the slope's own scale, and the sums' roundings over 2 h
        size = (g.double().abs() * u.double().abs()).sum().item()
        assert abs(by - (g.double() * u.double()).sum().item()) <= size * (h * h + M.attn_tol(64, 70) / h)


def test_same_bits_streams_and_graphs(L):
    q, k, v, do = inputs(2, 4, 2, 1300, 64)
    first = K.window_run(L, q, k, v, do, 60, 4)
    for a, b in zip(first, K.window_run(L, q, k, v, do, 60, 4)):
        assert torch.equal(a, b)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = K.window_run(L, q, k, v, do, 60, 4)
    side.synchronize()
    for a, b in zip(first, other):
        assert torch.equal(a, b)

    o, lse = torch.empty_like(q), torch.empty(q.shape[:3], device="cuda")
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ws = M.scratch(L.aar_window_attn_bwd_workspace_bytes(2, 4, 2, 1300, 64, 60, 4))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.window_fwd(L, q, k, v, o, lse, 60, 4)
        K.window_bwd(L, q, k, v, o, lse, do, dq, dk, dv, 60, 4, ws=ws)
    for i in range(3):
        q.copy_(rand(20 + i, *q.shape))
        for t in (o, lse, dq, dk, dv):
            t.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((o, lse, dq, dk, dv), K.window_run(L, q, k, v, do, 60, 4)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("shape", [
    (43, 6, 3, 250, 64, 90, 3), (22, 6, 6, 200, 40, 200, 0), (5, 2, 2, 161, 64, 3, 170), (3, 4, 1, 128, 128, 40, 4),
    (2, 6, 2, 1500, 64, 33, 700), (1, 4, 1, 2600, 128, 20, 2100), (1, 2, 2, 5000, 64, 64, 60), (70, 4, 4, 260, 36, 300, 2),
    (9, 8, 8, 1100, 64, 200, 1)])
def test_every_form_of_the_grid(L, shape):
    """Texts in LDS with one and two workgroups a head, rings of both depths, the sinks' far
    queries in parts and, of too many sinks, not."""
    B, H, Hkv, T, d, window, sinks = shape
    check(L, *inputs(B, H, Hkv, T, d), window, sinks)


def test_the_forward_holds_to_its_workspace(L):
    q, k, v, _ = inputs(1, 2, 1, 600, 64)
    o, lse = torch.empty_like(q), torch.empty(1, 2, 600, device="cuda")
    dims = (1, 2, 1, 600, 64)
    nb = L.aar_window_attn_fwd_workspace_bytes(*dims, 30, 2)
    assert nb > 0 and L.aar_window_attn_fwd_workspace_bytes(1, 2, 1, 64, 64, 30, 2) == 0
    ws = torch.full((nb + 64,), 123, dtype=torch.uint8, device="cuda")
    args, st = [t.data_ptr() for t in (q, k, v, o, lse)], M.strides3(q, k, v, o)
    assert L.aar_window_attn_fwd_f32(*args, *dims, st, 30, 2, 0.125, ws.data_ptr(), nb, M.stream()) == 0
    assert (ws[nb:] == 123).all()
    for p, n in ((None, nb), (ws.data_ptr(), nb - 1), (ws.data_ptr() + 4, nb)):
        assert L.aar_window_attn_fwd_f32(*args, *dims, st, 30, 2, 0.125, p, n, M.stream()) == M.EWORKSPACE


def test_workspace_is_held_to(L):
    """Nothing is written past the bytes that were asked for, and less is refused."""
    q, k, v, do = inputs(1, 2, 1, 600, 64)
    o, lse = K.window_run(L, q, k, v, None, 30, 2)
    dims = (1, 2, 1, 600, 64)
    nb = L.aar_window_attn_bwd_workspace_bytes(*dims, 30, 2)
    ws = torch.full((nb + 64,), 123, dtype=torch.uint8, device="cuda")
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    K.window_bwd(L, q, k, v, o, lse, do, dq, dk, dv, 30, 2, ws=ws)
    assert (ws[nb:] == 123).all()
    args = [t.data_ptr() for t in (q, k, v, o, lse, do, dq, dk, dv)]
    st = M.strides3(q, k, v, o, do, dq, dk, dv)
    for p, n in ((None, nb), (ws.data_ptr(), nb - 1), (ws.data_ptr() + 4, nb)):
        assert L.aar_window_attn_bwd_f32(*args, *dims, st, 30, 2, 0.125, p, n, M.stream()) == M.EWORKSPACE
