"""Per-head norms of queries and keys with the position rotation
(aar_qk_norm_rope_*, ag.qk_norm_rope, nn.MultiHeadAttention(qk_norm=True)) on the
GPU against the definition in 64 bits."""
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


def exact(x, wq, wk, pos, hq, hk, d, r, base, eps, gy=None):
    """x [rows, (hq + hk) d] in 64 bits on the CPU: y (and dx, dwq, dwk)."""
    x, wq, wk = (t.detach().double().cpu().requires_grad_() for t in (x, wq, wk))
    rows = x.shape[0]
    xs = x.view(rows, hq + hk, d)
    w = torch.cat([wq[None].repeat(hq, 1), wk[None].repeat(hk, 1)])
    u = xs / torch.sqrt(xs.pow(2).mean(-1, keepdim=True) + eps) * w
    if r:
        p = pos.cpu().double().repeat(rows // pos.numel())
        a = p[:, None, None] * base ** (torch.arange(r // 2, dtype=torch.float64) * (-2.0 / r))
        u1, u2 = u[..., : r // 2], u[..., r // 2: r]
        u = torch.cat([u1 * a.cos() - u2 * a.sin(), u2 * a.cos() + u1 * a.sin(), u[..., r:]], -1)
    y = u.reshape(rows, -1)
    if gy is None:
        return y.detach()
    y.backward(gy.double().cpu())
    return y.detach(), x.grad, wq.grad if hq else torch.zeros(d), wk.grad if hk else torch.zeros(d)


def tol_of(d, terms=1):
    """Half steps of an element: a sum of d squares (random walk), the root, three
    products, the turned pair's two products and the angle's own; a weight's
    gradient sums `terms` of them.  Four standard deviations."""
    return 4 * M.U * (math.sqrt(d) + 12 + math.sqrt(terms))


def run(L, x, wq, wk, pos, hq, hk, d, r, base=10000.0, eps=1e-6, gy=None, width=None):
    """Over rows of `width` columns, of which the heads are the first."""
    rows, n = x.shape[0], (hq + hk) * d
    width = n if width is None else width
    wide = torch.full((rows, width), 9.0, device="cuda")
    wide[:, :n] = x
    y = torch.full((rows, width), 5.0, device="cuda")
    p, count = (pos.data_ptr(), pos.numel()) if r else (None, 0)
    M.ok(L.aar_qk_norm_rope_fwd_f32(wide.data_ptr(), width, M.ptr(wq), M.ptr(wk), p, count, y.data_ptr(), width, rows, hq,
                                    hk, d, r, base, eps, M.stream()))
    assert (y[:, n:] == 5.0).all()
    if gy is None:
        return y[:, :n]
    gw = torch.full((rows, width), 3.0, device="cuda")
    gw[:, :n] = gy
    dx, dwq, dwk = torch.full((rows, width), 5.0, device="cuda"), torch.full((d,), 5.0, device="cuda"), torch.full((d,), 5.0, device="cuda")
    nb = L.aar_qk_norm_rope_bwd_workspace_bytes(rows, hq, hk, d)
    ws = M.scratch(nb)
    M.ok(L.aar_qk_norm_rope_bwd_f32(gw.data_ptr(), width, wide.data_ptr(), width, M.ptr(wq), M.ptr(wk), p, count,
                                    dx.data_ptr(), width, dwq.data_ptr(), dwk.data_ptr(), rows, hq, hk, d, r, base, eps,
                                    ws.data_ptr(), nb, M.stream()))
    assert (dx[:, n:] == 5.0).all()
    return y[:, :n], dx[:, :n], dwq, dwk


# rows, positions, hq, hk, d, r, spare columns
CASES = [
    (1, 1, 1, 1, 64, 64, 0), (7, 7, 6, 6, 64, 64, 384), (512, 128, 6, 6, 64, 64, 384), (33, 33, 8, 2, 128, 128, 0),
    (5, 5, 3, 1, 32, 32, 0), (64, 16, 12, 12, 96, 96, 0), (10, 10, 5, 5, 40, 40, 0), (9, 3, 2, 1, 256, 256, 4),
    (6, 6, 1, 2, 8, 8, 0), (21, 7, 4, 4, 30, 30, 0), (12, 12, 4, 2, 64, 32, 0), (12, 4, 3, 3, 64, 0, 0),
    (8, 8, 2, 2, 64, 64, 3), (5, 5, 1, 1, 2, 2, 0), (6, 6, 3, 2, 7, 4, 1), (40, 40, 4, 0, 64, 64, 0),
    (40, 40, 0, 4, 64, 64, 0), (3000, 1000, 5, 3, 64, 64, 0), (2, 2, 60, 12, 128, 128, 0), (4, 4, 2, 2, 255, 254, 0),
    (5000, 1000, 4, 2, 30, 30, 0), (4500, 1500, 2, 1, 200, 100, 0), (4200, 4200, 3, 3, 100, 50, 2),
]


@pytest.mark.parametrize("case", CASES)
def test_against_the_definition(L, case):
    rows, npos, hq, hk, d, r, spare = case
    n = (hq + hk) * d
    x, gy = rand(1, rows, n, scale=1.5), rand(2, rows, n)
    wq, wk = 1 + rand(3, d, scale=0.2), 1 + rand(4, d, scale=0.2)
    pos = torch.arange(npos, device="cuda") * 3 - 5
    got = run(L, x, wq, wk, pos, hq, hk, d, r, gy=gy, width=n + spare)
    ref = exact(x, wq, wk, pos, hq, hk, d, r, 10000.0, 1e-6, gy)
    for name, g, e, terms in zip(("y", "dx", "dwq", "dwk"), got, ref, (1, 1, rows * max(hq, 1), rows * max(hk, 1))):
        M.near(g, e, tol_of(d, terms), name)


@pytest.mark.parametrize("d", [64, 30])
def test_far_positions(L, d):
    """Angles of positions up to 2^40 in both directions: the turn is formed in 64
    bits, where position * frequency itself keeps 2^-53 of its turns."""
    pos = torch.tensor([0, 1, 131071, -131071, 10 ** 6 + 1, 2 ** 31 + 7, 2 ** 40 + 3, -(2 ** 40)], device="cuda")
    x, gy = rand(1, 8, 4 * d), rand(2, 8, 4 * d)
    w = torch.ones(d, device="cuda")
    got = run(L, x, w, w, pos, 2, 2, d, d, gy=gy)
    ref = exact(x, w, w, pos, 2, 2, d, d, 10000.0, 1e-6, gy)
    # 2^40 radians at 2^-52 relative (the frequency's own steps) are 2.4e-4 radians in both
    for i in range(8):
        far = abs(int(pos[i])) * 2.0 ** -50
        M.near(got[0][i], ref[0][i], tol_of(d) + far, f"y at {int(pos[i])}")
        M.near(got[1][i], ref[1][i], tol_of(d) + far, f"dx at {int(pos[i])}")


def test_in_place(L):
    x, gy, w = rand(1, 50, 8 * 64), rand(2, 50, 8 * 64), 1 + rand(3, 64, scale=0.1)
    pos = torch.arange(50, device="cuda")
    y, dx, dwq, dwk = run(L, x, w, w, pos, 4, 4, 64, 64, gy=gy)
    for d, r in ((64, 64), (64, 32)):
        y, dx, dwq, dwk = run(L, x, w, w, pos, 4, 4, d, r, gy=gy)
        z, g = x.clone(), gy.clone()
        M.ok(L.aar_qk_norm_rope_fwd_f32(z.data_ptr(), 512, w.data_ptr(), w.data_ptr(), pos.data_ptr(), 50, z.data_ptr(), 512,
                                        50, 4, 4, d, r, 10000.0, 1e-6, M.stream()))
        assert torch.equal(z, y)
        q, k = torch.empty_like(w), torch.empty_like(w)
        nb = L.aar_qk_norm_rope_bwd_workspace_bytes(50, 4, 4, d)
        ws = M.scratch(nb)
        M.ok(L.aar_qk_norm_rope_bwd_f32(g.data_ptr(), 512, x.data_ptr(), 512, w.data_ptr(), w.data_ptr(), pos.data_ptr(), 50,
                                        g.data_ptr(), 512, q.data_ptr(), k.data_ptr(), 50, 4, 4, d, r, 10000.0, 1e-6,
                                        ws.data_ptr(), nb, M.stream()))
        assert torch.equal(g, dx) and torch.equal(q, dwq) and torch.equal(k, dwk)


def test_zero_rows_heads_and_values(L):
    w = torch.ones(64, device="cuda")
    q, k = torch.full((64,), 5.0, device="cuda"), torch.full((64,), 5.0, device="cuda")
    for rows, heads in ((0, 2), (3, 0)):
        x = torch.empty(rows, 128, device="cuda")
        M.ok(L.aar_qk_norm_rope_fwd_f32(M.ptr(x), 128, w.data_ptr(), w.data_ptr(), None, 0, M.ptr(x), 128, rows, heads,
                                        0, 64, 0, 1e4, 1e-6, M.stream()))
        M.ok(L.aar_qk_norm_rope_bwd_f32(M.ptr(x), 128, M.ptr(x), 128, w.data_ptr(), w.data_ptr(), None, 0, M.ptr(x), 128,
                                        q.data_ptr(), k.data_ptr(), rows, heads, 0, 64, 0, 1e4, 1e-6, None, 0,
                                        M.stream()))
        assert (q == 0).all() and (k == 0).all()
        q.fill_(5.0), k.fill_(5.0)
    # a head of zeros stays zeros, its gradient is rsqrt(eps) w g
    x, gy, pos = torch.zeros(2, 128, device="cuda"), rand(1, 2, 128), torch.zeros(2, dtype=torch.int64, device="cuda")
    y, dx, _, _ = run(L, x, w, w, pos, 1, 1, 64, 64, gy=gy)
    assert (y == 0).all()
    M.near(dx, gy * 1e3, tol_of(64), "dx")


def test_gradients_against_differences(L):
    x, gy = rand(1, 6, 4 * 64), rand(2, 6, 4 * 64)
    wq, wk = 1 + rand(3, 64, scale=0.2), 1 + rand(4, 64, scale=0.2)
    pos = torch.arange(6, device="cuda") + 100
    _, dx, dwq, dwk = run(L, x, wq, wk, pos, 2, 2, 64, 64, gy=gy)
    h = 2.0 ** -6
    for i, (t, g) in enumerate(((x, dx), (wq, dwq), (wk, dwk))):
        dirn = rand(10 + i, *t.shape)
        args = [x, wq, wk]
        vals = []
        for s in (h, -h):
            args[i] = t + s * dirn
            vals.append((run(L, args[0], args[1], args[2], pos, 2, 2, 64, 64).double() * gy.double()).sum().item())
        want = (g.double() * dirn.double()).sum().item()
        bound = (h * h + tol_of(64) / h) * gy.norm().item() * max(dirn.norm().item(), 10.0)
        assert abs((vals[0] - vals[1]) / (2 * h) - want) <= bound


def test_captured_graph_and_streams(L):
    x, gy = rand(1, 256, 12 * 64), rand(2, 256, 12 * 64)
    wq, wk = 1 + rand(3, 64, scale=0.2), 1 + rand(4, 64, scale=0.2)
    pos = torch.arange(64, device="cuda")
    y, dx, dwq, dwk = torch.empty_like(x), torch.empty_like(x), torch.empty_like(wq), torch.empty_like(wq)
    nb = L.aar_qk_norm_rope_bwd_workspace_bytes(256, 6, 6, 64)
    ws = M.scratch(nb)

    def both():
        M.ok(L.aar_qk_norm_rope_fwd_f32(x.data_ptr(), 768, wq.data_ptr(), wk.data_ptr(), pos.data_ptr(), 64, y.data_ptr(), 768,
                                        256, 6, 6, 64, 64, 1e4, 1e-6, M.stream()))
        M.ok(L.aar_qk_norm_rope_bwd_f32(gy.data_ptr(), 768, x.data_ptr(), 768, wq.data_ptr(), wk.data_ptr(), pos.data_ptr(),
                                        64, dx.data_ptr(), 768, dwq.data_ptr(), dwk.data_ptr(), 256, 6, 6, 64, 64, 1e4, 1e-6,
                                        ws.data_ptr(), nb, M.stream()))

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for i in range(3):
        x.copy_(rand(20 + i, 256, 768))
        pos.add_(7)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((y, dx, dwq, dwk), run(L, x, wq, wk, pos, 6, 6, 64, 64, base=1e4, gy=gy)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rotary_dim,heads", [(None, 6), (32, 6), (0, 4)])
def test_ops_and_module(gpu, rotary_dim, heads):
    """nn.MultiHeadAttention with norms: the fused path against its explicit views
    and the whole against 64 bits; positions of each row."""
    rng = np.random.default_rng(3)
    B, T, D = 2, 37, heads * 64
    m = gpu.nn.MultiHeadAttention(D, heads, causal=True, rng=rng, qk_norm=True, rotary_dim=rotary_dim)
    for p, s in ((m.q_norm, 0.3), (m.k_norm, 0.3)):
        p.tensor = dev(gpu, 1 + s * rng.standard_normal(64).astype(np.float32))
    m.to(gpu.Device.CUDA)
    x = rng.standard_normal((B, T, D)).astype(np.float32)
    gy = rng.standard_normal((B, T, D)).astype(np.float32)
    pos = (np.arange(T) + np.array([[0], [1000]])).astype(np.int64)
    params = list(m.parameters())
    assert params[0] is m.q_norm and params[1] is m.k_norm
    r = 64 if rotary_dim is None else rotary_dim
    for given in (None, pos):
        tp = None if given is None or r == 0 else gpu.from_numpy(given).to(gpu.Device.CUDA)
        outs = []
        for forward in (m.forward, m.forward_views):
            m.zero_grad()
            tx = dev(gpu, x, True)
            y = forward(tx, tp)
            y.backward(dev(gpu, gy))
            outs.append([host(gpu, t) for t in (y, tx.grad, *(p.tensor.grad for p in params))])
        X = torch.from_numpy(x).double().requires_grad_()
        w = [torch.from_numpy(host(gpu, p.tensor)).double().requires_grad_() for p in params]
        qkv = (X @ w[2].t() + w[3]).view(B, T, 3, heads, 64)
        rows = torch.from_numpy(np.tile(pos[0], (B, 1)) if tp is None else pos).double()

        def turn(u, wt):
            u = u / torch.sqrt(u.pow(2).mean(-1, keepdim=True) + 1e-6) * wt
            if r == 0:
                return u
            a = rows[:, :, None, None] * 10000.0 ** (torch.arange(r // 2, dtype=torch.float64) * (-2.0 / r))
            u1, u2 = u[..., : r // 2], u[..., r // 2: r]
            return torch.cat([u1 * a.cos() - u2 * a.sin(), u2 * a.cos() + u1 * a.sin(), u[..., r:]], -1)

        q, k, v = turn(qkv[:, :, 0], w[0]).transpose(1, 2), turn(qkv[:, :, 1], w[1]).transpose(1, 2), qkv[:, :, 2].transpose(1, 2)
        s = (q @ k.transpose(2, 3) / 8).masked_fill(torch.ones(T, T).triu(1).bool(), -math.inf)
        ref = (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B, T, D) @ w[4].t() + w[5]
        ref.backward(torch.from_numpy(gy).double())
        want = [ref.detach(), X.grad, *(t.grad for t in w)]
        # normed heads have scores up to sqrt(64); products of D and B T terms around them
        tol = 4 * M.attn_tol(D, max(T, B * T), 16.0)
        for got in outs:
            for i, (g, e) in enumerate(zip(got, want)):
                M.near(g, e, tol, f"output {i}")
