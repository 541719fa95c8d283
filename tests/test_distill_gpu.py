"""Distillation from a teacher's top logits (aar_distill_*, ag.distill_loss,
nn.DistillationLoss) on the GPU against the definition in 64 bits."""
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


def exact(z, t, ids, tau, grad=1.0):
    """loss and dz in 64 bits (CPU, torch's differentiation)."""
    z = z.detach().double().cpu().requires_grad_()
    t, ids = t.double().cpu(), ids.cpu()
    V = z.shape[1]
    bad = ((ids < -1) | (ids >= V)).any(-1)
    rows = ((ids >= 0) & (t != -math.inf)).any(-1) & ~bad
    there = ids[rows] >= 0
    x = (t[rows] / tau).masked_fill(~there, -math.inf)
    m = x.amax(-1, keepdim=True) if rows.any() else x[:, :1]
    e = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
    s = e.sum(-1, keepdim=True)
    p = e / torch.where(s == 0, torch.ones_like(s), s)
    logq = torch.log_softmax(z[rows] / tau, -1).gather(1, ids[rows].clamp(min=0))
    terms = torch.xlogy(p, p) - torch.where(p > 0, p * logq, torch.zeros_like(p))
    loss = tau * tau * terms.sum() / max(int(rows.sum()), 1)
    loss.backward(torch.tensor(grad, dtype=torch.float64))
    return loss.detach().reshape(1), z.grad


def run(L, z, t, ids, tau, grad=1.0, err=None):
    n, V, K = z.shape[0], z.shape[1], ids.shape[1]
    loss, stats = torch.full((1,), 7.0, device="cuda"), torch.empty(2 * n + 1, device="cuda")
    dz, g = torch.empty(n * V + 4, device="cuda").fill_(7.0), torch.tensor([grad], device="cuda")
    # dz where z's rows stand against 16 bytes, and elsewhere
    off = (z.data_ptr() // 4) % 4
    dz = dz[off:off + n * V].view(n, V)
    nb = L.aar_distill_workspace_bytes(n)
    ws = M.scratch(nb)
    M.ok(L.aar_distill_fwd_f32(z.data_ptr(), t.data_ptr(), ids.data_ptr(), loss.data_ptr(), stats.data_ptr(), n, V, K, tau,
                               M.ptr(err), ws.data_ptr(), nb, M.stream()))
    M.ok(L.aar_distill_bwd_f32(g.data_ptr(), z.data_ptr(), t.data_ptr(), ids.data_ptr(), stats.data_ptr(), dz.data_ptr(), n,
                               V, K, tau, M.stream()))
    return loss, dz


def make(n, V, K, seed=1, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(n, V, generator=g) * spread
    t, ids = (torch.randn(n, V, generator=g) * 1.5 + 0.6 * z).topk(K, -1)
    return z.cuda(), t.cuda().contiguous(), ids.cuda().contiguous()


def check(L, z, t, ids, tau, grad=1.0, what=""):
    loss, dz = run(L, z, t, ids, tau, grad)
    rl, rd = exact(z, t, ids, tau, grad)
    span = float((z.max() - z[torch.isfinite(z)].min()).abs()) / tau
    # q: the exponent's three roundings on up to `span`, sums in chains of 24; p the
    # same over the teacher's entries, so an element is off by so many half steps of
    # q + p; exponentials below 2^-126 are flushed to zero
    steps = 4 * (span + 32)
    n = max(int((((ids >= 0) & (t != -math.inf)).any(-1) & ~((ids < -1) | (ids >= z.shape[1])).any(-1)).sum()), 1)
    bound = torch.zeros_like(rd) + rd.abs()
    c = abs(grad) * tau / n
    at = ids.cpu().clamp(0, z.shape[1] - 1)
    bound.scatter_add_(1, at, torch.full(at.shape, 2 * c, dtype=torch.float64))  # q + p <= |q - p| + 2 p, p <= 1
    far = (dz.double().cpu() - rd).abs() > steps * M.U * bound + 2.0 ** -126 * max(1.0, 2 * c)
    assert int(far.sum() + torch.isnan(dz).sum()) == 0, (what, far.nonzero()[:5].tolist())
    # a row's loss is a difference of numbers up to span + ln V
    assert abs(loss.item() - rl.item()) <= steps * M.U * tau * tau * (span + math.log(z.shape[1]) + 2), what


@pytest.mark.parametrize("tau", [1.0, 2.5])
@pytest.mark.parametrize("n,V,K", [(1, 1, 1), (1, 2, 2), (5, 7, 3), (3, 65, 8), (1000, 65, 8), (77, 1000, 64),
                                   (9, 2047, 5), (10, 2049, 37), (6, 5003, 1), (515, 4096, 16), (3, 50001, 64),
                                   (2, 16384, 1000), (600, 16387, 7), (2, 1024, 1024), (33, 16, 16), (33, 80, 16),
                                   (33, 81, 16), (33, 80, 17), (18, 256, 64), (33, 2048, 9), (255, 16384, 3),
                                   (257, 16384, 3)])
def test_against_the_definition(L, n, V, K, tau):
    check(L, *make(n, V, K), tau, grad=0.7)


@pytest.mark.parametrize("V", [65, 5003, 20001])
def test_absent_entries_and_rows(L, V):
    z, t, ids = make(40, V, 12)
    kept = torch.arange(40, device="cuda")[:, None] % 13
    ids = torch.where(torch.arange(12, device="cuda") < kept, ids, torch.full_like(ids, -1))
    t = torch.where(ids < 0, torch.full_like(t, math.nan), t)  # absent entries' logits are not looked at
    z[::13] = math.nan  # nor those of rows without entries
    loss, dz = run(L, z, t, ids, 1.5)
    on = (ids >= 0).any(-1)
    assert (dz[~on] == 0).all()
    check(L, z.nan_to_num(), t.nan_to_num(), ids, 1.5)
    rl, rd = run(L, z.nan_to_num(), t.nan_to_num(), ids, 1.5)
    assert torch.equal(rl, loss) and torch.equal(rd, dz)
    # none at all
    loss, dz = run(L, z, t, torch.full_like(ids, -1), 1.5)
    assert loss.item() == 0 and (dz == 0).all()


@pytest.mark.parametrize("V", [65, 5003, 20001])
def test_repeated_ids(L, V):
    z, t, ids = make(12, V, 10)
    ids[:, 3] = ids[:, 1]
    ids[:, 9] = ids[:, 1]
    ids[5] = ids[5, 0]
    check(L, z, t, ids, 2.0)


@pytest.mark.parametrize("V", [65, 5003])
def test_ids_outside(L, V):
    z, t, ids = make(12, V, 10)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    run(L, z, t, ids, 1.0, err=err)
    assert int(err) == 0
    ids[3, 2] = V
    ids[7, 9] = -2
    ids[9, 0] = 2 ** 40
    loss, dz = run(L, z, t, ids, 1.0, err=err)
    assert int(err) == 1 and (dz[[3, 7, 9]] == 0).all()
    check(L, z, t, ids, 1.0)


@pytest.mark.parametrize("V", [65, 5003])
def test_extreme_logits(L, V):
    # a masked vocabulary, a teacher with -inf entries, large magnitudes
    z, t, ids = make(8, V, 6)
    hidden = torch.ones(8, V, dtype=torch.bool, device="cuda").scatter_(1, ids, False)
    hidden[:, V // 2:] &= False
    z = z.masked_fill(hidden, -math.inf)
    t[:, 4:] = -math.inf
    t[2] = -math.inf  # nothing to learn from: left out
    check(L, z, t, ids, 1.0, what="masked")
    assert (run(L, z, t, ids, 1.0)[1][2] == 0).all()
    z, t, ids = make(8, V, 6, spread=1.0)
    check(L, z * 300, t * 300, ids, 1.0, what="large")
    check(L, z + 1e4, t - 1e4, ids, 4.0, what="offset")
    # a student that excludes what the teacher names: an infinite loss, the gradient of p alone there
    z[0, ids[0, 0]] = -math.inf
    loss, dz = run(L, z, t, ids, 1.0)
    assert loss.item() == math.inf and torch.isfinite(dz).all()


@pytest.mark.parametrize("V,offset", [(64, 1), (65, 2), (5003, 3), (4096, 1)])
def test_alignment(L, V, offset):
    z, t, ids = make(9, V, 5)
    buf = torch.empty(9 * V + 4, device="cuda")
    moved = buf[offset:offset + 9 * V].view(9, V)
    moved.copy_(z)
    check(L, moved, t, ids, 1.0)
    # z and dz that stand differently against 16 bytes
    n, K = 9, 5
    loss, stats, g = torch.empty(1, device="cuda"), torch.empty(2 * n + 1, device="cuda"), torch.ones(1, device="cuda")
    dz, ws = torch.empty(n, V, device="cuda"), M.scratch(4 * n)
    M.ok(L.aar_distill_fwd_f32(moved.data_ptr(), t.data_ptr(), ids.data_ptr(), loss.data_ptr(), stats.data_ptr(), n, V, K,
                               1.0, None, ws.data_ptr(), 4 * n, M.stream()))
    M.ok(L.aar_distill_bwd_f32(g.data_ptr(), moved.data_ptr(), t.data_ptr(), ids.data_ptr(), stats.data_ptr(), dz.data_ptr(),
                               n, V, K, 1.0, M.stream()))
    assert torch.equal(dz, run(L, moved, t, ids, 1.0)[1])


def test_gradient_against_differences(L):
    z, t, ids = make(20, 300, 8)
    _, dz = run(L, z, t, ids, 1.5)
    w = torch.randn(20, 300, generator=torch.Generator().manual_seed(3)).cuda()
    h = 2.0 ** -5
    up, down = run(L, z + h * w, t, ids, 1.5)[0].item(), run(L, z - h * w, t, ids, 1.5)[0].item()
    want = (dz.double() * w.double()).sum().item()
    # the loss is a mean of log-sums of directions of unit variance: third derivatives of order 1
    assert abs((up - down) / (2 * h) - want) <= h * h + 40 * M.U * 20 / h


def test_captured_graph_and_streams(L):
    z, t, ids = make(64, 3001, 9)
    n, V, K = 64, 3001, 9
    loss, stats, g = torch.empty(1, device="cuda"), torch.empty(2 * n + 1, device="cuda"), torch.ones(1, device="cuda")
    dz, ws = torch.empty(n, V, device="cuda"), M.scratch(4 * n)

    def both():
        M.ok(L.aar_distill_fwd_f32(z.data_ptr(), t.data_ptr(), ids.data_ptr(), loss.data_ptr(), stats.data_ptr(), n, V, K,
                                   2.0, None, ws.data_ptr(), 4 * n, M.stream()))
        M.ok(L.aar_distill_bwd_f32(g.data_ptr(), z.data_ptr(), t.data_ptr(), ids.data_ptr(), stats.data_ptr(),
                                   dz.data_ptr(), n, V, K, 2.0, M.stream()))

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for i in range(3):
        a, b, c = make(n, V, K, 10 + i)
        c[i * 5:i * 9] = -1
        z.copy_(a), t.copy_(b), ids.copy_(c)
        graph.replay()
        torch.cuda.synchronize()
        rl, rd = run(L, z, t, ids, 2.0)
        assert torch.equal(loss, rl) and torch.equal(dz, rd)


def test_ops_and_module(gpu):
    z, t, ids = make(30, 65, 8)
    ids[4:9, 3:] = -1
    crit = gpu.nn.DistillationLoss(2.0)
    tz = dev(gpu, z.cpu().numpy().reshape(5, 6, 65), True)
    tt = dev(gpu, t.cpu().numpy().reshape(5, 6, 8))
    ti = gpu.from_numpy(ids.cpu().numpy().reshape(5, 6, 8)).to(gpu.Device.CUDA)
    loss = crit(tz, tt, ti)
    loss.backward()
    rl, rd = exact(z, t, ids, 2.0)
    M.near(host(gpu, loss).reshape(1), rl, 64 * M.U, "loss")
    M.near(host(gpu, tz.grad).reshape(30, 65), rd, 64 * M.U, "dz")
    bad = ids.clone()
    bad[0, 0] = 65
    with pytest.raises(IndexError, match="distill_loss"):
        host(gpu, gpu.distill_loss(dev(gpu, z.cpu().numpy()), dev(gpu, t.cpu().numpy()),
                                   gpu.from_numpy(bad.cpu().numpy()).to(gpu.Device.CUDA)))
    assert np.isfinite(host(gpu, gpu.distill_loss(dev(gpu, z.cpu().numpy()), dev(gpu, t.cpu().numpy()),
                                                  gpu.from_numpy(ids.cpu().numpy()).to(gpu.Device.CUDA))))
