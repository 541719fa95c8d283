"""Scaled embedding and its gradient by sorted tokens (aar_embedding_scaled_fwd_f32,
aar_embedding_sorted_bwd_f32, ag.embedding_scaled, nn.Embedding(scale=...)) on the
GPU.  The lookup is one fp32 product, so exact; a gradient's element sums c
products, off by at most c + 1 half steps of the sum of their magnitudes, in any
order."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import lmops as M
from devutil import dev, host

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L(gpu):
    return M.lib()


def grad(L, g, ids, vocab, scale, ws=None):
    n, dim = g.shape
    dw = torch.full((vocab, dim), 7.0, device="cuda")
    nb = L.aar_embedding_sorted_bwd_workspace_bytes(n, vocab, dim)
    ws = M.scratch(nb) if ws is None else ws
    M.ok(L.aar_embedding_sorted_bwd_f32(M.ptr(g), M.ptr(ids), dw.data_ptr(), n, vocab, dim, scale, ws.data_ptr(), nb,
                                        M.stream()))
    return dw


def check_grad(L, g, ids, vocab, scale=1.5):
    dw = grad(L, g, ids, vocab, scale).double()
    inside = (ids >= 0) & (ids < vocab)
    at, rows = ids[inside], g[inside].double()
    ref = torch.zeros(vocab, g.shape[1], dtype=torch.float64, device="cuda").index_add_(0, at, rows) * scale
    mass = torch.zeros_like(ref).index_add_(0, at, rows.abs()) * abs(scale)
    count = torch.bincount(at, minlength=vocab)[:, None].double()
    assert ((dw - ref).abs() <= (count + 1) * M.U * mass).all()
    assert (dw[count[:, 0] == 0] == 0).all()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ids_of(kind, n, vocab, seed=1):
    g = gen(seed)
    if kind == "uniform":
        return torch.randint(0, vocab, (n,), generator=g, device="cuda")
    if kind == "one":
        return torch.full((n,), vocab - 1, device="cuda", dtype=torch.int64)
    if kind == "sorted":
        return torch.sort(torch.randint(0, vocab, (n,), generator=g, device="cuda")).values
    if kind == "two":  # two tokens share nearly all
        return torch.where(torch.rand(n, generator=g, device="cuda") < 0.7, 0, vocab // 2).long()
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    rank = torch.exp(u * np.log(vocab + 1.0)).long().sub_(1).clamp_(0, vocab - 1)
    return torch.randperm(vocab, generator=g, device="cuda")[rank]


@pytest.mark.parametrize("kind", ["uniform", "one", "sorted", "two", "zipf"])
@pytest.mark.parametrize("n,vocab,dim", [
    (1, 1, 4), (1, 5000, 384), (2, 1, 1), (15, 16, 3), (16, 65, 64), (17, 65, 260), (1023, 65, 384), (1025, 257, 5),
    (4096, 1000, 256), (16384, 65, 384), (16385, 50001, 68), (5000, 300001, 12), (40000, 7, 33), (70000, 1024, 8), (32768, 300, 20),
    (32769, 300, 20), (65536, 65, 4), (65537, 33, 7)])
def test_gradient(L, n, vocab, dim, kind):
    g = torch.randn(n, dim, generator=gen(2), device="cuda")
    check_grad(L, g, ids_of(kind, n, vocab), vocab)


def test_gradient_of_ids_outside(L):
    ids = ids_of("uniform", 3000, 500)
    ids[::7] = -1
    ids[3::11] = 500
    ids[5::13] = 2 ** 40
    ids[6::17] = -(2 ** 40)
    check_grad(L, torch.randn(3000, 128, generator=gen(2), device="cuda"), ids, 500)
    check_grad(L, torch.randn(100, 128, generator=gen(2), device="cuda"), torch.full((100,), -1, device="cuda"), 500)


def test_gradient_alignment_and_reproducibility(L):
    n, vocab, dim = 9000, 3001, 64
    ids = ids_of("zipf", n, vocab)
    buf = torch.randn(n * dim + 1, generator=gen(2), device="cuda")
    check_grad(L, buf[1:].view(n, dim), ids, vocab)  # unaligned rows: element-wise
    g = buf[:-1].view(n, dim)
    first = grad(L, g, ids, vocab, 2.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = grad(L, g, ids, vocab, 2.0)
    side.synchronize()
    assert torch.equal(first, second)


def test_gradient_of_a_captured_graph(L):
    n, vocab, dim = 5000, 700, 96
    ids, g = ids_of("zipf", n, vocab), torch.randn(n, dim, generator=gen(2), device="cuda")
    dw = torch.empty(vocab, dim, device="cuda")
    nb = L.aar_embedding_sorted_bwd_workspace_bytes(n, vocab, dim)
    ws = M.scratch(nb)

    def call():
        M.ok(L.aar_embedding_sorted_bwd_f32(g.data_ptr(), ids.data_ptr(), dw.data_ptr(), n, vocab, dim, 0.5, ws.data_ptr(),
                                            nb, M.stream()))

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(3):
        ids.copy_(ids_of(("uniform", "one", "two")[i], n, vocab, 10 + i))
        g.copy_(torch.randn(n, dim, generator=gen(20 + i), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dw, grad(L, g, ids, vocab, 0.5))


@pytest.mark.parametrize("n,vocab,dim,offset", [(1, 1, 1, 0), (5, 7, 4, 0), (1000, 65, 384, 0), (333, 5000, 30, 0),
                                                (64, 100, 64, 1)])
def test_lookup(gpu, L, n, vocab, dim, offset):
    w = torch.randn(vocab * dim + offset, generator=gen(1), device="cuda")[offset:].view(vocab, dim)
    ids = ids_of("uniform", n, vocab)
    out = torch.full((n, dim), 7.0, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    call = lambda: M.ok(L.aar_embedding_scaled_fwd_f32(w.data_ptr(), ids.data_ptr(), out.data_ptr(), n, vocab, dim, 2.3,  # noqa: E731
                                                       err.data_ptr(), M.stream()))
    call()
    assert torch.equal(out, w[ids] * torch.tensor(2.3, device="cuda")) and int(err) == 0
    ids[0] = vocab
    call()
    assert (out[0] == 0).all() and int(err) == 1


def test_ops_and_module(gpu):
    rng = np.random.default_rng(2)
    V, D = 1000, 48
    emb = gpu.nn.Embedding(V, D, rng=np.random.default_rng(7), scale=D ** 0.5)
    plain = gpu.nn.Embedding(V, D, rng=np.random.default_rng(7))
    emb.to(gpu.Device.CUDA), plain.to(gpu.Device.CUDA)
    ids = rng.integers(0, V, (6, 50)).astype(np.int64)
    ti = gpu.from_numpy(ids).to(gpu.Device.CUDA)
    gy = rng.standard_normal((6, 50, D)).astype(np.float32)
    y = emb(ti)
    np.testing.assert_array_equal(host(gpu, y), host(gpu, plain(ti)) * np.float32(D ** 0.5))
    y.backward(dev(gpu, gy))
    ref = np.zeros((V, D))
    np.add.at(ref, ids.ravel(), gy.reshape(-1, D).astype(np.float64) * D ** 0.5)
    mass = np.zeros((V, D))
    np.add.at(mass, ids.ravel(), np.abs(gy.reshape(-1, D)).astype(np.float64) * D ** 0.5)
    # at most 8 tokens share a row here; the scale itself is rounded once
    assert np.bincount(ids.ravel()).max() <= 8
    assert (np.abs(host(gpu, emb.weight.tensor.grad) - ref) <= 10 * M.U * mass).all()
    with pytest.raises(IndexError):
        host(gpu, emb(gpu.from_numpy(np.array([V], np.int64)).to(gpu.Device.CUDA)))


def test_large_vocabulary_through_the_plain_embedding(gpu):
    """n * vocab above 2^30, which the one-hot product refuses: ag.embedding takes
    the sorted gradient."""
    V, D, n = 300000, 8, 4096
    rng = np.random.default_rng(4)
    w = dev(gpu, rng.standard_normal((V, D)).astype(np.float32), True)
    ids = rng.integers(0, V, n).astype(np.int64)
    gy = rng.standard_normal((n, D)).astype(np.float32)
    gpu.embedding(w, gpu.from_numpy(ids).to(gpu.Device.CUDA)).backward(dev(gpu, gy))
    ref = np.zeros((V, D))
    np.add.at(ref, ids, gy.astype(np.float64))
    mass = np.zeros((V, D))
    np.add.at(mass, ids, np.abs(gy).astype(np.float64))
    assert np.bincount(ids).max() <= 8
    assert (np.abs(host(gpu, w.grad) - ref) <= 9 * M.U * mass).all()
