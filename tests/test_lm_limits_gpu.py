"""The encoder-reading decoder's operators at the ends of what they take: large tables,
many rows, many lengths, extreme temperatures."""
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


def test_positions_of_many_lengths(gpu):
    """nn.MultiHeadAttention makes the positions 0 .. T-1 itself; what it keeps of them does
    not grow with every length it meets."""
    m = gpu.nn.MultiHeadAttention(16, 2, qk_norm=True, rng=np.random.default_rng(0)).to(gpu.Device.CUDA)
    rng = np.random.default_rng(1)
    x = rng.standard_normal((2, 1000, 16)).astype(np.float32)
    m(dev(gpu, x))
    gpu.cuda_synchronize()
    before = gpu._core._memory_in_use()
    for T in range(1, 1000, 13):
        part = np.ascontiguousarray(x[:, :T])
        y = host(gpu, m(dev(gpu, part)))
        ramp = gpu.from_numpy(np.arange(T, dtype=np.int64)).to(gpu.Device.CUDA)
        np.testing.assert_array_equal(y, host(gpu, m(dev(gpu, part), ramp)))
        del ramp
    assert gpu._core._memory_in_use() == before
    assert host(gpu, m(dev(gpu, x[:, :0]))).shape == (2, 0, 16)


@pytest.mark.parametrize("dim", [1, 4])
def test_gradient_of_a_table_past_2_28_rows(L, dim):
    """Every row of the table is written: the sums of the rows that have tokens, zeros
    elsewhere."""
    vocab, n = 2 ** 28 + 77, 40
    at = torch.tensor([0, 1, 5, 2 ** 20, 2 ** 28 - 1, 2 ** 28, vocab - 2, vocab - 1], device="cuda")
    ids = at.repeat(5)
    g = torch.randint(-8, 9, (n, dim), generator=torch.Generator().manual_seed(3)).float().cuda()  # exact sums
    dw = torch.full((vocab, dim), 7.0, device="cuda")
    nb = L.aar_embedding_sorted_bwd_workspace_bytes(n, vocab, dim)
    ws = M.scratch(nb)
    M.ok(L.aar_embedding_sorted_bwd_f32(g.data_ptr(), ids.data_ptr(), dw.data_ptr(), n, vocab, dim, 2.0, ws.data_ptr(), nb,
                                        M.stream()))
    want = 2.0 * g.view(5, 8, dim).sum(0)
    assert torch.equal(dw[at], want)
    dw[at] = 0.0
    assert int(torch.count_nonzero(dw)) == 0


def test_gradient_of_rows_of_a_million_columns(L):
    """Columns of more than one launch; the tokens that are not named are never read, so
    their gradients need not be there."""
    n, vocab, dim = 16384, 5, 1048579
    at = torch.arange(0, n, 257, device="cuda")
    ids = torch.full((n,), -1, dtype=torch.int64, device="cuda")
    ids[at] = torch.where(torch.arange(len(at), device="cuda") < 50, 3, 1)  # 50 tokens: four chunks of sorted tokens
    g = torch.empty(n, dim, device="cuda")
    g[at] = torch.randint(-8, 9, (len(at), dim), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").float()
    dw = torch.full((vocab, dim), 7.0, device="cuda")
    nb = L.aar_embedding_sorted_bwd_workspace_bytes(n, vocab, dim)
    ws = M.scratch(nb)
    M.ok(L.aar_embedding_sorted_bwd_f32(g.data_ptr(), ids.data_ptr(), dw.data_ptr(), n, vocab, dim, 1.0, ws.data_ptr(), nb,
                                        M.stream()))
    assert torch.equal(dw[3], g[at[:50]].sum(0)) and torch.equal(dw[1], g[at[50:]].sum(0))
    assert int(torch.count_nonzero(dw[[0, 2, 4]])) == 0
    del g, ws, dw
    torch.cuda.empty_cache()


def distill(L, z, t, ids, tau, grad=1.0):
    n, V, K = z.shape[0], z.shape[1], ids.shape[1]
    loss, stats = torch.full((1,), 7.0, device="cuda"), torch.empty(2 * n + 1, device="cuda")
    dz, g = torch.full_like(z, 7.0), torch.tensor([grad], device="cuda")
    nb = L.aar_distill_workspace_bytes(n)
    ws = M.scratch(nb)
    M.ok(L.aar_distill_fwd_f32(z.data_ptr(), t.data_ptr(), ids.data_ptr(), loss.data_ptr(), stats.data_ptr(), n, V, K, tau,
                               None, ws.data_ptr(), nb, M.stream()))
    M.ok(L.aar_distill_bwd_f32(g.data_ptr(), z.data_ptr(), t.data_ptr(), ids.data_ptr(), stats.data_ptr(), dz.data_ptr(), n,
                               V, K, tau, M.stream()))
    return loss, dz


@pytest.mark.parametrize("V", [5, 96])
def test_distillation_of_many_rows(L, V):
    """16384 sequences of 256 tokens, and one row more: the loss is the mean over all of
    them, a row's gradient that of the same row in a small batch, but for the mean."""
    n, part = 16384 * 256 + 1, 1024
    gen = torch.Generator(device="cuda").manual_seed(1)
    z = torch.randn(n, V, generator=gen, device="cuda")
    t = torch.randn(n, 2, generator=gen, device="cuda")
    ids = torch.randint(0, V, (n, 2), generator=gen, device="cuda")
    loss, dz = distill(L, z, t, ids, 1.0, float(n))
    for at in (0, 16384 * 255, n - part):
        one, dpart = distill(L, z[at:at + part].clone(), t[at:at + part].clone(), ids[at:at + part].clone(), 1.0, float(part))
        # grad / rows is 1 in both
        assert torch.equal(dz[at:at + part], dpart)
    p = torch.softmax(t.double(), -1)
    logq = torch.log_softmax(z.double(), -1).gather(1, ids)
    want = (torch.xlogy(p, p) - p * logq).sum(-1).mean().item()
    # each row's loss is a difference of numbers of up to 16: 64 half steps, as for small batches
    assert abs(loss.item() - want) <= 64 * M.U * 16


@pytest.mark.parametrize("tau", [2.0 ** -61, 2.0 ** -40, 2.0 ** 40, 2.0 ** 61])
def test_distillation_at_extreme_temperatures(L, tau):
    """The loss, up to tau^2 ln V, stays in fp32's range, so loss and gradient are finite, and infinite where the
    student excludes what the teacher names."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    for V, K in ((33, 5), (3001, 20)):
        z = torch.randn(6, V, generator=gen, device="cuda")
        t, ids = (torch.randn(6, V, generator=gen, device="cuda")).topk(K, -1)
        loss, dz = distill(L, z, t.contiguous(), ids, tau)
        p = torch.softmax(t.double() / tau, -1)
        logq = torch.log_softmax(z.double() / tau, -1)
        want = (tau * tau * (torch.xlogy(p, p) - p * logq.gather(1, ids)).sum(-1).mean()).item()
        # a row's loss is a difference of numbers up to 12 / tau + ln V, each off by 64 half steps
        assert abs(loss.item() - want) <= 64 * M.U * tau * tau * (12 / tau + 9)
        dref = tau / 6 * torch.exp(logq).scatter_add(1, ids, -p)
        # entries of q and p are at most 1; no two logits are so near that a small tau leaves their weights open
        assert ((dz.double() - dref).abs() <= tau / 6 * 64 * M.U).all()
        z[0, ids[0, 0]] = -float("inf")
        assert distill(L, z, t.contiguous(), ids, tau)[0].item() == float("inf")
