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
