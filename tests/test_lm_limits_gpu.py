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
