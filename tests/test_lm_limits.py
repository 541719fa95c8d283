"""CPU checks of the sizes that the encoder-reading decoder's entry points take and
refuse: a size query and its call agree, before any launch."""
from __future__ import annotations

import numpy as np
import pytest

import lmops as M

X = 4096  # a pointer that is never dereferenced: every call below returns before any device work


@pytest.fixture(scope="module")
def L():
    return M.lib()


def test_sorted_gradient_sizes(L):
    most = 2 ** 31 - 65537
    for n, vocab, dim, fine in ((4, 2 ** 28 + 77, 1, True), (4, most, 4, True), (4, most + 1, 4, False), (most, 65, 4, True),
                                (most + 1, 65, 4, False), (16384, 5, 1048579, True), (32768, 5, 2 ** 31 - 1, True),
                                (32768, 5, 2 ** 31, False)):
        nb = L.aar_embedding_sorted_bwd_workspace_bytes(n, vocab, dim)
        rc = L.aar_embedding_sorted_bwd_f32(X, X, X, n, vocab, dim, 1.0, None, 0, None)
        assert (nb > 0, rc) == ((True, M.EWORKSPACE) if fine else (False, M.EUNSUPPORTED)), (n, vocab, dim)
        assert not fine or nb >= 8 * n + 4 * vocab


def test_distillation_sizes(L):
    for vocab, top, most in ((80, 16, 2 ** 28 - 16), (81, 16, 2 ** 26 - 4), (80, 17, 2 ** 26 - 4), (2048, 1, 2 ** 26 - 4),
                             (2049, 1, 2 ** 24 - 1), (50000, 64, 2 ** 24 - 1)):
        for n, fine in ((most, True), (most + 1, False)):
            rc = L.aar_distill_fwd_f32(X, X, X, X, X, n, vocab, top, 1.0, None, None, 0, None)
            assert rc == (M.EWORKSPACE if fine else M.EUNSUPPORTED), (vocab, top, n)
            if not fine:
                assert L.aar_distill_bwd_f32(X, X, X, X, X, X, n, vocab, top, 1.0, None) == M.EUNSUPPORTED


def test_temperatures(L, ag):
    """The loss is up to tau^2 ln V, which fp32 holds."""
    up, down = 2.0 ** 61 * 1.001, 2.0 ** -61 * 0.999
    for tau, rc in ((2.0 ** 61, M.EWORKSPACE), (2.0 ** -61, M.EWORKSPACE), (up, M.EINVAL), (down, M.EINVAL), (1e38, M.EINVAL)):
        assert L.aar_distill_fwd_f32(X, X, X, X, X, 4, 8, 2, tau, None, None, 0, None) == rc, tau
    for tau in (up, down, 1e30):
        assert L.aar_distill_bwd_f32(X, X, X, X, X, X, 4, 8, 2, tau, None) == M.EINVAL
        with pytest.raises(ValueError, match="temperature"):
            ag.nn.DistillationLoss(tau)
        with pytest.raises(ValueError, match="temperature"):
            f = ag.from_numpy(np.zeros((4, 8), np.float32))
            ag.distill_loss(f, f, ag.from_numpy(np.zeros((4, 8), np.int64)), tau)
