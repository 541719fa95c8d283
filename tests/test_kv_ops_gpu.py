"""window_attention, KVCache and MultiHeadAttention's window and decode through the host
layer: values and gradients against 64 bits, text generated through the cache against
what it holds, forks, windows that give pages back."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import kvops as K
import lmops as M
from devutil import dev, host

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def on_gpu(gpu):
    pass


def randn(seed, *shape, scale=1.0):
    return (np.random.default_rng(seed).standard_normal(shape) * scale).astype(np.float32)


def t64(x):
    return torch.from_numpy(np.asarray(x)).double()


@pytest.mark.parametrize("shape", [(2, 4, 2, 90, 64, 20, 3), (1, 3, 3, 33, 30, 7, 0), (1, 8, 1, 140, 128, 500, 0)])
def test_window_attention(ag, shape):
    B, H, Hkv, T, d, window, sinks = shape
    q, k, v, w = randn(1, B, H, T, d), randn(2, B, Hkv, T, d), randn(3, B, Hkv, T, d), randn(4, B, H, T, d)
    tq, tk, tv = (dev(ag, x, True) for x in (q, k, v))
    out = ag.window_attention(tq, tk, tv, window, sinks)
    ag.sum_all(ag.mul(out, dev(ag, w))).backward()
    ref, mass = K.window_exact(*(torch.from_numpy(x).cuda() for x in (q, k, v, w)), window, sinks)
    tol = M.attn_tol(d, T * H // Hkv)
    M.near(host(ag, out), ref[0], tol, "o")
    for name, t, r in zip(("dq", "dk", "dv"), (tq, tk, tv), ref[2:]):
        M.near(host(ag, t.grad), r, 2 * tol, name, mass.get(name))


def test_window_attention_reads_views(ag):
    """Head views of a packed projection, heads and rows in other orders."""
    B, T, H, d = 2, 50, 3, 64
    x = dev(ag, randn(1, B, T, 3, H, d), True)
    view = lambda i: ag.transpose(ag.squeeze(ag.slice(x, 2, i, i + 1), 2), 1, 2)  # noqa: E731
    out = ag.window_attention(view(0), view(1), view(2), 9, 1)
    dense = ag.window_attention(*(ag.contiguous(view(i)) for i in range(3)), 9, 1)
    assert np.array_equal(host(ag, out), host(ag, dense))
    # head and row swapped: rows closer together than their length
    y = dev(ag, randn(2, B, d, T, H))
    swapped = ag.transpose(y, 1, 3)  # [B, H, T, d], strides (.., 1, H, T H)
    assert np.array_equal(host(ag, ag.window_attention(swapped, swapped, swapped, 5, 0)),
                          host(ag, ag.window_attention(*[ag.contiguous(swapped)] * 3, 5, 0)))


@pytest.mark.parametrize("qk_norm", [False, True])
def test_multi_head_attention_window(ag, qk_norm):
    """The packed and the per-head paths agree, and a window of the whole text is
    causal attention."""
    rng = np.random.default_rng(3)
    x, w = randn(4, 2, 70, 96), randn(5, 2, 70, 96)

    def grads(m, call):
        m.zero_grad()
        out = call(dev(ag, x))
        ag.sum_all(ag.mul(out, dev(ag, w))).backward()
        return [host(ag, out)] + [host(ag, p.tensor.grad) for p in m.parameters()]

    m = ag.nn.MultiHeadAttention(96, 4, causal=True, rng=rng, qk_norm=qk_norm, window=16, sinks=2).to(ag.Device.CUDA)
    for a, b in zip(grads(m, m.forward), grads(m, m.forward_views)):
        M.near(a, t64(b), 4 * M.attn_tol(96, 140), "views")
    plain = ag.nn.MultiHeadAttention(96, 4, causal=True, rng=np.random.default_rng(9), qk_norm=qk_norm)
    wide = ag.nn.MultiHeadAttention(96, 4, causal=True, rng=np.random.default_rng(9), qk_norm=qk_norm, window=70)
    for a, b in zip(*(grads(n.to(ag.Device.CUDA), n.forward) for n in (wide, plain))):
        M.near(a, t64(b), 8 * M.attn_tol(96, 140), "causal")


def heads_of(m, x, positions, ag):
    q, k, v = m._split_heads(m.qkv_proj(x))
    if m.qk_norm:
        q, k = m._rotate_heads(q, k, positions)
    return (host(ag, ag.contiguous(t)) for t in (q, k, v))


@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3)])
def test_decode_against_what_the_cache_holds(ag, qk_norm, window, sinks):
    """Prompts of several lengths, then token by token: every step's output is attention
    over the numbers that the cache then holds, and these are the model's keys and values
    to half a step of their scale."""
    B, D, H, lens = 3, 128, 2, (50, 7, 64)
    m = ag.nn.MultiHeadAttention(D, H, causal=True, rng=np.random.default_rng(1), qk_norm=qk_norm, window=window,
                                 sinks=sinks).to(ag.Device.CUDA)
    cache = ag.KVCache(2, B, H, D // H, 140, page=32, window=window or 0, sinks=sinks)
    text = randn(2, B, 140, D)
    done = np.zeros(B, np.int64)
    wo, bo = t64(host(ag, m.out_proj.weight.tensor)), t64(host(ag, m.out_proj.bias.tensor))
    for counts in (lens, (1, 1, 1), (20, 0, 33), (1, 1, 1), (1, 40, 0), (1, 1, 1)):
        T = max(counts)
        x = np.zeros((B, T, D), np.float32)
        pos = np.zeros((B, T), np.int64)
        for b, n in enumerate(counts):
            x[b, :n] = text[b, done[b] : done[b] + n]
            pos[b] = done[b] + np.arange(T)
        cache.extend(list(counts))
        done += counts
        assert list(cache.lengths) == list(done)
        out = host(ag, m.decode(dev(ag, x), cache, 1))
        assert np.array_equal(host(ag, cache.positions()), pos)
        q, k, v = heads_of(m, dev(ag, x), ag.from_numpy(pos).to(ag.Device.CUDA), ag)
        kc, vc = (host(ag, t) for t in cache.read(1, 0, 140))
        for b, n in enumerate(counts):
            if n == 0:
                continue
            for got, new in ((kc, k), (vc, v)):
                assert np.abs(got[b, :, done[b] - n : done[b]] - new[b, :, :n]).max() <= np.abs(text).max() * 64 / 127
        ref = K.cache_exact(torch.from_numpy(q), [t64(kc[b, :, : done[b]]) for b in range(B)],
                            [t64(vc[b, :, : done[b]]) for b in range(B)], done, counts, window or 1 << 62, sinks)
        ref = ref.permute(0, 2, 1, 3).reshape(B, T, D) @ wo.t() + bo
        # the projection's sums of D products on top of the attention's
        M.near(out, ref, 2 * M.attn_tol(D // H, 140) + 4 * M.U * math.sqrt(D), "out")
    ag.cuda_synchronize()


def test_chunks_leave_the_same_cache(ag):
    """A text at once and token by token through the class: the same keys and values."""
    k, v = randn(1, 1, 2, 100, 40), randn(2, 1, 2, 100, 40)
    a, b = (ag.KVCache(1, 1, 2, 40, 100, page=32) for _ in range(2))
    a.extend([100])
    a.append(0, dev(ag, k), dev(ag, v))
    for t in range(100):
        b.extend([1])
        b.append(0, dev(ag, k[:, :, t : t + 1]), dev(ag, v[:, :, t : t + 1]))
    for x, y, rows in zip(a.read(0, 0, 100), b.read(0, 0, 100), (k, v)):
        assert np.array_equal(host(ag, x), host(ag, y))
        for h in range(2):
            M.near(host(ag, x)[0, h], K.quantised(torch.from_numpy(rows[0, h]), 32), M.U, "held")


def test_forks_and_frees(ag):
    """A fork shares full pages, goes its own way, and outlives its parent."""
    H, d = 2, 64
    cache = ag.KVCache(2, 3, H, d, 128, page=32, pages=9)
    x = randn(1, 3, H, 200, d)

    def step(layer_rows, counts):
        cache.extend(counts)
        for layer in (0, 1):
            cache.append(layer, dev(ag, layer_rows + layer), dev(ag, layer_rows - layer))

    step(x[:, :, :70], [70, 0, 0])
    assert cache.free_pages == 6
    cache.fork(0, 2)
    assert list(cache.lengths) == [70, 0, 70] and cache.free_pages == 5  # two shared, one copied
    same = [host(ag, t) for layer in (0, 1) for t in cache.read(layer, 0, 70)]
    assert all(np.array_equal(t[0], t[2]) for t in same)
    step(x[:, :, 100:130], [30, 0, 10])
    a = [host(ag, t) for layer in (0, 1) for t in cache.read(layer, 0, 100)]
    for t in a:
        assert np.array_equal(t[0, :, :64], t[2, :, :64]) and not np.array_equal(t[0, :, 70:80], t[2, :, 70:80])
    assert cache.free_pages == 4
    cache.free(0)
    assert list(cache.lengths) == [0, 0, 80] and cache.free_pages == 4 + 2  # the shared two stay
    b = [host(ag, t) for layer in (0, 1) for t in cache.read(layer, 0, 100)]
    for s, t in zip(a, b):
        assert np.array_equal(s[2], t[2]) and (t[0] == 0).all()
    with pytest.raises(RuntimeError):  # 6 free pages, 7 needed; nothing changes
        cache.extend([97, 97, 0])
    assert list(cache.lengths) == [0, 0, 80] and cache.free_pages == 6
    cache.fork(2, 2)
    cache.fork(2, 0)
    cache.free(2)
    cache.free(0)
    assert cache.free_pages == 9
    ag.cuda_synchronize()


def test_a_window_gives_pages_back(ag):
    """Text without end in a pool that holds the window's pages and the sinks'."""
    H, d, window, sinks = 2, 64, 50, 3
    cache = ag.KVCache(1, 1, H, d, 1000, page=32, pages=5, window=window, sinks=sinks)
    k, v, q = randn(1, 1, H, 1000, d), randn(2, 1, H, 1000, d), randn(3, 1, 2 * H, 1000, d)
    at = 0
    for n in (40, 1, 30, 1, 1, 29) + (31, 1) * 20:
        cache.extend([n])
        cache.append(0, dev(ag, k[:, :, at : at + n]), dev(ag, v[:, :, at : at + n]))
        out = host(ag, ag.contiguous(cache.attend(0, dev(ag, q[:, :, at : at + n]))))
        at += n
    kq = [torch.stack([K.quantised(torch.from_numpy(x[0, h, :at]), 32) for h in range(H)]) for x in (k, v)]
    ref = K.cache_exact(torch.from_numpy(q[:, :, at - n : at]), [kq[0]], [kq[1]], [at], [n], window, sinks)
    M.near(out, ref, M.attn_tol(d, window + sinks), "o")
    ag.cuda_synchronize()


def test_errors(ag):
    cache = ag.KVCache(1, 2, 2, 64, 64, page=32)
    x = dev(ag, randn(1, 2, 2, 5, 64))
    for bad in ([1], [1, 2, 3], [-1, 0], [65, 0]):
        with pytest.raises(ValueError):
            cache.extend(bad)
    cache.extend([5, 3])
    with pytest.raises(IndexError):
        cache.append(1, x, x)
    with pytest.raises(IndexError):
        cache.attend(-1, x)
    with pytest.raises(IndexError):
        cache.fork(0, 2)
    with pytest.raises(IndexError):
        cache.free(-1)
    for k, v in ((x, dev(ag, randn(1, 2, 2, 4, 64))), (dev(ag, randn(1, 2, 4, 5, 64)), x), (dev(ag, randn(1, 2, 5, 64)), x)):
        with pytest.raises(ValueError):
            cache.append(0, k, v)
    with pytest.raises(ValueError):
        cache.attend(0, dev(ag, randn(1, 2, 3, 5, 64)))
    with pytest.raises(RuntimeError):
        cache.append(0, ag.from_numpy(randn(1, 2, 2, 5, 64)), x)
    cache.append(0, x, x)
    assert (host(ag, ag.contiguous(cache.attend(0, x)))[1, :, 3:] == 0).all()
    cache.extend([0, 0])
    none = dev(ag, np.zeros((2, 2, 0, 64), np.float32))
    cache.append(0, none, none)
    assert list(cache.attend(0, none).shape) == [2, 2, 0, 64]
    m = ag.nn.MultiHeadAttention(128, 2, causal=True, window=8).to(ag.Device.CUDA)
    with pytest.raises(ValueError):
        m.decode(dev(ag, randn(1, 2, 5, 128)), cache, 0)


def test_the_order_of_a_step_is_kept(ag):
    """Twice the same rows, attention before them, a fork between them and layers that miss
    a step are refused, and change nothing."""
    cache = ag.KVCache(2, 2, 2, 64, 128, page=32)
    x, y = dev(ag, randn(1, 2, 2, 40, 64)), dev(ag, randn(2, 2, 2, 1, 64))
    cache.extend([40, 33])
    with pytest.raises(RuntimeError):
        cache.attend(0, x)
    with pytest.raises(RuntimeError):
        cache.read(0, 0, 1)
    cache.append(0, x, x)
    with pytest.raises(RuntimeError):
        cache.append(0, x, x)
    with pytest.raises(RuntimeError):
        cache.fork(0, 1)
    cache.append(1, x, x)
    before = [host(ag, t) for t in cache.read(1, 0, 64)]
    out = host(ag, ag.contiguous(cache.attend(1, x)))
    with pytest.raises(RuntimeError):
        cache.append(1, x, x)
    assert all(np.array_equal(a, host(ag, b)) for a, b in zip(before, cache.read(1, 0, 64)))
    assert np.array_equal(out, host(ag, ag.contiguous(cache.attend(1, x))))
    cache.extend([0, 0])  # no tokens: nothing is missed
    cache.extend([1, 1])
    cache.append(1, y, y)
    cache.extend([0, 1])  # layer 0 has missed a step
    cache.append(1, y, y)
    with pytest.raises(RuntimeError):
        cache.append(0, y, y)
    with pytest.raises(RuntimeError):
        cache.attend(0, y)
    with pytest.raises(RuntimeError):
        cache.read(0, 0, 1)
    cache.fork(1, 0)
    assert list(cache.lengths) == [35, 35]
    rows = host(ag, cache.read(1, 0, 35)[0])
    assert np.array_equal(rows[0], rows[1])
    cache.free(0)
    cache.free(1)
    cache.extend([1, 0])
    cache.append(0, y, y)
    assert np.isfinite(host(ag, ag.contiguous(cache.attend(0, y)))).all()
    ag.cuda_synchronize()
