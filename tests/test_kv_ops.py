"""Argument checks of window_attention, KVCache and MultiHeadAttention's window; no GPU."""
from __future__ import annotations

import numpy as np
import pytest


def cpu(ag, *shape):
    return ag.from_numpy(np.zeros(shape, np.float32))


def test_window_attention_refusals(ag):
    q, k = cpu(ag, 1, 4, 3, 8), cpu(ag, 1, 2, 3, 8)
    for args, kw in (((q, cpu(ag, 1, 3, 3, 8), cpu(ag, 1, 3, 3, 8)), {}), ((q, k, cpu(ag, 1, 2, 4, 8)), {}),
                     ((q, cpu(ag, 1, 2, 4, 8), cpu(ag, 1, 2, 4, 8)), {}), ((cpu(ag, 4, 3, 8), k, k), {}),
                     ((q, k, k), {"window": 0}), ((q, k, k), {"window": -3}), ((q, k, k), {"sinks": -1}),
                     ((cpu(ag, 1, 2, 3, 129), cpu(ag, 1, 2, 3, 129), cpu(ag, 1, 2, 3, 129)), {}),
                     ((ag.from_numpy(np.zeros((1, 4, 3, 8), np.int64)), k, k), {})):
        with pytest.raises(ValueError):
            ag.window_attention(*args, **{"window": 2, **kw})
    with pytest.raises(RuntimeError):
        ag.window_attention(q, k, k, 2)  # no compute on the host
    for args in ((cpu(ag, 3, 32), 3, 3, 2), (cpu(ag, 3, 32), 0, 1, 2), (cpu(ag, 3, 30), 3, 2, 2), (cpu(ag, 32), 2, 1, 2),
                 (cpu(ag, 3, 32), 2, 1, 0), (cpu(ag, 3, 32), 2, 1, 2, -1)):
        with pytest.raises(ValueError):
            ag._core._window_attention_qkv(*args)


def test_kv_cache_refusals(ag):
    good = dict(layers=1, sequences=2, kv_heads=2, d_head=64, max_tokens=100)
    for bad in ({"layers": 0}, {"sequences": 0}, {"kv_heads": 0}, {"d_head": 0}, {"d_head": 129}, {"max_tokens": 0},
                {"max_tokens": 1 << 30}, {"page": 16}, {"page": 96}, {"pages": -1}, {"window": -1}, {"sinks": -1},
                {"kv_heads": 1 << 17}, {"sequences": 1 << 23}, {"sequences": 1 << 21, "kv_heads": 4}):
        with pytest.raises(ValueError):
            ag.KVCache(**{**good, **bad})


def test_multi_head_attention_window_refusals(ag):
    for bad in ({"window": 4}, {"window": 0, "causal": True}, {"window": 4, "sinks": -1, "causal": True},
                {"sinks": 2, "causal": True}):
        with pytest.raises(ValueError):
            ag.nn.MultiHeadAttention(32, 4, **bad)
