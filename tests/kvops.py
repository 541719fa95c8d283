"""Helpers of the tests of window attention and of the paged 8-bit key/value cache:
their C ABI on torch tensors, and definitions in 64 bits."""
from __future__ import annotations

import ctypes
import math

import torch

import lmops as M

VP, I64, SZ, I32, F32 = M.VP, M.I64, M.SZ, M.I32, M.F32

SIGNATURES = {
    "aar_window_attn_fwd_workspace_bytes": (SZ, [I64] * 7),
    "aar_window_attn_fwd_f32": (I32, [VP] * 5 + [I64] * 5 + [VP, I64, I64, F32, VP, SZ, VP]),
    "aar_window_attn_bwd_workspace_bytes": (SZ, [I64] * 7),
    "aar_window_attn_bwd_f32": (I32, [VP] * 9 + [I64] * 5 + [VP, I64, I64, F32, VP, SZ, VP]),
    "aar_kv_cache_page_bytes": (SZ, [I64] * 3),
    "aar_kv_cache_append_f32": (I32, [VP] * 6 + [I64, VP, VP]),
    "aar_kv_cache_read_f32": (I32, [VP] * 6 + [I64, VP, VP]),
    "aar_kv_cache_attn_workspace_bytes": (SZ, [VP] + [I64] * 4),
    "aar_kv_cache_attn_f32": (I32, [VP] * 6 + [I64] * 4 + [F32, VP, SZ, VP, VP]),
}


class Cache(ctypes.Structure):
    """aar_kv_cache."""

    _fields_ = [(n, VP) for n in ("pages", "scales", "open", "table")] + [
        (n, I64) for n in ("sequences", "table_width", "n_pages", "kv_heads", "page", "d")]


def lib():
    L = M.lib()
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(L, name)
        fn.restype, fn.argtypes = res, args
    return L


# ------------------------------------------------------------------ window attention

def window_fwd(L, q, k, v, o, lse, window, sinks, scale=None):
    B, H, T, d = q.shape
    dims = (B, H, k.shape[1], T, d)
    nb = L.aar_window_attn_fwd_workspace_bytes(*dims, window, sinks)
    ws = M.scratch(nb)
    M.ok(L.aar_window_attn_fwd_f32(M.ptr(q), M.ptr(k), M.ptr(v), M.ptr(o), M.ptr(lse), *dims, M.strides3(q, k, v, o),
                                   window, sinks, d ** -0.5 if scale is None else scale, ws.data_ptr(), nb, M.stream()))


def window_bwd(L, q, k, v, o, lse, do, dq, dk, dv, window, sinks, scale=None, ws=None):
    B, H, T, d = q.shape
    dims = (B, H, k.shape[1], T, d)
    nb = L.aar_window_attn_bwd_workspace_bytes(*dims, window, sinks)
    ws = M.scratch(nb) if ws is None else ws
    M.ok(L.aar_window_attn_bwd_f32(M.ptr(q), M.ptr(k), M.ptr(v), M.ptr(o), M.ptr(lse), M.ptr(do), M.ptr(dq), M.ptr(dk),
                                   M.ptr(dv), *dims, M.strides3(q, k, v, o, do, dq, dk, dv), window, sinks,
                                   d ** -0.5 if scale is None else scale, ws.data_ptr(), nb, M.stream()))


def window_run(L, q, k, v, do, window, sinks, scale=None):
    B, H, T, d = q.shape
    o, lse = torch.full((B, H, T, d), 7.0, device="cuda"), torch.full((B, H, T), 7.0, device="cuda")
    window_fwd(L, q, k, v, o, lse, window, sinks, scale)
    if do is None:
        return o, lse
    dq, dk, dv = (torch.full(tuple(t.shape), 7.0, device="cuda") for t in (q, k, v))
    window_bwd(L, q, k, v, o, lse, do, dq, dk, dv, window, sinks, scale)
    return o, lse, dq, dk, dv


def window_mask(T, window, sinks):
    i, j = torch.arange(T)[:, None], torch.arange(T)
    return (j <= i) & ((i - j < window) | (j < sinks))


def window_exact(q, k, v, do, window, sinks, scale=None):
    """O, lse (dq, dk, dv) in 64 bits, and the magnitudes whose roundings reach lse, dq
    and dk (as lmops.cross_mass has them); torch's differentiation, on the GPU."""
    q, k, v = (t.detach().double().requires_grad_() for t in (q, k, v))
    T, d = q.shape[2:]
    G = q.shape[1] // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    sees = window_mask(T, window, sinks).to(q.device)
    kk, vv = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = (torch.matmul(q, kk.transpose(2, 3).contiguous()) * scale).masked_fill(~sees, -math.inf)
    p = torch.softmax(s, -1)
    o, lse = torch.matmul(p, vv), torch.logsumexp(s, -1).detach()
    if do is None:
        return (o.detach(), lse), {}
    o.backward(do.double())
    p, s = p.detach(), s.detach().masked_fill(~sees, 0.0)
    spread = (do.double().norm(dim=-1, keepdim=True) * vv.detach().norm(dim=-1).unsqueeze(-2)).masked_fill(~sees, 0.0)
    ds = abs(scale) * p * (spread + (p * spread).sum(-1, keepdim=True))
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q.detach().abs())
    mass = {"lse": s.abs().amax(-1) + math.log(T) + 1, "dq": torch.matmul(ds, kk.detach().abs()),
            "dk": dk.view(k.shape[0], k.shape[1], G, T, d).sum(2)}
    return (o.detach(), lse, q.grad, k.grad, v.grad), mass


# ------------------------------------------------------------------ the cache

# byte p of a group's column holds token ORDER[p] of the group's 32
ORDER = [4 * int(f"{g:03b}"[::-1], 2) + i for g in range(8) for i in range(4)]


def up(n, m):
    return (n + m - 1) // m * m


class Pool:
    """A cache on the GPU with its own table; pages are handed out in a shuffled order,
    and what stands in pages, scales and open rows at first is garbage."""

    def __init__(self, B, Hkv, d, page, width, spare=3, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.B, self.Hkv, self.d, self.P, self.width = B, Hkv, d, page, width
        self.n = B * width + spare
        self.dp = up(d, 16)
        self.bytes = torch.randint(0, 256, (self.n, Hkv, 2, page * self.dp), dtype=torch.uint8, generator=g).cuda()
        self.scales = torch.full((self.n, Hkv, 2), math.nan).cuda()
        self.open = torch.full((B, Hkv, 2, page, d), math.nan).cuda()
        self.table = torch.randperm(self.n, generator=g)[: B * width].view(B, width).cuda()
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")

    def struct(self):
        return Cache(M.ptr(self.bytes), M.ptr(self.scales), M.ptr(self.open), M.ptr(self.table), self.B, self.width,
                     self.n, self.Hkv, self.P, self.d)

    def append(self, L, k, v, lens, new_lens=None):
        """k, v [B, Hkv, T, d]."""
        c = self.struct()
        M.ok(L.aar_kv_cache_append_f32(ctypes.byref(c), M.ptr(k), M.ptr(v), M.strides3(k, v), M.ptr(lens),
                                       M.ptr(new_lens), k.shape[2], self.err.data_ptr(), M.stream()))

    def read(self, L, lens, T, first=None):
        c = self.struct()
        out = torch.full((2, self.B, self.Hkv, T, self.d), 7.0, device="cuda")
        M.ok(L.aar_kv_cache_read_f32(ctypes.byref(c), M.ptr(first), M.ptr(lens), M.ptr(out[0]), M.ptr(out[1]),
                                     M.strides3(out[0], out[1]), T, self.err.data_ptr(), M.stream()))
        return out

    def attend(self, L, q, lens, new_lens=None, window=1 << 62, sinks=0, scale=None, out=None, ws=None):
        B, H, T, d = q.shape
        c = self.struct()
        o = torch.full((B, H, T, d), 7.0, device="cuda") if out is None else out
        nb = L.aar_kv_cache_attn_workspace_bytes(ctypes.byref(c), H, T, window, sinks)
        ws = M.scratch(nb) if ws is None else ws
        M.ok(L.aar_kv_cache_attn_f32(ctypes.byref(c), M.ptr(q), M.ptr(o), M.strides3(q, o), M.ptr(lens),
                                     M.ptr(new_lens), H, T, window, sinks, d ** -0.5 if scale is None else scale,
                                     ws.data_ptr(), nb, self.err.data_ptr(), M.stream()))
        return o

    def values(self):
        """What the pages stand for, by the documented layout: [n, Hkv, 2, P, d], 64 bits."""
        x = self.bytes.cpu().double() - 128.0
        k = x[:, :, 0].view(self.n, self.Hkv, self.P, self.dp)
        v = x[:, :, 1].view(self.n, self.Hkv, self.P // 32, self.dp, 32)
        rows = torch.empty(self.n, self.Hkv, self.P // 32, 32, self.dp, dtype=torch.float64)
        rows[:, :, :, ORDER] = v.transpose(3, 4)
        both = torch.stack([k, rows.view(self.n, self.Hkv, self.P, self.dp)], 2)
        return both[..., : self.d] * self.scales.cpu().double()[..., None, None]


def quantised(rows, page):
    """What a cache holds of rows [n, d] (fp32), in 64 bits: page by page, the scale
    rounded to fp32, numbers to nearest with ties to even."""
    out = torch.empty(rows.shape, dtype=torch.float64)
    for a in range(0, rows.shape[0], page):
        x = rows[a : a + page].double()
        scale = (x.abs().max() / 127.0).float().double()
        out[a : a + page] = (x / scale).round().clamp(-127, 127) * scale if scale > 0 else 0.0 * x
    return out


def cache_exact(q, k, v, lens, new, window, sinks, scale=None):
    """q [B, H, T, d]; k, v lists of [Hkv, len_b, d] in 64 bits; new[b] tokens of b."""
    B, H, T, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    o = torch.zeros(B, H, T, d, dtype=torch.float64)
    for b in range(B):
        n, m = int(lens[b]), int(new[b])
        if m == 0:
            continue
        G = H // k[b].shape[0]
        i, j = torch.arange(n - m, n)[:, None], torch.arange(n)
        sees = (j <= i) & ((i - j < window) | (j < sinks))
        x = q[b, :, :m].double().cpu()
        s = (x @ k[b].repeat_interleave(G, 0).transpose(1, 2).contiguous() * scale).masked_fill(~sees, -math.inf)
        o[b, :, :m] = torch.softmax(s, -1) @ v[b].repeat_interleave(G, 0)
    return o
