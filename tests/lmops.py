"""Helpers of the tests of the encoder-reading decoder's operators: their C ABI
on torch tensors, definitions in 64 bits on the CPU, and comparisons."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

from devutil import LIB

U = 2.0 ** -24  # half a step of fp32, relative
VP, I64, SZ, I32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_size_t, ctypes.c_int
F32, F64 = ctypes.c_float, ctypes.c_double
EINVAL, EWORKSPACE, EUNSUPPORTED = -1, -2, -3

SIGNATURES = {
    "aar_cross_attn_fwd_workspace_bytes": (SZ, [I64] * 6),
    "aar_cross_attn_fwd_f32": (I32, [VP] * 6 + [I64] * 6 + [VP, F32, VP, SZ, VP]),
    "aar_cross_attn_bwd_workspace_bytes": (SZ, [I64] * 6),
    "aar_cross_attn_bwd_f32": (I32, [VP] * 10 + [I64] * 6 + [VP, F32, VP, SZ, VP]),
    "aar_qk_norm_rope_fwd_f32": (I32, [VP, I64, VP, VP, VP, I64, VP, I64] + [I64] * 5 + [F64, F32, VP]),
    "aar_qk_norm_rope_bwd_workspace_bytes": (SZ, [I64] * 4),
    "aar_qk_norm_rope_bwd_f32": (I32, [VP, I64, VP, I64, VP, VP, VP, I64, VP, I64, VP, VP] + [I64] * 5 +
                                 [F64, F32, VP, SZ, VP]),
    "aar_embedding_scaled_fwd_f32": (I32, [VP, VP, VP, I64, I64, I64, F32, VP, VP]),
    "aar_embedding_sorted_bwd_workspace_bytes": (SZ, [I64] * 3),
    "aar_embedding_sorted_bwd_f32": (I32, [VP, VP, VP, I64, I64, I64, F32, VP, SZ, VP]),
    "aar_distill_workspace_bytes": (SZ, [I64]),
    "aar_distill_fwd_f32": (I32, [VP] * 5 + [I64] * 3 + [F32, VP, VP, SZ, VP]),
    "aar_distill_bwd_f32": (I32, [VP] * 6 + [I64] * 3 + [F32, VP]),
}


def lib():
    L = ctypes.CDLL(str(LIB))
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(L, name)
        fn.restype, fn.argtypes = res, args
    return L


def ok(rc):
    assert rc == 0, rc


def ptr(t):
    return None if t is None or t.numel() == 0 else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def scratch(nbytes):
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device="cuda")


def strides3(*tensors):
    """(sb, sh, st) of [B, H, T, d] tensors as the ABI takes them."""
    out = []
    for t in tensors:
        assert t.shape[-1] == 1 or t.stride(-1) == 1
        out += [t.stride(0), t.stride(1), t.stride(2)]
    return (I64 * len(out))(*out)


def cross_fwd(L, q, k, v, lens, o, lse, scale=None, ws=None):
    B, H, Tq, d = q.shape
    Hkv, Tk = k.shape[1], k.shape[2]
    dims = (B, H, Hkv, Tq, Tk, d)
    nb = L.aar_cross_attn_fwd_workspace_bytes(*dims)
    ws = scratch(nb) if ws is None else ws
    ok(L.aar_cross_attn_fwd_f32(ptr(q), ptr(k), ptr(v), ptr(lens), ptr(o), ptr(lse), *dims, strides3(q, k, v, o),
                                d ** -0.5 if scale is None else scale, ws.data_ptr(), nb, stream()))


def cross_bwd(L, q, k, v, lens, o, lse, do, dq, dk, dv, scale=None, ws=None):
    B, H, Tq, d = q.shape
    dims = (B, H, k.shape[1], Tq, k.shape[2], d)
    nb = L.aar_cross_attn_bwd_workspace_bytes(*dims)
    ws = scratch(nb) if ws is None else ws
    ok(L.aar_cross_attn_bwd_f32(ptr(q), ptr(k), ptr(v), ptr(lens), ptr(o), ptr(lse), ptr(do), ptr(dq), ptr(dk), ptr(dv),
                                *dims, strides3(q, k, v, o, do, dq, dk, dv), d ** -0.5 if scale is None else scale,
                                ws.data_ptr(), nb, stream()))


def cross_exact(q, k, v, lens=None, do=None, scale=None):
    """O, lse (and dq, dk, dv) in 64 bits by torch's differentiation (CPU)."""
    q, k, v = (t.detach().double().cpu().requires_grad_() for t in (q, k, v))
    B, H, Tq, d = q.shape
    G = H // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    kk, vv = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = (q @ kk.transpose(2, 3)) * scale
    if lens is not None:
        seen = torch.arange(k.shape[2]) < lens.cpu().clamp(0, k.shape[2]).view(B, 1, 1, 1)
        s = s.masked_fill(~seen, -math.inf)
        vv = torch.where(seen.transpose(2, 3), vv, torch.zeros_like(vv))
    m = s.amax(-1, keepdim=True) if k.shape[2] else torch.full((B, H, Tq, 1), -math.inf, dtype=torch.float64)
    e = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m).detach())
    total = e.sum(-1, keepdim=True)
    o = (e / torch.where(total == 0, torch.ones_like(total), total)) @ vv
    lse = (m + torch.log(total))[..., 0].detach()
    if do is None:
        return o.detach(), lse
    o.backward(do.double().cpu())
    zero = lambda t: t.grad if t.grad is not None else torch.zeros_like(t)  # noqa: E731
    return o.detach(), lse, zero(q), zero(k), zero(v)


def attn_tol(d, n, smax=6.0):
    """What the roundings of an fp32 attention add up to, relative to its output:
    a score is a sum of d products, off by about sqrt(d) half steps of smax; the
    row's sums have n terms; four standard deviations of the two.  Where operands
    stand in two fp16 parts, each off by 2^-22 = 4 U at most, and the product of the
    second parts is left out, a product is off by 12 U at most and a score of d of them
    by some 4 U of a score: less than a quarter of its own sums' share."""
    return 4 * U * (math.sqrt(d) * smax + math.sqrt(n) + 8)


def cross_mass(q, k, v, lens, do, scale=None):
    """The magnitudes whose roundings reach lse, dq and dk: where their terms cancel
    (lse = m + ln l, dS = P (dP - D) with dP = D for a single key) the results are
    smaller than these, their errors are not.  dP and D are sums of d products of
    |dO| and |v|, off by half steps of that; so dq is off by half steps of
    scale P (|dP| + |D|) |K|, and dk likewise."""
    G = q.shape[1] // k.shape[1]
    q, k, v, do = (t.detach().double().cpu() for t in (q, k, v, do))
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    kk, vv = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    seen = torch.ones(q.shape[0], 1, 1, k.shape[2], dtype=torch.bool)
    if lens is not None:
        seen = torch.arange(k.shape[2]) < lens.cpu().clamp(0, k.shape[2]).view(-1, 1, 1, 1)
    s = (q @ kk.transpose(2, 3)) * scale
    p = torch.softmax(s.masked_fill(~seen, -1e300), -1) * seen
    spread = (do.abs().norm(dim=-1, keepdim=True) * vv.norm(dim=-1).unsqueeze(-2)).masked_fill(~seen, 0.0)
    ds = abs(scale) * p * (spread + (p * spread).sum(-1, keepdim=True))
    dq = ds @ torch.where(seen.transpose(2, 3), kk, torch.zeros_like(kk)).abs()
    dk = (ds.transpose(2, 3) @ q.abs()).view(k.shape[0], k.shape[1], G, k.shape[2], -1).sum(2)
    lse = s.masked_fill(~seen, -math.inf).abs().masked_fill(~seen, 0.0).amax(-1) + math.log(k.shape[2]) + 1
    return {"lse": lse, "dq": dq, "dk": dk}


def near(got, ref, tol, what="", mass=None):
    """max|g - r| <= 4 tol max|mass| and ||g - r|| <= tol ||mass||, non-finite values
    alike; mass: the magnitudes whose roundings count, the results' own if None."""
    g = got.detach().double().cpu() if torch.is_tensor(got) else torch.from_numpy(np.asarray(got, np.float64))
    r = ref.detach().double().cpu() if torch.is_tensor(ref) else torch.from_numpy(np.asarray(ref, np.float64))
    assert g.shape == r.shape, (what, g.shape, r.shape)
    fine = torch.isfinite(r)
    assert torch.equal(torch.isfinite(g), fine), f"{what}: non-finite values differ"
    assert torch.equal(g[~fine].nan_to_num(nan=7.0), r[~fine].nan_to_num(nan=7.0)), what
    g, r, w = g[fine], r[fine], (r if mass is None else mass)[fine]
    if not r.numel():
        return
    err, top = (g - r).abs().max().item(), w.abs().max().item()
    rel, norm = (g - r).norm().item(), w.norm().item()
    # the largest element's error counts against four times the tolerance: it is a maximum over all of them
    assert err <= 4 * tol * top and rel <= tol * norm, f"{what}: max {err / max(top, 1e-300):.3g} rel {rel / max(norm, 1e-300):.3g} tol {tol:.3g}"
