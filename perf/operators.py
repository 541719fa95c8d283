"""Operators of a decoder that reads an encoder's states and learns from a
larger teacher: cross attention, per-head norms of queries and keys with the
position rotation, the scaled embedding with its gradient by sorted tokens, and
distillation from a teacher's top logits.

Where `own` is false a pass computes the operator in elementary torch
operations; where it is true it calls the C ABI (include/aar_hip.h,
libaar_hip.so), the entry points a C++ core binds, on tensors that torch holds
on the GPU.  Training cases run forward and backward.
"""
from __future__ import annotations

import ctypes
import functools
import math
from pathlib import Path

import torch

own = False

DEV = "cuda"
LIB = Path(__file__).resolve().parent.parent / "aar-vlm_amd" / "aargrad" / "libaar_hip.so"


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # one new token for each of 32 sequences against a cached, padded encoder (serving: bytes of K and V)
        {"name": "cross_token", "kind": "cross", "B": 32, "H": 6, "Hkv": 6, "T": 1, "S": 2048, "d": 64, "ragged": True,
         "train": False},
        # the training step's cross attention over 24 x 24 patches and a class token, padded
        {"name": "cross_train", "kind": "cross", "B": 64, "H": 6, "Hkv": 6, "T": 256, "S": 577, "d": 64, "ragged": True,
         "train": True},
        # a prompt's pass over an encoder with shared key/value heads of the largest head size, odd lengths
        {"name": "cross_prompt", "kind": "cross", "B": 4, "H": 16, "Hkv": 4, "T": 301, "S": 1111, "d": 128,
         "ragged": False, "train": False},
        # long text against a long encoder, forward and backward (the largest case)
        {"name": "cross_long", "kind": "cross", "B": 8, "H": 12, "Hkv": 12, "T": 1024, "S": 4096, "d": 64,
         "ragged": False, "train": True},
        # queries and keys of one new token for each of 32 sequences, at positions of their own (the smallest case)
        {"name": "rotate_token", "kind": "rotate", "rows": 32, "T": 0, "Hq": 6, "Hk": 6, "d": 64, "train": False},
        # the packed projection of a training batch of 64 x 256 tokens, forward and backward
        {"name": "rotate_train", "kind": "rotate", "rows": 16384, "T": 256, "Hq": 6, "Hk": 6, "d": 64, "train": True},
        # a wide model's projection, fewer key heads, larger than the caches, forward and backward
        {"name": "rotate_wide", "kind": "rotate", "rows": 32768, "T": 4096, "Hq": 32, "Hk": 8, "d": 128, "train": True},
        # a character vocabulary: every row of the table takes hundreds of tokens
        {"name": "embed_chars", "kind": "embed", "n": 16384, "vocab": 65, "dim": 384},
        # a subword vocabulary: most rows take none, a few take thousands
        {"name": "embed_words", "kind": "embed", "n": 32768, "vocab": 50000, "dim": 768},
        # the character model's loss against a teacher's eight best
        {"name": "distill_chars", "kind": "distill", "n": 16384, "vocab": 65, "top": 8, "tau": 2.0},
        # a subword vocabulary, larger than the caches
        {"name": "distill_words", "kind": "distill", "n": 4096, "vocab": 50000, "top": 64, "tau": 1.0},
        # rows that are no multiple of a vector, an odd number of teacher entries
        {"name": "distill_odd", "kind": "distill", "n": 1001, "vocab": 32003, "top": 37, "tau": 1.5},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _extent(rng, lo, hi):
    """A size spread over the logarithm: a third a multiple of 64, else any."""
    n = _log_int(rng, lo, hi)
    return max(lo, n // 64 * 64) if rng.random() < 0.34 and n >= 64 else n


def draw(rng):
    kind = rng.choice(["cross", "cross", "cross", "rotate", "rotate", "embed", "embed", "distill", "distill"])
    while True:
        if kind == "cross":
            kv = rng.choice([1, 2, 4, 6, 8, 12])
            c = {"kind": kind, "B": _log_int(rng, 1, 64), "H": kv * rng.choice([1, 1, 1, 2, 4]), "Hkv": kv,
                 "T": 1 if rng.random() < 0.25 else _extent(rng, 2, 2048), "S": _extent(rng, 1, 8192),
                 "d": rng.choice([64, 64, 64, 128, 32, 96, 40, 30]), "ragged": rng.random() < 0.5,
                 "train": rng.random() < 0.6}
        elif kind == "rotate":
            heads = rng.choice([1, 2, 4, 6, 8, 12])
            c = {"kind": kind, "rows": _log_int(rng, 1, 256), "T": 0, "Hq": heads * rng.choice([1, 1, 4]), "Hk": heads,
                 "d": rng.choice([64, 64, 128, 32, 96, 40, 30]), "train": rng.random() < 0.6}
            if rng.random() < 0.75:
                c["T"] = _extent(rng, 2, 4096)
                c["rows"] = c["T"] * _log_int(rng, 1, 64)
        elif kind == "embed":
            c = {"kind": kind, "n": _extent(rng, 1, 131072), "vocab": _log_int(rng, 40, 200000),
                 "dim": _extent(rng, 32, 4096)}
        else:
            vocab = _log_int(rng, 40, 200000)
            c = {"kind": kind, "n": _extent(rng, 1, 32768), "vocab": vocab,
                 "top": min(vocab, _log_int(rng, 1, 128)), "tau": rng.choice([1.0, 1.5, 2.0, 4.0])}
        w = work(c)
        if w["flops"] <= 3.6e11 and w["bytes"] <= 2.0e9:
            return c


def work(case):
    """Bytes (each input read once, each output written once) and FLOPs of one pass."""
    c, k = case, case["kind"]
    if k == "cross":
        seen = 0.75 if c["ragged"] else 1.0  # of the keys, on average
        q, kv = c["B"] * c["T"] * c["H"] * c["d"], 2.0 * c["B"] * c["S"] * seen * c["Hkv"] * c["d"]
        pairs = float(c["B"] * c["H"] * c["T"]) * c["S"] * seen * c["d"]
        if not c["train"]:
            return {"bytes": 4.0 * (2 * q + kv), "flops": 4.0 * pairs}
        return {"bytes": 4.0 * (4 * q + 2 * kv), "flops": 14.0 * pairs}
    if k == "rotate":
        n = float(c["rows"]) * (c["Hq"] + c["Hk"]) * c["d"]
        return {"bytes": (16.0 if c["train"] else 8.0) * n, "flops": (20.0 if c["train"] else 7.0) * n}
    if k == "embed":
        n, d, v = float(c["n"]), c["dim"], float(c["vocab"])
        # the table's rows that a Zipf law's n tokens are expected to touch
        p = torch.log1p(1.0 / torch.arange(1, c["vocab"] + 1, dtype=torch.float64)) / math.log(v + 1.0)
        rows = float((1.0 - torch.exp(n * torch.log1p(-p.clamp(max=0.999999)))).sum())
        return {"bytes": 4.0 * d * (rows + 2 * n + v) + 8.0 * n, "flops": 2.0 * n * d}
    n, v, t = float(c["n"]), float(c["vocab"]), float(c["top"])
    return {"bytes": 8.0 * n * v + 12.0 * n * t, "flops": 8.0 * n * v}


# ------------------------------------------------------------------ inputs

def _rand(gen, *shape, scale=1.0):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).mul_(scale)


def _new(*shape):
    return torch.empty(shape, dtype=torch.float32, device=DEV)


def _inputs(c, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    k = c["kind"]
    if k == "cross":
        B, H, Hkv, T, S, d = (c[n] for n in ("B", "H", "Hkv", "T", "S", "d"))
        s = {"q": _rand(gen, B, T, H, d), "kv": _rand(gen, B, S, 2, Hkv, d), "lens": None}
        if c["ragged"]:
            s["lens"] = torch.randint((S + 1) // 2, S + 1, (B,), generator=gen, device=DEV, dtype=torch.int64)
        if c["train"]:
            s["do"] = _rand(gen, B, T, H, d, scale=0.1)
        return s
    if k == "rotate":
        heads = c["Hq"] + 2 * c["Hk"]  # the packed projection holds the values as well
        s = {"x": _rand(gen, c["rows"], heads * c["d"], scale=1.5),
             "wq": 1.0 + _rand(gen, c["d"], scale=0.1), "wk": 1.0 + _rand(gen, c["d"], scale=0.1)}
        if c["T"]:
            s["pos"] = torch.arange(c["T"], device=DEV, dtype=torch.int64)
        else:
            s["pos"] = torch.randint(0, 131072, (c["rows"],), generator=gen, device=DEV, dtype=torch.int64)
        if c["train"]:
            s["gy"] = _rand(gen, c["rows"], (c["Hq"] + c["Hk"]) * c["d"], scale=0.1)
        return s
    if k == "embed":
        n, v, d = c["n"], c["vocab"], c["dim"]
        # ids by a Zipf law (log-uniform ranks), the ranks spread over the table
        u = torch.rand(n, generator=gen, device=DEV, dtype=torch.float64)
        rank = torch.exp(u * math.log(v + 1.0)).long().sub_(1).clamp_(0, v - 1)
        place = torch.randperm(v, generator=gen, device=DEV)
        return {"w": _rand(gen, v, d, scale=d ** -0.5), "ids": place[rank].contiguous(),
                "g": _rand(gen, n, d, scale=1e-2)}
    n, v, t = c["n"], c["vocab"], c["top"]
    z = _rand(gen, n, v, scale=2.0)
    teacher = _rand(gen, n, v, scale=1.5).add_(z, alpha=0.6)
    best, ids = teacher.topk(t, dim=-1)
    # the entries a teacher's probability cut kept, and padded rows without any
    kept = torch.randint(1, t + 1, (n, 1), generator=gen, device=DEV)
    kept *= torch.rand(n, 1, generator=gen, device=DEV) > 0.03
    ids = torch.where(torch.arange(t, device=DEV) < kept, ids, torch.full_like(ids, -1))
    return {"z": z, "best": best.contiguous(), "ids": ids.contiguous(), "grad": torch.ones(1, device=DEV)}


def prepare(case, seed):
    """Inputs on the GPU, and the outputs a program allocates once."""
    c, k = dict(case), case["kind"]
    s = _inputs(c, seed)
    s["case"] = c
    if k == "cross":
        B, H, Hkv, T, S, d = (c[n] for n in ("B", "H", "Hkv", "T", "S", "d"))
        s.update(o=_new(B, T, H, d), lse=_new(B, H, T))
        if c["train"]:
            s.update(dq=_new(B, T, H, d), dkv=_new(B, S, 2, Hkv, d))
    elif k == "rotate":
        s["y"] = _new(c["rows"], (c["Hq"] + c["Hk"]) * c["d"])
        if c["train"]:
            s.update(dx=torch.empty_like(s["x"]), dwq=_new(c["d"]), dwk=_new(c["d"]))
    elif k == "embed":
        s.update(out=_new(c["n"], c["dim"]), dw=_new(c["vocab"], c["dim"]))
    else:
        s.update(loss=_new(1), stats=_new(2 * c["n"] + 1), dz=_new(c["n"], c["vocab"]))
    return s


ROPE_BASE, NORM_EPS = 10000.0, 1e-6


# ------------------------------------------------------------------ one pass

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"cross": _own_cross, "rotate": _own_rotate, "embed": _own_embed, "distill": _own_distill}[kind](state)
    return {"cross": _plain_cross, "rotate": _plain_rotate, "embed": _plain_embed, "distill": _plain_distill}[kind](state)


def _plain_cross(s):
    c = s["case"]
    B, H, Hkv, T, S, d = (c[n] for n in ("B", "H", "Hkv", "T", "S", "d"))
    G, scale = H // Hkv, 1.0 / math.sqrt(d)

    def heads(x):  # [B, T, H, d] -> [B, Hkv, G * T, d], the query heads of a shared one in a row
        return x.permute(0, 2, 1, 3).reshape(B, Hkv, G * T, d)

    def back(x):
        return x.reshape(B, H, T, d).permute(0, 2, 1, 3).contiguous()

    q = heads(s["q"])
    k, v = s["kv"].permute(2, 0, 3, 1, 4).contiguous().unbind(0)
    kt, vt = k.transpose(2, 3).contiguous(), v.transpose(2, 3).contiguous()
    score = torch.matmul(q, kt).mul_(scale)
    if s["lens"] is not None:
        score.masked_fill_(torch.arange(S, device=DEV) >= s["lens"].view(B, 1, 1, 1), -math.inf)
    m = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = torch.matmul(p, v)
    out = {"o": back(o), "lse": (m + torch.log(total)).reshape(B, H, T)}
    if c["train"]:
        do = heads(s["do"])
        ds = p * (torch.matmul(do, vt) - (do * o).sum(-1, keepdim=True)) * scale
        dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
        dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
        out["dq"] = back(torch.matmul(ds, k))
        out["dkv"] = torch.stack([dk, dv]).permute(1, 3, 0, 2, 4).contiguous()
    return out


def _plain_rotate(s):
    c = s["case"]
    rows, Hq, Hk, d = c["rows"], c["Hq"], c["Hk"], c["d"]
    H, h = Hq + Hk, d // 2
    x = s["x"][:, : H * d].reshape(rows, H, d)
    w = torch.cat([s["wq"].expand(Hq, d), s["wk"].expand(Hk, d)])
    # far positions: the angle in 64 bits
    freq = ROPE_BASE ** (torch.arange(h, device=DEV, dtype=torch.float64) * (-2.0 / d))
    angle = s["pos"].double()[:, None] * freq
    cos, sin = angle.cos().float(), angle.sin().float()
    n = s["pos"].numel()
    cos, sin = (t.view(1, n, 1, h).expand(rows // n, n, 1, h).reshape(rows, 1, h) for t in (cos, sin))
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + NORM_EPS)
    xh = x * rstd
    u = xh * w
    a, b = u[..., :h], u[..., h:]
    out = {"y": torch.cat([a * cos - b * sin, b * cos + a * sin], -1).reshape(rows, H * d)}
    if c["train"]:
        gy = s["gy"].reshape(rows, H, d)
        ga, gb = gy[..., :h], gy[..., h:]
        g = torch.cat([ga * cos + gb * sin, gb * cos - ga * sin], -1)
        gw = g * w
        dw = (g * xh).sum(0)
        out["dx"] = (rstd * (gw - xh * (gw * xh).mean(-1, keepdim=True))).reshape(rows, H * d)
        out["dwq"], out["dwk"] = dw[:Hq].sum(0), dw[Hq:].sum(0)
    return out


def _plain_embed(s):
    c = s["case"]
    scale = math.sqrt(c["dim"])
    dw = torch.zeros(c["vocab"], c["dim"], device=DEV).index_add_(0, s["ids"], s["g"])
    return {"out": s["w"][s["ids"]] * scale, "dw": dw.mul_(scale)}


def _plain_distill(s):
    c = s["case"]
    tau, ids = c["tau"], s["ids"]
    there = ids >= 0
    at = ids.clamp(min=0)
    active = there.any(-1)
    t = torch.where(there, s["best"] / tau, torch.full_like(s["best"], -math.inf))
    m = t.amax(-1, keepdim=True)
    e = torch.exp(t - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    logp = torch.where(p > 0, torch.log(p), torch.zeros_like(p))
    z = s["z"] / tau
    mz = z.amax(-1, keepdim=True)
    ez = torch.exp(z - mz)
    sz = ez.sum(-1, keepdim=True)
    logq = z.gather(1, at) - mz - torch.log(sz)
    row = torch.where(p > 0, p * (logp - logq), torch.zeros_like(p)).sum(-1)
    count = active.sum()
    loss = (tau * tau) * row.sum() / count.clamp(min=1)
    q = ez.div_(sz).mul_(active[:, None])
    dz = q.scatter_add_(1, at, -p).mul_(s["grad"] * tau / count.clamp(min=1))
    return {"loss": loss.reshape(1), "dz": dz}


# ------------------------------------------------------------------ the framework's calls

@functools.lru_cache(maxsize=1)
def _lib():
    lib = ctypes.CDLL(str(LIB))
    vp, i64, sz, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_size_t, ctypes.c_int
    f32, f64 = ctypes.c_float, ctypes.c_double

    def sign(name, res, args):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args

    sign("aar_cross_attn_fwd_workspace_bytes", sz, [i64] * 6)
    sign("aar_cross_attn_fwd_f32", i32, [vp] * 6 + [i64] * 6 + [vp, f32, vp, sz, vp])
    sign("aar_cross_attn_bwd_workspace_bytes", sz, [i64] * 6)
    sign("aar_cross_attn_bwd_f32", i32, [vp] * 10 + [i64] * 6 + [vp, f32, vp, sz, vp])
    sign("aar_qk_norm_rope_fwd_f32", i32, [vp, i64, vp, vp, vp, i64, vp, i64] + [i64] * 5 + [f64, f32, vp])
    sign("aar_qk_norm_rope_bwd_workspace_bytes", sz, [i64] * 4)
    sign("aar_qk_norm_rope_bwd_f32", i32, [vp, i64, vp, i64, vp, vp, vp, i64, vp, i64, vp, vp] + [i64] * 5 +
         [f64, f32, vp, sz, vp])
    sign("aar_embedding_scaled_fwd_f32", i32, [vp, vp, vp, i64, i64, i64, f32, vp, vp])
    sign("aar_embedding_sorted_bwd_workspace_bytes", sz, [i64] * 3)
    sign("aar_embedding_sorted_bwd_f32", i32, [vp, vp, vp, i64, i64, i64, f32, vp, sz, vp])
    sign("aar_distill_workspace_bytes", sz, [i64])
    sign("aar_distill_fwd_f32", i32, [vp] * 5 + [i64] * 3 + [f32, vp, vp, sz, vp])
    sign("aar_distill_bwd_f32", i32, [vp] * 6 + [i64] * 3 + [f32, vp])
    return lib


def _ok(rc):
    if rc != 0:
        raise RuntimeError("aar status %d" % rc)


def _plan(s, make):
    """What a program keeps beside its tensors: sizes asked once, strides, scratch."""
    if "plan" not in s:
        s["plan"] = make()
    return s["plan"]


def _scratch(nbytes):
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=DEV)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_cross(s):
    c, L = s["case"], _lib()
    B, H, Hkv, T, S, d = (c[n] for n in ("B", "H", "Hkv", "T", "S", "d"))

    def make():
        dims = (B, H, Hkv, T, S, d)
        fb, bb = L.aar_cross_attn_fwd_workspace_bytes(*dims), 0
        if c["train"]:
            bb = L.aar_cross_attn_bwd_workspace_bytes(*dims)
        q, kv = [T * H * d, d, H * d], [S * 2 * Hkv * d, d, 2 * Hkv * d]
        fwd = (ctypes.c_int64 * 12)(*(q + kv + kv + q))
        bwd = (ctypes.c_int64 * 24)(*(q + kv + kv + q + q + q + kv + kv))
        return _scratch(max(fb, bb)), fb, bb, fwd, bwd

    ws, fb, bb, fwd, bwd = _plan(s, make)
    kv, lens, st = s["kv"].data_ptr(), s["lens"].data_ptr() if s["lens"] is not None else None, _stream()
    q, o, lse, half, scale = s["q"].data_ptr(), s["o"].data_ptr(), s["lse"].data_ptr(), 4 * Hkv * d, 1.0 / math.sqrt(d)
    _ok(L.aar_cross_attn_fwd_f32(q, kv, kv + half, lens, o, lse, B, H, Hkv, T, S, d, fwd, scale, ws.data_ptr(), fb, st))
    out = {"o": s["o"], "lse": s["lse"]}
    if c["train"]:
        dkv = s["dkv"].data_ptr()
        _ok(L.aar_cross_attn_bwd_f32(q, kv, kv + half, lens, o, lse, s["do"].data_ptr(), s["dq"].data_ptr(), dkv,
                                     dkv + half, B, H, Hkv, T, S, d, bwd, scale, ws.data_ptr(), bb, st))
        out.update(dq=s["dq"], dkv=s["dkv"])
    return out


def _own_rotate(s):
    c, L = s["case"], _lib()
    rows, Hq, Hk, d = c["rows"], c["Hq"], c["Hk"], c["d"]
    wide, narrow, st = (Hq + 2 * Hk) * d, (Hq + Hk) * d, _stream()
    x, wq, wk, pos, count = s["x"].data_ptr(), s["wq"].data_ptr(), s["wk"].data_ptr(), s["pos"].data_ptr(), s["pos"].numel()
    _ok(L.aar_qk_norm_rope_fwd_f32(x, wide, wq, wk, pos, count, s["y"].data_ptr(), narrow, rows, Hq, Hk, d, d, ROPE_BASE,
                                   NORM_EPS, st))
    if not c["train"]:
        return {"y": s["y"]}
    ws = _plan(s, lambda: _scratch(L.aar_qk_norm_rope_bwd_workspace_bytes(rows, Hq, Hk, d)))
    _ok(L.aar_qk_norm_rope_bwd_f32(s["gy"].data_ptr(), narrow, x, wide, wq, wk, pos, count, s["dx"].data_ptr(), wide,
                                   s["dwq"].data_ptr(), s["dwk"].data_ptr(), rows, Hq, Hk, d, d, ROPE_BASE, NORM_EPS,
                                   ws.data_ptr(), ws.numel(), st))
    return {"y": s["y"], "dx": s["dx"][:, :narrow], "dwq": s["dwq"], "dwk": s["dwk"]}


def _own_embed(s):
    c, L = s["case"], _lib()
    n, v, d, st = c["n"], c["vocab"], c["dim"], _stream()
    scale = math.sqrt(d)
    ws = _plan(s, lambda: _scratch(L.aar_embedding_sorted_bwd_workspace_bytes(n, v, d)))
    _ok(L.aar_embedding_scaled_fwd_f32(s["w"].data_ptr(), s["ids"].data_ptr(), s["out"].data_ptr(), n, v, d, scale, None,
                                       st))
    _ok(L.aar_embedding_sorted_bwd_f32(s["g"].data_ptr(), s["ids"].data_ptr(), s["dw"].data_ptr(), n, v, d, scale,
                                       ws.data_ptr(), ws.numel(), st))
    return {"out": s["out"], "dw": s["dw"]}


def _own_distill(s):
    c, L = s["case"], _lib()
    n, v, t, tau, st = c["n"], c["vocab"], c["top"], c["tau"], _stream()
    ws = _plan(s, lambda: _scratch(L.aar_distill_workspace_bytes(n)))
    z, best, ids, stats = s["z"].data_ptr(), s["best"].data_ptr(), s["ids"].data_ptr(), s["stats"].data_ptr()
    _ok(L.aar_distill_fwd_f32(z, best, ids, s["loss"].data_ptr(), stats, n, v, t, tau, None, ws.data_ptr(), ws.numel(),
                              st))
    _ok(L.aar_distill_bwd_f32(s["grad"].data_ptr(), z, best, ids, stats, s["dz"].data_ptr(), n, v, t, tau, st))
    return {"loss": s["loss"], "dz": s["dz"]}


# ------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    """The definitions in 64 bits, gradients by torch's own differentiation."""
    c, k = case, case["kind"]
    s = {n: t.double().requires_grad_() if t is not None and t.is_floating_point() else t
         for n, t in _inputs(c, seed).items()}
    if k == "cross":
        B, H, Hkv, T, S, d = (c[n] for n in ("B", "H", "Hkv", "T", "S", "d"))
        o = torch.empty(B, T, H, d, dtype=torch.float64, device=DEV)
        lse = torch.empty(B, H, T, dtype=torch.float64, device=DEV)
        dq, dkv = torch.zeros_like(o), torch.zeros(B, S, 2, Hkv, d, dtype=torch.float64, device=DEV)
        for b in range(B):
            seen = int(s["lens"][b]) if c["ragged"] else S
            for h in range(H):
                hk = h * Hkv // H
                q = s["q"].detach()[b, :, h].clone().requires_grad_()
                kv = s["kv"].detach()[b, :seen, :, hk].clone().requires_grad_()
                score = (q @ kv[:, 0].t()) / math.sqrt(d)
                got = torch.softmax(score, -1) @ kv[:, 1]
                o[b, :, h], lse[b, h] = got.detach(), torch.logsumexp(score.detach(), -1)
                if c["train"]:
                    got.backward(s["do"].detach()[b, :, h])
                    dq[b, :, h] = q.grad
                    dkv[b, :seen, :, hk] += kv.grad
        return {"o": o, "lse": lse, "dq": dq, "dkv": dkv} if c["train"] else {"o": o, "lse": lse}
    if k == "rotate":
        rows, Hq, Hk, d = c["rows"], c["Hq"], c["Hk"], c["d"]
        x = s["x"][:, : (Hq + Hk) * d].reshape(rows, Hq + Hk, d)
        w = torch.cat([s["wq"][None].repeat(Hq, 1), s["wk"][None].repeat(Hk, 1)])
        u = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + NORM_EPS) * w
        pos = s["pos"].repeat(rows // s["pos"].numel()).double()
        turn = pos[:, None] / ROPE_BASE ** (2.0 * torch.arange(d // 2, device=DEV, dtype=torch.float64) / d)
        y = torch.complex(u[..., : d // 2], u[..., d // 2:]) * torch.polar(torch.ones_like(turn), turn)[:, None]
        y = torch.cat([y.real, y.imag], -1).reshape(rows, -1)
        if not c["train"]:
            return {"y": y.detach()}
        y.backward(s["gy"].detach())
        return {"y": y.detach(), "dx": s["x"].grad[:, : (Hq + Hk) * d].contiguous(), "dwq": s["wq"].grad,
                "dwk": s["wk"].grad}
    if k == "embed":
        out = torch.nn.functional.embedding(s["ids"], s["w"]) * math.sqrt(c["dim"])
        out.backward(s["g"].detach())
        return {"out": out.detach(), "dw": s["w"].grad}
    ids, tau = s["ids"], c["tau"]
    there, rows = ids >= 0, (ids >= 0).any(-1)
    p = torch.softmax((s["best"].detach() / tau).masked_fill(~there, -math.inf)[rows], -1)
    logq = torch.log_softmax(s["z"] / tau, -1)[rows].gather(1, ids[rows].clamp(min=0))
    terms = torch.xlogy(p, p) - p * logq
    loss = tau * tau * terms.sum() / max(int(rows.sum()), 1)
    loss.backward()
    return {"loss": loss.detach().reshape(1), "dz": s["z"].grad}
