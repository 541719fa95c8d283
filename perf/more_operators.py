"""Operators of a decoder whose text is longer than what it attends to, and of its
serving: causal attention with a sliding window and a few first tokens that stay
visible (sinks), a key/value cache in pages of 8-bit numbers with a scale for each
page and head, and the attention of new tokens over that cache.

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
EVERY = 1 << 30  # a window that hides nothing


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # a short text of one sequence, forward and backward (the training call that latency counts in)
        {"name": "window_short", "kind": "window", "B": 1, "H": 6, "Hkv": 6, "T": 200, "W": 64, "S": 2, "d": 64,
         "train": True},
        # the training step's attention, 64 x 256 tokens, half of the text in the window
        {"name": "window_train", "kind": "window", "B": 64, "H": 6, "Hkv": 6, "T": 256, "W": 128, "S": 4, "d": 64,
         "train": True},
        # a prompt's pass with shared key/value heads of the largest head size, odd lengths
        {"name": "window_prompt", "kind": "window", "B": 4, "H": 16, "Hkv": 4, "T": 1777, "W": 500, "S": 1, "d": 128,
         "train": False},
        # long text of a grouped-head model, forward and backward (the largest case)
        {"name": "window_long", "kind": "window", "B": 2, "H": 12, "Hkv": 4, "T": 16384, "W": 1024, "S": 4, "d": 64,
         "train": True},
        # one new token for each of 32 sequences into the cache, and its page read back
        {"name": "append_token", "kind": "append", "B": 32, "Hkv": 6, "T": 1, "len": 2048, "page": 64, "d": 64},
        # prompts of up to 1000 tokens into an empty cache, and what it holds of them
        {"name": "append_prompt", "kind": "append", "B": 16, "Hkv": 8, "T": 1000, "len": 1000, "page": 32, "d": 128},
        # one new token of a single user's text (the smallest case)
        {"name": "cache_one", "kind": "cache", "B": 1, "H": 6, "Hkv": 6, "T": 1, "len": 1000, "W": EVERY, "S": 0,
         "page": 64, "d": 64},
        # one new token for each of 32 sequences
        {"name": "cache_token", "kind": "cache", "B": 32, "H": 12, "Hkv": 12, "T": 1, "len": 4096, "W": EVERY, "S": 0,
         "page": 64, "d": 64},
        # text without end: the window's pages and the sinks' are all that is kept
        {"name": "cache_stream", "kind": "cache", "B": 64, "H": 16, "Hkv": 4, "T": 1, "len": 20000, "W": 2000, "S": 4,
         "page": 32, "d": 128},
        # long contexts of a grouped-head model (bytes of the cache)
        {"name": "cache_long", "kind": "cache", "B": 16, "H": 32, "Hkv": 4, "T": 1, "len": 32768, "W": EVERY, "S": 0,
         "page": 128, "d": 128},
        # a chunk of each prompt behind what the cache holds already, odd lengths
        {"name": "cache_prompt", "kind": "cache", "B": 4, "H": 12, "Hkv": 12, "T": 250, "len": 4096, "W": EVERY, "S": 0,
         "page": 64, "d": 64},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _extent(rng, lo, hi):
    """A size spread over the logarithm: a third a multiple of 64, else any."""
    n = _log_int(rng, lo, hi)
    return max(lo, n // 64 * 64) if rng.random() < 0.34 and n >= 64 else n


def draw(rng):
    kind = rng.choice(["window", "window", "append", "cache", "cache"])
    while True:
        kv, d = rng.choice([1, 2, 4, 6, 8, 12]), rng.choice([64, 64, 64, 128, 128, 32, 96, 40, 30])
        H = kv * rng.choice([1, 1, 2, 4, 8])
        window, sinks = _extent(rng, 16, 4096), rng.choice([0, 1, 4, 4, _log_int(rng, 1, 100)])
        if kind == "window":
            c = {"kind": kind, "B": _log_int(rng, 1, 64), "H": H, "Hkv": kv, "T": _extent(rng, 1, 16384), "W": window,
                 "S": sinks, "d": d, "train": rng.random() < 0.6}
        elif kind == "append":
            T = 1 if rng.random() < 0.4 else _extent(rng, 2, 4096)
            c = {"kind": kind, "B": _log_int(rng, 1, 64), "Hkv": kv, "T": T, "len": T + _log_int(rng, 1, 8192),
                 "page": rng.choice([32, 64, 128]), "d": d}
        else:
            T = 1 if rng.random() < 0.6 else _extent(rng, 2, 1024)
            if rng.random() < 0.6:
                window, sinks = EVERY, 0
            c = {"kind": kind, "B": _log_int(rng, 1, 64), "H": H, "Hkv": kv, "T": T,
                 "len": max(2 * T, _extent(rng, 1, 32768)), "W": window, "S": sinks, "page": rng.choice([32, 64, 128]),
                 "d": d}
        w = work(c)
        if w["flops"] <= 3.2e11 and w["bytes"] <= 4.0e8:
            return c


def _pairs(T, window, sinks):
    """Pairs of a query and a key that it sees, of T tokens from the first one on."""
    full = min(T, window + sinks)  # queries that see everything before them
    seen = full * (full + 1) / 2.0
    return seen + (T - full) * float(window + sinks)


def work(case):
    """Bytes (each input read once, each output written once) and FLOPs of one pass."""
    c, k = case, case["kind"]
    if k == "window":
        q, kv = float(c["B"]) * c["T"] * c["H"] * c["d"], 2.0 * c["B"] * c["T"] * c["Hkv"] * c["d"]
        pairs = c["B"] * c["H"] * c["d"] * _pairs(c["T"], c["W"], c["S"])
        if not c["train"]:
            return {"bytes": 4.0 * (2 * q + kv), "flops": 4.0 * pairs}
        return {"bytes": 4.0 * (4 * q + 2 * kv), "flops": 14.0 * pairs}
    if k == "append":
        heads = 2.0 * c["B"] * c["Hkv"] * c["d"]
        if c["T"] == 1:  # the page's rows so far, kept and read back; its bytes
            return {"bytes": heads * c["page"] * (4 * 0.5 + 1 + 4), "flops": 4.0 * heads * c["page"]}
        rows = 0.75 * c["T"]
        return {"bytes": heads * (rows * (4 + 1 + 1) + 4.0 * c["T"]), "flops": 4.0 * heads * rows}
    held = 0.75 * c["len"]  # tokens of a sequence, on average
    seen = min(held, c["W"] + c["S"] + c["T"] - 1.0)
    pairs = float(c["T"]) * min(held - (c["T"] - 1) / 2.0, c["W"] + c["S"])
    return {"bytes": 2.0 * c["B"] * c["Hkv"] * c["d"] * seen + 8.0 * c["B"] * c["H"] * c["T"] * c["d"],
            "flops": 4.0 * c["B"] * c["H"] * c["d"] * pairs}


# ------------------------------------------------------------------ inputs

def _rand(gen, *shape, scale=1.0):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).mul_(scale)


def _new(*shape):
    return torch.empty(shape, dtype=torch.float32, device=DEV)


def _up(n, m):
    return (n + m - 1) // m * m


def _table(gen, lens, pages, width, first):
    """Each sequence's pages, scattered over the pool: those from `first` tokens back
    and the sinks' are held, the others' entries are -1."""
    B = lens.numel()
    place = torch.randperm(pages, generator=gen, device=DEV)
    at = torch.arange(width, device=DEV)
    held = at < first[:, 1:2]
    held &= (at >= first[:, :1]) | (at < first[:, 2:])
    count = held.flatten().cumsum(0).view(B, width) - 1
    return torch.where(held, place[count.clamp(min=0)], torch.full_like(count, -1)).contiguous()


def _inputs(c, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    k = c["kind"]
    if k == "window":
        B, H, Hkv, T, d = (c[n] for n in ("B", "H", "Hkv", "T", "d"))
        s = {"q": _rand(gen, B, T, H, d), "kv": _rand(gen, B, T, 2, Hkv, d)}
        if c["train"]:
            s["do"] = _rand(gen, B, T, H, d, scale=0.1)
        return s
    B, Hkv, T, d, P = (c[n] for n in ("B", "Hkv", "T", "d", "page"))
    most = c["len"]
    if k == "append":
        # what a projection gives: keys with a few large columns, values
        new = _rand(gen, B, T, 2, Hkv, d)
        new[:, :, 0] *= 1.0 + 5.0 * (torch.rand(Hkv, d, generator=gen, device=DEV) > 0.95)
        s = {"new": new, "open": _rand(gen, B, Hkv, 2, P, d)}
        if T == 1:
            lens = torch.randint((most + 1) // 2, most + 1, (B,), generator=gen, device=DEV)
            s["new_lens"] = None
            s["from"] = (lens - 1) // P * P
        else:  # prompts of several lengths behind whole pages that others share
            s["new_lens"] = torch.randint((T + 1) // 2, T + 1, (B,), generator=gen, device=DEV)
            s["from"] = torch.randint(0, (most - T) // P + 1, (B,), generator=gen, device=DEV) * P
            lens = s["from"] + s["new_lens"]
        width = _up(most, P) // P
        first = torch.stack([torch.zeros_like(lens), (lens + P - 1) // P, torch.zeros_like(lens)], 1)
        pages = B * width
    else:
        lens = torch.randint((most + 1) // 2, most + 1, (B,), generator=gen, device=DEV)
        s = {"q": _rand(gen, B, T, c["H"], d), "new_lens": None}
        width = _up(most, P) // P
        kept = min(width, (min(most, c["W"]) + T) // P + 2)
        back = (lens - (T - 1) - min(most, c["W"])).clamp(min=0) // P
        shown = torch.full_like(lens, (min(most, c["S"]) + P - 1) // P)
        first = torch.stack([back, (lens + P - 1) // P, shown], 1)
        pages = B * min(width, kept + (min(most, c["S"]) + P - 1) // P)
        # keys and values of about standard deviation 1, in steps of their page's scale
        n = pages * Hkv * 2 * P * d
        s["pool"] = torch.empty(pages + 1, Hkv, 2, P, d, dtype=torch.int8, device=DEV)
        flat = s["pool"].view(-1)
        for at in range(0, n, 1 << 26):
            part = torch.randn(min(1 << 26, n - at), generator=gen, device=DEV)
            flat[at : at + part.numel()] = part.mul_(40.0).round_().clamp_(-127, 127).to(torch.int8)
        flat[n:] = 0
        s["scales"] = 0.025 * (1.0 + 0.3 * torch.rand(pages + 1, Hkv, 2, generator=gen, device=DEV))
    s.update(lens=lens, table=_table(gen, lens, pages, width, first), pages=pages)
    return s


# a page's bytes hold number + 128: the keys' rows, padded to dp columns, then the values
# with the 32 tokens of a group beside each other in every column, in this order
_ORDER = [4 * int(f"{g:03b}"[::-1], 2) + i for g in range(8) for i in range(4)]


def _pack(pool):
    """[pages, Hkv, 2, P, d] numbers in the layout that include/aar_hip.h states."""
    n, Hkv, _, P, d = pool.shape
    dp = _up(d, 16)
    out = torch.empty(n, Hkv, 2, P * dp, dtype=torch.uint8, device=DEV)
    order = torch.tensor(_ORDER, device=DEV)
    step = max(1, (1 << 27) // (Hkv * P * dp))
    for at in range(0, n, step):
        x = torch.nn.functional.pad((pool[at : at + step].short() + 128).to(torch.uint8), (0, dp - d), value=128)
        out[at : at + step, :, 0] = x[:, :, 0].reshape(-1, Hkv, P * dp)
        v = x[:, :, 1].reshape(-1, Hkv, P // 32, 32, dp)[:, :, :, order]
        out[at : at + step, :, 1] = v.transpose(3, 4).reshape(-1, Hkv, P * dp)
    return out


def prepare(case, seed):
    """Inputs on the GPU, the cache that a program holds, and the outputs it allocates once."""
    c, k = dict(case), case["kind"]
    s = _inputs(c, seed)
    s["case"] = c
    if k == "window":
        B, H, Hkv, T, d = (c[n] for n in ("B", "H", "Hkv", "T", "d"))
        s.update(o=_new(B, T, H, d), lse=_new(B, H, T))
        if c["train"]:
            s.update(dq=_new(B, T, H, d), dkv=_new(B, T, 2, Hkv, d))
        return s
    B, Hkv, T, d, P = (c[n] for n in ("B", "Hkv", "T", "d", "page"))
    if k == "append":
        s["read"] = _new(B, P if T == 1 else T, 2, Hkv, d)
        if own:
            s["bytes"] = torch.empty(s["pages"], Hkv, 2 * P * _up(d, 16), dtype=torch.uint8, device=DEV)
            s["scales"] = _new(s["pages"], Hkv, 2)
        else:
            s["pool"] = torch.empty(s["pages"] + 1, Hkv, 2, P, d, dtype=torch.int8, device=DEV)
            s["scales"] = _new(s["pages"] + 1, Hkv, 2)
        return s
    s["o"] = _new(B, T, c["H"], d)
    if own:
        s["bytes"] = _pack(s.pop("pool")[:-1])
        s["scales"] = s["scales"][:-1].contiguous()
    return s


# ------------------------------------------------------------------ one pass

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"window": _own_window, "append": _own_append, "cache": _own_cache}[kind](state)
    return {"window": _plain_window, "append": _plain_append, "cache": _plain_cache}[kind](state)


def _plain_window(s):
    """Blocks of queries against the sinks and the keys of their windows."""
    c = s["case"]
    B, H, Hkv, T, W, S, d = (c[n] for n in ("B", "H", "Hkv", "T", "W", "S", "d"))
    G, scale = H // Hkv, 1.0 / math.sqrt(d)
    q = s["q"].permute(0, 2, 1, 3).reshape(B, Hkv, G, T, d)
    k, v = s["kv"].permute(2, 0, 3, 1, 4).contiguous().unbind(0)
    o = torch.empty(B, Hkv, G, T, d, device=DEV)
    lse = torch.empty(B, Hkv, G, T, device=DEV)
    if c["train"]:
        do = s["do"].permute(0, 2, 1, 3).reshape(B, Hkv, G, T, d)
        dq, dk, dv = torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    block = max(64, min(T, 1024, W))
    for a in range(0, T, block):
        b = min(T, a + block)
        lo = max(0, a - W + 1)
        first = min(S, lo)
        at = torch.cat([torch.arange(first, device=DEV), torch.arange(lo, b, device=DEV)])
        row = torch.arange(a, b, device=DEV)[:, None]
        hidden = (at > row) | ((at <= row - W) & (at >= S))
        kb = torch.cat([k[:, :, :first], k[:, :, lo:b]], 2)
        vb = torch.cat([v[:, :, :first], v[:, :, lo:b]], 2)
        n, m = b - a, kb.shape[2]
        qb = q[:, :, :, a:b].reshape(B, Hkv, G * n, d)
        score = torch.matmul(qb, kb.transpose(2, 3).contiguous()).mul_(scale).view(B, Hkv, G, n, m)
        score.masked_fill_(hidden, -math.inf)
        top = score.amax(-1, keepdim=True)
        p = torch.exp(score - top)
        total = p.sum(-1, keepdim=True)
        p = (p / total).view(B, Hkv, G * n, m)
        ob = torch.matmul(p, vb)
        o[:, :, :, a:b] = ob.view(B, Hkv, G, n, d)
        lse[:, :, :, a:b] = (top + torch.log(total))[..., 0]
        if c["train"]:
            g = do[:, :, :, a:b].reshape(B, Hkv, G * n, d)
            ds = p * (torch.matmul(g, vb.transpose(2, 3).contiguous()) - (g * ob).sum(-1, keepdim=True)) * scale
            dq[:, :, :, a:b] = torch.matmul(ds, kb).view(B, Hkv, G, n, d)
            gk = torch.matmul(ds.transpose(2, 3).contiguous(), qb)
            gv = torch.matmul(p.transpose(2, 3).contiguous(), g)
            dk[:, :, :first] += gk[:, :, :first]
            dk[:, :, lo:b] += gk[:, :, first:]
            dv[:, :, :first] += gv[:, :, :first]
            dv[:, :, lo:b] += gv[:, :, first:]

    def back(x):
        return x.reshape(B, H, T, d).permute(0, 2, 1, 3).contiguous()

    out = {"o": back(o), "lse": lse.reshape(B, H, T)}
    if c["train"]:
        out["dq"] = back(dq)
        out["dkv"] = torch.stack([dk, dv]).permute(1, 3, 0, 2, 4).contiguous()
    return out


def _over_127(x):
    return x / torch.full_like(x, 127.0)  # a division by a plain number would multiply by its rounded inverse


def _page_rows(c, s):
    """The rows of the pages that an append touches, [B, Hkv, 2, pages, P, d], zeros
    where there is none, and how many rows of them there are."""
    B, Hkv, T, d, P = (c[n] for n in ("B", "Hkv", "T", "d", "page"))
    new = s["new"].permute(0, 3, 2, 1, 4)
    if T == 1:
        rows = s["lens"] - s["from"]
        at = torch.arange(P, device=DEV)
        kept, last = (at < rows[:, None] - 1).view(B, 1, 1, P, 1), (at == rows[:, None] - 1).view(B, 1, 1, P, 1)
        x = torch.where(last, new, torch.where(kept, s["open"], torch.zeros_like(s["open"])))
        return x.view(B, Hkv, 2, 1, P, d), rows
    there = (torch.arange(T, device=DEV) < s["new_lens"][:, None]).view(B, 1, 1, T, 1)
    x = torch.zeros(B, Hkv, 2, _up(T, P), d, device=DEV, dtype=new.dtype)
    x[:, :, :, :T] = torch.where(there, new, torch.zeros_like(new))
    return x.view(B, Hkv, 2, -1, P, d), s["new_lens"]


def _plain_append(s):
    c = s["case"]
    B, Hkv, T, d, P = (c[n] for n in ("B", "Hkv", "T", "d", "page"))
    x, rows = _page_rows(c, s)
    n = x.shape[3]
    scale = _over_127(x.abs().amax((-2, -1)).double()).float()
    # a number's border may be as near as 2^-24 of it: in 64 bits
    step = torch.where(scale > 0, scale, torch.ones_like(scale)).double()[..., None, None]
    q = torch.round(x.double() / step).clamp_(-127, 127)
    value = q.float() * scale[..., None, None]
    index = torch.arange(n, device=DEV)
    used = index * P < rows[:, None]
    page = (s["from"] // P)[:, None] + index
    page = torch.where(used, s["table"].gather(1, page.clamp(max=s["table"].shape[1] - 1)), torch.full_like(page, s["pages"]))
    s["pool"][page] = q.to(torch.int8).permute(0, 3, 1, 2, 4, 5)
    s["scales"][page] = scale.permute(0, 3, 1, 2)
    # the last page's rows, where it is not full, are kept as they are
    left = rows % P
    last = (rows // P).clamp(max=n - 1).view(B, 1, 1, 1, 1, 1).expand(B, Hkv, 2, 1, P, d)
    mine = (torch.arange(P, device=DEV) < left[:, None]).view(B, 1, 1, P, 1)
    s["open"] = torch.where(mine, x.gather(3, last)[:, :, :, 0], s["open"])
    value = value.reshape(B, Hkv, 2, n * P, d)[:, :, :, : P if T == 1 else T]
    return {"read": value.permute(0, 3, 2, 1, 4).contiguous(), "open": s["open"]}


def _seen(c, s):
    """Positions of the tokens that a chunk's queries may see [B, n], each once, and
    which query sees which [B, T, n]."""
    T, W, S, lens = c["T"], c["W"], c["S"], s["lens"]
    most = c["len"]
    n = min(most, W + T - 1)
    low = (lens - n).clamp(min=0)[:, None]
    near = low + torch.arange(n, device=DEV)
    first = torch.arange(min(S, most), device=DEV).expand(lens.numel(), -1)
    at = torch.cat([torch.where(first < low, first, torch.full_like(first, EVERY)), near], 1)
    row = (lens[:, None] - T + torch.arange(T, device=DEV))[:, :, None]
    there = at[:, None, :]
    return at, (there <= row) & ((there > row - W) | (there < S))


def _plain_cache(s):
    c = s["case"]
    B, H, Hkv, T, d, P = (c[n] for n in ("B", "H", "Hkv", "T", "d", "page"))
    G, scale = H // Hkv, 1.0 / math.sqrt(d)
    at, sees = _seen(c, s)
    page = s["table"].gather(1, (at // P).clamp(max=s["table"].shape[1] - 1))
    page = torch.where((page >= 0) & (at < s["lens"][:, None]), page, torch.full_like(page, s["pages"]))
    kv = s["pool"][page, :, :, at % P].float() * s["scales"][page][..., None]  # [B, n, Hkv, 2, d]
    k, v = kv.permute(3, 0, 2, 1, 4).contiguous().unbind(0)
    q = s["q"].permute(0, 2, 1, 3).reshape(B, Hkv, G * T, d)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale).view(B, Hkv, G, T, -1)
    score.masked_fill_(~sees[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = torch.matmul(p.view(B, Hkv, G * T, -1), v)
    return {"o": o.view(B, H, T, d).permute(0, 2, 1, 3).contiguous()}


# ------------------------------------------------------------------ the framework's calls

class _Cache(ctypes.Structure):
    _fields_ = [("pages", ctypes.c_void_p), ("scales", ctypes.c_void_p), ("open", ctypes.c_void_p),
                ("table", ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in
                                               ("sequences", "table_width", "n_pages", "kv_heads", "page", "d")]


@functools.lru_cache(maxsize=1)
def _lib():
    lib = ctypes.CDLL(str(LIB))
    vp, i64, sz, i32, f32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_size_t, ctypes.c_int, ctypes.c_float

    def sign(name, res, args):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args

    sign("aar_window_attn_fwd_workspace_bytes", sz, [i64] * 7)
    sign("aar_window_attn_fwd_f32", i32, [vp] * 5 + [i64] * 5 + [vp, i64, i64, f32, vp, sz, vp])
    sign("aar_window_attn_bwd_workspace_bytes", sz, [i64] * 7)
    sign("aar_window_attn_bwd_f32", i32, [vp] * 9 + [i64] * 5 + [vp, i64, i64, f32, vp, sz, vp])
    sign("aar_kv_cache_append_f32", i32, [vp] * 6 + [i64, vp, vp])
    sign("aar_kv_cache_read_f32", i32, [vp] * 6 + [i64, vp, vp])
    sign("aar_kv_cache_attn_workspace_bytes", sz, [vp] + [i64] * 4)
    sign("aar_kv_cache_attn_f32", i32, [vp] * 6 + [i64] * 4 + [f32, vp, sz, vp, vp])
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


def _ptr(t):
    return None if t is None else t.data_ptr()


def _own_window(s):
    c, L = s["case"], _lib()
    B, H, Hkv, T, W, S, d = (c[n] for n in ("B", "H", "Hkv", "T", "W", "S", "d"))

    def make():
        dims = (B, H, Hkv, T, d, W, S)
        fb, bb = L.aar_window_attn_fwd_workspace_bytes(*dims), 0
        if c["train"]:
            bb = L.aar_window_attn_bwd_workspace_bytes(*dims)
        q, kv = [T * H * d, d, H * d], [T * 2 * Hkv * d, d, 2 * Hkv * d]
        fwd = (ctypes.c_int64 * 12)(*(q + kv + kv + q))
        bwd = (ctypes.c_int64 * 24)(*(q + kv + kv + q + q + q + kv + kv))
        return _scratch(max(fb, bb)), fb, bb, fwd, bwd

    ws, fb, bb, fwd, bwd = _plan(s, make)
    kv, st = s["kv"].data_ptr(), _stream()
    q, o, lse, half, scale = s["q"].data_ptr(), s["o"].data_ptr(), s["lse"].data_ptr(), 4 * Hkv * d, 1.0 / math.sqrt(d)
    _ok(L.aar_window_attn_fwd_f32(q, kv, kv + half, o, lse, B, H, Hkv, T, d, fwd, W, S, scale, ws.data_ptr(), fb, st))
    out = {"o": s["o"], "lse": s["lse"]}
    if c["train"]:
        dkv = s["dkv"].data_ptr()
        _ok(L.aar_window_attn_bwd_f32(q, kv, kv + half, o, lse, s["do"].data_ptr(), s["dq"].data_ptr(), dkv, dkv + half,
                                      B, H, Hkv, T, d, bwd, W, S, scale, ws.data_ptr(), bb, st))
        out.update(dq=s["dq"], dkv=s["dkv"])
    return out


def _cache(s):
    c = s["case"]
    return _Cache(s["bytes"].data_ptr(), s["scales"].data_ptr(), _ptr(s.get("open")), s["table"].data_ptr(), c["B"],
                  s["table"].shape[1], s["pages"], c["Hkv"], c["page"], c["d"])


def _own_append(s):
    c, L = s["case"], _lib()
    Hkv, T, d, half = c["Hkv"], c["T"], c["d"], 4 * c["Hkv"] * c["d"]

    def make():
        def strides(n):
            return [n * 2 * Hkv * d, d, 2 * Hkv * d] * 2

        rows = s["read"].shape[1]
        return _cache(s), (ctypes.c_int64 * 6)(*strides(T)), (ctypes.c_int64 * 6)(*strides(rows)), rows

    cache, new, read, rows = _plan(s, make)
    x, y, lens, st = s["new"].data_ptr(), s["read"].data_ptr(), s["lens"].data_ptr(), _stream()
    _ok(L.aar_kv_cache_append_f32(ctypes.byref(cache), x, x + half, new, lens, _ptr(s["new_lens"]), T, None, st))
    _ok(L.aar_kv_cache_read_f32(ctypes.byref(cache), s["from"].data_ptr(), lens, y, y + half, read, rows, None, st))
    return {"read": s["read"], "open": s["open"]}


def _own_cache(s):
    c, L = s["case"], _lib()
    H, T, W, S, d = (c[n] for n in ("H", "T", "W", "S", "d"))

    def make():
        cache = _cache(s)
        ws = _scratch(L.aar_kv_cache_attn_workspace_bytes(ctypes.byref(cache), H, T, W, S))
        return cache, (ctypes.c_int64 * 6)(*([T * H * d, d, H * d] * 2)), ws

    cache, strides, ws = _plan(s, make)
    _ok(L.aar_kv_cache_attn_f32(ctypes.byref(cache), s["q"].data_ptr(), s["o"].data_ptr(), strides, s["lens"].data_ptr(),
                                _ptr(s["new_lens"]), H, T, W, S, 1.0 / math.sqrt(d), ws.data_ptr(), ws.numel(), None,
                                _stream()))
    return {"o": s["o"]}


# ------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    """The definitions in 64 bits, gradients by torch's own differentiation.  A page's
    scale is a number of 32 bits by definition, its elements whole numbers."""
    c, k = case, case["kind"]
    s = _inputs(c, seed)
    if k == "window":
        return _exact_window(c, s)
    if k == "append":
        B, Hkv, T, d, P = (c[n] for n in ("B", "Hkv", "T", "d", "page"))
        rows = P if T == 1 else T
        read = torch.zeros(B, rows, 2, Hkv, d, dtype=torch.float64, device=DEV)
        kept = s["open"].double()
        for b in range(B):
            end = int(s["lens"][b]) - int(s["from"][b])
            x = s["new"][b].permute(2, 1, 0, 3).double()  # [Hkv, 2, T, d]
            x = torch.cat([kept[b, :, :, : end - 1], x], 2) if T == 1 else x[:, :, :end]
            for a in range(0, end, P):
                part = x[:, :, a : a + P]
                scale = _over_127(part.abs().amax((2, 3))).float().double()[..., None, None]
                read[b, a : a + P][:end - a] = (torch.round(part / scale) * scale).permute(2, 1, 0, 3)
            if end % P:
                kept[b, :, :, : end % P] = x[:, :, end // P * P :]
        return {"read": read, "open": kept}
    B, H, Hkv, T, d, P, W, S = (c[n] for n in ("B", "H", "Hkv", "T", "d", "page", "W", "S"))
    if float(B) * H * c["len"] * T * d > 4e11:
        return None
    o = torch.zeros(B, T, H, d, dtype=torch.float64, device=DEV)
    for b in range(B):
        n = int(s["lens"][b])
        at = torch.arange(n, device=DEV)
        page = s["table"][b, at // P]
        kv = s["pool"][page, :, :, at % P].double() * s["scales"][page].double()[..., None]  # [n, Hkv, 2, d]
        row = torch.arange(n - T, n, device=DEV)[:, None]
        sees = (at <= row) & ((row - at < W) | (at < S)) & (page >= 0)
        for h in range(H):
            x = kv[:, h * Hkv // H]
            score = (s["q"][b, :, h].double() @ x[:, 0].t()) / math.sqrt(d)
            o[b, :, h] = torch.softmax(score.masked_fill(~sees, -math.inf), -1) @ x[:, 1]
    return {"o": o}


def _exact_window(c, s):
    B, H, Hkv, T, W, S, d = (c[n] for n in ("B", "H", "Hkv", "T", "W", "S", "d"))
    o = torch.empty(B, T, H, d, dtype=torch.float64, device=DEV)
    lse = torch.empty(B, H, T, dtype=torch.float64, device=DEV)
    dq, dkv = torch.zeros_like(o), torch.zeros(B, T, 2, Hkv, d, dtype=torch.float64, device=DEV)
    at = torch.arange(T, device=DEV)
    for b in range(B):
        for h in range(H):
            hk = h * Hkv // H
            for a in range(0, T, 4096):  # rows at once, against every key
                e = min(T, a + 4096)
                row = at[a:e, None]
                sees = (at[:e] <= row) & ((row - at[:e] < W) | (at[:e] < S))
                q = s["q"][b, a:e, h].double().requires_grad_()
                kv = s["kv"][b, :e, :, hk].double().requires_grad_()
                score = ((q @ kv[:, 0].t()) / math.sqrt(d)).masked_fill(~sees, -math.inf)
                got = torch.softmax(score, -1) @ kv[:, 1]
                o[b, a:e, h], lse[b, h, a:e] = got.detach(), torch.logsumexp(score.detach(), -1)
                if c["train"]:
                    got.backward(s["do"][b, a:e, h].double())
                    dq[b, a:e, h] = q.grad
                    dkv[b, :e, :, hk] += kv.grad
    return {"o": o, "lse": lse, "dq": dq, "dkv": dkv} if c["train"] else {"o": o, "lse": lse}
