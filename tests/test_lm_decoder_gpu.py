"""The operators as they are used: training steps of a small decoder that reads a
padded encoder and learns from a teacher (scaled embedding, normed and rotated
self attention, cross attention with shared heads, MLP, vocabulary head,
distillation), its loss and every parameter's gradient against 64 bits, and the
same decoder token by token against the projected context."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import lmops as M
from devutil import dev, host

pytestmark = pytest.mark.gpu

V, D, H, HKV, LAYERS, C, K = 300, 128, 4, 2, 2, 72, 7
B, T, S, TAU = 3, 40, 90, 2.0
d = D // H


def build(ag, rng):
    nn = ag.nn

    class Block(nn.Module):
        def __init__(self):
            super().__init__()
            self.ln1, self.ln2, self.ln3 = nn.LayerNorm(D), nn.LayerNorm(D), nn.LayerNorm(D)
            self.attn = nn.MultiHeadAttention(D, H, causal=True, bias=False, rng=rng, qk_norm=True)
            self.cross = nn.CrossAttention(D, H, d_context=C, n_kv_heads=HKV, bias=False, rng=rng)
            self.up, self.down = nn.Linear(D, 2 * D, bias=True, rng=rng), nn.Linear(2 * D, D, bias=True, rng=rng)

        def forward(self, x, context, lens):
            x = ag.add(x, self.attn(self.ln1(x)))
            x = ag.add(x, self.cross(self.ln2(x), context, lens))
            return ag.add(x, self.down(ag.gelu(self.up(self.ln3(x)))))

    class Decoder(nn.Module):
        def __init__(self):
            super().__init__()
            self.emb = nn.Embedding(V, D, rng=rng, scale=0.5)
            self.blocks = nn.Sequential(*[Block() for _ in range(LAYERS)])
            self.norm = nn.LayerNorm(D)
            self.head = nn.Linear(D, V, rng=rng)

        def forward(self, ids, context, lens):
            x = self.emb(ids)
            for blk in self.blocks._modules.values():
                x = blk(x, context, lens)
            return self.head(self.norm(x))

    return Decoder()


def reference(params, ids, context, lens, best, tids):
    """Loss and logits in 64 bits; params in the module's order."""
    it = iter(params)
    nxt = lambda: next(it)  # noqa: E731
    rows = torch.arange(T, dtype=torch.float64)
    angle = rows[:, None, None] * 10000.0 ** (torch.arange(d // 2, dtype=torch.float64) * (-2.0 / d))

    def norm(x, w, b):
        return torch.nn.functional.layer_norm(x, (D,), w, b, 1e-5)

    def turn(u, w):
        u = u / torch.sqrt(u.pow(2).mean(-1, keepdim=True) + 1e-6) * w
        a, b = u[..., : d // 2], u[..., d // 2:]
        return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)

    def attend(q, k, v, hide):
        s = (q.transpose(1, 2) @ k.transpose(1, 2).transpose(2, 3)) / math.sqrt(d)
        p = torch.softmax(s.masked_fill(hide, -1e300), -1) * ~hide
        return (p @ v.transpose(1, 2)).transpose(1, 2).reshape(B, T, D)

    x = nxt()[ids] * 0.5
    for _ in range(LAYERS):
        ln = [(nxt(), nxt()) for _ in range(3)]
        qn, kn, wqkv, wo, cq, ckv, co, w1, b1, w2, b2 = (nxt() for _ in range(11))
        qkv = (norm(x, *ln[0]) @ wqkv.t()).view(B, T, 3, H, d)
        a = attend(turn(qkv[:, :, 0], qn), turn(qkv[:, :, 1], kn), qkv[:, :, 2], torch.ones(T, T).triu(1).bool())
        x = x + a @ wo.t()
        q = (norm(x, *ln[1]) @ cq.t()).view(B, T, H, d)
        kv = (context @ ckv.t()).view(B, S, 2, HKV, d).repeat_interleave(H // HKV, 3)
        hidden = (torch.arange(S) >= lens.view(B, 1, 1, 1)).expand(B, 1, T, S)
        x = x + attend(q, kv[:, :, 0], kv[:, :, 1], hidden) @ co.t()
        x = x + torch.nn.functional.gelu(norm(x, *ln[2]) @ w1.t() + b1) @ w2.t() + b2
    nw, nb, head = nxt(), nxt(), nxt()
    logits = norm(x, nw, nb) @ head.t()
    z = logits.reshape(B * T, V)
    on = (tids >= 0).any(-1)
    p = torch.softmax((best[on] / TAU).masked_fill(tids[on] < 0, -math.inf), -1)
    logq = torch.log_softmax(z / TAU, -1)[on].gather(1, tids[on].clamp(min=0))
    return TAU * TAU * (torch.xlogy(p, p) - p * logq).sum() / on.sum(), logits


def data():
    rng = np.random.default_rng(11)
    ids = rng.integers(0, V, (B, T)).astype(np.int64)
    context = rng.standard_normal((B, S, C)).astype(np.float32)
    lens = np.array([S, 0, 33], np.int64)
    best = rng.standard_normal((B * T, K)).astype(np.float32)
    tids = np.argsort(rng.random((B * T, V)), -1)[:, :K].astype(np.int64)
    tids[::9] = -1
    tids[4::5, 3:] = -1
    return ids, context, lens, best, tids


def test_training_steps(gpu):
    model = build(gpu, np.random.default_rng(0)).to(gpu.Device.CUDA)
    ids, context, lens, best, tids = data()
    up = lambda a: gpu.from_numpy(a).to(gpu.Device.CUDA)  # noqa: E731
    crit = gpu.nn.DistillationLoss(TAU)
    params = list(model.parameters())
    opt = gpu.optim.SGD(params, lr=0.05)
    # roundings of two blocks' products (up to 2 D terms) and attentions, one after
    # another: about twelve stages, each as large as one attention's
    tol = 12 * M.attn_tol(2 * D, B * T)
    for step in range(3):
        w = [torch.from_numpy(host(gpu, p.tensor)).double().requires_grad_() for p in params]
        model.zero_grad()
        tc = dev(gpu, context, True)
        logits = model(up(ids), tc, up(lens))
        loss = crit(gpu.reshape(logits, [B * T, V]), dev(gpu, best), up(tids))
        loss.backward()
        C64 = torch.from_numpy(context).double().requires_grad_()
        rl, rz = reference(w, torch.from_numpy(ids), C64, torch.from_numpy(lens), torch.from_numpy(best).double(),
                           torch.from_numpy(tids))
        rl.backward()
        M.near(host(gpu, logits), rz, tol, f"step {step} logits")
        M.near(host(gpu, loss).reshape(1), rl.reshape(1), tol, f"step {step} loss")
        for i, (p, r) in enumerate(zip(params, w)):
            M.near(host(gpu, p.tensor.grad), r.grad, tol, f"step {step} parameter {i}")
        M.near(host(gpu, tc.grad), C64.grad, tol, f"step {step} context")
        opt.step()


def test_serving_steps(gpu):
    """Each token by itself: rotation at its own position, cross attention over the
    context projected once."""
    model = build(gpu, np.random.default_rng(0)).to(gpu.Device.CUDA)
    blk = next(iter(model.blocks._modules.values()))
    ids, context, lens, _, _ = data()
    up = lambda a: gpu.from_numpy(a).to(gpu.Device.CUDA)  # noqa: E731
    x, tl = model.emb(up(ids)), up(lens)
    kv = blk.cross.project_context(dev(gpu, context))
    whole = host(gpu, blk.cross(x, dev(gpu, context), tl))
    qkv = blk.attn.qkv_proj(x)
    w = blk.attn.q_norm.tensor, blk.attn.k_norm.tensor
    qk = gpu.contiguous(gpu.slice(qkv, 2, 0, 2 * D))
    rotated = host(gpu, gpu.qk_norm_rope(qk, *w, up(np.arange(T, dtype=np.int64)), H, H))
    for t in range(0, T, 7):
        one = gpu.contiguous(gpu.slice(x, 1, t, t + 1))
        M.near(host(gpu, blk.cross.attend(one, kv, tl))[:, 0], whole[:, t], 2 * M.attn_tol(D, S), f"token {t}")
        row = gpu.contiguous(gpu.slice(qk, 1, t, t + 1))
        pos = up(np.full((B, 1), t, np.int64))
        M.near(host(gpu, gpu.qk_norm_rope(row, *w, pos, H, H))[:, 0], rotated[:, t], 8 * M.U * math.sqrt(d), f"rotation {t}")
