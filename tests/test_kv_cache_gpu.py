"""The paged 8-bit key/value cache (aar_kv_cache_*) on the GPU against its definition
in 64 bits: what pages hold whatever chunks tokens came in, reading back, attention of
single tokens, chunks and prompts with and without a window, padded calls, pages
without an id, unaligned rows, other streams and captured graphs."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import kvops as K
import lmops as M

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L(gpu):
    return K.lib()


def rand(seed, *shape, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).cuda()


def ints(*x):
    return torch.tensor(x, dtype=torch.int64, device="cuda")


def held(k, v, lens, page):
    """What a cache holds of the first lens[b] rows of k, v [B, Hkv, T, d]: lists of
    [Hkv, len, d] in 64 bits."""
    out = []
    for x in (k, v):
        out.append([torch.stack([K.quantised(x[b, h, : int(lens[b])].cpu(), page) for h in range(x.shape[1])])
                    for b in range(x.shape[0])])
    return out


def check_read(L, pool, k, v, lens):
    T = k.shape[2]
    got = pool.read(L, lens, T).cpu().double()
    for g, rows in zip(got, held(k, v, lens, pool.P)):
        for b in range(k.shape[0]):
            n = int(lens[b])
            # a value is a whole number times the scale, rounded once
            assert ((g[b, :, :n] - rows[b]).abs() <= M.U * rows[b].abs() + 2.0 ** -150).all()
            assert (g[b, :, n:] == 0).all()


@pytest.mark.parametrize("page", [32, 64, 128])
@pytest.mark.parametrize("d", [64, 128, 1, 30, 40, 96])
def test_pages_do_not_depend_on_the_chunks(L, page, d):
    """All at once, token by token, and in ragged chunks: the same bytes, the ones that
    the definition gives, in the documented layout."""
    B, Hkv, T = 3, 2, 2 * page + 21
    k, v = rand(1, B, Hkv, T, d), rand(2, B, Hkv, T, d, scale=3.0)
    lens = ints(T, page, page + 5)
    width = K.up(T, page) // page
    whole = K.Pool(B, Hkv, d, page, width)
    whole.append(L, k, v, lens, lens)
    check_read(L, whole, k, v, lens)
    ref = held(k, v, lens, page)
    values = whole.values()
    for b in range(B):
        for j in range(int(lens[b])):
            at = whole.table[b, j // page].item()
            for kv in (0, 1):
                assert torch.equal(values[at, :, kv, j % page], ref[kv][b][:, j])
    steps = [[1] * T, [7, 1, 40, 13, 1, 2], [page - 1, 2, page + 3, 1]]
    for sizes in steps:
        pool = K.Pool(B, Hkv, d, page, width)
        done = torch.zeros(B, dtype=torch.int64)
        while (done < lens.cpu()).any():
            n = sizes[0] if len(sizes) > 1 else T
            sizes = sizes[1:] or sizes
            new = torch.minimum(lens.cpu() - done, torch.tensor(n))
            x = torch.full((2, B, Hkv, n, d), math.nan, device="cuda")  # rows past new_lens are not read
            for b in range(B):
                m = int(new[b])
                x[0, b, :, :m] = k[b, :, int(done[b]) : int(done[b]) + m]
                x[1, b, :, :m] = v[b, :, int(done[b]) : int(done[b]) + m]
            done += new
            pool.append(L, x[0], x[1], done.cuda(), new.cuda())
        for b in range(B):
            for i in range(-(-int(lens[b]) // page)):
                at = whole.table[b, i]
                assert torch.equal(pool.bytes[at], whole.bytes[at]) and torch.equal(pool.scales[at], whole.scales[at])
    assert whole.err.item() == 0


def test_other_pages_are_left_alone(L):
    pool = K.Pool(2, 2, 40, 32, 3)
    before = pool.bytes.clone()
    k = rand(1, 2, 2, 50, 40)
    pool.append(L, k, k, ints(50, 20), ints(50, 20))
    used = {pool.table[0, 0].item(), pool.table[0, 1].item(), pool.table[1, 0].item()}
    for at in range(pool.n):
        if at not in used:
            assert torch.equal(pool.bytes[at], before[at]) and torch.isnan(pool.scales[at]).all()
    assert torch.isnan(pool.open[0, :, :, 18:]).all() and torch.isnan(pool.open[1, :, :, 20:]).all()
    assert torch.equal(pool.open[0, :, 0, :18], k[0, :, 32:50])


@pytest.mark.parametrize("power", [-149, -140, -126, -110, -99, -30, 60, 120, 127])
def test_magnitudes_and_ties(L, power):
    """Rows of every magnitude, and numbers that are exactly between two."""
    P, d = 32, 64
    x = torch.randn(P, d, generator=torch.Generator().manual_seed(3), dtype=torch.float64)
    x = (x.clamp(-0.9, 0.9) * 2.0 ** power).float()
    x[0, 0] = 2.0 ** power
    tie = torch.zeros(P, d)
    tie[0, 0] = 127.0
    tie.view(-1)[1:255] = torch.arange(-127, 127) + 0.5
    tie = (tie.double() * 2.0 ** max(-149, min(power, 120))).float()
    for rows in (x, tie):
        pool = K.Pool(1, 1, d, P, 1)
        t = rows.view(1, 1, P, d).cuda()
        pool.append(L, t, t, ints(P))
        check_read(L, pool, t, t, ints(P))


def test_infinities_and_nan_in_a_page(L):
    """They make their page's head NaN, keys or values apart, and nothing else."""
    k, v = rand(1, 2, 2, 70, 64), rand(2, 2, 2, 70, 64)
    k[0, 1, 3, 5], v[1, 0, 40, 6] = math.inf, math.nan
    pool = K.Pool(2, 2, 64, 32, 3)
    lens = ints(70, 70)
    pool.append(L, k, v, lens)
    got = pool.read(L, lens, 70)
    bad = torch.zeros(2, 2, 2, 70, 64, dtype=torch.bool, device="cuda")
    bad[0, 0, 1, :32] = True
    bad[1, 1, 0, 32:64] = True
    assert torch.equal(torch.isnan(got), bad)
    # a token that sees neither page
    q = rand(3, 2, 2, 1, 64)
    o = pool.attend(L, q, lens, window=6)
    assert torch.isfinite(o).all()
    o = pool.attend(L, q, lens)
    assert torch.equal(torch.isnan(o).all(-1)[..., 0], torch.tensor([[False, True], [True, False]], device="cuda"))
    # a chunk whose first tokens see the page and whose last do not
    q = rand(4, 2, 2, 12, 64)
    o = pool.attend(L, q, lens, window=3)
    want = torch.zeros(2, 2, 12, dtype=torch.bool, device="cuda")
    want[1, 0, :8] = True  # positions 58 .. 65 see one of the tokens up to 63
    assert torch.equal(torch.isnan(o).any(-1), want)
    zero = torch.zeros(1, 1, 32, 64, device="cuda")
    pool = K.Pool(1, 1, 64, 32, 1)
    pool.append(L, zero, zero, ints(32))
    assert (pool.read(L, ints(32), 32) == 0).all() and (pool.attend(L, q[:1, :1], ints(32)) == 0).all()


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("scale", [None, 0.0])
def test_keys_that_are_not_finite(L, bad, scale):
    """Queries that see the page are NaN, whatever the scale, others do not change."""
    k, v, q = rand(1, 1, 1, 90, 64), rand(2, 1, 1, 90, 64), rand(3, 1, 2, 50, 64)
    lens = ints(90)
    pool = K.Pool(1, 1, 64, 32, 3)
    pool.append(L, k, v, lens)
    fine = pool.attend(L, q, lens, window=9, scale=scale)
    k[0, 0, 40, 7] = bad
    pool.append(L, k, v, lens)
    o = pool.attend(L, q, lens, window=9, scale=scale)
    sees = torch.arange(40, 90, device="cuda") - 9 < 63  # tokens 32 .. 63 share the page
    assert torch.equal(torch.isnan(o).all(-1), sees.expand(1, 2, 50)) and torch.equal(torch.isnan(o).any(-1), torch.isnan(o).all(-1))
    assert torch.equal(o[:, :, ~sees], fine[:, :, ~sees])


@pytest.mark.parametrize("first", [None, (0, 5, 40), (-7, 33, 100), (64, 96, -200)])
def test_reading_ranges(L, first):
    B, Hkv, T, d = 3, 2, 100, 36
    k, v = rand(1, B, Hkv, T, d), rand(2, B, Hkv, T, d)
    lens = ints(100, 64, 37)
    pool = K.Pool(B, Hkv, d, 32, 4)
    pool.append(L, k, v, lens, lens)
    whole = pool.read(L, lens, T)
    got = pool.read(L, lens, 45, None if first is None else ints(*first))
    for b in range(B):
        f = 0 if first is None else first[b]
        for i in range(45):
            want = whole[:, b, :, f + i] if 0 <= f + i < T else torch.zeros_like(got[:, b, :, i])
            assert torch.equal(got[:, b, :, i], want)


# B, H, Hkv, d, page, T, lens, window, sinks
EVERY = 1 << 62
CASES = [
    (1, 1, 1, 64, 32, 1, (1,), EVERY, 0), (1, 2, 2, 64, 64, 1, (31,), EVERY, 0), (2, 6, 6, 64, 64, 1, (33, 500), EVERY, 0),
    (3, 8, 2, 128, 32, 1, (129, 1, 777), EVERY, 0), (2, 16, 1, 64, 128, 1, (300, 128), EVERY, 0),
    (1, 32, 1, 96, 64, 1, (1000,), EVERY, 0), (1, 64, 1, 32, 32, 1, (400,), EVERY, 0), (2, 2, 2, 1, 32, 1, (40, 7), EVERY, 0),
    (2, 4, 2, 30, 64, 1, (100, 65), EVERY, 0), (1, 6, 6, 64, 64, 1, (4000,), EVERY, 0), (2, 4, 4, 64, 32, 1, (900, 63), 100, 4),
    (2, 4, 2, 128, 64, 1, (900, 40), 1, 0), (2, 4, 2, 64, 128, 1, (900, 1000), 300, 130), (1, 3, 3, 40, 32, 1, (2000,), 64, 1),
    (1, 1, 1, 64, 32, 2, (2,), EVERY, 0), (2, 4, 2, 64, 64, 5, (5, 100), EVERY, 0), (2, 2, 2, 128, 32, 17, (40, 17), EVERY, 0),
    (1, 4, 1, 64, 64, 40, (300,), EVERY, 0), (2, 3, 3, 64, 32, 100, (100, 260), EVERY, 0), (1, 8, 2, 128, 128, 70, (500,), EVERY, 0),
    (1, 2, 2, 36, 64, 130, (200,), 50, 3), (2, 4, 2, 64, 32, 65, (65, 400), 30, 40), (1, 2, 1, 64, 64, 33, (1000,), 1, 1),
    (1, 16, 2, 64, 32, 9, (700,), 90, 0), (1, 2, 2, 3, 32, 40, (90,), EVERY, 0), (4, 12, 12, 64, 64, 1, (2000, 1, 64, 65), EVERY, 0),
]


def filled(L, B, Hkv, d, page, lens, seed=5):
    T = max(lens)
    k, v = rand(seed, B, Hkv, T, d), rand(seed + 1, B, Hkv, T, d)
    pool = K.Pool(B, Hkv, d, page, K.up(T, page) // page + 1)
    pool.append(L, k, v, ints(*lens), ints(*lens))
    return pool, held(k, v, lens, page)


@pytest.mark.parametrize("case", CASES)
def test_attention_against_the_definition(L, case):
    B, H, Hkv, d, page, T, lens, window, sinks = case
    pool, (k, v) = filled(L, B, Hkv, d, page, lens)
    q = rand(9, B, H, T, d)
    ref = K.cache_exact(q, k, v, lens, [T] * B, window, sinks)
    o = pool.attend(L, q, ints(*lens), None, window, sinks)
    M.near(o, ref, M.attn_tol(d, min(max(lens), window + sinks)), "o")
    assert pool.err.item() == 0
    # q scaled row by row by powers of two that its scale takes back: the same
    o2 = pool.attend(L, q * 2.0 ** 90, ints(*lens), None, window, sinks, scale=d ** -0.5 * 2.0 ** -90)
    assert torch.equal(o, o2)
    o3 = pool.attend(L, q * 2.0 ** -100, ints(*lens), None, window, sinks, scale=d ** -0.5 * 2.0 ** 100)
    assert torch.equal(o, o3)


@pytest.mark.parametrize("T", [1, 8, 70])
def test_padded_calls(L, T):
    """Sequences with no, one, some and all of the call's tokens; rows behind them are
    zeros, as are those of a sequence whose numbers do not fit, which says so."""
    lens = (0, 200, 150, 70 + T, 100)
    new = (0, 1, (T + 1) // 2, T, 0)
    B, H, Hkv, d = 5, 4, 2, 64
    pool, (k, v) = filled(L, B, Hkv, d, 32, lens)
    q = rand(9, B, H, T, d)
    for b in range(B):
        q[b, :, new[b] :] = math.nan
    ref = K.cache_exact(q, k, v, lens, new, EVERY, 0)
    o = pool.attend(L, q, ints(*lens), ints(*new))
    M.near(o, ref, M.attn_tol(d, 200), "o")
    for b in range(B):
        assert (o[b, :, new[b] :] == 0).all()
    assert pool.err.item() == 0
    most = pool.width * pool.P
    for bad_len, bad_new in (((-1, 200, most + 1, 70 + T, 1 << 40), new), (lens, (1, -1, T + 1, 70 + T + 1, 1 << 40))):
        pool.err.zero_()
        got = pool.attend(L, q, ints(*bad_len), ints(*bad_new))
        assert pool.err.item() == 1
        for b in range(B):
            if bad_len[b] == lens[b] and bad_new[b] == new[b]:
                assert torch.equal(got[b], o[b])
            elif not (0 <= bad_len[b] <= most and 0 <= bad_new[b] <= min(T, bad_len[b])):
                assert (got[b] == 0).all()


def test_sequences_that_do_not_fit_are_not_stored(L):
    k = rand(1, 3, 2, 40, 64)
    pool = K.Pool(3, 2, 64, 32, 2)
    before = pool.bytes.clone()
    for lens, new in (((65, -3, 20), (40, 0, 21)), ((1 << 50, 5, 64), (1, 6, -1))):
        pool.append(L, k, k, ints(*lens), ints(*new))
        assert pool.err.item() == 1 and torch.equal(pool.bytes, before) and torch.isnan(pool.open).all()
        pool.err.zero_()
    # and ids outside the pool: that page alone is left out
    pool.table[1, 0], pool.table[2, 1] = pool.n, -1
    pool.append(L, k, k, ints(40, 40, 40))
    assert pool.err.item() == 1
    pool.err.zero_()
    got = pool.read(L, ints(40, 40, 40), 40)
    assert pool.err.item() == 1
    pool.err.zero_()
    fine = [rows for rows in held(k[:1], k[:1], (40,), 32)[0]]
    assert (got[0, 1, :, :32] == 0).all() and (got[0, 2, :, 32:] == 0).all()
    M.near(got[0, 0], fine[0], M.U, "read")
    # attention: hidden keys, whoever asks
    q = rand(2, 3, 2, 1, 64)
    lens = ints(40, 40, 40)
    o = pool.attend(L, q, lens)
    assert pool.err.item() == 1
    ref = held(k, k, (40, 40, 40), 32)[0]
    for b, rows in ((1, slice(32, 40)), (2, slice(0, 32))):
        x = ref[b][:, rows]
        s = (q[b].double().cpu() @ x.transpose(1, 2).contiguous()) / 8.0
        M.near(o[b], torch.softmax(s, -1) @ x, M.attn_tol(64, 40), "o")
    # a page that the window passes over is not looked up
    pool.err.zero_()
    pool.table[1, 0] = -5
    pool.attend(L, q[:, :, :1], lens, window=8)
    assert pool.err.item() == 1  # sequence 2's last page
    pool.table[2, 1] = pool.table[0, 1]
    pool.err.zero_()
    assert torch.isfinite(pool.attend(L, q, lens, window=8)).all() and pool.err.item() == 0
    # nothing at all to see
    pool.table[0, :] = -1
    assert (pool.attend(L, q, lens)[0] == 0).all()


def test_shared_pages(L):
    """Sequences whose first pages are the same."""
    k, v = rand(1, 1, 2, 128, 64), rand(2, 1, 2, 128, 64)
    pool = K.Pool(3, 2, 64, 64, 3)
    pool.table[1:, :2] = pool.table[:1, :2]
    lens = ints(128, 0, 0)
    pool.append(L, k.expand(3, 2, 128, 64), v.expand(3, 2, 128, 64), lens, lens)
    new = rand(3, 3, 2, 1, 64)
    lens = ints(129, 129, 129)
    pool.append(L, new, new, lens)
    q = rand(4, 3, 4, 1, 64)
    o = pool.attend(L, q, lens)
    kk, vv = (torch.cat([x.expand(3, 2, 128, 64), new], 2) for x in (k, v))
    M.near(o, K.cache_exact(q, *held(kk, vv, [129] * 3, 64), [129] * 3, [1] * 3, EVERY, 0), M.attn_tol(64, 129), "o")


@pytest.mark.parametrize("d", [64, 128, 36])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("T", [1, 37])
def test_strided_rows(L, d, offset, T):
    """Views of a packed projection, outputs in [B, T, H, d] order, unaligned bases."""
    B, H, Hkv = 2, 4, 2

    def rows(*shape):
        n = math.prod(shape)
        return torch.full((n + 4,), 3.0, device="cuda")[offset : offset + n].view(shape)

    packed = rows(B, T, H + 2 * Hkv, d)
    packed.copy_(rand(1, *packed.shape))
    q, k, v = (t.transpose(1, 2) for t in (packed[:, :, :H], packed[:, :, H : H + Hkv], packed[:, :, H + Hkv :]))
    lens = ints(T, T)
    a, b = K.Pool(B, Hkv, d, 32, 2), K.Pool(B, Hkv, d, 32, 2)
    a.append(L, k, v, lens)
    b.append(L, k.contiguous(), v.contiguous(), lens)
    for i in range(B):
        for at in a.table[i, : -(-T // 32)]:
            assert torch.equal(a.bytes[at], b.bytes[at])
    o = rows(B, T, H, d)
    a.attend(L, q, lens, out=o.transpose(1, 2))
    dense = b.attend(L, q.contiguous(), lens)
    assert torch.equal(o.transpose(1, 2), dense)
    read = rows(2, B, T, Hkv, d)
    c = a.struct()
    M.ok(L.aar_kv_cache_read_f32(ctypes.byref(c), None, lens.data_ptr(), read[0].data_ptr(), read[1].data_ptr(),
                                 M.strides3(read[0].transpose(1, 2), read[1].transpose(1, 2)), T, None, M.stream()))
    assert torch.equal(read.transpose(2, 3), b.read(L, lens, T))


def test_same_bits_streams_and_graphs(L):
    """A captured step (append, then attention) replayed over a growing text."""
    B, H, Hkv, d, n0 = 2, 4, 2, 64, 300
    k, v = rand(1, B, Hkv, n0 + 40, d), rand(2, B, Hkv, n0 + 40, d)
    q = rand(3, B, H, n0 + 40, d)
    pools = []
    for _ in range(2):
        pool = K.Pool(B, Hkv, d, 32, 12)
        pool.append(L, k[:, :, :n0], v[:, :, :n0], ints(n0, n0))
        pools.append(pool)
    lens, kn, vn, qn = ints(n0, n0), *(torch.empty(B, h, 1, d, device="cuda") for h in (Hkv, Hkv, H))
    out = torch.empty(B, H, 1, d, device="cuda")
    c = pools[0].struct()
    ws = M.scratch(L.aar_kv_cache_attn_workspace_bytes(ctypes.byref(c), H, 1, 200, 4))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens.add_(1)
        pools[0].append(L, kn, vn, lens)
        pools[0].attend(L, qn, lens, None, 200, 4, out=out, ws=ws)
    assert lens.tolist() == [n0, n0]
    side = torch.cuda.Stream()
    for t in range(n0, n0 + 40):
        for dst, src in ((kn, k), (vn, v), (qn, q)):
            dst.copy_(src[:, :, t : t + 1])
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            n = ints(t + 1, t + 1)
            pools[1].append(L, k[:, :, t : t + 1], v[:, :, t : t + 1], n)
            o = pools[1].attend(L, q[:, :, t : t + 1], n, None, 200, 4)
        side.synchronize()
        assert torch.equal(o, out)
    assert lens.tolist() == [n0 + 40] * 2
    full = held(k, v, [n0 + 40] * B, 32)
    ref = K.cache_exact(q[:, :, -1:], *full, [n0 + 40] * B, [1] * B, 200, 4)
    M.near(out, ref, M.attn_tol(d, 204), "o")


def test_workspace_is_held_to(L):
    pool, _ = filled(L, 1, 1, 64, 32, (5000,))
    q = rand(1, 1, 2, 1, 64)
    c, lens = pool.struct(), ints(5000)
    nb = L.aar_kv_cache_attn_workspace_bytes(ctypes.byref(c), 2, 1, EVERY, 0)
    assert nb > 0
    ws = torch.full((nb + 64,), 123, dtype=torch.uint8, device="cuda")
    o = pool.attend(L, q, lens, ws=ws)
    assert (ws[nb:] == 123).all()
    st = M.strides3(q, o)
    for p, n in ((None, nb), (ws.data_ptr(), nb - 1), (ws.data_ptr() + 4, nb)):
        assert L.aar_kv_cache_attn_f32(ctypes.byref(c), q.data_ptr(), o.data_ptr(), st, lens.data_ptr(), None, 2, 1, EVERY,
                                       0, 0.125, p, n, None, M.stream()) == M.EWORKSPACE


def test_pages_past_32_bits(L):
    """A pool of more than 4 GiB, its last page and its first in one sequence."""
    page, d, Hkv = 128, 128, 8
    per = L.aar_kv_cache_page_bytes(Hkv, page, d)
    n = (1 << 32) // per + 2
    pool = K.Pool(1, Hkv, d, page, 2, spare=0)
    pool.bytes = torch.empty(n * per, dtype=torch.uint8, device="cuda")
    pool.scales = torch.zeros(n, Hkv, 2, device="cuda")
    pool.n = n
    pool.table = ints(n - 1, 0).view(1, 2)
    k, v, q = rand(1, 1, Hkv, 200, d), rand(2, 1, Hkv, 200, d), rand(3, 1, Hkv, 1, d)
    pool.append(L, k, v, ints(200))
    check_read(L, pool, k, v, ints(200))
    ref = K.cache_exact(q, *held(k, v, (200,), page), [200], [1], EVERY, 0)
    M.near(pool.attend(L, q, ints(200)), ref, M.attn_tol(d, 200), "o")
