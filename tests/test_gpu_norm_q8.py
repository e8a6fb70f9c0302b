"""The 8-bit products and the norm's gates on the GPU against their definitions in
64-bit integers.  All results are ring words, so every comparison is of all bits."""
import ctypes as C

import numpy as np
import pytest

import mpcx
from test_gpu_transformer import dev, host, words

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


@pytest.fixture(scope="module", params=[32, 64])
def ctx(request):
    c = mpcx.Ctx(bw=request.param, scale=12)
    yield c
    c.close()


# ---------------- 8-bit weights ----------------
def q8_rows(w):
    """Weights (N, K) in -128..127 as rows of whole 16, the bytes past K arbitrary."""
    N, K = w.shape
    full = np.full((N, (K + 15) // 16 * 16), 77, np.int8)
    full[:, :K] = w
    return mpcx.to_dev(full.view(np.uint8)).view(_torch().int8)


def q8_plain(a, w, scale=None, tok=None):
    with np.errstate(over="ignore"):
        out = np.matmul(a.astype(np.uint64), w.T.astype(np.int64).astype(np.uint64))
        if scale is not None:
            out = out * scale.astype(np.int64).astype(np.uint64)
        if tok is not None:
            out = out * tok.astype(np.int64).astype(np.uint64)[:, None]
        return out.astype(a.dtype)


def steps(rng, n):
    s = rng.integers(-(1 << 31), 1 << 31, n).astype(np.int32)
    s[0], s[-1] = -(1 << 31), (1 << 31) - 1
    return s


# a token, few and many; rows, columns and sums one below, at and one past the tiles
Q8_SHAPES = [(1, 1, 1), (1, 15, 5), (1, 4096, 64), (1, 8192, 2047), (2, 16, 16), (3, 17, 17), (4, 128, 48), (5, 129, 33),
             (8, 1000, 200), (15, 127, 300), (16, 512, 130), (17, 257, 65), (31, 640, 16), (32, 64, 257), (33, 95, 1),
             (48, 2049, 63), (64, 312, 1024), (65, 1024, 129), (100, 160, 300), (127, 113, 255), (130, 300, 260),
             (257, 129, 31), (300, 384, 520), (513, 2100, 700)]


@pytest.mark.parametrize("M,K,N", Q8_SHAPES)
def test_q8(ctx, M, K, N):
    rng = np.random.default_rng(M * 7 + K * 3 + N)
    a, w = words(rng, (M, K), ctx.bw), rng.integers(-128, 128, (N, K))
    scale, tok = steps(rng, N), steps(rng, M)
    da, dq, ds, dt = dev(a), q8_rows(w), dev(scale), dev(tok)
    for s, t, x, y in ((ds, dt, scale, tok), (ds, None, scale, None), (None, dt, None, tok), (None, None, None, None)):
        assert np.array_equal(host(ctx.ring_gemm_q8(da, dq, s, t), ctx.bw), q8_plain(a, w, x, y))


@pytest.mark.parametrize("M", [1, 6, 40, 200])
@pytest.mark.parametrize("word", [0x8080808080808080, 0x7F7F7F7F7F7F7F7F, (1 << 64) - 1])
def test_q8_largest_sums(ctx, M, word):
    """Every digit and weight at its end over a K whose sums pass 31 bits."""
    K, N = 300001, 3
    w = np.full((N, K), -128, np.int8)
    w[1] = 127
    w[2, ::2] = 127
    a = np.full((M, K), word, np.uint64).astype(ctx.T)
    scale = np.array([-5, 1, 1 << 30], np.int32)
    got = host(ctx.ring_gemm_q8(dev(a), q8_rows(w), dev(scale)), ctx.bw)
    with np.errstate(over="ignore"):
        want = w.sum(1, dtype=np.int64).astype(np.uint64) * np.uint64(a[0, 0]) * scale.astype(np.int64).astype(np.uint64)
    assert np.array_equal(got, np.tile(want.astype(ctx.T), (M, 1)))


@pytest.mark.parametrize("M", [1, 3, 16, 37, 140])
def test_q8_rows_apart(ctx, M):
    """Operands inside larger arrays, activations one word off a 16-byte boundary; what is
    beside the output stays."""
    torch = _torch()
    rng = np.random.default_rng(M)
    K, N = 200, 77
    big, w = words(rng, (M, K + 13), ctx.bw), rng.integers(-128, 128, (N, K))
    wide = np.full((N, 256), -99, np.int8)
    wide[:, 16:16 + K] = w
    scale = rng.integers(-5000, 5000, N).astype(np.int32)
    to = torch.full((M, N + 9), 17, dtype=torch.int32 if ctx.bw == 32 else torch.int64, device="cuda")
    q = mpcx.to_dev(wide.view(np.uint8)).view(torch.int8)[:, 16:16 + K]
    ctx.ring_gemm_q8(dev(big)[:, 5:5 + K], q, dev(scale), out=to[:, 3:3 + N])
    got = host(to, ctx.bw)
    assert np.array_equal(got[:, 3:3 + N], q8_plain(big[:, 5:5 + K], w, scale))
    assert (got[:, :3] == 17).all() and (got[:, 3 + N:] == 17).all()


def q8_wide(a, w):
    """q8_plain without scales, by float64 products of 16-bit limbs: below 2^53, so exact."""
    wide = w.T.astype(np.float64)
    with np.errstate(over="ignore"):
        return sum((np.matmul((a >> a.dtype.type(16 * i) & a.dtype.type(0xFFFF)).astype(np.float64), wide).astype(np.int64)
                    .astype(np.uint64) << np.uint64(16 * i) for i in range(a.itemsize // 2)), np.uint64(0)).astype(a.dtype)


# rows and columns for which a small tile is 1, 2, 3, 4 times 64 columns wide and, with some
# steps of K, a large one 3 or 4 times; K one step, a few, a whole number, and past the last
@pytest.mark.parametrize("M,N", [(256, 4096), (384, 4096), (640, 4096), (1000, 4096), (320, 4096), (500, 4096), (20, 20000),
                                 (20, 40000), (20, 60000), (70, 20001), (17, 33000), (33, 33001)])
@pytest.mark.parametrize("K", [16, 127, 128, 130, 384, 500, 640, 769])
def test_q8_tiles(ctx, M, K, N):
    rng = np.random.default_rng(M + K)
    a, w = words(rng, (M, K), ctx.bw), rng.integers(-128, 128, (N, K)).astype(np.int8)
    assert np.array_equal(host(ctx.ring_gemm_q8(dev(a), q8_rows(w)), ctx.bw), q8_wide(a, w))


# more steps, by small and large tiles of each width, some with K in parts, most in one ring only
@pytest.mark.parametrize("M,K,N", [(1000, 1100, 4096), (640, 2049, 4096), (500, 2049, 4096), (320, 2049, 4096), (70, 4097, 2003),
                                   (34, 4046, 4406), (130, 8191, 1003), (33, 4082, 3369), (196, 8986, 2317), (1028, 7444, 587),
                                   (273, 4046, 208), (49, 8659, 4120), (715, 7163, 420), (568, 1969, 72)])
def test_q8_tiles_of_long_rows(ctx, M, K, N):
    rng = np.random.default_rng(N)
    a, w = words(rng, (M, K), ctx.bw), rng.integers(-128, 128, (N, K)).astype(np.int8)
    scale, tokens = steps(rng, N), steps(rng, M)
    with np.errstate(over="ignore"):
        want = q8_wide(a, w) * scale.astype(np.int64).astype(ctx.T) * tokens.astype(np.int64).astype(ctx.T)[:, None]
    assert np.array_equal(host(ctx.ring_gemm_q8(dev(a), q8_rows(w), dev(scale), dev(tokens)), ctx.bw), want)


# a few rows by many columns or a long K, by either kernel
@pytest.mark.parametrize("M", [1, 2, 3, 5, 8, 9, 16, 17, 24, 32])
@pytest.mark.parametrize("K,N", [(2048, 500), (4099, 4096), (8191, 2048), (130, 30001), (20001, 100), (2001, 4200), (3200, 4201), (9000, 2500),
                                 (4099, 4097), (1, 40), (2, 40), (3, 40), (4, 40), (5, 40), (7, 33)])
def test_q8_few_or_many(ctx, M, K, N):
    rng = np.random.default_rng(M * N)
    a, w = words(rng, (M, K), ctx.bw), rng.integers(-128, 128, (N, K)).astype(np.int8)
    assert np.array_equal(host(ctx.ring_gemm_q8(dev(a), q8_rows(w)), ctx.bw), q8_wide(a, w))


# K in parts: their sums added up in memory
@pytest.mark.parametrize("M,K,N", [(20, 8191, 300), (33, 4096, 100), (100, 4097, 500), (17, 20000, 20), (64, 1100, 64)])
def test_q8_parts_of_k(ctx, M, K, N):
    torch = _torch()
    rng = np.random.default_rng(K)
    a, w, scale = words(rng, (M, K), ctx.bw), rng.integers(-128, 128, (N, K)).astype(np.int8), steps(rng, N)
    to = torch.full((M, N + 5), 41, dtype=torch.int32 if ctx.bw == 32 else torch.int64, device="cuda")
    for _ in range(2):  # the output is not added to
        ctx.ring_gemm_q8(dev(a), q8_rows(w), dev(scale), out=to[:, 2:2 + N])
        got = host(to, ctx.bw)
        with np.errstate(over="ignore"):
            assert np.array_equal(got[:, 2:2 + N], q8_wide(a, w) * scale.astype(np.int64).astype(ctx.T))
        assert (got[:, :2] == 41).all() and (got[:, 2 + N:] == 41).all()


def test_q8_long_sums_of_a_token(ctx):
    """One token, a K past what a wave sums in 32 bits."""
    K, N = (1 << 21) + 5, 3
    w = np.full((N, K), -128, np.int8)
    w[1, 7::2] = 127
    a = np.full((1, K), 0x8080808080808080, np.uint64).astype(ctx.T)
    got = host(ctx.ring_gemm_q8(dev(a), q8_rows(w)), ctx.bw)
    with np.errstate(over="ignore"):
        assert np.array_equal(got[0], w.sum(1, dtype=np.int64).astype(np.uint64).astype(ctx.T) * a[0, 0])


@pytest.mark.parametrize("M", [1, 2, 5, 20])
def test_q8_rows_far_apart(ctx, M):
    """Rows and weights further apart than a workgroup's 32-bit places reach."""
    torch = _torch()
    rng = np.random.default_rng(M)
    K, N, ld, ldq = 40, 3, 1 << 24, 1 << 23
    a, w = words(rng, (M, K), ctx.bw), rng.integers(-128, 128, (N, K)).astype(np.int8)
    big = torch.empty(((M - 1) * ld + K,), dtype=torch.int32 if ctx.bw == 32 else torch.int64, device="cuda")
    wide = torch.empty(((N - 1) * ldq + 48,), dtype=torch.int8, device="cuda")
    x, q = big.as_strided((M, K), (ld, 1)), wide.as_strided((N, K), (ldq, 1))
    x.copy_(dev(a))
    q.copy_(q8_rows(w)[:, :K])
    torch.cuda.synchronize()
    assert np.array_equal(host(ctx.ring_gemm_q8(x, q), ctx.bw), q8_plain(a, w))


@pytest.mark.parametrize("M", [5, 16, 20, 40])
def test_q8_rows_as_far_apart_as_a_workgroup_reaches(ctx, M):
    """Rows and weights one place nearer than that."""
    torch = _torch()
    rng = np.random.default_rng(M)
    K, N, ld, ldq = 140, 20, (1 << 24) - 1, (1 << 23) - 16
    a, w = words(rng, (M, K), ctx.bw), rng.integers(-128, 128, (N, K)).astype(np.int8)
    big = torch.empty(((M - 1) * ld + K,), dtype=torch.int32 if ctx.bw == 32 else torch.int64, device="cuda")
    wide = torch.empty(((N - 1) * ldq + 144,), dtype=torch.int8, device="cuda")
    x, q = big.as_strided((M, K), (ld, 1)), wide.as_strided((N, K), (ldq, 1))
    x.copy_(dev(a))
    q.copy_(q8_rows(w)[:, :K])
    torch.cuda.synchronize()
    assert np.array_equal(host(ctx.ring_gemm_q8(x, q), ctx.bw), q8_plain(a, w))


def test_q8_padding_tokens(ctx):
    """A token scale of zero clears its row, the others stay."""
    rng = np.random.default_rng(8)
    a, w = words(rng, (20, 96), ctx.bw), rng.integers(-128, 128, (40, 96))
    tok = np.where(np.arange(20) % 3 == 2, 0, 7).astype(np.int32)
    got = host(ctx.ring_gemm_q8(dev(a), q8_rows(w), None, dev(tok)), ctx.bw)
    assert np.array_equal(got, q8_plain(a, w, None, tok)) and not got[2::3].any()


def test_q8_no_token(ctx):
    out = ctx.ring_gemm_q8(dev(words(np.random.default_rng(0), (0, 32), ctx.bw)), q8_rows(np.ones((4, 32), np.int8)))
    assert out.shape == (0, 4)


# ---------------- the norm's gates ----------------
NORM_SHAPES = [(1, 1), (1, 64), (1, 4096), (1, 70001), (2, 63), (3, 65), (5, 129), (7, 1000), (16, 256), (37, 1279),
               (64, 312), (130, 2048), (600, 96), (1025, 33), (3000, 4), (2, 32768), (3, 49155), (64, 32769)]


def up(n):
    return (n + 255) // 256 * 256


def key_planes(k, T, first, second):
    tb = np.dtype(T).itemsize
    raw = k.cpu().numpy().view(np.uint8)
    at = up(first * tb)
    return raw[:first * tb].view(T), raw[at:at + second * tb].view(T)


def two(T):
    return T(2)


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("rows,dim", NORM_SHAPES)
def test_norm_sums(ctx, rows, dim, residual):
    """Keys, the sums from them, and each party's message."""
    rng = np.random.default_rng(rows * 3 + dim + residual)
    rx, x = words(rng, (rows, dim), ctx.bw), words(rng, (rows, dim), ctx.bw)
    rd, d = (words(rng, (rows, dim), ctx.bw), words(rng, (rows, dim), ctx.bw)) if residual else (None, None)
    k0, k1, rh, rs = ctx.norm_sums_keygen(dev(rx), dev(rd) if residual else None, seed=9, gate=5)
    rh, rs = host(rh, ctx.bw), host(rs, ctx.bw)
    (a0, c0), (a1, c1) = (key_planes(k, ctx.T, rows * dim, rows) for k in (k0, k1))
    with np.errstate(over="ignore"):
        assert np.array_equal(rh, rx + rd if residual else rx)
        assert np.array_equal((a0 + a1).reshape(rows, dim), rh)
        assert np.array_equal(c0 + c1, rs + np.square(rh).sum(1, dtype=ctx.T))
        h = x + d if residual else x
        want = np.square(h).sum(1, dtype=ctx.T)
        hhat, xhat = h + rh, dev(x + rx)
        dhat = dev(d + rd) if residual else None
    before = ctx.bytes_exchanged, ctx.rounds
    got_h, got = ctx.norm_sums_eval(k0, k1, xhat, dhat)
    assert (ctx.bytes_exchanged - before[0], ctx.rounds - before[1]) == (2 * rows * ctx.bw // 8, 1)
    assert np.array_equal(host(got_h, ctx.bw), hhat)
    with np.errstate(over="ignore"):
        assert np.array_equal(host(got, ctx.bw) - rs, want)
        total = 0
        for p, key in enumerate((k0, k1)):
            hp, m = ctx.norm_sums_message(p, key, xhat, dhat)
            a, c = (a0, a1)[p].reshape(rows, dim), (c0, c1)[p]
            own = (hhat * (hhat - two(ctx.T) * a)).sum(1, dtype=ctx.T) if p == 0 else \
                np.zeros(rows, ctx.T) - two(ctx.T) * (hhat * a).sum(1, dtype=ctx.T)
            assert np.array_equal(host(m, ctx.bw), own + c)
            assert np.array_equal(host(hp, ctx.bw), hhat)
            total = total + host(m, ctx.bw)
        assert np.array_equal(total, host(got, ctx.bw))


@pytest.mark.parametrize("gain", [True, False])
@pytest.mark.parametrize("rows,dim", NORM_SHAPES)
def test_norm_scale(ctx, rows, dim, gain):
    rng = np.random.default_rng(rows * 5 + dim + gain)
    rh, h = words(rng, (rows, dim), ctx.bw), words(rng, (rows, dim), ctx.bw)
    rv, v = words(rng, (rows,), ctx.bw), words(rng, (rows,), ctx.bw)
    g = words(rng, (dim,), ctx.bw) if gain else np.ones(dim, ctx.T)
    s0, s1, _, _ = ctx.norm_sums_keygen(dev(rh), seed=4, gate=1)
    dg = dev(g) if gain else None
    k0, k1, ry = ctx.norm_scale_keygen(s0, s1, dev(rv), dim, dg, seed=4, gate=2)
    ry = host(ry, ctx.bw)
    a0, a1 = (key_planes(k, ctx.T, rows * dim, rows)[0].reshape(rows, dim) for k in (s0, s1))
    (b0, c0), (b1, c1) = (key_planes(k, ctx.T, rows, rows * dim) for k in (k0, k1))
    with np.errstate(over="ignore"):
        assert np.array_equal(b0 + b1, rv)
        assert np.array_equal((c0 + c1).reshape(rows, dim), ry + g * (rh * rv[:, None] - a0 * b0[:, None]))
        hhat, vhat, want = h + rh, v + rv, g * h * v[:, None]
    before = ctx.bytes_exchanged, ctx.rounds
    got = host(ctx.norm_scale_eval(k0, k1, s0, s1, dev(hhat), dev(vhat), dg), ctx.bw)
    assert (ctx.bytes_exchanged - before[0], ctx.rounds - before[1]) == (2 * rows * dim * ctx.bw // 8, 1)
    with np.errstate(over="ignore"):
        assert np.array_equal(got - ry, want)
        m0 = host(ctx.norm_scale_message(0, k0, s0, dev(hhat), dev(vhat), dg), ctx.bw)
        m1 = host(ctx.norm_scale_message(1, k1, s1, dev(hhat), dev(vhat), dg), ctx.bw)
        assert np.array_equal(m0, g * (hhat - a0) * (vhat - b0)[:, None] + c0.reshape(rows, dim))
        assert np.array_equal(m1, c1.reshape(rows, dim) - g * (hhat * b1[:, None] + a1 * vhat[:, None]))
        assert np.array_equal(m0 + m1, got)


@pytest.mark.parametrize("rows,dim", [(9, 200), (130, 1024), (3, 5000)])
def test_norm_in_place_and_apart(ctx, rows, dim):
    """Rows as columns of larger matrices, one word off a 16-byte boundary, and outputs in
    their inputs' place: the same words, and what is beside them stays."""
    torch = _torch()
    rng = np.random.default_rng(dim)
    x, d, v = words(rng, (rows, dim), ctx.bw), words(rng, (rows, dim), ctx.bw), dev(words(rng, (rows,), ctx.bw))
    k0, k1, _, _ = ctx.norm_sums_keygen(dev(x), dev(d), seed=2)
    q0, q1, _ = ctx.norm_scale_keygen(k0, k1, v, dim, None, seed=3)
    h, s = ctx.norm_sums_eval(k0, k1, dev(x), dev(d))
    y = ctx.norm_scale_eval(q0, q1, k0, k1, h, v)
    h, s, y = (host(t, ctx.bw) for t in (h, s, y))

    def wide(a):
        t = torch.full((rows, dim + 11), 23, dtype=torch.int32 if ctx.bw == 32 else torch.int64, device="cuda")
        t[:, 3:3 + dim] = dev(a)
        return t, t[:, 3:3 + dim]

    for place in ("apart", "x", "d"):
        (bx, vx), (bd, vd), (bo, vo) = wide(x), wide(d), wide(x)
        to = {"apart": vo, "x": vx, "d": vd}[place]
        got_h, got_s = ctx.norm_sums_eval(k0, k1, vx, vd, out=to)
        assert got_h is to and np.array_equal(host(to, ctx.bw), h) and np.array_equal(host(got_s, ctx.bw), s)
        (by, vy) = wide(x)
        for dest in (vy, to):
            ctx.norm_scale_eval(q0, q1, k0, k1, to, v, out=dest)
            assert np.array_equal(host(dest, ctx.bw), y)
        for b in (bx, bd, bo, by):
            e = host(b, ctx.bw)
            assert (e[:, :3] == 23).all() and (e[:, 3 + dim:] == 23).all()


def test_norm_no_row(ctx):
    z = dev(np.zeros((0, 8), ctx.T))
    before = ctx.rounds
    k0, k1, rh, rs = ctx.norm_sums_keygen(z, z)
    h, s = ctx.norm_sums_eval(k0, k1, z, z)
    q0, q1, ry = ctx.norm_scale_keygen(k0, k1, rs, 8)
    y = ctx.norm_scale_eval(q0, q1, k0, k1, h, s)
    assert h.shape == y.shape == ry.shape == (0, 8) and s.shape == (0,) and ctx.rounds == before


def test_norm_keys_differ_by_gate(ctx):
    """The shares are pseudorandom: another gate id or seed, other keys."""
    r = dev(words(np.random.default_rng(1), (4, 40), ctx.bw))
    keys = [ctx.norm_sums_keygen(r, seed=s, gate=g)[0].cpu().numpy() for s, g in ((1, 1), (1, 2), (2, 1))]
    assert not any(np.array_equal(a[:160], b[:160]) for a, b in ((keys[0], keys[1]), (keys[0], keys[2])))


def test_norm_gates_of_one_id(ctx):
    """The two gates of a norm under one seed and gate id, as the defaults give them, and the other
    gates' masks and shares under the same: no two draw the same words."""
    rng = np.random.default_rng(3)
    rows, dim = 40, 3
    r, rv = dev(words(rng, (rows, dim), ctx.bw)), dev(words(rng, (rows,), ctx.bw))
    k0, k1, _, rs = ctx.norm_sums_keygen(r)
    q0, _, ry = ctx.norm_scale_keygen(k0, k1, rv, dim)
    drawn = [*key_planes(k0, ctx.T, rows * dim, rows), host(rs, ctx.bw), *key_planes(q0, ctx.T, rows, rows * dim),
             host(ry, ctx.bw).reshape(-1), host(ctx.split_mask(rv)[0], ctx.bw),
             host(ctx.gate_keygen(mpcx.TR, rv)[2], ctx.bw)]
    first = [tuple(d[:rows].tolist()) for d in drawn]
    assert len(set(first)) == len(first)
    q0, _, ry = ctx.norm_scale_keygen(k0, k1, rv, dim, gate=2)  # another id, other words
    again = [host(ry, ctx.bw).reshape(-1), *key_planes(q0, ctx.T, rows, rows * dim)]
    assert not set(first) & {tuple(d[:rows].tolist()) for d in again}
