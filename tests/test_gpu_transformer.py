"""The transformer operators on the GPU against their definitions in 64-bit
integers: products with 4-bit weights, the paged cache, and the two attention
gates (values, keys, single parties' messages).  All results are ring words, so
every comparison is of all bits."""
import ctypes as C

import numpy as np
import pytest

import mpcx

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


def dev(a):
    """uint32 / uint64 words as the int tensor that holds them."""
    return mpcx.to_dev(np.ascontiguousarray(a)).reshape(a.shape)


def host(t, bw):
    return t.cpu().numpy().view(np.uint32 if bw == 32 else np.uint64)


def words(rng, shape, bw):
    """Ring words, the ends of the digits' and the ring's ranges among them."""
    x = rng.integers(0, 1 << 64, shape, dtype=np.uint64)
    ends = np.array([0, 1, (1 << 64) - 1, 1 << 63, (1 << 63) - 1, 0x7F7F7F7F7F7F7F7F, 0x8080808080808080,
                     0x7F7F7F7F80808080, 0xFF80FF80FF80FF80], np.uint64)
    at = rng.random(shape) < 0.1
    x[at] = ends[rng.integers(0, ends.size, int(at.sum()))]
    return x.astype(np.uint32) if bw == 32 else x


@pytest.fixture(scope="module", params=[32, 64])
def ctx(request):
    c = mpcx.Ctx(bw=request.param, scale=12)
    yield c
    c.close()


# ---------------- 4-bit weights ----------------
def q4_pack(w):
    """Weights (N, K) in -8..7 as rows of whole 32, the halves past K arbitrary."""
    N, K = w.shape
    full = np.full((N, (K + 31) // 32 * 32), 5, np.int64)
    full[:, :K] = w
    full &= 15
    return (full[:, 0::2] | full[:, 1::2] << 4).astype(np.uint8)


def q4_plain(a, w, scale, group):
    a = a.astype(np.uint64)
    out = np.zeros((a.shape[0], w.shape[0]), np.uint64)
    for g in range(scale.shape[0]):
        k = slice(g * group, (g + 1) * group)
        out += np.matmul(a[:, k], w[:, k].T.astype(np.uint64)) * scale[g].astype(np.int64).astype(np.uint64)
    return out


Q4_SHAPES = [(1, 1, 1, 32), (1, 31, 5, 32), (1, 4096, 64, 128), (2, 32, 16, 32), (3, 33, 17, 32), (4, 128, 48, 64),
             (5, 129, 33, 128), (8, 1000, 200, 96), (16, 512, 130, 64), (17, 257, 65, 128), (31, 640, 16, 640),
             (33, 95, 1, 32), (64, 312, 1024, 32), (65, 1024, 129, 256), (100, 160, 300, 160), (130, 300, 260, 64),
             (257, 129, 31, 4096), (300, 384, 520, 128)]


@pytest.mark.parametrize("M,K,N,group", Q4_SHAPES)
def test_q4(ctx, M, K, N, group):
    rng = np.random.default_rng(M * 7 + K * 3 + N)
    a, w = words(rng, (M, K), ctx.bw), rng.integers(-8, 8, (N, K))
    scale = rng.integers(-(1 << 31), 1 << 31, (-(-K // group), N)).astype(np.int32)
    scale.flat[0], scale.flat[-1] = -(1 << 31), (1 << 31) - 1
    got = host(ctx.ring_gemm_q4(dev(a), dev(q4_pack(w)), dev(scale), group), ctx.bw)
    assert np.array_equal(got, q4_plain(a, w, scale, group).astype(ctx.T))


@pytest.mark.parametrize("M", [1, 40])
@pytest.mark.parametrize("word", [0x8080808080808080, 0x7F7F7F7F7F7F7F7F, (1 << 64) - 1])
def test_q4_largest_sums(ctx, M, word):
    """Every digit and weight at its end, one group over all of a long K."""
    K, N, group = 140000, 3, 160000
    a = np.full((M, K), word, np.uint64).astype(ctx.T)
    w = np.full((N, K), -8)
    w[1] = 7
    w[2, ::2] = 7
    scale = np.array([[-5, 1, 1 << 30]], np.int32)
    got = host(ctx.ring_gemm_q4(dev(a), dev(q4_pack(w)), dev(scale), group), ctx.bw)
    with np.errstate(over="ignore"):
        want = (w.sum(1).astype(np.uint64) * np.uint64(a[0, 0]) * scale[0].astype(np.int64).astype(np.uint64))
    assert np.array_equal(got, np.tile(want.astype(ctx.T), (M, 1)))


@pytest.mark.parametrize("M", [2, 37, 140])
def test_q4_rows_apart(ctx, M):
    """Operands inside larger arrays, one word off a 16-byte boundary; what is
    beside the output stays."""
    torch = _torch()
    rng = np.random.default_rng(M)
    K, N, group = 200, 77, 64
    big, w = words(rng, (M, K + 13), ctx.bw), rng.integers(-8, 8, (N, K))
    scale = rng.integers(-5000, 5000, (-(-K // group), N)).astype(np.int32)
    to = torch.full((M, N + 9), 17, dtype=torch.int32 if ctx.bw == 32 else torch.int64, device="cuda")
    ctx.ring_gemm_q4(dev(big)[:, 5:5 + K], dev(q4_pack(w)), dev(scale), group, out=to[:, 3:3 + N])
    got = host(to, ctx.bw)
    assert np.array_equal(got[:, 3:3 + N], q4_plain(big[:, 5:5 + K], w, scale, group).astype(ctx.T))
    assert (got[:, :3] == 17).all() and (got[:, 3 + N:] == 17).all()


# ---------------- the cache ----------------
def rotate_plain(x, cos, sin, shift, pairs):
    """x (tokens, heads, dim), tables (tokens, half)."""
    h = cos.shape[1]
    y = x << np.uint64(shift).astype(x.dtype)
    i = np.arange(h)
    u, v = (2 * i, 2 * i + 1) if pairs else (i, i + h)
    c, s = cos[:, None], sin[:, None]
    y[..., u] = c * x[..., u] - s * x[..., v]
    y[..., v] = s * x[..., u] + c * x[..., v]
    return y


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,half,page,planes,extra", [
    (1, 1, 2, 1, 1, 1, 0), (1, 8, 128, 64, 16, 6, 0), (7, 3, 5, 2, 4, 2, 3), (40, 2, 72, 36, 24, 6, 8),
    (33, 4, 80, 20, 16, 8, 1), (5, 2, 64, 3, 1, 3, 64), (300, 1, 96, 48, 256, 4, 0)])
def test_cache_append(ctx, tokens, heads, dim, half, page, planes, extra, pairs):
    rng = np.random.default_rng(tokens + dim + planes)
    n_pages, n_pos, shift = -(-tokens // page) + 2, 50, 11
    rows = [words(rng, (tokens, heads * dim + extra), ctx.bw) for _ in range(planes)]
    pools = [words(rng, (n_pages, heads, page, dim), ctx.bw) for _ in range(planes)]
    cos, sin = words(rng, (n_pos, half), ctx.bw), words(rng, (n_pos, half), ctx.bw)
    slot = rng.permutation(n_pages * page)[:tokens].astype(np.int64)
    pos = rng.integers(0, n_pos, tokens).astype(np.int32)
    if tokens > 4:  # padding, slots past the cache, positions outside the tables
        slot[1], slot[2] = -1, n_pages * page
        pos[3], pos[4] = n_pos, -1
    want = [p.copy() for p in pools]
    for i in range(planes):
        x = rows[i][:, extra:].reshape(tokens, heads, dim)
        y = rotate_plain(x, cos[np.clip(pos, 0, n_pos - 1)], sin[np.clip(pos, 0, n_pos - 1)], shift, pairs)
        for t in range(tokens):
            if not 0 <= slot[t] < n_pages * page or (i % 2 == 0 and not 0 <= pos[t] < n_pos):
                continue
            want[i][slot[t] // page, :, slot[t] % page] = (y if i % 2 == 0 else x)[t]
    d = [dev(p) for p in pools]
    ctx.cache_append([(dev(r)[:, extra:].unflatten(1, (heads, dim)), p, i % 2 == 0) for i, (r, p) in
                      enumerate(zip(rows, d))], dev(slot), dev(pos), mpcx.Rotation(dev(cos), dev(sin), shift, pairs))
    for w, p in zip(want, d):
        assert np.array_equal(host(p, ctx.bw), w)


def test_cache_append_without_rotation(ctx):
    rng = np.random.default_rng(4)
    rows, pool = words(rng, (9, 2, 7), ctx.bw), words(rng, (3, 2, 5, 7), ctx.bw)
    slot = np.array([0, 14, 3, 9, -5, 7, 1 << 40, 8, 2], np.int64)
    d = dev(pool)
    ctx.cache_append([(dev(rows), d, False)], dev(slot))
    for t, s in enumerate(slot):
        if 0 <= s < 15:
            pool[s // 5, :, s % 5] = rows[t]
    assert np.array_equal(host(d, ctx.bw), pool)
    ctx.cache_append([(dev(rows)[:0], d, False)], dev(slot)[:0])  # no token
    assert np.array_equal(host(d, ctx.bw), pool)


# ---------------- the attention gates ----------------
class Batch:
    """A random batch, its cache (masked rows, shares) and the plain products."""

    def __init__(self, bw, seqs, q, keys, heads, kv, dim, page, mask, seed=0, gap=0):
        rng = self.rng = np.random.default_rng(seed + seqs * 131 + q * 17 + keys + heads + dim + page)
        self.bw, self.heads, self.kv, self.dim, self.page = bw, heads, kv, dim, page
        nq, nk = [], []
        for b in range(seqs):
            n = q if b == 0 else int(rng.integers(0, q + 1))  # a sequence may have no token
            nq.append(n)
            nk.append(keys if b == 0 else int(rng.integers(max(n, 1), max(keys, n, 1) + 1)))
        self.seq = np.repeat(np.arange(seqs), nq)
        self.tokens = self.seq.size
        self.qstart = np.concatenate([[0], np.cumsum(nq)]).astype(np.int32)
        at = np.arange(self.tokens) - self.qstart[self.seq]
        self.pos = (np.array(nk)[self.seq] - np.array(nq)[self.seq] + at).astype(np.int32)
        self.lo, self.hi = np.zeros(self.tokens, np.int32), self.pos + 1
        if mask == "prefix":
            self.hi = np.maximum(self.hi, np.array(nk)[self.seq] // 2)
        elif mask == "window":
            self.lo = np.maximum(0, self.hi - max(1, keys // 3)).astype(np.int32)
        elif mask == "ragged":  # any range, empty and reversed ones among them
            self.lo = rng.integers(0, np.array(nk)[self.seq] + 1).astype(np.int32)
            self.hi = rng.integers(0, np.array(nk)[self.seq] + 1).astype(np.int32)
        self.hi = self.hi.astype(np.int32)
        width = np.maximum(0, self.hi.astype(np.int64) - self.lo)
        order = rng.permutation(self.tokens) if gap else np.arange(self.tokens)  # blocks in any order, apart
        self.off = np.zeros(self.tokens, np.int64)
        end = gap
        for t in order:
            self.off[t] = end
            end += heads * int(width[t]) + gap
        self.n = end
        used = [-(-k // page) for k in nk]
        self.n_pages = sum(used) + 3
        perm = rng.permutation(self.n_pages)
        self.table = np.full((seqs, max(used) + 1), -1, np.int32)
        done = 0
        for b, u in enumerate(used):
            self.table[b, :u] = perm[done:done + u]
            done += u
        shape = (self.n_pages, kv, page, dim)
        self.y, self.b0, self.b1 = (words(rng, shape, bw) for _ in range(3))
        self.max_q, self.max_keys = max(max(nq), 1), max(nk)

    def gpu(self):
        return mpcx.AttnBatch(dev(self.table), dev(self.qstart), dev(self.lo), dev(self.hi), dev(self.off), self.n,
                              self.heads, self.max_q, self.max_keys)

    def lines(self, plane):
        """Rows of a sequence, head by head (pages outside the cache: zeros)."""
        out = np.zeros((self.table.shape[0], self.kv, self.table.shape[1] * self.page, self.dim), plane.dtype)
        for b, row in enumerate(self.table):
            for i, p in enumerate(row):
                if 0 <= p < self.n_pages:
                    out[b, :, i * self.page:(i + 1) * self.page] = plane[p]
        return out

    def blocks(self):
        """(token, head, words of its block) that see something."""
        m = self.heads // self.kv
        for t in range(self.tokens):
            w = int(self.hi[t]) - int(self.lo[t])
            if w <= 0:
                continue
            for h in range(self.heads):
                o = int(self.off[t]) + h * w
                yield t, h, h // m, slice(o, o + w)

    def scores(self, x, y):
        """The plain products of queries x and a plane y, zero outside the blocks."""
        out = np.zeros(self.n, x.dtype)
        ln = self.lines(y)
        for t, h, k, o in self.blocks():
            out[o] = ln[self.seq[t], k, self.lo[t]:self.hi[t]] @ x[t, h]
        return out

    def mix(self, p, y):
        out = np.zeros((self.tokens, self.heads, self.dim), p.dtype)
        ln = self.lines(y)
        for t, h, k, o in self.blocks():
            out[t, h] = p[o] @ ln[self.seq[t], k, self.lo[t]:self.hi[t]]
        return out

    def bias(self, slope):
        out = np.zeros(self.n, slope.dtype)
        for t, h, _, o in self.blocks():
            out[o] = slope[h] * (np.arange(self.lo[t], self.hi[t]) - self.pos[t]).astype(slope.dtype)
        return out

    def inside(self):
        m = np.zeros(self.n, bool)
        for *_, o in self.blocks():
            m[o] = True
        return m


ATTN = [
    # seqs, q, keys, heads, kv, dim, page, mask
    (1, 1, 1, 1, 1, 1, 1, "causal"), (1, 1, 2, 2, 1, 3, 1, "causal"), (1, 1, 500, 8, 8, 64, 16, "causal"),
    (3, 1, 333, 8, 2, 128, 64, "window"), (2, 1, 70, 17, 1, 16, 7, "causal"), (5, 2, 40, 6, 3, 20, 16, "ragged"),
    (1, 1, 1500, 4, 1, 72, 16, "causal"), (2, 33, 33, 4, 2, 64, 16, "causal"), (3, 20, 65, 5, 1, 80, 24, "prefix"),
    (1, 130, 130, 2, 2, 33, 32, "window"), (4, 19, 40, 3, 3, 96, 1, "ragged"), (1, 70, 200, 16, 2, 130, 256, "causal"),
    (2, 9, 17, 40, 8, 8, 5, "prefix"), (1, 4, 100, 4, 4, 300, 16, "ragged")]


@pytest.mark.parametrize("seqs,q,keys,heads,kv,dim,page,mask", ATTN)
@pytest.mark.parametrize("gap", [0, 3])
def test_attn_scores(ctx, seqs, q, keys, heads, kv, dim, page, mask, gap):
    """Values, keygen and both messages of the scores gate."""
    B = Batch(ctx.bw, seqs, q, keys, heads, kv, dim, page, mask, gap=gap)
    rq, qhat = words(B.rng, (B.tokens, heads, dim), ctx.bw), words(B.rng, (B.tokens, heads, dim), ctx.bw)
    slope = words(B.rng, (heads,), ctx.bw) if gap else None
    g, planes = B.gpu(), [dev(v) for v in (B.y, B.b0, B.b1)]
    k0, k1, rs = ctx.attn_scores_keygen(g, dev(rq), planes[1], planes[2], seed=3, gate=9)
    rs = host(rs, ctx.bw)
    extra = dict(slope=dev(slope), pos=dev(B.pos)) if gap else {}
    got = host(ctx.attn_scores_eval(g, k0, k1, dev(qhat), *planes, **extra), ctx.bw)
    with np.errstate(over="ignore"):
        want = B.scores(qhat - rq, B.y - B.b0 - B.b1) + rs + (B.bias(slope) if gap else 0)
        m = B.inside()
        assert np.array_equal(got[m], want[m])
        parts = [host(ctx.attn_scores_message(p, g, k, dev(qhat), planes[0], planes[1 + p], **extra), ctx.bw)
                 for p, k in ((0, k0), (1, k1))]
        assert np.array_equal((parts[0] + parts[1])[m], want[m])
        # party 0's message from its own key alone
        tb = ctx.bw // 8
        key = k0.cpu().numpy()
        n = rq.size
        a0 = key[:n * tb].view(ctx.T).reshape(rq.shape)
        at = (n * tb + 255) // 256 * 256
        c0 = key[at:at + B.n * tb].view(ctx.T)
        want0 = B.scores(qhat - a0, B.y - B.b0) + c0 + (B.bias(slope) if gap else 0)
        assert np.array_equal(parts[0][m], want0[m])
        if rs.size >= 32:  # a mask, not zeros
            assert np.unique(rs).size > rs.size // 2


@pytest.mark.parametrize("seqs,q,keys,heads,kv,dim,page,mask", ATTN)
@pytest.mark.parametrize("gap", [0, 3])
def test_attn_mix(ctx, seqs, q, keys, heads, kv, dim, page, mask, gap):
    B = Batch(ctx.bw, seqs, q, keys, heads, kv, dim, page, mask, seed=5, gap=gap)
    rp, phat = words(B.rng, (B.n,), ctx.bw), words(B.rng, (B.n,), ctx.bw)
    g, planes = B.gpu(), [dev(v) for v in (B.y, B.b0, B.b1)]
    k0, k1, ro = ctx.attn_mix_keygen(g, dev(rp), planes[1], planes[2], seed=4, gate=2)
    got = host(ctx.attn_mix_eval(g, k0, k1, dev(phat), *planes), ctx.bw)
    with np.errstate(over="ignore"):
        want = B.mix(phat - rp, B.y - B.b0 - B.b1) + host(ro, ctx.bw)
        assert np.array_equal(got, want)
        parts = [host(ctx.attn_mix_message(p, g, k, dev(phat), planes[0], planes[1 + p]), ctx.bw)
                 for p, k in ((0, k0), (1, k1))]
        assert np.array_equal(parts[0] + parts[1], want)


def test_attn_long_range(ctx):
    """Sums over more keys than the digit sums hold at once, digits at their ends."""
    n, dim = 70000, 24
    B = Batch(ctx.bw, 1, 1, n, 2, 1, dim, 64, "causal")
    top = np.uint64(0x8080808080808080).astype(ctx.T)
    B.y[:], B.b0[:], B.b1[:] = top, 0, top
    phat, rp = np.full(B.n, top), words(B.rng, (B.n,), ctx.bw)
    g, planes = B.gpu(), [dev(v) for v in (B.y, B.b0, B.b1)]
    k0, k1, ro = ctx.attn_mix_keygen(g, dev(rp), planes[1], planes[2])
    got = host(ctx.attn_mix_eval(g, k0, k1, dev(phat), *planes), ctx.bw)
    with np.errstate(over="ignore"):
        assert np.array_equal(got, B.mix(phat - rp, B.y - B.b0 - B.b1) + host(ro, ctx.bw))
        q, rq = np.full((1, 2, dim), top), words(B.rng, (1, 2, dim), ctx.bw)
        k0, k1, rs = ctx.attn_scores_keygen(g, dev(rq), planes[1], planes[2])
        got = host(ctx.attn_scores_eval(g, k0, k1, dev(q), *planes), ctx.bw)
        assert np.array_equal(got, B.scores(q - rq, B.y - B.b0 - B.b1) + host(rs, ctx.bw))


def test_attn_ranges_outside_see_nothing(ctx):
    """Ranges that leave the page row and blocks that leave the scores are taken
    as empty; page numbers outside the cache read as zeros; nothing else is
    written."""
    torch = _torch()
    B = Batch(ctx.bw, 1, 6, 30, 2, 1, 16, 8, "causal")
    width = B.table.shape[1] * B.page
    B.lo[0] = -1
    B.hi[1] = width + 1
    B.off[2] = -1
    B.off[3] = B.n - 5
    B.off[4] = 1 << 62
    g, planes = B.gpu(), [dev(v) for v in (B.y, B.b0, B.b1)]
    x = words(B.rng, (6, 2, 16), ctx.bw)
    k0, k1, rs = ctx.attn_scores_keygen(g, dev(x), planes[1], planes[2])
    word = torch.int32 if ctx.bw == 32 else torch.int64
    out = torch.full((B.n,), 99, dtype=word, device="cuda")
    a = ctx._attn(g, planes[0])
    torch.cuda.synchronize()
    xd = dev(x)
    ctx.check(ctx.lib.mpcx_attn_scores_eval(ctx.h, C.byref(a), k0.data_ptr(), k1.data_ptr(), xd.data_ptr(),
                                            *[p.data_ptr() for p in planes], None, None, out.data_ptr()), "eval")
    ctx.sync()
    got = host(out, ctx.bw)
    for t in range(5):
        B.lo[t] = B.hi[t] = 0
    with np.errstate(over="ignore"):
        want = B.scores(x - x, B.y) + host(rs, ctx.bw)
    m = B.inside()
    assert m.sum() > 0 and np.array_equal(got[m], want[m]) and (got[~m] == 99).all()
    p = words(B.rng, (B.n,), ctx.bw)
    k0, k1, ro = ctx.attn_mix_keygen(g, dev(np.zeros(B.n, ctx.T)), planes[1], planes[2])
    got = host(ctx.attn_mix_eval(g, k0, k1, dev(p), *planes), ctx.bw)
    with np.errstate(over="ignore"):
        assert np.array_equal(got, B.mix(p, B.y - B.b0 - B.b1) + host(ro, ctx.bw))


def test_attn_pages_outside_read_as_zeros(ctx):
    B = Batch(ctx.bw, 1, 5, 60, 4, 2, 40, 8, "causal")
    B.table[0, 1], B.table[0, 3] = -7, B.n_pages
    g, planes = B.gpu(), [dev(v) for v in (B.y, B.b0, B.b1)]
    rng = B.rng
    q, p = words(rng, (5, 4, 40), ctx.bw), words(rng, (B.n,), ctx.bw)
    zq, zp = np.zeros_like(q), np.zeros_like(p)
    with np.errstate(over="ignore"):
        k0, k1, rs = ctx.attn_scores_keygen(g, dev(zq), planes[1], planes[2])
        got = host(ctx.attn_scores_eval(g, k0, k1, dev(q), *planes), ctx.bw)
        assert np.array_equal(got, B.scores(q, B.y - B.b0 - B.b1) + host(rs, ctx.bw))
        k0, k1, ro = ctx.attn_mix_keygen(g, dev(zp), planes[1], planes[2])
        got = host(ctx.attn_mix_eval(g, k0, k1, dev(p), *planes), ctx.bw)
        assert np.array_equal(got, B.mix(p, B.y - B.b0 - B.b1) + host(ro, ctx.bw))


def test_launch_hints_do_not_change_results(ctx):
    B = Batch(ctx.bw, 3, 40, 90, 4, 2, 48, 16, "prefix")
    planes = [dev(v) for v in (B.y, B.b0, B.b1)]
    q, p = dev(words(B.rng, (B.tokens, 4, 48), ctx.bw)), dev(words(B.rng, (B.n,), ctx.bw))
    ks = ctx.attn_scores_keygen(B.gpu(), q, planes[1], planes[2])
    km = ctx.attn_mix_keygen(B.gpu(), p, planes[1], planes[2])
    ref = None
    for mq, mk in ((40, 90), (1, 1), (7, 1 << 20), (100000, 2)):
        g = B.gpu()._replace(max_q=mq, max_keys=mk)
        got = [host(ctx.attn_scores_eval(g, ks[0], ks[1], q, *planes), ctx.bw),
               host(ctx.attn_mix_eval(g, km[0], km[1], p, *planes), ctx.bw)]
        ref = ref or got
        assert all(np.array_equal(a, b) for a, b in zip(ref, got))


def test_offsets_past_32_bits():
    """A cache plane of more than 2^31 words, rows at its end."""
    torch = _torch()
    ctx = mpcx.Ctx(bw=32, scale=12)
    kv, page, dim = 2, 64, 128
    n_pages = (1 << 31) // (kv * page * dim) + 40
    rng = np.random.default_rng(1)
    pool = torch.zeros((n_pages, kv, page, dim), dtype=torch.int32, device="cuda")
    rows = words(rng, (100, kv, dim), 32)
    slot = np.arange((n_pages - 2) * page, (n_pages - 2) * page + 100).astype(np.int64)
    ctx.cache_append([(dev(rows), pool, False)], dev(slot))
    assert np.array_equal(host(pool[n_pages - 2], 32), rows[:64].transpose(1, 0, 2))
    assert np.array_equal(host(pool[n_pages - 1][:, :36], 32), rows[64:].transpose(1, 0, 2))
    table = np.array([[n_pages - 2, n_pages - 1]], np.int32)
    i32 = np.int32
    g = mpcx.AttnBatch(dev(table), dev(np.array([0, 1], i32)), dev(np.array([0], i32)), dev(np.array([100], i32)),
                       dev(np.array([0], np.int64)), 400, 4, 1, 100)
    q, p = words(rng, (1, 4, dim), 32), words(rng, (400,), 32)
    zero = torch.zeros_like(pool)
    k = ctx.attn_scores_keygen(g, dev(np.zeros_like(q)), zero, zero)
    got = host(ctx.attn_scores_eval(g, k[0], k[1], dev(q), pool, zero, zero), 32) - host(k[2], 32)
    want = np.concatenate([rows[:, h // 2] @ q[0, h] for h in range(4)])
    assert np.array_equal(got, want)
    k = ctx.attn_mix_keygen(g, dev(np.zeros_like(p)), zero, zero)
    got = host(ctx.attn_mix_eval(g, k[0], k[1], dev(p), pool, zero, zero), 32) - host(k[2], 32)
    assert np.array_equal(got[0], np.stack([p[h * 100:(h + 1) * 100] @ rows[:, h // 2] for h in range(4)]))
    ctx.close()
    del pool, zero
    torch.cuda.empty_cache()


def test_split_mask(ctx):
    rng = np.random.default_rng(2)
    m = words(rng, (1003,), ctx.bw)
    s0, s1 = (host(s, ctx.bw) for s in ctx.split_mask(dev(m), seed=8, gate=3))
    with np.errstate(over="ignore"):
        assert np.array_equal(s0 + s1, m)
    assert np.unique(s0).size > 900
    t0, _ = ctx.split_mask(dev(m), seed=9, gate=3)
    assert not np.array_equal(host(t0, ctx.bw), s0)


# ---------------- order, counters, graphs ----------------
def test_on_torch_streams(ctx):
    """Behind a busy stream: the calls wait for their inputs, and on the caller's
    own stream they are in its order."""
    torch = _torch()
    rng = np.random.default_rng(6)
    a, w = words(rng, (3, 256), ctx.bw), rng.integers(-8, 8, (40, 256))
    scale = rng.integers(1, 99, (2, 40)).astype(np.int32)
    want = q4_plain(a, w, scale, 128).astype(ctx.T)
    d, q, s = dev(a), dev(q4_pack(w)), dev(scale)
    late = torch.zeros_like(d)
    big = torch.empty(1 << 29, dtype=torch.uint8, device="cuda")
    for stream in (None, torch.cuda.Stream()):
        ctx.set_stream(stream)
        with torch.cuda.stream(stream):  # None: torch's own
            for k in range(32):
                big.fill_(k)
            late.zero_()
            late.copy_(d)
            got = ctx.ring_gemm_q4(late, q, s, 128) + 0
            torch.cuda.current_stream().synchronize()
        assert np.array_equal(host(got, ctx.bw), want)
    ctx.set_stream(None)


def test_graph_replays(ctx):
    """Captured once, replayed on new inputs with eager work between."""
    torch = _torch()
    B = Batch(ctx.bw, 2, 1, 300, 4, 2, 64, 16, "causal")
    planes = [dev(v) for v in (B.y, B.b0, B.b1)]
    g = B.gpu()
    q, p = dev(words(B.rng, (B.tokens, 4, 64), ctx.bw)), dev(words(B.rng, (B.n,), ctx.bw))
    ks = ctx.attn_scores_keygen(g, q, planes[1], planes[2])
    km = ctx.attn_mix_keygen(g, p, planes[1], planes[2])
    w, scale = dev(q4_pack(B.rng.integers(-8, 8, (50, 64)))), dev(B.rng.integers(1, 99, (2, 50)).astype(np.int32))
    slot = dev(np.arange(B.tokens).astype(np.int64))

    def step():
        s = ctx.attn_scores_eval(g, ks[0], ks[1], q, *planes)
        o = ctx.attn_mix_eval(g, km[0], km[1], p, *planes)
        z = ctx.ring_gemm_q4(q.view(-1, 64), w, scale, 32)
        ctx.cache_append([(q[:, :2], planes[0], False)], slot)
        return s, o, z

    stream = torch.cuda.Stream()
    ctx.set_stream(stream)
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs = step()
        for i in range(4):
            q.copy_(dev(words(B.rng, (B.tokens, 4, 64), ctx.bw)))
            p.copy_(dev(words(B.rng, (B.n,), ctx.bw)))
            keep = planes[0].clone()
            graph.replay()
            stream.synchronize()
            after = planes[0].clone()
            planes[0].copy_(keep)
            want = step()
            stream.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(outs, want)) and torch.equal(after, planes[0])
    ctx.set_stream(None)


def test_exchange_is_counted(ctx):
    B = Batch(ctx.bw, 2, 3, 20, 4, 2, 8, 4, "causal")
    planes = [dev(v) for v in (B.y, B.b0, B.b1)]
    q, p = dev(words(B.rng, (B.tokens, 4, 8), ctx.bw)), dev(words(B.rng, (B.n,), ctx.bw))
    ks = ctx.attn_scores_keygen(B.gpu(), q, planes[1], planes[2])
    km = ctx.attn_mix_keygen(B.gpu(), p, planes[1], planes[2])
    ctx.reset_counters()
    ctx.attn_scores_eval(B.gpu(), ks[0], ks[1], q, *planes)
    assert (ctx.rounds, ctx.bytes_exchanged) == (1, 2 * B.n * ctx.bw // 8)
    ctx.attn_mix_eval(B.gpu(), km[0], km[1], p, *planes)
    assert (ctx.rounds, ctx.bytes_exchanged) == (2, 2 * (B.n + q.numel()) * ctx.bw // 8)


# ---------------- refusals ----------------
def test_refusals(ctx):
    torch = _torch()
    L, h, EINVAL = ctx.lib, ctx.h, 1
    t = torch.zeros(4096, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    d = t.data_ptr()

    def q4(M=2, K=64, N=4, g=32, a=d, lda=64, q=d, s=d, o=d + 16384, ldc=4, w=d + 24576):
        return L.mpcx_ring_gemm_q4(h, M, K, N, g, a, lda, q, s, o, ldc, w)

    for bad in (dict(M=0), dict(K=0), dict(N=0), dict(g=0), dict(g=48), dict(g=16), dict(lda=63), dict(ldc=3),
                dict(a=None), dict(q=None), dict(s=None), dict(o=None), dict(q=d + 8), dict(a=d + 2), dict(s=d + 1),
                dict(o=d + 3), dict(M=-1)):
        assert q4(**bad) == EINVAL, bad
    assert q4() == 0
    cache = mpcx.Cache(2, 8, 4, 3)
    rot = mpcx._Rotation(4, 0, 8, 3, d, d)

    def append(cache=cache, n=2, slot=d, pos=d, rot=rot, planes=((d, 16, d + 8192, 1),)):
        arr = (mpcx._CachePlane * 16)(*[mpcx._CachePlane(*p) for p in planes])
        return L.mpcx_cache_append(h, C.byref(cache), n, slot, pos, C.byref(rot) if rot else None, len(planes), arr)

    one = (d, 16, d + 8192, 1)
    for bad in (dict(cache=mpcx.Cache(0, 8, 4, 3)), dict(cache=mpcx.Cache(2, 0, 4, 3)),
                dict(cache=mpcx.Cache(2, 8, 0, 3)), dict(cache=mpcx.Cache(2, 8, 4, 0)),
                dict(cache=mpcx.Cache(1 << 20, 1 << 20, 1 << 20, 1 << 20)), dict(slot=None), dict(pos=None),
                dict(rot=None), dict(planes=()), dict(planes=(one,) * 9), dict(planes=((d, 15, d + 8192, 1),)),
                dict(planes=((None, 16, d, 1),)), dict(planes=((d, 16, None, 1),)), dict(planes=((d + 1, 16, d, 1),)),
                dict(rot=mpcx._Rotation(5, 0, 8, 3, d, d)), dict(rot=mpcx._Rotation(0, 0, 8, 3, d, d)),
                dict(rot=mpcx._Rotation(4, 0, 0, 3, d, d)), dict(rot=mpcx._Rotation(4, 0, 8, ctx.bw, d, d)),
                dict(rot=mpcx._Rotation(4, 0, 8, -1, d, d)), dict(rot=mpcx._Rotation(4, 0, 8, 3, None, d)),
                dict(n=1 << 61)):
        assert append(**bad) == EINVAL, bad
    assert append(n=0, slot=None, pos=None) == 0 and append() == 0
    assert L.mpcx_split_mask(h, 3, None, 1, 1, d, d) == EINVAL and L.mpcx_split_mask(h, 0, None, 1, 1, None, None) == 0

    z = torch.zeros(64, dtype=torch.int32, device="cuda")
    z[1] = 1
    torch.cuda.synchronize()
    i = z.data_ptr()

    def attn(call="eval", over=(), **kw):
        a = mpcx._Attn(mpcx.Cache(2, 8, 4, 3), 4, 1, 1, 2, 1, 8, 32, i, i, i, i, i)
        for k, v in dict(over).items():
            setattr(a, k, v)
        v = dict(k0=d, k1=d, x=d, y=d, b0=d, b1=d, slope=None, pos=None, out=d + 16384)
        v.update(kw)
        if call == "eval":
            return L.mpcx_attn_scores_eval(h, C.byref(a), v["k0"], v["k1"], v["x"], v["y"], v["b0"], v["b1"],
                                           v["slope"], v["pos"], v["out"])
        if call == "mix":
            return L.mpcx_attn_mix_eval(h, C.byref(a), v["k0"], v["k1"], v["x"], v["y"], v["b0"], v["b1"], v["out"])
        return L.mpcx_attn_scores_keygen(h, C.byref(a), v["x"], v["b0"], v["b1"], v["out"], 1, 1, v["k0"], v["k1"])

    for call in ("eval", "mix", "keygen"):
        for bad in (dict(n_heads=0), dict(n_heads=3), dict(n_tok=-1), dict(n_seq=-1), dict(max_pages=-1),
                    dict(max_q=0), dict(max_keys=0), dict(n_scores=-1), dict(d_pages=None), dict(d_off=None),
                    dict(cache=mpcx.Cache(2, 0, 4, 3))):
            assert attn(call, bad.items()) == EINVAL, (call, bad)
        for bad in (dict(k0=None), dict(k1=None), dict(x=None), dict(b0=None), dict(b1=None), dict(out=None),
                    dict(x=d + 1), dict(k0=d + 4)):
            assert attn(call, **bad) == EINVAL, (call, bad)
    assert attn(slope=d) == EINVAL and attn(y=None) == EINVAL
    assert L.mpcx_attn_scores_message(h, 2, None, *[d] * 7) == EINVAL
    assert L.mpcx_attn_mix_message(h, -1, None, *[d] * 5) == EINVAL
    assert attn(over=dict(n_tok=0).items(), x=None, k0=d) == 0  # nothing to do
    assert attn() == 0
    ctx.sync()
    assert L.mpcx_ring_gemm_q4(None, 1, 1, 1, 32, d, 1, d, d, d, 1, None) == EINVAL


def test_binding_refusals(ctx):
    torch = _torch()
    word = torch.int32 if ctx.bw == 32 else torch.int64
    other = torch.int64 if ctx.bw == 32 else torch.int32
    q = torch.zeros((4, 32), dtype=torch.uint8, device="cuda")
    s = torch.ones((2, 4), dtype=torch.int32, device="cuda")
    a = torch.zeros((2, 64), dtype=word, device="cuda")
    for args in ((a.to(other), q, s, 32), (a.cpu(), q, s, 32), (a.t(), q, s, 32), (a, q[:, :16], s, 32),
                 (a, q, s[:1], 32), (a, q, s.long(), 32)):
        with pytest.raises(mpcx.MpcxError):
            ctx.ring_gemm_q4(*args)
    pool = torch.zeros((2, 1, 4, 8), dtype=word, device="cuda")
    rows, slot = torch.zeros((3, 1, 8), dtype=word, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for planes, at in (([(rows, pool, False)], slot.int()), ([(rows[:2], pool, False)], slot),
                       ([(rows, pool.to(other), False)], slot), ([(rows, pool, True)], slot)):
        with pytest.raises(mpcx.MpcxError):
            ctx.cache_append(planes, at)


# ---------------- together, and one party at a time ----------------
@pytest.mark.parametrize("bw", [32, 64])
def test_attention_layer(bw):
    """The operators in one layer, prompt and single tokens, with the framework's
    truncation and ReLU gates between: the plain fixed-point layer bit for bit."""
    import attention
    said = []
    assert attention.run(bw, say=said.append), said
    assert len(said) == 5


def test_parties_reconstruct_the_gates(ctx):
    """Each party's message from its own key and shares, exchanged over a channel:
    both hold the gate's output."""
    import threading
    torch = _torch()
    B = Batch(ctx.bw, 2, 5, 30, 4, 2, 24, 8, "prefix", seed=8)
    g, planes = B.gpu(), [dev(v) for v in (B.y, B.b0, B.b1)]
    q, p = dev(words(B.rng, (B.tokens, 4, 24), ctx.bw)), dev(words(B.rng, (B.n,), ctx.bw))
    slope, pos = dev(words(B.rng, (4,), ctx.bw)), dev(B.pos)
    ks = ctx.attn_scores_keygen(g, q, planes[1], planes[2])
    km = ctx.attn_mix_keygen(g, p, planes[1], planes[2])
    want = [host(ctx.attn_scores_eval(g, ks[0], ks[1], q, *planes, slope=slope, pos=pos), ctx.bw),
            host(ctx.attn_mix_eval(g, km[0], km[1], p, *planes), ctx.bw).reshape(-1)]
    peers, got, errors = mpcx.Peer.pair(), {}, []

    def party(i):
        try:
            c = mpcx.Ctx(bw=ctx.bw, scale=12)
            s = c.attn_scores_message(i, g, ks[i], q, planes[0], planes[1 + i], slope=slope, pos=pos)
            o = c.attn_mix_message(i, g, km[i], p, planes[0], planes[1 + i])
            got[i] = [c.party_reconstruct(peers[i], host(v, ctx.bw).reshape(-1)) for v in (s, o)]
            c.close()
        except Exception as e:  # a thread's failure is the test's
            errors.append(e)

    threads = [threading.Thread(target=party, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors and len(got) == 2, errors
    for i in (0, 1):
        assert all(np.array_equal(a, b) for a, b in zip(got[i], want))
    for peer in peers:
        peer.close()
    torch.cuda.synchronize()


def test_sizes_past_the_bounds_are_refused(ctx):
    L, h = ctx.lib, ctx.h
    d = _torch().zeros(64, dtype=_torch().int64, device="cuda").data_ptr()
    assert L.mpcx_ring_gemm_q4(h, 1, (1 << 24) + 1, 1, 32, d, (1 << 24) + 1, d, d, d, 1, d) == 1
    a = mpcx._Attn(mpcx.Cache(1, 8, 4, 3), 1 << 16, 1 << 16, 1, 1, 1, 1, 0, d, d, d, d, d)
    assert L.mpcx_attn_mix_eval(h, C.byref(a), d, d, d, d, d, d, d) == 1  # 2^32 rows
    big = mpcx.Cache(1 << 16, 1 << 16, 1, 1)
    plane = (mpcx._CachePlane * 1)(mpcx._CachePlane(d, 1 << 32, d, 0))
    assert L.mpcx_cache_append(h, C.byref(big), 1, d, None, None, 1, plane) == 1


def test_outputs_over_inputs_are_refused(ctx):
    B = Batch(ctx.bw, 1, 4, 20, 2, 2, 16, 4, "causal", seed=9)
    g, planes = B.gpu(), [dev(v) for v in (B.y, B.b0, B.b1)]
    q, p = dev(words(B.rng, (B.tokens, 2, 16), ctx.bw)), dev(words(B.rng, (B.n,), ctx.bw))
    ks, km = ctx.attn_scores_keygen(g, q, *planes[1:]), ctx.attn_mix_keygen(g, p, *planes[1:])
    L, h, a = ctx.lib, ctx.h, ctx._attn(g, planes[0])
    y, b0, b1 = (t.data_ptr() for t in planes)
    for out in (q, ks[0], ks[1], *planes):
        assert L.mpcx_attn_scores_eval(h, C.byref(a), ks[0].data_ptr(), ks[1].data_ptr(), q.data_ptr(), y, b0, b1, None,
                                       None, out.data_ptr()) == 1
    for out in (p, km[0], km[1], *planes):
        assert L.mpcx_attn_mix_eval(h, C.byref(a), km[0].data_ptr(), km[1].data_ptr(), p.data_ptr(), y, b0, b1,
                                    out.data_ptr()) == 1
    assert b"overlaps" in L.mpcx_last_error(h)
