"""The transformer operators where sizes, launches and buffers meet their ends, and
the kernel instances that small shapes do not choose, against the definitions in
64-bit integers.  All results are ring words, so every comparison is of all bits."""
import ctypes as C

import numpy as np
import pytest

import mpcx
from test_gpu_transformer import Batch, dev, host, q4_pack, q4_plain, words

pytestmark = pytest.mark.gpu
EINVAL = 1


@pytest.fixture(scope="module", params=[32, 64])
def ctx(request):
    c = mpcx.Ctx(bw=request.param, scale=12)
    yield c
    c.close()


def q4_case(ctx, M, K, N, group, seed=0):
    rng = np.random.default_rng(seed + M * 7 + K * 3 + N)
    a, w = words(rng, (M, K), ctx.bw), rng.integers(-8, 8, (N, K))
    scale = rng.integers(-(1 << 31), 1 << 31, (-(-K // group), N)).astype(np.int32)
    scale.flat[0], scale.flat[-1] = -(1 << 31), (1 << 31) - 1
    return a, w, scale


# ---------------- 4-bit weights ----------------
@pytest.mark.parametrize("M", [1, 2, 40, 90])
@pytest.mark.parametrize("K,N,group", [(1, 1, 128), (31, 16, 64), (32, 5, 64), (32, 17, 128), (33, 5, 128), (64, 5, 128),
                                       (65, 3, 128), (96, 5, 128), (97, 18, 256), (127, 16, 128), (40, 9, 192)])
def test_q4_rows_shorter_than_a_chunk(ctx, M, K, N, group):
    a, w, scale = q4_case(ctx, M, K, N, group)
    got = host(ctx.ring_gemm_q4(dev(a), dev(q4_pack(w)), dev(scale), group), ctx.bw)
    assert np.array_equal(got, q4_plain(a, w, scale, group).astype(ctx.T))


# Instances by the launch's rules on 256 compute units: a row tile is 4 rows of Z_2^32 or
# 2 of Z_2^64, so `tiles` of them are the same instance in both rings.
#   up to 16 tiles: the kernel of few rows, of 1, 2 or 4 tiles a workgroup, from digits in
#   the workspace where tiles x K x column tiles pass 2^20;
#   more: column tiles a wave, the most of 4 (groups of 64 and 128), 2 and 1 that give 512
#   workgroups of 8 row tiles and 32 times as many columns.
Q4_INSTANCES = [
    # tiles, K, N, group: few rows, digits in the workspace
    (1, 4200, 4100, 128), (2, 2111, 4097, 128), (4, 1000, 4500, 128), (16, 900, 2003, 256),
    (1, 4200, 4100, 64), (2, 2111, 4097, 64), (13, 700, 2600, 192),
    (1, 4200, 4100, 32), (2, 2111, 4097, 96), (3, 1500, 4200, 32),
    # many rows: 4, 2 and 1 column tiles a wave
    (125, 130, 4090, 128), (130, 200, 4095, 64), (126, 257, 2090, 128), (125, 100, 2100, 64),
    (127, 161, 2081, 32), (250, 95, 1030, 96), (17, 1300, 100, 128), (40, 300, 333, 64), (21, 190, 258, 32)]


@pytest.mark.parametrize("scales", ["any", "small", "few large"])
@pytest.mark.parametrize("tiles,K,N,group", Q4_INSTANCES)
def test_q4_instances(ctx, tiles, K, N, group, scales):
    M = tiles * (4 if ctx.bw == 32 else 2) - 1
    a, w, scale = q4_case(ctx, M, K, N, group, seed=11)
    if scales != "any":  # scales within 24 bits, and among them some that are not
        rng = np.random.default_rng(K)
        small = rng.integers(-(1 << 23), 1 << 23, scale.shape).astype(np.int32)
        small.flat[:2] = -(1 << 23), (1 << 23) - 1
        scale = np.where(rng.random(scale.shape) < 0.01, scale, small) if scales == "few large" else small
    got = host(ctx.ring_gemm_q4(dev(a), dev(q4_pack(w)), dev(scale), group), ctx.bw)
    if ctx.bw == 32:  # the same modulo 2^32 in float64 halves: 2^16 * 2^3 * K < 2^53
        a64 = np.stack([a & 0xFFFF, a >> 16]).astype(np.float64)
        want = np.zeros((M, N), np.uint64)
        for g in range(scale.shape[0]):
            k = slice(g * group, (g + 1) * group)
            lo, hi = (a64[:, :, k] @ w[:, k].T.astype(np.float64)).astype(np.int64).astype(np.uint64)
            want += (lo + (hi << np.uint64(16))) * scale[g].astype(np.int64).astype(np.uint64)
    else:
        want = q4_plain(a, w, scale, group)
    assert np.array_equal(got, want.astype(ctx.T))


def test_q4_work_bytes_at_the_ends_of_the_sizes(ctx):
    """What the rows' digits take, whole tiles of 32 or 16 rows and steps of 128 words;
    nothing for sizes that are refused."""
    def want(M, K):
        rows = 32 if ctx.bw == 32 else 16
        return -(-M // rows) * rows * ctx.bw // 8 * (-(-K // 128) * 128)

    top = (1 << 31) - 1
    for M, K in ((1, 1), (33, 129), (1, 1 << 24), (top - 255, 1), (top - 255, 1 << 24)):
        assert ctx.lib.mpcx_ring_gemm_q4_work_bytes(ctx.h, M, K) == want(M, K)
    for M, K in ((0, 1), (1, 0), (-1, 5), (top, 1), (top - 254, 1), (1, top), (1, (1 << 24) + 1)):
        assert ctx.lib.mpcx_ring_gemm_q4_work_bytes(ctx.h, M, K) == 0


def test_q4_sizes_past_the_bounds(ctx):
    import torch
    t = torch.zeros(64, dtype=torch.int64, device="cuda").data_ptr()
    top, wide = (1 << 31) - 1, 1 << 40
    for M, K, N in ((top, 1, 1), (top - 254, 1, 1), (1, 1, top), (1, 1, top - 254), (1, (1 << 24) + 1, 1), (1, top, 1)):
        assert ctx.lib.mpcx_ring_gemm_q4(ctx.h, M, K, N, 32, t, wide, t, t, t + 256, wide, t) == EINVAL, (M, K, N)
        assert b"bad argument" in ctx.lib.mpcx_last_error(ctx.h)


# ---------------- launches ----------------
def test_q4_columns_past_one_launch(ctx):
    """16 waves a column tile: columns past 2^26 are more threads than a launch may have."""
    import torch
    M, K, N, group = 1, 512, (1 << 26) + 37, 544
    gen = torch.Generator(device="cuda").manual_seed(ctx.bw)
    q = torch.empty((N, K // 2), dtype=torch.uint8, device="cuda")
    for i in range(0, N, 1 << 24):
        q[i:i + (1 << 24)].random_(0, 256, generator=gen)
    scale = torch.randint(-(1 << 31), 1 << 31, (1, N), dtype=torch.int64, device="cuda", generator=gen).int()
    rng = np.random.default_rng(5)
    a = words(rng, (M, K), ctx.bw)
    out = ctx.ring_gemm_q4(dev(a), q, scale, group)
    at = np.unique(np.concatenate([np.arange(64), np.arange(N - 128, N), rng.integers(0, N, 4000)]))
    t = torch.from_numpy(at).cuda()
    byte = q[t].cpu().numpy().astype(np.int64)
    w = np.stack([byte & 15, byte >> 4], -1).reshape(at.size, K)
    want = q4_plain(a, (w ^ 8) - 8, scale[:, t].cpu().numpy(), group).astype(ctx.T)
    assert np.array_equal(host(out[:, t], ctx.bw), want)
    del q, scale, out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("max_q,max_keys", [(1 << 20, 1), (1 << 20, 60), ((1 << 31) - 1, (1 << 31) - 1)])
def test_launch_hints_of_any_size(ctx, max_q, max_keys):
    """8 sequences of 8 cache heads: 2^20 tokens a sequence, taken at their word, are
    more threads than a launch may have."""
    B = Batch(ctx.bw, 8, 3, 60, 32, 8, 16, 16, "causal", seed=3)
    g, planes = B.gpu()._replace(max_q=max_q, max_keys=max_keys), [dev(v) for v in (B.y, B.b0, B.b1)]
    rq, q = words(B.rng, (B.tokens, 32, 16), ctx.bw), words(B.rng, (B.tokens, 32, 16), ctx.bw)
    rp, p = words(B.rng, (B.n,), ctx.bw), words(B.rng, (B.n,), ctx.bw)
    with np.errstate(over="ignore"):
        k0, k1, rs = ctx.attn_scores_keygen(g, dev(rq), *planes[1:])
        got = host(ctx.attn_scores_eval(g, k0, k1, dev(q), *planes), ctx.bw)
        assert np.array_equal(got, B.scores(q - rq, B.y - B.b0 - B.b1) + host(rs, ctx.bw))
        k0, k1, ro = ctx.attn_mix_keygen(g, dev(rp), *planes[1:])
        got = host(ctx.attn_mix_eval(g, k0, k1, dev(p), *planes), ctx.bw)
        assert np.array_equal(got, B.mix(p - rp, B.y - B.b0 - B.b1) + host(ro, ctx.bw))


# ---------------- the attention kernels' instances ----------------
TWO_TILES = [  # rows enough for two tiles of them a workgroup in both rings
    (4, 32, 50, 64, 8, 64, 16, "causal"), (4, 33, 70, 64, 8, 33, 16, "prefix"), (3, 70, 90, 32, 8, 128, 24, "window"),
    (5, 20, 40, 96, 8, 100, 16, "ragged"), (16, 17, 33, 32, 16, 24, 7, "ragged")]


@pytest.mark.parametrize("seqs,q,keys,heads,kv,dim,page,mask", TWO_TILES)
@pytest.mark.parametrize("gap", [0, 3])
def test_scores_of_two_tiles(ctx, seqs, q, keys, heads, kv, dim, page, mask, gap):
    """Both parties together, the dealer's form and each party's message, with the bias
    and without."""
    B = Batch(ctx.bw, seqs, q, keys, heads, kv, dim, page, mask, seed=7, gap=gap)
    rq, qhat = words(B.rng, (B.tokens, heads, dim), ctx.bw), words(B.rng, (B.tokens, heads, dim), ctx.bw)
    slope = words(B.rng, (heads,), ctx.bw)
    g, planes = B.gpu(), [dev(v) for v in (B.y, B.b0, B.b1)]
    k0, k1, rs = ctx.attn_scores_keygen(g, dev(rq), planes[1], planes[2], seed=3, gate=9)
    extra = dict(slope=dev(slope), pos=dev(B.pos)) if gap else {}
    got = host(ctx.attn_scores_eval(g, k0, k1, dev(qhat), *planes, **extra), ctx.bw)
    parts = [host(ctx.attn_scores_message(p, g, k, dev(qhat), planes[0], planes[1 + p], **extra), ctx.bw)
             for p, k in ((0, k0), (1, k1))]
    with np.errstate(over="ignore"):
        want = B.scores(qhat - rq, B.y - B.b0 - B.b1) + host(rs, ctx.bw) + (B.bias(slope) if gap else 0)
        m = B.inside()
        assert np.array_equal(got[m], want[m])
        assert np.array_equal((parts[0] + parts[1])[m], want[m])


def test_sums_past_the_matrix_cores_sums(ctx):
    """Every digit at -128 and every term of the gate the same product, over more keys a
    wave than 31 bits of digit sums hold (Z_2^32 wraps, Z_2^64 folds in between)."""
    import torch
    seqs, keys, dim, page = 256, 100000, 4, 64  # a workgroup for each sequence: no splits
    w = (-sum(128 << (8 * p) for p in range(ctx.bw // 8))) % (1 << ctx.bw)
    word = torch.int32 if ctx.bw == 32 else torch.int64

    def full(shape, v):
        v %= 1 << ctx.bw
        return torch.full(shape, v - (1 << ctx.bw) if v >> (ctx.bw - 1) else v, dtype=word, device="cuda")

    n, pages, i32 = seqs * keys, -(-keys // page), np.int32
    g = mpcx.AttnBatch(dev(np.tile(np.arange(pages, dtype=i32), (seqs, 1))), dev(np.arange(seqs + 1, dtype=i32)),
                       dev(np.zeros(seqs, i32)), dev(np.full(seqs, keys, i32)), dev(np.arange(seqs) * keys), n, 1, 1, keys)
    shape, tail = (pages, 1, page, dim), torch.zeros(-(-seqs * dim * ctx.bw // 2048) * 256, dtype=torch.uint8, device="cuda")
    assert n * ctx.bw // 8 % 256 == 0
    # (x - a0)(y - b0) = (-x) b1 = (-a1) y = w w
    k0, k1 = (torch.cat((full((n,), v).view(torch.uint8), tail)) for v in (-2 * w, -w))
    got = host(ctx.attn_mix_eval(g, k0, k1, full((n,), -w), full(shape, w), full(shape, 0), full(shape, w)), ctx.bw)
    assert (got == 3 * keys * w * w % (1 << ctx.bw)).all()


# ---------------- buffers ----------------
def test_q4_output_or_workspace_over_another_buffer(ctx):
    import torch
    M, K, N, group, tb = 6, 64, 40, 32, ctx.bw // 8
    nb = ctx.lib.mpcx_ring_gemm_q4_work_bytes(ctx.h, M, K)
    buf = torch.zeros(5 * (1 << 16), dtype=torch.uint8, device="cuda")
    a, q, s, c, w = (buf.data_ptr() + (i << 16) for i in range(5))
    assert nb < 1 << 16
    torch.cuda.synchronize()

    def call(a=a, lda=K, q=q, s=s, c=c, ldc=N, w=w):
        return ctx.lib.mpcx_ring_gemm_q4(ctx.h, M, K, N, group, a, lda, q, s, c, ldc, w)

    assert call() == 0
    for bad in (dict(c=a), dict(c=a + K * tb - tb), dict(c=a + ((M - 1) * K + K - 1) * tb), dict(c=q), dict(c=q + N * 32 - tb),
                dict(c=s), dict(c=s + 2 * N * 4 - tb), dict(c=w), dict(c=w + nb - tb), dict(w=a), dict(w=q), dict(w=s),
                dict(w=c), dict(a=w + nb - 8), dict(lda=K + N, c=a + (K - 1) * tb, ldc=K + N),
                dict(lda=K + N, c=a + (K + 1) * tb, ldc=K + N), dict(lda=K + N, c=a + K * tb, ldc=K + N + 1)):
        assert call(**bad) == EINVAL, bad
        assert b"overlaps" in ctx.lib.mpcx_last_error(ctx.h)
    ctx.sync()


@pytest.mark.parametrize("M", [3, 70])
def test_q4_into_columns_of_its_operand(ctx, M):
    """Input and output side by side in one matrix."""
    K, N, group = 96, 50, 32
    a, w, scale = q4_case(ctx, M, K, N, group)
    big = words(np.random.default_rng(M), (M, K + N + 3), ctx.bw)
    big[:, :K] = a
    d = dev(big)
    ctx.ring_gemm_q4(d[:, :K], dev(q4_pack(w)), dev(scale), group, out=d[:, K + 1:K + 1 + N])
    big[:, K + 1:K + 1 + N] = q4_plain(a, w, scale, group)
    assert np.array_equal(host(d, ctx.bw), big)


def test_cache_append_pool_over_another_buffer(ctx):
    import torch
    tb = ctx.bw // 8
    cache, n, row = mpcx.Cache(2, 8, 4, 3), 5, 16
    pool = 2 * 8 * 4 * 3 * tb
    buf = torch.zeros(8 << 18, dtype=torch.uint8, device="cuda")
    rows0, rows1, pool0, pool1, slot, pos, cos, sin = (buf.data_ptr() + (i << 18) for i in range(8))
    buf[4 << 18:(4 << 18) + 8 * n].view(torch.int64).copy_(torch.arange(n))
    torch.cuda.synchronize()

    def call(rows0=rows0, ld0=row, pool0=pool0, rows1=rows1, pool1=pool1, slot=slot, pos=pos, cos=cos, sin=sin, turn=1):
        planes = (mpcx._CachePlane * 2)(mpcx._CachePlane(rows0, ld0, pool0, turn), mpcx._CachePlane(rows1, row, pool1, 0))
        return ctx.lib.mpcx_cache_append(ctx.h, C.byref(cache), n, slot, pos, C.byref(mpcx._Rotation(4, 0, 8, 3, cos, sin)),
                                         2, planes)

    assert call() == 0
    for bad in (dict(pool0=rows0), dict(pool0=rows1), dict(pool1=rows0 + (n * row - 1) * tb), dict(pool1=pool0),
                dict(pool1=pool0 + pool - tb), dict(pool0=pool1 + pool - tb), dict(pool0=slot), dict(pool1=slot + 8 * n - 8),
                dict(pool0=pos), dict(pool1=cos), dict(pool1=sin + 32 * tb - tb), dict(rows0=pool1 - tb),
                dict(ld0=4096, pool1=rows0 + 4096 * tb * (n - 1) - tb)):
        assert call(**bad) == EINVAL, bad
        assert b"overlaps" in ctx.lib.mpcx_last_error(ctx.h)
    # between the rows, at a table that no plane uses, and just past the rows
    assert call(ld0=4096, pool1=rows0 + 4096 * tb + row * tb) == 0
    assert call(turn=0, pool0=cos) == 0 and call(pool0=rows0 + n * row * tb) == 0
    ctx.sync()


@pytest.mark.parametrize("heads,dim", [(1, 8), (1, 1), (3, 1)])
def test_cache_append_rows_of_single_heads_and_dims(ctx, heads, dim):
    """Rows cut out of wider ones."""
    rng = np.random.default_rng(heads + dim)
    big, pool = words(rng, (6, heads, dim + 5), ctx.bw), words(rng, (3, heads, 4, dim), ctx.bw)
    if heads > 1:
        big = words(rng, (6, dim + 4, heads), ctx.bw)
    slot = rng.permutation(12)[:6].astype(np.int64)
    d, p = dev(big), dev(pool)
    rows = d[:, :, 2:2 + dim] if heads == 1 else d[:, 1:1 + dim].transpose(1, 2)
    ctx.cache_append([(rows, p, False)], dev(slot))
    for t, s in enumerate(slot):
        pool[s // 4, :, s % 4] = big[t, :, 2:2 + dim] if heads == 1 else big[t, 1:1 + dim].T
    assert np.array_equal(host(p, ctx.bw), pool)


class Gate:
    """The buffers of an attention gate, each at a place of its own, as the C calls
    take them."""

    def __init__(self, ctx, scores):
        import torch
        self.ctx, self.scores, self.tb = ctx, scores, ctx.bw // 8
        names = "pages qstart lo hi off slope pos x y b0 b1 k0 k1 out".split()
        self.buf = torch.zeros(len(names) << 18, dtype=torch.uint8, device="cuda")
        self.at = {n: self.buf.data_ptr() + (i << 18) for i, n in enumerate(names)}
        for name, values in dict(pages=[2, 0], qstart=[0, 3], lo=[0, 0, 1], hi=[2, 3, 5], off=[0, 8, 20, 36],
                                 pos=[1, 2, 4]).items():
            t = torch.tensor(values[:3], dtype=torch.int64 if name == "off" else torch.int32)
            self.buf[self.at[name] - self.buf.data_ptr():][:t.numel() * t.element_size()] = t.view(torch.uint8).cuda()
        self.rows, self.wide = 3 * 4 * 8, 36
        self.left, self.to = (self.rows, self.wide) if scores else (self.wide, self.rows)
        self.bytes = dict(pages=8, qstart=8, lo=12, hi=12, off=24, slope=4 * self.tb, pos=12, x=self.left * self.tb,
                          y=192 * self.tb, b0=192 * self.tb, b1=192 * self.tb, out=self.to * self.tb)
        key = (self.left * self.tb + 255) // 256 * 256 + (self.to * self.tb + 255) // 256 * 256
        self.bytes.update(k0=key, k1=key)
        torch.cuda.synchronize()

    def batch(self, v):
        return mpcx._Attn(mpcx.Cache(2, 8, 4, 3), 4, 3, 1, 2, 3, 5, self.wide, v["pages"], v["qstart"], v["lo"], v["hi"],
                          v["off"])

    def eval(self, **over):
        v = {**self.at, **over}
        f = self.ctx.lib.mpcx_attn_scores_eval if self.scores else self.ctx.lib.mpcx_attn_mix_eval
        extra = [v["slope"], v["pos"]] if self.scores else []
        return f(self.ctx.h, C.byref(self.batch(v)), *[v[n] for n in ("k0", "k1", "x", "y", "b0", "b1")], *extra, v["out"])

    def keygen(self, **over):
        """x is the left operand's mask, out the output's."""
        v = {**self.at, **over}
        f = self.ctx.lib.mpcx_attn_scores_keygen if self.scores else self.ctx.lib.mpcx_attn_mix_keygen
        return f(self.ctx.h, C.byref(self.batch(v)), v["x"], v["b0"], v["b1"], v["out"], 1, 1, v["k0"], v["k1"])


@pytest.mark.parametrize("scores", [True, False])
def test_attn_output_over_an_input(ctx, scores):
    g = Gate(ctx, scores)
    assert g.eval() == 0
    for n in g.at:
        if n == "out" or (not scores and n in ("slope", "pos")):
            continue
        for out in (g.at[n], g.at[n] + (g.bytes[n] - 1) // g.tb * g.tb, g.at[n] - g.bytes["out"] + g.tb):
            assert g.eval(out=out) == EINVAL, (n, out)
            assert b"overlaps" in ctx.lib.mpcx_last_error(ctx.h)
        assert g.eval(out=g.at[n] + (g.bytes[n] + g.tb - 1) // g.tb * g.tb) == 0, n
    ctx.sync()


@pytest.mark.parametrize("scores", [True, False])
def test_attn_keygen_output_over_another_buffer(ctx, scores):
    g = Gate(ctx, scores)
    assert g.keygen() == 0
    for to in ("out", "k0", "k1"):
        step = 16 if to != "out" else g.tb  # keys are aligned to 16 bytes
        for n in g.at:
            if n == to or n in ("y", "slope", "pos"):
                continue
            past = -(-(g.at[n] + g.bytes[n]) // step) * step
            for at in (g.at[n], past - step, (g.at[n] - g.bytes[to]) // step * step + step):
                assert g.keygen(**{to: at}) == EINVAL, (to, n, at)
                assert b"overlaps" in ctx.lib.mpcx_last_error(ctx.h)
            assert g.keygen(**{to: past}) == 0, (to, n)
    ctx.sync()


@pytest.mark.parametrize("scores", [True, False])
def test_misaligned_tables(ctx, scores):
    g = Gate(ctx, scores)
    calls = [(g.eval, "pages qstart lo hi off".split() + ["pos"] * scores), (g.keygen, "pages qstart lo hi off".split())]
    for call, names in calls:
        for n in names:
            for by in (1, 2) + (4,) * (n == "off"):
                assert call(**{n: g.at[n] + by}) == EINVAL, (n, by)
                assert b"misaligned" in ctx.lib.mpcx_last_error(ctx.h)
    planes = (mpcx._CachePlane * 1)(mpcx._CachePlane(g.at["x"], 16, g.at["y"], 0))
    cache = mpcx.Cache(2, 8, 4, 3)
    for slot, pos in ((4, 0), (1, 0), (0, 2)):
        assert ctx.lib.mpcx_cache_append(ctx.h, C.byref(cache), 1, g.at["off"] + slot, g.at["pos"] + pos, None, 1,
                                         planes) == EINVAL
    ctx.sync()


def test_split_mask_buffers(ctx):
    import torch
    n, tb = 300, ctx.bw // 8
    buf = torch.zeros(3 << 16, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    m, s0, s1 = (buf.data_ptr() + (i << 16) for i in range(3))

    def call(m=m, s0=s0, s1=s1):
        return ctx.lib.mpcx_split_mask(ctx.h, n, m, 1, 1, s0, s1)

    assert call() == 0
    for bad in (dict(s0=s1), dict(s0=s1 + (n - 1) * tb), dict(s0=m + tb), dict(s1=m + (n - 1) * tb), dict(m=s0 + tb),
                dict(m=s0 + 1), dict(s0=m + n * tb + 1), dict(s1=s1 + tb // 2), dict(s0=m, s1=m)):
        assert call(**bad) == EINVAL, bad
    ctx.sync()
    mask = words(np.random.default_rng(3), (n,), ctx.bw)
    want = [host(s, ctx.bw) for s in ctx.split_mask(dev(mask), seed=5, gate=6)]
    for place in (0, 1):  # a share in the mask's place
        d, other = dev(mask), dev(mask)
        torch.cuda.synchronize()
        to = [other.data_ptr(), other.data_ptr()]
        to[place] = d.data_ptr()
        assert ctx.lib.mpcx_split_mask(ctx.h, n, d.data_ptr(), 5, 6, *to) == 0
        ctx.sync()
        assert np.array_equal(host(d, ctx.bw), want[place]) and np.array_equal(host(other, ctx.bw), want[1 - place])


# ---------------- lengths of zero ----------------
def test_attn_without_pages(ctx):
    """Sequences that have no page yet: every token sees nothing."""
    B = Batch(ctx.bw, 2, 3, 5, 4, 2, 8, 4, "causal", seed=2)
    i32 = np.int32
    none = dev(np.zeros(B.tokens, i32))
    g = mpcx.AttnBatch(dev(np.zeros((2, 0), i32)), dev(B.qstart), none, none, dev(np.zeros(B.tokens, np.int64)), 0, 4, 3, 1)
    planes = [dev(v) for v in (B.y, B.b0, B.b1)]
    nothing = dev(np.zeros(0, ctx.T))
    k0, k1, ro = ctx.attn_mix_keygen(g, nothing, *planes[1:], seed=3)
    assert np.array_equal(host(ctx.attn_mix_eval(g, k0, k1, nothing, *planes), ctx.bw), host(ro, ctx.bw))
    q = dev(words(B.rng, (B.tokens, 4, 8), ctx.bw))
    k0, k1, rs = ctx.attn_scores_keygen(g, q, *planes[1:])
    assert rs.shape == (0,) and ctx.attn_scores_eval(g, k0, k1, q, *planes).shape == (0,)


# ---------------- what a party sends ----------------
def test_messages_hold_nothing_of_earlier_memory(ctx):
    """Words of no token's block and rows of tokens of no sequence go to the other
    party with the rest."""
    import torch
    B = Batch(ctx.bw, 2, 4, 30, 4, 2, 8, 4, "ragged", seed=4, gap=9)
    B.qstart[-1] -= 1  # the last token is of no sequence
    last = B.tokens - 1
    g, planes = B.gpu(), [dev(v) for v in (B.y, B.b0, B.b1)]
    q, p = dev(words(B.rng, (B.tokens, 4, 8), ctx.bw)), dev(words(B.rng, (B.n,), ctx.bw))
    ks, km = ctx.attn_scores_keygen(g, q, *planes[1:]), ctx.attn_mix_keygen(g, p, *planes[1:])
    seen = B.inside()
    for t, _, _, o in B.blocks():
        if t == last:
            seen[o] = False
    assert (~seen).sum() > 9
    for i in (0, 1):
        for scores in (True, False):
            old = torch.full((B.n,) if scores else tuple(q.shape), 0x5A5A5A5A, dtype=q.dtype, device="cuda")
            torch.cuda.synchronize()
            del old  # its memory is the next tensor's of this size
            if scores:
                m = host(ctx.attn_scores_message(i, g, ks[i], q, planes[0], planes[1 + i]), ctx.bw)
                assert (m[~seen] == 0).all() and m[seen].any()
            else:
                m = host(ctx.attn_mix_message(i, g, km[i], p, planes[0], planes[1 + i]), ctx.bw)
                assert (m[last] == 0).all() and m[:last].any()


def test_gate_eval_keys(ctx):
    """A key of another gate or of fewer words is refused; a gate without keys takes none."""
    x = dev(words(np.random.default_rng(1), (100,), ctx.bw))
    k0, k1, _ = ctx.gate_keygen(mpcx.TRRELU, x)
    short, _, _ = ctx.gate_keygen(mpcx.TRRELU, x[:40].contiguous())
    other, _, _ = ctx.gate_keygen(mpcx.TR, x)
    assert other.numel() < k0.numel()
    ctx.gate_eval(mpcx.TRRELU, k0, k1, x)
    for a, b in ((short, k1), (k0, short), (other, k1), (k0, k1.cpu()), (k0[1:], k1)):
        with pytest.raises(mpcx.MpcxError):
            ctx.gate_eval(mpcx.TRRELU, a, b, x)
    word = host(x, ctx.bw).view(np.int32 if ctx.bw == 32 else np.int64)
    assert np.array_equal(host(ctx.gate_eval(mpcx.LOCALARS, None, None, x), ctx.bw).view(word.dtype), word >> 12)


# ---------------- streams ----------------
def test_which_calls_wait_for_their_stream(ctx):
    """On the caller's stream the products only enqueue; the gates' evaluations and
    the keygens wait."""
    import torch
    B = Batch(ctx.bw, 1, 2, 20, 2, 1, 16, 4, "causal", seed=6)
    g, planes = B.gpu(), [dev(v) for v in (B.y, B.b0, B.b1)]
    q, p = dev(words(B.rng, (B.tokens, 2, 16), ctx.bw)), dev(words(B.rng, (B.n,), ctx.bw))
    w, scale = dev(q4_pack(B.rng.integers(-8, 8, (50, 32)))), dev(B.rng.integers(1, 99, (1, 50)).astype(np.int32))
    slot, rows = dev(np.arange(B.tokens)), q[:, :1]
    stream, big = torch.cuda.Stream(), torch.empty(1 << 30, dtype=torch.uint8, device="cuda")
    ctx.set_stream(stream)
    with torch.cuda.stream(stream):
        ks, km = ctx.attn_scores_keygen(g, q, *planes[1:]), ctx.attn_mix_keygen(g, p, *planes[1:])
        k0, k1, _ = ctx.gate_keygen(mpcx.TR, q)
        calls = {
            "ring_gemm_q4": lambda: ctx.ring_gemm_q4(q.view(-1, 32), w, scale, 32),
            "cache_append": lambda: ctx.cache_append([(rows, planes[0], False)], slot),
            "split_mask": lambda: ctx.split_mask(q),
            "attn_scores_eval": lambda: ctx.attn_scores_eval(g, *ks[:2], q, *planes),
            "attn_mix_eval": lambda: ctx.attn_mix_eval(g, *km[:2], p, *planes),
            "attn_scores_message": lambda: ctx.attn_scores_message(0, g, ks[0], q, *planes[:2]),
            "attn_mix_message": lambda: ctx.attn_mix_message(0, g, km[0], p, *planes[:2]),
            "gate_eval": lambda: ctx.gate_eval(mpcx.TR, k0, k1, q),
            "attn_scores_keygen": lambda: ctx.attn_scores_keygen(g, q, *planes[1:]),
            "attn_mix_keygen": lambda: ctx.attn_mix_keygen(g, p, *planes[1:])}
        for call in calls.values():
            call()
        done = {}
        for name, call in calls.items():
            torch.cuda.synchronize()
            for k in range(64):  # some 20 ms
                big.fill_(k)
            call()
            done[name] = stream.query()
        torch.cuda.synchronize()
    ctx.set_stream(None)
    waits = {"gate_eval", "attn_scores_keygen", "attn_mix_keygen"}
    assert done == {name: name in waits for name in calls}


# ---------------- the layer ----------------
def test_layer_evaluates_without_host_data(monkeypatch):
    """Weights, tables and the bias are on the GPU before the first step."""
    import attention
    took = []
    evaluate, copy = attention.Layer.evaluate, mpcx.to_dev

    def watched(self, *a):
        monkeypatch.setattr(mpcx, "to_dev", lambda x: took.append(x.shape) or copy(x))
        try:
            return evaluate(self, *a)
        finally:
            monkeypatch.setattr(mpcx, "to_dev", copy)

    monkeypatch.setattr(attention.Layer, "evaluate", watched)
    assert attention.run(32, singles=1, say=lambda line: None)
    assert took == []
