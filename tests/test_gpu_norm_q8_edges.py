"""The 8-bit products and the norm's gates where buffers, streams, graphs and sizes meet
their ends.  All results are ring words, so every comparison is of all bits."""
import numpy as np
import pytest

import mpcx
from test_gpu_norm_q8 import key_planes, q8_plain, q8_rows, q8_wide
from test_gpu_transformer import dev, host, words

pytestmark = pytest.mark.gpu
EINVAL = 1


@pytest.fixture(scope="module", params=[32, 64])
def ctx(request):
    c = mpcx.Ctx(bw=request.param, scale=12)
    yield c
    c.close()


def places(n, apart=1 << 18):
    """Addresses of n buffers of one allocation, `apart` bytes from each other."""
    import torch
    buf = torch.zeros(n * apart, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    return buf, [buf.data_ptr() + i * apart for i in range(n)]


def refused(ctx, call, what, cases):
    for bad in cases:
        assert call(**bad) == EINVAL, bad
        assert what in ctx.lib.mpcx_last_error(ctx.h), bad


# ---------------- refusals ----------------
def test_q8_refusals(ctx):
    tb = ctx.bw // 8
    buf, (a, q, s, t, c) = places(5)
    M, K, N, ldq = 6, 72, 40, 80

    def call(M=M, K=K, N=N, a=a, lda=K, q=q, ldq=ldq, s=s, t=t, c=c, ldc=N):
        return ctx.lib.mpcx_ring_gemm_q8(ctx.h, M, K, N, a, lda, q, ldq, s, t, c, ldc)

    assert call() == 0 and call(s=None) == 0 and call(t=None) == 0
    refused(ctx, call, b"bad argument", [
        dict(M=0), dict(K=0), dict(N=0), dict(M=-1), dict(K=-1), dict(N=-5), dict(M=(1 << 31) - 1), dict(N=(1 << 31) - 1),
        dict(K=(1 << 24) + 1, lda=1 << 25, ldq=1 << 25), dict(lda=K - 1), dict(ldc=N - 1), dict(ldq=K - 8), dict(ldq=K),
        dict(ldq=88), dict(ldq=0)])
    refused(ctx, call, b"null pointer", [dict(a=None), dict(q=None), dict(c=None)])
    refused(ctx, call, b"misaligned", [dict(a=a + 1), dict(a=a + tb // 2), dict(q=q + 8), dict(q=q + 1), dict(s=s + 2),
                                       dict(t=t + 1), dict(c=c + tb // 2)])
    refused(ctx, call, b"overlaps", [
        dict(c=a), dict(c=a + (M * K - 1) * tb), dict(a=c + (M * N - 1) * tb), dict(c=q), dict(c=q + (N - 1) * ldq + 64),
        dict(c=s), dict(c=s + 4 * N - tb), dict(c=t), dict(c=t + 4 * M - tb), dict(lda=K + N, c=a + (K - 1) * tb, ldc=K + N),
        dict(lda=K + N, c=a + (K + 1) * tb, ldc=K + N)])
    # side by side in one matrix; between the weights' rows; just past them
    assert call(lda=K + N, c=a + K * tb, ldc=K + N) == 0
    assert call(M=1, N=1, c=q + 72, ldq=80) == 0 and call(c=q + (N - 1) * ldq + 72) == 0
    ctx.sync()


def test_norm_sums_refusals(ctx):
    tb = ctx.bw // 8
    buf, (k0, k1, x, d, h, s) = places(6)
    rows, dim, kb = 6, 50, ctx.lib.mpcx_norm_sums_key_bytes(ctx.h, 6, 50)
    n = rows * dim * tb

    def call(rows=rows, dim=dim, k0=k0, k1=k1, x=x, ldx=dim, d=d, ldd=dim, h=h, ldh=dim, s=s):
        return ctx.lib.mpcx_norm_sums_eval(ctx.h, rows, dim, k0, k1, x, ldx, d, ldd, h, ldh, s)

    def message(party=0, k0=k0, **kw):
        v = dict(rows=rows, dim=dim, x=x, ldx=dim, d=d, ldd=dim, h=h, ldh=dim, s=s)
        v.update(kw)
        return ctx.lib.mpcx_norm_sums_message(ctx.h, party, v["rows"], v["dim"], k0, v["x"], v["ldx"], v["d"], v["ldd"],
                                              v["h"], v["ldh"], v["s"])

    def keygen(k0=k0, k1=k1, **kw):
        v = dict(rows=rows, dim=dim, x=x, ldx=dim, d=d, ldd=dim, h=h, ldh=dim, s=s)
        v.update(kw)
        return ctx.lib.mpcx_norm_sums_keygen(ctx.h, v["rows"], v["dim"], v["x"], v["ldx"], v["d"], v["ldd"], v["h"],
                                             v["ldh"], v["s"], 1, 1, k0, k1)

    for f in (call, message, keygen):
        assert f() == 0 and f(d=None, h=None) == 0 and f(h=x) == 0 and f(h=d) == 0 and f(x=d) == 0
        assert f(ldx=99, ldd=60, ldh=51) == 0 and f(ldx=60, h=x, ldh=60) == 0
        assert f(rows=0, x=None, d=None, h=None, s=None) == 0
        refused(ctx, f, b"bad argument", [dict(dim=0), dict(dim=-3), dict(rows=1 << 60), dict(rows=(1 << 64) - 1, dim=1)])
        refused(ctx, f, b"rows overlap", [dict(ldx=dim - 1), dict(ldd=dim - 1), dict(ldh=0)])
        refused(ctx, f, b"null pointer", [dict(x=None), dict(s=None), dict(h=None), dict(k0=None)])
        refused(ctx, f, b"without a residual", [dict(d=None)])
        refused(ctx, f, b"misaligned", [dict(x=x + tb // 2), dict(d=d + 1), dict(h=h + 1), dict(s=s + tb // 2),
                                        dict(k0=k0 + 8)])
        refused(ctx, f, b"overlaps", [
            dict(h=x + tb), dict(h=x + n - tb), dict(h=d + tb), dict(s=x), dict(s=d + n - tb), dict(s=h), dict(h=s),
            dict(h=k0), dict(s=k0 + kb - tb), dict(h=x, ldh=dim + 1), dict(h=x, x=x, ldx=60, ldh=61), dict(h=k0 + kb - tb)])
    for f in (call, keygen):
        refused(ctx, f, b"null pointer", [dict(k1=None)])
        refused(ctx, f, b"overlaps", [dict(h=k1), dict(s=k1 + n - tb)])
        refused(ctx, f, b"misaligned", [dict(k1=k1 + 8)])
    refused(ctx, keygen, b"overlaps", [dict(k0=k1), dict(k0=k1 + kb - 16), dict(k1=x), dict(k0=d), dict(x=k1 + n - tb)])
    refused(ctx, message, b"bad party", [dict(party=2), dict(party=-1)])
    assert message(party=1, k0=k1) == 0
    ctx.sync()


def test_norm_scale_refusals(ctx):
    tb = ctx.bw // 8
    buf, (k0, k1, a0, a1, h, v, g, y) = places(8)
    rows, dim, kb = 6, 50, ctx.lib.mpcx_norm_scale_key_bytes(ctx.h, 6, 50)
    n = rows * dim * tb

    def call(rows=rows, dim=dim, k0=k0, k1=k1, a0=a0, a1=a1, h=h, ldh=dim, v=v, g=g, y=y, ldy=dim):
        return ctx.lib.mpcx_norm_scale_eval(ctx.h, rows, dim, k0, k1, a0, a1, h, ldh, v, g, y, ldy)

    def message(party=0, rows=rows, dim=dim, k0=k0, a0=a0, h=h, ldh=dim, v=v, g=g, y=y, ldy=dim):
        return ctx.lib.mpcx_norm_scale_message(ctx.h, party, rows, dim, k0, a0, h, ldh, v, g, y, ldy)

    def keygen(rows=rows, dim=dim, a0=a0, a1=a1, v=v, g=g, y=y, k0=k0, k1=k1):
        return ctx.lib.mpcx_norm_scale_keygen(ctx.h, rows, dim, a0, a1, v, g, y, 1, 1, k0, k1)

    for f in (call, message, keygen):
        assert f() == 0 and f(g=None) == 0 and f(rows=0, y=None) == 0
        refused(ctx, f, b"bad argument", [dict(dim=0), dict(dim=-3), dict(rows=1 << 60)])
        refused(ctx, f, b"null pointer", [dict(k0=None), dict(a0=None), dict(v=None), dict(y=None)])
        refused(ctx, f, b"misaligned", [dict(k0=k0 + 8), dict(a0=a0 + 1), dict(v=v + tb // 2), dict(g=g + 1), dict(y=y + 1)])
        refused(ctx, f, b"overlaps", [dict(y=k0 + kb - tb), dict(y=a0), dict(y=a0 + n - tb), dict(y=v), dict(y=g + dim * tb - tb)])
    for f in (call, message):
        assert f(y=h) == 0 and f(ldh=60, ldy=77) == 0 and f(y=h, ldh=60, ldy=60) == 0
        refused(ctx, f, b"rows overlap", [dict(ldh=dim - 1), dict(ldy=dim - 1)])
        refused(ctx, f, b"null pointer", [dict(h=None)])
        refused(ctx, f, b"overlaps", [dict(y=h + tb), dict(y=h, ldy=51), dict(y=h + n - tb)])
    for f in (call, keygen):
        refused(ctx, f, b"null pointer", [dict(k1=None), dict(a1=None)])
        refused(ctx, f, b"overlaps", [dict(y=k1), dict(y=a1 + tb)])
    refused(ctx, keygen, b"overlaps", [dict(k0=k1), dict(k1=a0), dict(k0=a1 + n - 16), dict(k0=v), dict(k1=g)])
    refused(ctx, message, b"bad party", [dict(party=2)])
    ctx.sync()


def test_key_bytes(ctx):
    tb, up = ctx.bw // 8, lambda n: (n + 255) // 256 * 256
    for rows, dim in ((1, 1), (3, 100), (1 << 33, 5)):
        assert ctx.lib.mpcx_norm_sums_key_bytes(ctx.h, rows, dim) == up(up(rows * dim * tb) + rows * tb)
        assert ctx.lib.mpcx_norm_scale_key_bytes(ctx.h, rows, dim) == up(up(rows * tb) + rows * dim * tb)
    for f in (ctx.lib.mpcx_norm_sums_key_bytes, ctx.lib.mpcx_norm_scale_key_bytes):
        assert f(ctx.h, 5, 0) == f(ctx.h, 5, -1) == f(ctx.h, (1 << 60) + 1, 1) == f(None, 5, 5) == f(ctx.h, 0, 5) == 0


@pytest.mark.parametrize("M", [3, 70])
def test_q8_into_columns_of_its_operand(ctx, M):
    """Input and output side by side in one matrix."""
    rng = np.random.default_rng(M)
    K, N = 96, 50
    big, w = words(rng, (M, K + N + 3), ctx.bw), rng.integers(-128, 128, (N, K))
    d = dev(big)
    ctx.ring_gemm_q8(d[:, :K], q8_rows(w), out=d[:, K + 1:K + 1 + N])
    big[:, K + 1:K + 1 + N] = q8_plain(big[:, :K], w)
    assert np.array_equal(host(d, ctx.bw), big)


# ---------------- streams and graphs ----------------
def calls_of(ctx, rng, M):
    """Each call on inputs of its own, with the tensors that change between replays and the
    outputs; products that split K, that do not, and of few rows."""
    import torch
    out = []
    for K, N in ((2000, 70), (100, 300)):
        a, q, s = dev(words(rng, (M, K), ctx.bw)), q8_rows(rng.integers(-128, 128, (N, K))), dev(
            rng.integers(1, 99, N).astype(np.int32))
        c = torch.empty((M, N), dtype=a.dtype, device="cuda")
        out.append((a, lambda a=a, q=q, s=s, c=c: ctx.ring_gemm_q8(a, q, s, out=c), (c,)))
    x, d = dev(words(rng, (M, 200), ctx.bw)), dev(words(rng, (M, 200), ctx.bw))
    v, g = dev(words(rng, (M,), ctx.bw)), dev(words(rng, (200,), ctx.bw))
    k0, k1, _, _ = ctx.norm_sums_keygen(x, d, seed=3)
    q0, q1, _ = ctx.norm_scale_keygen(k0, k1, v, 200, g, seed=4)
    h, y, m = (torch.empty_like(x) for _ in range(3))
    s0, s1 = torch.empty_like(v), torch.empty_like(v)
    out.append((x, lambda: s0.copy_(ctx.norm_sums_eval(k0, k1, x, d, h)[1]), (h, s0)))
    out.append((d, lambda: s1.copy_(ctx.norm_sums_message(1, k1, x, d, y)[1]), (y, s1)))
    out.append((v, lambda: ctx.norm_scale_eval(q0, q1, k0, k1, d, v, g, m), (m,)))
    return out


@pytest.mark.parametrize("M", [1, 7, 40])
def test_graph_replays(ctx, M):
    """All evaluations captured in one graph; inputs change between replays, eager calls and
    synchronizations run in between, and every replay gives the eager results."""
    import torch
    rng = np.random.default_rng(M)
    stream = torch.cuda.Stream()
    ctx.set_stream(stream)
    try:
        with torch.cuda.stream(stream):
            calls = calls_of(ctx, rng, M)
            for _, call, _ in calls:
                call()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                for _, call, _ in calls:
                    call()
            for _ in range(4):
                for x, _, outs in calls:
                    x.copy_(dev(words(rng, tuple(x.shape), ctx.bw)))
                    for o in outs:
                        o.fill_(77)
                graph.replay()
                stream.synchronize()
                got = [[o.clone() for o in outs] for _, _, outs in calls]
                for _, call, _ in calls:
                    call()
                torch.cuda.synchronize()
                for g, (_, _, outs) in zip(got, calls):
                    assert all(torch.equal(a, b) for a, b in zip(g, outs))
    finally:
        ctx.set_stream(None)


def test_which_calls_wait_for_their_stream(ctx):
    """On the caller's stream the evaluations and messages only enqueue; the keygens wait."""
    import torch
    rng = np.random.default_rng(5)
    stream, big = torch.cuda.Stream(), torch.empty(1 << 30, dtype=torch.uint8, device="cuda")
    ctx.set_stream(stream)
    try:
        with torch.cuda.stream(stream):
            x, v, d = dev(words(rng, (9, 200), ctx.bw)), dev(words(rng, (9,), ctx.bw)), dev(words(rng, (9, 200), ctx.bw))
            k0, k1, _, _ = ctx.norm_sums_keygen(x, d)
            q0, q1, _ = ctx.norm_scale_keygen(k0, k1, v, 200)
            q = q8_rows(rng.integers(-128, 128, (70, 200)))
            calls = {
                "ring_gemm_q8": lambda: ctx.ring_gemm_q8(x, q),
                "norm_sums_eval": lambda: ctx.norm_sums_eval(k0, k1, x, d),
                "norm_sums_message": lambda: ctx.norm_sums_message(0, k0, x, d),
                "norm_scale_eval": lambda: ctx.norm_scale_eval(q0, q1, k0, k1, x, v),
                "norm_scale_message": lambda: ctx.norm_scale_message(0, q0, k0, x, v),
                "norm_sums_keygen": lambda: ctx.norm_sums_keygen(x, d),
                "norm_scale_keygen": lambda: ctx.norm_scale_keygen(k0, k1, v, 200)}
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
    finally:
        ctx.set_stream(None)
    assert done == {name: name.endswith("keygen") for name in calls}


def test_two_streams_at_once(ctx):
    """Two contexts on two streams, their products and gates interleaved."""
    import torch
    rng = np.random.default_rng(6)
    other = mpcx.Ctx(bw=ctx.bw, scale=12)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    want, made = [], []
    for c, s in zip((ctx, other), streams):
        made.append(calls_of(c, rng, 40))
        for _, call, outs in made[-1]:
            call()
        torch.cuda.synchronize()
        want.append([[o.clone() for o in outs] for _, _, outs in made[-1]])
        c.set_stream(s)
    for _, _, outs in made[0] + made[1]:
        for o in outs:
            o.zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(len(made[0])):
            for s, calls in zip(streams, made):
                with torch.cuda.stream(s):
                    calls[i][1]()
    torch.cuda.synchronize()
    ctx.set_stream(None)
    other.close()
    for w, calls in zip(want, made):
        for a, (_, _, outs) in zip(w, calls):
            assert all(torch.equal(x, y) for x, y in zip(a, outs))


def test_calls_from_another_stream(ctx):
    """Inputs made on torch's current stream, the context on its own: the calls wait for them,
    and are done when they return."""
    import torch
    rng = np.random.default_rng(7)
    big = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    a, w = words(rng, (30, 300), ctx.bw), rng.integers(-128, 128, (40, 300))
    q, src, x = q8_rows(w), dev(a), dev(np.zeros((30, 300), ctx.T))
    for k in range(40):
        big.fill_(k)
    x.copy_(src)
    assert np.array_equal(host(ctx.ring_gemm_q8(x, q), ctx.bw), q8_plain(a, w))


# ---------------- sizes ----------------
def test_places_past_32_bits():
    """Rows and outputs of more than 2^32 words: the last ones are right."""
    import torch
    c = mpcx.Ctx(bw=32, scale=12)
    rng = np.random.default_rng(8)
    M, K, N = (1 << 17) + 3, 16, 1 << 15
    w, last = rng.integers(-128, 128, (N, K)).astype(np.int8), words(rng, (40, K), 32)
    a = torch.zeros((M, K), dtype=torch.int32, device="cuda")
    a[M - 40:] = dev(last)
    out = torch.empty((M, N), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    c.ring_gemm_q8(a, q8_rows(w), out=out)
    assert np.array_equal(host(out[M - 40:], 32), q8_wide(last, w)) and not bool(out[:1000].any())
    del a
    # the gates' last rows, with shares of zero but the second party's of three
    v, a0, a1 = dev(words(rng, (M,), 32)), torch.zeros_like(out), torch.full_like(out, 3)
    nb = c.lib.mpcx_norm_sums_key_bytes(c.h, M, N), c.lib.mpcx_norm_scale_key_bytes(c.h, M, N)
    key = torch.zeros(max(nb), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    h = host(out[M - 40:], 32)
    _, s = c.norm_sums_eval(key, key, out)
    c.norm_scale_eval(key, key, a0, a1, out, v, out=out)
    with np.errstate(over="ignore"):
        assert np.array_equal(host(s[M - 40:], 32), np.square(h).sum(1, dtype=np.uint32))
        vv = host(v[M - 40:], 32)[:, None]
        assert np.array_equal(host(out[M - 40:], 32), h * vv - np.uint32(3) * vv)
    c.close()


def test_long_rows(ctx):
    """Rows of 2^20 words and one, single and a few."""
    rng = np.random.default_rng(9)
    for rows in (1, 3):
        dim = (1 << 20) + 1
        rx, x = words(rng, (rows, dim), ctx.bw), words(rng, (rows, dim), ctx.bw)
        k0, k1, _, rs = ctx.norm_sums_keygen(dev(rx))
        with np.errstate(over="ignore"):
            _, s = ctx.norm_sums_eval(k0, k1, dev(x + rx))
            assert np.array_equal(host(s, ctx.bw) - host(rs, ctx.bw), np.square(x).sum(1, dtype=ctx.T))


@pytest.mark.parametrize("rows,dim", [(1, 40001), (100, 65537)])
def test_graph_of_long_rows(ctx, rows, dim):
    """Sums that parts of a row add up: every replay begins them anew."""
    import torch
    rng = np.random.default_rng(dim)
    k0, k1, _, _ = ctx.norm_sums_keygen(dev(words(rng, (rows, dim), ctx.bw)))
    x = dev(words(rng, (rows, dim), ctx.bw))
    stream = torch.cuda.Stream()
    ctx.set_stream(stream)
    try:
        with torch.cuda.stream(stream):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                _, s = ctx.norm_sums_eval(k0, k1, x)
            for i in range(3):
                x.add_(i)
                graph.replay()
                stream.synchronize()
                assert torch.equal(s, ctx.norm_sums_eval(k0, k1, x)[1])
        with np.errstate(over="ignore"):
            v, a = host(x, ctx.bw), sum(key_planes(k, ctx.T, rows * dim, rows)[0].reshape(rows, dim) for k in (k0, k1))
            c = sum(key_planes(k, ctx.T, rows * dim, rows)[1] for k in (k0, k1))
            assert np.array_equal(host(s, ctx.bw), (v * (v - ctx.T(2) * a)).sum(1, dtype=ctx.T) + c)
    finally:
        ctx.set_stream(None)


@pytest.mark.parametrize("value", [0, 1 << 63, (1 << 64) - 1, 0x8000000080000000])
def test_rows_of_one_value(ctx, value):
    """Zeros, and words at the ends of the ring."""
    rows, dim = 5, 300
    x = np.full((rows, dim), value, np.uint64).astype(ctx.T)
    z = dev(x)
    k0, k1, _, rs = ctx.norm_sums_keygen(z, z)  # masks of the same value
    (a0, c0), (a1, c1) = (key_planes(k, ctx.T, rows * dim, rows) for k in (k0, k1))
    with np.errstate(over="ignore"):
        h = x + x
        assert np.array_equal(a0 + a1, h.reshape(-1)) and np.array_equal(
            c0 + c1, host(rs, ctx.bw) + np.square(h).sum(1, dtype=ctx.T))
        hh, s = ctx.norm_sums_eval(k0, k1, z, z)  # masked values that hide zeros
    assert np.array_equal(host(hh, ctx.bw), h) and np.array_equal(host(s, ctx.bw), host(rs, ctx.bw))


def test_key_bytes_at_their_end(ctx):
    """The most rows there are have keys whose bytes can be counted; one row more is refused."""
    tb, buf, (k0, k1, x, s) = ctx.bw // 8, *places(4)
    for most, dim in ((1 << 59, 1), ((1 << 59) // 3, 3)):
        for f in (ctx.lib.mpcx_norm_sums_key_bytes, ctx.lib.mpcx_norm_scale_key_bytes):
            assert f(ctx.h, most, dim) >= most * (dim + 1) * tb and f(ctx.h, most + 1, dim) == 0
            assert f(ctx.h, 1 << 60, 1) == 0
        refused(ctx, lambda rows: ctx.lib.mpcx_norm_sums_eval(ctx.h, rows, dim, k0, k1, x, dim, None, 0, None, 0, s),
                b"bad argument", [dict(rows=most + 1), dict(rows=1 << 60)])


def test_parties_reconstruct_the_norm(ctx):
    """Each party's messages from its own keys and shares, exchanged over a channel: both hold
    the gates' outputs."""
    import threading
    rng = np.random.default_rng(10)
    rows, dim = 7, 150
    x, d, g = (dev(words(rng, s, ctx.bw)) for s in ((rows, dim), (rows, dim), (dim,)))
    v = dev(words(rng, (rows,), ctx.bw))
    ks = ctx.norm_sums_keygen(x, d)
    kv = ctx.norm_scale_keygen(ks[0], ks[1], v, dim, g)
    h, s = ctx.norm_sums_eval(ks[0], ks[1], x, d)
    want = [host(s, ctx.bw), host(ctx.norm_scale_eval(kv[0], kv[1], ks[0], ks[1], h, v, g), ctx.bw).reshape(-1)]
    peers, got, errors = mpcx.Peer.pair(), {}, []

    def party(i):
        try:
            c = mpcx.Ctx(bw=ctx.bw, scale=12)
            hi, s = c.norm_sums_message(i, ks[i], x, d)
            y = c.norm_scale_message(i, kv[i], ks[i], hi, v, g)
            got[i] = [c.party_reconstruct(peers[i], host(m, ctx.bw).reshape(-1)) for m in (s, y)]
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
