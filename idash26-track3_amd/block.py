"""A secure decoder: blocks of norm, attention, norm and 8-bit layers, one after another.

Two parties evaluate, on masked values, pre-norm transformer blocks with public weights:
the residual's addition and root-mean-square norm, the attention layer of attention.py,
the norm again, and two layers of 8-bit weights with ReLU between them; behind the last
block a norm and the output layer.  The norm is the two gates norm_sums and norm_scale;
between them the reciprocal root of one word a token is taken with the gates there are,
a table of 256 entries and one Newton step.  A prompt's tokens and single tokens take the
same calls.  The dealer makes the keys of a step beforehand, by the same steps on the
masks: a step is written once (Decoder.step) and run by the dealer, by the parties and in
plain integers.

`python block.py [--bw 64]` runs a prompt and a few single tokens of two sequences and
compares the outputs with plain fixed-point arithmetic, bit for bit.
"""
import argparse
import time

import numpy as np

import attention
import mpcx


class Weights8:
    """A public matrix (N, K) as 8-bit weights with a scale for each output channel:
    steps at the fixed-point scale s, w ~ step * q, q in -127..127."""

    def __init__(self, w, s):
        self.step = np.maximum(1, np.round(np.abs(w).max(1) / 127 * (1 << s))).astype(np.int64)
        self.q = np.clip(np.round(w * (1 << s) / self.step[:, None]), -127, 127).astype(np.int8)
        rows = np.zeros((w.shape[0], (w.shape[1] + 15) // 16 * 16), np.int8)  # rows of whole 16 bytes
        rows[:, :w.shape[1]] = self.q
        self.rows = mpcx.to_dev(rows.view(np.uint8)).view(mpcx._torch().int8)
        self.scale = mpcx.to_dev(self.step.astype(np.int32))

    def __call__(self, ctx, x):
        return ctx.ring_gemm_q8(x, self.rows, self.scale)

    def plain(self, x):
        return x @ self.q.T.astype(np.int64) * self.step


class Norm:
    """y = gain * h / rms(h) for rows h of dim words at scale s.  The mean square, at
    scale s + 2, is looked up in steps of 1/64 (up to 4: index i holds half the reciprocal
    root of (i + 1/2) / 64) and refined by v = p (3 - 4 m p^2), m the mean square."""

    def __init__(self, ctx, dim, gain=None):
        s = self.s = ctx.s
        self.per = round((1 << (s + 2)) / dim)
        self.table = np.round((1 << s) / 2 / np.sqrt((np.arange(256) + 0.5) / 64)).astype(np.int64)
        self.dev_table = _words(ctx, self.table)
        self.gain = gain
        self.dev_gain = _words(ctx, gain) if gain is not None else None

    def root(self, m, z):
        """1 / rms from the sum of squares (scale 2 s)."""
        ms = m.gate(mpcx.TR, m.gate(mpcx.TR, z) * self.per)
        p = m.lookup(m.gate(mpcx.TR, ms * 16), self)
        b = m.gate(mpcx.TR, m.product(ms, m.gate(mpcx.TR, m.product(p, p))))
        return m.gate(mpcx.TR, m.product(p, m.shifted(b * -1, 3 << self.s)))

    def __call__(self, m, x, d):
        """x + d (x where d is None), and its norm."""
        h, z, shares = m.sums(x, d)
        y = m.gate(mpcx.TR, m.scaled(h, self.root(m, z), shares, self))
        return h, (m.gate(mpcx.TR, y) if self.gain is not None else y)


def _words(ctx, v):
    return mpcx.to_dev(np.ascontiguousarray(v).astype(np.int64).astype(np.int32 if ctx.bw == 32 else np.int64))


class _Calls:
    """What the dealer and the parties share: calls on GPU tensors, gate by gate."""

    def __init__(self, ctx):
        self.ctx = ctx

    def _call(self, name, *args):
        """A C call on tensors, in torch's order."""
        same = self.ctx._enter()
        ptrs = [a.data_ptr() if hasattr(a, "data_ptr") else a for a in args]
        self.ctx.check(getattr(self.ctx.lib, "mpcx_" + name)(self.ctx.h, *ptrs), name)
        self.ctx._leave(same)

    def _map(self, n):  # element i of both operands of a product
        torch = mpcx._torch()
        return torch.arange(n, dtype=torch.int32, device=self.ctx._device)

    def linear(self, w, x):
        return w(self.ctx, x)


class Dealer(_Calls):
    """A step on the masks: the keys of its gates, in order."""

    def __init__(self, ctx, seed):
        super().__init__(ctx)
        self.seed, self.keys = seed, []

    def _id(self):
        return 16 * len(self.keys)

    def _keep(self, k0, k1):
        self.keys.append((k0, k1))

    def _keys(self, nb):
        self._keep(mpcx.empty_dev(nb, self.ctx._device), mpcx.empty_dev(nb, self.ctx._device))
        return self.keys[-1]

    def gate(self, kind, x):
        k0, k1, r = self.ctx.gate_keygen(kind, x.contiguous(), self.seed, self._id())
        self._keep(k0, k1)
        return r

    def product(self, x, y):
        n, r, g, at = x.numel(), self.ctx._new(x.shape), self._id(), self._map(x.numel())
        keys = self._keys(self.ctx.lib.mpcx_mul_key_bytes(self.ctx.h, n, n, n))
        self._call("mul_keygen", n, n, n, at, at, x, y, r, self.seed, g, *keys)
        self.ctx.sync()  # the call is only enqueued: its operands are read until then
        return r

    def lookup(self, x, norm):
        n, r, g = x.numel(), self.ctx._new(x.shape), self._id()
        keys = self._keys(self.ctx.lib.mpcx_lut8_key_bytes(self.ctx.h, n))
        self._call("lut8_keygen", n, x, r, self.seed, g, *keys)
        self.ctx.sync()
        return r

    def shifted(self, x, c):
        return x  # a public addend has no mask

    def sums(self, x, d):
        k0, k1, h, z = self.ctx.norm_sums_keygen(x, d, self.seed, self._id())
        self._keep(k0, k1)
        return h, z, (k0, k1)

    def scaled(self, h, v, shares, norm):
        k0, k1, r = self.ctx.norm_scale_keygen(*shares, v, h.shape[1], norm.dev_gain, self.seed, self._id())
        self._keep(k0, k1)
        return r

    def attend(self, layer, cache, place, x):
        keys, r = layer.deal(cache, *place[:3], x.contiguous(), self.seed + ((len(self.keys) + 1) << 32))
        self.keys.append(keys)
        return r


class Parties(_Calls):
    """A step on masked values, both parties, with the keys of the dealer's step."""

    def __init__(self, ctx, keys):
        super().__init__(ctx)
        self.keys = iter(keys)

    def gate(self, kind, x):
        return self.ctx.gate_eval(kind, *next(self.keys), x.contiguous())

    def product(self, x, y):
        n, z, at = x.numel(), self.ctx._new(x.shape), self._map(x.numel())
        self._call("mul_eval", n, n, n, at, at, *next(self.keys), x, y, z)
        return z

    def lookup(self, x, norm):
        y = self.ctx._new(x.shape)
        self._call("lut8_eval", x.numel(), *next(self.keys), norm.dev_table, x, y)
        return y

    def shifted(self, x, c):
        return x + c

    def sums(self, x, d):
        keys = next(self.keys)
        return (*self.ctx.norm_sums_eval(*keys, x, d), keys)

    def scaled(self, h, v, shares, norm):
        return self.ctx.norm_scale_eval(*next(self.keys), *shares, h, v, norm.dev_gain)

    def attend(self, layer, cache, place, x):
        return layer.evaluate(cache, *place[:3], next(self.keys), x.contiguous())


class Plain:
    """A step in plain fixed-point integers (numpy); states: each layer's keys and values."""

    def __init__(self, s, states):
        self.s, self.states = s, states

    def gate(self, kind, x):
        return np.maximum(x >> self.s, 0) if kind == mpcx.TRRELU else x >> self.s

    def product(self, x, y):
        return x * y

    def lookup(self, x, norm):
        return norm.table[x & 255]

    def shifted(self, x, c):
        return x + c

    def sums(self, x, d):
        h = x if d is None else x + d
        return h, (h * h).sum(1), None

    def scaled(self, h, v, shares, norm):
        return h * v[:, None] * (1 if norm.gain is None else norm.gain)

    def linear(self, w, x):
        return w.plain(x)

    def attend(self, layer, cache, place, x):
        return layer.plain(self.states[id(layer)], place[3], x)


class Decoder:
    def __init__(self, ctx, blocks, model, heads, kv, dim, hidden, words, seed=5):
        """Weights of random initialisation.  The 64-bit ring has room for a norm's gain
        (three scales); over the 32-bit one it is taken to be in the weights behind it."""
        rng = np.random.default_rng(seed)
        self.ctx, s = ctx, ctx.s

        def norm():
            gain = np.round(rng.normal(1, 0.1, model) * (1 << s)).astype(np.int64)
            return Norm(ctx, model, gain if ctx.bw == 64 else None)

        def weights(n, k, std):
            return Weights8(rng.normal(0, std / k ** 0.5, (n, k)), s)

        def layer(i):  # its weights as small as rows of root mean square one need
            a = attention.Layer(ctx, model, heads, kv, dim, seed=seed + 1 + i)
            a.w_in = attention.Weights(rng.normal(0, 0.3 / model ** 0.5, ((heads + 2 * kv) * dim, model)), s)
            return a

        self.blocks = [(norm(), layer(i), norm(), weights(hidden, model, 0.8), weights(model, hidden, 0.6))
                       for i in range(blocks)]
        self.last, self.head = norm(), weights(words, model, 0.5)

    def caches(self, seqs, page, pages):
        return [attention.Cache(self.ctx, seqs, b[1].kv, b[1].dim, page, pages) for b in self.blocks]

    def places(self, caches, counts):
        """Each layer's room for the step's tokens."""
        return [b[1].batch(c, counts) for b, c in zip(self.blocks, caches)]

    def step(self, m, caches, places, x):
        """The outputs of a step's tokens (tokens, words) from their rows (tokens, model)."""
        d = None
        for (norm1, layer, norm2, up, down), cache, place in zip(self.blocks, caches, places):
            x, y = norm1(m, x, d)
            d = m.attend(layer, cache, place, y)
            x, y = norm2(m, x, d)
            d = m.gate(mpcx.TR, m.linear(down, m.gate(mpcx.TRRELU, m.linear(up, y))))
        x, y = self.last(m, x, d)
        return m.gate(mpcx.TR, m.linear(self.head, y))


def run(bw=32, blocks=2, model=96, heads=4, kv=2, dim=24, hidden=200, words=130, page=8, prompts=(21, 13), singles=3,
        say=print):
    """A prompt and some single tokens of each sequence; returns whether every output
    is the plain one."""
    ctx = mpcx.Ctx(bw=bw, scale=12)
    net = Decoder(ctx, blocks, model, heads, kv, dim, hidden, words)
    caches = net.caches(len(prompts), page, -(-(max(prompts) + singles) // page))
    states = {id(b[1]): [([], []) for _ in prompts] for b in net.blocks}
    rng = np.random.default_rng(2)
    same = True
    for step in range(1 + singles):
        counts = list(prompts) if step == 0 else [1] * len(prompts)
        x = np.round(rng.normal(0, 0.5, (sum(counts), model)) * (1 << ctx.s)).astype(np.int64)
        rx = rng.integers(-(1 << 63), 1 << 63, x.shape, dtype=np.int64)
        places = net.places(caches, counts)
        dealer = Dealer(ctx, seed=100 + step)
        rout = net.step(dealer, caches, places, _words(ctx, rx))
        xhat = _words(ctx, x + rx)
        ctx.reset_counters()
        t = time.perf_counter()
        yhat = net.step(Parties(ctx, dealer.keys), caches, places, xhat)
        ctx.sync()
        t = time.perf_counter() - t
        y = (yhat - rout).cpu().numpy().astype(np.int64)
        ok = bool(np.array_equal(y, net.step(Plain(ctx.s, states), caches, places, x)))
        same &= ok
        say(f"{sum(counts)} tokens: {t * 1e3:.2f} ms, {ctx.rounds} rounds, {ctx.bytes_exchanged} bytes exchanged, "
            f"{'bit-exact' if ok else 'DIFFERS from the plain decoder'}")
    ctx.close()
    return same


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--bw", type=int, default=32, choices=(32, 64))
    raise SystemExit(0 if run(ap.parse_args().bw) else 1)
