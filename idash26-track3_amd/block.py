"""A secure decoder: blocks of norm, attention, norm and 8-bit layers, one after another.

Two parties evaluate, on masked values, pre-norm transformer blocks with public weights:
the residual's addition and root-mean-square norm, the attention layer of attention.py,
the norm again, and two layers of 8-bit weights with ReLU between them; behind the last
block a norm and the output layer.  The norm is the two gates norm_sums and norm_scale;
between them the reciprocal root of one word a token is taken with the gates there are,
tables of 256 entries and one Newton step.  A prompt's tokens and single tokens take the
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


class Table:
    """A public function of a word in 0..255, as 256 ring words."""

    def __init__(self, ctx, values):
        self.values = np.asarray(values, np.int64)
        self.dev = _words(ctx, self.values)


class Norm:
    """y = gain * h / rms(h) for rows h of dim words at scale s.

    Within 1% (and the last floors: a unit of 2^-s, with a gain two) for rows of a root mean
    square in [low, high], a range of 64.  In Z_2^64 that is 0.34 to 15 at every width (0.24 to
    21 at some).  In Z_2^32 a sum of squares has to stay below 2^31 at twice the scale and the
    range ends there, at scale 12 at sqrt(120 / dim): 0.017 to 1.1 for 96 words, 0.0027 to
    0.17 for 4096.  Larger rows, up to the ring's end, are divided by `high`; smaller ones
    by something between 2/3 of `low` and `low`, as with an epsilon added, and rows of
    zeros stay zeros.  Widths and scales that leave no room are refused.

    The sum of squares z is cut to w, 240 2^e at the range's end and no more.  Three bands of
    w, each 16 times the last, have 8-bit indexes w >> e - 8, e - 4, e, of which 15 to 239 are
    the band's; below and above, a table holds the values at the band's ends, so that the
    bands' entries add up to the one of the band that w is in.  With z0 the middle of an
    entry's sums the tables hold p = 1 / (2 rms(z0)) and g, 1 / z0 in w's units, and v =
    p (3 - w g): one Newton step from p, off by 3/8 of the square of z / z0 - 1, which
    is 1/30 at most.  The width is in the tables, so nothing is divided by it."""

    BANDS = 3

    def __init__(self, ctx, dim, gain=None):
        s, bits, dim = ctx.s, ctx.bw - 1, int(dim)
        if dim < 1:
            raise ValueError(f"Norm: rows of {dim} words")
        wide = bits == 63
        high = min((dim - 1).bit_length() + 2 * s, bits - 8)  # sums of 240 2^high end the range
        drops = -(-(high - s) // s)                           # truncations to w
        e = high - drops * s
        lift = s - e if drops > 1 else 0                      # a shift behind the first, where there is room
        e += lift
        steps = dim * 4.0 ** s                                # sums over this: mean squares
        self.low, self.high = (15 * 2.0 ** (high - 8) / steps) ** 0.5, (240 * 2.0 ** high / steps) ** 0.5
        # w g has wg bits behind its truncations, v v_scale: 3 p, at most 1.5 / low, has to fit
        # the ring before v's
        wg, g_drops, v_drops = (s + 6, 1, 2) if wide else (26 - s, 1, 1) if s >= 12 else (8, 2, 1)
        v_scale = min(s, int(np.floor(bits + np.log2(self.low / 1.5))) - v_drops * s)
        p_end = 2.0 ** (v_scale + v_drops * s - wg) / (2 * self.high)  # the last entries
        g_end = 2.0 ** (g_drops * s + wg) / (240 * 2.0 ** e)
        # a word of the output before its truncations: sqrt(dim), where a row has but one word other
        # than zero (and 32/30 of that between the range's end and the ring's), and the gain
        word = 32 / 30 * dim ** 0.5 * 4.0 ** s * (1 if gain is None else max(int(np.abs(gain).max()), 1))
        if e < 10 or min(p_end, g_end) < 128 or word >= 2.0 ** bits:
            raise ValueError(f"Norm: rows of {dim} words at scale {s} in Z_2^{ctx.bw}: no room")
        self.s, self.e, self.lift, self.drops, self.wg, self.g_drops = s, e, lift, drops, wg, g_drops
        self.v_drops, self.v_scale = v_drops, v_scale
        at = np.arange(255, -1, -1)                           # the index is looked up from 255 down
        z = np.where((at < 15) | (at >= 240), 240, at + 0.5)  # in the last band, in 2^high

        def table(f, grows):  # at the band's lower end `grows` times what is at its upper
            v = np.round(f).astype(np.int64)
            return Table(ctx, np.where(at < 15, grows * v, v))

        self.p = table(p_end * np.sqrt(240 / z), 4)
        self.g = table(g_end * 240 / z, 16)
        # 256 2^s - 1 - 2^(s - e_j) w, w = 240 2^e - 1 - left
        by = [1 << (s - e + 4 * (self.BANDS - 1 - j)) for j in range(self.BANDS)]
        self.spread = Spread(ctx, by, [(256 << s) - 1 - k * ((240 << e) - 1) for k in by])
        self.gain = gain
        self.dev_gain = _words(ctx, gain) if gain is not None else None

    def _entry(self, m, index, table, grows):
        """The entry of the band that each word is in: a band's are `grows` times the next one's."""
        *below, total = m.lookup(index, table)  # a row for each
        weights = [grows ** (j + 1) for j in range(len(below))]
        for x, w in zip(reversed(below), weights):
            total = m.plus(total, x, w)
        return m.shifted(total, -int(table.values[0]) * sum(weights))  # the bands below give their upper ends

    def root(self, m, z):
        """1 / rms at scale v_scale from the sum of squares (scale 2 s)."""
        s, end = self.s, 240 << self.e
        for i in range(self.drops - 1):
            z = m.gate(mpcx.TR, z)
            z = z << self.lift if i == 0 and self.lift else z
        # w, rounded, is end - 1 less what is left of it, if that is positive
        left = m.gate(mpcx.TRRELU, m.less((end << s) - 1 - (1 << (s - 1)), z))
        index = m.gate(mpcx.TRRELU, m.spread(left, self.spread))  # 255 less it
        p, g = self._entry(m, index, self.p, 4), self._entry(m, index, self.g, 16)
        b = m.product(m.less(end - 1, left), g)
        for _ in range(self.g_drops):
            b = m.gate(mpcx.TR, b)
        v = m.product(p, m.less(3 << self.wg, b))
        for i in range(self.v_drops):
            v = m.gate(mpcx.TR, m.shifted(v, 1 << (s - 1)) if i + 1 == self.v_drops else v)
        return v

    def __call__(self, m, x, d):
        """x + d (x where d is None), and its norm."""
        h, z, shares = m.sums(x, d)
        y = m.scaled(h, self.root(m, z), shares, self)
        y = m.gate(mpcx.TR, y << (self.s - self.v_scale) if self.s > self.v_scale else y)
        return h, (m.gate(mpcx.TR, y) if self.gain is not None else y)


class Spread:
    """Words of `left` into the bands' indexes: times `by`, and `plus`, a row for each band."""

    def __init__(self, ctx, by, plus):
        self.by, self.plus = (np.array(v, np.int64)[:, None] for v in (by, plus))
        self.dev_by, self.dev_plus = _words(ctx, self.by), _words(ctx, self.plus)


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

    def plus(self, x, y, k):
        return mpcx._torch().add(x, y, alpha=k)


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

    def lookup(self, x, table):
        n, r, g = x.numel(), self.ctx._new(x.shape), self._id()
        keys = self._keys(self.ctx.lib.mpcx_lut8_key_bytes(self.ctx.h, n))
        self._call("lut8_keygen", n, x, r, self.seed, g, *keys)
        self.ctx.sync()
        return r

    def shifted(self, x, c):
        return x  # a public addend has no mask

    def less(self, c, x):
        return -x

    def spread(self, x, s):
        return x * s.dev_by

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

    def lookup(self, x, table):
        y = self.ctx._new(x.shape)
        self._call("lut8_eval", x.numel(), *next(self.keys), table.dev, x, y)
        return y

    def shifted(self, x, c):
        return x + c

    def less(self, c, x):
        return c - x

    def spread(self, x, s):
        return mpcx._torch().addcmul(s.dev_plus, x, s.dev_by)

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

    def lookup(self, x, table):
        return table.values[x & 255]

    def plus(self, x, y, k):
        return x + y * k

    def shifted(self, x, c):
        return x + c

    def less(self, c, x):
        return c - x

    def spread(self, x, s):
        return x * s.by + s.plus

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
        (three scales); over the 32-bit one it is taken to be in the weights behind it.  The
        residual stream's rows have to stay in the norms' range (Norm)."""
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
