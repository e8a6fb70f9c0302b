"""A secure attention layer over a paged cache: the transformer operators together.

Two parties evaluate, on masked values, one layer of ReLU attention with public
4-bit weights: projections, positions rotated, keys and values kept in a paged
cache of masked rows, scores with a bias that depends on distance, ReLU, weighted
sums, output projection; every product is followed by the exact truncation gate.
A prompt's tokens and single tokens take the same calls.  The dealer makes the
keys of a step beforehand, by the same calls on the masks.

`python attention.py [--bw 64]` runs a prompt and a few single tokens of two
sequences and compares the outputs with plain fixed-point arithmetic, bit for bit.
"""
import argparse
import time

import numpy as np
import torch

import mpcx


class Weights:
    """A public matrix (N, K) as 4-bit weights with group scales: steps at the
    fixed-point scale s, w ~ scale * q, q in -8..7."""

    def __init__(self, w, s, group=32):
        n, k = w.shape
        groups = -(-k // group)
        step = np.zeros((groups, n), np.int64)
        q = np.zeros((n, (k + 31) // 32 * 32), np.int64)
        for g in range(groups):
            part = w[:, g * group:(g + 1) * group]
            step[g] = np.maximum(1, np.round(np.abs(part).max(1) / 7 * (1 << s)))
            q[:, g * group:g * group + part.shape[1]] = np.clip(np.round(part * (1 << s) / step[g][:, None]), -8, 7)
        self.q, self.step, self.group, self.k = q[:, :k], step, group, k
        bits = q & 15
        self.packed = mpcx.to_dev((bits[:, 0::2] | bits[:, 1::2] << 4).astype(np.uint8))
        self.scale = mpcx.to_dev(step.astype(np.int32))

    def __call__(self, ctx, x):
        return ctx.ring_gemm_q4(x, self.packed, self.scale, self.group)

    def plain(self, x):
        w = self.q * np.repeat(self.step, self.group, 0)[:self.k].T
        return x @ w.T


class Cache:
    """Pages of one plane each for keys and values: masked rows and both parties'
    shares of their masks; and which pages a sequence has."""

    def __init__(self, ctx, seqs, kv, dim, page, pages_per_seq):
        self.page, self.seqs = page, seqs
        shape = (seqs * pages_per_seq, kv, page, dim)
        self.keys = [ctx._new(shape).zero_() for _ in range(3)]
        self.values = [ctx._new(shape).zero_() for _ in range(3)]
        order = np.random.default_rng(7).permutation(seqs * pages_per_seq)
        self.table = order.reshape(seqs, pages_per_seq).astype(np.int32)
        self.used = [0] * seqs

    def room(self, counts):
        """Slots and positions of the next counts[b] tokens of each sequence."""
        if max(u + n for u, n in zip(self.used, counts)) > self.table.shape[1] * self.page:
            raise ValueError("the sequences' pages are full")
        slot, pos, seq = [], [], []
        for b, n in enumerate(counts):
            for i in range(self.used[b], self.used[b] + n):
                slot.append(int(self.table[b, i // self.page]) * self.page + i % self.page)
                pos.append(i)
                seq.append(b)
            self.used[b] += n
        return np.array(slot, np.int64), np.array(pos, np.int32), np.array(seq, np.int32)


class Layer:
    def __init__(self, ctx, model, heads, kv, dim, seed=3, max_pos=512):
        rng = np.random.default_rng(seed)
        self.ctx, self.heads, self.kv, self.dim, self.model = ctx, heads, kv, dim, model
        s = ctx.s
        self.w_in = Weights(rng.normal(0, 0.6 / model ** 0.5, ((heads + 2 * kv) * dim, model)), s)
        self.w_out = Weights(rng.normal(0, 0.3 / (heads * dim) ** 0.5, (model, heads * dim)), s)
        angle = np.arange(max_pos)[:, None] * 10000.0 ** (-np.arange(dim // 2) * 2 / dim)
        self.cos, self.sin = np.round(np.cos(angle) * (1 << s)).astype(np.int64), \
            np.round(np.sin(angle) * (1 << s)).astype(np.int64)
        self.slope = np.round(2.0 ** (-np.arange(1, heads + 1)) * (1 << (2 * s)) / 64).astype(np.int64)
        self.bias = self._dev(self.slope)
        self.rotation = mpcx.Rotation(self._dev(self.cos), self._dev(self.sin), s)

    def _dev(self, v):
        return mpcx.to_dev(np.ascontiguousarray(v).astype(np.int64).astype(np.int32 if self.ctx.bw == 32 else np.int64))

    def batch(self, cache, counts):
        """The tokens of a step: where they go and what they see (each its sequence
        up to itself)."""
        if max(u + n for u, n in zip(cache.used, counts)) > len(self.cos):  # a row without a table row is not written
            raise ValueError(f"the rotation's tables have {len(self.cos)} positions")
        slot, pos, seq = cache.room(counts)
        start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        hi = pos + 1
        off = np.concatenate([[0], np.cumsum(self.heads * hi.astype(np.int64))])
        to = mpcx.to_dev
        b = mpcx.AttnBatch(to(cache.table).view(cache.seqs, -1), to(start), to(np.zeros_like(pos)), to(hi), to(off[:-1]),
                           int(off[-1]), self.heads, max(counts), max(cache.used))
        return b, to(slot), to(pos), (pos, seq)

    def _rotated(self, rows, n_heads, pos):
        """Rows with their positions turned, at twice the scale: appended to a scratch
        cache of one slot a page."""
        n = rows.shape[0]
        out = self.ctx._new((n, n_heads, 1, self.dim))
        slot = torch.arange(n, device=rows.device)
        self.ctx.cache_append([(rows, out, True)], slot, pos, self.rotation)
        return out.view(n, n_heads, self.dim)

    def _split(self, x):
        """Queries, keys and values of the joint projection's rows."""
        n, (h, k, d) = x.shape[0], (self.heads, self.kv, self.dim)
        return (x[:, a * d:b * d].unflatten(1, (b - a, d)) for a, b in ((0, h), (h, h + k), (h + k, h + 2 * k)))

    def deal(self, cache, batch, slot, pos, rx, seed):
        """The dealer's run of a step on the input's mask: every gate's keys, the
        shares that go into the cache, and the output's mask."""
        ctx, keys = self.ctx, {}

        def gate(name, kind, mask):
            keys[name] = ctx.gate_keygen(kind, mask.contiguous(), seed, len(keys) * 16)
            return keys[name][2]

        q, k, v = self._split(gate("in", mpcx.TR, self.w_in(ctx, rx)))
        q = gate("q", mpcx.TR, self._rotated(q, self.heads, pos))
        k = gate("k", mpcx.TR, self._rotated(k, self.kv, pos))
        ks, vs = ctx.split_mask(k, seed, 1000), ctx.split_mask(v.contiguous(), seed, 1001)
        planes = [(s, p, False) for s, p in zip(ks + vs, cache.keys[1:] + cache.values[1:])]
        ctx.cache_append(planes, slot)
        keys["scores"] = ctx.attn_scores_keygen(batch, q, *cache.keys[1:], seed=seed, gate=2000)
        p = gate("p", mpcx.TRRELU, keys["scores"][2])
        keys["mix"] = ctx.attn_mix_keygen(batch, p, *cache.values[1:], seed=seed, gate=2001)
        o = gate("o", mpcx.TR, keys["mix"][2])
        return keys, gate("out", mpcx.TR, self.w_out(ctx, o.flatten(1)))

    def evaluate(self, cache, batch, slot, pos, keys, xhat):
        """Both parties' run on masked values: the masked output (tokens, model)."""
        ctx = self.ctx

        def gate(name, kind, x):
            return ctx.gate_eval(kind, *keys[name][:2], x.contiguous())

        q, k, v = self._split(gate("in", mpcx.TR, self.w_in(ctx, xhat)))
        q = gate("q", mpcx.TR, self._rotated(q, self.heads, pos))
        k = gate("k", mpcx.TR, self._rotated(k, self.kv, pos))
        ctx.cache_append([(k, cache.keys[0], False), (v, cache.values[0], False)], slot)
        s = ctx.attn_scores_eval(batch, *keys["scores"][:2], q, *cache.keys, slope=self.bias, pos=pos)
        p = gate("p", mpcx.TRRELU, s)
        o = gate("o", mpcx.TR, ctx.attn_mix_eval(batch, *keys["mix"][:2], p, *cache.values))
        return gate("out", mpcx.TR, self.w_out(ctx, o.flatten(1)))

    def plain(self, state, where, x):
        """The same in plain fixed-point integers; state: the sequences' keys and values."""
        s, (h, kv, d) = self.ctx.s, (self.heads, self.kv, self.dim)
        pos, seq = where
        y = self.w_in.plain(x) >> s
        q, k, v = (y[:, a * d:b * d].reshape(len(x), b - a, d) for a, b in ((0, h), (h, h + kv), (h + kv, h + 2 * kv)))

        def turned(r):
            a, b, c, t = r[..., :d // 2], r[..., d // 2:], self.cos[pos][:, None], self.sin[pos][:, None]
            return np.concatenate([c * a - t * b, t * a + c * b], -1) >> s

        q, k = turned(q), turned(k)
        out = np.zeros((len(x), h * d), np.int64)
        for i, b in enumerate(seq):
            state[b][0].append(k[i])
            state[b][1].append(v[i])
            ks, vs = (np.repeat(np.stack(r), h // kv, 1) for r in state[b])
            score = np.einsum("hd,jhd->hj", q[i], ks) + self.slope[:, None] * (np.arange(len(ks)) - pos[i])
            out[i] = (np.einsum("hj,jhd->hd", np.maximum(score >> s, 0), vs) >> s).reshape(-1)
        return self.w_out.plain(out) >> s


def run(bw=32, model=96, heads=6, kv=2, dim=32, page=8, prompts=(21, 13), singles=4, say=print):
    """A prompt and some single tokens of each sequence; returns whether every output
    is the plain one."""
    ctx = mpcx.Ctx(bw=bw, scale=12)
    layer = Layer(ctx, model, heads, kv, dim)
    cache = Cache(ctx, len(prompts), kv, dim, page, -(-(max(prompts) + singles) // page))
    state = [([], []) for _ in prompts]
    rng = np.random.default_rng(1)
    same = True
    for step in range(1 + singles):
        counts = list(prompts) if step == 0 else [1] * len(prompts)
        x = np.round(rng.normal(0, 0.5, (sum(counts), model)) * (1 << ctx.s)).astype(np.int64)
        rx = rng.integers(-(1 << 63), 1 << 63, x.shape, dtype=np.int64)
        batch, slot, pos, where = layer.batch(cache, counts)
        keys, rout = layer.deal(cache, batch, slot, pos, layer._dev(rx), seed=100 + step)
        ctx.reset_counters()
        t = time.perf_counter()
        yhat = layer.evaluate(cache, batch, slot, pos, keys, layer._dev(x + rx))
        ctx.sync()
        t = time.perf_counter() - t
        y = (yhat - rout).cpu().numpy().astype(np.int64)
        ok = bool(np.array_equal(y, layer.plain(state, where, x)))
        same &= ok
        say(f"{sum(counts)} tokens: {t * 1e3:.2f} ms, {ctx.rounds} rounds, {ctx.bytes_exchanged} bytes exchanged, "
            f"{'bit-exact' if ok else 'DIFFERS from the plain layer'}")
    ctx.close()
    return same


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--bw", type=int, default=32, choices=(32, 64))
    raise SystemExit(0 if run(ap.parse_args().bw) else 1)
