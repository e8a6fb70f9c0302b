"""The operators of secure transformer inference as cases that can be timed.

Four operators on ring words (modulo 2^bw, bw = 32 or 64), each exact:

- "q4": masked activations times public 4-bit weights with group scales;
- "append": masked keys and values, with both parties' shares of their masks,
  into a paged cache, positions rotated on the way;
- "scores": the Beaver gate of the products query . key over that cache, with a
  bias that depends on distance and a range of visible keys per query token;
- "mix": the Beaver gate of the weighted sums of values over the same ranges.

`listed()` gives the named cases, `draw(rng)` one more of the same ranges,
`prepare` what a program holds before the call, `run` one pass and its outputs
(plain torch operations, or the framework's calls where `own` is true), `work`
the bytes and operations a pass cannot do without, `exact` the outputs from the
definition on the CPU.

Ring words are held in int32 (bw = 32) or int64 tensors.  Masked values and mask
shares are uniform words, which is how the parties see them.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False  # True: `run` calls the framework's operators

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "idash26-track3_amd")
F = 12  # fixed-point scale of the rotation tables


def listed():
    return [
        # one token through a square projection: the latency of a decode step
        {"name": "q4 1x4096x4096", "op": "q4", "bw": 32, "M": 1, "K": 4096, "N": 4096, "group": 128},
        # a few tokens through a wide layer of odd width in the 64-bit ring
        {"name": "q4 5x8192x2047 ring64", "op": "q4", "bw": 64, "M": 5, "K": 8192, "N": 2047, "group": 64},
        # the affinity model's first fully connected layer on a batch of 64
        {"name": "q4 64x312x1024", "op": "q4", "bw": 32, "M": 64, "K": 312, "N": 1024, "group": 32},
        # the tokens of a prompt through a projection
        {"name": "q4 768x4096x4096", "op": "q4", "bw": 32, "M": 768, "K": 4096, "N": 4096, "group": 128},
        # a decode step of 48 sequences: one row each into the cache
        {"name": "append 48", "op": "append", "bw": 32, "tokens": 48, "kv": 8, "dim": 128, "rot": 128,
         "pairs": False, "page": 16},
        # prompts of 6000 tokens, only half of each head rotated, 64-bit ring
        {"name": "append 6000 ring64", "op": "append", "bw": 64, "tokens": 6000, "kv": 4, "dim": 80, "rot": 40,
         "pairs": True, "page": 32},
        # one sequence at the start of its answer, 64-bit ring: the smallest call
        {"name": "scores 1x500 ring64", "op": "scores", "bw": 64, "seqs": 1, "q": 1, "keys": 500, "heads": 8, "kv": 8,
         "dim": 64, "page": 16, "mask": "causal", "bias": False},
        # a decode step of 8 sequences with a few thousand keys each, shared heads
        {"name": "scores 8x4096", "op": "scores", "bw": 32, "seqs": 8, "q": 1, "keys": 4096, "heads": 32, "kv": 8,
         "dim": 128, "page": 64, "mask": "causal", "bias": True},
        # four prompts with a prefix visible to every token, bias by distance
        {"name": "scores prompt 4x512", "op": "scores", "bw": 32, "seqs": 4, "q": 512, "keys": 512, "heads": 8, "kv": 2,
         "dim": 64, "page": 16, "mask": "prefix", "bias": True},
        # the weighted sums of the decode step above
        {"name": "mix 8x4096", "op": "mix", "bw": 32, "seqs": 8, "q": 1, "keys": 4096, "heads": 32, "kv": 8,
         "dim": 128, "page": 64, "mask": "causal"},
        # one long document, one token
        {"name": "mix 1x50000", "op": "mix", "bw": 32, "seqs": 1, "q": 1, "keys": 50000, "heads": 16, "kv": 4,
         "dim": 128, "page": 128, "mask": "causal"},
        # ragged prompts in a padded batch (tokens that see nothing), odd sizes, 64-bit ring
        {"name": "mix prompt 3x301 ring64", "op": "mix", "bw": 64, "seqs": 3, "q": 301, "keys": 301, "heads": 6,
         "kv": 3, "dim": 72, "page": 16, "mask": "padded"},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, its logarithm uniform."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["q4", "q4", "append", "scores", "mix"])
    c = {"op": op, "bw": rng.choice([32, 64])}
    if op == "q4":
        c["group"] = rng.choice([32, 64, 128])
        c["K"], c["N"] = _log(rng, 256, 8192), _log(rng, 256, 8192)
        c["M"] = _log(rng, 1, max(1, min(1024, (768 * 4096 * 4096 >> (c["bw"] == 64)) // (c["K"] * c["N"]))))
    elif op == "append":
        c["tokens"], c["kv"] = _log(rng, 1, 8000), rng.choice([1, 2, 4, 8])
        c["dim"] = rng.choice([64, 72, 80, 96, 128])
        c["rot"] = rng.choice([c["dim"], c["dim"] // 4 * 2])
        c["pairs"], c["page"] = rng.random() < 0.5, rng.choice([1, 16, 24, 64, 256])
    else:
        c["kv"] = rng.choice([1, 2, 3, 4, 8])
        c["heads"] = c["kv"] * rng.choice([1, 2, 4, 5, 8])
        c["dim"] = rng.choice([64, 72, 80, 96, 128])
        c["page"] = rng.choice([1, 16, 24, 64, 256])
        c["mask"] = rng.choice(["causal", "prefix", "window", "padded"])
        if rng.random() < 0.6:  # single tokens
            c["q"], c["seqs"] = rng.choice([1, 1, 1, 2, 3]), _log(rng, 1, 32)
            c["keys"] = _log(rng, 16, max(17, min(50000, (1 << 24 if c["bw"] == 32 else 1 << 23)
                                                   // (c["seqs"] * c["kv"] * c["dim"]))))
        else:
            c["seqs"] = rng.choice([1, 2, 3, 4])
            c["q"] = _log(rng, 16, max(17, int(math.sqrt((1 << 22) / (c["seqs"] * c["heads"])))))
            c["keys"] = c["q"] + rng.choice([0, 0, rng.randint(1, 500)])
        if op == "scores":
            c["bias"] = rng.random() < 0.5
    return c


# ---------------- inputs ----------------
def _words(g, shape, bw):
    """Uniform ring words."""
    n = math.prod(shape) if isinstance(shape, (tuple, list)) else shape
    b = torch.randint(0, 256, (n * bw // 8,), dtype=torch.uint8, device="cuda", generator=g)
    return b.view(torch.int32 if bw == 32 else torch.int64).view(shape)


def _up(n):
    """Key planes start at whole 256 bytes."""
    return (n + 255) // 256 * 256


def _ragged(c):
    """Lengths and visible ranges of an attention case, by its sizes alone: per
    sequence the query tokens and keys, per token its sequence, its place in it,
    its position, and the range [lo, hi) of keys it sees."""
    r = random.Random("%(seqs)d %(q)d %(keys)d %(heads)d %(kv)d" % c)
    nq, nk, seq, at, pos, lo, hi = [], [], [], [], [], [], []
    for b in range(c["seqs"]):
        n = c["q"] if b == 0 else r.randint((c["q"] + 1) // 2, c["q"])
        k = c["keys"] if b == 0 else r.randint(max(n, c["keys"] // 2), c["keys"])
        nq.append(n)
        nk.append(k)
        for i in range(n):
            p = k - n + i  # the queries are the sequence's last tokens
            a, z = 0, p + 1
            if c["mask"] == "prefix":
                z = max(z, k // 4)
            elif c["mask"] == "window":
                a = max(0, z - max(1, c["keys"] // 4))
            elif c["mask"] == "padded" and i % 8 == 7:  # a padding token sees nothing
                a = z = 0
            seq.append(b)
            at.append(i)
            pos.append(p)
            lo.append(a)
            hi.append(z)
    return nq, nk, seq, at, pos, lo, hi


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    bw = c["bw"]

    def whole(lo, hi, shape, dtype=torch.int32):
        return torch.randint(lo, hi, shape, dtype=dtype, device="cuda", generator=g)

    s = {"op": c["op"], "bw": bw}
    if c["op"] == "q4":
        groups = -(-c["K"] // c["group"])
        s["group"], s["K"] = c["group"], c["K"]
        s["a"] = _words(g, (c["M"], c["K"]), bw)
        # two weights a byte, the even one in the low half; rows of whole 32
        s["q"] = whole(0, 256, (c["N"], (c["K"] + 31) // 32 * 16), torch.uint8)
        # group scales: steps of a few hundredths at scale 12 to a few units at scale 12
        s["scale"] = whole(16, 1 << 14, (groups, c["N"]))
        return s
    if c["op"] == "append":
        t, kv, d = c["tokens"], c["kv"], c["dim"]
        n_pages = -(-t // c["page"]) + 8
        s |= {"rot": c["rot"], "pairs": c["pairs"], "kv": kv, "dim": d}
        # the projections' outputs hold queries, keys and values side by side
        s["rows"] = [_words(g, (t, 4 * kv * d), bw) for _ in range(3)]
        s["pools"] = [_words(g, (n_pages, kv, c["page"], d), bw) for _ in range(6)]
        order = torch.randperm(n_pages * c["page"], generator=g, device="cuda")[:t]
        s["slot"] = order.to(torch.int64)
        s["pos"] = whole(0, 8192, (t,))
        angle = torch.arange(8192, device="cuda", dtype=torch.float64)[:, None] * torch.pow(
            10000.0, -torch.arange(c["rot"] // 2, device="cuda", dtype=torch.float64) * 2 / c["rot"])
        word = torch.int32 if bw == 32 else torch.int64
        s["cos"] = torch.round(torch.cos(angle) * (1 << F)).to(word)
        s["sin"] = torch.round(torch.sin(angle) * (1 << F)).to(word)
        return s
    nq, nk, seq, at, pos, lo, hi = _ragged(c)
    tokens, heads, kv, d, page = len(seq), c["heads"], c["kv"], c["dim"], c["page"]
    off = [0]
    for a, z in zip(lo, hi):
        off.append(off[-1] + heads * (z - a))
    s["n_scores"] = off[-1]
    used = [-(-k // page) for k in nk]
    n_pages = sum(used) + 4
    perm = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((c["seqs"], max(used)), dtype=torch.int32, device="cuda")
    done = 0
    for b, u in enumerate(used):
        table[b, :u] = perm[done:done + u]
        done += u

    def ints(v, dtype=torch.int32):
        return torch.tensor(v, dtype=dtype, device="cuda")

    start = [0]
    for n in nq:
        start.append(start[-1] + n)
    s |= {"heads": heads, "max_q": max(nq), "max_keys": max(nk), "pages": table, "qstart": ints(start), "lo": ints(lo),
          "hi": ints(hi), "off": ints(off[:-1], torch.int64), "pos": ints(pos), "seq": ints(seq, torch.int64),
          "at": ints(at, torch.int64)}
    s["cache"] = [_words(g, (n_pages, kv, page, d), bw) for _ in range(3)]  # masked rows, party 0's shares, party 1's
    tb = bw // 8
    rows, wide = tokens * heads * d * tb, s["n_scores"] * tb
    first, second = (rows, wide) if c["op"] == "scores" else (wide, rows)
    # both parties' keys: the share of the left operand's mask, then of the product term
    s["key"] = [torch.randint(0, 256, (_up(first) + _up(second),), dtype=torch.uint8, device="cuda", generator=g)
                for _ in range(2)]
    s["x"] = _words(g, (tokens, heads, d) if c["op"] == "scores" else (s["n_scores"],), bw)
    s["dim"] = d
    s["slope"] = _words(g, (heads,), bw) % 4096 if c.get("bias") else None
    return s


# ---------------- the plain forms ----------------
def _limbs(x, bw):
    """16-bit limbs of ring words, as float64: products of limbs and their sums
    are exact there."""
    return [((x.to(torch.int64) >> (16 * i)) & 0xFFFF).double() for i in range(bw // 16)]


def _ring_matmul(x, y, bw):
    """x (..., M, K) times y (..., K, N) modulo 2^bw."""
    xs, ys = _limbs(x, bw), _limbs(y, bw)
    n = bw // 16
    parts = [torch.matmul(xs[i], ys[j]).to(torch.int64) << (16 * (i + j)) for i in range(n) for j in range(n - i)]
    return sum(parts[1:], parts[0]).to(x.dtype)


def _plain_q4(s):
    q, bw = s["q"], s["bw"]
    w = torch.stack((q & 15, q >> 4), dim=-1).view(q.shape[0], -1)[:, :s["K"]].to(torch.int32)
    w = (w ^ 8) - 8
    scale = s["scale"].t().repeat_interleave(s["group"], dim=1)[:, :s["K"]]
    w = (w * scale).double().t()  # below 2^53 beside a 16-bit limb and K terms
    parts = [torch.matmul(x, w).to(torch.int64) << (16 * i) for i, x in enumerate(_limbs(s["a"], bw))]
    return sum(parts[1:], parts[0]).to(s["a"].dtype)


def _split(s):
    """The rows to append: queries, keys, values side by side in each plane."""
    kd = s["kv"] * s["dim"]
    keys = [r[:, 2 * kd:3 * kd].view(-1, s["kv"], s["dim"]) for r in s["rows"]]
    values = [r[:, 3 * kd:].view(-1, s["kv"], s["dim"]) for r in s["rows"]]
    return keys, values


def _plain_append(s):
    keys, values = _split(s)
    h, pos = s["rot"] // 2, s["pos"].to(torch.int64)
    cos, sin = s["cos"][pos][:, None, :], s["sin"][pos][:, None, :]
    page = s["pools"][0].shape[2]
    at, off = s["slot"] // page, s["slot"] % page

    def rotated(x):
        a, b = (x[..., 0:2 * h:2], x[..., 1:2 * h:2]) if s["pairs"] else (x[..., :h], x[..., h:2 * h])
        u, v = cos * a - sin * b, sin * a + cos * b
        front = torch.stack((u, v), dim=-1).flatten(-2) if s["pairs"] else torch.cat((u, v), dim=-1)
        return torch.cat((front, x[..., 2 * h:] << F), dim=-1)

    [pool.__setitem__((at, slice(None), off), y) for pool, y in zip(s["pools"], [rotated(k) for k in keys] + values)]
    return s["pools"]


def _dense_cache(s):
    """The pages of each sequence, as (plane)(sequence, head, key, dim)."""
    pages = s["pages"].to(torch.int64)
    return [p[pages].permute(0, 2, 1, 3, 4).flatten(2, 3) for p in s["cache"]]


def _packed_index(s):
    """Per packed score: its token, head and key."""
    n = s["n_scores"]
    width = (s["hi"] - s["lo"]).to(torch.int64)
    tok = torch.repeat_interleave(torch.arange(width.numel(), device="cuda"), width * s["heads"], output_size=n)
    rem = torch.arange(n, device="cuda") - s["off"][tok]
    return tok, rem // width[tok], rem % width[tok] + s["lo"][tok]


def _key_planes(s, first, second):
    word = torch.int32 if s["bw"] == 32 else torch.int64
    tb = s["bw"] // 8
    a = [k[:first * tb].view(word) for k in s["key"]]
    b = [k[_up(first * tb):_up(first * tb) + second * tb].view(word) for k in s["key"]]
    return a, b


def _plain_scores(s):
    tokens, heads, d, bw = s["x"].shape[0], s["heads"], s["dim"], s["bw"]
    (a0, a1), (c0, c1) = _key_planes(s, tokens * heads * d, s["n_scores"])
    k, b0, b1 = [p.transpose(2, 3).contiguous() for p in _dense_cache(s)]  # (sequence, kv head, dim, key)
    kv, keys = k.shape[1], k.shape[3]

    def rows(x):  # (sequence, kv head, tokens x heads of it, dim)
        t = torch.zeros((k.shape[0], s["max_q"], heads, d), dtype=x.dtype, device="cuda")
        t[s["seq"], s["at"]] = x.view(tokens, heads, d)
        return t.view(k.shape[0], s["max_q"], kv, heads // kv, d).transpose(1, 2).flatten(2, 3)

    x, a0, a1 = rows(s["x"]), rows(a0), rows(a1)
    z = _ring_matmul(x - a0, k - b0, bw) - _ring_matmul(x, b1, bw) - _ring_matmul(a1, k, bw)
    z = z.view(k.shape[0], kv, s["max_q"], heads // kv, keys).transpose(1, 2).flatten(2, 3)
    tok, head, key = _packed_index(s)
    out = z[s["seq"][tok], s["at"][tok], head, key] + c0 + c1
    if s["slope"] is not None:
        out = out + s["slope"][head] * (key - s["pos"][tok]).to(out.dtype)
    return out


def _plain_mix(s):
    tokens, heads, d, bw = s["lo"].numel(), s["heads"], s["dim"], s["bw"]
    (a0, a1), (c0, c1) = _key_planes(s, s["n_scores"], tokens * heads * d)
    v, b0, b1 = _dense_cache(s)
    kv, keys = v.shape[1], v.shape[2]
    tok, head, key = _packed_index(s)

    def rows(x):  # (sequence, kv head, tokens x heads of it, key), zero where nothing is seen
        t = torch.zeros((v.shape[0], s["max_q"], heads, keys), dtype=x.dtype, device="cuda")
        t[s["seq"][tok], s["at"][tok], head, key] = x
        return t.view(v.shape[0], s["max_q"], kv, heads // kv, keys).transpose(1, 2).flatten(2, 3)

    x, a0, a1 = rows(s["x"]), rows(a0), rows(a1)
    z = _ring_matmul(x - a0, v - b0, bw) - _ring_matmul(x, b1, bw) - _ring_matmul(a1, v, bw)
    z = z.view(v.shape[0], kv, s["max_q"], heads // kv, d).transpose(1, 2).flatten(2, 3)
    return z[s["seq"], s["at"]] + (c0 + c1).view(tokens, heads, d)


# ---------------- the framework's calls ----------------
_ctx = {}


def _context(bw):
    """The program's context of this ring and the stream it works on."""
    if bw not in _ctx:
        if PKG not in sys.path:
            sys.path.insert(0, PKG)
        import mpcx

        stream = torch.cuda.Stream()
        ctx = mpcx.Ctx(bw=bw, scale=F)
        ctx.set_stream(stream)
        _ctx[bw] = (mpcx, ctx, stream)
    return _ctx[bw]


def _own_run(s):
    mpcx, ctx, stream = _context(s["bw"])
    with torch.cuda.stream(stream):
        if s["op"] == "q4":
            return ctx.ring_gemm_q4(s["a"], s["q"], s["scale"], s["group"])
        if s["op"] == "append":
            keys, values = _split(s)
            rotation = mpcx.Rotation(s["cos"], s["sin"], F, pairs=s["pairs"])
            planes = [(r, p, i < 3) for i, (r, p) in enumerate(zip(keys + values, s["pools"]))]
            ctx.cache_append(planes, s["slot"], s["pos"], rotation)
            return s["pools"]
        batch = mpcx.AttnBatch(s["pages"], s["qstart"], s["lo"], s["hi"], s["off"], s["n_scores"], s["heads"],
                               s["max_q"], s["max_keys"])
        if s["op"] == "scores":
            return ctx.attn_scores_eval(batch, *s["key"], s["x"], *s["cache"], slope=s["slope"], pos=s["pos"])
        return ctx.attn_mix_eval(batch, *s["key"], s["x"], *s["cache"])


def run(state):
    if own:
        return _own_run(state)
    return {"q4": _plain_q4, "append": _plain_append, "scores": _plain_scores, "mix": _plain_mix}[state["op"]](state)


def work(case):
    """Each input read once, each output written once; a ring multiply-add counts
    as two operations."""
    c, tb = case, case["bw"] // 8
    if c["op"] == "q4":
        m, k, n = c["M"], c["K"], c["N"]
        return {"bytes": m * k * tb + n * ((k + 31) // 32 * 16) + 4 * n * -(-k // c["group"]) + m * n * tb,
                "flops": 2 * m * k * n}
    if c["op"] == "append":
        rows = c["tokens"] * c["kv"] * c["dim"]
        return {"bytes": 12 * rows * tb + c["tokens"] * (12 + min(c["tokens"], 8192) / c["tokens"] * c["rot"] * tb),
                "flops": 3 * c["tokens"] * c["kv"] * c["rot"] * 3}
    nq, nk, seq, at, pos, lo, hi = _ragged(c)
    scores = c["heads"] * sum(z - a for a, z in zip(lo, hi))
    seen = 0
    for b in range(c["seqs"]):
        r = [(a, z) for a, z, q in zip(lo, hi, seq) if q == b and z > a]
        seen += max(z for _, z in r) - min(a for a, _ in r) if r else 0
    rows = len(seq) * c["heads"] * c["dim"]
    return {"bytes": 3 * (rows + scores + seen * c["kv"] * c["dim"]) * tb, "flops": 6 * scores * c["dim"]}


# ---------------- from the definition, on the CPU ----------------
def exact(case, seed):
    c = case
    if work(c)["flops"] > 4e9:
        return None
    s = prepare(c, seed)
    bits = np.uint32 if c["bw"] == 32 else np.uint64

    def host(t):
        return t.cpu().numpy().view(bits)

    def out(x):
        return torch.from_numpy(np.ascontiguousarray(x).view(np.int32 if c["bw"] == 32 else np.int64))

    if c["op"] == "q4":
        nib = s["q"].cpu().numpy()
        w = np.zeros((c["N"], c["K"]), np.int64)
        w[:, 0::2] = (nib & 15)[:, :(c["K"] + 1) // 2]
        w[:, 1::2] = (nib >> 4)[:, :c["K"] // 2]
        w[w > 7] -= 16
        a, scale = host(s["a"]).astype(np.uint64), s["scale"].cpu().numpy().astype(np.int64)
        z = np.zeros((c["M"], c["N"]), np.uint64)
        for i in range(scale.shape[0]):
            k = slice(i * c["group"], (i + 1) * c["group"])
            z += np.matmul(a[:, k], w[:, k].T.astype(np.uint64)) * scale[i].astype(np.uint64)
        return out(z.astype(bits))
    if c["op"] == "append":
        kd, h, page = c["kv"] * c["dim"], c["rot"] // 2, c["page"]
        cos, sin = host(s["cos"]), host(s["sin"])
        pools = [host(p).copy() for p in s["pools"]]
        slot, pos = s["slot"].cpu().numpy(), s["pos"].cpu().numpy()
        rows = [host(r) for r in s["rows"]]
        for t in range(c["tokens"]):
            co, si = cos[pos[t]], sin[pos[t]]
            for p in range(3):
                x = rows[p][t, 2 * kd:3 * kd].reshape(c["kv"], c["dim"])
                y = x << bits(F)
                i = np.arange(h)
                u, v = (2 * i, 2 * i + 1) if c["pairs"] else (i, i + h)
                y[:, u] = co * x[:, u] - si * x[:, v]
                y[:, v] = si * x[:, u] + co * x[:, v]
                pools[p][slot[t] // page, :, slot[t] % page] = y
                pools[3 + p][slot[t] // page, :, slot[t] % page] = rows[p][t, 3 * kd:].reshape(c["kv"], c["dim"])
        return [out(p) for p in pools]
    nq, nk, seq, at, pos, lo, hi = _ragged(c)
    heads, d, page, group = c["heads"], c["dim"], c["page"], c["heads"] // c["kv"]
    rows, n = len(seq) * heads * d, s["n_scores"]
    first, second = (rows, n) if c["op"] == "scores" else (n, rows)
    key = [k.cpu().numpy() for k in s["key"]]
    tb = c["bw"] // 8
    a0, a1 = [k[:first * tb].view(bits) for k in key]
    c0, c1 = [k[_up(first * tb):_up(first * tb) + second * tb].view(bits) for k in key]
    cache, table, x = [host(p) for p in s["cache"]], s["pages"].cpu().numpy(), host(s["x"]).reshape(-1)
    slope = host(s["slope"]) if s["slope"] is not None else None
    z = c0 + c1
    done = 0
    lines = [[p[table[b]].transpose(1, 0, 2, 3).reshape(c["kv"], -1, d) for p in cache] for b in range(c["seqs"])]
    for t in range(len(seq)):
        w = hi[t] - lo[t]
        for h in range(heads):
            y, y0, y1 = [p[h // group, lo[t]:hi[t]] for p in lines[seq[t]]]
            wide, row = slice(done, done + w), slice((t * heads + h) * d, (t * heads + h + 1) * d)
            left, to = (row, wide) if c["op"] == "scores" else (wide, row)
            if c["op"] == "scores":
                y, y0, y1 = y.T, y0.T, y1.T
            p, r0, r1 = x[left], a0[left], a1[left]
            if w:
                z[to] += np.matmul(p - r0, y - y0) - np.matmul(p, y1) - np.matmul(r1, y)
                if slope is not None:
                    z[to] += slope[h] * (np.arange(lo[t], hi[t]) - pos[t]).astype(bits)
            done += w
    return out(z if c["op"] == "scores" else z.reshape(len(seq), heads, d))
