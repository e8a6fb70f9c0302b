"""The 8-bit products and the norm of secure transformer inference as cases that can
be timed.

Three operators on ring words (modulo 2^bw, bw = 32 or 64), each exact:

- "q8": masked activations times public 8-bit weights, with a scale for each output
  channel and, where given, for each token;
- "sums": the residual's addition and, as a Beaver gate, each token's sum of squares
  (what a root-mean-square norm divides by);
- "scale": the Beaver gate of each token's row times its factor, with a public gain
  for each channel.

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
import sys

import numpy as np
import torch

own = False  # True: `run` calls the framework's operators

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "idash26-track3_amd")


def listed():
    return [
        # one token through a square projection: the latency of a decode step
        {"name": "q8 1x4096x4096", "op": "q8", "bw": 32, "M": 1, "K": 4096, "N": 4096, "tokens": False},
        # a decode step of a few sequences out of a layer of odd width, 64-bit ring
        {"name": "q8 6x8191x2048 ring64", "op": "q8", "bw": 64, "M": 6, "K": 8191, "N": 2048, "tokens": False},
        # the affinity model's first fully connected layer on a batch of 64
        {"name": "q8 64x312x1024", "op": "q8", "bw": 32, "M": 64, "K": 312, "N": 1024, "tokens": True},
        # a short ragged batch of prompts into a vocabulary of odd size, 64-bit ring
        {"name": "q8 150x1000x4099 ring64", "op": "q8", "bw": 64, "M": 150, "K": 1000, "N": 4099, "tokens": True},
        # the tokens of long prompts through a projection: the largest
        {"name": "q8 1000x4096x4096", "op": "q8", "bw": 32, "M": 1000, "K": 4096, "N": 4096, "tokens": False},
        # a decode step of one sequence: the smallest calls
        {"name": "sums 1x4096", "op": "sums", "bw": 32, "rows": 1, "dim": 4096, "residual": True},
        # a decode step of some sequences, odd width, 64-bit ring
        {"name": "sums 37x1279 ring64", "op": "sums", "bw": 64, "rows": 37, "dim": 1279, "residual": True},
        # a network's input, which has no residual yet, 64-bit ring
        {"name": "sums 4000x1000 ring64", "op": "sums", "bw": 64, "rows": 4000, "dim": 1000, "residual": False},
        # long prompts
        {"name": "sums 6000x4096", "op": "sums", "bw": 32, "rows": 6000, "dim": 4096, "residual": True},
        {"name": "scale 1x4096", "op": "scale", "bw": 32, "rows": 1, "dim": 4096, "gain": True},
        {"name": "scale 37x1279 ring64", "op": "scale", "bw": 64, "rows": 37, "dim": 1279, "gain": False},
        {"name": "scale 6000x4096", "op": "scale", "bw": 32, "rows": 6000, "dim": 4096, "gain": True},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, its logarithm uniform."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    c = {"op": rng.choice(["q8", "q8", "sums", "scale"]), "bw": rng.choice([32, 64])}
    if c["op"] == "q8":
        c["K"], c["N"] = _log(rng, 256, 8192), _log(rng, 256, 8192)
        c["M"] = _log(rng, 1, max(1, min(1024, (1000 * 4096 * 4096 >> (c["bw"] == 64)) // (c["K"] * c["N"]))))
        c["tokens"] = rng.random() < 0.5
        return c
    c["dim"] = _log(rng, 64, 8192)
    c["rows"] = _log(rng, 1, min(8192, (6000 * 4096 >> (c["bw"] == 64)) // c["dim"]))
    c["residual" if c["op"] == "sums" else "gain"] = rng.random() < 0.7
    return c


# ---------------- inputs ----------------
def _words(g, shape, bw):
    """Uniform ring words."""
    b = torch.randint(0, 256, (math.prod(shape) * bw // 8,), dtype=torch.uint8, device="cuda", generator=g)
    return b.view(torch.int32 if bw == 32 else torch.int64).view(shape)


def _up(n):
    """Key planes start at whole 256 bytes."""
    return (n + 255) // 256 * 256


def prepare(case, seed):
    c, bw = case, case["bw"]
    if own:
        _context(bw)  # before the inputs: they are made on its stream
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"op": c["op"], "bw": bw}

    def whole(lo, hi, shape, dtype=torch.int32):
        return torch.randint(lo, hi, shape, dtype=dtype, device="cuda", generator=g)

    def key(first, second):
        """A party's key: two planes of ring words."""
        return whole(0, 256, (_up(_up(first * bw // 8) + second * bw // 8),), torch.uint8)

    if c["op"] == "q8":
        s["K"] = c["K"]
        s["a"] = _words(g, (c["M"], c["K"]), bw)
        # rows of weights take whole 16 bytes
        s["q"] = whole(-128, 128, (c["N"], (c["K"] + 15) // 16 * 16), torch.int8)
        # channel scales: thousandths to a few units at scale 12; token scales about one
        s["scale"] = whole(4, 1 << 14, (c["N"],))
        s["tokens"] = whole(0, 1 << 13, (c["M"],)) if c["tokens"] else None
        return s
    t, d = c["rows"], c["dim"]
    s["h"] = _words(g, (t, d), bw)
    if c["op"] == "sums":
        s["d"] = _words(g, (t, d), bw) if c["residual"] else None
        s["key"] = [key(t * d, t) for _ in range(2)]  # shares of the rows' mask, then of the sums' term
        return s
    s["v"] = _words(g, (t,), bw)
    s["share"] = [_words(g, (t, d), bw) for _ in range(2)]
    s["key"] = [key(t, t * d) for _ in range(2)]  # shares of the factors' mask, then of the product term
    s["gain"] = _words(g, (d,), bw) % 8192 if c["gain"] else None
    return s


# ---------------- the plain forms ----------------
def _planes(s, first, second):
    """Both parties' two key planes."""
    word, tb = (torch.int32 if s["bw"] == 32 else torch.int64), s["bw"] // 8
    a = [k[:first * tb].view(word) for k in s["key"]]
    b = [k[_up(first * tb):_up(first * tb) + second * tb].view(word) for k in s["key"]]
    return a, b


def _plain_q8(s):
    a, bw = s["a"], s["bw"]
    w = s["q"][:, :s["K"]].double().t()
    out = 0
    for i in range(bw // 16):  # 16-bit limbs: their products and sums are exact in float64
        limb = ((a.to(torch.int64) >> (16 * i)) & 0xFFFF).double()
        out = out + (torch.matmul(limb, w).to(torch.int64) << (16 * i))
    out = out * s["scale"]
    if s["tokens"] is not None:
        out = out * s["tokens"][:, None]
    return out.to(a.dtype)


def _plain_sums(s):
    t, d = s["h"].shape
    (a0, a1), (c0, c1) = _planes(s, t * d, t)
    h = s["h"] + s["d"] if s["d"] is not None else s["h"]
    total = (h * (h - 2 * (a0 + a1).view(t, d))).sum(1).to(h.dtype) + c0 + c1
    return (h, total) if s["d"] is not None else total


def _plain_scale(s):
    h, v = s["h"], s["v"][:, None]
    t, d = h.shape
    (b0, b1), (c0, c1) = _planes(s, t, t * d)
    a0, a1 = s["share"]
    z = (h - a0) * (v - b0[:, None]) - h * b1[:, None] - a1 * v
    if s["gain"] is not None:
        z = z * s["gain"]
    return z + (c0 + c1).view(t, d)


# ---------------- the framework's calls ----------------
_ctx = {}


def _context(bw):
    """The program's context of this ring.  The program works on a stream of its own: from
    its first context on it is torch's current one, on which inputs are made, the
    calls enqueue and outputs are used.  Where a caller has made another stream current
    the calls wait for that one, and for their own work at their end."""
    if "stream" not in _ctx:
        stream = _ctx["stream"] = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.set_stream(stream)
    if bw not in _ctx:
        if PKG not in sys.path:
            sys.path.insert(0, PKG)
        import mpcx

        _ctx[bw] = mpcx.Ctx(bw=bw, scale=12)
        _ctx[bw].set_stream(_ctx["stream"])
    return _ctx[bw]


def _own_run(s):
    ctx = _context(s["bw"])
    if s["op"] == "q8":
        return ctx.ring_gemm_q8(s["a"], s["q"], s["scale"], s["tokens"])
    if s["op"] == "sums":
        h, total = ctx.norm_sums_eval(*s["key"], s["h"], s["d"])
        return (h, total) if s["d"] is not None else total
    return ctx.norm_scale_eval(*s["key"], *s["share"], s["h"], s["v"], s["gain"])


def run(state):
    if own:
        return _own_run(state)
    return {"q8": _plain_q8, "sums": _plain_sums, "scale": _plain_scale}[state["op"]](state)


def work(case):
    """Each input read once, each output written once; a ring multiply-add counts
    as two operations."""
    c, tb = case, case["bw"] // 8
    if c["op"] == "q8":
        m, k, n = c["M"], c["K"], c["N"]
        return {"bytes": m * k * tb + n * k + 4 * n + 4 * m * c["tokens"] + m * n * tb, "flops": 2 * m * k * n}
    t, d = c["rows"], c["dim"]
    if c["op"] == "sums":
        return {"bytes": (t * d * (5 if c["residual"] else 3) + 3 * t) * tb, "flops": 4 * t * d}
    return {"bytes": (t * d * 6 + 3 * t + d * c["gain"]) * tb, "flops": (6 + c["gain"]) * t * d}


# ---------------- from the definition, on the CPU ----------------
def exact(case, seed):
    c = case
    if work(c)["flops"] > 4e9:
        return None
    s = prepare(c, seed)
    bits = np.uint32 if c["bw"] == 32 else np.uint64
    tb = c["bw"] // 8

    def host(t):
        return t.cpu().numpy().view(bits)

    def out(x):
        return torch.from_numpy(np.ascontiguousarray(x).view(np.int32 if c["bw"] == 32 else np.int64))

    if c["op"] == "q8":
        a, q = host(s["a"]), s["q"].cpu().numpy()[:, :c["K"]].astype(np.int64).astype(bits)
        z = np.matmul(a, np.ascontiguousarray(q.T))
        z = z * s["scale"].cpu().numpy().astype(np.int64).astype(bits)
        if s["tokens"] is not None:
            z = z * s["tokens"].cpu().numpy().astype(np.int64).astype(bits)[:, None]
        return out(z)
    t, d = c["rows"], c["dim"]
    first, second = (t * d, t) if c["op"] == "sums" else (t, t * d)
    key = [k.cpu().numpy() for k in s["key"]]
    (l0, l1) = [k[:first * tb].view(bits) for k in key]
    (c0, c1) = [k[_up(first * tb):_up(first * tb) + second * tb].view(bits) for k in key]
    h = host(s["h"])
    # each party's message from its own shares, then their sum
    if c["op"] == "sums":
        if s["d"] is not None:
            h = h + host(s["d"])
        two, squares = bits(2), np.square(h)
        p0 = (squares - two * h * l0.reshape(t, d)).sum(1, dtype=bits) + c0
        p1 = c1 - two * (h * l1.reshape(t, d)).sum(1, dtype=bits)
        total = out(p0 + p1)
        return (out(h), total) if s["d"] is not None else total
    a0, a1 = [host(x) for x in s["share"]]
    v = host(s["v"])[:, None]
    gain = host(s["gain"]) if s["gain"] is not None else bits(1)
    p0 = gain * (h - a0) * (v - l0[:, None]) + c0.reshape(t, d)
    p1 = c1.reshape(t, d) - gain * (h * l1[:, None] + a1 * v)
    return out(p0 + p1)
