"""The example decoder's norm in plain integers, on the CPU, against 64-bit floats: widths of
ordinary decoders, the whole range of sizes that it states, and what lies outside."""
import types

import numpy as np
import pytest

import block
import mpcx


class Ring(block.Plain):
    """Plain integers, none of which may leave the ring's signed range."""

    def __init__(self, bw, s):
        super().__init__(s, None)
        self.end = 1 << (bw - 1)

    def held(self, x):
        assert np.abs(x.astype(object) if x.size < 100 else x).max(initial=0) < self.end
        return x

    def gate(self, kind, x):
        return super().gate(kind, self.held(x))

    def product(self, x, y):
        assert (np.abs(x.astype(np.float64) * y) < self.end).all()
        return super().product(x, y)

    def lookup(self, x, *table):
        assert ((x >= 0) & (x < 256)).all()  # not wrapped
        return super().lookup(x, *table)

    def sums(self, x, d):
        h, z, shares = super().sums(x, d)
        assert ((h.astype(np.float64) ** 2).sum(1) < self.end).all()
        return h, z, shares

    def scaled(self, h, v, shares, norm):
        y = super().scaled(h, v, shares, norm)
        gain = 1 if norm.gain is None else np.abs(norm.gain)
        assert (np.abs(h.astype(np.float64)) * np.abs(v[:, None]) * gain < self.end).all()
        return y


@pytest.fixture
def norm(monkeypatch):
    monkeypatch.setattr(block, "_words", lambda ctx, v: None)
    return lambda bw, dim, gain=None, s=12: block.Norm(types.SimpleNamespace(s=s, bw=bw), dim, gain)


WIDE = [1, 2, 5, 64, 96, 200, 987, 1000, 1279, 2560, 3000, 4095, 4096, 4097, 5120, 6144, 7168, 8192,
        11008, 16384, 32768, 65537]
NARROW = [8, 30, 64, 96, 200, 987, 1000, 2560, 4096, 5120, 11008, 13000]


# What the root may lose, relative (by ring; the first and the third meet only where w is small or v is):
#   w       its last step's half unit and one unit of the floors before, in 15 of 2^-8 of the
#           top's step: 120 units (32 bits), 240: half of 1.5 / 120, 1.5 / 240          2^-7.3, 2^-8.3
#   index   half a step in 15: 3/8 (1/30)^2                                             2^-11.2
#   p       half a unit in its last entry: 132 (32), 5900                                2^-8, 2^-13.5
#   g       half a unit in its last entry: 136 (32), 1092, halved in the root            2^-9.1, 2^-12
#   v       half a unit in 2^V / high: 1058 (32), 186                                   2^-11, 2^-8.5
# together 2^-6.5 at most (32 bits, at the lower end) and 2^-7.3 (64, there); from twice the
# lower end on 2^-7.3 and 2^-8.
@pytest.mark.parametrize("bw,dim", [(64, d) for d in WIDE] + [(32, d) for d in NARROW])
def test_root(norm, bw, dim):
    n = norm(bw, dim)
    if bw == 64:
        assert n.low <= 0.35 and n.high >= 15
    else:  # up to the ring's end, 2^31 at twice the scale
        assert 115 / dim < n.high ** 2 < 128 / dim and n.low < n.high / 60
    rms = np.geomspace(n.low, n.high, 50001)
    z = np.floor(dim * rms * rms * 2 ** 24).astype(np.int64)
    v = n.root(Ring(bw, 12), z) / 2.0 ** n.v_scale
    true = np.sqrt(dim * 2.0 ** 24 / z)
    off = np.abs(v / true - 1)
    assert off.max() < 0.01
    assert off[rms > 2 * n.low].max() < 2 ** -7.3


@pytest.mark.parametrize("bw,dim", [(64, d) for d in (1, 96, 2560, 4096, 6144, 16384)] +
                         [(32, d) for d in (8, 96, 4096, 13000)])
def test_root_outside_its_range(norm, bw, dim):
    """Above: the factor of the range's upper end.  Below: never more than the true factor, nor than
    1.5 times that of the lower end."""
    n, m = norm(bw, dim), Ring(bw, 12)
    top = int(dim * n.high ** 2 * 2 ** 24)
    z = np.unique(np.geomspace(top, 2 ** (bw - 1) - 2049, 2001).astype(np.int64))
    v = n.root(m, z)
    assert v.min() == v.max() > 0 and abs(v[0] / 2.0 ** n.v_scale * n.high - 1) < 0.01
    z = np.arange(0, int(dim * n.low ** 2 * 2 ** 24), max(1, int(dim * n.low ** 2 * 2 ** 24) // 5000))
    v = n.root(m, z) / 2.0 ** n.v_scale
    assert (v > 0).all() and v.max() < 1.5 / n.low * 1.01
    assert (v[1:] * np.sqrt(z[1:] / (dim * 2.0 ** 24)) < 1.01).all()


@pytest.mark.parametrize("bw,dim,gain", [(64, 96, True), (64, 2560, False), (64, 3000, True), (64, 4096, True),
                                         (64, 6144, True), (64, 11008, False), (64, 16384, True), (32, 96, False), (32, 2560, False),
                                         (32, 4096, False), (32, 11008, False)])
def test_norm(norm, bw, dim, gain):
    """Whole rows, both ends of the range among them, and rows of zeros; one floor of a unit, with
    a gain two."""
    rng = np.random.default_rng(dim + bw)
    g = np.round(rng.normal(1, 0.1, dim) * 4096).astype(np.int64) if gain else None
    n = norm(bw, dim, g)
    rms = np.geomspace(n.low * 1.02, n.high * 0.98, 13)[:, None]
    x = rng.normal(0, 1, (13, dim))
    x = np.round(x / np.sqrt((x * x).mean(1, keepdims=True)) * rms * 4096).astype(np.int64)
    x = np.concatenate([x, np.zeros((1, dim), np.int64)])
    d = rng.integers(-1, 2, x.shape)
    d[-1] = 0
    h, y = n(Ring(bw, 12), x, d)
    size = np.sqrt((h.astype(np.float64) ** 2).mean(1, keepdims=True))
    want = h / np.maximum(size, 1e-9) * (1 if g is None else g / 4096)
    assert np.array_equal(h, x + d)
    assert (np.abs(y / 4096 - want) <= 0.01 * np.abs(want) + 2 / 4096).all()
    assert not y[-1].any()


def test_a_row_of_one_large_word(norm):
    """The largest word that a normed row can have."""
    for bw, dim in ((64, 16384), (32, 4096), (32, 13000)):
        n = norm(bw, dim)
        x = np.zeros((1, dim), np.int64)
        x[0, 3] = int(n.high * 0.99 * dim ** 0.5 * 4096)
        _, y = n(Ring(bw, 12), x, None)
        assert abs(y[0, 3] / 4096 / dim ** 0.5 - 1) < 0.01 and not y[0, 4:].any()


@pytest.mark.parametrize("s", [10, 11, 13, 14, 16, 18])
def test_other_scales(norm, s):
    for bw in (64, 32) if s <= 13 else (64,):
        for dim in (96, 1000, 4000):
            try:
                n = norm(bw, dim, None, s)
            except ValueError:
                assert bw == 32 and s >= 13  # rows' words past the ring
                continue
            z = np.floor(dim * np.geomspace(n.low, n.high, 20001) ** 2 * 4.0 ** s).astype(np.int64)
            v = n.root(Ring(bw, s), z) / 2.0 ** n.v_scale
            assert np.abs(v * np.sqrt(z / (dim * 4.0 ** s)) - 1).max() < (0.01 if s > 10 else 0.02)


@pytest.mark.parametrize("bw,dim,gain,s", [(64, 0, None, 12), (64, -4, None, 12), (32, 15000, None, 12), (32, 5, None, 12),
                                           (32, 40000, None, 12), (32, 96, 1.0, 12), (64, 96, None, 9), (64, 96, None, 30), (64, 16384, 600.0, 16),
                                           (32, 96, None, 14), (64, 96, 1.0, 21)])
def test_refusals(norm, bw, dim, gain, s):
    """Widths, scales and gains whose words do not fit the ring."""
    with pytest.raises(ValueError):
        norm(bw, dim, None if gain is None else np.full(max(dim, 1), int(gain * (1 << s)), np.int64), s)


def test_gates(norm):
    """A root's gates: ten of a word a token, or fewer in the 32-bit ring."""
    class Count(Ring):
        calls = 0

        def gate(self, kind, x):
            Count.calls += 1
            assert kind in (mpcx.TR, mpcx.TRRELU)
            return super().gate(kind, x)

    for bw, most in ((64, 6), (32, 4)):
        Count.calls = 0
        norm(bw, 4096).root(Count(bw, 12), np.array([1 << 24, 0]))
        assert Count.calls <= most


def test_widths_of_numpy(norm):
    """A width as an array's shape or a numpy number holds it."""
    assert np.array_equal(norm(64, np.int64(1000)).p.values, norm(64, 1000).p.values)
