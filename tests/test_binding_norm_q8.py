"""What the binding's 8-bit products and norm gates check before they enter the library,
and the example decoder's norm: on the CPU, with stand-ins for tensors and library."""
import types

import numpy as np
import pytest

import mpcx
from test_binding_transformer import BIG, BYTE, INT, LONG, Tensor, ctx  # noqa: F401 (ctx: the fixture)

INT8 = types.SimpleNamespace(name="int8", size=1)
KEY = Tensor((1000,), BYTE)


@pytest.fixture
def c(ctx, monkeypatch):  # noqa: F811
    mpcx._torch_module.int8 = INT8
    mpcx._torch_module.empty_like = lambda t: Tensor(t.shape, t.dtype, t.device_index)
    monkeypatch.setattr(Tensor, "new_empty", lambda t, n: Tensor(n if isinstance(n, tuple) else (n,), t.dtype, t.device_index),
                        raising=False)
    return ctx


def q8(c, a=None, q=None, scale=None, tokens=None, out=None):
    return c.ring_gemm_q8(a or Tensor((5, 40)), q or Tensor((7, 48), INT8), scale, tokens, out)


def test_q8_takes(c):
    q8(c)
    q8(c, a=Tensor((5, 40), stride=(90, 1)), scale=Tensor((7,)), tokens=Tensor((5,)), out=Tensor((5, 7), stride=(9, 1)))
    q8(c, q=Tensor((7, 40), INT8, stride=(64, 1)))  # rows without their padding
    q8(c, a=Tensor((5, 1)), q=Tensor((7, 1), INT8, stride=(16, 3)), out=Tensor((5, 7)))
    q8(c, q=Tensor((1, 40), INT8), out=Tensor((5, 1)))
    assert [x[0] for x in c.lib.calls] == ["mpcx_ring_gemm_q8"] * 5
    strides = [(x[1][5], x[1][7], x[1][11]) for x in c.lib.calls]
    assert strides == [(40, 48, 7), (90, 48, 9), (40, 64, 7), (1, 16, 7), (40, 48, 1)]
    assert q8(c, a=Tensor((0, 40))).shape == (0, 7) and len(c.lib.calls) == 5  # no token: no call


@pytest.mark.parametrize("bad", [
    dict(a=Tensor((5, 40), LONG)), dict(a=Tensor((5, 40), device=1)), dict(a=Tensor((5, 40), stride=(40, 2))),
    dict(a=Tensor((200,))), dict(a=Tensor((BIG, 40))), dict(a=Tensor((5, BIG)), q=Tensor((7, BIG), INT8)),
    dict(q=Tensor((BIG, 48), INT8)), dict(q=Tensor((7, 48), BYTE)), dict(q=Tensor((7, 48), INT8, device=-1)),
    dict(q=Tensor((7, 32), INT8)), dict(q=Tensor((7, 64), INT8)), dict(q=Tensor((7, 40), INT8)),
    dict(q=Tensor((7, 48), INT8, stride=(1, 7))), dict(q=Tensor((7, 48), INT8, stride=(0, 1))),
    dict(q=Tensor((7, 48), INT8, stride=(32, 1))), dict(scale=Tensor((8,))), dict(scale=Tensor((7,), LONG)),
    dict(scale=Tensor((7,), stride=(2,))), dict(scale=Tensor((7,), device=1)), dict(tokens=Tensor((7,))),
    dict(tokens=Tensor((5, 1))), dict(out=Tensor((7, 5))), dict(out=Tensor((5, 7), LONG)),
    dict(out=Tensor((5, 7), stride=(1, 5)))])
def test_q8_refuses(c, bad):
    with pytest.raises(mpcx.MpcxError):
        q8(c, **bad)
    assert not c.lib.calls


def sums(c, x=None, d=None, out=None, keys=(KEY, KEY)):
    return c.norm_sums_eval(*keys, x or Tensor((5, 40)), d, out)


def test_sums_takes(c):
    x, d, wide = Tensor((5, 40)), Tensor((5, 40)), Tensor((5, 40), stride=(90, 1))
    assert sums(c, x)[0] is x and sums(c, x)[1].shape == (5,)
    assert sums(c, x, d)[0].shape == (5, 40) and sums(c, x, wide, x)[0] is x
    assert sums(c, wide, d, wide)[0] is wide
    c.norm_sums_message(1, KEY, x, d)
    k0, k1, rh, rs = c.norm_sums_keygen(x, d)
    assert rh.shape == (5, 40) and rs.shape == (5,) and c.norm_sums_keygen(x)[2] is x
    assert sums(c, Tensor((0, 8), stride=(0, 0)), Tensor((0, 8)))[1].shape == (0,)
    calls = [n for n, _ in c.lib.calls]
    assert calls == ["mpcx_norm_sums_eval"] * 5 + ["mpcx_norm_sums_message"] + ["mpcx_norm_sums_keygen"] * 2 + \
        ["mpcx_norm_sums_eval"]
    assert c.lib.calls[0][1][7:11] == (None, 0, None, 0) and c.lib.calls[3][1][6:11:2] == (40, 90, 40)


@pytest.mark.parametrize("bad", [
    dict(x=Tensor((5, 40), LONG)), dict(x=Tensor((200,))), dict(x=Tensor((5, 8, 5))), dict(x=Tensor((5, 40), device=1)),
    dict(x=Tensor((5, 40), stride=(1, 5))), dict(x=Tensor((5, BIG))), dict(d=Tensor((5, 41))), dict(d=Tensor((6, 40))),
    dict(d=Tensor((5, 40), LONG)), dict(d=Tensor((5, 40), device=-1)), dict(out=Tensor((5, 40))),
    dict(d=Tensor((5, 40)), out=Tensor((5, 41))), dict(d=Tensor((5, 40)), out=Tensor((5, 40), LONG)),
    dict(keys=(Tensor((999,), BYTE), KEY)), dict(keys=(KEY, Tensor((1000,), BYTE, device=-1))),
    dict(keys=(KEY, Tensor((1000,), BYTE, stride=(2,))))])
def test_sums_refuses(c, bad):
    with pytest.raises(mpcx.MpcxError):
        sums(c, **bad)
    if "keys" not in bad and "out" not in bad:
        with pytest.raises(mpcx.MpcxError):
            c.norm_sums_keygen(bad.get("x") or Tensor((5, 40)), bad.get("d"))
    assert not c.lib.calls


def scale(c, keys=(KEY, KEY), shares=None, h=None, v=None, gain=None, out=None):
    return c.norm_scale_eval(*keys, *(shares or (Tensor((800,), BYTE), Tensor((800,), BYTE))), h or Tensor((5, 40)),
                             v or Tensor((5,)), gain, out)


def test_scale_takes(c):
    h = Tensor((5, 40), stride=(90, 1))
    assert scale(c).shape == (5, 40) and scale(c, h=h, gain=Tensor((40,)), out=h) is h
    c.norm_scale_message(0, KEY, Tensor((5, 40)), h, Tensor((5,)))
    assert c.norm_scale_keygen(KEY, KEY, Tensor((5,)), 40, Tensor((40,)))[2].shape == (5, 40)
    assert [n for n, _ in c.lib.calls] == ["mpcx_norm_scale_eval"] * 2 + ["mpcx_norm_scale_message", "mpcx_norm_scale_keygen"]
    assert c.lib.calls[1][1][8] == c.lib.calls[1][1][12] == 90


@pytest.mark.parametrize("bad", [
    dict(h=Tensor((5, 40), LONG)), dict(h=Tensor((200,))), dict(h=Tensor((5, 40), stride=(1, 5))), dict(h=Tensor((5, BIG))),
    dict(v=Tensor((4,))), dict(v=Tensor((5, 1))), dict(v=Tensor((5,), LONG)), dict(v=Tensor((5,), stride=(2,))),
    dict(gain=Tensor((41,))), dict(gain=Tensor((40,), LONG)), dict(gain=Tensor((40,), device=1)), dict(out=Tensor((40, 5))),
    dict(out=Tensor((5, 40), LONG)), dict(keys=(KEY, Tensor((999,), BYTE))),
    dict(shares=(Tensor((799,), BYTE), Tensor((800,), BYTE))), dict(shares=(Tensor((800,), BYTE), Tensor((800,), BYTE, 1)))])
def test_scale_refuses(c, bad):
    with pytest.raises(mpcx.MpcxError):
        scale(c, **bad)
    assert not c.lib.calls


@pytest.mark.parametrize("bad", [dict(dim=0), dict(dim=-1), dict(dim=BIG), dict(rv=Tensor((5, 1))), dict(rv=Tensor((5,), LONG)),
                                 dict(a0=Tensor((799,), BYTE)), dict(gain=Tensor((39,)))])
def test_scale_keygen_refuses(c, bad):
    args = dict(a0=KEY, a1=KEY, rv=Tensor((5,)), dim=40)
    with pytest.raises(mpcx.MpcxError):
        c.norm_scale_keygen(**{**args, **bad})
    assert not c.lib.calls


# ---------------- the example's norm ----------------
@pytest.mark.parametrize("bw,dim", [(32, 96), (64, 96), (64, 200)])
def test_norm_of_the_example(monkeypatch, bw, dim):
    """Rows of root mean square between 0.36 and 1.9 (the sum of squares of 96 then stays below
    2^31 at scale 24 only up to 1.1), against 64-bit floats.  What may be lost: the mean
    square's factor round(2^14 / dim), half a unit of 80 or more (2^-7.3), its index (a
    half step of 1/64 in 1/8: one Newton step leaves 1.5 (1/32)^2), five floors of a unit in
    500 or more, half of each in the root: 1% together; and the last floors of the row, one
    unit each, with a gain two."""
    import block
    monkeypatch.setattr(block, "_words", lambda ctx, v: None)
    rng = np.random.default_rng(dim)
    gain = np.round(rng.normal(1, 0.1, dim) * 4096).astype(np.int64) if bw == 64 else None
    norm = block.Norm(types.SimpleNamespace(s=12, bw=bw), dim, gain)
    rms = np.linspace(0.36, 1.9 if bw == 64 else 1.1, 40)[:, None]
    x = rng.normal(0, 1, (40, dim))
    x = np.round(x / np.sqrt((x * x).mean(1, keepdims=True)) * rms * 4096).astype(np.int64)
    d = np.round(rng.normal(0, 0.01, x.shape) * 4096).astype(np.int64)
    h, y = norm(block.Plain(12, None), x, d)
    want = h / np.sqrt((h.astype(np.float64) ** 2).mean(1, keepdims=True)) * (1 if gain is None else gain / 4096)
    assert np.array_equal(h, x + d)
    assert (np.abs(y / 4096 - want) <= 0.01 * np.abs(want) + 2 / 4096).all()
