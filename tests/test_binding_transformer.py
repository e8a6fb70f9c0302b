"""What the binding's tensor calls check before they enter the library: on the CPU,
with stand-ins for the tensors and the library."""
import math
import types

import pytest

import mpcx

INT, LONG, BYTE = (types.SimpleNamespace(name=n, size=s) for n, s in (("int32", 4), ("int64", 8), ("uint8", 1)))


class Tensor:
    """Shape, strides and place of a GPU tensor."""

    def __init__(self, shape, dtype=None, device=0, stride=None):
        self.shape, self.dtype, self.device_index = tuple(shape), dtype or INT, device
        self.strides = stride or tuple(math.prod(self.shape[i + 1:]) for i in range(len(self.shape)))

    is_cuda = property(lambda self: self.device_index >= 0)

    def get_device(self):
        return self.device_index

    def is_contiguous(self):
        want = 1
        for n, s in zip(reversed(self.shape), reversed(self.strides)):
            if n != 1 and s != want:
                return False
            want *= n
        return True

    def stride(self, d=None):
        return self.strides if d is None else self.strides[d]

    def dim(self):
        return len(self.shape)

    def numel(self):
        return math.prod(self.shape)

    def element_size(self):
        return self.dtype.size

    def data_ptr(self):
        return 4096

    def zero_(self):
        return self


class Lib:
    """Says that a key or workspace has 1000 bytes; records the other calls."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*a):
            if name.endswith("_bytes"):
                return 1000
            if name != "mpcx_synchronize":
                self.calls.append((name, a))
            return 0
        return call


@pytest.fixture
def ctx(monkeypatch):
    stream = types.SimpleNamespace(cuda_stream=7, synchronize=lambda: None)
    torch = types.SimpleNamespace(int32=INT, int64=LONG, uint8=BYTE, empty=lambda shape, dtype=None, device=None: Tensor(
        shape if isinstance(shape, tuple) else (shape,), dtype, device),
        zeros=lambda n, dtype=None, device=None: Tensor((n,), dtype, 0 if device == "cuda" else device),
        cuda=types.SimpleNamespace(current_stream=lambda device=None: stream))
    monkeypatch.setattr(mpcx, "_torch_module", torch)
    monkeypatch.setattr(mpcx, "_torch", lambda: torch)
    c = mpcx.Ctx.__new__(mpcx.Ctx)
    c.lib, c.h, c.bw, c._word, c._device, c._stream_id = Lib(), None, 32, INT, 0, 7
    return c


@pytest.mark.parametrize("bad", [dict(shape=(999,)), dict(shape=(1000,), device=-1), dict(shape=(1000,), stride=(2,)),
                                 dict(shape=(0,))])
def test_gate_eval_checks_its_keys(ctx, bad):
    key, x = Tensor((1000,), BYTE), Tensor((5,))
    ctx.gate_eval(mpcx.TR, key, key, x)
    assert [c[0] for c in ctx.lib.calls] == ["mpcx_tr_eval"]
    for keys in ((Tensor(dtype=BYTE, **bad), key), (key, Tensor(dtype=BYTE, **bad))):
        with pytest.raises(mpcx.MpcxError):
            ctx.gate_eval(mpcx.TR, *keys, x)
    assert len(ctx.lib.calls) == 1


@pytest.mark.parametrize("group", [0, -32])
def test_q4_groups_of_nothing(ctx, group):
    with pytest.raises(mpcx.MpcxError):
        ctx.ring_gemm_q4(Tensor((2, 64)), Tensor((4, 32), BYTE), Tensor((2, 4)), group)
    assert not ctx.lib.calls


BIG = (1 << 32) + 2  # 2 where a C int is taken


@pytest.mark.parametrize("M,K,N", [(BIG, 64, 4), (2, BIG, 4), (2, 64, BIG)])
def test_q4_sizes_past_a_c_int(ctx, M, K, N):
    args = Tensor((M, K)), Tensor((N, (K + 31) // 32 * 16), BYTE), Tensor((-(-K // 32), N))
    with pytest.raises(mpcx.MpcxError):
        ctx.ring_gemm_q4(*args, 32)
    assert not ctx.lib.calls
    ctx.ring_gemm_q4(Tensor((2, 64)), Tensor((4, 32), BYTE), Tensor((2, 4)), 32)
    assert len(ctx.lib.calls) == 1


def batch(seqs=1, tokens=2, pages=3, **kw):
    v = dict(n_scores=8, heads=2, max_q=2, max_keys=4)
    v.update(kw)
    return mpcx.AttnBatch(Tensor((seqs, pages)), Tensor((seqs + 1,)), Tensor((tokens,)), Tensor((tokens,)),
                          Tensor((tokens,), LONG), **v)


def mix(ctx, b, pool=(5, 2, 4, 8)):
    key = Tensor((1000,), BYTE)
    return ctx.attn_mix_eval(b, key, key, Tensor((b.n_scores,)), *[Tensor(pool) for _ in range(3)])


@pytest.mark.parametrize("over", [dict(tokens=BIG), dict(seqs=BIG), dict(pages=BIG), dict(heads=BIG), dict(max_q=BIG),
                                  dict(max_keys=BIG)])
def test_attn_sizes_past_a_c_int(ctx, over):
    with pytest.raises(mpcx.MpcxError):
        mix(ctx, batch(**over))
    assert not ctx.lib.calls
    assert mix(ctx, batch()).shape == (2, 2, 8)


@pytest.mark.parametrize("at", [1, 2, 3])
def test_cache_sizes_past_a_c_int(ctx, at):
    pool = [5, 2, 4, 8]
    pool[at] = BIG
    with pytest.raises(mpcx.MpcxError):
        mix(ctx, batch(), tuple(pool))
    with pytest.raises(mpcx.MpcxError):
        ctx.cache_append([(Tensor((2, pool[1], pool[3])), Tensor(pool), False)], Tensor((2,), LONG))
    with pytest.raises(mpcx.MpcxError):  # the table's sizes
        ctx.cache_append([(Tensor((2, 2, 8)), Tensor((5, 2, 4, 8)), True)], Tensor((2,), LONG), Tensor((2,)),
                         mpcx.Rotation(Tensor((BIG, 4)), Tensor((BIG, 4)), 12))
    assert not ctx.lib.calls
    ctx.cache_append([(Tensor((2, 2, 8)), Tensor((5, 2, 4, 8)), True)], Tensor((2,), LONG), Tensor((2,)),
                     mpcx.Rotation(Tensor((9, 4)), Tensor((9, 4)), 12))
    assert len(ctx.lib.calls) == 1


def test_keys_are_made_on_the_contexts_gpu(ctx):
    ctx._device = 1
    keys = ctx.gate_keygen(mpcx.TR, Tensor((5,), device=1))
    b = batch()._replace(**{n: Tensor(getattr(batch(), n).shape, getattr(batch(), n).dtype, 1)
                            for n in ("pages", "qstart", "lo", "hi", "off")})
    keys += ctx.attn_mix_keygen(b, Tensor((8,), device=1), Tensor((5, 2, 4, 8), device=1), Tensor((5, 2, 4, 8), device=1))
    assert [k.get_device() for k in keys] == [1] * 6


CALLS = {
    "ring_gemm_q4": (lambda c, *t: c.ring_gemm_q4(*t, 32), [(2, 64), ((4, 32), BYTE), (2, 4)]),
    "cache_append": (lambda c, r, p, s, pos, co, si: c.cache_append([(r, p, True)], s, pos, mpcx.Rotation(co, si, 12)),
                     [(2, 2, 8), (5, 2, 4, 8), ((2,), LONG), (2,), (9, 4), (9, 4)]),
    "gate_keygen": (lambda c, m: c.gate_keygen(mpcx.TR, m), [(5,)]),
    "gate_eval": (lambda c, a, b, x: c.gate_eval(mpcx.TR, a, b, x), [((1000,), BYTE), ((1000,), BYTE), (5,)]),
    "split_mask": (lambda c, m: c.split_mask(m), [(5,)]),
    "attn_scores_eval": (
        lambda c, pages, q, lo, hi, off, slope, pos, *t: c.attn_scores_eval(
            mpcx.AttnBatch(pages, q, lo, hi, off, 8, 2, 2, 4), *t, slope=slope, pos=pos),
        [(1, 3), (2,), (2,), (2,), ((2,), LONG), (2,), (2,), ((1000,), BYTE), ((1000,), BYTE), (2, 2, 8), (5, 2, 4, 8),
         (5, 2, 4, 8), (5, 2, 4, 8)]),
    "attn_mix_message": (
        lambda c, pages, q, lo, hi, off, *t: c.attn_mix_message(1, mpcx.AttnBatch(pages, q, lo, hi, off, 8, 2, 2, 4), *t),
        [(1, 3), (2,), (2,), (2,), ((2,), LONG), ((1000,), BYTE), (8,), (5, 2, 4, 8), (5, 2, 4, 8)]),
}


@pytest.mark.parametrize("name", sorted(CALLS))
def test_tensors_of_another_gpu(ctx, name):
    call, shapes = CALLS[name]
    made = [(s if isinstance(s[0], tuple) else (s, INT)) for s in shapes]
    call(ctx, *[Tensor(*m) for m in made])
    assert len(ctx.lib.calls) == 1
    for i in range(len(made)):
        for device in (1, -1):
            with pytest.raises(mpcx.MpcxError):
                call(ctx, *[Tensor(*m, device=device if i == j else 0) for j, m in enumerate(made)])
    assert len(ctx.lib.calls) == 1


@pytest.mark.parametrize("heads,dim,stride,ok", [
    (1, 8, (24, 24, 1), True), (1, 8, (8, 1, 1), True), (1, 1, (5, 7, 3), True), (3, 1, (9, 1, 4), True),
    (2, 8, (16, 8, 1), True), (2, 8, (40, 8, 1), True), (2, 8, (40, 9, 1), False), (1, 8, (8, 8, 2), False),
    (2, 1, (9, 4, 1), False), (2, 8, (8, 16, 1), False)])
def test_cache_append_strides_of_single_heads_and_dims(ctx, heads, dim, stride, ok):
    """A stride counts where there is more than one of its dimension."""
    rows, pool = Tensor((4, heads, dim), stride=stride), Tensor((5, heads, 4, dim))
    if not ok:
        with pytest.raises(mpcx.MpcxError):
            ctx.cache_append([(rows, pool, False)], Tensor((4,), LONG))
        return
    ctx.cache_append([(rows, pool, False)], Tensor((4,), LONG))
    (_, args), = ctx.lib.calls
    assert args[-1][0].ld == stride[0]
