"""The example decoder on the GPU: norm, attention and 8-bit layers together, a prompt of two
sequences and single tokens, against plain integers bit for bit."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bw,kw", [(32, {}), (64, {}), (64, dict(blocks=3, model=80, heads=5, kv=1, dim=16, hidden=77, words=33,
                                                                 prompts=(1, 9, 4), page=3)),
                                   (32, dict(blocks=1, model=64, hidden=300, words=1000, prompts=(70,), page=16))])
def test_decoder(bw, kw):
    import block
    lines = []
    assert block.run(bw, say=lines.append, **kw), lines
    assert len(lines) == 4


@pytest.mark.parametrize("bw,kw", [(64, dict(blocks=1, model=2560, hidden=96, words=40, prompts=(5,), singles=2)),
                                   (64, dict(blocks=1, model=6144, hidden=48, words=24, prompts=(3,), singles=2))])
def test_decoder_of_ordinary_width(bw, kw):
    """Norms of rows whose width is no power of two, one of them past 4096 (a truncation more)."""
    import block
    lines = []
    assert block.run(bw, say=lines.append, **kw), lines
