"""A paged decoder over a window that takes back tokens behind which pages have gone: what two requests answer from then on,
against the model's formulas in 64 bits."""
import numpy as np
import pytest

from test_gpu_paged_decoder_windows import Windowed
from test_gpu_paged_model import BOUND, SMALL, off, weights_of
from test_gpu_serving import types

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,dtype", [("f16", "f16"), ("int8", "bf16"), ("int4", "f16")])
@pytest.mark.parametrize("window,sinks,back_to", [(50, 4, 0), (50, 4, 10), (50, 40, 20), (1, 0, 96)])
def test_two_requests_after_a_rewind(cuda, fmt, dtype, window, sinks, back_to):
    from bgtq import PagedDecoder, device_status
    g, bound = SMALL["llama"], BOUND[dtype]
    w = weights_of(g, dtype)
    dec = PagedDecoder(w, g, pages=14, page_size=16, format=fmt, dtype=types()[dtype], window=window, sinks=sinks)
    rng = np.random.default_rng(7)
    a, b = dec.open(), dec.open()
    plain = {r: Windowed(w, dec, r, bound) for r in (a, b)}

    def prompt(counts):
        tokens = [rng.integers(0, g.vocab, n) for n in counts.values()]
        for r, t, got in zip(counts, tokens, dec.prompt(list(counts), tokens)):
            assert off(got[None], plain[r].forward(t)[-1:]) < bound, (r, dec.length(r))

    def step():
        tokens = rng.integers(0, g.vocab, 2)
        for r, t, got in zip((a, b), tokens, dec.step([a, b], tokens)):
            assert off(got[None], plain[r].forward([t])) < bound, (r, dec.length(r))

    prompt({b: 20})
    for _ in range(12):
        prompt({a: 30})
    dec.rewind(a, back_to)
    plain[a].length = back_to
    prompt({a: 40, b: 30})
    for _ in range(20):
        step()
    prompt({b: 40, a: 25})
    step()
    held = [p for h in dec._held.values() for p in h[0] if p >= 0]
    assert sorted(dec._free + held) == list(range(14)) and device_status(0) == 0
