"""A call of the paged decoder that fails on the way leaves its requests as they were: lengths, pages,
and what the next calls answer.  The failures are made on the host."""
import numpy as np
import pytest

from test_gpu_paged_model import SMALL, weights_of
from test_gpu_serving import types

pytestmark = pytest.mark.gpu


def decoder(pages=12):
    from bgtq import PagedDecoder
    g = SMALL["llama"]
    return PagedDecoder(weights_of(g, "f16"), g, pages=pages, page_size=16, format="int8", dtype=types()["f16"])


def failing(dec, monkeypatch, layer, method, calls):
    """The layer's cache raises in the given method from its call number `calls` on, counted from 1."""
    cache, seen = dec.caches[layer], [0]
    was = getattr(cache, method)

    def instead(*a, **k):
        seen[0] += 1
        if seen[0] >= calls:
            raise MemoryError("made by the test")
        return was(*a, **k)

    monkeypatch.setattr(cache, method, instead)


def state(dec, requests):
    return [dec.length(r) for r in requests], [list(dec._held[r][0]) for r in requests], list(dec._free)


@pytest.mark.parametrize("layer,method", [(0, "write"), (2, "write"), (1, "read")])
def test_a_prompt_that_fails_changes_nothing(cuda, monkeypatch, layer, method):
    import torch
    dec, same = decoder(), decoder()
    rng = np.random.default_rng(4)
    first, second = [rng.integers(0, 331, n) for n in (17, 30)], [rng.integers(0, 331, n) for n in (40, 3)]
    answers = []
    for d in (same, dec):
        held = [d.open(), d.open()]
        d.prompt(held, first)
        if d is dec:
            was = state(d, held)
            with monkeypatch.context() as m:
                failing(d, m, layer, method, 1)
                with pytest.raises(MemoryError):
                    d.prompt(held, second)
            assert state(d, held) == was
        answers.append((d.prompt(held, second), d.step(held, [5, 6])))
    for a, b in zip(*answers):
        assert torch.equal(a, b)


@pytest.mark.parametrize("calls", [1, 2])      # before the recording of the step, and while it is recorded
def test_a_step_that_fails_changes_nothing(cuda, monkeypatch, calls):
    import torch
    dec, same = decoder(), decoder()
    tokens = [np.arange(16), np.arange(5)]     # the first needs a page for its next token
    answers = []
    for d in (same, dec):
        held = [d.open(), d.open()]
        d.prompt(held, tokens)
        if d is dec:
            was = state(d, held)
            with monkeypatch.context() as m:
                failing(d, m, 1, "attend", calls)
                with pytest.raises(MemoryError):
                    d.step(held, [5, 6])
            assert state(d, held) == was
        answers.append((d.step(held, [5, 6]), d.step(held, [7, 8])))
    for a, b in zip(*answers):
        assert torch.equal(a, b)


def test_failures_do_not_eat_pages(cuda, monkeypatch):
    dec = decoder(pages=3)
    r = dec.open()
    for _ in range(3):
        with monkeypatch.context() as m:
            failing(dec, m, 0, "write", 1)
            with pytest.raises(MemoryError):
                dec.prompt([r], [np.arange(40)])
    assert dec.length(r) == 0 and dec.free_pages == 3
    dec.prompt([r], [np.arange(40)])
    assert dec.length(r) == 40 and dec.free_pages == 0
