"""The paged decoder's pages, without a device: which requests hold which, and which are free."""
import numpy as np
import pytest

from bgtq import _lib
from bgtq.paged_model import PagedDecoder


def books(pages, window=None, sinks=0, page_size=16):
    """A decoder that has its books alone."""
    dec = PagedDecoder.__new__(PagedDecoder)
    dec.window, dec.sinks, dec.page_size = window, sinks, page_size
    dec._free, dec._held, dec._next = list(range(pages))[::-1], {}, 0
    return dec


def grow(dec, request, tokens):
    with dec._grown([request], [tokens]) as (held, before):
        return dec._slots(held[0][0], before[0], held[0][1])


def every_page_once(dec, pages):
    held = [p for h in dec._held.values() for p in h[0] if p >= 0]
    assert sorted(dec._free + held) == list(range(pages))


@pytest.mark.parametrize("window,sinks,length", [(50, 4, 0), (50, 4, 3), (50, 4, 10), (50, 4, 16), (50, 40, 20), (50, 40, 48), (50, 0, 0),
                                                 (1, 0, 96), (1, 0, 112), (1, 20, 0), (1, 20, 32), (1, 20, 96)])
def test_a_rewind_past_pages_that_were_given_back(window, sinks, length):
    """To nothing, into the first tokens, and, with a window of one, to a page's end, however many pages behind have gone."""
    dec = books(14, window, sinks)
    a, b = dec.open(), dec.open()
    slots = grow(dec, b, 20)
    for _ in range(18):
        grow(dec, a, 20)
    assert -1 in dec._held[a][0] and dec.length(a) == 360
    dec.rewind(a, length)
    every_page_once(dec, 14)
    assert dec.length(a) == length and len(dec._held[a][0]) == -(-length // 16)
    mine = grow(dec, a, 60)
    every_page_once(dec, 14)
    assert mine.min() >= 0 and len(np.unique(mine // 16 * 16 + mine % 16)) == 60 and not set(mine // 16) & set(slots // 16)
    for r in (a, b):
        dec.close(r)
    assert sorted(dec._free) == list(range(14))


def test_a_rewind_to_tokens_that_have_gone_is_refused():
    dec = books(14, 50, 4)
    a = dec.open()
    for _ in range(18):
        grow(dec, a, 20)
    was = list(dec._held[a][0]), list(dec._free)
    for length in (17, 100, 330):
        with pytest.raises(_lib.RangeError, match="given back"):
            dec.rewind(a, length)
    assert (dec._held[a][0], dec._free) == was and dec.length(a) == 360
    dec.rewind(a, 355)
    every_page_once(dec, 14)


def state(dec):
    return {r: (list(h[0]), h[1]) for r, h in dec._held.items()}, list(dec._free)


def test_a_refused_call_changes_nothing():
    """A call of too many tokens, and what a rewind takes back after it."""
    dec = books(14, 50, 4)
    a, b = dec.open(), dec.open()
    grow(dec, a, 80)
    was = state(dec)
    for requests, counts in (([a], [400]), ([b, a], [1, 400])):
        with pytest.raises(_lib.RangeError, match="pages wanted, 9 free"):
            with dec._grown(requests, counts):
                pass
        assert state(dec) == was
    dec.rewind(a, 60)
    assert dec.length(a) == 60
    every_page_once(dec, 14)


@pytest.mark.parametrize("free", [0, 1, 2, 6])
@pytest.mark.parametrize("count,taken", [(1, 1), (16, 1), (17, 2), (32, 2)])
def test_a_call_that_fails_gives_back_what_it_took(free, count, taken):
    """Of 7 pages the second and the third are behind the window: the last that a call takes, and, where it did not,
    the request's again when it fails."""
    dec = books(7 + free, 50, 4)
    a = dec.open()
    grow(dec, a, 112)
    was, free_was = state(dec)
    with pytest.raises(MemoryError):
        with dec._grown([a], [count]) as (held, before):
            assert before == [112] and held[0][0][1:3] == [-1, -1] and len(held[0][0]) == 7 + taken
            raise MemoryError("made by the test")
    every_page_once(dec, 7 + free)
    lost = max(0, taken - free)
    pages = dec._held[a][0]
    assert dec.length(a) == 112 and len(dec._free) == free + lost and pages[1:3].count(-1) == lost
    assert pages[:1] + pages[3:] == was[a][0][:1] + was[a][0][3:]
    if not lost:
        assert state(dec) == (was, free_was)
    grow(dec, a, 10)
    every_page_once(dec, 7 + free)


def test_a_request_still_grows_past_the_pool():
    dec = books(6, 50, 4)
    a = dec.open()
    for _ in range(40):
        grow(dec, a, 16)
        every_page_once(dec, 6)
    assert dec.length(a) == 640
