"""Which steps the paged decoder records: batches that change size find theirs again."""
import numpy as np
import pytest

from test_gpu_paged_decoder_failures import decoder

pytestmark = pytest.mark.gpu


def recordings(dec, monkeypatch):
    made, was = [], dec._record

    def instead(*a):
        made.append(a)
        return was(*a)

    monkeypatch.setattr(dec, "_record", instead)
    return made


def test_places_hold_the_requests_and_are_few():
    from bgtq.paged_model import _RECORDED, _places
    assert all(n <= _places(n) < 2 * n + 1 for n in range(1, 400)) and _places(65535) == 65535
    assert len({_places(n) for n in range(1, 65)}) <= _RECORDED // 2


def test_a_batch_that_wanders_is_recorded_once_for_each_size(cuda, monkeypatch):
    dec = decoder(pages=80)
    held = [dec.open() for _ in range(20)]
    dec.prompt(held, [np.arange(2)] * 20)
    made = recordings(dec, monkeypatch)
    for lap in range(3):
        for n in range(1, 21):
            dec.step(held[:n], [lap] * n)
        assert len(made) <= 6, (lap, made)     # 1, 2, 4, 8, 16, 32 places


def test_the_step_unused_for_longest_goes_first(cuda, monkeypatch):
    from bgtq import paged_model
    monkeypatch.setattr(paged_model, "_RECORDED", 2)
    dec = decoder(pages=20)
    held = [dec.open() for _ in range(4)]
    dec.prompt(held, [np.arange(2)] * 4)
    made = recordings(dec, monkeypatch)
    for n in (1, 2, 1, 4, 1, 1):
        dec.step(held[:n], [5] * n)
    assert [m[0] for m in made] == [1, 2, 4] and len(dec._steps) == 2


def test_places_left_over_change_nothing(cuda):
    """Three requests in four places answer like themselves in a step of three and a stranger's."""
    import torch
    a, b = decoder(pages=20), decoder(pages=20)
    for d in (a, b):
        d.prompt([d.open() for _ in range(4)], [np.arange(3 + i) for i in range(4)])
    first = a.step([1, 2, 3], [7, 8, 9])
    assert [a.length(r) for r in (1, 2, 3, 4)] == [4, 5, 6, 6]
    assert torch.equal(first, b.step([1, 2, 3, 4], [7, 8, 9, 10])[:3])
    # the stranger's rows are as its prompt left them
    assert torch.equal(a.step([4], [10]), a_alone(4, [10]))


def a_alone(i, token):
    d = decoder(pages=20)
    d.prompt([d.open() for _ in range(4)], [np.arange(3 + j) for j in range(4)])
    return d.step([i], token)
