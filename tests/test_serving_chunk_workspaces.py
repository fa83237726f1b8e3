"""Which workspace a chunk's call takes, and which are made ready again, for devices that are made up."""
import pytest


@pytest.fixture
def serving(monkeypatch):
    import torch
    from bgtq import _lib, serving

    class device:
        def __init__(self, d):
            pass

        def __enter__(self):
            pass

        def __exit__(self, *a):
            pass

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device: None)
    monkeypatch.setattr(_lib, "call", lambda *a: None)
    monkeypatch.setattr(serving, "_room", lambda size, on: (4096, size, torch.ones(2 * _lib.WORKSPACE_ZEROED, dtype=torch.uint8)))
    return serving


def made_up(serving, device=1, works=None):
    import torch
    c = serving.PagedCache.__new__(serving.PagedCache)
    c._ref, c._on, c.device, c.dim = None, torch.device("cuda", device), device, 64
    c._chunk_work = serving._Workspaces() if works is None else works
    return c


def test_a_cache_keeps_its_workspaces_where_it_was_told_to(serving):
    mine, other = made_up(serving), made_up(serving)
    work = serving._chunk_workspace(mine, 8, 77)
    assert dict(mine._chunk_work) == {(1, 64, 77): work}
    assert not other._chunk_work and (1, 64, 77) not in serving._chunk_work


def test_all_of_a_devices_workspaces_are_made_ready_again(serving):
    from bgtq import _lib
    caches = [made_up(serving, 1), made_up(serving, 1), made_up(serving, 2)]
    rooms = [serving._chunk_workspace(c, 8, 77)[2] for c in caches]
    serving._ready_again(1)
    for room, zeroed in zip(rooms, (True, True, False)):
        assert bool(room[:_lib.WORKSPACE_ZEROED].any()) != zeroed and bool(room[_lib.WORKSPACE_ZEROED:].all())
