"""Workspaces of a windowed decoder's recorded steps: nobody else's calls may use them while a step is replayed."""
import numpy as np
import pytest

from test_gpu_paged_model import SMALL, weights_of
from test_gpu_serving import randn, types

pytestmark = pytest.mark.gpu


def recorded(streams, fmt="int8"):
    """Decoders whose recording streams are the given ones, each with a request of 4000 tokens, of which a step reads
    3000 in parts; and the graphs and logits of their steps."""
    from bgtq import PagedDecoder
    g = SMALL["llama"]
    w = weights_of(g, "f16")
    decs = []
    for i, side in enumerate(streams):
        dec = PagedDecoder(w, g, pages=260, page_size=16, format=fmt, dtype=types()["f16"], window=3000, sinks=4)
        dec._side = side
        r = dec.open()
        dec.prompt([r], [np.random.default_rng(i).integers(0, g.vocab, 4000)])
        dec.step([r], [3 + i])
        decs.append(dec)
    return decs, [next(iter(d._steps.values())) for d in decs]


def test_a_recording_has_the_decoders_own_workspace(cuda):
    import torch
    from bgtq import serving
    side = torch.cuda.Stream()
    decs, _ = recorded([side, side])
    mine = [{work[0] for work in d.caches[0]._chunk_work.values()} for d in decs]
    assert all(mine) and not mine[0] & mine[1]
    assert not (mine[0] | mine[1]) & {work[0] for work in serving._chunk_work.values()}
    assert all(c._chunk_work is d.caches[0]._chunk_work for d in decs for c in d.caches)


def test_steps_replayed_beside_each_other_and_beside_calls_on_their_recording_stream(cuda):
    import torch
    from bgtq import PagedCache
    side = torch.cuda.Stream()
    decs, steps = recorded([side, side])  # (a decoder owns what its graphs use)
    cache = PagedCache(1, 64, 250, 16, "int8")
    cache.write(randn(1, 4000, 1, 64, dtype="f16"), randn(2, 4000, 1, 64, dtype="f16"), torch.arange(4000, device="cuda"))
    q = randn(3, 1, 3, 64, dtype="f16")
    table, lengths = torch.arange(250, dtype=torch.int32, device="cuda")[None], torch.tensor([4000], dtype=torch.int32, device="cuda")
    call = lambda: cache.attend(q, table, lengths, window=3000, sinks=4)
    want, wants = call(), []
    for graph, _, logits in steps:
        graph.replay()
        torch.cuda.synchronize()
        wants.append(logits.clone())
    on, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    torch.cuda.synchronize()
    for _ in range(100):
        for s, (graph, _, _) in zip(on, steps):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(side):
            got.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    assert all(torch.equal(logits, w) for (_, _, logits), w in zip(steps, wants)) and len(decs) == 2


def test_all_chunk_workspaces_are_ready_again_after_a_wait_that_ran_out(cuda):
    """The counters that such a call leaves are made up; they stay within the launch's parts."""
    import torch
    from bgtq import _lib, serving
    decs, steps = recorded([torch.cuda.Stream()])
    graph, _, logits = steps[0]
    want = logits.clone()
    torch.cuda.synchronize()
    rooms = [work[2] for work in decs[0].caches[0]._chunk_work.values()]
    assert rooms and not any(room[:_lib.WORKSPACE_ZEROED].any() for room in rooms)
    for room in rooms:
        room.view(torch.int32)[:64] = 1
    serving._ready_again(0)
    assert not any(room[:_lib.WORKSPACE_ZEROED].any() for room in rooms)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(logits, want)
    del decs, steps, graph
