"""Workspaces of the serving operators: what has to be zero in them, and what it costs to make one."""
import ctypes as C

import pytest

from bgtq import _lib
from test_gpu_serving import randn, starts_of

pytestmark = pytest.mark.gpu


def case():
    """A prompt and a token over long keys, each done in several parts."""
    import torch
    from bgtq import PagedCache
    n = 4000
    k, v = randn(1, n, 2, 64, dtype="f16"), randn(2, n, 2, 64, dtype="f16")
    cache = PagedCache(2, 64, 250, 16, "int8")
    cache.write(k, v, torch.arange(n, device="cuda"))
    return dict(k=k, v=v, cache=cache, q1=randn(3, 1, 14, 64, dtype="f16"), q2=randn(4, 16, 14, 64, dtype="f16"),
                table=torch.arange(250, dtype=torch.int32, device="cuda")[None],
                lengths=torch.tensor([n], dtype=torch.int32, device="cuda"), starts=starts_of([16]), keys=starts_of([n]))


def test_only_the_front_of_a_workspace_has_to_be_zero(cuda):
    import torch
    from bgtq import prompt_attention
    c = case()
    want = c["cache"].attend(c["q1"], c["table"], c["lengths"]), prompt_attention(c["q2"], c["k"], c["v"], c["starts"], c["keys"])
    need = [C.c_size_t(), C.c_size_t()]
    _lib.call("bgtq_paged_attend_workspace", c["cache"]._ref, 14, C.byref(need[0]))
    _lib.call("bgtq_prompt_workspace", 0, 64, C.byref(need[1]))
    rooms = [torch.full((n.value,), 255, dtype=torch.uint8, device="cuda") for n in need]     # NaN behind the front
    out = torch.empty_like(want[0]), torch.empty_like(want[1])
    for room in rooms:
        room[:_lib.WORKSPACE_ZEROED] = 0
    p = _lib.PromptDesc(0, _lib.F16, 1, 14, 2, 64, 16, 4000, c["q2"].data_ptr(), c["k"].data_ptr(), c["v"].data_ptr(), 14 * 64, 64,
                        128, 64, 128, 64, c["starts"].data_ptr(), c["keys"].data_ptr(), 1, 0.0, out[1].data_ptr(), None,
                        rooms[1].data_ptr(), need[1].value)
    for _ in range(3):
        for o in out:
            o.zero_()
        _lib.call("bgtq_paged_attend", c["cache"]._ref, c["q1"].data_ptr(), _lib.F16, 1, 14, 14 * 64, 64, c["table"].data_ptr(), 250,
                  250, c["lengths"].data_ptr(), 0.0, out[0].data_ptr(), None, rooms[0].data_ptr(), need[0].value,
                  torch.cuda.current_stream().cuda_stream)
        _lib.call("bgtq_prompt_attend", C.byref(p), torch.cuda.current_stream().cuda_stream)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_a_recording_on_a_new_stream_zeroes_the_front_alone(cuda):
    """What a recorded call fills is repeated by every replay."""
    import torch
    from torch.utils._python_dispatch import TorchDispatchMode
    from bgtq import prompt_attention

    class Filled(TorchDispatchMode):
        most = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            if func.overloadpacket in (torch.ops.aten.zeros, torch.ops.aten.zero_, torch.ops.aten.fill_, torch.ops.aten.full):
                self.most = max(self.most, out.numel() * out.element_size())
            return out

    c = case()
    want = c["cache"].attend(c["q1"], c["table"], c["lengths"]), prompt_attention(c["q2"], c["k"], c["v"], c["starts"], c["keys"])
    torch.cuda.synchronize()
    g, filled = torch.cuda.CUDAGraph(), Filled()
    with torch.cuda.graph(g), filled:
        got = c["cache"].attend(c["q1"], c["table"], c["lengths"]), prompt_attention(c["q2"], c["k"], c["v"], c["starts"], c["keys"])
    assert 0 < filled.most <= _lib.WORKSPACE_ZEROED
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_workspace_is_ready_again_after_a_wait_that_ran_out(cuda, monkeypatch):
    """The status is made up, and so are the counters that such a call leaves; they stay within the launch's parts."""
    import torch
    import bgtq
    from bgtq import prompt_attention, serving
    c = case()
    run = lambda: prompt_attention(c["q2"], c["k"], c["v"], c["starts"], c["keys"])
    want = run()
    torch.cuda.synchronize()
    work = serving._prompt_work[0, 64, torch.cuda.current_stream().cuda_stream][2]
    assert not work[:_lib.WORKSPACE_ZEROED // 8].any()
    work.view(torch.int32)[:64] = 1
    real = _lib.call

    def call(name, *args):
        real(name, *args)
        if name == "bgtq_device_status":
            args[1]._obj.value |= 1

    monkeypatch.setattr(_lib, "call", call)
    assert bgtq.device_status() & 1
    assert torch.equal(run(), want)
    assert not work[:_lib.WORKSPACE_ZEROED // 8].any()


def test_the_layers_of_a_decoder_share_a_workspace(cuda):
    import numpy as np
    from test_gpu_paged_decoder_failures import decoder
    dec = decoder()
    r = dec.open()
    dec.prompt([r], [np.arange(20)])
    dec.step([r], [3])
    assert len({work[0] for cache in dec.caches for work in cache._workspace.values()}) == 1
