"""What the serving operators do on the host: arguments at the ends of their ranges, refused before a device is
touched, and workspaces of devices that are made up."""
import ctypes as C

import pytest

from test_serving_refusals import attend, cache, prompt, refused


@pytest.mark.parametrize("scale", [3e38, 2.4e38])
def test_a_scale_whose_product_with_log2_e_overflows(scale):
    refused("scale", *attend(cache(), scale=scale))
    refused("scale", "bgtq_prompt_attend", C.byref(prompt(scale=scale)), None)


@pytest.mark.parametrize("what", ["prompt", "token"])
@pytest.mark.parametrize("recording", [True, False])
def test_a_recording_is_looked_for_on_the_tensors_device(monkeypatch, what, recording):
    """A workspace that is made within a recording on device 1 belongs to the graph and is not kept for the
    stream, while device 0 is the current one."""
    import torch
    from bgtq import _lib, serving
    current = [0]

    class device:
        def __init__(self, d):
            self.to, self.back = torch.device(d).index, current[0]

        def __enter__(self):
            current[0] = self.to

        def __exit__(self, *a):
            current[0] = self.back

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: recording and current[0] == 1)
    monkeypatch.setattr(_lib, "call", lambda *a: None)
    monkeypatch.setattr(serving, "_room", lambda size, on: (4096, size, None))
    kept = {}
    if what == "prompt":
        monkeypatch.setattr(serving, "_prompt_work", kept)
        assert serving._prompt_workspace(torch.device("cuda", 1), 64, 77)[0] == 4096
    else:
        c = serving.PagedCache.__new__(serving.PagedCache)
        c._ref, c._on, c._workspace = None, torch.device("cuda", 1), kept
        assert c._work(8, 77)[0] == 4096
    assert bool(kept) != recording and current[0] == 0
