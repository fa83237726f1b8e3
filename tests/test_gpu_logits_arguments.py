"""The serving operators at the C ABI: arguments that stand beside a null array, and a call after one that failed."""
import ctypes as C

import pytest

from bgtq import _lib
from test_gpu_serving import randn

pytestmark = pytest.mark.gpu


def put(x, out, **kw):
    import torch
    d = dict(device=0, dtype=_lib.F32, batch=x.shape[0], vocab=x.shape[1], logits=x.data_ptr(), logits_stride=x.stride(0), out=out.data_ptr(),
             out_stride=out.stride(0), id_bytes=4)
    d.update(kw)
    _lib.call("bgtq_adjust_logits", C.byref(_lib.LogitsDesc(**d)), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("entries", [1, 256, 257, 100000, 2**31 - 1])
def test_a_number_of_biases_without_biases_says_nothing(cuda, entries):
    import torch
    x = randn(1, 3, 5000)
    assert torch.equal(put(x, torch.empty_like(x), entries=entries, bias_stride=entries), x)
    ids = torch.zeros((3, 4), dtype=torch.int32, device="cuda")
    one = torch.ones(3, device="cuda")
    got = put(x, torch.empty_like(x), entries=entries, tokens=ids.data_ptr(), tokens_stride=4, width=4, presence=one.data_ptr())
    want = x.clone()
    want[:, 0] -= 1
    assert torch.equal(got, want)


def test_a_call_after_one_on_a_device_that_is_not_there(cuda):
    """The error is the call's own."""
    import torch
    from bgtq import PagedCache
    assert torch.cuda.device_count() < 60
    x, cache = randn(1, 3, 500), PagedCache(1, 64, 4, 16, "f16")
    rows, at = randn(2, 20, 1, 64), torch.arange(20, device="cuda")
    want = cache.append(rows, rows, rows, at, randn(3, 20, 64))
    q, table, lengths = randn(4, 1, 1, 64, dtype="f16"), torch.arange(2, dtype=torch.int32, device="cuda")[None], torch.tensor([20], dtype=torch.int32, device="cuda")
    for call in (lambda: put(x, torch.empty_like(x)), lambda: cache.append(rows, rows, rows, at, randn(3, 20, 64)),
                 lambda: cache.attend_chunk(q, None, table, lengths), lambda: cache.attend(q, table, lengths), lambda: cache.read(at)):
        with pytest.raises(_lib.DeviceError):
            put(x, torch.empty_like(x), device=61)
        call()
    assert torch.equal(cache.append(rows, rows, rows, at, randn(3, 20, 64)), want)
