"""What the serving operators refuse, at the C ABI: every check comes before a device is touched,
so these run without one."""
import ctypes as C

import pytest

from bgtq import _lib

GOOD = 1 << 20  # an aligned address that is never followed


def cache(**kw):
    d = dict(device=0, format=_lib.PAGES_INT8, kv_heads=2, dim=64, page_size=16, pages=4, k=GOOD, v=GOOD, k_scales=GOOD,
             v_scales=GOOD)
    d.update(kw)
    return _lib.PagedCacheDesc(**d)


def refused(message, name, *args):
    with pytest.raises(_lib.RangeError, match=message) as e:
        _lib.call(name, *args)
    assert e.value.status == _lib.EINVAL


def write(c, k=GOOD, v=GOOD, dtype=_lib.F16, tokens=3, slots=GOOD):
    return "bgtq_paged_write", C.byref(c), k, v, dtype, tokens, 128, 64, 128, 64, slots, None


def read(c, slots=GOOD, tokens=3, k=GOOD, v=GOOD, dtype=_lib.F16):
    return "bgtq_paged_read", C.byref(c), slots, tokens, k, v, dtype, None


def attend(c, q=GOOD, dtype=_lib.F16, batch=2, heads=4, table=GOOD, width=4, lengths=GOOD, scale=0.0, out=GOOD, lse=None):
    return ("bgtq_paged_attend", C.byref(c), q, dtype, batch, heads, 256, 64, table, 4, width, lengths, scale, out, lse,
            GOOD, 1 << 30, None)


@pytest.mark.parametrize("change,message", [
    (dict(dim=96), "head dim"), (dict(dim=0), "head dim"), (dict(format=0), "format"), (dict(format=5), "format"),
    (dict(page_size=24), "page size"), (dict(page_size=8), "page size"), (dict(page_size=512), "page size"),
    (dict(kv_heads=0), "head or page count"), (dict(kv_heads=1025), "head or page count"),
    (dict(pages=0), "head or page count"), (dict(pages=1 << 31), "head or page count"), (dict(k=None), "16-byte"),
    (dict(v=GOOD + 8), "16-byte"), (dict(k_scales=None), "scales"), (dict(v_scales=GOOD + 8), "scales")])
def test_every_call_refuses_a_wrong_cache(change, message):
    c = cache(**change)
    for call in (write(c), read(c), attend(c)):
        refused(message, *call)
    refused(message, "bgtq_paged_attend_workspace", C.byref(c), 2, C.byref(C.c_size_t()))


def test_null_cache():
    refused("null", "bgtq_paged_write", None, GOOD, GOOD, _lib.F16, 1, 128, 64, 128, 64, GOOD, None)
    refused("null", "bgtq_prompt_attend", None, None)


def test_write_and_read_refusals():
    c = cache()
    refused("FP16, BF16 or FP32", *write(c, dtype=7))
    refused("FP16, BF16 or FP32", *read(c, dtype=0))
    refused("null", *write(c, k=None))
    refused("null", *write(c, slots=None))
    refused("null", *read(c, v=None))
    refused("misaligned", *write(c, k=GOOD + 1))
    refused("misaligned", *write(c, v=GOOD + 2, dtype=_lib.F32))
    refused("misaligned", *write(c, slots=GOOD + 4))
    refused("misaligned", *read(c, k=GOOD + 8))
    refused("too many", *write(c, tokens=1 << 31))
    refused("too many", *read(c, tokens=1 << 40))
    _lib.call(*write(c, tokens=0))
    _lib.call(*read(c, tokens=0))


def test_attend_refusals():
    c = cache()
    refused("queries must be", *attend(c, dtype=_lib.F32))
    for fmt, dt in ((_lib.PAGES_F16, _lib.BF16), (_lib.PAGES_BF16, _lib.F16)):
        refused("type of 16-bit pages", *attend(cache(format=fmt), dtype=dt))
    refused("head count", *attend(c, heads=3))
    refused("head count", *attend(c, heads=0))
    for scale in (-1.0, float("inf"), float("nan")):
        refused("scale", *attend(c, scale=scale))
    for null in ("q", "table", "lengths", "out"):
        refused("null", *attend(c, **{null: None}))
    refused("too many requests", *attend(c, batch=65536))
    refused("2\\^31", *attend(c, width=1 << 27))
    refused("misaligned", *attend(c, q=GOOD + 1))
    refused("misaligned", *attend(c, out=GOOD + 8))
    refused("misaligned", *attend(c, lengths=GOOD + 2))
    _lib.call(*attend(c, batch=0))


def prompt(**kw):
    d = dict(device=0, dtype=_lib.F16, sequences=1, q_heads=4, kv_heads=2, dim=64, q_tokens=8, k_tokens=8, q=GOOD, k=GOOD,
             v=GOOD, q_token_stride=256, q_head_stride=64, k_token_stride=128, k_head_stride=64, v_token_stride=128,
             v_head_stride=64, starts=GOOD, key_starts=None, causal=1, scale=0.0, out=GOOD, lse=None)
    d.update(kw)
    return _lib.PromptDesc(**d)


@pytest.mark.parametrize("change,message", [
    (dict(dim=80), "head dim"), (dict(dtype=_lib.F32), "FP16 or BF16"), (dict(q_heads=3), "head count"),
    (dict(kv_heads=0), "head count"), (dict(q_heads=258, kv_heads=2), "head count"), (dict(scale=-0.5), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(q_tokens=1 << 31), "too many tokens"), (dict(q=None), "null"),
    (dict(v=None), "null"), (dict(starts=None), "null"), (dict(out=None), "null"), (dict(k=GOOD + 8), "misaligned"),
    (dict(starts=GOOD + 2), "misaligned"), (dict(q_token_stride=250), "strides"), (dict(k_head_stride=0), "strides"),
    (dict(v_token_stride=-128), "strides")])
def test_prompt_refusals(change, message):
    refused(message, "bgtq_prompt_attend", C.byref(prompt(**change)), None)


def test_prompt_without_work():
    _lib.call("bgtq_prompt_attend", C.byref(prompt(q_tokens=0)), None)
    _lib.call("bgtq_prompt_attend", C.byref(prompt(sequences=0)), None)


def test_prompt_workspace_refusals():
    refused("head dim", "bgtq_prompt_workspace", 0, 80, C.byref(C.c_size_t()))
    refused("null|invalid|head dim", "bgtq_prompt_workspace", 0, 64, None)


def test_python_refusals():
    import torch
    from bgtq import PagedCache, prompt_attention
    for kw in (dict(format="fp8"), dict(dim=96), dict(page_size=20), dict(kv_heads=0), dict(pages=0)):
        with pytest.raises(_lib.RangeError):
            PagedCache(**{**dict(kv_heads=2, dim=64, pages=4, page_size=16, format="int8"), **kw})
    with pytest.raises(_lib.RangeError, match="CUDA tensor"):
        PagedCache(2, 64, 4, 16, "f16", storage=dict(k=torch.zeros(4, 2, 16, 64).half(), v=torch.zeros(4, 2, 16, 64).half()))
    x, s = torch.zeros(4, 2, 64).half(), torch.tensor([0, 4], dtype=torch.int32)
    for args in ((x, x, x, s), (x.float(), x.float(), x.float(), s), (x[:, :, :32], x, x, s), (x, x, x[:2], s)):
        with pytest.raises(_lib.RangeError):
            prompt_attention(*args)
