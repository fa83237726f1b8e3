"""What the operators of a serving step refuse, at the C ABI: every check comes before a device is touched,
so these run without one."""
import ctypes as C

import pytest

from bgtq import _lib
from test_serving_refusals import GOOD, cache, refused


def append(c, **kw):
    d = dict(dtype=_lib.BF16, q_heads=4, tokens=3, q=GOOD, k=GOOD, v=GOOD, q_token_stride=512, q_head_stride=64,
             k_token_stride=512, k_head_stride=64, v_token_stride=512, v_head_stride=64, slots=GOOD, rotary=GOOD,
             rotary_rows=100, positions=GOOD, q_norm=GOOD, k_norm=None, eps=1e-6, out_dtype=_lib.BF16, q_out=GOOD,
             k_out=None)
    d.update(kw)
    return "bgtq_paged_append", C.byref(c), C.byref(_lib.AppendDesc(**d)), None


def chunk(c, **kw):
    d = dict(dtype=_lib.BF16, batch=2, q_heads=4, q_tokens=7, q=GOOD, q_token_stride=256, q_head_stride=64, starts=GOOD,
             table=GOOD, table_stride=4, table_width=4, lengths=GOOD, scale=0.0, window=0, sinks=0, out=GOOD, lse=None,
             workspace=GOOD, workspace_bytes=1 << 40)
    d.update(kw)
    return "bgtq_paged_attend_chunk", C.byref(c), C.byref(_lib.ChunkDesc(**d)), None


def logits(**kw):
    d = dict(device=0, dtype=_lib.F32, batch=2, vocab=100, logits=GOOD, logits_stride=100, tokens=GOOD,
             tokens_stride=10, width=10, id_bytes=8, lengths=GOOD, repetition=GOOD, presence=None, frequency=None,
             bias_ids=GOOD, bias=GOOD, bias_stride=3, entries=3, mask=GOOD, mask_stride=4, out=GOOD, out_stride=100)
    d.update(kw)
    return "bgtq_adjust_logits", C.byref(_lib.LogitsDesc(**d)), None


@pytest.mark.parametrize("change,message", [
    (dict(dim=96), "head dim"), (dict(format=5), "format"), (dict(page_size=24), "page size"),
    (dict(kv_heads=0), "head or page count"), (dict(pages=0), "head or page count"), (dict(k=None), "16-byte"),
    (dict(v_scales=GOOD + 8), "scales")])
def test_a_wrong_cache(change, message):
    c = cache(**change)
    for call in (append(c), chunk(c)):
        refused(message, *call)
    refused(message, "bgtq_paged_chunk_workspace", C.byref(c), 2, C.byref(C.c_size_t()))


@pytest.mark.parametrize("change,message", [
    (dict(dtype=0), "source must be"), (dict(out_dtype=4), "output must be"), (dict(q_heads=0), "head count"),
    (dict(q_heads=65536), "head count"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(eps=float("inf")), "eps"), (dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"),
    (dict(slots=None), "null"), (dict(rotary=None), "null"), (dict(q_out=None), "null"), (dict(q=GOOD + 1), "misaligned"),
    (dict(dtype=_lib.F32, v=GOOD + 2), "misaligned"), (dict(slots=GOOD + 4), "misaligned"),
    (dict(positions=GOOD + 4), "misaligned"), (dict(rotary=GOOD + 4), "misaligned"), (dict(q_norm=GOOD + 4), "misaligned"),
    (dict(k_norm=GOOD + 8), "misaligned"), (dict(q_out=GOOD + 8), "misaligned"), (dict(k_out=GOOD + 8), "misaligned"),
    (dict(tokens=1 << 29), "too many rows"), (dict(tokens=1 << 60), "too many rows"),
    (dict(rotary_rows=1 << 31), "cosines"), (dict(positions=None, rotary_rows=2), "cosines")])
def test_append_refusals(change, message):
    refused(message, *append(cache(), **change))


def test_append_of_nothing():
    refused("null", "bgtq_paged_append", C.byref(cache()), None, None)
    _lib.call(*append(cache(), tokens=0, q=None))


@pytest.mark.parametrize("change,message", [
    (dict(dtype=_lib.F32), "queries must be"), (dict(q_heads=3), "head count"), (dict(q_heads=0), "head count"),
    (dict(q_heads=258), "head count"), (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=3e38), "scale"), (dict(window=1 << 31), "window"),
    (dict(sinks=1 << 31), "window"), (dict(batch=65536), "too many"), (dict(q_tokens=1 << 31), "too many"),
    (dict(q_tokens=1 << 62), "too many"), (dict(starts=None), "one query row"), (dict(q=None), "null"),
    (dict(table=None), "null"), (dict(lengths=None), "null"), (dict(out=None), "null"), (dict(table_width=1 << 27), "2\\^31"),
    (dict(q=GOOD + 8), "misaligned"), (dict(out=GOOD + 8), "misaligned"), (dict(starts=GOOD + 2), "misaligned"),
    (dict(table=GOOD + 1), "misaligned"), (dict(lengths=GOOD + 2), "misaligned"), (dict(lse=GOOD + 2), "misaligned"),
    (dict(q_token_stride=0), "strides"), (dict(q_token_stride=-256), "strides"), (dict(q_head_stride=60), "strides"),
    (dict(q_head_stride=1 << 40), "strides")])
def test_chunk_refusals(change, message):
    refused(message, *chunk(cache(), **change))


def test_chunk_types_and_nothing():
    for fmt, dt in ((_lib.PAGES_F16, _lib.BF16), (_lib.PAGES_BF16, _lib.F16)):
        refused("type of 16-bit pages", *chunk(cache(format=fmt), dtype=dt))
    refused("null", "bgtq_paged_attend_chunk", C.byref(cache()), None, None)
    _lib.call(*chunk(cache(), batch=0, q=None))
    _lib.call(*chunk(cache(), q_tokens=0, q=None))
    _lib.call(*chunk(cache(), batch=0, q_tokens=0, starts=None, q=None))
    refused("head count", "bgtq_paged_chunk_workspace", C.byref(cache()), 3, C.byref(C.c_size_t()))
    refused("head count", "bgtq_paged_chunk_workspace", C.byref(cache()), 4, None)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=0), "must be FP16"), (dict(vocab=0), "vocabulary"), (dict(vocab=1 << 31), "vocabulary"),
    (dict(batch=65536), "too many rows"), (dict(width=1 << 31), "too many tokens"), (dict(entries=1 << 31), "too many tokens"),
    (dict(id_bytes=2), "4 or 8"), (dict(logits=None), "null"), (dict(out=None), "null"), (dict(bias=None), "null"),
    (dict(bias_ids=None), "null"), (dict(logits=GOOD + 2), "misaligned"), (dict(out=GOOD + 1), "misaligned"),
    (dict(tokens=GOOD + 4), "misaligned"), (dict(id_bytes=4, tokens=GOOD + 2), "misaligned"),
    (dict(lengths=GOOD + 2), "misaligned"), (dict(repetition=GOOD + 1), "misaligned"), (dict(mask=GOOD + 2), "misaligned"),
    (dict(bias=GOOD + 2), "misaligned"), (dict(bias_ids=GOOD + 2), "misaligned")])
def test_logits_refusals(change, message):
    refused(message, *logits(**change))


def test_logits_of_nothing():
    refused("null", "bgtq_adjust_logits", None, None)
    _lib.call(*logits(batch=0, logits=None))
