"""Serving requests of different lengths: packed prompts and a paged, quantised K/V cache.

    prompt_attention   a whole batch of prompts, packed one after the other, in one call
    PagedCache         K and V of every request in the pages of one pool, in 16, 8 or 4 bits:
                       ``write`` quantises new rows, ``read`` gives back what rows stand for,
                       ``attend`` runs one new token of every request over its own pages

No counterpart in the reference, whose stores hold one sequence each.  CUDA tensors in, CUDA
tensors out, ordered on the current stream of the tensors' device; nothing synchronises, and
nothing is differentiated: results do not require gradients, whatever the arguments do.
Indices that only the GPU sees (slots, page tables, lengths, starts) are checked there: what
lies outside the cache is left out and sets a bit of `device_status` (4: slot or page, 8:
length or starts).

Attention keeps a workspace for every stream that it has been called on.  A CUDA graph
recorded on such a stream uses that one, so it is not replayed at the same time as calls there or
other graphs that were recorded there; recorded on a stream without one, it has its own.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

_DTYPE = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
_HALF = {torch.float16: "f16", torch.bfloat16: "bf16"}
# format: (code, element type)
_FORMATS = {"f16": (_lib.PAGES_F16, torch.float16), "bf16": (_lib.PAGES_BF16, torch.bfloat16),
            "int8": (_lib.PAGES_INT8, torch.int8), "int4": (_lib.PAGES_INT4, torch.uint8)}
_LEAST_SCALE = 2.0 ** -149  # the least FP32: a zero stands for the default at the C ABI


def _refuse(message: str):
    raise _lib.RangeError(_lib.EINVAL, message)


def _room(size: int, device):
    """A workspace, its counters zeroed: address, bytes, tensor."""
    have = torch.empty(size, dtype=torch.uint8, device=device)
    have[:_lib.WORKSPACE_ZEROED].zero_()
    return have.data_ptr(), size, have


def _recording(device) -> bool:
    with torch.cuda.device(device):  # the tensors' device need not be the current one
        return torch.cuda.is_current_stream_capturing()


def _stream(device: int) -> int:
    return torch.cuda.current_stream(device).cuda_stream


class PagedCache:
    """K and V rows of ``pages`` pages of ``page_size`` tokens for ``kv_heads`` heads.

    format "f16" / "bf16" (rounded rows), "int8" (one BF16 scale a row) or "int4" (one BF16
    scale for every 32 dimensions).  The memory is the tensors ``k``, ``v`` [pages, kv_heads,
    page_size, row] and ``k_scales``, ``v_scales`` [pages, kv_heads, page_size, groups] (None
    in 16 bits), allocated zeroed here or taken from ``storage`` (a dict of those four).  Which
    page belongs to which request is the caller's business: rows are addressed by slots (page *
    page_size + row), requests by rows of a page table."""

    def __init__(self, kv_heads: int, dim: int, pages: int, page_size: int = 64, format: str = "int8",
                 device: int = 0, storage: dict | None = None):
        if format not in _FORMATS:
            _refuse(f"Paged cache: format must be one of {sorted(_FORMATS)}")
        if dim not in (64, 128):
            _refuse("Paged cache: head dim must be 64 or 128")
        if page_size not in (16, 32, 64, 128, 256):
            _refuse("Paged cache: page size must be a power of two from 16 to 256")
        if not 1 <= kv_heads <= 1024 or not 1 <= pages < 2**31:
            _refuse("Paged cache: invalid head or page count")
        code, dtype = _FORMATS[format]
        groups = {"int8": 1, "int4": dim // 32}.get(format, 0)
        want = dict(k=(dtype, dim // 2 if format == "int4" else dim), k_scales=(torch.bfloat16, groups))
        want.update(v=want["k"], v_scales=want["k_scales"])
        tensors = {}
        for name, (dt, width) in want.items():
            shape = (pages, kv_heads, page_size, width)
            if not width:
                t = None
                if storage is not None and storage.get(name) is not None:
                    _refuse(f"Paged cache: {format} pages have no {name}")
            elif storage is None:
                t = torch.zeros(shape, dtype=dt, device=torch.device("cuda", device))
            else:
                t = storage.get(name)
                if t is None or not t.is_cuda or t.dtype != dt or tuple(t.shape) != shape or not t.is_contiguous():
                    _refuse(f"Paged cache: {name} must be a contiguous CUDA tensor {list(shape)} of {dt}")
            tensors[name] = t
        self.k, self.v, self.k_scales, self.v_scales = (tensors[n] for n in ("k", "v", "k_scales", "v_scales"))
        if any(t is not None and t.device != self.k.device for t in tensors.values()):
            _refuse("Paged cache: all storage must be on one device")
        self.kv_heads, self.dim, self.pages, self.page_size = int(kv_heads), int(dim), int(pages), int(page_size)
        self.format, self.device = format, self.k.device.index
        self._desc = _lib.PagedCacheDesc(self.device, code, kv_heads, dim, page_size, pages, self.k.data_ptr(),
                                         self.v.data_ptr(), *(None if t is None else t.data_ptr()
                                                              for t in (self.k_scales, self.v_scales)))
        self._ref = C.byref(self._desc)
        self._on = self.k.device
        self._workspace = {}
        library = _lib.lib()
        self._write, self._read = library.bgtq_paged_write, library.bgtq_paged_read
        self._attend = library.bgtq_paged_attend

    def _check_slots(self, slots) -> None:
        if slots.dtype != torch.int64 or slots.device != self._on or slots.dim() != 1 or not slots.is_contiguous():
            _refuse("Paged cache: slots must be a contiguous one-dimensional int64 tensor on the cache's device")

    def write(self, k, v, slots) -> None:
        """Store rows k, v [tokens, kv_heads, dim] (float16, bfloat16 or float32; any strides with
        a contiguous last dimension) at ``slots`` [tokens].  Negative slots are padding."""
        self._check_slots(slots)
        shape = (slots.shape[0], self.kv_heads, self.dim)
        if k.shape != shape or v.shape != shape:
            _refuse("Paged write: K and V must be [tokens, kv_heads, dim] with one slot a token")
        dtype = _DTYPE.get(k.dtype)
        if dtype is None or v.dtype != k.dtype:
            _refuse("Paged write: K and V must both be float16, bfloat16 or float32")
        if k.device != self._on or v.device != self._on:
            _refuse("Paged write: K and V must be on the cache's device")
        k0, k1, k2 = k.stride()
        v0, v1, v2 = v.stride()
        if k2 != 1 or v2 != 1:
            _refuse("Paged write: the last dimension must be contiguous")
        status = self._write(self._ref, k.data_ptr(), v.data_ptr(), dtype, shape[0], k0, k1, v0, v1, slots.data_ptr(),
                             _stream(self.device))
        if status:
            _lib.check(status)

    def read(self, slots, dtype=None):
        """(k, v) [tokens, kv_heads, dim]: the values that the rows at ``slots`` stand for, as
        dtype (default: the pages' own type, bfloat16 for 8- and 4-bit pages); zeros for
        negative slots."""
        self._check_slots(slots)
        if dtype is None:
            dtype = torch.float16 if self.format == "f16" else torch.bfloat16
        code = _DTYPE.get(dtype)
        if code is None:
            _refuse("Paged read: dtype must be float16, bfloat16 or float32")
        n = slots.shape[0]
        k = slots.new_empty((n, self.kv_heads, self.dim), dtype=dtype)
        v = torch.empty_like(k)
        status = self._read(self._ref, slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), code, _stream(self.device))
        if status:
            _lib.check(status)
        return k, v

    def attend(self, q, table, lengths, scale: float | None = None, out=None, lse: bool = False):
        """One new token of every request: q [batch, q_heads, dim] (float16 or bfloat16, the
        pages' type over 16-bit pages) over the first ``lengths`` [batch] (int32) tokens of the
        pages in ``table`` [batch, width] (int32).  Returns out [batch, q_heads, dim], with
        ``lse`` also the log sums [batch, q_heads] (float32).  scale: 1 / sqrt(dim) if None."""
        shape = q.shape
        if len(shape) != 3 or shape[2] != self.dim or shape[1] < 1 or shape[1] % self.kv_heads:
            _refuse("Paged attention: Q must be [batch, q_heads, dim], q_heads a multiple of kv_heads")
        batch, heads, _ = shape
        dtype = q.dtype
        if dtype not in _HALF or self.format in _HALF.values() and self.format != _HALF[dtype]:
            _refuse("Paged attention: Q must be float16 or bfloat16, and of the type of 16-bit pages")
        q0, q1, q2 = q.stride()
        if q.device != self._on or q2 != 1:
            _refuse("Paged attention: Q must be on the cache's device with a contiguous last dimension")
        if (table.dim() != 2 or table.shape[0] != batch or table.dtype != torch.int32 or table.device != self._on
                or (table.shape[1] > 1 and table.stride(1) != 1)):
            _refuse("Paged attention: the table must be int32 [batch, width] on the cache's device")
        if (lengths.dim() != 1 or lengths.shape[0] != batch or lengths.dtype != torch.int32
                or lengths.device != self._on or (batch > 1 and lengths.stride(0) != 1)):
            _refuse("Paged attention: lengths must be int32 [batch] on the cache's device")
        if scale is not None and not 0.0 < scale < float("inf"):
            _refuse("Paged attention: scale must be positive and finite")
        if out is None:
            out = q.new_empty(shape)
        elif out.shape != shape or out.dtype != dtype or out.device != self._on or not out.is_contiguous():
            _refuse("Paged attention: out must be contiguous, of Q's shape, type and device")
        sums = q.new_empty((batch, heads), dtype=torch.float32) if lse else None
        st = _stream(self.device)
        work = self._workspace.get((st, heads)) or self._work(heads, st)
        status = self._attend(self._ref, q.data_ptr(), _DTYPE[dtype], batch, heads, q0, q1, table.data_ptr(),
                              table.stride(0), table.shape[1], lengths.data_ptr(), 0.0 if scale is None else max(scale, _LEAST_SCALE),
                              out.data_ptr(), sums.data_ptr() if lse else None, work[0], work[1], st)
        if status:
            _lib.check(status)
        return (out, sums) if lse else out

    def _work(self, heads: int, stream: int):
        """The stream's own workspace (calls on different streams may overlap): address, bytes, tensor."""
        need = C.c_size_t()
        _lib.call("bgtq_paged_attend_workspace", self._ref, heads, C.byref(need))
        work = _room(need.value, self._on)
        if not _recording(self._on):  # a graph's own is zeroed by its replays alone
            self._workspace[stream, heads] = work
        return work


_prompt_work = {}


def _prompt_workspace(device, dim: int, stream: int):
    """The stream's own workspace (calls on different streams may overlap): address, bytes, tensor."""
    need = C.c_size_t()
    _lib.call("bgtq_prompt_workspace", device.index, dim, C.byref(need))
    work = _room(need.value, device)
    if not _recording(device):  # a graph's own is zeroed by its replays alone
        _prompt_work[device.index, dim, stream] = work
    return work


def _ready_again(device: int):
    """Zeroes the counters of the device's prompt workspaces: a call whose wait ran out ends without its joins.
    (One-token attention waits for nothing, and a graph's own workspace is zeroed by its replays.)"""
    torch.cuda.synchronize(device)
    for (on, _, _), work in _prompt_work.items():
        if on == device:
            work[2][:_lib.WORKSPACE_ZEROED].zero_()
    torch.cuda.synchronize(device)


def _even(t):
    """t, or a packed copy of it where the kernels' loads cannot follow its strides or address, and its
    token and head strides (that of a dimension of one element is never used)."""
    s0, s1, s2 = t.stride()
    n0, n1, _ = t.shape
    if s2 != 1 or n0 > 1 and (s0 <= 0 or s0 % 8) or n1 > 1 and (s1 <= 0 or s1 % 8) or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        s0, s1, _ = t.stride()
    return t, s0 if n0 > 1 else 8, s1 if n1 > 1 else 8


def prompt_attention(q, k, v, starts, key_starts=None, causal: bool = True, scale: float | None = None, out=None,
                     lse: bool = False):
    """Attention of a packed batch of prompts: q [tokens, q_heads, dim], k and v [key tokens,
    kv_heads, dim] (float16 or bfloat16, one type; q_heads a multiple of kv_heads).  Sequence s
    is query rows starts[s] .. starts[s + 1] and key rows key_starts[s] .. key_starts[s + 1]
    (int32 [sequences + 1]; key_starts None: the same as starts).  Causal rows see their
    sequence's keys up to their own, counted from the end, so a chunk whose prefix is cached
    passes more keys than queries.  Rows that see nothing are zeros; rows that no sequence holds are
    not written (of a new output they are whatever its memory held).  Any strides with a
    contiguous last dimension; a tensor whose strides or address are not multiples of 16
    bytes is copied.  Returns out [tokens, q_heads, dim], with ``lse`` also the log sums
    [tokens, q_heads] (float32)."""
    shape, keys = q.shape, k.shape
    if len(shape) != 3 or len(keys) != 3 or v.shape != keys or shape[2] != keys[2]:
        _refuse("Prompt attention: Q must be [tokens, q_heads, dim], K and V [key tokens, kv_heads, dim]")
    dtype, on = q.dtype, q.device
    if dtype not in _HALF or k.dtype != dtype or v.dtype != dtype:
        _refuse("Prompt attention: Q, K and V must all be float16 or all bfloat16")
    if on.type != "cuda" or k.device != on or v.device != on:
        _refuse("Prompt attention: Q, K and V must be CUDA tensors on one device")
    tokens, heads, dim = shape
    if dim not in (64, 128) or keys[1] < 1 or heads < 1 or heads % keys[1]:
        _refuse("Prompt attention: head dim must be 64 or 128 and q_heads a multiple of kv_heads")
    for s in (starts,) if key_starts is None else (starts, key_starts):
        if (s.dim() != 1 or s.shape[0] != starts.shape[0] or s.shape[0] < 1 or s.dtype != torch.int32 or s.device != on
                or not s.is_contiguous()):
            _refuse("Prompt attention: starts must be int32 [sequences + 1] on Q's device")
    if key_starts is None and keys[0] != tokens:
        _refuse("Prompt attention: key_starts are needed when K has other tokens than Q")
    if scale is not None and not 0.0 < scale < float("inf"):
        _refuse("Prompt attention: scale must be positive and finite")
    if out is None:
        out = q.new_empty(shape)
    elif out.shape != shape or out.dtype != dtype or out.device != on or not out.is_contiguous():
        _refuse("Prompt attention: out must be contiguous, of Q's shape, type and device")
    sums = q.new_empty((tokens, heads), dtype=torch.float32) if lse else None
    q, q0, q1 = _even(q)
    k, k0, k1 = _even(k)
    v, v0, v1 = _even(v)
    dev = on.index
    st = _stream(dev)
    work = _prompt_work.get((dev, dim, st)) or _prompt_workspace(on, dim, st)
    p = _lib.PromptDesc(dev, _DTYPE[dtype], starts.shape[0] - 1, heads, keys[1], dim, tokens, keys[0], q.data_ptr(),
                        k.data_ptr(), v.data_ptr(), q0, q1, k0, k1, v0, v1, starts.data_ptr(),
                        None if key_starts is None else key_starts.data_ptr(), 1 if causal else 0,
                        0.0 if scale is None else max(scale, _LEAST_SCALE), out.data_ptr(), sums.data_ptr() if lse else None, work[0], work[1])
    status = _lib.lib().bgtq_prompt_attend(C.byref(p), st)
    if status:
        _lib.check(status)
    return (out, sums) if lse else out
