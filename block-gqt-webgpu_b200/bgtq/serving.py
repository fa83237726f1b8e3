"""Serving requests of different lengths: packed prompts and a paged, quantised K/V cache.

    prompt_attention   a whole batch of prompts, packed one after the other, in one call
    PagedCache         K and V of every request in the pages of one pool, in 16, 8 or 4 bits:
                       ``write`` quantises new rows, ``append`` rotates them (and norms their
                       heads) on the way, ``read`` gives back what rows stand for, ``attend`` runs
                       one new token of every request over its own pages, ``attend_chunk`` any
                       number of them; both over all tokens or a window and the first few
    adjust_logits      penalties for repeated tokens, biases and grammar masks, before a token is
                       chosen

No counterpart in the reference, whose stores hold one sequence each.  CUDA tensors in, CUDA
tensors out, ordered on the current stream of the tensors' device; nothing synchronises, and
nothing is differentiated: results do not require gradients, whatever the arguments do.
Indices that only the GPU sees (slots, page tables, lengths, starts) are checked there: what
lies outside the cache is left out and sets a bit of `device_status` (4: slot or page, 8:
length or starts).

Attention keeps a workspace for every stream that it has been called on (`PagedDecoder` has workspaces
of its own).  A CUDA graph recorded on such a stream uses that one, so it is not replayed at the same
time as calls there or other graphs that were recorded there; recorded on a stream without one, it
has its own.
"""
from __future__ import annotations

import ctypes as C
import weakref

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


# torch.cuda.current_stream(device).cuda_stream without the objects in between, which are a microsecond of a call
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device: int) -> int:
    return torch.cuda.current_stream(device).cuda_stream if _raw_stream is None else _raw_stream(device)


class _Workspaces(dict):
    """(device, head dim, stream): (address, bytes, tensor).  `_ready_again` finds them all."""
    made = weakref.WeakSet()
    __hash__, __eq__ = object.__hash__, object.__eq__

    def __init__(self):
        super().__init__()
        _Workspaces.made.add(self)


_prompt_work, _chunk_work = _Workspaces(), _Workspaces()


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
        self._workspace, self._chunk_work = {}, _chunk_work
        library = _lib.lib()
        self._write, self._read = library.bgtq_paged_write, library.bgtq_paged_read
        self._attend = library.bgtq_paged_attend
        self._append, self._chunk = library.bgtq_paged_append, library.bgtq_paged_attend_chunk

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

    def append(self, q, k, v, slots, rotary, positions=None, q_norm=None, k_norm=None, eps: float = 1e-6, dtype=None,
               keys: bool = False):
        """New tokens in one pass: heads of q [tokens, q_heads, dim] and k [tokens, kv_heads, dim] are
        normed, where q_norm / k_norm [dim] (float32) are given (x norm / sqrt(mean(x^2) + eps)), and rotated;
        k and v [tokens, kv_heads, dim] are stored at ``slots`` [tokens] as ``write`` stores them.  All
        three are float16, bfloat16 or float32, of any strides with a contiguous last dimension.
        Dimension i < dim / 2 is rotated with dimension i + dim / 2 by the token's row of ``rotary``
        [rows, dim] (float32: dim / 2 cosines, then sines), row positions[t] (int64) or, without
        positions, row t.  Negative slots are padding: nothing is stored of them; others come once in a call.  A token whose
        position is outside the table is not stored and its results are zeros.
        Returns the queries, as dtype (default: q's own), with ``keys`` also the keys."""
        self._check_slots(slots)
        n, shape = slots.shape[0], q.shape
        if len(shape) != 3 or shape[0] != n or shape[1] < 1 or shape[2] != self.dim:
            _refuse("Paged append: Q must be [tokens, q_heads, dim] with one slot a token")
        if k.shape != (n, self.kv_heads, self.dim) or v.shape != k.shape:
            _refuse("Paged append: K and V must be [tokens, kv_heads, dim] with one slot a token")
        code = _DTYPE.get(q.dtype)
        if code is None or k.dtype != q.dtype or v.dtype != q.dtype:
            _refuse("Paged append: Q, K and V must all be float16, bfloat16 or float32")
        to = q.dtype if dtype is None else dtype
        out = _DTYPE.get(to)
        if out is None:
            _refuse("Paged append: dtype must be float16, bfloat16 or float32")
        on = self._on
        if q.device != on or k.device != on or v.device != on:
            _refuse("Paged append: Q, K and V must be on the cache's device")
        q0, q1, q2 = q.stride()
        k0, k1, k2 = k.stride()
        v0, v1, v2 = v.stride()
        if q2 != 1 or k2 != 1 or v2 != 1:
            _refuse("Paged append: the last dimension must be contiguous")
        if (rotary.dim() != 2 or rotary.shape[1] != self.dim or rotary.dtype != torch.float32 or rotary.device != on
                or not rotary.is_contiguous()):
            _refuse("Paged append: rotary must be a contiguous float32 tensor [rows, dim] on the cache's device")
        if positions is None:
            if rotary.shape[0] < n:
                _refuse("Paged append: without positions rotary must have a row for every token")
        elif positions.shape != (n,) or positions.dtype != torch.int64 or positions.device != on or not positions.is_contiguous():
            _refuse("Paged append: positions must be a contiguous int64 tensor [tokens] on the cache's device")
        for w in (q_norm, k_norm):
            if w is not None and (w.shape != (self.dim,) or w.dtype != torch.float32 or w.device != on
                                  or not w.is_contiguous()):
                _refuse("Paged append: norms must be contiguous float32 tensors [dim] on the cache's device")
        if not 0.0 <= eps < float("inf"):
            _refuse("Paged append: eps must be nonnegative and finite")
        q_out = q.new_empty(shape, dtype=to)
        k_out = q.new_empty(k.shape, dtype=to) if keys else None
        p = _lib.AppendDesc(code, shape[1], n, q.data_ptr(), k.data_ptr(), v.data_ptr(), q0, q1, k0, k1, v0, v1,
                            slots.data_ptr(), rotary.data_ptr(), rotary.shape[0],
                            None if positions is None else positions.data_ptr(),
                            None if q_norm is None else q_norm.data_ptr(),
                            None if k_norm is None else k_norm.data_ptr(), eps, out, q_out.data_ptr(),
                            k_out.data_ptr() if keys else None)
        status = self._append(self._ref, C.byref(p), _stream(self.device))
        if status:
            _lib.check(status)
        return (q_out, k_out) if keys else q_out

    def attend(self, q, table, lengths, scale: float | None = None, out=None, lse: bool = False,
               window: int | None = None, sinks: int = 0):
        """One new token of every request: q [batch, q_heads, dim] (float16 or bfloat16, the
        pages' type over 16-bit pages) over the first ``lengths`` [batch] (int32) tokens of the
        pages in ``table`` [batch, width] (int32), with ``window`` only over the last of them and
        the first ``sinks`` (as `attend_chunk` does it).  Returns out [batch, q_heads, dim], with
        ``lse`` also the log sums [batch, q_heads] (float32).  scale: 1 / sqrt(dim) if None."""
        if window is not None:
            return self.attend_chunk(q, None, table, lengths, scale, window, sinks, out, lse)
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

    def attend_chunk(self, q, starts, table, lengths, scale: float | None = None, window: int | None = None,
                     sinks: int = 0, out=None, lse: bool = False):
        """Any number of new tokens of every request over its pages, which hold their rows already:
        q [tokens, q_heads, dim] (float16 or bfloat16, the pages' type over 16-bit pages), rows
        starts[b] .. starts[b + 1] (int32 [batch + 1]) the last tokens of the ``lengths`` [batch]
        (int32) that the pages in ``table`` [batch, width] (int32) hold of request b; starts None: one
        row each.  A row sees the tokens up to its own, with ``window`` the last so many of them, its own
        included, and the first ``sinks``.  Rows that see nothing are zeros; rows that no
        request holds are not written (of a new output they are whatever its memory held).  Any
        strides of q with a contiguous last dimension; one whose strides or address are not
        multiples of 16 bytes is copied.  Returns out [tokens, q_heads, dim], with ``lse`` also the
        log sums [tokens, q_heads] (float32).  scale: 1 / sqrt(dim) if None."""
        shape = q.shape
        if len(shape) != 3 or shape[2] != self.dim or shape[1] < 1 or shape[1] % self.kv_heads:
            _refuse("Chunk attention: Q must be [tokens, q_heads, dim], q_heads a multiple of kv_heads")
        tokens, heads, _ = shape
        if heads // self.kv_heads > 128:
            _refuse("Chunk attention: at most 128 query heads for a KV head")
        dtype, on = q.dtype, self._on
        if dtype not in _HALF or self.format in _HALF.values() and self.format != _HALF[dtype]:
            _refuse("Chunk attention: Q must be float16 or bfloat16, and of the type of 16-bit pages")
        if q.device != on:
            _refuse("Chunk attention: Q must be on the cache's device")
        batch = tokens if starts is None else starts.shape[0] - 1 if starts.dim() == 1 else -1
        if starts is not None and (batch < 0 or starts.dtype != torch.int32 or starts.device != on
                                   or not starts.is_contiguous()):
            _refuse("Chunk attention: starts must be int32 [batch + 1] on the cache's device")
        if (table.dim() != 2 or table.shape[0] != batch or table.dtype != torch.int32 or table.device != on
                or (table.shape[1] > 1 and table.stride(1) != 1)):
            _refuse("Chunk attention: the table must be int32 [batch, width] on the cache's device")
        if (lengths.dim() != 1 or lengths.shape[0] != batch or lengths.dtype != torch.int32 or lengths.device != on
                or (batch > 1 and lengths.stride(0) != 1)):
            _refuse("Chunk attention: lengths must be int32 [batch] on the cache's device")
        if scale is not None and not 0.0 < scale < float("inf"):
            _refuse("Chunk attention: scale must be positive and finite")
        if window is not None and not 1 <= window < 2**31 or not 0 <= sinks < 2**31:
            _refuse("Chunk attention: window must be positive and sinks nonnegative, both below 2^31")
        if out is None:
            out = q.new_empty(shape)
        elif out.shape != shape or out.dtype != dtype or out.device != on or not out.is_contiguous():
            _refuse("Chunk attention: out must be contiguous, of Q's shape, type and device")
        sums = q.new_empty((tokens, heads), dtype=torch.float32) if lse else None
        q, q0, q1 = _even(q)
        st = _stream(self.device)
        work = self._chunk_work.get((self.device, self.dim, st)) or _chunk_workspace(self, heads, st)
        p = _lib.ChunkDesc(_DTYPE[dtype], batch, heads, tokens, q.data_ptr(), q0, q1,
                           None if starts is None else starts.data_ptr(), table.data_ptr(), table.stride(0),
                           table.shape[1], lengths.data_ptr(), 0.0 if scale is None else max(scale, _LEAST_SCALE),
                           window or 0, sinks, out.data_ptr(), sums.data_ptr() if lse else None, work[0], work[1])
        status = self._chunk(self._ref, C.byref(p), st)
        if status:
            _lib.check(status)
        return (out, sums) if lse else out


def _prompt_workspace(device, dim: int, stream: int):
    """The stream's own workspace (calls on different streams may overlap): address, bytes, tensor."""
    need = C.c_size_t()
    _lib.call("bgtq_prompt_workspace", device.index, dim, C.byref(need))
    work = _room(need.value, device)
    if not _recording(device):  # a graph's own is zeroed by its replays alone
        _prompt_work[device.index, dim, stream] = work
    return work


def _chunk_workspace(cache, heads: int, stream: int):
    """The same for chunks over pages: one for all caches of a device and head dim, but for a decoder's."""
    need = C.c_size_t()
    _lib.call("bgtq_paged_chunk_workspace", cache._ref, heads, C.byref(need))
    work = _room(need.value, cache._on)
    if not _recording(cache._on):
        cache._chunk_work[cache.device, cache.dim, stream] = work
    return work


def _ready_again(device: int):
    """Zeroes the counters of the device's prompt and chunk workspaces: a call whose wait ran out ends without its
    joins.  (One-token attention waits for nothing, and a graph's own workspace is zeroed by its replays.)"""
    torch.cuda.synchronize(device)
    for works in list(_Workspaces.made):
        for (on, _, _), work in list(works.items()):
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


def _per_row(x, batch: int, device, name: str):
    """A penalty as float32 [batch]: a tensor as it is, a number filled in."""
    if not isinstance(x, torch.Tensor):
        x = C.c_float(x).value  # what FP32 makes of it: infinity and zero among it
        if not -float("inf") < x < float("inf") or name == "repetition" and x <= 0.0:
            _refuse(f"Logits: {name} must be finite" + (" and positive" if name == "repetition" else "") + " in FP32")
        return torch.full((batch,), x, dtype=torch.float32, device=device)
    if x.shape != (batch,) or x.dtype != torch.float32 or x.device != device or not x.is_contiguous():
        _refuse(f"Logits: {name} must be a number or a contiguous float32 tensor [batch] on the logits' device")
    return x


def _rows(t, batch: int, device, name: str, shape: str):
    """The row stride of [batch or 1, n] (one row for all: 0)."""
    if t.dim() != 2 or t.shape[0] not in (1, batch) or t.device != device or t.shape[1] > 1 and t.stride(1) != 1:
        _refuse(f"Logits: {name} must be {shape} on the logits' device, with a contiguous last dimension")
    return t.stride(0) if t.shape[0] > 1 else 0


def adjust_logits(logits, tokens=None, lengths=None, repetition=None, presence=None, frequency=None, bias_ids=None,
                  bias=None, mask=None, out=None):
    """Penalties for repeated tokens, biases and a grammar's mask on logits [batch, vocab] (float16, bfloat16 or
    float32), in this order, where they are given; FP32 within, rounded once:

        repetition   x / repetition if x > 0, else x * repetition   for tokens of the row's history
        presence     x - presence                                   for tokens of the row's history
        frequency    x - frequency * (how often the history has the token)
        bias         x + bias[b, j] for token bias_ids[b, j]        (one that comes twice is added twice)
        mask         -inf where bit v % 32 of mask[b, v // 32] is not set

    The history of row b is the first lengths[b] (int32 [batch]; None: all) of tokens [batch, width] (int32 or
    int64), negative ones left out.  Penalties are numbers or float32 [batch]; repetition is positive.  bias_ids (int32) and bias
    (float32) are [batch, n] or, for all rows alike, [1, n]; mask (int32, the bits of 32 tokens a word) [batch,
    ceil(vocab / 32)] or [1, ...].  Token ids past the vocabulary are left out and set bit 4 of `device_status`, lengths
    outside 0 .. width are cut and set bit 8.  Returns the result, a new tensor or ``out``, which may be the logits
    themselves and else shares no memory with them."""
    if logits.dim() != 2 or not logits.is_cuda or logits.shape[1] < 1 or logits.stride(1) != 1 and logits.shape[1] > 1:
        _refuse("Logits: logits must be a CUDA tensor [batch, vocab] with a contiguous last dimension")
    batch, vocab = logits.shape
    dtype, on = _DTYPE.get(logits.dtype), logits.device
    if dtype is None:
        _refuse("Logits: logits must be float16, bfloat16 or float32")
    tokens_stride = width = 0
    if tokens is not None:
        if (tokens.dim() != 2 or tokens.shape[0] != batch or tokens.dtype not in (torch.int32, torch.int64)
                or tokens.device != on or tokens.shape[1] > 1 and tokens.stride(1) != 1):
            _refuse("Logits: tokens must be int32 or int64 [batch, width] on the logits' device, with a contiguous "
                    "last dimension")
        tokens_stride, width = tokens.stride(0), tokens.shape[1]
    if lengths is not None and (tokens is None or lengths.shape != (batch,) or lengths.dtype != torch.int32
                                or lengths.device != on or not lengths.is_contiguous()):
        _refuse("Logits: lengths must be a contiguous int32 tensor [batch] on the logits' device, with tokens")
    if tokens is None and not repetition is presence is frequency is None:
        _refuse("Logits: penalties need tokens")
    if repetition is not None:
        repetition = _per_row(repetition, batch, on, "repetition")
    if presence is not None:
        presence = _per_row(presence, batch, on, "presence")
    if frequency is not None:
        frequency = _per_row(frequency, batch, on, "frequency")
    bias_stride = mask_stride = entries = 0
    if (bias is None) != (bias_ids is None):
        _refuse("Logits: bias and bias_ids come together")
    if bias is not None:
        if bias.dtype != torch.float32 or bias_ids.dtype != torch.int32 or bias.shape != bias_ids.shape:
            _refuse("Logits: bias must be float32 and bias_ids int32, of one shape")
        bias_stride = _rows(bias, batch, on, "bias", "[batch, n] or [1, n]")
        if _rows(bias_ids, batch, on, "bias_ids", "[batch, n] or [1, n]") != bias_stride:
            bias, bias_ids = bias.contiguous(), bias_ids.contiguous()
            bias_stride = bias.shape[1] if bias.shape[0] > 1 else 0
        entries = bias.shape[1]
    if mask is not None:
        mask_stride = _rows(mask, batch, on, "mask", "[batch, ceil(vocab / 32)] or [1, ceil(vocab / 32)]")
        if mask.dtype != torch.int32 or mask.shape[1] != (vocab + 31) // 32:
            _refuse("Logits: mask must be int32, a bit for each token of the vocabulary")
    if out is None:
        out = logits.new_empty((batch, vocab))
    elif (out.shape != logits.shape or out.dtype != logits.dtype or out.device != on
          or out.stride(1) != 1 and vocab > 1 or batch > 1 and out.stride(0) < vocab):
        _refuse("Logits: out must be of the logits' shape, type and device, with a contiguous last dimension")
    p = _lib.LogitsDesc(on.index, dtype, batch, vocab, logits.data_ptr(), logits.stride(0),
                        None if tokens is None else tokens.data_ptr(), tokens_stride, width,
                        8 if tokens is not None and tokens.dtype == torch.int64 else 4,
                        None if lengths is None else lengths.data_ptr(),
                        None if repetition is None else repetition.data_ptr(),
                        None if presence is None else presence.data_ptr(),
                        None if frequency is None else frequency.data_ptr(),
                        None if bias_ids is None else bias_ids.data_ptr(), None if bias is None else bias.data_ptr(),
                        bias_stride, entries, None if mask is None else mask.data_ptr(), mask_stride, out.data_ptr(),
                        out.stride(0))
    status = _lib.lib().bgtq_adjust_logits(C.byref(p), _stream(on.index))
    if status:
        _lib.check(status)
    return out
