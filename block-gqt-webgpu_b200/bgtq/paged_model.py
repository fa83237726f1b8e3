"""The decoder families of `bgtq.model` over a paged cache: requests that come, grow and go one by one.

`model.Decoder` advances equal sequences together over the Block-GTQ key stores
(src/model/decoder.ts:15-83); this one serves requests of different lengths over 16-, 8- or
4-bit pages.  A call of `prompt` runs the new tokens of any number of requests as one packed
batch: their rows are quantised into the pages (`PagedCache.write`), the rows of earlier calls
are read back (`PagedCache.read`) in front of them, and `prompt_attention` runs over both.  A
call of `step` runs one new token of each request: it is rotated into the pages
(`PagedCache.append`), then every head reads its request's pages (`PagedCache.attend`).  Over
16-bit pages, which hold rows as they are, and with a window a prompt's chunk does the same
(`PagedCache.attend_chunk`), and so does a call of `verify`, which answers for every one of a
few drafted tokens what `step` would have answered one after the other.  `generate` chooses
after penalties, biases and masks (`adjust_logits`).  Geometry, weights, RoPE and norms are the
ones of `model` (src/model/kernels.wgsl:11-54); the projections are plain GEMMs.
"""
from __future__ import annotations

import contextlib

import numpy as np
import torch
import torch.nn.functional as F

from .model import ModelGeometry
from .serving import PagedCache, adjust_logits, prompt_attention, _Workspaces, _per_row, _refuse


_PENALTIES = ("repetition", "presence", "frequency")
_RECORDED = 16  # steps that a decoder keeps recorded, by requests and table width, both rounded up


def _places(requests: int) -> int:
    """The places of the recorded step that so many requests take: powers of two up to 16, then multiples of 16."""
    return 1 << (requests - 1).bit_length() if requests <= 16 else min(-(-requests // 16) * 16, max(requests, 65535))


class PagedDecoder:
    """pages: pages of page_size tokens that all requests share (one pool a layer, one table
    for all).  format: "f16" / "bf16" (dtype's own), "int8" or "int4" pages.  dtype: float16 or
    bfloat16, the type of GEMMs and attention; the residual stream is FP32.  window, sinks: a
    token sees the last `window` tokens, itself among them, and the first `sinks` of its request
    (None: all); pages that no later token sees are given back when their request grows, so that a
    request may become longer than the pool."""

    def __init__(self, weights, geometry: ModelGeometry, pages: int, page_size: int = 64, format: str = "int8",
                 dtype=torch.bfloat16, device: int = 0, window: int | None = None, sinks: int = 0):
        if dtype not in (torch.float16, torch.bfloat16):
            _refuse("Paged decoder: dtype must be float16 or bfloat16")
        if format in ("f16", "bf16") and (format == "f16") != (dtype == torch.float16):
            _refuse("Paged decoder: 16-bit pages must be of dtype")
        if window is not None and not 1 <= window < 2**31 or not 0 <= sinks < 2**31:
            _refuse("Paged decoder: window must be positive and sinks nonnegative, both below 2^31")
        self.window, self.sinks = window, int(sinks)
        g = self.g = geometry
        self.dtype, self.page_size = dtype, int(page_size)
        self.dev = torch.device("cuda", device)
        self.caches = [PagedCache(g.kv_heads, g.head_dim, pages, page_size, format, device) for _ in range(g.layers)]
        # The layers follow each other on one stream: one workspace serves all.  It is the decoder's own, for chunks too:
        # torch hands the recording stream's handle to others as well, and recorded steps are replayed on any.
        work = _Workspaces()
        for c in self.caches:
            c._workspace, c._chunk_work = self.caches[0]._workspace, work
        w = {k: v.detach().to(self.dev, dtype) for k, v in weights.items()}  # (attention has no gradient)
        self.emb, self.final_norm = w["model.embed_tokens.weight"], w["model.norm.weight"].float()
        self.layers = []
        for layer in range(g.layers):
            a, m = f"model.layers.{layer}.self_attn.", f"model.layers.{layer}.mlp."
            names = [a + n for n in ("q_proj", "k_proj", "v_proj")]
            self.layers.append(dict(
                ln1=w[f"model.layers.{layer}.input_layernorm.weight"].float(),
                ln2=w[f"model.layers.{layer}.post_attention_layernorm.weight"].float(),
                qkv=torch.cat([w[n + ".weight"] for n in names]).contiguous(),
                qkv_b=torch.cat([w[n + ".bias"] for n in names]).contiguous() if g.qkv_bias else None,
                o=w[a + "o_proj.weight"],
                gate_up=torch.cat([w[m + "gate_proj.weight"], w[m + "up_proj.weight"]]).contiguous(),
                down=w[m + "down_proj.weight"]))
        pairs = g.head_dim // 2
        # theta to a power in FP32, as src/model/kernels.wgsl:52 takes it
        self.inv_freq = torch.pow(torch.tensor(float(g.rope_theta), dtype=torch.float32),
                                  -torch.arange(pairs, dtype=torch.float32) / pairs).to(self.dev)
        self._free = list(range(pages))[::-1]
        self._held = {}        # request: [its pages in order, its tokens]
        self._next = 0
        self._steps, self._side, self._pool = {}, torch.cuda.Stream(self.dev), torch.cuda.graph_pool_handle()

    # ---- requests and pages ----
    def open(self) -> int:
        """A new, empty request."""
        self._next += 1
        self._held[self._next] = [[], 0]
        return self._next

    def close(self, request: int) -> None:
        """Ends a request; its pages are free for others."""
        self._free += [p for p in self._request(request)[0][::-1] if p >= 0]
        del self._held[request]

    def rewind(self, request: int, length: int) -> None:
        """Takes back the last tokens of a request, so that `length` are left: what a draft was
        verified to be wrong in.  Pages that are left over are free for others."""
        pages, have = held = self._request(request)
        if not 0 <= length <= have:
            _refuse(f"Paged decoder: a length of 0 to {have} can be left")
        keep = -(-length // self.page_size)
        if length and -1 in pages[self._first(length) // self.page_size:keep]:
            _refuse("Paged decoder: pages of tokens that would be seen again have been given back")
        self._free += [p for p in pages[keep:][::-1] if p >= 0]
        held[0], held[1] = pages[:keep], length

    def _first(self, length: int) -> int:
        """The first token that the next one sees, but for sinks."""
        return 0 if self.window is None else max(0, length - self.window + 1)

    def _unseen(self, held):
        """Places of the pages of tokens that no later one sees, in order (those given back before lie in front of them)."""
        pages, length = held
        first, end = -(-self.sinks // self.page_size), min(self._first(length) // self.page_size, len(pages))
        at = end
        while at > first and pages[at - 1] >= 0:
            at -= 1
        return range(at, end)

    def length(self, request: int) -> int:
        """Tokens of a request whose rows the pages hold."""
        return self._request(request)[1]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _request(self, request):
        if request not in self._held:
            _refuse("Paged decoder: no such request")
        return self._held[request]

    @contextlib.contextmanager
    def _grown(self, requests, counts):
        """Pages for counts[i] more tokens of requests[i], all of them or a refusal, which changes nothing: what
        each holds now and its length before.  Pages that their later tokens do not see are given back (-1 stands
        for them from then on).  A body that fails has written no rows to count on, so it leaves lengths and pages
        as they were; but of the pages given back, those that the call took again have lost their rows, and stay
        free.  They are the last that a call takes."""
        requests = requests.tolist() if hasattr(requests, "tolist") else list(requests)
        if not requests or len(set(requests)) < len(requests):
            _refuse("Paged decoder: requests must be one or more, each once")
        held = [self._request(r) for r in requests]
        back = [(h[0], i, h[0][i]) for h in held for i in self._unseen(h)] if self.window is not None else []
        need = [-(-(h[1] + n) // self.page_size) - len(h[0]) for h, n in zip(held, counts)]
        if sum(need) > len(self._free) + len(back):
            _refuse(f"Paged decoder: {sum(need)} pages wanted, {len(self._free) + len(back)} free")
        before = [h[1] for h in held]
        for pages, i, _ in back:
            pages[i] = -1
        kept = back[max(0, sum(need) - len(self._free)):]
        self._free[:0] = [page for _, _, page in back[::-1]]
        for h, n, more in zip(held, counts, need):
            h[0] += [self._free.pop() for _ in range(more)]
            h[1] += n
        try:
            yield held, before
        except BaseException:
            for h, start, more in reversed(list(zip(held, before, need))):
                self._free += h[0][len(h[0]) - more:][::-1]
                del h[0][len(h[0]) - more:]
                h[1] = start
            for pages, i, page in kept:
                pages[i] = page
            del self._free[:len(kept)]
            raise

    def _slots(self, pages, first: int, upto: int):
        t = np.arange(first, upto)
        return np.asarray(pages, np.int64)[t // self.page_size] * self.page_size + t % self.page_size

    def _table(self, held, places: int, width: int):
        table = np.zeros((places, width), np.int32)  # (a page that was given back is not followed)
        for row, h in zip(table, held):
            row[:len(h[0])] = np.maximum(h[0], 0)
        return table

    def _to(self, array, dtype):
        return torch.as_tensor(np.asarray(array), dtype=dtype).to(self.dev, non_blocking=True)

    # ---- the model ----
    def prompt(self, requests, tokens):
        """The next tokens[i] (a sequence of one or more) of each requests[i], its first or a
        later chunk: logits [requests, vocab] (FP32) of each one's last token."""
        tokens = [np.asarray(t.cpu() if torch.is_tensor(t) else t, np.int64).reshape(-1) for t in tokens]
        if len(tokens) != len(requests) or any(not len(t) for t in tokens):
            _refuse("Paged decoder: one or more tokens for every request")
        flat = self._vocabulary(np.concatenate(tokens)) if tokens else None
        counts = [len(t) for t in tokens]
        with self._grown(requests, counts) as (held, before):
            return self._prompt(flat, counts, held, before)

    def verify(self, requests, tokens):
        """The next tokens[i] (one or more) of each requests[i], drafted by whatever means: logits
        [all tokens, vocab] (FP32) of every one of them, one request's after the other's, as `step`
        would answer them one at a time.  `rewind` takes back the ones that were wrong."""
        tokens = [np.asarray(t.cpu() if torch.is_tensor(t) else t, np.int64).reshape(-1) for t in tokens]
        if len(tokens) != len(requests) or any(not len(t) for t in tokens):
            _refuse("Paged decoder: one or more tokens for every request")
        flat = self._vocabulary(np.concatenate(tokens)) if tokens else None
        counts = [len(t) for t in tokens]
        with self._grown(requests, counts) as (held, before):
            return self._chunk(flat, counts, held, before, None)

    def _chunk(self, flat, counts, held, before, last):
        """New tokens through the pages."""
        slots, positions, starts = self._rows(counts, held, before)
        table = self._to(self._table(held, len(held), max(len(h[0]) for h in held)), torch.int32)
        lengths = self._to([h[1] for h in held], torch.int32)

        def attention(cache, q, k, v, rotary):
            q = cache.append(q, k, v, slots, rotary)
            return cache.attend_chunk(q, starts, table, lengths, window=self.window, sinks=self.sinks)

        return self._forward(self._to(flat, torch.int64), positions, attention, last)

    def _rows(self, counts, held, before):
        """Slots and positions of new rows, and where each request's begin."""
        return (self._to(np.concatenate([self._slots(h[0], b, h[1]) for h, b in zip(held, before)]), torch.int64),
                self._to(np.concatenate([np.arange(b, h[1]) for h, b in zip(held, before)]), torch.float32),
                self._to(np.concatenate([[0], np.cumsum(counts)]), torch.int32))

    def _prompt(self, flat, counts, held, before):
        ends = np.cumsum(counts)
        last = self._to(ends - 1, torch.int64)
        if self.window is not None or self.caches[0].k_scales is None:
            return self._chunk(flat, counts, held, before, last)
        # 8- and 4-bit pages: a chunk sees its own rows as they are, and the rows of earlier calls as they are stored
        slots, positions, starts = self._rows(counts, held, before)
        earlier = None
        if any(before):
            # keys of a request: the rows of earlier calls from the pages, then this call's own as they are
            # (a negative slot reads nothing: those rows are filled in)
            key_ends = np.cumsum([h[1] for h in held])
            rows = [np.concatenate([self._slots(h[0], 0, b), np.full(h[1] - b, -1)]) for h, b in zip(held, before)]
            new = [np.arange(e - n, e) for e, n in zip(key_ends, counts)]
            earlier = (self._to(np.concatenate(rows), torch.int64), self._to(np.concatenate(new), torch.int64),
                       self._to(np.concatenate([[0], key_ends]), torch.int32))

        def attention(cache, q, k, v, rotary):
            q, k, v = self._rope(q.float(), rotary), self._rope(k.float(), rotary), v.float()
            cache.write(k, v, slots)
            q, k, v = q.to(self.dtype), k.to(self.dtype), v.to(self.dtype)
            if earlier is None:
                return prompt_attention(q, k, v, starts)
            all_k, all_v = cache.read(earlier[0], self.dtype)
            all_k[earlier[1]], all_v[earlier[1]] = k, v
            return prompt_attention(q, all_k, all_v, starts, key_starts=earlier[2])

        return self._forward(self._to(flat, torch.int64), positions, attention, last)

    def step(self, requests, tokens):
        """One token of each request: logits [requests, vocab] (FP32).  Replays a CUDA graph that is
        recorded at the first step of about so many requests and pages; of the places that are
        left over, nothing is written or read.  The graphs used last are kept."""
        tokens = np.asarray(tokens.cpu() if torch.is_tensor(tokens) else tokens, np.int64).reshape(-1)
        if len(tokens) != len(requests):
            _refuse("Paged decoder: one token for every request")
        self._vocabulary(tokens)
        with self._grown(requests, [1] * len(tokens)) as (held, before):
            return self._step(tokens, held, before)

    def _step(self, tokens, held, before):
        n, places = len(held), _places(len(held))
        width = 1 << max(4, (max(len(h[0]) for h in held) - 1).bit_length())
        key = places, width
        graph, inputs, logits = self._steps[key] = self._steps.pop(key, None) or self._record(places, width)
        slots = [h[0][b // self.page_size] * self.page_size + b % self.page_size for h, b in zip(held, before)]
        for buffer, values, rest in zip(inputs, (tokens, before, slots, [h[1] for h in held]), (0, 0, -1, 0)):
            row = np.full(places, rest, np.float32 if buffer.is_floating_point() else np.int64)
            row[:n] = values
            buffer.copy_(torch.as_tensor(row).to(buffer.dtype))
        inputs[-1].copy_(torch.as_tensor(self._table(held, places, width)))
        graph.replay()
        return logits[:n].clone()

    def _record(self, batch: int, width: int):
        """A step of batch requests over tables of width pages: graph, inputs, logits."""
        tokens, positions, slots, lengths, table = inputs = (
            self._to(np.zeros(batch), torch.int64), self._to(np.zeros(batch), torch.float32),
            self._to(np.full(batch, -1), torch.int64), self._to(np.zeros(batch), torch.int32),
            self._to(np.zeros((batch, width)), torch.int32))

        def attention(cache, q, k, v, rotary):
            q = cache.append(q, k, v, slots, rotary)
            if self.window is None:
                return cache.attend(q, table, lengths)
            return cache.attend(q, table, lengths, window=self.window, sinks=self.sinks)

        # once beside the recording, for what is set up at first calls: no row is written, none is read
        self._side.wait_stream(torch.cuda.current_stream(self.dev))
        with torch.cuda.stream(self._side):
            self._forward(tokens, positions, attention, None)
        torch.cuda.current_stream(self.dev).wait_stream(self._side)
        graph = torch.cuda.CUDAGraph()
        # one pool for all: a replay's logits are copied before the next one, whichever it is
        with torch.cuda.graph(graph, pool=self._pool, stream=self._side):
            logits = self._forward(tokens, positions, attention, None)
        while len(self._steps) >= _RECORDED:
            del self._steps[next(iter(self._steps))]
        return graph, inputs, logits

    def generate(self, prompts, count: int, **choice):
        """Greedy: count tokens after each of prompts (sequences of tokens), as an int64 array
        [prompts, count].  choice: what is put on the logits before each token is chosen, as
        `adjust_logits` takes it (repetition, presence, frequency, bias_ids, bias, mask; the history is
        a request's prompt and what it was answered).  Its requests are closed before it returns."""
        penalties = [name for name in _PENALTIES if choice.get(name) is not None]
        if set(choice) - {*_PENALTIES, "bias_ids", "bias", "mask"}:
            _refuse(f"Paged decoder: choice is of {', '.join(_PENALTIES)}, bias_ids, bias and mask")
        history = None
        if penalties:
            texts = [np.asarray(p.cpu() if torch.is_tensor(p) else p, np.int64).reshape(-1) for p in prompts]
            lengths = [len(p) for p in texts]
            row = np.full((len(texts), max(lengths, default=0) + max(count, 0)), -1, np.int64)
            for r, p in zip(row, texts):
                r[:len(p)] = p
            history = self._to(row, torch.int64)
            # (numbers are filled in once, not for every token)
            choice.update({name: _per_row(choice[name], len(texts), history.device, name) for name in penalties})
            at = torch.as_tensor(lengths, device=self.dev)[:, None]
        requests = [self.open() for _ in prompts]

        def chosen(logits):
            if choice:
                adjust_logits(logits, history, out=logits, **choice)
            token = logits.argmax(-1)
            if history is not None and count > 0:  # (places past the answers hold -1: they are left out)
                history.scatter_(1, at + len(out), token[:, None])
            return token

        out = []
        try:
            out.append(chosen(self.prompt(requests, prompts)))
            while len(out) < count:
                out.append(chosen(self.step(requests, out[-1])))
            return torch.stack(out[:count], 1).cpu().numpy() if count > 0 else np.zeros((len(prompts), 0), np.int64)
        finally:
            for r in requests:
                self.close(r)

    def _vocabulary(self, tokens):
        if len(tokens) and (tokens.min() < 0 or tokens.max() >= self.g.vocab):
            _refuse("Paged decoder: token outside the vocabulary")
        return tokens

    def _norm(self, x, w):
        return F.rms_norm(x, (self.g.hidden,), w, self.g.rms_eps).to(self.dtype)

    def _rope(self, x, rotary):
        cos, sin = rotary[:, None].chunk(2, -1)
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    def _forward(self, tokens, positions, attention, last):
        g = self.g
        qw, kvw = g.q_heads * g.head_dim, g.kv_heads * g.head_dim
        angle = positions[:, None] * self.inv_freq
        rotary = torch.cat([angle.cos(), angle.sin()], -1)
        h = self.emb[tokens].float()
        for lw, cache in zip(self.layers, self.caches):
            qkv = F.linear(self._norm(h, lw["ln1"]), lw["qkv"], lw["qkv_b"])
            q, k, v = (x.unflatten(1, (-1, g.head_dim)) for x in qkv.split((qw, kvw, kvw), 1))
            h = h + F.linear(attention(cache, q, k, v, rotary).flatten(1), lw["o"]).float()
            gate, up = F.linear(self._norm(h, lw["ln2"]), lw["gate_up"]).chunk(2, -1)
            h = h + F.linear(F.silu(gate) * up, lw["down"]).float()
        if last is not None:
            h = h[last]
        return F.linear(self._norm(h, self.final_norm), self.emb).float()
