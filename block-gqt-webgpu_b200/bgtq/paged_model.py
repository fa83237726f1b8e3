"""The decoder families of `bgtq.model` over a paged cache: requests that come, grow and go one by one.

`model.Decoder` advances equal sequences together over the Block-GTQ key stores
(src/model/decoder.ts:15-83); this one serves requests of different lengths over 16-, 8- or
4-bit pages.  A call of `prompt` runs the new tokens of any number of requests as one packed
batch: their rows are quantised into the pages (`PagedCache.write`), the rows of earlier calls
are read back (`PagedCache.read`) in front of them, and `prompt_attention` runs over both.  A
call of `step` runs one new token of each request: its row is written, then every head reads
its request's pages (`PagedCache.attend`).  Geometry, weights, RoPE and norms are the ones of
`model` (src/model/kernels.wgsl:11-54); the projections are plain GEMMs.
"""
from __future__ import annotations

import contextlib

import numpy as np
import torch
import torch.nn.functional as F

from .model import ModelGeometry
from .serving import PagedCache, prompt_attention, _refuse


_RECORDED = 16  # steps that a decoder keeps recorded, by requests and table width, both rounded up


def _places(requests: int) -> int:
    """The places of the recorded step that so many requests take: powers of two up to 16, then multiples of 16."""
    return 1 << (requests - 1).bit_length() if requests <= 16 else min(-(-requests // 16) * 16, max(requests, 65535))


class PagedDecoder:
    """pages: pages of page_size tokens that all requests share (one pool a layer, one table
    for all).  format: "f16" / "bf16" (dtype's own), "int8" or "int4" pages.  dtype: float16 or
    bfloat16, the type of GEMMs and attention; the residual stream is FP32."""

    def __init__(self, weights, geometry: ModelGeometry, pages: int, page_size: int = 64, format: str = "int8",
                 dtype=torch.bfloat16, device: int = 0):
        if dtype not in (torch.float16, torch.bfloat16):
            _refuse("Paged decoder: dtype must be float16 or bfloat16")
        if format in ("f16", "bf16") and (format == "f16") != (dtype == torch.float16):
            _refuse("Paged decoder: 16-bit pages must be of dtype")
        g = self.g = geometry
        self.dtype, self.page_size = dtype, int(page_size)
        self.dev = torch.device("cuda", device)
        self.caches = [PagedCache(g.kv_heads, g.head_dim, pages, page_size, format, device) for _ in range(g.layers)]
        for c in self.caches[1:]:  # the layers follow each other on one stream: one workspace serves all
            c._workspace = self.caches[0]._workspace
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
        self._free += self._request(request)[0][::-1]
        del self._held[request]

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
        """Pages for counts[i] more tokens of requests[i], all of them or a refusal: what each holds now and
        its length before.  A body that fails has written no rows to count on, so it leaves lengths and
        pages as they were."""
        requests = requests.tolist() if hasattr(requests, "tolist") else list(requests)
        if not requests or len(set(requests)) < len(requests):
            _refuse("Paged decoder: requests must be one or more, each once")
        held = [self._request(r) for r in requests]
        need = [-(-(h[1] + n) // self.page_size) - len(h[0]) for h, n in zip(held, counts)]
        if sum(need) > len(self._free):
            _refuse(f"Paged decoder: {sum(need)} pages wanted, {len(self._free)} free")
        before = [h[1] for h in held]
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
            raise

    def _slots(self, pages, first: int, upto: int):
        t = np.arange(first, upto)
        return np.asarray(pages, np.int64)[t // self.page_size] * self.page_size + t % self.page_size

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

    def _prompt(self, flat, counts, held, before):
        ends = np.cumsum(counts)
        slots = self._to(np.concatenate([self._slots(h[0], b, h[1]) for h, b in zip(held, before)]), torch.int64)
        positions = self._to(np.concatenate([np.arange(b, h[1]) for h, b in zip(held, before)]), torch.float32)
        starts = self._to(np.concatenate([[0], ends]), torch.int32)
        earlier = None
        if any(before):
            # keys of a request: the rows of earlier calls from the pages, then this call's own as they are
            # (a negative slot reads nothing: those rows are filled in)
            key_ends = np.cumsum([h[1] for h in held])
            rows = [np.concatenate([self._slots(h[0], 0, b), np.full(h[1] - b, -1)]) for h, b in zip(held, before)]
            new = [np.arange(e - n, e) for e, n in zip(key_ends, counts)]
            earlier = (self._to(np.concatenate(rows), torch.int64), self._to(np.concatenate(new), torch.int64),
                       self._to(np.concatenate([[0], key_ends]), torch.int32))

        def attention(cache, q, k, v):
            cache.write(k, v, slots)
            q, k, v = q.to(self.dtype), k.to(self.dtype), v.to(self.dtype)
            if earlier is None:
                return prompt_attention(q, k, v, starts)
            all_k, all_v = cache.read(earlier[0], self.dtype)
            all_k[earlier[1]], all_v[earlier[1]] = k, v
            return prompt_attention(q, all_k, all_v, starts, key_starts=earlier[2])

        return self._forward(self._to(flat, torch.int64), positions, attention, self._to(ends - 1, torch.int64))

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
        table = np.zeros((places, width), np.int32)
        for row, h in zip(table, held):
            row[:len(h[0])] = h[0]
        inputs[-1].copy_(torch.as_tensor(table))
        graph.replay()
        return logits[:n].clone()

    def _record(self, batch: int, width: int):
        """A step of batch requests over tables of width pages: graph, inputs, logits."""
        tokens, positions, slots, lengths, table = inputs = (
            self._to(np.zeros(batch), torch.int64), self._to(np.zeros(batch), torch.float32),
            self._to(np.full(batch, -1), torch.int64), self._to(np.zeros(batch), torch.int32),
            self._to(np.zeros((batch, width)), torch.int32))

        def attention(cache, q, k, v):
            cache.write(k, v, slots)
            return cache.attend(q.to(self.dtype), table, lengths)

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

    def generate(self, prompts, count: int):
        """Greedy: count tokens after each of prompts (sequences of tokens), as an int64 array
        [prompts, count].  Its requests are closed before it returns."""
        requests = [self.open() for _ in prompts]
        try:
            out = [self.prompt(requests, prompts).argmax(-1)]
            while len(out) < count:
                out.append(self.step(requests, out[-1]).argmax(-1))
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

    def _rope(self, x, cos, sin):
        half = self.g.head_dim // 2
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    def _forward(self, tokens, positions, attention, last):
        g = self.g
        qw, kvw = g.q_heads * g.head_dim, g.kv_heads * g.head_dim
        angle = positions[:, None, None] * self.inv_freq
        cos, sin = angle.cos(), angle.sin()
        h = self.emb[tokens].float()
        for lw, cache in zip(self.layers, self.caches):
            qkv = F.linear(self._norm(h, lw["ln1"]), lw["qkv"], lw["qkv_b"]).float()
            q = self._rope(qkv[:, :qw].unflatten(1, (g.q_heads, g.head_dim)), cos, sin)
            k = self._rope(qkv[:, qw:qw + kvw].unflatten(1, (g.kv_heads, g.head_dim)), cos, sin)
            v = qkv[:, qw + kvw:].unflatten(1, (g.kv_heads, g.head_dim))
            h = h + F.linear(attention(cache, q, k, v).flatten(1), lw["o"]).float()
            gate, up = F.linear(self._norm(h, lw["ln2"]), lw["gate_up"]).chunk(2, -1)
            h = h + F.linear(F.silu(gate) * up, lw["down"]).float()
        if last is not None:
            h = h[last]
        return F.linear(self._norm(h, self.final_norm), self.emb).float()
