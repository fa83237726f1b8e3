"""The paged decoder on the GPU: chunks of prompts, single tokens, pages that come and go, against
the model's formulas in 64 bits over the rows that the pages hold.

A code is a step function of its row, and a step that falls the other way goes through softmax into
every later layer, so the plain form takes the rows of earlier tokens from the pages (by its own
decoding), after it has seen that each is the row it computes itself to half a step.

Tolerances, from the arithmetic: with activations of unit roundoff u (2^-11 FP16, 2^-8 BF16), each
layer rounds about ten times along the residual path (two norms, projections, Q, K, V, attention,
the gated product, two sums), each independent and of relative size u / sqrt(3): three layers and
the last norm and product come to sqrt(32 / 3) u = 3.3 u, 0.0016 and 0.013; the bounds, relative
2-norm, leave room for what softmax and the gates add: 0.02 FP16, 0.05 BF16.  A stored value is half
a step of its group, and four times that bound of the row's root mean square, from the plain one.
"""
import math

import numpy as np
import pytest

from bgtq import _lib
from bgtq.model import ModelGeometry, weight_names
from test_gpu_serving import codes_of, types

pytestmark = pytest.mark.gpu
SMALL = {"llama": ModelGeometry("smollm2", 3, 192, 320, 3, 1, 1e4, 1e-5, 331, False),
         "biased": ModelGeometry("qwen2", 3, 256, 448, 4, 2, 1e6, 1e-6, 407, True)}
BOUND = {"f16": 0.02, "bf16": 0.05}


def weights_of(g, dtype, seed=3):
    """Larger than a checkpoint's start, so that attention decides and layers add to what is there."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = {}
    for name, shape in weight_names(g).items():
        if name.endswith("norm.weight"):
            out[name] = (1 + 0.1 * torch.randn(shape, generator=gen, device="cuda")).to(types()[dtype])
        else:
            scale = 1.5 / math.sqrt(shape[-1]) if "proj" in name and len(shape) == 2 else 0.5
            out[name] = (scale * torch.randn(shape, generator=gen, device="cuda")).to(types()[dtype])
    return out


class Plain:
    """One request of a decoder by the formulas, in 64 bits."""

    def __init__(self, weights, dec, request, bound):
        self.w, self.g, self.dec, self.request, self.bound = {k: v.double() for k, v in weights.items()}, dec.g, dec, request, bound
        self.length = 0

    def held(self, layer, name, upto):
        """What the pages hold of the first tokens: [heads, upto, dim]; half a step of each value."""
        import torch
        cache, page = self.dec.caches[layer], self.dec.page_size
        t = torch.arange(upto, device="cuda")
        pages = torch.tensor(self.dec._held[self.request][0], device="cuda")[t // page]
        x, scales = getattr(cache, name).double(), getattr(cache, name + "_scales")
        half = torch.zeros_like(x)
        if scales is not None:
            codes = codes_of(cache, name)
            s = scales.double().repeat_interleave(codes.shape[-1] // scales.shape[-1], -1)
            x, half = codes * s, 0.5 * s
        return tuple(y[pages, :, t % page].transpose(0, 1) for y in (x, half))

    def rows(self, layer, name, new):
        """The rows of all tokens as they are held; the new ones are seen to be those of `new`."""
        n = new.shape[1]
        got, half = self.held(layer, name, self.length + n)
        far = (got[:, self.length:] - new).abs()
        rms = new.square().mean(-1, keepdim=True).sqrt()
        assert bool((far <= 1.01 * half[:, self.length:] + 4 * self.bound * rms).all()), (layer, name)
        return got

    def norm(self, x, w):
        import torch
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + self.g.rms_eps) * self.w[w]

    def forward(self, tokens, single, lost=None):
        import torch
        g, w = self.g, self.w
        d, n = g.head_dim, len(tokens)
        start = self.length
        inv = g.rope_theta ** (-torch.arange(d // 2, device="cuda").double() / (d // 2))
        angle = (start + torch.arange(n, device="cuda").double())[:, None] * inv
        cos, sin = angle.cos(), angle.sin()

        def rope(x):
            a, b = x[..., :d // 2], x[..., d // 2:]
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

        def linear(x, name):
            y = x @ w[name + ".weight"].T
            return y + w[name + ".bias"] if name + ".bias" in w else y

        h = w["model.embed_tokens.weight"][torch.as_tensor(tokens, device="cuda")]
        for layer in range(g.layers):
            p = f"model.layers.{layer}."
            x = self.norm(h, p + "input_layernorm.weight")
            q, k, v = (linear(x, p + f"self_attn.{c}_proj").unflatten(1, (-1, d)).transpose(0, 1) for c in "qkv")
            q, k = rope(q), rope(k)
            kept = [self.rows(layer, c, x) for c, x in (("k", k), ("v", v))]
            keys, values = kept if single else (torch.cat([a[:, :start], b], 1) for a, b in zip(kept, (k, v)))
            if lost is not None:
                values = values.clone()
                values[:, lost] = 0
            keys, values = (t.repeat_interleave(g.gqa, 0) for t in (keys, values))
            s = q @ keys.transpose(1, 2) / math.sqrt(d)
            seen = torch.arange(start + n, device="cuda")[None] <= start + torch.arange(n, device="cuda")[:, None]
            s = torch.where(seen, s, -math.inf)
            h = h + linear((s.softmax(-1) @ values).transpose(0, 1).flatten(1), p + "self_attn.o_proj")
            x = self.norm(h, p + "post_attention_layernorm.weight")
            gate = linear(x, p + "mlp.gate_proj")
            h = h + linear(gate * torch.sigmoid(gate) * linear(x, p + "mlp.up_proj"), p + "mlp.down_proj")
        self.length += n
        return self.norm(h[-1], "model.norm.weight") @ w["model.embed_tokens.weight"].T


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("name,fmt,dtype", [("llama", "f16", "f16"), ("llama", "int8", "bf16"), ("biased", "bf16", "bf16"),
                                            ("biased", "int8", "f16"), ("biased", "int4", "f16"), ("llama", "int4", "bf16")])
def test_chunks_and_steps_match_the_formulas(cuda, name, fmt, dtype):
    from bgtq import PagedDecoder
    g = SMALL[name]
    w = weights_of(g, dtype)
    bound = BOUND[dtype]
    dec = PagedDecoder(w, g, pages=24, page_size=16, format=fmt, dtype=types()[dtype])
    rng = np.random.default_rng(5)
    plain = {}

    def prompt(lengths):
        tokens = {r: rng.integers(0, g.vocab, n) for r, n in lengths.items()}
        got = dec.prompt(list(tokens), list(tokens.values()))
        for row, (r, t) in zip(got, tokens.items()):
            assert off(row, plain[r].forward(t, False)) < bound, (r, len(t))

    def step(requests):
        tokens = rng.integers(0, g.vocab, len(requests))
        got = dec.step(requests, tokens)
        for row, r, t in zip(got, requests, tokens):
            assert off(row, plain[r].forward([t], True)) < bound, r

    def new():
        r = dec.open()
        plain[r] = Plain(w, dec, r, bound)
        return r

    a, b, c = new(), new(), new()
    prompt({a: 37, b: 1, c: 16})
    for _ in range(3):
        step([c, a, b])
    prompt({b: 70, a: 5})            # a later chunk over rows read back, another order, not all requests
    step([a, b, c])
    dec.close(a)
    e = new()                        # takes pages that a has left
    prompt({e: 20, c: 13})
    step([e, c])
    assert [dec.length(r) for r in (b, c, e)] == [75, 34, 21] and dec.free_pages == 24 - 5 - 3 - 2


def test_the_bound_sees_one_missing_row(cuda):
    """The plain form that has lost one stored row is outside the tolerance."""
    from bgtq import PagedDecoder
    g = SMALL["llama"]
    w = weights_of(g, "f16")
    dec = PagedDecoder(w, g, pages=4, page_size=16, format="int8", dtype=types()["f16"])
    tokens = np.random.default_rng(1).integers(0, g.vocab, 20)
    r = dec.open()
    dec.prompt([r], [tokens])
    got = dec.step([r], [7])[0]
    plain = Plain(w, dec, r, BOUND["f16"])
    plain.length = 20
    right = plain.forward([7], True)
    plain.length = 20
    assert off(got, right) < BOUND["f16"]
    with pytest.raises(AssertionError):  # by the logits, or by the rows of the layers behind it
        assert off(got, plain.forward([7], True, lost=3)) < BOUND["f16"]


def test_generate_is_the_same_alone_and_in_company(cuda):
    from bgtq import PagedDecoder
    g = SMALL["biased"]
    dec = PagedDecoder(weights_of(g, "f16"), g, pages=16, page_size=16, format="int8", dtype=types()["f16"])
    prompts = [np.arange(n) % g.vocab for n in (9, 33, 2)]
    got = dec.generate(prompts, 6)
    assert got.shape == (3, 6) and dec.free_pages == 16
    assert dec.generate(prompts[:1], 0).shape == (1, 0)
    # the first token of each is the argmax of its own prompt's logits, unless two are within rounding
    for p, row in zip(prompts, got):
        r = dec.open()
        logits = dec.prompt([r], [p])[0]
        dec.close(r)
        assert float(logits.max() - logits[row[0]]) <= 2 * BOUND["f16"] * float(logits.norm()) / math.sqrt(g.vocab)


def test_refusals_change_nothing(cuda):
    import torch
    from bgtq import PagedDecoder
    g = SMALL["llama"]
    w = weights_of(g, "f16")
    for kw, message in [(dict(dtype=torch.float32), "dtype"), (dict(dtype=torch.float16, format="bf16"), "16-bit pages"),
                        (dict(format="int3"), "format"), (dict(page_size=24), "page size")]:
        with pytest.raises(_lib.RangeError, match=message):
            PagedDecoder(w, g, pages=2, **{"page_size": 16, **kw})
    dec = PagedDecoder(w, g, pages=2, page_size=16, format="int8", dtype=torch.float16)
    r = dec.open()
    dec.prompt([r], [list(range(30))])
    for call, message in [(lambda: dec.prompt([r], [[1, 2, 3]]), "1 pages wanted, 0 free"),
                          (lambda: dec.prompt([r, r], [[1], [2]]), "each once"), (lambda: dec.prompt([], []), "one or more"),
                          (lambda: dec.prompt([r], [[]]), "one or more tokens"), (lambda: dec.step([r], [1, 2]), "one token"),
                          (lambda: dec.prompt([r], [[g.vocab]]), "vocabulary"), (lambda: dec.step([r], [-1]), "vocabulary"),
                          (lambda: dec.step([r + 1], [1]), "no such request"), (lambda: dec.close(r + 1), "no such request")]:
        with pytest.raises(_lib.RangeError, match=message):
            call()
    assert dec.length(r) == 30 and dec.free_pages == 0
    dec.step([r], [1])
    dec.close(r)
    assert dec.free_pages == 2


def test_steps_of_changing_batches_and_widths(cuda):
    """Recorded steps of other batches and table widths, more of them than are kept, on another stream
    too, follow the requests."""
    import torch
    from bgtq import PagedDecoder, paged_model
    g = SMALL["llama"]
    w = weights_of(g, "f16")
    dec = PagedDecoder(w, g, pages=64, page_size=16, format="int8", dtype=types()["f16"])
    rng = np.random.default_rng(2)
    held = [dec.open() for _ in range(18)]
    plain = {r: Plain(w, dec, r, BOUND["f16"]) for r in held}
    lengths = [250] + [3 + i for i in range(17)]     # the first grows past 16 pages, to tables of 32
    tokens = [rng.integers(0, g.vocab, n) for n in lengths]
    for row, r, t in zip(dec.prompt(held, tokens), held, tokens):
        assert off(row, plain[r].forward(t, False)) < BOUND["f16"], r
    side = torch.cuda.Stream()
    for batch in [*range(1, 19), 1, 2, 1]:
        some = held[:batch]
        t = rng.integers(0, g.vocab, batch)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side if batch % 2 else torch.cuda.current_stream()):
            got = dec.step(some, t)
        torch.cuda.synchronize()
        for row, r, x in zip(got, some, t):
            assert off(row, plain[r].forward([x], True)) < BOUND["f16"], (batch, r)
    assert len(dec._steps) <= paged_model._RECORDED
