"""The paged decoder over windows, in verified drafts and with what is put on logits, against the model's formulas in
64 bits over the rows that the pages hold (tolerances: test_gpu_paged_model)."""
import math

import numpy as np
import pytest

from bgtq import _lib
from test_gpu_paged_model import BOUND, SMALL, Plain, off, weights_of
from test_gpu_serving import types

pytestmark = pytest.mark.gpu


class Windowed(Plain):
    """One request whose tokens see a window and the first few; rows are taken from the pages where the decoder
    still holds them, and kept here."""

    def __init__(self, weights, dec, request, bound):
        super().__init__(weights, dec, request, bound)
        self.kept = {}

    def rows(self, layer, name, new):
        import torch
        n = new.shape[1]
        pages = self.dec._held[self.request][0]
        upto = self.length + n
        first = upto - n
        assert min(pages[first // self.dec.page_size:]) >= 0
        held, pages[:] = list(pages), [max(p, 0) for p in pages]
        try:
            got, half = self.held(layer, name, upto)
        finally:
            pages[:] = held
        far = (got[:, self.length:] - new).abs()
        rms = new.square().mean(-1, keepdim=True).sqrt()
        assert bool((far <= 1.01 * half[:, self.length:] + 4 * self.bound * rms).all()), (layer, name)
        old = self.kept.get((layer, name))
        now = got[:, self.length:] if old is None else torch.cat([old[:, :self.length], got[:, self.length:]], 1)
        self.kept[layer, name] = now
        return now

    def forward(self, tokens):
        """Logits of every token."""
        import torch
        g, w, d, n, start = self.g, self.w, self.g.head_dim, len(tokens), self.length
        inv = g.rope_theta ** (-torch.arange(d // 2, device="cuda").double() / (d // 2))
        angle = (start + torch.arange(n, device="cuda").double())[:, None] * inv
        cos, sin = angle.cos(), angle.sin()

        def rope(x):
            a, b = x[..., :d // 2], x[..., d // 2:]
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

        def linear(x, name):
            y = x @ w[name + ".weight"].T
            return y + w[name + ".bias"] if name + ".bias" in w else y

        t, p = torch.arange(start + n, device="cuda")[None], start + torch.arange(n, device="cuda")[:, None]
        seen = t <= p
        if self.dec.window is not None:
            seen = seen & ((t > p - self.dec.window) | (t < self.dec.sinks))
        h = w["model.embed_tokens.weight"][torch.as_tensor(tokens, device="cuda")]
        for layer in range(g.layers):
            pre = f"model.layers.{layer}."
            x = self.norm(h, pre + "input_layernorm.weight")
            q, k, v = (linear(x, pre + f"self_attn.{c}_proj").unflatten(1, (-1, d)).transpose(0, 1) for c in "qkv")
            keys, values = (self.rows(layer, c, y).repeat_interleave(g.gqa, 0) for c, y in (("k", rope(k)), ("v", v)))
            s = torch.where(seen, rope(q) @ keys.transpose(1, 2) / math.sqrt(d), -math.inf)
            h = h + linear((s.softmax(-1) @ values).transpose(0, 1).flatten(1), pre + "self_attn.o_proj")
            x = self.norm(h, pre + "post_attention_layernorm.weight")
            gate = linear(x, pre + "mlp.gate_proj")
            h = h + linear(gate * torch.sigmoid(gate) * linear(x, pre + "mlp.up_proj"), pre + "mlp.down_proj")
        self.length += n
        return self.norm(h, "model.norm.weight") @ w["model.embed_tokens.weight"].T


@pytest.mark.parametrize("name,fmt,dtype", [("llama", "f16", "f16"), ("llama", "int8", "bf16"), ("biased", "bf16", "bf16"), ("biased", "int4", "f16")])
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 5), (33, 0)])
def test_prompts_drafts_and_steps_match_the_formulas(cuda, name, fmt, dtype, window, sinks):
    from bgtq import PagedDecoder
    g, bound = SMALL[name], BOUND[dtype]
    w = weights_of(g, dtype)
    dec = PagedDecoder(w, g, pages=30, page_size=16, format=fmt, dtype=types()[dtype], window=window, sinks=sinks)
    rng = np.random.default_rng(5)
    a, b = dec.open(), dec.open()
    plain = {r: Windowed(w, dec, r, bound) for r in (a, b)}

    def same(got, lengths, call):
        tokens = [rng.integers(0, g.vocab, n) for n in lengths.values()]
        rows = got(list(lengths), tokens if call != "step" else [t[0] for t in tokens])
        at = 0
        for i, (r, t) in enumerate(zip(lengths, tokens)):
            want = plain[r].forward(t)
            have = rows[at:at + len(t)] if call == "verify" else rows[i:i + 1]
            at += len(t)
            assert off(have, want if call == "verify" else want[-1:]) < bound, (call, r, len(t))

    if window is not None or fmt in ("f16", "bf16"):
        same(dec.prompt, {a: 100, b: 1}, "prompt")
        same(dec.prompt, {b: 70}, "prompt")
    else:      # (a prompt's chunk over 8- and 4-bit pages sees its own rows as they are: drafts do not)
        same(dec.verify, {a: 100, b: 71}, "verify")
    same(dec.step, {b: 1, a: 1}, "step")
    same(dec.verify, {a: 5, b: 3}, "verify")
    for r, back in ((a, 2), (b, 3)):
        dec.rewind(r, dec.length(r) - back)
        plain[r].length -= back
    same(dec.step, {a: 1, b: 1}, "step")
    same(dec.verify, {b: 1}, "verify")
    for _ in range(20):
        same(dec.step, {a: 1}, "step")
    for r in (a, b):
        dec.close(r)
    assert dec.free_pages == 30


def test_drafts_answer_what_steps_answer(cuda):
    """Over stored rows both do the same arithmetic up to rounding."""
    from bgtq import PagedDecoder
    g = SMALL["biased"]
    w = weights_of(g, "f16")
    one, two = (PagedDecoder(w, g, pages=20, page_size=16, format="int8", dtype=types()["f16"]) for _ in range(2))
    tokens = np.random.default_rng(1).integers(0, g.vocab, 60)
    rows = []
    for d in (one, two):
        r = d.open()
        d.prompt([r], [tokens[:40]])
        rows.append([d.step([r], [t])[0] for t in tokens[40:48]] if d is one else list(d.verify([r], [tokens[40:48]])))
    for x, y in zip(*rows):
        assert off(x, y.double()) < BOUND["f16"]


def test_a_request_grows_past_the_pool(cuda):
    """With a window, pages that no later token sees go back: 8 pages of 16 hold a request of any length."""
    from bgtq import PagedDecoder
    g = SMALL["llama"]
    w = weights_of(g, "f16")
    dec = PagedDecoder(w, g, pages=8, page_size=16, format="f16", dtype=types()["f16"], window=50, sinks=4)
    r = dec.open()
    plain = Windowed(w, dec, r, BOUND["f16"])
    rng = np.random.default_rng(3)
    for i in range(12):
        t = rng.integers(0, g.vocab, 30)
        assert off(dec.prompt([r], [t])[0], plain.forward(t)[-1]) < BOUND["f16"], i
        assert off(dec.step([r], t[:1])[0], plain.forward(t[:1])[-1]) < BOUND["f16"], i
    assert dec.length(r) == 12 * 31 and dec._held[r][0][0] >= 0 and -1 in dec._held[r][0]
    with pytest.raises(_lib.RangeError, match="given back"):
        dec.rewind(r, 200)
    held = 8 - dec.free_pages
    dec.close(r)
    assert held <= 6 and dec.free_pages == 8 and sorted(dec._free) == list(range(8))


def test_generate_with_penalties_biases_and_a_mask(cuda):
    import torch
    from bgtq import PagedDecoder
    g = SMALL["biased"]
    dec = PagedDecoder(weights_of(g, "f16"), g, pages=16, page_size=16, format="int8", dtype=types()["f16"])
    prompts = [np.arange(9), torch.arange(33) % g.vocab, [5, 5]]
    # only a few tokens allowed, each of them once
    allowed = np.zeros((1, (g.vocab + 31) // 32), np.uint32)
    some = [3, 40, 64, 95, 200, 406]
    for t in some:
        allowed[0, t // 32] |= np.uint32(1 << t % 32)
    mask = torch.as_tensor(allowed.view(np.int32), device="cuda")
    got = dec.generate(prompts, 6, presence=1e6, mask=mask)
    assert all(set(row) <= set(some) for row in got)
    assert sorted(got[2]) == some
    # tokens of a prompt are penalised too: 3 is in the first two
    assert got[0][:5].tolist().count(3) == 0
    # a large bias decides, for all rows or for one
    ids, bias = torch.tensor([[17]], dtype=torch.int32, device="cuda"), torch.tensor([[1e5]], device="cuda")
    assert (dec.generate(prompts, 3, bias_ids=ids, bias=bias) == 17).all()
    assert (dec.generate(prompts, 3) == dec.generate(prompts, 3, repetition=1.0)).all()
    assert dec.generate(prompts[:1], 0, presence=1.0).shape == (1, 0) and dec.free_pages == 16


def test_generate_refuses_before_it_opens_requests(cuda):
    import torch
    from bgtq import PagedDecoder
    g = SMALL["llama"]
    dec = PagedDecoder(weights_of(g, "f16"), g, pages=4, page_size=16, dtype=torch.float16)
    for kw in (dict(repetition=0.0), dict(presence=math.nan), dict(frequency=torch.zeros(3, device="cuda")), dict(out=1), dict(lengths=1),
               dict(tokens=1), dict(temperature=1.0), dict(bias=torch.zeros(1, 1, device="cuda")), dict(mask=torch.zeros(1, 1, device="cuda"))):
        with pytest.raises(_lib.RangeError):
            dec.generate([[1, 2]], 2, **kw)
        assert not dec._held and dec.free_pages == 4
    assert (dec.generate([np.array([[1, 2, 3]])], 3, frequency=0.0) == dec.generate([[1, 2, 3]], 3)).all()


def test_refusals(cuda):
    import torch
    from bgtq import PagedDecoder
    g = SMALL["llama"]
    w = weights_of(g, "f16")
    for kw in (dict(window=0), dict(window=2**31), dict(window=5, sinks=-1)):
        with pytest.raises(_lib.RangeError, match="window"):
            PagedDecoder(w, g, pages=2, page_size=16, dtype=torch.float16, **kw)
    dec = PagedDecoder(w, g, pages=3, page_size=16, dtype=torch.float16)
    r = dec.open()
    dec.verify([r], [list(range(30))])
    for call, message in [(lambda: dec.verify([r], [[1], [2]]), "one or more tokens"), (lambda: dec.verify([r], [[]]), "one or more tokens"),
                          (lambda: dec.verify([r], [[g.vocab]]), "vocabulary"), (lambda: dec.verify([r], [list(range(19))]), "pages wanted"),
                          (lambda: dec.verify([], []), "one or more"), (lambda: dec.rewind(r, 31), "0 to 30"), (lambda: dec.rewind(r, -1), "0 to 30"),
                          (lambda: dec.rewind(r + 1, 0), "no such request")]:
        with pytest.raises(_lib.RangeError, match=message):
            call()
    assert dec.length(r) == 30 and dec.free_pages == 1
    dec.rewind(r, 16)
    assert dec.length(r) == 16 and dec.free_pages == 2
    dec.rewind(r, 0)
    assert dec.length(r) == 0 and dec.free_pages == 3
    dec.step([r], [4])
    assert dec.length(r) == 1


def test_a_draft_that_fails_changes_nothing(cuda, monkeypatch):
    import torch
    from test_gpu_paged_decoder_failures import decoder, failing, state
    dec, same = decoder(), decoder()
    answers = []
    for d in (same, dec):
        held = [d.open(), d.open()]
        d.prompt(held, [np.arange(17), np.arange(30)])
        if d is dec:
            was = state(d, held)
            for method in ("append", "attend_chunk"):
                with monkeypatch.context() as m:
                    failing(d, m, 1, method, 1)
                    with pytest.raises(MemoryError):
                        d.verify(held, [[1, 2, 3], [4] * 20])
                assert state(d, held) == was
        answers.append((d.verify(held, [[1, 2, 3], [4] * 20]), d.step(held, [5, 6])))
    for a, b in zip(*answers):
        assert torch.equal(a, b)
