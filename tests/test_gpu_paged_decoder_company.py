"""What a request of the paged decoder answers does not depend on whom it is served with, up to rounding, nor
on whether its weights are a training program's."""
import math

import numpy as np
import pytest

from test_gpu_paged_model import BOUND, SMALL, weights_of
from test_gpu_serving import types

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name,fmt,dtype", [("biased", "int8", "f16"), ("llama", "f16", "f16"), ("biased", "int4", "bf16")])
def test_every_token_of_company_is_one_that_the_request_alone_would_choose(cuda, name, fmt, dtype):
    """Each sequence generated in company is followed alone, through the chunk and every step: its tokens are
    the largest logits there, or within the rounding of two logits (BOUND of the logits' size, twice)."""
    from bgtq import PagedDecoder
    g = SMALL[name]
    dec = PagedDecoder(weights_of(g, dtype), g, pages=32, page_size=16, format=fmt, dtype=types()[dtype])
    prompts = [np.arange(n) * 3 % g.vocab for n in (9, 33, 2, 70)]
    got = dec.generate(prompts, 8)
    for p, row in zip(prompts, got):
        r = dec.open()
        logits = dec.prompt([r], [p])[0]
        for i, t in enumerate(row):
            assert float(logits.max() - logits[t]) <= 2 * BOUND[dtype] * float(logits.norm()) / math.sqrt(g.vocab), (len(p), i)
            logits = dec.step([r], [t])[0]
        dec.close(r)
    assert dec.free_pages == 32


def test_weights_that_require_gradients(cuda):
    """Logits carry no graph, which would leave attention out, and no step's memory is kept for one."""
    import torch
    from bgtq import PagedDecoder
    g = SMALL["llama"]
    w = weights_of(g, "f16")
    answers = []
    for weights in (w, {k: v.clone().requires_grad_() for k, v in w.items()}):
        dec = PagedDecoder(weights, g, pages=8, page_size=16, format="int8", dtype=torch.float16)
        r = dec.open()
        answers.append((dec.prompt([r], [np.arange(20)]), dec.prompt([r], [[4, 5]]), dec.step([r], [6])))
    for a, b in zip(*answers):
        assert not b.requires_grad and torch.equal(a, b)


def test_requests_in_an_array(cuda):
    """Requests may stand in an array or a tensor, like tokens."""
    import torch
    from test_gpu_paged_decoder_failures import decoder
    dec, same = decoder(), decoder()
    held = [d.open() for d in (dec, same) for _ in range(2)][:2]
    for wrap in (np.array, torch.tensor):
        tokens = [np.arange(5), np.arange(9)]
        assert torch.equal(dec.prompt(wrap(held), tokens), same.prompt(held, tokens))
        assert torch.equal(dec.step(wrap(held), [3, 4]), same.step(held, [3, 4]))
