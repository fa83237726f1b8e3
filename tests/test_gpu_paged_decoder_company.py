"""What a request of the paged decoder answers does not depend on whom it is served with, up to rounding."""
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
