"""The serving operators at the ends of their types' ranges, against plain formulas in 64 bits: what a
row does not see, or sees with next to no weight, leaves it as it was, however large it is.

A key that a row does not see has probability zero, and one whose logit is 200 under the row's largest
has less than 2^-288: times the largest BF16 value, 2^128, that is under 2^-160, which no sum of values
of size 1 shows.  Those rows have to come out bit by bit.
"""
import math

import pytest

from bgtq import device_status
from test_gpu_serving import randn, starts_of, types

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("big", [1e30, -3e38])
def test_prompt_large_values_do_not_reach_rows_before_them(cuda, dim, big):
    """A large finite value at every place of a stretch of 16 keys leaves the earlier rows bit by bit."""
    import torch
    from bgtq import prompt_attention
    n, st = 200, starts_of([200])
    q, k, v = (randn(s, n, 2, dim, dtype="bf16") for s in (1, 2, 3))
    want, want_lse = prompt_attention(q, k, v, st, lse=True)
    for at in range(120, 136):
        v2 = v.clone()
        v2[at] = big
        out, lse = prompt_attention(q, k, v2, st, lse=True)
        assert torch.equal(out[:at], want[:at]) and torch.equal(lse, want_lse), at


@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_large_values_of_keys_without_weight(cuda, dim):
    """Every row sees keys whose weight is next to nothing: their values, however large, add nothing."""
    import torch
    from bgtq import prompt_attention
    n, m = 9, 333
    q, k, v = randn(1, n, 2, dim, dtype="bf16"), randn(2, m, 2, dim, dtype="bf16"), randn(3, m, 2, dim, dtype="bf16")
    q[..., 0], k[..., 0] = 1.0, 0.0
    far = torch.arange(m, device="cuda") % 3 == 1
    k[far] = 0.0
    k[far, :, 0] = -4096.0          # a logit of -256 or less at either head dim's scale
    st, ks = starts_of([n]), starts_of([m])
    want, want_lse = prompt_attention(q, k, v, st, ks, causal=False, lse=True)
    v[far] = 3e38
    out, lse = prompt_attention(q, k, v, st, ks, causal=False, lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("nq,nk", [(150, 150), (3, 5000)])     # an item as a whole, and one in parts
def test_prompt_rows_whose_logits_are_all_minus_infinity(cuda, dtype, dim, nq, nk):
    """They have no weights: zeros, and minus infinity for the log sum, like rows that see nothing."""
    import torch
    from bgtq import prompt_attention
    q, k, v = (randn(s, n, 2, dim, dtype=dtype) for s, n in ((1, nq), (2, nk), (3, nk)))
    q[..., 0], k[..., 0] = 1.0, 0.0
    st, ks = starts_of([nq]), starts_of([nk])
    want, want_lse = prompt_attention(q, k, v, st, ks, lse=True)
    k[:, 1, 0] = -math.inf                                     # every key of the second head
    out, lse = prompt_attention(q, k, v, st, ks, lse=True)
    assert torch.equal(out[:, 0], want[:, 0]) and torch.equal(lse[:, 0], want_lse[:, 0])
    assert not out[:, 1].any() and bool((lse[:, 1] == -math.inf).all())
    assert device_status(0) == 0
