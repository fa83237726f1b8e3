"""The serving operators at the ends of their types' ranges, against plain formulas in 64 bits: what a
row does not see, or sees with next to no weight, leaves it as it was, however large it is.

A key that a row does not see has probability zero, and one whose logit is 200 under the row's largest
has less than 2^-288: times the largest BF16 value, 2^128, that is under 2^-160, which no sum of values
of size 1 shows.  Those rows have to come out bit by bit.
"""
import math

import pytest

from bgtq import device_status
from test_gpu_serving import U, attention64, randn, starts_of, types

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


# What FP16 holds of a probability at least: half its last place, 2^-25, over what it is multiplied by
LEAST = {"prompt": 2.0 ** -25 / 2 ** 7, "token": 2.0 ** -25 / 2 ** 12}


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kind", ["prompt", "token"])
@pytest.mark.parametrize("n", [900, 8193])                 # prompts: an item as a whole, and one in parts
@pytest.mark.parametrize("gap", [14.0, 16.8, 17.4, 18.5])  # nats: 2^-20 to 2^-27
def test_many_small_probabilities_beside_a_large_one(cuda, kind, dim, n, gap):
    """One key has nearly all of the weight and a value of zero; what the others, each of them small,
    add up to is the answer.  Tolerance: the roundings of an output and its probabilities, 3e-5 of them
    for FP32, and what FP16 drops of a small probability."""
    import torch
    from bgtq import PagedCache, prompt_attention
    q = torch.zeros((1, 2, dim), dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0
    k = torch.zeros((n, 1, dim), dtype=torch.float16, device="cuda")
    k[5, 0, 0] = gap
    k[:, 0, 1:] = 0.0
    v = (64 + 16 * randn(3, n, 1, dim)).half()     # outputs above 2^-14, where FP16 rounds by 2^-11
    v[5] = 0
    if kind == "prompt":
        out, lse = prompt_attention(q, k, v, starts_of([1]), starts_of([n]), scale=1.0, lse=True)
    else:
        pages = (n + 15) // 16
        cache = PagedCache(1, dim, pages, 16, "f16")
        cache.write(k, v, torch.arange(n, device="cuda"))
        out, lse = cache.attend(q, torch.arange(pages, dtype=torch.int32, device="cuda")[None],
                                torch.tensor([n], dtype=torch.int32, device="cuda"), scale=1.0, lse=True)
    for h in range(2):
        want, want_lse, mag, small = attention64(q[:, h], k[:, 0], v[:, 0], torch.ones((1, n), dtype=torch.bool, device="cuda"), 1.0)
        tol = U["f16"] * want.abs() + (U["f16"] + 3e-5) * mag + LEAST[kind] * small
        assert bool(((out[:, h].double() - want).abs() <= tol).all()), float(((out[:, h].double() - want).abs() / tol).max())
        assert float((lse[:, h].double() - want_lse).abs().max()) <= 3e-5


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("nq,nk", [(300, 300), (40, 4000)])    # items as a whole, and one in parts
@pytest.mark.parametrize("early,late,both", [(math.nan, math.inf, math.nan), (-math.inf, math.inf, math.nan),
                                             (math.inf, -math.inf, math.nan), (math.inf, math.inf, math.inf)])
def test_prompt_infinities_and_nan_of_far_and_near_keys_add_up(cuda, dtype, dim, nq, nk, early, late, both):
    """One value is in a tile that every row sees, one where only the later rows see it."""
    import torch
    from bgtq import prompt_attention
    q, k, v = (randn(s, n, 2, dim, dtype=dtype) for s, n in ((1, nq), (2, nk), (3, nk)))
    st, ks = starts_of([nq]), starts_of([nk])
    want = prompt_attention(q, k, v, st, ks)
    v[3, :, 5], v[nk - 10, :, 5] = early, late
    out = prompt_attention(q, k, v, st, ks)
    rest = [i for i in range(dim) if i != 5]
    assert torch.equal(out[..., rest], want[..., rest])
    row = torch.arange(nq, device="cuda") + nk - nq          # the last key that each row sees
    expect = torch.where(row >= nk - 10, both, torch.where(row >= 3, early, 0.0))[:, None].expand(nq, 2)
    got = torch.where(row[:, None] >= 3, out[..., 5].float(), 0.0)
    assert torch.equal(got.nan_to_num(nan=7.0, posinf=8.0, neginf=9.0), expect.nan_to_num(nan=7.0, posinf=8.0, neginf=9.0))


def pages_of(k, v, fmt):
    """A cache that holds rows k, v [tokens, heads, dim], its table, and the rows as they stand there."""
    import torch
    from bgtq import PagedCache
    n = k.shape[0]
    pages = (n + 15) // 16
    cache = PagedCache(k.shape[1], k.shape[2], pages, 16, fmt)
    slots = torch.arange(n, device="cuda")
    cache.write(k, v, slots)
    table, length = torch.arange(pages, dtype=torch.int32, device="cuda")[None], torch.tensor([n], dtype=torch.int32, device="cuda")
    return cache, table, length, cache.read(slots, torch.float32)


def check_quantised(cache, q, table, length, rows, dtype, scale):
    """Tolerance: the roundings of an output and of its probabilities, 3e-5 of them for FP32, and for every
    token FP16's half of a last place, 2^-25 / 2^10 of the head's largest contribution.  A contribution is a
    probability x a scale in 8 bits, whose codes are up to the row's largest / scale; in 4 bits a probability x a
    power of two of at least half the token's largest scale, with codes x scales up to 16 of it: with the row's
    largest, 7 scales or more, that is 2^-35 and 16 x 2^-35 / 7 of probability x row at most, 2^-33 for both."""
    import torch
    out, lse = cache.attend(q, table, length, scale=scale, lse=True)
    k, v = (x[:, 0].double() for x in rows)
    s = (q[0].double() @ k.T) * scale
    p = torch.softmax(s, -1)
    want = p @ v
    least = k.shape[0] * 2.0 ** -33 * (p * v.abs().amax(-1)).amax(-1, keepdim=True)
    tol = U[dtype] * want.abs() + (U[dtype] + 3e-5) * (p @ v.abs()) + least
    off = (out[0].double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    assert float((lse[0].double() - torch.logsumexp(s, -1)).abs().max()) <= 3e-5 * max(1.0, float(s.abs().max()) / 64)
    return out


@pytest.mark.parametrize("fmt,dtype", [("int8", "f16"), ("int8", "bf16"), ("int4", "f16"), ("int4", "bf16")])
@pytest.mark.parametrize("dim,heads", [(64, 2), (64, 14), (128, 3), (128, 16)])
@pytest.mark.parametrize("big", [1e5, 1e12, 1e30, 3e38])
@pytest.mark.parametrize("where", ["first", "middle", "last", "half"])
def test_token_large_values_without_weight(cuda, fmt, dtype, dim, heads, big, where):
    """Rows of large values that no head gives weight to leave the others as they are."""
    import torch
    n = 700
    far = torch.zeros(n, dtype=torch.bool, device="cuda")
    if where == "half":
        far[1::2] = True
    else:
        far[{"first": 0, "middle": 333, "last": n - 1}[where]] = True
    k, v = randn(1, n, 1, dim), randn(2, n, 1, dim) + 0.5
    k[:, 0, 0] = 0
    k[far] = 0
    k[far, 0, 0] = -2400.0                     # logits of -300: weights below 2^-420
    v[far] = big
    q = randn(3, 1, heads, dim, dtype=dtype)
    q[..., 0] = 1.0
    cache, table, length, rows = pages_of(k, v, fmt)
    check_quantised(cache, q, table, length, rows, dtype, 1.0 / 8)


@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("big", [1e6, 1e25])
def test_token_heads_that_see_values_of_different_size(cuda, fmt, dim, big):
    """Of the heads of a KV head some give all their weight to large values, some to small ones."""
    import torch
    n = 600
    k, v = randn(1, n, 1, dim, spread=0.5), randn(2, n, 1, dim) + 0.5
    k[:, 0, 0] = torch.where(torch.arange(n, device="cuda") % 7 == 3, 30.0, -30.0)
    v[k[:, 0, 0] > 0] *= big
    q = randn(3, 1, 10, dim, dtype="bf16")
    q[0, :, 0] = torch.where(torch.arange(10, device="cuda") % 3 == 0, 16.0, -16.0).bfloat16()
    cache, table, length, rows = pages_of(k, v, fmt)
    check_quantised(cache, q, table, length, rows, "bf16", 1.0 / 8)


@pytest.mark.parametrize("fmt", ["int8", "int4"])
def test_token_climbing_logits_after_a_large_value(cuda, fmt):
    """The large value leads at first; by the end of a slow climb its weight is 2^-115."""
    import torch
    n = 3000
    k = torch.zeros((n, 1, 64), device="cuda")
    k[:, 0, 0] = torch.linspace(-40, 40, n, device="cuda")
    v = randn(2, n, 1, 64) + 0.5
    v[0] = 1e20
    q = torch.zeros((1, 4, 64), device="cuda", dtype=torch.bfloat16)
    q[..., 0] = 1.0
    cache, table, length, rows = pages_of(k, v, fmt)
    check_quantised(cache, q, table, length, rows, "bf16", 1.0)


@pytest.mark.parametrize("scale", [1e-50, 1e-46, 1e-44])
def test_scales_below_fp32(cuda, scale):
    """A scale of next to nothing gives equal weights, not the default scale."""
    import torch
    from bgtq import prompt_attention
    n = 50
    q, k, v = (randn(s, n, 1, 64, dtype="f16") for s in (1, 2, 3))
    want = v[:, 0].double().mean(0)
    tol = U["f16"] * want.abs() + (U["f16"] + 3e-5) * v[:, 0].double().abs().mean(0)
    out = prompt_attention(q, k, v, starts_of([n]), causal=False, scale=scale)
    assert bool(((out[:, 0].double() - want).abs() <= tol).all())
    cache, table, length, _ = pages_of(k, v, "f16")
    out = cache.attend(q[:1], table, length, scale=scale)
    assert bool(((out[0, 0].double() - want).abs() <= tol).all())


@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("dim,heads", [(64, 3), (128, 10)])
@pytest.mark.parametrize("q_size,k_size", [(1.0, 1e36), (1e36, 1.0), (1e-30, 1e32), (1e32, 1e-30)])
def test_token_large_queries_and_keys(cuda, fmt, dim, heads, q_size, k_size):
    """Logits that FP32 holds, from queries or keys near the ends of BF16."""
    k, v = randn(1, 300, 1, dim) * k_size, randn(2, 300, 1, dim) + 0.5
    q = (randn(3, 1, heads, dim) * q_size).bfloat16()
    cache, table, length, rows = pages_of(k, v, fmt)
    check_quantised(cache, q, table, length, rows, "bf16", 1.0 / 8)
