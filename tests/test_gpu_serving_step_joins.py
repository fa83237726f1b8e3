"""Chunks of one long request, which many CTAs take in parts: every number of rows in a block, row tile and item, and
infinities and NaN in one part only."""
import math

import pytest

from test_gpu_serving_step import FORMATS, check_chunk, paged, randn, seen_of, starts_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,dtype", FORMATS)
@pytest.mark.parametrize("dim,hq,hk", [(64, 16, 2), (64, 7, 1), (128, 16, 2), (128, 5, 1)])
@pytest.mark.parametrize("n", [5, 9, 13, 17, 33, 70, 150])
def test_rows_of_one_long_request(cuda, fmt, dtype, dim, hq, hk, n):
    cache, table, lens = paged(31, [4001], hk, dim, 64, fmt)
    check_chunk(cache, randn(3, n, hq, dim, dtype=dtype), [n], table, lens, dtype)


@pytest.mark.parametrize("fmt,dtype", FORMATS)
@pytest.mark.parametrize("lengths", [[257, 300, 1000], [256, 255, 64, 1025], [2000, 1024, 100]])
@pytest.mark.parametrize("n", [5, 8, 9])
def test_short_and_long_requests_of_few_rows(cuda, fmt, dtype, lengths, n):
    for dim, hq, hk in ((128, 32, 8), (64, 56, 8)):
        cache, table, lens = paged(32, lengths, hk, dim, 32, fmt)
        check_chunk(cache, randn(4, n * len(lengths), hq, dim, dtype=dtype), [n] * len(lengths), table, lens, dtype)


@pytest.mark.parametrize("fmt,dtype", FORMATS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [5, 60])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("window,sinks", [(None, 0), (2000, 70)])
def test_special_values_in_one_part(cuda, fmt, dtype, dim, n, bad, window, sinks):
    import torch
    length, last = 4001, dim - 1
    cache, table, lens = paged(33, [length], 2, dim, 64, fmt)
    q = randn(3, n, 16, dim, dtype=dtype)
    want, want_lse = check_chunk(cache, q, [n], table, lens, dtype, window, sinks)
    t = torch.arange(length, device="cuda")
    slots = table[0].long()[t // 64] * 64 + t % 64
    plain = fmt in ("f16", "bf16")
    cut = slice(last, last + 1) if plain else slice(-1, None)
    dims = cut if plain else slice(dim - 32 if fmt == "int4" else 0, dim)
    rest = torch.ones(dim, dtype=torch.bool, device="cuda")
    rest[dims] = False
    seen = seen_of(n, length, window, sinks)
    pool = cache.v if plain else cache.v_scales
    for at in (length - 1, length - 3, length - 2000, length - 2002, 69, 40):
        s = slots[at]
        old = pool[s // 64, 1, s % 64, cut].clone()
        pool[s // 64, 1, s % 64, cut] = bad
        out, lse = cache.attend_chunk(q, starts_of([n]), table, lens, window=window, sinks=sinks, lse=True)
        pool[s // 64, 1, s % 64, cut] = old
        blind = ~seen[:, at]
        assert torch.equal(lse, want_lse), at
        assert torch.equal(out[blind], want[blind]) and torch.equal(out[:, :8], want[:, :8]), at
        assert torch.equal(out[..., rest], want[..., rest]), at
        hit = out[~blind][:, 8:, dims].float()
        # (a scale of infinity makes +-infinity of codes and NaN of zeros, and either of their sum)
        wrong = ~(hit.isnan() | (hit == bad)) if plain else ~hit.isnan() if math.isnan(bad) else hit.isfinite()
        assert not bool(wrong.any()), at
    again, _ = check_chunk(cache, q, [n], table, lens, dtype, window, sinks)
    assert torch.equal(again, want)
