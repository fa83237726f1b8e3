"""Chunks over 8-bit pages lose no bit of a value, however many rows a request has.

Tolerances (u = 2^-11, FP16's unit roundoff): a value is its code times its scale, exactly; the product of a probability and its
scale, or the scale's mantissa, is rounded to FP16 once, the output once; exponentials and FP32 sums 3e-5 of A = sum p_t |v_t|;
products are held to 2^-34 of the row's largest probability x value scale, times a code of at most 2^7: 2^-25 (A + B + 1), B = sum |v_t| over the row's sum, holds them.  Where all
seen tokens have the same probability it is a power of two of the row, and its product with a scale's eight bits is exact: what
remains is u |o| + 3e-5 A + 2^-25 (A + B + 1)."""
import pytest

from test_gpu_serving import U, attention64, paged, randn, starts_of, types
from test_gpu_serving_step import NEW, seen_of

pytestmark = pytest.mark.gpu


def within(cache, out, q, new, table, lengths, dtype, products):
    import math
    import torch
    group, ps, at = q.shape[1] // cache.kv_heads, cache.page_size, 0
    for b, (n, length) in enumerate(zip(new, lengths.tolist())):
        rows, at = slice(at, at + n), at + n
        if not n:
            continue
        t = torch.arange(length, device="cuda")
        k, v = cache.read(table[b].long()[t // ps] * ps + t % ps, dtype=torch.float32)
        for h in sorted({0, q.shape[1] // 2, q.shape[1] - 1}):
            want, _, mag, small = attention64(q[rows, h], k[:, h // group], v[:, h // group], seen_of(n, length, None, 0), 1 / math.sqrt(cache.dim))
            off = (out[rows, h].double() - want).abs()
            tol = U[dtype] * want.abs() + (products + 3e-5) * mag + 2.0 ** -25 * (small + mag + 1)
            assert bool((off <= tol).all()), (b, h, float((off / tol).max()))


@pytest.mark.parametrize("new", sorted(NEW))
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim,hq,hk,page", [(64, 9, 3, 16), (128, 8, 2, 64), (64, 14, 2, 128), (128, 32, 4, 32)])
def test_products_are_rounded_once(cuda, new, dtype, dim, hq, hk, page):
    n, lengths = NEW[new]
    cache, table, lens = paged(10, lengths, hk, dim, page, "int8")
    q = randn(11, sum(n), hq, dim, dtype=dtype)
    out = cache.attend_chunk(q, starts_of(n), table, lens)
    within(cache, out, q, n, table, lens, dtype, U["f16"])


@pytest.mark.parametrize("n", [1, 2, 40, 300])
@pytest.mark.parametrize("dim,hq", [(64, 2), (64, 14), (128, 4), (128, 16)])
@pytest.mark.parametrize("spread", [1.0, 8.0, 3000.0, 1e6])
def test_values_that_cancel(cuda, n, dim, hq, spread):
    """Rows of three kinds one after the other, the third of which takes back most of the first two, of scales as far apart as
    `spread`; no row of queries prefers one."""
    import torch
    from bgtq import PagedCache
    length = 400
    cache = PagedCache(2, dim, 25, 16, "int8")
    base = randn(5, 2, 2, dim)
    kinds = torch.cat([base * torch.tensor([1.0, spread], device="cuda")[:, None, None], randn(6, 1, 2, dim)])
    kinds[2] -= kinds[0] + kinds[1]
    t = torch.arange(length, device="cuda")
    cache.write(randn(7, length, 2, dim), kinds[t % 3], t)
    table, lens = torch.arange(25, dtype=torch.int32, device="cuda")[None], torch.tensor([length], dtype=torch.int32, device="cuda")
    q = torch.zeros((n, hq, dim), dtype=torch.float16, device="cuda")
    # (in FP16 the outputs of spread 1e6 are infinite: those are asked for in BF16, whose own rounding is coarser)
    dtype = "bf16" if spread > 1e4 else "f16"
    q = q.to(types()[dtype])
    out = cache.attend_chunk(q, starts_of([n]), table, lens)
    within(cache, out, q, [n], table, lens, dtype, 0.0)
