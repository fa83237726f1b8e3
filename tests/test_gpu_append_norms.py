"""Head norms of rows whose squares FP32 does not hold, and next to where it does, against the formula in 64 bits
(tolerances: test_gpu_serving_step)."""
import math

import pytest

from test_gpu_serving import randn, types
from test_gpu_serving_step import check_append, table_of

pytestmark = pytest.mark.gpu

SIZES = [1e-44, 3e-39, 1e-30, 1e-20, 1e-13, 8e-13, 1.2e-12, 1e-3, 1.0, 1e10, 1e17, 9e17, 1.1e18, 3e18, 1e19, 1e30, 5e37]


@pytest.mark.parametrize("fmt", ["f16", "bf16", "int8", "int4"])
@pytest.mark.parametrize("source", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-6])
def test_heads_of_any_size(cuda, fmt, source, dim, eps):
    """A head whose root mean square is far above eps' root comes out of one size, whatever its own; below it the result is
    as small as the head over that root, and where FP32 has fewer bits for it the formula's is not asked for."""
    import torch
    from bgtq import PagedCache
    sizes = [s for s in SIZES if s * s > 1e-12 * eps]
    n = 3 * len(sizes)
    cache, other = (PagedCache(2, dim, n // 16 + 1, 16, fmt) for _ in range(2))
    by = torch.tensor(sizes * 3, device="cuda", dtype=torch.float64)[:, None, None]
    q, k = ((randn(s, n, h, dim).double().clamp(-6, 6) * by).float().to(types()[source]) for s, h in ((1, 3), (2, 2)))
    q[-1, 0, 1:] = 0
    k[-1, 0, 1:] = 0
    v = randn(3, n, 2, dim, dtype=source)
    norms = [1 + randn(s, dim, spread=0.3) for s in (4, 5)]
    out, slots, rotary = "f32" if source == "f32" else "bf16", torch.arange(n, device="cuda"), table_of(n, dim)
    # (BF16 has no 1e-44: a head of zeros, which is NaN without eps and zeros with one)
    none = [~x.bool().any(-1) for x in (q, k)]
    got = other.append(q, k, v, slots, rotary, None, *norms, eps=eps, dtype=types()[out], keys=True)
    for x, zeros in zip(got, none):
        assert bool((x[zeros].isnan() if eps == 0 else x[zeros] == 0).all()) and bool(torch.isfinite(x[~zeros]).all())
    some = ~(none[0].any(-1) | none[1].any(-1))
    assert int(some.sum()) >= n - 3
    check_append(cache, q[some], k[some], v[some], slots[some], rotary[some], None, *norms, eps, out)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_heads_without_a_size(cuda, fmt):
    """Zeros are zeros with an eps and NaN without; an infinity or a NaN makes of its own head what the formula makes."""
    import torch
    from bgtq import PagedCache
    cache = PagedCache(1, 64, 1, 16, fmt)
    one, w = torch.zeros(6, 64, device="cuda"), torch.ones(64, device="cuda")
    one[:, :32] = 1.0
    x = randn(1, 6, 1, 64)
    x[0] = 0
    x[1, 0, 5], x[2, 0, 40], x[3, 0, 7] = math.inf, -math.inf, math.nan
    x[4] = 1e30
    for eps in (0.0, 1e-40, 1e-6, 1e38):
        got, keys = cache.append(x, x, x, torch.arange(6, device="cuda"), one, q_norm=w, k_norm=w, eps=eps, keys=True)
        d = x.double()
        want = (d / (d.square().mean(-1, keepdim=True) + torch.tensor(eps).double().item()).sqrt()).float()
        for have in (got, keys):
            fin = torch.isfinite(want)
            # (rotating by nothing adds zero times the head's other half, which makes a NaN of an infinity's pair)
            pair = torch.isfinite(want.roll(32, -1))
            assert torch.equal(have.isnan() & pair, want.isnan() & pair) and not bool(torch.isfinite(have)[~fin].any())
            assert torch.allclose(have[fin & pair], want[fin & pair], rtol=1e-5, atol=1e-40), eps
