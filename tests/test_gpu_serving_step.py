"""The operators of a serving step on the GPU - new tokens rotated into the pages, chunks of them over
the pages, what is put on logits - against plain formulas in 64 bits.

Tolerances, from the arithmetic (u = unit roundoff, 2^-24 FP32, 2^-11 FP16, 2^-8 BF16):
append   a rotated value is three FP32 roundings of a c and b s, of at most |a| + |b|; a norm's factor
         is the root of a mean of at most 128 squares, summed 16 in a row and then by pairs (20 roundings),
         a root, a quotient and two products: 24 u in all.  32 u (|a| + |b|) holds both, and the result is
         rounded once.  Rows that become codes are 64-bit and rounded to FP32 once: their codes are those
         of the 64-bit row, but for ties.
chunk    what test_gpu_serving says: u |o| + (u + 3e-5) A, A = sum p_t |v_t|, for the roundings of probabilities
         and outputs; over 8- and 4-bit pages probabilities are rounded to FP16, whatever the queries' type, and values
         in 8 bits too (2 u + u^2 of FP16 in place of u), and products are held to 2^-34 of the row's largest
         probability x value scale, times a code of at most 2^4 of it (4 bits) or 2^7 (8 bits): 2^-25 (A + 1) covers it
         for rows of one size.  The log sum is FP32 throughout: 3e-5 absolute.
logits   every step is one FP32 rounding of what it gives: 5 u of the sum of the steps' magnitudes.
"""
import math
import subprocess
import sys

import numpy as np
import pytest

from bgtq import _lib, device_status
from conftest import ROOT
from test_gpu_serving import FORMATS, U, attention64, codes_of, paged, randn, starts_of, types

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24


# ---- new tokens into the pages ------------------------------------------------------------------

def table_of(rows, dim, theta=1e4):
    import torch
    angle = torch.arange(rows, device="cuda").double()[:, None] * theta ** (-torch.arange(dim // 2, device="cuda") / (dim / 2))
    return torch.cat([angle.cos(), angle.sin()], -1).float()


def turned64(x, row, norm, eps):
    """Heads [tokens, heads, dim] normed and rotated, in 64 bits, and what their FP32 roundings are relative to."""
    import torch
    x = x.double()
    if norm is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * norm.double()
    h = x.shape[-1] // 2
    c, s = row.double()[:, None, :h], row.double()[:, None, h:]
    a, b = x[..., :h], x[..., h:]
    mag = (a.abs() + b.abs()).repeat(1, 1, 2)
    return torch.cat([a * c - b * s, b * c + a * s], -1), mag


def stored_by_product(x, fmt):
    """(x / scale, codes, scales) of FP32 rows by the documented formula: a scale is max|x| times FP32 1 / top, an FP32
    product rounded to BF16 (where that is a tie within an FP32 rounding, max|x| / top has another)."""
    import torch
    top, group = (127.0, x.shape[-1]) if fmt == "int8" else (7.0, 32)
    y = x.reshape(*x.shape[:-1], -1, group)
    s = (y.abs().amax(-1, keepdim=True) * torch.tensor(1 / top, device="cuda", dtype=torch.float32)).bfloat16()
    ratio = torch.where(s > 0, y.double() / s.double(), 0.0)
    return ratio.reshape(x.shape), ratio.round().clamp(-top, top).reshape(x.shape), s.squeeze(-1)


def near(got, want, mag, dtype):
    import torch
    u = U.get(dtype, U32)
    assert torch.isfinite(got).all()
    tol = u * want.abs() + 32 * U32 * mag * (1 + u) + (2.0 ** -25 if dtype == "f16" else 0)
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


def check_append(cache, q, k, v, slots, rotary, positions, q_norm, k_norm, eps, dtype):
    """One call, all of its results against the formula."""
    import torch
    dim, page, H = cache.dim, cache.page_size, cache.kv_heads
    before = [getattr(cache, n).clone() for n in ("k", "v")]
    got, keys = cache.append(q, k, v, slots, rotary, positions, q_norm=q_norm, k_norm=k_norm, eps=eps, dtype=types()[dtype],
                             keys=True)
    row = rotary[:len(slots)] if positions is None else rotary[positions]
    want, mag = turned64(q, row, q_norm, eps)
    near(got, want, mag, dtype)
    want, mag = turned64(k, row, k_norm, eps)
    near(keys, want, mag, dtype)
    live = slots >= 0
    pg, at = slots[live] // page, slots[live] % page
    free = torch.ones(cache.pages * page, dtype=torch.bool, device="cuda")
    free[slots[live]] = False
    for name, old, x in (("k", before[0], want), ("v", before[1], v.double())):
        pool = getattr(cache, name)
        assert torch.equal(pool.transpose(1, 2).flatten(0, 1)[free], old.transpose(1, 2).flatten(0, 1)[free])
        if cache.format in ("f16", "bf16"):
            near(pool[pg, :, at], x[live], mag[live] if name == "k" else 0 * mag[live], cache.format)
            continue
        ratio, codes, scale = stored_by_product(x.float(), cache.format)
        assert torch.equal(getattr(cache, name + "_scales")[pg, :, at], scale[live])
        diff = (codes_of(cache, name)[pg, :, at] - codes[live]).abs()
        tie = ((ratio - ratio.floor() - 0.5).abs() <= ratio.abs() * 2.0 ** -23)[live]
        assert not bool((diff[~tie] != 0).any()) and float(diff.max() if diff.numel() else 0) <= 1
    assert device_status(0) == 0


@pytest.mark.parametrize("fmt", ["f16", "bf16", "int8", "int4"])
@pytest.mark.parametrize("source", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("dim,hq,hk,page,n", [(64, 9, 3, 16, 1), (64, 14, 2, 16, 37), (128, 32, 8, 64, 133), (128, 1, 1, 256, 300)])
@pytest.mark.parametrize("norm", [False, True])
def test_append_matches_the_formula(cuda, fmt, source, dim, hq, hk, page, n, norm):
    import torch
    from bgtq import PagedCache
    pages = (n + page - 1) // page + 2
    cache = PagedCache(hk, dim, pages, page, fmt)
    qkv = randn(1, n, (hq + 2 * hk) * dim, dtype=source, spread=3.0)
    q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([hq * dim, hk * dim, hk * dim], 1))
    g = torch.Generator(device="cuda").manual_seed(3)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:n]
    slots = torch.where(torch.arange(n, device="cuda") % 5 == 4, -1, slots)
    rotary = table_of(700, dim)
    positions = torch.randint(0, 700, (n,), generator=g, device="cuda")
    norms = [1 + randn(s, dim, spread=0.3) if norm else None for s in (4, 5)]
    for where in (positions, None):
        check_append(cache, q, k, v, slots, rotary, where, *norms, 1e-5, "f16" if fmt == "f16" else "bf16")


@pytest.mark.parametrize("which", ["q", "k"])
@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
def test_append_with_one_norm_and_every_result_type(cuda, which, out):
    import torch
    from bgtq import PagedCache
    cache = PagedCache(2, 64, 8, 16, "int8")
    q, k, v = randn(1, 50, 6, 64), randn(2, 50, 2, 64), randn(3, 50, 2, 64)
    w = 1 + randn(4, 64, spread=0.3)
    norms = (w, None) if which == "q" else (None, w)
    check_append(cache, q, k, v, torch.randperm(128, device="cuda")[:50], table_of(50, 64), None, *norms, 0.0 if which == "q" else 0.5, out)


def test_append_strides_and_addresses(cuda):
    """Views that 16-byte loads cannot follow, broadcast and turned ones give what packed copies give."""
    import torch
    from bgtq import PagedCache
    n, H, d = 50, 3, 64
    base = {t: randn(1, n, 20 * d + 1, dtype=t) for t in ("f32", "bf16")}
    slots, rotary = torch.randperm(128, device="cuda")[:n], table_of(n, d)
    for fmt in ("int8", "int4", "bf16"):
        for x in base.values():
            cut = lambda at, heads: x[:, at:at + heads * d].unflatten(1, (heads, d))
            views = [(cut(1, 6), cut(8 * d, H), cut(11 * d, H)), (cut(0, 6), cut(8 * d + 1, H), cut(11 * d, H)),
                     (cut(0, 6), cut(8 * d, H), cut(12 * d + 1, H)), (cut(0, 6), cut(6 * d, 1).expand(n, H, d), cut(9 * d, H)),
                     (cut(0, 6).flip(0).contiguous().transpose(0, 1).contiguous().transpose(0, 1), cut(6 * d, H), cut(9 * d, H))]
            for q, k, v in views:
                a, b = PagedCache(H, d, 8, 16, fmt), PagedCache(H, d, 8, 16, fmt)
                got = a.append(q, k, v, slots, rotary, keys=True)
                want = b.append(q.contiguous(), k.contiguous(), v.contiguous(), slots, rotary, keys=True)
                assert all(torch.equal(s, t) for s, t in zip(got, want)) and torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
                assert a.k_scales is None or (torch.equal(a.k_scales, b.k_scales) and torch.equal(a.v_scales, b.v_scales))


def test_append_special_values(cuda):
    """Zero heads with and without a norm, infinities and NaN: what holds one is NaN as a whole where it is
    quantised, its neighbours are untouched."""
    import torch
    from bgtq import PagedCache
    for fmt, group in (("int8", 64), ("int4", 32)):
        q, k, v = randn(1, 9, 2, 64), randn(2, 9, 2, 64), randn(3, 9, 2, 64)
        k[1, 0] = 0
        k[2, 1, 5], v[3, 0, 40], k[4, 0, 33] = math.nan, math.inf, -math.inf
        clean = [x.nan_to_num(1.0, 1.0, 1.0) for x in (k, v)]
        slots, rotary = torch.arange(9, device="cuda"), table_of(9, 64)
        one = torch.ones(64, device="cuda")
        for norm in (None, one):
            a, b = PagedCache(2, 64, 1, 16, fmt), PagedCache(2, 64, 1, 16, fmt)
            qa, ka = a.append(q, k, v, slots, rotary, k_norm=norm, keys=True)
            qb, kb = b.append(q, *clean, slots, rotary, k_norm=norm, keys=True)
            assert torch.equal(qa, qb)
            (k1, v1), (k2, v2) = a.read(slots, torch.float32), b.read(slots, torch.float32)
            hurt = torch.zeros((9, 2), dtype=torch.bool, device="cuda")
            hurt[2, 1] = hurt[4, 0] = True
            assert torch.equal(k1[~hurt], k2[~hurt]) and torch.equal(ka[~hurt], kb[~hurt]) and not k1[1, 0].any()
            pair = torch.arange(64, device="cuda") % 32 == 5
            if norm is None and group == 64:
                assert bool(torch.isnan(k1[hurt]).all())
            if norm is None:
                assert bool(torch.isnan(ka[2, 1][pair]).all()) and torch.equal(ka[2, 1][~pair], kb[2, 1][~pair])
            hurt_v = torch.zeros((9, 2, 64), dtype=torch.bool, device="cuda")
            hurt_v[3, 0, (0 if group == 64 else 32):] = True
            assert bool(torch.isnan(v1[hurt_v]).all()) and torch.equal(v1[~hurt_v], v2[~hurt_v])


def test_append_far_rows_of_a_large_pool(cuda):
    """Pages that begin more than 2^32 bytes, and 2^31 elements, into the pool."""
    import torch
    from bgtq import PagedCache
    pages = (2**32 // (256 * 8 * 128 * 2)) + 8
    cache = PagedCache(8, 128, pages, 256, "f16")
    slots = torch.arange((pages - 4) * 256, (pages - 4) * 256 + 300, device="cuda")
    q, k, v = (randn(s, 300, h, 128, dtype="f16") for s, h in ((1, 16), (2, 8), (3, 8)))
    rotary = table_of(300, 128)
    _, keys = cache.append(q, k, v, slots, rotary, keys=True)
    rk, rv = cache.read(slots)
    assert torch.equal(rk, keys) and torch.equal(rv, v)


def test_append_in_a_graph_and_on_a_stream(cuda):
    import torch
    from bgtq import PagedCache
    a, b = PagedCache(2, 64, 4, 16, "int8"), PagedCache(2, 64, 4, 16, "int8")
    q, k, v = randn(1, 5, 4, 64, dtype="bf16"), randn(2, 5, 2, 64, dtype="bf16"), randn(3, 5, 2, 64, dtype="bf16")
    slots, rotary = torch.tensor([3, 40, -1, 7, 63], device="cuda"), table_of(64, 64)
    where = torch.tensor([5, 1, 2, 63, 0], device="cuda")
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        out = a.append(q, k, v, slots, rotary, where)
    for seed in (7, 8):
        q.copy_(randn(seed, 5, 4, 64, dtype="bf16"))
        slots.copy_(slots.roll(1))
        g.replay()
        want = b.append(q, k, v, slots, rotary, where)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(a.k, b.k) and torch.equal(a.v_scales, b.v_scales)


def test_append_refusals_on_the_device(cuda):
    import torch
    from bgtq import PagedCache
    c = PagedCache(2, 64, 4, 16, "int8")
    q, k = randn(1, 3, 4, 64, dtype="bf16"), randn(2, 3, 2, 64, dtype="bf16")
    s, r, p = torch.arange(3, device="cuda"), table_of(9, 64), torch.arange(3, device="cuda")
    for args, message in [((q[:2], k, k, s, r), "one slot"), ((q, k[:, :1], k, s, r), "one slot"), ((q, k, k, s.int(), r), "int64"),
                          ((q.float(), k, k, s, r), "must all be"), ((q.cpu(), k, k, s, r), "device"),
                          ((q, k, k, s, r[:2]), "a row for every"), ((q, k, k, s, r.half()), "rotary"), ((q, k, k, s, r[:, :32]), "rotary"),
                          ((q, k, k, s, r, p.int()), "positions"), ((q, k, k, s, r, p[:2]), "positions"),
                          ((q, k, k, s, r, p, torch.ones(32, device="cuda")), "norms"),
                          ((q, k, k, s, r, p, None, torch.ones(64, device="cuda").half()), "norms"),
                          ((q, k, k, s, r, p, None, None, -1.0), "eps"), ((q, k, k, s, r, p, None, None, 1e-6, torch.int32), "dtype"),
                          ((q.transpose(0, 2).contiguous().transpose(0, 2), k, k, s, r), "contiguous")]:
        with pytest.raises(_lib.RangeError, match=message):
            c.append(*args)
    assert not c.k.any() and not c.v.any()
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert c.append(q[:0], k[:0], k[:0], none, r).shape == (0, 4, 64)


# ---- chunks of new tokens over the pages --------------------------------------------------------

def seen_of(n, length, window, sinks):
    import torch
    p = torch.arange(length - n, length, device="cuda")[:, None]
    t = torch.arange(length, device="cuda")[None]
    seen = t <= p
    if window is not None:
        seen = seen & ((t > p - window) | (t < sinks))
    return seen


def close_chunk(out, lse, ref, dtype, fmt):
    import torch
    want, want_lse, mag, small = ref
    u = U[dtype] if fmt in ("f16", "bf16") else U["f16"] if fmt == "int4" else 2 * U["f16"] + U["f16"] ** 2
    tol = U[dtype] * want.abs() + (u + 3e-5) * mag + 1e-30
    if dtype == "f16" or fmt not in ("f16", "bf16"):
        tol = tol + 2.0 ** -25 * (small + mag + (1 if dtype == "f16" else 0))
    off = (out.double() - want).abs()
    bad = ~(off <= tol) & ~(torch.isnan(want) & torch.isnan(out)) & ~(torch.isinf(want) & (out.double() == want))
    assert not bool(bad.any()), (int(bad.sum()), float((off / tol).nan_to_num(0).max()))
    fin = torch.isfinite(want_lse)
    assert bool((torch.isfinite(lse) == fin).all()) and bool((lse[~fin].nan_to_num(7.0) == want_lse[~fin].float().nan_to_num(7.0)).all())
    assert float((lse.double() - want_lse)[fin].abs().max() if bool(fin.any()) else 0.0) <= 3e-5


def check_chunk(cache, q, new, table, lengths, dtype, window=None, sinks=0, scale=None, only=None, **kw):
    import torch
    out, lse = cache.attend_chunk(q, starts_of(new), table, lengths, scale=scale, window=window, sinks=sinks, lse=True, **kw)
    sc = 1.0 / math.sqrt(cache.dim) if scale is None else scale
    group, ps, at = q.shape[1] // cache.kv_heads, cache.page_size, 0
    for b, (n, length) in enumerate(zip(new, lengths.tolist())):
        rows, at = slice(at, at + n), at + n
        if not n or only is not None and b not in only:
            continue
        t = torch.arange(length, device="cuda")
        slots = table[b].long()[t // ps] * ps + t % ps
        k, v = cache.read(slots, dtype=torch.float32)
        seen = seen_of(n, length, window, sinks)
        for h in sorted({0, q.shape[1] // 2, q.shape[1] - 1}):
            ref = attention64(q[rows, h], k[:, h // group], v[:, h // group], seen, sc)
            close_chunk(out[rows, h], lse[rows, h], ref, dtype, cache.format)
    assert device_status(0) == 0
    return out, lse


NEW = {"steps": ([1, 1, 1, 1, 1], [1, 16, 17, 300, 64]), "drafts": ([5, 1, 3, 8, 2], [5, 90, 64, 1000, 130]),
       "ragged": ([0, 130, 1, 64, 0, 300, 17], [3, 130, 70, 200, 0, 901, 1500]), "whole": ([200, 63, 65], [200, 63, 65])}


@pytest.mark.parametrize("new", sorted(NEW))
@pytest.mark.parametrize("fmt,dtype", FORMATS)
@pytest.mark.parametrize("dim,hq,hk,page", [(64, 9, 3, 16), (128, 8, 2, 64), (64, 14, 2, 128), (128, 5, 5, 32)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 3), (64, 64), (1, 0)])
def test_chunk_matches_the_formula(cuda, new, fmt, dtype, dim, hq, hk, page, window, sinks):
    n, lengths = NEW[new]
    cache, table, lens = paged(10, lengths, hk, dim, page, fmt)
    check_chunk(cache, randn(3, sum(n), hq, dim, dtype=dtype, spread=1.5), n, table, lens, dtype, window, sinks)


@pytest.mark.parametrize("fmt,dtype", FORMATS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1500, 100), (4000, 1)])
def test_chunk_long_histories_are_split_and_joined(cuda, fmt, dtype, dim, window, sinks):
    n, lengths = [3, 0, 40, 1], [9000, 50, 5001, 7000]
    cache, table, lens = paged(20, lengths, 2, dim, 32, fmt)
    check_chunk(cache, randn(3, sum(n), 6, dim, dtype=dtype), n, table, lens, dtype, window, sinks)


@pytest.mark.parametrize("fmt,dtype", [("f16", "f16"), ("int8", "bf16"), ("int4", "f16"), ("int4", "bf16")])
@pytest.mark.parametrize("hq,hk", [(1, 1), (16, 1), (17, 1), (48, 2), (71, 1), (128, 1)])
@pytest.mark.parametrize("n", [1, 2, 33])
def test_chunk_head_groups(cuda, fmt, dtype, hq, hk, n):
    cache, table, lens = paged(30, [700, 33], hk, 128, 128, fmt)
    check_chunk(cache, randn(3, 2 * n, hq, 128, dtype=dtype), [n, n], table, lens, dtype, 200, 5)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("fmt,dtype", [("bf16", "bf16"), ("int8", "f16"), ("int4", "bf16")])
@pytest.mark.parametrize("most", [4, 60])
def test_chunk_many_requests(cuda, page, fmt, dtype, most):
    rng = np.random.default_rng(5)
    n = rng.integers(0, most + 1, 150).tolist()
    lengths = [a + int(b) for a, b in zip(n, rng.integers(0, 400, 150))]
    cache, table, lens = paged(40, lengths, 2, 64, page, fmt)
    check_chunk(cache, randn(3, sum(n), 8, 64, dtype=dtype), n, table, lens, dtype, only=[*range(0, 150, 11), 149])


@pytest.mark.parametrize("fmt,dtype", FORMATS)
def test_chunk_large_windows_and_sinks_are_no_window(cuda, fmt, dtype):
    """A window of all tokens, or sinks that reach the window, leave nothing out."""
    import torch
    n, lengths = [20, 1], [700, 300]
    cache, table, lens = paged(25, lengths, 2, 64, 16, fmt)
    q = randn(3, 21, 4, 64, dtype=dtype)
    want, want_lse = check_chunk(cache, q, n, table, lens, dtype)
    for window, sinks in ((700, 0), (2**31 - 1, 2**31 - 1), (1, 2**31 - 1), (64, 700)):
        out, lse = check_chunk(cache, q, n, table, lens, dtype, window, sinks)
        assert torch.equal(lse.isfinite(), want_lse.isfinite())


@pytest.mark.parametrize("fmt,dtype", FORMATS)
@pytest.mark.parametrize("dim", [64, 128])
def test_attend_with_a_window_is_a_chunk_of_one(cuda, fmt, dtype, dim):
    import torch
    lengths = [1, 900, 0, 64, 5000, 33]
    cache, table, lens = paged(26, lengths, 2, dim, 32, fmt)
    q = randn(3, 6, 4, dim, dtype=dtype)
    out, lse = cache.attend(q, table, lens, window=100, sinks=4, lse=True)
    # (no request of length 0 among those that are compared: its row sees nothing)
    assert not out[2].any() and bool((lse[2] == -math.inf).all())
    keep = [0, 1, 3, 4, 5]
    o, l = check_chunk(cache, q[keep], [1] * 5, table[keep], lens[keep], dtype, 100, 4)
    for a, b in ((out[keep], o), (lse[keep], l)):
        assert float((a.double() - b.double()).abs().max()) <= 0.05
    full, plain = cache.attend(q, table, lens, window=9000), cache.attend(q, table, lens)
    assert float((full.double() - plain.double()).abs().max()) <= 4 * U["bf16"] * float(plain.abs().max())


@pytest.mark.parametrize("n", [2, 40])
def test_chunk_rows_before_the_first_token_see_nothing(cuda, n):
    """More new rows than the pages hold tokens: the first of them are at negative positions."""
    import torch
    cache, table, lens = paged(27, [3, 30], 1, 64, 16, "f16")
    lens = torch.tensor([1, 30], dtype=torch.int32, device="cuda")
    q = randn(3, n + 30, 3, 64, dtype="f16")
    for window in (None, 5):
        out, lse = cache.attend_chunk(q, starts_of([n, 30]), table, lens, window=window, sinks=2, lse=True)
        assert not out[:n - 1].any() and bool((lse[:n - 1] == -math.inf).all())
        k, v = cache.read(table[0, :1].long() * 16, dtype=torch.float32)
        assert torch.equal(out[n - 1], v[0].half().expand(3, 64))
        assert bool(torch.isfinite(lse[n - 1:]).all())


@pytest.mark.parametrize("fmt", ["f16", "int8", "int4"])
@pytest.mark.parametrize("n", [1, 30])
def test_chunk_rising_maximum_and_large_logits(cuda, fmt, n):
    import torch
    from bgtq import PagedCache
    length = 3000
    cache = PagedCache(1, 64, 200, 16, fmt)
    ramp = torch.linspace(-4, 4, length, device="cuda")
    k = ramp[:, None, None] * torch.ones((1, 1, 64), device="cuda")
    table = torch.arange(200, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([length], dtype=torch.int32, device="cuda")
    q = torch.ones((n, 8, 64), device="cuda", dtype=torch.float16)
    for keys in (k, k.flip(0)):
        cache.write(keys, randn(1, length, 1, 64), torch.arange(length, device="cuda"))
        check_chunk(cache, q, [n], table, lens, "f16")
        check_chunk(cache, q, [n], table, lens, "f16", 700, 100)


@pytest.mark.parametrize("fmt,dtype", FORMATS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [2, 100])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("window,sinks", [(None, 0), (70, 10)])
def test_chunk_what_a_row_does_not_see_does_not_reach_it(cuda, fmt, dtype, dim, n, bad, window, sinks):
    """Infinities and NaN in keys and values of later tokens, and of tokens that have left the window, leave rows
    that do not see them bit by bit; rows that do have them in the places where the formula has them."""
    import torch
    length = 400
    cache, table, lens = paged(28, [length], 2, dim, 16, fmt)
    q = randn(3, n, 4, dim, dtype=dtype)
    want, want_lse = check_chunk(cache, q, [n], table, lens, dtype, window, sinks)
    t = torch.arange(length, device="cuda")
    slots = table[0].long()[t // 16] * 16 + t % 16
    if fmt in ("f16", "bf16"):
        where = (cache.v, cache.k)
        cut = slice(5, 6)
    else:
        where = (cache.v_scales, cache.k_scales)
        cut = slice(0, 1)
    seen = seen_of(n, length, window, sinks)
    for pool in where:
        for at in (length - 1, length - n // 2 - 1, length - 75, length - 150, 15, 3):
            s = slots[at]
            old = pool[s // 16, 1, s % 16, cut].clone()
            pool[s // 16, 1, s % 16, cut] = bad if fmt in ("f16", "bf16") else math.nan
            out, lse = cache.attend_chunk(q, starts_of([n]), table, lens, window=window, sinks=sinks, lse=True)
            pool[s // 16, 1, s % 16, cut] = old
            blind = ~seen[:, at]
            assert torch.equal(out[blind], want[blind]) and torch.equal(lse[blind], want_lse[blind]), at
            assert torch.equal(out[:, :2], want[:, :2]) and torch.equal(lse[:, :2], want_lse[:, :2]), at
            if pool is where[0]:
                assert torch.equal(lse, want_lse)
                dims = cut if fmt in ("f16", "bf16") else slice(0, 32 if fmt == "int4" else dim)
                hit = out[~blind][:, 2:, dims].float()
                if fmt in ("f16", "bf16") and bad == math.inf:
                    assert bool(((hit == bad) | hit.isnan()).all())
                else:
                    assert bool(hit.isnan().all()), at
                rest = torch.ones(dim, dtype=torch.bool, device="cuda")
                rest[dims] = False
                assert torch.equal(out[..., rest], want[..., rest]), at


def test_chunk_rows_that_no_request_holds(cuda):
    """Rows before the first request, behind the last one and of skipped requests are left as they were."""
    import torch
    cache, table, lens = paged(29, [50, 20, 300], 2, 64, 16, "int8")
    for n, tail in (([2, 1, 2], 3), ([20, 1, 100], 30)):
        q = randn(3, 4 + sum(n) + tail, 4, 64, dtype="bf16")
        st = starts_of(n) + 4
        out = torch.full_like(q, 7.0)
        cache.attend_chunk(q, st, table, lens, out=out)
        assert bool((out[:4] == 7).all()) and bool((out[4 + sum(n):] == 7).all())
        want = cache.attend_chunk(q[4:4 + sum(n)], st - 4, table, lens)
        assert float((out[4:4 + sum(n)].double() - want.double()).abs().max()) <= 4 * U["bf16"] * float(want.abs().max())


def test_chunk_strides_tables_and_streams(cuda):
    import torch
    n, lengths = [1, 30, 2, 150], [100, 900, 5, 1500]
    cache, table, lens = paged(50, lengths, 2, 64, 16, "f16")
    wide = torch.full((4, table.shape[1] + 9), 2**31 - 1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    for count in (n, [1, 1, 1, 1]):
        st = starts_of(count)
        for off in (0, 1, 8):
            qkv = randn(3, sum(count), 10 * 64 + 8, dtype="f16")
            q = qkv[:, off:6 * 64 + off].unflatten(1, (6, 64))
            want = cache.attend_chunk(q.contiguous(), st, table, lens)
            assert torch.equal(cache.attend_chunk(q, st, wide[:, :table.shape[1]], lens), want)
            assert torch.equal(cache.attend_chunk(q, st, wide, lens), want)
        turned = q.transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(cache.attend_chunk(turned, st, table, lens), want)
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = []
        for _ in range(4):
            for s in streams:
                with torch.cuda.stream(s):
                    got.append(cache.attend_chunk(q, st, table, lens))
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("fmt", ["f16", "int8", "int4"])
def test_chunk_in_a_graph_while_requests_grow(cuda, fmt):
    """Recorded on a stream without a workspace, replayed over other starts, lengths and pages."""
    import torch
    from bgtq import PagedCache
    cache = PagedCache(1, 64, 64, 16, fmt)
    table = torch.arange(64, dtype=torch.int32, device="cuda").view(2, 32)
    t = torch.arange(1024, device="cuda")
    cache.write(randn(1, 1024, 1, 64), randn(2, 1024, 1, 64), t)
    for rows in (6, 150):
        lens = torch.tensor([rows, 400], dtype=torch.int32, device="cuda")
        st = starts_of([rows - 3, 3])
        q = randn(3, rows, 4, 64, dtype="f16")
        out = torch.zeros_like(q)
        cache.attend_chunk(q, st, table, lens, out=out, window=90, sinks=3)
        torch.cuda.synchronize()
        side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            cache.attend_chunk(q, st, table, lens, out=out, window=90, sinks=3)
        for a, b, c in ((1, 101, 200), (rows - 1, 512, 512), (0, 0, 300)):
            lens.copy_(torch.tensor([b, c], dtype=torch.int32))
            st.copy_(torch.tensor([0, a, rows], dtype=torch.int32))
            q.copy_(randn(a, rows, 4, 64, dtype="f16"))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, cache.attend_chunk(q, st, table, lens, window=90, sinks=3))


@pytest.mark.parametrize("fmt", ["bf16", "int8", "int4"])
def test_chunk_repeated_over_changing_lengths(cuda, fmt):
    """Calls that follow each other without a pause, whole and in parts in turn, give the bits of a call alone."""
    import torch
    calls = []
    for i, (n, lengths) in enumerate([([1, 700, 33, 257], [9, 900, 33, 1000]), ([600], [5000]), ([2] * 40, [64] * 40),
                                      ([5, 100, 1], [4000, 101, 7000])]):
        cache, table, lens = paged(60 + i, lengths, 2, 128, 32, fmt)
        calls.append((cache, (randn(i, sum(n), 8, 128, dtype="bf16"), starts_of(n), table, lens)))
    want = []
    for cache, args in calls:
        want.append(cache.attend_chunk(*args))
        torch.cuda.synchronize()
    got = [calls[i % 4][0].attend_chunk(*calls[i % 4][1]) for i in range(60)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 4]) for i, g in enumerate(got)) and device_status() == 0


@pytest.mark.parametrize("n", [2, 200])
def test_chunk_offsets_past_32_bits(cuda, n):
    """Pages that begin more than 2^32 bytes, and 2^31 elements, into the pool."""
    import torch
    from bgtq import PagedCache
    pages = (2**32 // (256 * 8 * 128 * 2)) + 8
    cache = PagedCache(8, 128, pages, 256, "f16")
    slots = torch.arange((pages - 4) * 256, (pages - 4) * 256 + 700, device="cuda")
    cache.write(randn(1, 700, 8, 128, dtype="f16"), randn(2, 700, 8, 128, dtype="f16"), slots)
    table = torch.arange(pages - 4, pages - 1, dtype=torch.int32, device="cuda")[None].contiguous()
    check_chunk(cache, randn(3, n, 16, 128, dtype="f16"), [n], table, torch.tensor([700], dtype=torch.int32, device="cuda"), "f16", 300, 20)


@pytest.mark.parametrize("fmt", ["int8", "int4"])
@pytest.mark.parametrize("n", [2, 90])
def test_chunk_sizes_of_rows(cuda, fmt, n):
    """Key and value rows of very different size: the scales span BF16's range, not FP16's."""
    import torch
    from bgtq import PagedCache
    length = 500
    cache = PagedCache(1, 64, 40, 16, fmt)
    size = torch.logspace(-20, 3, length, device="cuda")[:, None, None]
    small = torch.logspace(-9, 0.3, length, device="cuda")[:, None, None]
    table = torch.arange(40, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([length], dtype=torch.int32, device="cuda")
    for dtype, by in (("bf16", 1.0), ("bf16", 1e-6), ("f16", 1e-2)):
        cache.write(randn(1, length, 1, 64) * small / by, randn(2, length, 1, 64) * (size if dtype == "bf16" else small), torch.arange(length, device="cuda"))
        check_chunk(cache, (randn(3, n, 3, 64) * by).to(types()[dtype]), [n], table, lens, dtype)


@pytest.mark.parametrize("fmt,dtype", [("int8", "f16"), ("int8", "bf16"), ("int4", "f16"), ("int4", "bf16")])
@pytest.mark.parametrize("dim,hq", [(64, 2), (64, 7), (128, 3), (128, 16)])
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("big", [1e5, 1e12, 1e30])
@pytest.mark.parametrize("where", ["first", "last", "half"])
def test_chunk_large_values_without_weight(cuda, fmt, dtype, dim, hq, n, big, where):
    """Rows of large values that no row gives weight to leave the others as they are, and so do keys that are next to
    nothing beside them.  Tolerance: as test_gpu_serving_extremes derives it for one token, 2^-33 of the row's largest
    probability x value for every token, and FP16's rounding of values in 8 bits."""
    import torch
    from bgtq import PagedCache
    length = 700
    far = torch.zeros(length, dtype=torch.bool, device="cuda")
    if where == "half":
        far[1::2] = True
    else:
        far[{"first": 0, "last": length - n}[where]] = True
    k, v = randn(1, length, 1, dim), randn(2, length, 1, dim) + 0.5
    k[::5] *= 1e-13
    k[:, 0, 0] = 0
    k[far] = 0
    k[far, 0, 0] = -2400.0                     # logits of -300: weights below 2^-420
    v[far] = big
    q = randn(3, n, hq, dim, dtype=dtype)
    q[..., 0] = 1.0
    cache = PagedCache(1, dim, 44, 16, fmt)
    t = torch.arange(length, device="cuda")
    cache.write(k, v, t)
    table = torch.arange(44, dtype=torch.int32, device="cuda")[None]
    out, lse = cache.attend_chunk(q, starts_of([n]), table, torch.tensor([length], dtype=torch.int32, device="cuda"), scale=1.0 / 8, lse=True)
    rk, rv = (x[:, 0].double() for x in cache.read(t, torch.float32))
    for h in range(hq):
        s = (q[:, h].double() @ rk.T / 8).masked_fill(~seen_of(n, length, None, 0), -math.inf)
        p = torch.softmax(s, -1)
        want, mag = p @ rv, p @ rv.abs()
        least = length * 2.0 ** -33 * (p * rv.abs().amax(-1)).amax(-1, keepdim=True)
        tol = U[dtype] * want.abs() + (2 * U["f16"] + 3e-5) * mag + least + (2.0 ** -25 if dtype == "f16" else 0)
        off = (out[:, h].double() - want).abs()
        assert bool((off <= tol).all()), float((off / tol).max())
        assert float((lse[:, h].double() - torch.logsumexp(s, -1)).abs().max()) <= 3e-5


def test_indices_outside_the_cache_are_left_out_and_reported(cuda):
    """In a process of its own: the device status word keeps its bits."""
    code = '''
import math, torch, bgtq
from bgtq import PagedCache, adjust_logits, device_status
dev = "cuda"
i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
i64 = lambda *x: torch.tensor(x, device=dev)
table = torch.randn(10, 64, device=dev)
for fmt in ("int8", "int4", "f16"):
    c = PagedCache(2, 64, 4, 16, fmt)
    x, q = torch.randn(4, 2, 64, device=dev), torch.randn(4, 3, 64, device=dev)
    good = c.append(q, x, x, i64(5, 6, 7, 8), table, i64(0, 1, 2, 3))
    kept = c.k.clone()
    got = c.append(q, x + 1, x + 1, i64(64, 2**40, 2**62, -5), table, i64(0, 1, 2, 3))
    assert torch.equal(got, good) and torch.equal(c.k, kept)
assert device_status(0) == 4
for fmt in ("int8", "f16"):
    c = PagedCache(2, 64, 4, 16, fmt)
    got, keys = c.append(q, x, x, i64(5, 6, 7, 8), table, i64(0, 10, -1, 2**40), keys=True)
    assert torch.equal(got[0], good[0]) and not got[1:].any() and not keys[1:].any() and c.k[0, :, 5].any() and not c.k[0, :, 6:].any()
assert device_status(0) == 12
for fmt in ("f16", "int8", "int4"):
    c = PagedCache(1, 64, 4, 16, fmt)
    y = torch.randn(64, 1, 64, device=dev).half()
    c.write(y, y, torch.arange(64, device=dev))
    w = c.read(torch.arange(64, device=dev), torch.float32)[0]
    for n in (1, 2, 40):
        q = torch.randn(2 * n, 2, 64, device=dev).half()
        st = i32(0, n, 2 * n)
        # a page that is not there: its tokens are left out
        b = c.attend_chunk(q, st, torch.stack([i32(0, 9999, 3), i32(0, -5, 7)]), i32(40, 48))
        for s, pages in ((0, (0, None, 3)), (1, (0, None, None))):
            length = (40, 48)[s]
            at = torch.tensor([p * 16 + i if p is not None else -1 for p in pages for i in range(16)], device=dev)[:length]
            pos = torch.arange(length - n, length, device=dev)[:, None]
            seen = (torch.arange(length, device=dev)[None] <= pos) & (at >= 0)[None]
            k = w[at.clamp(min=0), 0]
            for h in range(2):
                p = torch.softmax(((q[s * n:(s + 1) * n, h].float() @ k.T) / 8).masked_fill(~seen, -math.inf), -1) @ k
                p = torch.where(seen.any(-1, keepdim=True), p, 0.0)
                assert (b[s * n:(s + 1) * n, h] - p).abs().max() < 0.04, (fmt, n, s)
        # lengths past the table, and negative ones
        o, l = c.attend_chunk(q, st, i32(0, 1, 2, 3).view(2, 2), i32(1000, -3), lse=True)
        full, fl = c.attend_chunk(q, st, i32(0, 1, 2, 3).view(2, 2), i32(32, 0), lse=True)
        assert torch.equal(o, full) and torch.equal(l, fl) and not o[n:].any()
        # starts that fall, or pass the rows
        o = torch.full_like(q, 7.0)
        c.attend_chunk(q, i32(0, n, n - 1, 3 * n + 1, 3 * n + 1), i32(0, 1, 2, 3).view(4, 1), i32(9, 9, 9, 9), out=o)
        want = c.attend_chunk(q[:n], i32(0, n), i32(0).view(1, 1), i32(9))
        assert (o[:n] - want).abs().max() < 0.04 and bool((o[n:] == 7).all()), (fmt, n)
assert device_status(0) == 12
x = torch.randn(2, 33, device=dev)
got = adjust_logits(x, i32(3, 33, -1, 3, 9, 9).view(2, 3), i32(3, 3), presence=1.0)
want = x.clone()
want[0, 3] -= 1.0
want[1, [3, 9]] -= 1.0
assert torch.equal(got, want) and device_status(0) == 12
got = adjust_logits(x, i32(3, 32, -1, 3, 9, 9).view(2, 3), i32(9, -4), frequency=1.0, bias_ids=i32(2**31 - 1, -7).view(1, 2),
                    bias=torch.ones(1, 2, device=dev))
want = x.clone()
want[0, [3, 32]] -= 1.0
assert torch.equal(got, want) and device_status(0) == 12
print("fine")
'''
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       cwd=ROOT / "block-gqt-webgpu_b200")
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr


def test_chunk_refusals_on_the_device(cuda):
    import ctypes as C
    import torch
    from bgtq import PagedCache
    c = PagedCache(2, 64, 4, 16, "f16")
    q = randn(1, 5, 4, 64, dtype="f16")
    st, table, lengths = starts_of([2, 3]), torch.zeros((2, 2), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for args, message in [((q[:, :3], st, table, lengths), "multiple"), ((q.bfloat16(), st, table, lengths), "16-bit pages"),
                          ((q, st.long(), table, lengths), "starts"), ((q, st.view(3, 1), table, lengths), "starts"), ((q, st.cpu(), table, lengths), "starts"),
                          ((q, st[:2], table, lengths), "table"), ((q, None, table, lengths), "table"), ((q, st, table.long(), lengths), "table"),
                          ((q, st, table, lengths.long()), "lengths"), ((q, st, table, lengths[:1]), "lengths"),
                          ((q.cpu(), st, table, lengths), "device"), ((q, st, table, lengths, -1.0), "scale"),
                          ((q, st, table, lengths, None, 0), "window"), ((q, st, table, lengths, None, 5, -1), "window"),
                          ((q, st, table, lengths, None, 2**31), "window"), ((q, st, table, lengths, None, None, 0, q.float()), "out"),
                          ((randn(1, 5, 2 * 129, 64, dtype="f16"), st, table, lengths), "128 query heads")]:
        with pytest.raises(_lib.RangeError, match=message):
            c.attend_chunk(*args)
    with pytest.raises(_lib.RangeError, match="window"):
        c.attend(q[:2], table, lengths, window=0)
    assert c.attend_chunk(q[:0], starts_of([0, 0]), table, lengths).shape == (0, 4, 64)
    assert c.attend_chunk(q[:0], starts_of([]), table[:0], lengths[:0]).shape == (0, 4, 64)
    need = C.c_size_t()
    _lib.call("bgtq_paged_chunk_workspace", c._ref, 4, C.byref(need))
    room = torch.zeros(need.value + 128, dtype=torch.uint8, device="cuda")
    for address, size in ((None, need.value), (room.data_ptr(), need.value - 1), (room.data_ptr() + 16, need.value)):
        p = _lib.ChunkDesc(_lib.F16, 2, 4, 5, q.data_ptr(), 256, 64, st.data_ptr(), table.data_ptr(), 2, 2, lengths.data_ptr(), 0.0, 0, 0,
                           torch.empty_like(q).data_ptr(), None, address, size)
        with pytest.raises(_lib.RangeError, match="workspace"):
            _lib.call("bgtq_paged_attend_chunk", c._ref, C.byref(p), None)


# ---- what is put on logits ------------------------------------------------------------------------

def check_logits(x, ids=None, lengths=None, r=None, p=None, f=None, bias_ids=None, bias=None, mask=None, got=None, **kw):
    import torch
    from bgtq import adjust_logits
    old = x.clone()
    if got is None:
        got = adjust_logits(x, ids, lengths, repetition=r, presence=p, frequency=f, bias_ids=bias_ids, bias=bias, mask=mask, **kw)
    dtype = {t: n for n, t in types().items()}[x.dtype]
    want, mag = old.double(), old.double().abs()
    per = lambda v, b, none: none if v is None else float(v[b]) if torch.is_tensor(v) else float(np.float32(v))
    B, V = x.shape
    for b in range(B):
        if ids is not None:
            h = ids[b] if lengths is None else ids[b, :int(lengths[b])]
            h = h[(h >= 0) & (h < V)].long()
            c = torch.bincount(h, minlength=V).double()
            again, rr = c > 0, per(r, b, 1.0)
            want[b] = torch.where(again, torch.where(want[b] > 0, want[b] / rr, want[b] * rr), want[b])
            mag[b] += torch.where(again, want[b].abs(), 0.0)
            for step in (per(p, b, 0.0) * again, per(f, b, 0.0) * c):
                want[b] -= step
                mag[b] += 2 * step.abs()
        if bias is not None:
            i, y = bias_ids[b % len(bias_ids)].long(), bias[b % len(bias)].double()
            there = (i >= 0) & (i < V)
            want[b].index_put_((i[there],), y[there], accumulate=True)
            mag[b].index_put_((i[there],), 2 * y[there].abs(), accumulate=True)
        if mask is not None:
            bits = (mask[b % len(mask)].long()[:, None] >> torch.arange(32, device="cuda")) & 1
            want[b] = torch.where(bits.flatten()[:V] != 0, want[b], -math.inf)
    fin = torch.isfinite(want)
    assert torch.equal(got.double()[~fin].nan_to_num(7.0), want[~fin].nan_to_num(7.0))
    tol = U.get(dtype, U32) * want.abs() + 5 * U32 * mag + (2.0 ** -25 if dtype == "f16" else 0)
    off = (got.double() - want).abs()[fin]
    assert bool((off <= tol[fin]).all()), float((off / tol[fin]).max())
    assert device_status(0) == 0
    return got


def history(seed, batch, width, vocab, dtype="int32"):
    """Ids dense at the low end, every ninth one padding."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = (torch.rand((batch, width), generator=g, device="cuda") ** 3 * vocab).long().clamp(max=vocab - 1)
    ids = torch.where(torch.arange(width, device="cuda") % 9 == 4, -1, ids)
    return ids.to(getattr(torch, dtype))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("batch,vocab,width", [(1, 1, 3), (1, 49152, 300), (5, 331, 40), (3, 50001, 1), (37, 8193, 700), (2, 151936, 5000)])
@pytest.mark.parametrize("ids", ["int32", "int64"])
def test_logits_match_the_formula(cuda, dtype, batch, vocab, width, ids):
    import torch
    x = randn(1, batch, vocab, dtype=dtype, spread=4.0)
    h = history(2, batch, width, vocab, ids)
    lens = torch.tensor([(7 * b + width) % (width + 1) for b in range(batch)], dtype=torch.int32, device="cuda")
    r, p, f = 1 + randn(3, batch).abs(), randn(4, batch), randn(5, batch) * 0.3
    bias_ids = history(6, batch, 77, vocab)       # the same id many times
    bias = randn(7, batch, 77, spread=3.0)
    mask = torch.randint(-2**31, 2**31, (batch, (vocab + 31) // 32), device="cuda", generator=torch.Generator(device="cuda").manual_seed(8)).int()
    check_logits(x, h, lens, r, p, f, bias_ids, bias, mask)
    check_logits(x, h, None, r, p, f)
    check_logits(x, h, lens, r=1.3)
    check_logits(x, h, lens, p=0.5)
    check_logits(x, h, lens, f=-0.25)
    check_logits(x, bias_ids=bias_ids, bias=bias)
    check_logits(x, mask=mask)
    check_logits(x, h, lens, 1.1, 0.5, 0.25, bias_ids[:1], bias[:1], mask[:1])
    assert torch.equal(check_logits(x), x)


def test_logits_strides_in_place_and_another_output(cuda):
    import torch
    from bgtq import adjust_logits
    wide = randn(1, 6, 1003, spread=4.0)
    h, b = history(2, 6, 90, 997), randn(7, 6, 9)
    ids = history(3, 6, 9, 997)
    mask = torch.randint(-2**31, 2**31, (6, 40), device="cuda").int()
    for off in (0, 1, 4):
        x = wide[:, off:off + 997]
        want = check_logits(x.contiguous(), h, None, 1.2, 0.3, 0.1, ids, b, mask[:, :32].contiguous())
        args = dict(repetition=1.2, presence=0.3, frequency=0.1, bias_ids=ids, bias=b, mask=mask[:, :32])
        assert torch.equal(adjust_logits(x, h, **args), want)
        assert torch.equal(adjust_logits(x, h.long().repeat(1, 2)[:, :90], **args), want)
        room = torch.full((6, 1010), 7.0, device="cuda")
        got = adjust_logits(x, h, out=room[:, 3:1000], **args)
        assert torch.equal(got, want) and bool((room[:, :3] == 7).all()) and bool((room[:, 1000:] == 7).all())
        assert torch.equal(adjust_logits(x[:1].expand(6, 997), h, **args)[1:3], check_logits(x[:1].expand(6, 997).contiguous(), h, None, 1.2, 0.3, 0.1, ids, b, mask[:, :32].contiguous())[1:3])
        y = x.clone()
        back = adjust_logits(y, h, out=y, **args)
        assert back is y and torch.equal(y, want)


def test_logits_special_values(cuda):
    """Infinities and NaN stay what they are unless they are masked; zero is not divided."""
    import torch
    from bgtq import adjust_logits
    x = torch.tensor([[math.inf, -math.inf, math.nan, 0.0, -0.0, 3e38, -3e38, 1e-45]], device="cuda")
    h = torch.arange(8, device="cuda", dtype=torch.int32)[None]
    got = adjust_logits(x, h, repetition=2.0)
    assert torch.equal(got.nan_to_num(7.0, 8.0, 9.0), torch.tensor([[8.0, 9.0, 7.0, 0.0, 0.0, 1.5e38, 9.0, 0.0]], device="cuda"))
    assert bool((adjust_logits(x, mask=torch.zeros((1, 1), dtype=torch.int32, device="cuda")) == -math.inf).all())
    # a count that 16 bits do not hold
    h = torch.full((1, 70000), 5, dtype=torch.int32, device="cuda")
    assert float(adjust_logits(torch.zeros((1, 9), device="cuda"), h, frequency=1.0)[0, 5]) == -70000.0


def test_logits_in_a_graph_repeated_and_on_two_streams(cuda):
    import torch
    from bgtq import adjust_logits
    x, h = randn(1, 9, 5000, spread=4.0), history(2, 9, 600, 5000)
    lens = torch.full((9,), 600, dtype=torch.int32, device="cuda")
    ids, b = history(3, 9, 200, 50), randn(4, 9, 200)
    args = dict(repetition=torch.full((9,), 1.2, device="cuda"), frequency=torch.full((9,), 0.5, device="cuda"), bias_ids=ids, bias=b)
    want = adjust_logits(x, h, lens, **args)
    assert all(torch.equal(adjust_logits(x, h, lens, **args), want) for _ in range(20))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(adjust_logits(x, h, lens, **args))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = adjust_logits(x, h, lens, **args)
    lens.fill_(7)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, adjust_logits(x, h, lens, **args)) and not torch.equal(out, want)


def test_logits_refusals_on_the_device(cuda):
    import torch
    from bgtq import adjust_logits
    x, h = randn(1, 2, 100), history(2, 2, 9, 100)
    lens, ids, b = torch.ones(2, dtype=torch.int32, device="cuda"), history(3, 2, 4, 100), randn(4, 2, 4)
    mask = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    for kw, message in [(dict(logits=x[0]), "batch, vocab"), (dict(logits=x.cpu()), "CUDA"), (dict(logits=x.long()), "float16, bfloat16"),
                        (dict(logits=x.t().contiguous().t()), "contiguous"), (dict(tokens=h.short()), "int32 or int64"), (dict(tokens=h[:1]), "int32 or int64"),
                        (dict(tokens=h.cpu()), "int32 or int64"), (dict(tokens=h, lengths=lens.long()), "lengths"), (dict(lengths=lens), "with tokens"),
                        (dict(repetition=1.5), "need tokens"), (dict(tokens=h, repetition=0.0), "positive"), (dict(tokens=h, presence=math.inf), "finite"),
                        (dict(tokens=h, frequency=torch.ones(3, device="cuda")), "frequency"), (dict(tokens=h, presence=torch.ones(2)), "presence"),
                        (dict(bias=b), "together"), (dict(bias_ids=ids.long(), bias=b), "int32"), (dict(bias_ids=ids[:, :3], bias=b), "one shape"),
                        (dict(bias_ids=ids.repeat(2, 1), bias=b.repeat(2, 1)), "bias must be"), (dict(mask=mask[:, :3]), "a bit for each"),
                        (dict(mask=mask.long()), "int32"), (dict(mask=mask.repeat(2, 1)), "mask must be"), (dict(out=x.half()), "out must be"),
                        (dict(out=x[:1]), "out must be"), (dict(out=x[:1].expand(2, 100)), "out must be")]:
        with pytest.raises(_lib.RangeError, match=message):
            adjust_logits(**{"logits": x, **kw})
    assert adjust_logits(x[:0], h[:0], presence=1.0).shape == (0, 100)


# ---- together --------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt,dtype", FORMATS)
@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 2)])
def test_a_prompt_in_chunks_is_the_prompt_token_by_token(cuda, fmt, dtype, window, sinks):
    """Tokens appended and attended in chunks of any size, and one at a time, then a token chosen: both follow the
    formula over the rows that the pages hold, and choose alike."""
    import torch
    from bgtq import PagedCache, adjust_logits
    n, hq, hk, d = 90, 6, 2, 64
    qkv = randn(1, n, (hq + 2 * hk) * d, dtype=dtype)
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, hk * d, hk * d], 1))
    rotary, w = table_of(n, d), 1 + randn(2, d, spread=0.2)
    head = randn(3, hq * d, 500, dtype=dtype, spread=0.1)
    outs = []
    for sizes in ([1] * n, [37, 1, 2, 50], [n]):
        cache = PagedCache(hk, d, 9, 16, fmt)
        table = torch.tensor([[4, 0, 8, 2, 6, 1]], dtype=torch.int32, device="cuda")
        at, parts = 0, []
        for m in sizes:
            t = torch.arange(at, at + m, device="cuda")
            slots = table[0].long()[t // 16] * 16 + t % 16
            rq = cache.append(q[at:at + m], k[at:at + m], v[at:at + m], slots, rotary, t, q_norm=w, k_norm=w)
            at += m
            lens = torch.tensor([at], dtype=torch.int32, device="cuda")
            parts.append(cache.attend_chunk(rq, starts_of([m]), table, lens, window=window, sinks=sinks))
        outs.append(torch.cat(parts))
        if len(outs) == 1:
            t = torch.arange(n, device="cuda")
            rk, rv = cache.read(table[0].long()[t // 16] * 16 + t % 16, torch.float32)
            want_q = turned64(q, rotary, w, 1e-6)[0].to(types()[dtype])
            for h in range(hq):
                ref = attention64(want_q[:, h], rk[:, h // 3], rv[:, h // 3], seen_of(n, n, window, sinks), d ** -0.5)
                # (queries are rounded from FP32 here and from 64 bits there: an ulp of a few elements, which moves a
                # logit by at most 2 u times the largest |q||k| of a dimension: far inside of BF16's own tolerance)
                off = (outs[0][:, h].double() - ref[0]).abs()
                assert float((off / (ref[2] + 1e-30)).max()) <= 4 * U["bf16"]
    for o in outs[1:]:
        assert float((o.double() - outs[0].double()).norm() / outs[0].double().norm()) <= 2 * U["bf16"]
    logits = [(o[-1:].flatten(1).float() @ head.float()) for o in outs]
    mask = torch.full((1, 16), -1, dtype=torch.int32, device="cuda")
    best = [int(adjust_logits(x, torch.tensor([[3, 3, 9]], device="cuda"), presence=0.1, mask=mask).argmax()) for x in logits]
    gap = float(logits[0].topk(2)[0].diff().abs())
    assert len(set(best)) == 1 or gap <= 2 * U["bf16"] * float(logits[0].norm())
