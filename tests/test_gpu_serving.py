"""The serving operators on the GPU: packed prompts, the paged cache and one token over its
pages, against plain formulas in 64 bits.

Tolerances, from the arithmetic (u = unit roundoff of the 16-bit type, 2^-11 FP16, 2^-8 BF16):
an output o = sum p_t v_t, with the probabilities rounded to the queries' type before the
product and the result rounded once, is within u |o| + u A of the exact value, A = sum p_t
|v_t|; FP32 sums, the exponential and the logits' rounding (logits below 64, so 64 * 2^-23
relative on a probability) add at most 3e-5 A; an FP16 probability below 2^-14 is held to
2^-25 absolute, which adds 2^-25 sum |v_t| / l, l = sum exp(s_t - max) >= 1.  The log sum is
FP32 throughout: 3e-5 absolute.
Stored rows are exact: the formula's steps are FP32 with IEEE rounding; a 64-bit computation of
the scale (rounded to FP32 before BF16) gives the same one but for about one group in 2^17, whose
maximum / top is within an FP32 rounding of a BF16 tie (none of these inputs has one), and a code
can differ from the 64-bit one only where x / s falls on a half within an FP32 rounding; those
places are counted, and a code there may differ by one.
"""
import math
import subprocess
import sys

import numpy as np
import pytest

from bgtq import _lib, device_status
from conftest import ROOT

pytestmark = pytest.mark.gpu
U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def types():
    import torch
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def randn(seed, *shape, dtype="f32", spread=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * spread).to(types()[dtype])


# ---- plain forms in 64 bits ------------------------------------------------------------

def attention64(q, k, v, seen, scale):
    """q [n, d], k, v [m, d], seen [n, m]: (out, lse, sum p |v|, sum |v| / l) by definition.  Unseen
    keys and values take no part, whatever they hold."""
    import torch
    q, k, v = q.double(), k.double(), v.double()
    any_row = seen.any(0)
    k = torch.where(any_row[:, None], k, 0.0)
    s = (q @ k.T) * scale
    s = torch.where(seen, s, -math.inf)
    m = s.amax(-1, keepdim=True) if s.shape[1] else torch.full((s.shape[0], 1), -math.inf, device=s.device).double()
    m = torch.where(torch.isinf(m), 0.0, m)
    e = torch.where(seen, (s - m).exp(), 0.0)
    l = e.sum(-1, keepdim=True)
    p = e / torch.where(l > 0, l, 1.0)
    out = torch.zeros_like(q)
    mag = torch.zeros_like(q)
    for r0 in range(0, q.shape[0], 512):  # values masked row by row
        sl = slice(r0, r0 + 512)
        if bool(torch.isfinite(v).all()):
            out[sl], mag[sl] = p[sl] @ v, p[sl] @ v.abs()
        else:
            vv = torch.where(seen[sl][:, :, None], v[None], 0.0)
            out[sl] = torch.einsum("nm,nmd->nd", p[sl], vv)
            mag[sl] = torch.einsum("nm,nmd->nd", p[sl], vv.abs())
    small = v.abs().nan_to_num(0, 0, 0).sum(0) / torch.where(l > 0, l, 1.0)
    return out, (m + l.log()).squeeze(-1), mag, small


def close(out, lse, ref, dtype):
    import torch
    want, want_lse, mag, small = ref
    tol = U[dtype] * want.abs() + (U[dtype] + 3e-5) * mag + 1e-30
    if dtype == "f16":
        tol = tol + 2.0 ** -25 * small
    bad = ~((out.double() - want).abs() <= tol) & ~(torch.isnan(want) & torch.isnan(out))
    assert not bool(bad.any()), (int(bad.sum()), float(((out.double() - want).abs() / tol).nan_to_num(0).max()))
    fin = torch.isfinite(want_lse)
    assert bool((torch.isfinite(lse) == fin).all()) and bool((lse[~fin] == want_lse[~fin].float()).all())
    assert float((lse.double() - want_lse)[fin].abs().max() if bool(fin.any()) else 0.0) <= 3e-5


def stored64(x, fmt):
    """(codes, scales) of rows x by the formula, with the scale in 64 bits rounded to FP32 and BF16."""
    import torch
    top, group = (127.0, x.shape[-1]) if fmt == "int8" else (7.0, 32)
    y = x.double().reshape(*x.shape[:-1], -1, group)
    s = (y.abs().amax(-1, keepdim=True) / top).float().bfloat16()
    ratio = torch.where(s > 0, y / s.double(), 0.0)
    return ratio.reshape(x.shape), ratio.round().clamp(-top, top).reshape(x.shape), s.squeeze(-1)


def codes_of(cache, name):
    """The integer codes of every row of a quantised pool, [pages, heads, page, dim]."""
    import torch
    raw = getattr(cache, name)
    if cache.format == "int8":
        return raw.double()
    return torch.stack([raw & 15, raw >> 4], -1).flatten(-2).double() - 8


# ---- packed prompts --------------------------------------------------------------------------

def starts_of(lengths):
    import torch
    return torch.tensor([0] + list(np.cumsum(lengths)), dtype=torch.int32, device="cuda")


def check_prompt(q, k, v, nq, nk, causal, dtype, scale=None, seqs=None, **kw):
    import torch
    from bgtq import prompt_attention
    starts, kst = starts_of(nq), starts_of(nk)
    out, lse = prompt_attention(q, k, v, starts, None if nq == nk else kst, causal=causal, scale=scale, lse=True, **kw)
    sc = 1.0 / math.sqrt(q.shape[2]) if scale is None else scale
    group = q.shape[1] // k.shape[1]
    for s in range(len(nq)) if seqs is None else seqs:
        a, b = int(starts[s]), int(kst[s])
        n, m = nq[s], nk[s]
        if n == 0:
            continue
        i, j = torch.arange(n, device="cuda")[:, None], torch.arange(m, device="cuda")[None]
        seen = (j <= i + (m - n)) if causal else torch.ones((n, m), dtype=torch.bool, device="cuda")
        for h in sorted({0, q.shape[1] // 2, q.shape[1] - 1}):
            ref = attention64(q[a:a + n, h], k[b:b + m, h // group], v[b:b + m, h // group], seen, sc)
            close(out[a:a + n, h], lse[a:a + n, h], ref, dtype)
    return out, lse


LENGTHS = {"one": [1], "edges": [1, 2, 127, 128, 129, 3], "empty": [0, 5, 0, 130, 0], "ragged": [300, 17, 700, 64, 255],
           "long": [1500]}


@pytest.mark.parametrize("lengths", sorted(LENGTHS))
@pytest.mark.parametrize("dtype,dim,hq,hk", [("f16", 64, 9, 3), ("bf16", 64, 14, 2), ("bf16", 128, 8, 2), ("f16", 128, 5, 5)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_matches_the_formula(cuda, lengths, dtype, dim, hq, hk, causal):
    n = LENGTHS[lengths]
    q = randn(1, sum(n), hq, dim, dtype=dtype, spread=1.5)
    k, v = (randn(s, sum(n), hk, dim, dtype=dtype, spread=1.2) for s in (2, 3))
    check_prompt(q, k, v, n, n, causal, dtype)
    assert device_status(0) == 0


@pytest.mark.parametrize("hq,hk", [(1, 1), (16, 1), (33, 1), (128, 1), (40, 8), (6, 2)])
def test_prompt_head_groups(cuda, hq, hk):
    n = [70, 1, 200]
    q, k, v = randn(1, 271, hq, 64, dtype="bf16"), randn(2, 271, hk, 64, dtype="bf16"), randn(3, 271, hk, 64, dtype="bf16")
    check_prompt(q, k, v, n, n, True, "bf16")


@pytest.mark.parametrize("dtype,dim", [("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("nq,nk", [([5, 64, 1, 130], [300, 64, 513, 131]),    # cached prefixes
                                   ([40, 300, 9, 7], [10, 172, 0, 7])])          # rows that see nothing
def test_prompt_with_other_keys_than_queries(cuda, dtype, dim, causal, nq, nk):
    q = randn(4, sum(nq), 6, dim, dtype=dtype)
    k, v = (randn(s, sum(nk), 2, dim, dtype=dtype) for s in (5, 6))
    out, lse = check_prompt(q, k, v, nq, nk, causal, dtype)
    if causal and nk[0] == 10:
        assert not out[:30].any() and bool((lse[:30] == -math.inf).all())


def test_prompt_few_rows_over_long_keys(cuda):
    nq, nk = [1, 16, 3], [9001, 4096, 12345]
    q = randn(4, sum(nq), 8, 128, dtype="f16")
    k, v = (randn(s, sum(nk), 2, 128, dtype="f16") for s in (5, 6))
    check_prompt(q, k, v, nq, nk, True, "f16")


def test_prompt_without_any_key(cuda):
    import torch
    from bgtq import prompt_attention
    q = randn(1, 7, 4, 64, dtype="f16")
    k = torch.empty((0, 2, 64), dtype=torch.float16, device="cuda")
    out, lse = prompt_attention(q, k, k, starts_of([3, 4]), starts_of([0, 0]), lse=True)
    assert not out.any() and bool((lse == -math.inf).all())
    assert prompt_attention(q[:0], k, k, starts_of([0, 0])).shape == (0, 4, 64)


def test_prompt_strides_and_alignment(cuda):
    """Columns of one fused projection, head-major storage, an address off by one element, a broadcast
    key: the same numbers as their packed copies."""
    import torch
    from bgtq import prompt_attention
    n, hq, hk, d = [100, 61], 6, 2, 64
    T = sum(n)
    qkv = randn(7, T, (hq + 2 * hk) * d, dtype="bf16")
    q, k, v = (qkv[:, a:b].unflatten(1, (-1, d)) for a, b in ((0, 384), (384, 512), (512, 640)))
    want = prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), starts_of(n))
    assert torch.equal(prompt_attention(q, k, v, starts_of(n)), want)
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(prompt_attention(*turned, starts_of(n)), want)
    off = torch.empty(T * hk * d + 1, dtype=torch.bfloat16, device="cuda")[1:].view(T, hk, d)
    off.copy_(k)
    assert torch.equal(prompt_attention(q, off, v, starts_of(n)), want)
    one = k[:, :1].expand(T, hk, d)
    assert torch.equal(prompt_attention(q, one, v, starts_of(n)), prompt_attention(q, one.contiguous(), v, starts_of(n)))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_prompt_what_a_row_does_not_see_does_not_reach_it(cuda, dim, bad):
    """Infinities and NaN in one sequence's keys, values and queries leave the others as they were,
    and in a later position of a causal sequence leave its earlier rows as they were."""
    import torch
    from bgtq import prompt_attention
    n = [150, 131, 90]
    q = randn(1, sum(n), 4, dim, dtype="bf16")
    k, v = (randn(s, sum(n), 2, dim, dtype="bf16") for s in (2, 3))
    want, want_lse = prompt_attention(q, k, v, starts_of(n), lse=True)
    q2, k2, v2 = q.clone(), k.clone(), v.clone()
    at = n[0] + 77
    for t in (q2, k2, v2):
        t[at:n[0] + n[1], ..., 3] = bad
    out, lse = prompt_attention(q2, k2, v2, starts_of(n), lse=True)
    keep = torch.ones(sum(n), dtype=torch.bool, device="cuda")
    keep[at:n[0] + n[1]] = False
    assert torch.equal(out[keep], want[keep]) and torch.equal(lse[keep], want_lse[keep])
    # a value seen by its own and later rows is an infinity or a NaN there, and only in its dimension
    v3 = v.clone()
    v3[at, :, 5] = bad
    out = prompt_attention(q, k, v3, starts_of(n))
    late = torch.zeros(sum(n), dtype=torch.bool, device="cuda")
    late[at:n[0] + n[1]] = True
    assert torch.equal(out[~late], want[~late])
    rest = [i for i in range(dim) if i != 5]
    assert torch.equal(out[late][..., rest], want[late][..., rest])
    hit = out[late][..., 5].float()
    assert bool(torch.isnan(hit).all()) if math.isnan(bad) else bool((hit == bad).all())


def test_prompt_large_logits_and_scale(cuda):
    n = [200]
    q = randn(1, 200, 2, 64, dtype="bf16", spread=6.0)
    k, v = randn(2, 200, 1, 64, dtype="bf16", spread=1.0), randn(3, 200, 1, 64, dtype="bf16")
    check_prompt(q, k, v, n, n, True, "bf16", scale=0.15)
    check_prompt(q, k * -1, v, n, n, True, "bf16", scale=0.01)


def test_prompt_rising_maximum(cuda):
    """Logits that climb along the keys, so that the running maximum moves in every tile."""
    import torch
    n = 900
    q = torch.ones((n, 2, 64), device="cuda", dtype=torch.float16)
    ramp = torch.linspace(-6, 6, n, device="cuda").half()
    k = (ramp[:, None, None] * torch.ones((1, 2, 64), device="cuda")).half()
    v = randn(3, n, 2, 64, dtype="f16")
    check_prompt(q, k, v, [n], [n], True, "f16")
    check_prompt(q, k.flip(0).contiguous(), v, [n], [n], False, "f16")


def test_prompt_other_stream_and_repeat(cuda):
    import torch
    from bgtq import prompt_attention
    n = [333, 512]
    q, k, v = randn(1, 845, 8, 128, dtype="f16"), randn(2, 845, 2, 128, dtype="f16"), randn(3, 845, 2, 128, dtype="f16")
    want = prompt_attention(q, k, v, starts_of(n))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = [prompt_attention(q, k, v, starts_of(n)) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_prompt_in_a_graph(cuda):
    import torch
    from bgtq import prompt_attention
    n = [40, 90]
    q, k, v = randn(1, 130, 3, 64, dtype="bf16"), randn(2, 130, 1, 64, dtype="bf16"), randn(3, 130, 1, 64, dtype="bf16")
    st = starts_of(n)
    out = torch.empty_like(q)
    prompt_attention(q, k, v, st, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        prompt_attention(q, k, v, st, out=out)
    q.copy_(randn(9, 130, 3, 64, dtype="bf16"))
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, prompt_attention(q, k, v, st))


@pytest.mark.parametrize("dtype,dim,hq,hk", [("f16", 64, 14, 2), ("bf16", 128, 4, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_items_done_in_parts(cuda, dtype, dim, hq, hk, causal):
    """Few items over long keys: several CTAs have keys of one, and the last of them joins."""
    nq, nk = [5, 200, 0, 700], [5003, 1300, 64, 3001]
    q = randn(4, sum(nq), hq, dim, dtype=dtype)
    k, v = (randn(s, sum(nk), hk, dim, dtype=dtype) for s in (5, 6))
    check_prompt(q, k, v, nq, nk, causal, dtype)


@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_prompt_parts_with_values_not_every_row_sees(cuda, bad):
    """Infinities and NaN in the last keys of a long item: they reach the rows that see them, from
    whichever part holds them, and no others."""
    import torch
    n, m = 70, 4000
    q = randn(1, n, 4, 64, dtype="f16")
    k, v = (randn(s, m, 1, 64, dtype="f16") for s in (2, 3))
    clean, _ = check_prompt(q, k, v, [n], [m], True, "f16")
    v[m - 30, 0, 7] = bad
    k[m - 1, 0, 0] = math.nan          # the last row alone sees it
    from bgtq import prompt_attention
    out = prompt_attention(q, k, v, starts_of([n]), starts_of([m]))
    sees = torch.arange(n, device="cuda") >= n - 30
    want = clean.clone()
    want[sees, :, 7] = bad
    want[n - 1] = math.nan
    assert torch.equal(out.nan_to_num(nan=7.0, posinf=8.0), want.nan_to_num(nan=7.0, posinf=8.0))


def test_prompt_many_sequences_and_one_long(cuda):
    rng = np.random.default_rng(3)
    n = [int(x) for x in rng.integers(0, 60, 70)] + [2500] + [int(x) for x in rng.integers(0, 9, 20)]
    q = randn(4, sum(n), 6, 64, dtype="bf16")
    k, v = (randn(s, sum(n), 2, 64, dtype="bf16") for s in (5, 6))
    check_prompt(q, k, v, n, n, True, "bf16", seqs=[0, 3, 31, 32, 33, 69, 70, 71, 90])


@pytest.mark.parametrize("dim,hq,hk", [(64, 14, 2), (128, 8, 2)])
def test_prompt_repeated_over_changing_lengths(cuda, dim, hq, hk):
    """Calls that follow each other without a pause, items whole and in parts in turn, give the bits
    of a call alone."""
    import torch
    from bgtq import device_status, prompt_attention
    lengths = [[1, 700, 33, 257], [2100], [64] * 40, [5, 1025, 900]]
    calls = []
    for i, n in enumerate(lengths):
        q = randn(10 + i, sum(n), hq, dim, dtype="f16")
        k, v = (randn(s + i, sum(n), hk, dim, dtype="f16") for s in (20, 30))
        calls.append((q, k, v, starts_of(n)))
    want = []
    for c in calls:
        want.append(prompt_attention(*c))
        torch.cuda.synchronize()
    got = [prompt_attention(*calls[i % 4]) for i in range(80)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 4]) for i, g in enumerate(got)) and device_status() == 0


# ---- the paged cache --------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", ["f16", "bf16", "int8", "int4"])
@pytest.mark.parametrize("source", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("dim,heads,page,n", [(64, 3, 16, 1), (64, 3, 16, 37), (128, 2, 64, 200), (128, 1, 256, 513)])
def test_cache_write_stores_the_formula_and_read_gives_it_back(cuda, fmt, source, dim, heads, page, n):
    import torch
    from bgtq import PagedCache
    pages = (n + page - 1) // page + 2
    cache = PagedCache(heads, dim, pages, page, fmt)
    k, v = randn(1, n, heads, dim, dtype=source, spread=3.0), randn(2, n, heads, dim, dtype=source, spread=0.02)
    g = torch.Generator(device="cuda").manual_seed(3)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:n]
    slots = torch.where(torch.arange(n, device="cuda") % 5 == 4, -1, slots)
    cache.write(k, v, slots)
    live = slots >= 0
    pg, row = slots.clamp(min=0) // page, slots.clamp(min=0) % page
    free = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    free[slots[live]] = False
    for name, x in (("k", k), ("v", v)):
        pool = getattr(cache, name)
        spare = pool.transpose(1, 2).flatten(0, 1)[free]
        assert not spare.any(), "a row that no slot names was written"
        if fmt in ("f16", "bf16"):
            assert torch.equal(pool[pg, :, row][live], x.float().to(types()[fmt])[live])
            continue
        ratio, want, scale = stored64(x, fmt)
        got = codes_of(cache, name)[pg, :, row]
        assert torch.equal(getattr(cache, name + "_scales")[pg, :, row][live], scale[live])
        diff = (got - want)[live].abs()
        tie = ((ratio - ratio.floor() - 0.5).abs() <= ratio.abs() * 2.0 ** -23)[live]
        assert not bool((diff[~tie] != 0).any()) and float(diff.max() if diff.numel() else 0) <= 1
    for dtype in ("f16", "bf16", "f32"):
        rk, rv = cache.read(slots, dtype=types()[dtype])
        for name, r in (("k", rk), ("v", rv)):
            if fmt in ("f16", "bf16"):
                want = getattr(cache, name)[pg, :, row].float()
            else:
                sc = getattr(cache, name + "_scales")[pg, :, row].float()
                want = codes_of(cache, name)[pg, :, row].float() * sc.repeat_interleave(dim // sc.shape[-1], -1)
            want = torch.where(live[:, None, None], want, 0.0).to(types()[dtype])
            assert torch.equal(r, want)
    assert device_status(0) == 0


def test_cache_strided_sources_and_rewriting(cuda):
    import torch
    from bgtq import PagedCache
    n, H, d = 50, 3, 64
    qkv = randn(1, n, 11 * d + 1, dtype="f32")
    views = [(qkv[:, 2 * d:5 * d].unflatten(1, (H, d)), qkv[:, 5 * d:8 * d].unflatten(1, (H, d))),
             (qkv[:, 1:3 * d + 1].unflatten(1, (H, d)), qkv[:, 3 * d + 1:6 * d + 1].unflatten(1, (H, d)))]
    half = qkv.half()
    views += [(half[:, 1:3 * d + 1].unflatten(1, (H, d)), half[:, 4 * d:7 * d].unflatten(1, (H, d)))]
    views += [(half[:, :d].unflatten(1, (1, d)).expand(n, H, d), half[:, d:4 * d].unflatten(1, (H, d)))]
    views += [(randn(5, H, n, d, dtype="bf16").transpose(0, 1), randn(6, n, H, d, dtype="bf16"))]
    for fmt in ("int8", "int4", "bf16"):
        a, b = PagedCache(H, d, 8, 16, fmt), PagedCache(H, d, 8, 16, fmt)
        slots = torch.randperm(128, device="cuda")[:n]
        for k, v in views:
            a.write(k, v, slots)
            b.write(k.contiguous(), v.contiguous(), slots)
            assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
            assert a.k_scales is None or (torch.equal(a.k_scales, b.k_scales) and torch.equal(a.v_scales, b.v_scales))


def test_cache_special_values(cuda):
    """Zero rows, tiny and huge values, infinities and NaN: the group that holds one reads back as
    NaN, its neighbours are untouched."""
    import torch
    from bgtq import PagedCache
    for fmt, group in (("int8", 64), ("int4", 32)):
        x = randn(1, 9, 1, 64, dtype="f32")
        x[0] = 0
        x[1] *= 1e-42
        x[2] *= 1e30
        x[3, 0, 5] = math.nan
        x[4, 0, 40] = math.inf
        x[5, 0, 63] = -math.inf
        x[6, 0, :32] = 0
        x[7] = 3.0e38
        cache = PagedCache(1, 64, 1, 16, fmt)
        slots = torch.arange(9, device="cuda")
        cache.write(x, -x, slots)
        k, v = cache.read(slots, dtype=torch.float32)
        assert torch.equal(v.nan_to_num(7.0), (-k).nan_to_num(7.0))
        broken = ~torch.isfinite(x).reshape(9, -1, group).all(-1)
        assert torch.equal(torch.isnan(k).reshape(9, -1, group).all(-1), broken)
        assert torch.equal(torch.isnan(k).reshape(9, -1, group).any(-1), broken)
        assert not k[0].any() and not k[6, 0, :32].any()
        top = 127.0 if fmt == "int8" else 7.0
        y, z = x.reshape(9, -1, group), k.reshape(9, -1, group)
        for r in (2, 6, 7, 8):  # half a step, and a step's share for a scale rounded down by 2^-9
            step = y[r].abs().amax(-1, keepdim=True) / top
            assert bool(((y[r] - z[r]).abs() <= step * (0.5 + 2.0 ** -8 * top)).all())


def test_cache_nothing_to_do(cuda):
    import torch
    from bgtq import PagedCache
    cache = PagedCache(2, 64, 2, 16, "int8")
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    k = torch.empty((0, 2, 64), dtype=torch.float16, device="cuda")
    cache.write(k, k, none)
    assert cache.read(none)[0].shape == (0, 2, 64)
    assert cache.attend(torch.empty((0, 4, 64), dtype=torch.float16, device="cuda"),
                        torch.empty((0, 2), dtype=torch.int32, device="cuda"),
                        torch.empty(0, dtype=torch.int32, device="cuda")).shape == (0, 4, 64)


# ---- one token over the pages ------------------------------------------------------------------

def paged(seed, lengths, heads, dim, page, fmt, spread=1.0, extra=3):
    """A cache of random rows, its page table and lengths; unused rows and pages hold NaN."""
    import torch
    from bgtq import PagedCache
    need = [(n + page - 1) // page for n in lengths]
    pages, width = sum(need) + extra, max(max(need), 1)
    cache = PagedCache(heads, dim, pages, page, fmt)
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).tolist()
    table = np.full((len(lengths), width), 2**31 - 1, np.int64)  # entries past a length are not read
    used = torch.zeros((pages, page), dtype=torch.bool)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
        for t in range(0, lengths[b], page):
            used[int(table[b, t // page]), :min(page, lengths[b] - t)] = True
    slots = torch.nonzero(used.flatten()).flatten().cuda()
    k, v = randn(seed, len(slots), heads, dim, spread=spread), randn(seed + 1, len(slots), heads, dim)
    cache.write(k, v, slots)
    unused = ~used.cuda()
    if fmt in ("f16", "bf16"):
        for pool in (cache.k, cache.v):
            pool.transpose(1, 2)[unused] = math.nan
    else:
        for sc in (cache.k_scales, cache.v_scales):
            sc.transpose(1, 2)[unused] = math.nan
    return cache, torch.tensor(table, dtype=torch.int32).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()


def check_token(cache, q, table, lengths, dtype, scale=None, **kw):
    import torch
    out, lse = cache.attend(q, table, lengths, scale=scale, lse=True, **kw)
    sc = 1.0 / math.sqrt(cache.dim) if scale is None else scale
    group = q.shape[1] // cache.kv_heads
    ps = cache.page_size
    for b, n in enumerate(lengths.tolist()):
        t = torch.arange(n, device="cuda")
        slots = table[b].long()[t // ps] * ps + t % ps
        k, v = cache.read(slots, dtype=torch.float32)
        seen = torch.ones((group, n), dtype=torch.bool, device="cuda")
        for h in sorted({0, cache.kv_heads - 1}):
            rows = slice(h * group, (h + 1) * group)
            close(out[b, rows], lse[b, rows], attention64(q[b, rows], k[:, h], v[:, h], seen, sc), dtype)
    return out, lse


FORMATS = [("f16", "f16"), ("bf16", "bf16"), ("int8", "f16"), ("int8", "bf16"), ("int4", "f16"), ("int4", "bf16")]


@pytest.mark.parametrize("fmt,dtype", FORMATS)
@pytest.mark.parametrize("dim,hq,hk", [(64, 9, 3), (128, 8, 2), (64, 14, 2), (128, 5, 5)])
@pytest.mark.parametrize("page", [16, 64])
def test_token_matches_the_formula(cuda, fmt, dtype, dim, hq, hk, page):
    lengths = [1, 0, 15, 16, 17, 63, 64, 65, 129, 1000, 0, 2]
    cache, table, lens = paged(10, lengths, hk, dim, page, fmt)
    q = randn(3, len(lengths), hq, dim, dtype=dtype, spread=1.5)
    out, lse = check_token(cache, q, table, lens, dtype)
    assert not out[1].any() and bool((lse[10] == -math.inf).all())
    assert device_status(0) == 0


@pytest.mark.parametrize("fmt,dtype", FORMATS)
@pytest.mark.parametrize("lengths", [[20000], [9000, 1, 300], [5000, 4999, 5001, 0, 5003]])
def test_token_long_requests_are_split_and_joined(cuda, fmt, dtype, lengths):
    cache, table, lens = paged(20, lengths, 2, 64, 32, fmt)
    q = randn(3, len(lengths), 6, 64, dtype=dtype)
    check_token(cache, q, table, lens, dtype)


@pytest.mark.parametrize("fmt,dtype", [("f16", "f16"), ("int8", "bf16"), ("int4", "f16")])
@pytest.mark.parametrize("hq,hk", [(1, 1), (16, 1), (17, 1), (48, 2), (71, 1)])
def test_token_head_groups(cuda, fmt, dtype, hq, hk):
    cache, table, lens = paged(30, [700, 33], hk, 128, 128, fmt)
    check_token(cache, randn(3, 2, hq, 128, dtype=dtype), table, lens, dtype)


@pytest.mark.parametrize("page", [16, 32, 128, 256])
def test_token_many_requests(cuda, page):
    rng = np.random.default_rng(5)
    lengths = rng.integers(0, 600, 150).tolist()
    cache, table, lens = paged(40, lengths, 2, 64, page, "int8")
    check_token(cache, randn(3, 150, 8, 64, dtype="bf16"), table, lens, "bf16")


@pytest.mark.parametrize("fmt", ["f16", "int8", "int4"])
def test_token_rising_maximum_and_large_logits(cuda, fmt):
    import torch
    from bgtq import PagedCache
    n = 3000
    cache = PagedCache(1, 64, 200, 16, fmt)
    ramp = torch.linspace(-4, 4, n, device="cuda")
    k = ramp[:, None, None] * torch.ones((1, 1, 64), device="cuda")
    table = torch.arange(200, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    q = torch.ones((1, 2, 64), device="cuda", dtype=torch.float16)
    for keys in (k, k.flip(0)):
        cache.write(keys, randn(1, n, 1, 64), torch.arange(n, device="cuda"))
        check_token(cache, q, table, lens, "f16")


@pytest.mark.parametrize("fmt", ["int8", "int4"])
def test_token_tiny_and_huge_value_scales(cuda, fmt):
    """Value rows of very different size: the scales span BF16's range, not FP16's."""
    import torch
    from bgtq import PagedCache
    n = 500
    cache = PagedCache(1, 64, 40, 16, fmt)
    size = torch.logspace(-20, 3, n, device="cuda")[:, None, None]
    cache.write(randn(1, n, 1, 64), randn(2, n, 1, 64) * size, torch.arange(n, device="cuda"))
    table = torch.arange(40, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    check_token(cache, randn(3, 1, 3, 64, dtype="bf16"), table, lens, "bf16")


def test_token_strided_queries_tables_and_streams(cuda):
    import torch
    lengths = [100, 900, 5, 1500]
    cache, table, lens = paged(50, lengths, 2, 64, 16, "f16")
    qkv = randn(3, 4, 10 * 64 + 1, dtype="f16")
    q = qkv[:, 1:6 * 64 + 1].unflatten(1, (6, 64))
    want = cache.attend(q.contiguous(), table, lens)
    wide = torch.full((4, table.shape[1] + 9), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    assert torch.equal(cache.attend(q, wide[:, :table.shape[1]], lens), want)
    assert torch.equal(cache.attend(q, wide, lens), want)
    st = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in st:
            with torch.cuda.stream(s):
                got.append(cache.attend(q, table, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_token_in_a_graph_while_requests_grow(cuda):
    import torch
    from bgtq import PagedCache
    cache = PagedCache(1, 64, 64, 16, "int8")
    table = torch.arange(64, dtype=torch.int32, device="cuda").view(2, 32)
    lens = torch.tensor([3, 100], dtype=torch.int32, device="cuda")
    t = torch.arange(1024, device="cuda")
    cache.write(randn(1, 1024, 1, 64), randn(2, 1024, 1, 64), t)
    q = randn(3, 2, 4, 64, dtype="bf16")
    out = torch.empty_like(q)
    cache.attend(q, table, lens, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.attend(q, table, lens, out=out)
    for a, b in ((4, 101), (500, 512), (0, 1)):
        lens.copy_(torch.tensor([a, b], dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, cache.attend(q, table, lens))


def test_token_offsets_past_32_bits(cuda):
    """Pages that begin more than 2^32 bytes, and 2^31 elements, into the pool."""
    import torch
    from bgtq import PagedCache
    pages = (2**32 // (256 * 8 * 128 * 2)) + 8
    cache = PagedCache(8, 128, pages, 256, "f16")
    slots = torch.arange((pages - 4) * 256, (pages - 4) * 256 + 700, device="cuda")
    k, v = randn(1, 700, 8, 128, dtype="f16"), randn(2, 700, 8, 128, dtype="f16")
    cache.write(k, v, slots)
    rk, rv = cache.read(slots)
    assert torch.equal(rk, k) and torch.equal(rv, v)
    table = torch.arange(pages - 4, pages - 1, dtype=torch.int32, device="cuda")[None].contiguous()
    check_token(cache, randn(3, 1, 16, 128, dtype="f16"), table, torch.tensor([700], dtype=torch.int32, device="cuda"), "f16")


# ---- indices that only the GPU sees -------------------------------------------------------------

def test_indices_outside_the_cache_are_left_out_and_reported(cuda):
    """In a process of its own: the device status word keeps its bits."""
    code = '''
import math, torch, bgtq
from bgtq import PagedCache, prompt_attention, device_status
dev = "cuda"
i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
c = PagedCache(2, 64, 4, 16, "int8")
x = torch.randn(3, 2, 64, device=dev)
c.write(x, x, torch.tensor([5, 64, 2**40], device=dev))
assert device_status(0) == 4
k, v = c.read(torch.tensor([5, 64, -1], device=dev))
assert k[0].any() and not k[1:].any() and not v[1:].any()
c = PagedCache(1, 64, 4, 16, "f16")
y = torch.randn(64, 1, 64, device=dev).half()
c.write(y, y, torch.arange(64, device=dev))
q = torch.randn(2, 2, 64, device=dev).half()
a = c.attend(q, i32(0, 1, 3).view(1, 3).expand(2, 3), i32(40, 16))
b = c.attend(q, torch.stack([i32(0, 9999, 3), i32(0, -5, 7)]), i32(40, 48))
w = torch.cat([y[0:16], y[48:56]])
p = torch.softmax((q[0].float() @ w[:, 0].float().T) / 8, -1) @ w[:, 0].float()
assert (b[0] - p).abs().max() < 4e-3 and (a[1] - b[1]).abs().max() < 4e-3
assert device_status(0) == 4
o, l = c.attend(q, i32(0, 1, 2, 3).view(2, 2), i32(1000, -3), lse=True)
full = c.attend(q, i32(0, 1, 2, 3).view(2, 2), i32(32, 0))
assert torch.equal(o, full) and device_status(0) == 12
t = torch.randn(20, 2, 64, device=dev).half()
o = torch.full_like(t, 7.0)
prompt_attention(t, t, t, i32(0, 5, 3, 30, 30), out=o)
want = prompt_attention(t[:5], t[:5], t[:5], i32(0, 5))
assert torch.equal(o[:5], want) and not torch.isnan(o).any()
assert device_status(0) == 12
print("fine")
'''
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       cwd=ROOT / "block-gqt-webgpu_b200")
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr


def test_python_refusals_on_the_device(cuda):
    import ctypes as C
    import torch
    from bgtq import PagedCache, prompt_attention
    c = PagedCache(2, 64, 4, 16, "f16")
    x = randn(1, 3, 2, 64, dtype="f16")
    slots = torch.arange(3, device="cuda")
    for k, v, s, message in [(x, x, slots.int(), "int64"), (x, x, slots.cpu(), "cache's device"), (x, x, slots[:2], "one slot"),
                             (x, x.float(), slots, "both be"), (x, x.cpu(), slots, "device"), (x.long(), x.long(), slots, "both be"),
                             (x.transpose(0, 2).contiguous().transpose(0, 2), x, slots, "contiguous")]:
        with pytest.raises(_lib.RangeError, match=message):
            c.write(k, v, s)
    with pytest.raises(_lib.RangeError, match="dtype"):
        c.read(slots, torch.float64)
    q = randn(1, 2, 4, 64, dtype="f16")
    table, lengths = torch.zeros((2, 2), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for args, message in [((q[:, :3], table, lengths), "multiple"), ((q.bfloat16(), table, lengths), "16-bit pages"),
                          ((q, table.long(), lengths), "table"), ((q, table[:1], lengths), "table"),
                          ((q, table, lengths.long()), "lengths"), ((q, table, lengths.cpu()), "lengths"),
                          ((q.cpu(), table, lengths), "device"), ((q, table, lengths, -1.0), "scale"),
                          ((q, table, lengths, None, q.float()), "out")]:
        with pytest.raises(_lib.RangeError, match=message):
            c.attend(*args)
    st = starts_of([2])
    k = randn(2, 2, 2, 64, dtype="f16")
    for args, message in [((q, k, k, st.long()), "starts"), ((q, k.bfloat16(), k, st), "float16"), ((q, k[:1], k[:1], st), "key_starts"),
                          ((q, k, k, st, starts_of([1, 1])), "starts"), ((q[:, :3], k, k, st), "multiple")]:
        with pytest.raises(_lib.RangeError, match=message):
            prompt_attention(*args)
    # a workspace that is too small, or none
    need = C.c_size_t()
    _lib.call("bgtq_prompt_workspace", 0, 64, C.byref(need))
    room = torch.zeros(need.value + 128, dtype=torch.uint8, device="cuda")
    for address, size in ((None, need.value), (room.data_ptr(), need.value - 1), (room.data_ptr() + 4, need.value)):
        p = _lib.PromptDesc(0, _lib.F16, 1, 4, 2, 64, 2, 2, q.data_ptr(), k.data_ptr(), k.data_ptr(), 256, 64, 128, 64, 128, 64,
                            st.data_ptr(), None, 1, 0.0, torch.empty_like(q).data_ptr(), None, address, size)
        with pytest.raises(_lib.RangeError, match="workspace"):
            _lib.call("bgtq_prompt_attend", C.byref(p), None)


def test_first_call_of_a_stream_inside_a_recording(cuda):
    """The graph has a workspace of its own; a call on that stream before any replay has another."""
    import torch
    from bgtq import PagedCache, prompt_attention
    c = PagedCache(2, 64, 300, 16, "int8")
    n = 4000
    slots = torch.arange(n, device="cuda")
    k, v = randn(1, n, 2, 64, dtype="f16"), randn(2, n, 2, 64, dtype="f16")
    c.write(k, v, slots)
    table = torch.arange(300, dtype=torch.int32, device="cuda")[None]
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    q1, q2 = randn(3, 1, 14, 64, dtype="f16"), randn(4, 16, 14, 64, dtype="f16")
    st, ks = starts_of([16]), starts_of([n])
    want = c.attend(q1, table, lengths), prompt_attention(q2, k, v, st, ks)   # in several parts, both
    out = torch.zeros_like(want[0]), torch.zeros_like(want[1])
    torch.cuda.synchronize()
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        c.attend(q1, table, lengths, out=out[0])
        prompt_attention(q2, k, v, st, ks, out=out[1])
    with torch.cuda.stream(side):
        got = c.attend(q1, table, lengths), prompt_attention(q2, k, v, st, ks)
        for _ in range(3):
            g.replay()
    torch.cuda.synchronize()
    for a, b, w in zip(got, out, want):
        assert torch.equal(a, w) and torch.equal(b, w)
