"""The serving operators for requests of different lengths, in cases of real sizes.

Three operators that belong together: prompts of different lengths are attended as one
packed batch (`bgtq.prompt_attention`), their keys and values are quantised into the pages of
a shared cache and read back for a later chunk (`bgtq.PagedCache.write` / `.read`), and every
new token attends over its own pages (`bgtq.PagedCache.attend`).

    listed(), draw(rng)    the cases: dicts of plain values
    prepare(case, seed)    what a server has in hand before the call
    run(state)             one pass; `own` chooses the library's kernels or the plain form
    work(case)             bytes and operations that the pass cannot do without
    exact(case, seed)      the result by definition, in 64 bits
"""
import math

import torch

own = False  # False: elementary torch operations in 32 bits; True: the library's entry points

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
GROUP = 32  # dimensions that share one scale in a 4-bit row


# ---- the cases -------------------------------------------------------------------------

def listed():
    return [
        # --- writing a quantised cache and reading it back ---
        # one decode step of 16 requests, 3 KV heads of 64 (the small model's geometry): latency
        dict(name="cache-step", op="cache", tokens=16, kv_heads=3, dim=64, format="int8", source="f16", page=16,
             pad=0, fused=True),
        # a padded batch of FP32 projections of 2 KV heads: an odd token count, every 7th row is padding
        dict(name="cache-ragged", op="cache", tokens=4999, kv_heads=2, dim=64, format="int8", source="f32", page=16,
             pad=7, fused=True),
        # 16K prompt tokens of a wide layer into 4 bits: a bandwidth case
        dict(name="cache-prompt", op="cache", tokens=16384, kv_heads=8, dim=128, format="int4", source="bf16", page=64,
             pad=0, fused=False),
        # --- one new token per request over the pages ---
        # a single chat request with a 4096-token history, FP16 pages: latency, split over the length
        dict(name="token-single", op="token", batch=1, shortest=4096, longest=4096, q_heads=9, kv_heads=3, dim=64,
             format="f16", dtype="f16", page=16),
        # a mixed server batch, 1 to 8191 tokens, 8-bit pages, grouped heads of 128
        dict(name="token-ragged", op="token", batch=48, shortest=1, longest=8191, q_heads=32, kv_heads=8, dim=128,
             format="int8", dtype="bf16", page=64),
        # eight long documents in 4-bit pages, seven query heads per KV head
        dict(name="token-long", op="token", batch=8, shortest=20011, longest=32768, q_heads=14, kv_heads=2, dim=64,
             format="int4", dtype="f16", page=32),
        # a full machine: 128 requests of 16K to 32K tokens, 16-bit pages, 2.4 GB of cache
        dict(name="token-full", op="token", batch=128, shortest=16384, longest=32768, q_heads=9, kv_heads=3, dim=64,
             format="bf16", dtype="bf16", page=64),
        # --- prompts of different lengths in one packed batch ---
        # one short question: latency
        dict(name="prompt-short", op="prompt", batch=1, shortest=37, longest=37, prefix=0, q_heads=9, kv_heads=3,
             dim=64, dtype="f16", causal=True),
        # a dozen prompts of 1 to 2047 tokens
        dict(name="prompt-ragged", op="prompt", batch=12, shortest=1, longest=2047, prefix=0, q_heads=14, kv_heads=2,
             dim=64, dtype="bf16", causal=True),
        # chunks of three prompts whose earlier tokens are already cached: more keys than queries
        dict(name="prompt-chunk", op="prompt", batch=3, shortest=300, longest=512, prefix=3500, q_heads=32, kv_heads=8,
             dim=128, dtype="f16", causal=True),
        # two long documents, the 14 / 2 head geometry at 8192 positions
        dict(name="prompt-long", op="prompt", batch=2, shortest=8192, longest=8192, prefix=0, q_heads=14, kv_heads=2,
             dim=64, dtype="bf16", causal=True),
        # a prefill batch of a wide layer, 32 / 8 heads of 128
        dict(name="prompt-wide", op="prompt", batch=4, shortest=3500, longest=4096, prefix=0, q_heads=32, kv_heads=8,
             dim=128, dtype="bf16", causal=True),
    ]


def _log(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["cache", "token", "token", "prompt", "prompt"])
    dim = rng.choice([64, 128])
    kv = rng.choice([1, 2, 3, 4, 8])
    if op == "cache":
        tokens = min(_log(rng, 1, 16384), 16384 * 8 * 128 // (kv * dim))
        return dict(op=op, tokens=tokens, kv_heads=kv, dim=dim, format=rng.choice(["f16", "bf16", "int8", "int4"]),
                    source=rng.choice(["f16", "bf16", "f32"]), page=rng.choice([16, 32, 64, 128]),
                    pad=rng.choice([0, 0, 5, 13]), fused=rng.random() < 0.5)
    group = rng.choice([1, 2, 3, 4, 7, 8])
    dtype = rng.choice(["f16", "bf16"])
    if op == "token":
        batch = _log(rng, 1, 128)
        most = min(32768, int(128 * 24576 * 3 * 64 / (batch * kv * dim)))
        longest = _log(rng, 1, most)
        return dict(op=op, batch=batch, shortest=_log(rng, 1, longest), longest=longest, q_heads=kv * group,
                    kv_heads=kv, dim=dim, format=rng.choice([dtype, "int8", "int4"]), dtype=dtype,
                    page=rng.choice([16, 32, 64, 128]))
    batch = _log(rng, 1, 24)
    most = int(min(8192, math.sqrt(4 * 32 * 4096 * 4096 / (batch * kv * group * (dim / 64)))))
    longest = _log(rng, 1, most)
    prefix = 0 if rng.random() < 0.6 else _log(rng, 1, max(1, most - longest))
    return dict(op=op, batch=batch, shortest=_log(rng, 1, longest), longest=longest,
                prefix=prefix if longest + prefix <= most else 0, q_heads=kv * group, kv_heads=kv, dim=dim,
                dtype=dtype, causal=rng.random() < 0.8)


def lengths_of(case):
    """Every request's length: from the shortest to the longest on a logarithmic scale, in a mixed order."""
    b, low, high = case["batch"], case["shortest"], case["longest"]
    if b == 1:
        return [high]
    order = sorted(range(b), key=lambda i: (i * 7919 + 3) % 10007)
    return [int(round(low * (high / low) ** (i / (b - 1)))) for i in order]


def prefixes_of(case):
    """Keys that come before each prompt's own tokens: the prefix, less a different remainder for each prompt."""
    return [max(0, case["prefix"] - 37 * i) for i in range(case["batch"])]


# ---- what a server has in hand ------------------------------------------------------------

def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _spread(dim):
    """Standard deviations of a post-RoPE key's dimensions: the low-frequency pairs dominate."""
    pair = torch.arange(dim // 2, device="cuda", dtype=torch.float32)
    sigma = 0.5 + 3.0 * torch.exp(-(dim // 2 - 1 - pair) / (0.08 * dim))
    return torch.cat([sigma, sigma])


def _quantise(x, fmt):
    """Codes and scales of FP32 rows x [..., dim]: symmetric, one BF16 scale a row (8 bits) or for
    every 32 dimensions (4 bits, two to a byte, the even dimension in the low nibble)."""
    top, group = (127, x.shape[-1]) if fmt == "int8" else (7, GROUP)
    g = x.unflatten(-1, (-1, group))
    scale = (g.abs().amax(-1) / top).to(torch.bfloat16)
    s = scale.float().unsqueeze(-1)
    code = torch.where(s > 0, g / s, torch.zeros_like(g)).round().clamp(-top, top).flatten(-2)
    if fmt == "int8":
        return code.to(torch.int8), scale
    code = (code + 8).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def _values(codes, scales, fmt):
    """The FP32 values that stored rows stand for."""
    if fmt not in ("int8", "int4"):
        return codes.float()
    if fmt == "int4":
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
        x = codes.float() - 8
    else:
        x = codes.float()
    groups = scales.shape[-1]
    return (x.unflatten(-1, (groups, -1)) * scales.float().unsqueeze(-1)).flatten(-2)


def _pools(pages, case):
    """Zeroed pages as the cache lays them out: [pages, kv_heads, page, row] and their scales."""
    h, p, d, fmt = case["kv_heads"], case["page"], case["dim"], case["format"]
    row = {"int8": (d, torch.int8, 1), "int4": (d // 2, torch.uint8, d // GROUP)}.get(fmt, (d, DTYPES.get(fmt), 0))

    def pool():
        return torch.zeros((pages, h, p, row[0]), dtype=row[1], device="cuda")

    def scale():
        return torch.zeros((pages, h, p, row[2]), dtype=torch.bfloat16, device="cuda") if row[2] else None

    return dict(k=pool(), v=pool(), k_scales=scale(), v_scales=scale())


def prepare(case, seed):
    state = _inputs(case, seed)
    if own and "pools" in state:  # the cache object that a server keeps, over the same pages
        state["cache"] = _library().PagedCache(case["kv_heads"], case["dim"], state["pools"]["k"].shape[0],
                                               case["page"], case["format"], storage=state["pools"])
    return state


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    d, hk = case["dim"], case["kv_heads"]
    state = dict(case=case)
    if case["op"] == "cache":
        n, dt = case["tokens"], DTYPES[case["source"]]
        if case["fused"]:  # K and V are columns of one fused projection's output
            qkv = _normal(gen, (n, 4 * hk * d), dt)
            state["k"] = qkv[:, 2 * hk * d:3 * hk * d].unflatten(-1, (hk, d)).mul_(_spread(d))
            state["v"] = qkv[:, 3 * hk * d:].unflatten(-1, (hk, d))
        else:
            state["k"] = _normal(gen, (n, hk, d), dt).mul_(_spread(d))
            state["v"] = _normal(gen, (n, hk, d), dt)
        pages = (n + case["page"] - 1) // case["page"] + 3
        where = torch.randperm(pages, generator=gen, device="cuda")
        t = torch.arange(n, device="cuda")
        slots = where[t // case["page"]] * case["page"] + t % case["page"]
        if case["pad"]:
            slots = torch.where(t % case["pad"] == case["pad"] - 1, -1, slots)
        state.update(slots=slots, pools=_pools(pages, case))
    elif case["op"] == "token":
        lens, page, fmt = lengths_of(case), case["page"], case["format"]
        need = [(x + page - 1) // page for x in lens]
        pages = sum(need) + 5
        where = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        width = max(need)
        first = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
        at = first[:, None] + torch.arange(width, device="cuda")
        used = torch.arange(width, device="cuda") < torch.tensor(need, device="cuda")[:, None]
        state["table"] = torch.where(used, where[at.clamp(max=pages - 1)], 0)
        state["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        state["q"] = _normal(gen, (case["batch"], case["q_heads"], d), DTYPES[case["dtype"]])
        pools = {}
        for name in ("k", "v"):
            x = _normal(gen, (pages, hk, page, d), torch.bfloat16 if fmt == "bf16" else torch.float16)
            if name == "k":
                x.mul_(_spread(d))
            if fmt in ("int8", "int4"):
                pools[name], pools[name + "_scales"] = _quantise(x.float(), fmt)
            else:
                pools[name], pools[name + "_scales"] = x, None
            del x
        state["pools"] = pools
    else:
        lens, pre, dt, hq = lengths_of(case), prefixes_of(case), DTYPES[case["dtype"]], case["q_heads"]
        keys = [a + b for a, b in zip(lens, pre)]
        state["starts"] = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
        if case["prefix"]:
            state["key_starts"] = torch.tensor([0] + keys, device="cuda").cumsum(0).to(torch.int32)
            state["q"] = _normal(gen, (sum(lens), hq, d), dt)
            kv = _normal(gen, (2, sum(keys), hk, d), dt)
            state["k"], state["v"] = kv[0].mul_(_spread(d)), kv[1]
        else:  # Q, K and V are columns of one fused projection's output
            qkv = _normal(gen, (sum(lens), (hq + 2 * hk) * d), dt)
            state["key_starts"] = None
            state["q"] = qkv[:, :hq * d].unflatten(-1, (hq, d))
            state["k"] = qkv[:, hq * d:(hq + hk) * d].unflatten(-1, (hk, d)).mul_(_spread(d))
            state["v"] = qkv[:, (hq + hk) * d:].unflatten(-1, (hk, d))
    return state


def _library():
    import sys
    if "block-gqt-webgpu_b200" not in sys.path:
        sys.path.insert(0, "block-gqt-webgpu_b200")
    import bgtq
    return bgtq


# ---- one pass ---------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if case["op"] == "cache":
        if own:
            state["cache"].write(state["k"], state["v"], state["slots"])
            k, v = state["cache"].read(state["slots"], dtype=state["k"].dtype)
            return dict(k=k, v=v)
        return _plain_cache(state, case)
    if case["op"] == "token":
        if own:
            out, lse = state["cache"].attend(state["q"], state["table"], state["lengths"], lse=True)
            return dict(out=out, lse=lse)
        return _plain_token(state, case)
    if own:
        out, lse = _library().prompt_attention(state["q"], state["k"], state["v"], state["starts"],
                                               state["key_starts"], causal=case["causal"], lse=True)
        return dict(out=out, lse=lse)
    return _plain_prompt(state, case)


def _plain_cache(state, case):
    """Rows quantised in FP32 and stored at their slots (a negative slot is padding, not stored), then
    every slot's row read back as the values it stands for (padding: zeros)."""
    pools, slots, page, fmt = state["pools"], state["slots"], case["page"], case["format"]
    there = slots >= 0
    live = slots[there]
    pg, at = live // page, live % page

    def there_and_back(x, pool, scales):
        codes, sc = _quantise(x.float(), fmt) if scales is not None else (x.float().to(DTYPES[fmt]), None)
        pool[pg, :, at] = codes[there]
        if scales is not None:
            scales[pg, :, at] = sc[there]
        got = torch.zeros_like(x, memory_format=torch.contiguous_format)
        got[there] = _values(pool[pg, :, at], None if scales is None else scales[pg, :, at], fmt).to(x.dtype)
        return got

    return dict(k=there_and_back(state["k"], pools["k"], pools["k_scales"]),
                v=there_and_back(state["v"], pools["v"], pools["v_scales"]))


def _softmax_parts(s):
    """exp(s - max), its sum and log of the sum of exp(s); a row of -inf alone gives zeros and -inf."""
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = s.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    return e, total, (top + total.log()).squeeze(-1)


def _plain_token(state, case):
    pools, fmt, hk = state["pools"], case["format"], case["kv_heads"]
    q = state["q"].float().unflatten(1, (hk, -1))                       # [B, hk, g, d]
    table = state["table"].long()

    def rows(name):                                                     # [B, hk, tokens, d]
        sc = pools[name + "_scales"]
        x = _values(pools[name][table], None if sc is None else sc[table], fmt)
        return x.transpose(1, 2).flatten(2, 3)

    k = rows("k")
    s = torch.matmul(q, k.transpose(-1, -2)).div_(math.sqrt(case["dim"]))
    del k
    inside = torch.arange(s.shape[-1], device=s.device) < state["lengths"][:, None]
    s.masked_fill_(~inside[:, None, None], -math.inf)
    e, total, lse = _softmax_parts(s)
    v = rows("v").masked_fill_(~inside[:, None, :, None], 0)
    out = torch.matmul(e, v) / torch.where(total > 0, total, torch.ones_like(total))
    return dict(out=out.flatten(1, 2).to(state["q"].dtype), lse=lse.flatten(1, 2))


def _plain_prompt(state, case):
    hq, hk, dev = case["q_heads"], case["kv_heads"], state["q"].device
    qs = state["starts"].long()
    ks = qs if state["key_starts"] is None else state["key_starts"].long()
    nq, nk = qs[1:] - qs[:-1], ks[1:] - ks[:-1]
    lq = max(lengths_of(case))
    lk = max(a + b for a, b in zip(lengths_of(case), prefixes_of(case))) if case["prefix"] else lq

    def padded(x, first, count, n):                                     # [B, heads, n, d]
        i = torch.arange(n, device=dev)
        at = (first[:-1, None] + i).clamp(max=max(0, x.shape[0] - 1))
        y = x[at].float() * (i < count[:, None])[:, :, None, None]
        return y.transpose(1, 2)

    q, k, v = padded(state["q"], qs, nq, lq), padded(state["k"], ks, nk, lk), padded(state["v"], ks, nk, lk)
    q = q.unflatten(1, (hk, hq // hk)).flatten(2, 3)                    # [B, hk, g * lq, d]
    s = torch.matmul(q, k.transpose(-1, -2)).div_(math.sqrt(case["dim"])).unflatten(2, (hq // hk, lq))
    j, i = torch.arange(lk, device=dev), torch.arange(lq, device=dev)
    seen = (j < nk[:, None])[:, None, :].expand(-1, lq, -1)
    if case["causal"]:
        seen = seen & (j <= i[:, None] + (nk - nq)[:, None, None])
    s.masked_fill_(~seen[:, None, None], -math.inf)
    e, total, lse = _softmax_parts(s)
    out = torch.matmul(e.flatten(2, 3), v).unflatten(2, (hq // hk, lq)) / torch.where(total > 0, total, 1.0)
    t = torch.arange(state["q"].shape[0], device=dev)
    seq = (t[:, None] >= qs[1:]).sum(1)
    pos = t - qs[seq]
    out, lse = out.flatten(1, 2), lse.flatten(1, 2)                     # [B, hq, lq, d], [B, hq, lq]
    return dict(out=out[seq, :, pos].to(state["q"].dtype), lse=lse[seq, :, pos])


# ---- what a pass cannot do without ----------------------------------------------------------

def _row_bytes(case):
    d = case["dim"]
    return {"int8": d + 2, "int4": d // 2 + 2 * (d // GROUP)}.get(case["format"], 2 * d)


def work(case):
    d, hk = case["dim"], case["kv_heads"]
    if case["op"] == "cache":
        n, wide = case["tokens"], 4 if case["source"] == "f32" else 2
        live = n - (n // case["pad"] if case["pad"] else 0)
        # the source rows, the stored rows written and read, the values written (padding too), the slots twice
        return dict(bytes=2 * hk * (live * (d * wide + 2 * _row_bytes(case)) + n * d * wide) + 16 * n,
                    flops=2 * hk * live * d * 4)
    hq = case["q_heads"]
    if case["op"] == "token":
        total = sum(lengths_of(case))
        return dict(bytes=total * 2 * hk * _row_bytes(case) + case["batch"] * hq * (4 * d + 4), flops=4 * total * hq * d)
    pairs, queries, keys = 0, 0, 0
    for n, p in zip(lengths_of(case), prefixes_of(case)):
        pairs += n * p + n * (n + 1) // 2 if case["causal"] else n * (n + p)
        queries, keys = queries + n, keys + n + p
    return dict(bytes=queries * hq * (4 * d + 4) + keys * hk * 4 * d, flops=4 * pairs * hq * d)


# ---- the definition in 64 bits ----------------------------------------------------------------

def _exact_row(x, fmt):
    """What a stored row stands for, in 64 bits: the scale is rounded to BF16 where it is stored."""
    if fmt in ("f16", "bf16"):
        return x.to(DTYPES[fmt]).double()
    top, group = (127.0, x.shape[-1]) if fmt == "int8" else (7.0, GROUP)
    y = x.double().reshape(*x.shape[:-1], -1, group)
    step = (y.abs().max(-1, keepdim=True).values / top).float().bfloat16().double()
    return (torch.round(y / step.clamp(min=1e-300)).clamp(-top, top) * step).reshape(x.shape)


def exact(case, seed):
    state = _inputs(case, seed)
    if case["op"] == "cache":
        live = (state["slots"] >= 0)[:, None, None]
        return {n: (_exact_row(state[n], case["format"]) * live).double() for n in ("k", "v")}
    d, hq, hk = case["dim"], case["q_heads"], case["kv_heads"]
    group = hq // hk
    outs, lses = [], []
    if case["op"] == "token":
        for b, n in enumerate(lengths_of(case)):
            pages = state["table"][b, :(n + case["page"] - 1) // case["page"]].long()
            rows = {}
            for name in ("k", "v"):
                x = state["pools"][name][pages].permute(1, 0, 2, 3).reshape(hk, -1, state["pools"][name].shape[-1])
                if case["format"] in ("int8", "int4"):
                    sc = state["pools"][name + "_scales"][pages].permute(1, 0, 2, 3).double()
                    sc = sc.reshape(hk, x.shape[1], -1)
                    if case["format"] == "int4":
                        y = torch.empty((hk, x.shape[1], d), dtype=torch.float64, device=x.device)
                        y[..., 0::2], y[..., 1::2] = (x % 16).double() - 8, (x // 16).double() - 8
                    else:
                        y = x.double()
                    x = y * sc.repeat_interleave(d // sc.shape[-1], dim=-1)
                rows[name] = x[:, :n].double()
            q = state["q"][b].double().reshape(hk, group, d)
            s = torch.einsum("hgd,htd->hgt", q, rows["k"]) / math.sqrt(d)
            lses.append(torch.logsumexp(s, -1).reshape(hq))
            outs.append(torch.einsum("hgt,htd->hgd", torch.softmax(s, -1), rows["v"]).reshape(hq, d))
        return dict(out=torch.stack(outs), lse=torch.stack(lses))
    q0 = k0 = 0
    for n, p in zip(lengths_of(case), prefixes_of(case)):
        q = state["q"][q0:q0 + n].double()
        k, v = state["k"][k0:k0 + n + p].double(), state["v"][k0:k0 + n + p].double()
        q0, k0 = q0 + n, k0 + n + p
        out = torch.empty((n, hq, d), dtype=torch.float64, device=q.device)
        lse = torch.empty((n, hq), dtype=torch.float64, device=q.device)
        for h in range(hq):
            s = q[:, h] @ k[:, h // group].T / math.sqrt(d)
            if case["causal"]:
                late = torch.ones((n, n + p), dtype=torch.bool, device=q.device).triu(p + 1)
                s = s.masked_fill(late, -math.inf)
            lse[:, h] = torch.logsumexp(s, -1)
            out[:, h] = torch.softmax(s, -1) @ v[:, h // group]
        outs.append(out)
        lses.append(lse)
    return dict(out=torch.cat(outs), lse=torch.cat(lses))
