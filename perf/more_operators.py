"""The operators of a serving step, in cases of real sizes.

Three operators that follow one another in every step of `bgtq.PagedDecoder`: the new tokens'
queries and keys are normed (where the model does) and rotated, and keys and values go into the
pages in the same pass (`bgtq.PagedCache.append`); a chunk of new tokens of every request, from
one to thousands, attends over the request's pages, all of them or a window and the first few
(`bgtq.PagedCache.attend_chunk`); penalties, biases and grammar masks are put on the logits
(`bgtq.adjust_logits`).

    listed(), draw(rng)    the cases: dicts of plain values
    prepare(case, seed)    what a server has in hand before the call
    run(state)             one pass; `own` chooses the library's kernels or the plain form
    work(case)             bytes and operations that the pass cannot do without
    exact(case, seed)      the result by definition, in 64 bits
"""
import math

import torch

own = False  # False: elementary torch operations; True: the library's entry points

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
GROUP = 32  # dimensions that share one scale in a 4-bit row
EPS = 1e-6  # of the head norms


# ---- the cases -------------------------------------------------------------------------

def listed():
    return [
        # --- queries and keys rotated, keys and values into the pages ---
        # one decode step of 16 requests, 9 / 3 heads of 64 (the small model's geometry), 16-bit pages: latency
        dict(name="append-step", op="append", tokens=16, q_heads=9, kv_heads=3, dim=64, format="f16", source="f16",
             page=16, pad=0, norm=False),
        # a padded batch of short prompts, 14 / 2 heads of 64, 8-bit pages (their rows are read back): an odd token
        # count, every 7th row is padding
        dict(name="append-ragged", op="append", tokens=4999, q_heads=14, kv_heads=2, dim=64, format="int8",
             source="bf16", page=16, pad=7, norm=False),
        # a chunk of prompts from FP32 projections with head norms, 32 / 8 heads of 128
        dict(name="append-norm", op="append", tokens=2047, q_heads=32, kv_heads=8, dim=128, format="bf16",
             source="f32", page=32, pad=0, norm=True),
        # 16K prompt tokens of a wide layer with head norms, 4-bit pages (their rows are read back): a bandwidth case
        dict(name="append-prompt", op="append", tokens=16384, q_heads=32, kv_heads=8, dim=128, format="int4",
             source="bf16", page=64, pad=0, norm=True),
        # --- new tokens over their request's pages ---
        # a server's step in streaming use: 64 requests, one token each, window of 2048 and four first tokens
        dict(name="chunk-window", op="chunk", batch=64, new_least=1, new_most=1, old_least=100, old_most=32767,
             q_heads=14, kv_heads=2, dim=64, format="f16", dtype="f16", page=64, window=2048, sinks=4),
        # drafted tokens verified: 32 requests, five tokens each, 8-bit pages of up to 16K tokens
        dict(name="chunk-verify", op="chunk", batch=32, new_least=5, new_most=5, old_least=500, old_most=16000,
             q_heads=32, kv_heads=8, dim=128, format="int8", dtype="bf16", page=64, window=0, sinks=0),
        # a mixed step of a server: 20 requests, one to 700 new tokens over up to 9001, 16-bit pages
        dict(name="chunk-mixed", op="chunk", batch=20, new_least=1, new_most=700, old_least=1, old_most=9001,
             q_heads=32, kv_heads=8, dim=128, format="bf16", dtype="bf16", page=32, window=0, sinks=0),
        # the later chunk of two long documents, 14 / 2 heads of 64, 8-bit pages
        dict(name="chunk-long", op="chunk", batch=2, new_least=2048, new_most=2048, old_least=24000, old_most=30000,
             q_heads=14, kv_heads=2, dim=64, format="int8", dtype="f16", page=64, window=0, sinks=0),
        # later chunks of four prompts of a wide layer, 32 / 8 heads of 128, 16-bit pages
        dict(name="chunk-wide", op="chunk", batch=4, new_least=1024, new_most=1024, old_least=6000, old_most=8192,
             q_heads=32, kv_heads=8, dim=128, format="bf16", dtype="bf16", page=128, window=0, sinks=0),
        # --- penalties, biases and masks on the logits ---
        # one chat request, the small model's vocabulary: latency
        dict(name="logits-one", op="logits", batch=1, vocab=49152, shortest=300, longest=300, dtype="f32",
             entries=10, mask=False),
        # 37 requests of the small model in 16 bits, grammar masks, an odd history length
        dict(name="logits-half", op="logits", batch=37, vocab=49152, shortest=1, longest=2047, dtype="bf16",
             entries=33, mask=True),
        # 256 requests of the large vocabulary, long histories, grammar masks
        dict(name="logits-batch", op="logits", batch=256, vocab=151936, shortest=16, longest=8192, dtype="f32",
             entries=50, mask=True),
    ]


def _log(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    op = rng.choice(["append", "append", "chunk", "chunk", "chunk", "logits"])
    if op == "logits":
        vocab = rng.choice([49152, 151936, _log(rng, 1000, 151936)])
        longest = _log(rng, 1, 8192)
        return dict(op=op, batch=_log(rng, 1, min(256, 256 * 151936 // vocab)), vocab=vocab,
                    shortest=_log(rng, 1, longest), longest=longest, dtype=rng.choice(["f16", "bf16", "f32"]),
                    entries=rng.choice([0, _log(rng, 1, 300)]), mask=rng.random() < 0.5)
    dim = rng.choice([64, 128])
    kv = rng.choice([1, 2, 3, 4, 8])
    hq = kv * rng.choice([1, 2, 3, 4, 7, 8])
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        fmt = rng.choice(["f16", "bf16", "int8", "int4"])
        tokens = _log(rng, 1, min(16384, 16384 * 32 * 128 // (hq * dim)))
        return dict(op=op, tokens=tokens, q_heads=hq, kv_heads=kv, dim=dim, format=fmt,
                    source=rng.choice(["f16", "bf16", "f32"]), page=page, pad=rng.choice([0, 0, 5, 13]),
                    norm=rng.random() < 0.5)
    dtype = rng.choice(["f16", "bf16"])
    batch = _log(rng, 1, 48)
    rows = 4 * 32 * 1024 * 9216 // (batch * hq)           # new tokens x keys of a request, at most
    most = min(32768, (1 << 28) // (batch * kv * dim))    # keys of a request, at most
    new = _log(rng, 1, max(1, min(2048, most // 2, int(math.sqrt(rows)))))
    old = _log(rng, 1, max(1, min(most, rows // new) - new))
    return dict(op=op, batch=batch, new_least=_log(rng, 1, new), new_most=new, old_least=_log(rng, 1, old),
                old_most=old, q_heads=hq, kv_heads=kv, dim=dim, format=rng.choice([dtype, "int8", "int4"]),
                dtype=dtype, page=page, window=rng.choice([0, 0, _log(rng, 16, 8192)]),
                sinks=rng.choice([0, 1, 4, 70]))


def _spread_over(low, high, count, turn):
    """count numbers from low to high on a logarithmic scale, in a mixed order."""
    if count == 1:
        return [high]
    order = sorted(range(count), key=lambda i: (i * turn + 3) % 10007)
    return [int(round(low * (high / low) ** (i / (count - 1)))) for i in order]


def new_of(case):
    return _spread_over(case["new_least"], case["new_most"], case["batch"], 7919)


def lengths_of(case):
    """Tokens of every request that the pages hold, its new ones among them."""
    return [a + b for a, b in zip(_spread_over(case["old_least"], case["old_most"], case["batch"], 4243), new_of(case))]


def histories_of(case):
    return _spread_over(case["shortest"], case["longest"], case["batch"], 7919)


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
    scale = (g.abs().amax(-1) * torch.tensor(1.0 / top, dtype=torch.float32, device=x.device)).to(torch.bfloat16)
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
    return (x.unflatten(-1, (scales.shape[-1], -1)) * scales.float().unsqueeze(-1)).flatten(-2)


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
    return dict(append=_append_inputs, chunk=_chunk_inputs, logits=_logits_inputs)[case["op"]](case, gen)


def _append_inputs(case, gen):
    n, dt, d, hq, hk = case["tokens"], DTYPES[case["source"]], case["dim"], case["q_heads"], case["kv_heads"]
    state = dict(case=case)
    qkv = _normal(gen, (n, (hq + 2 * hk) * d), dt)  # Q, K and V are columns of one fused projection's output
    state["q"] = qkv[:, :hq * d].unflatten(-1, (hq, d))
    state["k"] = qkv[:, hq * d:(hq + hk) * d].unflatten(-1, (hk, d)).mul_(_spread(d))
    state["v"] = qkv[:, (hq + hk) * d:].unflatten(-1, (hk, d))
    # cosines and sines of the positions up to 8192, and the tokens' positions
    at = torch.arange(8192, device="cuda").double()[:, None]
    angle = at * torch.pow(1e5, -torch.arange(d // 2, device="cuda").double() / (d // 2))
    state["rotary"] = torch.cat([angle.cos(), angle.sin()], -1).float()
    state["positions"] = torch.randint(0, 8192, (n,), generator=gen, device="cuda")
    for name in ("q_norm", "k_norm"):
        state[name] = _normal(gen, (d,), torch.float32).mul_(0.2).add_(1) if case["norm"] else None
    pages = (n + case["page"] - 1) // case["page"] + 3
    where = torch.randperm(pages, generator=gen, device="cuda")
    t = torch.arange(n, device="cuda")
    slots = where[t // case["page"]] * case["page"] + t % case["page"]
    if case["pad"]:
        slots = torch.where(t % case["pad"] == case["pad"] - 1, -1, slots)
    state.update(slots=slots, pools=_pools(pages, case))
    return state


def _chunk_inputs(case, gen):
    d, hk, lens, page, fmt = case["dim"], case["kv_heads"], lengths_of(case), case["page"], case["format"]
    need = [(x + page - 1) // page for x in lens]
    pages = sum(need) + 5
    where = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    width = max(need)
    first = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    at = first[:, None] + torch.arange(width, device="cuda")
    used = torch.arange(width, device="cuda") < torch.tensor(need, device="cuda")[:, None]
    state = dict(case=case, table=torch.where(used, where[at.clamp(max=pages - 1)], 0))
    state["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    state["starts"] = torch.tensor([0] + new_of(case), device="cuda").cumsum(0).to(torch.int32)
    state["q"] = _normal(gen, (sum(new_of(case)), case["q_heads"], d), DTYPES[case["dtype"]])
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
    return state


def _logits_inputs(case, gen):
    b, n, lens = case["batch"], case["vocab"], histories_of(case)
    state = dict(case=case, logits=_normal(gen, (b, n), torch.float32).mul_(4).to(DTYPES[case["dtype"]]))
    # texts repeat frequent words: ids dense at the low end
    u = torch.rand((b, max(lens)), generator=gen, device="cuda", dtype=torch.float64)
    state["tokens"] = (u ** 3 * n).long().clamp(max=n - 1).to(torch.int32)
    state["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def uniform(low, high):
        return torch.rand(b, generator=gen, device="cuda") * (high - low) + low

    state.update(repetition=uniform(1.0, 1.5), presence=uniform(0.0, 1.0), frequency=uniform(0.0, 0.5))
    state["bias_ids"] = state["bias"] = state["mask"] = None
    if case["entries"]:  # each id once in a row
        i = torch.arange(case["entries"], device="cuda")
        first = torch.randint(0, n, (b, 1), generator=gen, device="cuda")
        state["bias_ids"] = ((first + i * (n // case["entries"])) % n).to(torch.int32)
        state["bias"] = _normal(gen, (b, case["entries"]), torch.float32).mul_(5)
    if case["mask"]:  # a bit for each id, 32 to a word: about half of them allowed
        state["mask"] = torch.randint(-2 ** 31, 2 ** 31, (b, (n + 31) // 32), generator=gen, device="cuda").to(torch.int32)
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
    if case["op"] == "append":
        return _own_append(state, case) if own else _plain_append(state, case)
    if case["op"] == "chunk":
        if own:
            out, lse = state["cache"].attend_chunk(state["q"], state["starts"], state["table"], state["lengths"],
                                                   window=case["window"] or None, sinks=case["sinks"], lse=True)
            return dict(out=out, lse=lse)
        return _plain_chunk(state, case)
    if own:
        return _library().adjust_logits(state["logits"], state["tokens"], state["lengths"],
                                        repetition=state["repetition"], presence=state["presence"],
                                        frequency=state["frequency"], bias_ids=state["bias_ids"], bias=state["bias"],
                                        mask=state["mask"])
    return _plain_logits(state, case)


def _half(case):
    return torch.float16 if "f16" in (case["source"], case["format"]) else torch.bfloat16


def _own_append(state, case):
    cache = state["cache"]
    q = cache.append(state["q"], state["k"], state["v"], state["slots"], state["rotary"], state["positions"],
                     q_norm=state["q_norm"], k_norm=state["k_norm"], eps=EPS, dtype=_half(case))
    if case["format"] in ("int8", "int4"):  # what the rows stand for
        k, v = cache.read(state["slots"], dtype=_half(case))
        return dict(q=q, k=k, v=v)
    return dict(q=q, k=cache.k, v=cache.v)


def _turned(x, norm, rotary):
    """Heads normed, if there are weights, and rotated, in 64 bits: a code is a step function of its
    row, so the row has to be right to FP32's last place."""
    x = x.double()
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * norm.double()
    a, b = x.chunk(2, -1)
    cos, sin = rotary.double()[:, None].chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).float()


def _plain_append(state, case):
    pools, slots, page, fmt = state["pools"], state["slots"], case["page"], case["format"]
    rotary = state["rotary"][state["positions"]]
    q = _turned(state["q"], state["q_norm"], rotary).to(_half(case))
    there = slots >= 0
    live = slots[there]
    pg, at = live // page, live % page

    def put(x, name):
        pool, scales = pools[name], pools[name + "_scales"]
        if scales is None:
            pool[pg, :, at] = x[there].to(pool.dtype)
            return pool
        codes, sc = _quantise(x, fmt)
        pool[pg, :, at] = codes[there]
        scales[pg, :, at] = sc[there]
        got = torch.zeros(x.shape, dtype=_half(case), device=x.device)
        got[there] = _values(pool[pg, :, at], scales[pg, :, at], fmt).to(got.dtype)
        return got

    return dict(q=q, k=put(_turned(state["k"], state["k_norm"], rotary), "k"), v=put(state["v"].float(), "v"))


def _plain_chunk(state, case):
    pools, fmt, hk, hq, dev = state["pools"], case["format"], case["kv_heads"], case["q_heads"], state["q"].device
    lens, first = state["lengths"].long(), state["starts"].long()
    count = first[1:] - first[:-1]
    lq, table = case["new_most"], state["table"].long()

    def rows(name):                                                     # [B, hk, tokens, d]
        sc = pools[name + "_scales"]
        x = _values(pools[name][table], None if sc is None else sc[table], fmt)
        return x.transpose(1, 2).flatten(2, 3)

    i = torch.arange(lq, device=dev)
    at = (first[:-1, None] + i).clamp(max=state["q"].shape[0] - 1)
    q = state["q"][at].float().transpose(1, 2)                          # [B, hq, lq, d]
    q = q.unflatten(1, (hk, hq // hk)).flatten(2, 3)                    # [B, hk, g * lq, d]
    k = rows("k")
    s = torch.matmul(q, k.transpose(-1, -2)).div_(math.sqrt(case["dim"])).unflatten(2, (hq // hk, lq))
    j = torch.arange(k.shape[2], device=dev)
    del k
    mine = (lens - count)[:, None, None] + i[:, None]                   # a row's own position
    seen = (j <= mine) & (i < count[:, None])[:, :, None]
    if case["window"]:
        seen &= (j > mine - case["window"]) | (j < case["sinks"])
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = s.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    v = rows("v").masked_fill_(~(j < lens[:, None])[:, None, :, None], 0)
    out = torch.matmul(e.flatten(2, 3), v).unflatten(2, (hq // hk, lq)) / torch.where(total > 0, total, 1.0)
    lse = (top + total.log()).squeeze(-1)
    t = torch.arange(state["q"].shape[0], device=dev)
    seq = (t[:, None] >= first[1:]).sum(1)
    pos = t - first[seq]
    out, lse = out.flatten(1, 2), lse.flatten(1, 2)                     # [B, hq, lq, d], [B, hq, lq]
    return dict(out=out[seq, :, pos].to(state["q"].dtype), lse=lse[seq, :, pos])


def _plain_logits(state, case):
    x, ids, n = state["logits"].float(), state["tokens"].long(), case["vocab"]
    there = torch.arange(ids.shape[1], device=x.device) < state["lengths"][:, None]
    count = torch.zeros((x.shape[0], n + 1), device=x.device).scatter_add_(1, torch.where(there, ids, n),
                                                                           there.float())[:, :n]
    again = count > 0
    r = state["repetition"][:, None]
    x = torch.where(again, torch.where(x > 0, x / r, x * r), x)
    x = x - state["presence"][:, None] * again - state["frequency"][:, None] * count
    if state["bias"] is not None:
        x = x.scatter_add(1, state["bias_ids"].long(), state["bias"])
    if state["mask"] is not None:
        v = torch.arange(n, device=x.device)
        allowed = (state["mask"][:, v // 32] >> (v % 32)) & 1
        x = torch.where(allowed != 0, x, -math.inf)
    return x.to(state["logits"].dtype)


# ---- what a pass cannot do without ----------------------------------------------------------

def _row_bytes(case):
    d = case["dim"]
    return {"int8": d + 2, "int4": d // 2 + 2 * (d // GROUP)}.get(case["format"], 2 * d)


def seen_by(case, n, length):
    """(pairs of a query and a key, keys that any of them sees) of a request's n new tokens of `length`."""
    w, sinks = case["window"], case["sinks"]
    pairs = sum(min(p + 1, w + min(sinks, max(0, p + 1 - w))) for p in range(length - n, length)) if w else \
        n * (length - n) + n * (n + 1) // 2
    keys = min(length, w + n - 1 + min(sinks, max(0, length - n - w + 1))) if w else length
    return pairs, keys


def work(case):
    if case["op"] == "logits":
        b, n = case["batch"], case["vocab"]
        wide = 4 if case["dtype"] == "f32" else 2
        return dict(bytes=b * (2 * n * wide + (n // 8 if case["mask"] else 0) + 8 * case["entries"] + 16) +
                    4 * sum(histories_of(case)), flops=b * n * 4)
    d, hk, hq = case["dim"], case["kv_heads"], case["q_heads"]
    if case["op"] == "append":
        n, wide = case["tokens"], 4 if case["source"] == "f32" else 2
        live = n - (n // case["pad"] if case["pad"] else 0)
        # queries in and out, rows of cosines and sines, positions and slots; keys and values in and into the pages
        moved = n * hq * d * (wide + 2) + min(n, 8192) * 4 * d + 16 * n + live * 2 * hk * (d * wide + _row_bytes(case))
        if case["format"] in ("int8", "int4"):  # and back
            moved += 2 * hk * (live * _row_bytes(case) + 2 * n * d) + 8 * n
        return dict(bytes=moved, flops=n * (hq + hk) * d * (6 if case["norm"] else 3))
    pairs = keys = queries = 0
    for n, length in zip(new_of(case), lengths_of(case)):
        p, k = seen_by(case, n, length)
        pairs, keys, queries = pairs + p, keys + k, queries + n
    return dict(bytes=keys * 2 * hk * _row_bytes(case) + queries * hq * (4 * d + 4), flops=4 * pairs * hq * d)


# ---- the definition in 64 bits ----------------------------------------------------------------

def exact(case, seed):
    state = _inputs(case, seed)
    return dict(append=_exact_append, chunk=_exact_chunk, logits=_exact_logits)[case["op"]](case, state)


def _exact_row(x, fmt):
    """What a stored row stands for, in 64 bits: the scale is rounded to BF16 where it is stored."""
    if fmt in ("f16", "bf16"):
        return x.to(DTYPES[fmt]).double()
    top, group = (127.0, x.shape[-1]) if fmt == "int8" else (7.0, GROUP)
    y = x.double().reshape(*x.shape[:-1], -1, group)
    step = (y.abs().max(-1, keepdim=True).values / top).float().bfloat16().double()
    return (torch.round(y / step.clamp(min=1e-300)).clamp(-top, top) * step).reshape(x.shape)


def _exact_append(case, state):
    d = case["dim"]
    table = state["rotary"][state["positions"]].double()
    turn = torch.complex(table[:, :d // 2], table[:, d // 2:])[:, None]

    def heads(name):
        x = state[name].double()
        if case["norm"]:
            x = x / (x.square().sum(-1, keepdim=True) / d + EPS).sqrt() * state[name + "_norm"].double()
        z = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:].contiguous()) * turn
        return torch.cat([z.real, z.imag], -1)

    slots, fmt = state["slots"], case["format"]
    got = dict(q=heads("q"))
    for name, x in (("k", heads("k")), ("v", state["v"].double())):
        rows = _exact_row(x, fmt)
        if fmt in ("int8", "int4"):
            got[name] = rows * (slots >= 0)[:, None, None]
        else:
            flat = torch.zeros((state["pools"]["k"].shape[0] * case["page"], case["kv_heads"], d), dtype=torch.float64,
                               device=x.device)
            flat[slots[slots >= 0]] = x[slots >= 0]
            got[name] = flat.unflatten(0, (-1, case["page"])).transpose(1, 2).contiguous()
    return got


def _exact_chunk(case, state):
    d, hq, hk, page = case["dim"], case["q_heads"], case["kv_heads"], case["page"]
    group, outs, lses, q0 = hq // hk, [], [], 0
    for b, (n, length) in enumerate(zip(new_of(case), lengths_of(case))):
        pages = state["table"][b, :(length + page - 1) // page].long()
        rows = {}
        for name in ("k", "v"):
            x = state["pools"][name][pages].permute(1, 0, 2, 3).reshape(hk, -1, state["pools"][name].shape[-1])
            if case["format"] in ("int8", "int4"):
                sc = state["pools"][name + "_scales"][pages].permute(1, 0, 2, 3).double().reshape(hk, x.shape[1], -1)
                if case["format"] == "int4":
                    y = torch.empty((hk, x.shape[1], d), dtype=torch.float64, device=x.device)
                    y[..., 0::2], y[..., 1::2] = (x % 16).double() - 8, (x // 16).double() - 8
                else:
                    y = x.double()
                x = y * sc.repeat_interleave(d // sc.shape[-1], dim=-1)
            rows[name] = x[:, :length].double()
        place = torch.arange(length - n, length, device="cuda")[:, None]
        key = torch.arange(length, device="cuda")[None]
        hidden = key > place
        if case["window"]:
            hidden |= (place - key >= case["window"]) & (key >= case["sinks"])
        out = torch.empty((n, hq, d), dtype=torch.float64, device="cuda")
        lse = torch.empty((n, hq), dtype=torch.float64, device="cuda")
        for h in range(hq):
            s = state["q"][q0:q0 + n, h].double() @ rows["k"][h // group].T / math.sqrt(d)
            s = s.masked_fill(hidden, -math.inf)
            lse[:, h] = torch.logsumexp(s, -1)
            out[:, h] = torch.softmax(s, -1) @ rows["v"][h // group]
        q0 += n
        outs.append(out)
        lses.append(lse)
    return dict(out=torch.cat(outs), lse=torch.cat(lses))


def _exact_logits(case, state):
    x = state["logits"].double()
    for b, n in enumerate(histories_of(case)):
        ids, counts = torch.unique(state["tokens"][b, :n].long(), return_counts=True)
        y, r = x[b, ids], state["repetition"][b].double()
        y = y * torch.where(y > 0, 1 / r, r)
        x[b, ids] = y - state["presence"][b].double() - state["frequency"][b].double() * counts
        if state["bias"] is not None:
            x[b, state["bias_ids"][b].long()] += state["bias"][b].double()
    if state["mask"] is not None:
        bits = (state["mask"].long()[:, :, None] >> torch.arange(32, device=x.device)) & 1
        x = x.masked_fill(bits.flatten(1)[:, :case["vocab"]] == 0, -math.inf)
    return x
