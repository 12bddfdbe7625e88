"""The operators of a step of several requests at once, as cases that can be timed and compared.

The framework's decoder serves one sequence with a contiguous cache.  Several requests at once keep their cache rows in
blocks ("pages") of a shared pool, start behind one prefix whose rows they share (a system prompt, or the prompt
whose continuations are sampled in parallel), and go through three operators in every step:

op "tables"     llama2_batch_tables: once a step, from the requests' lengths: new blocks out of the pool's free list, the
                block tables, first query row of every request, position and cache slot of every token.
op "rope"       llama2_batch_qk_norm_rope: once a layer: norm of every query and key head (where the model has one), rotation
                by the token's position, keys and values to their slots of the paged cache.
op "attention"  llama2_batch_attention: once a layer: causal attention of all tokens over the shared prefix and each
                request's own rows.

Head counts and sizes are those of synth.LLAMA2_7B (32 heads of 128), synth.LLAMA2_13B (40) and the small models of the
tests, and the same with fewer key/value heads, which the rotation takes already.  Everything is fp16, as in the whole framework.
Lengths are spread evenly over their logarithm between the bounds that a case names; the seed says which request has which.
"""
import math

import torch

own = False

_HALF, _INT = torch.float16, torch.int32


def listed():
    return [
        # one decode step of a busy server: 200 requests, launched for up to 256 (a captured step); most need no block
        dict(name="tables_decode_200", op="tables", requests=200, block=16, prefix=512, ctx_lo=1, ctx_hi=4000, new_lo=1,
             new_hi=1, pad=56, short=0),
        # a step that reads prompts; the pool runs dry before the last of them
        dict(name="tables_prompts_48", op="tables", requests=48, block=16, prefix=0, ctx_lo=0, ctx_hi=0, new_lo=1, new_hi=2000,
             pad=0, short=100),
        # one request of the 7B model: latency
        dict(name="rope_one_token", op="rope", requests=1, heads=32, kv_heads=32, head_size=128, block=16, prefix=0, ctx_lo=777,
             ctx_hi=777, new_lo=1, new_hi=1, pad=0, norms=False, fused=False, theta=10000.0),
        # a decode step of 64 requests of a model with normed queries and keys and 8 key/value heads, far into a long context
        dict(name="rope_norms_64", op="rope", requests=64, heads=32, kv_heads=8, head_size=128, block=32, prefix=100000,
             ctx_lo=1, ctx_hi=900, new_lo=1, new_hi=1, pad=0, norms=True, fused=True, theta=1000000.0),
        # prompts of the 13B model
        dict(name="rope_prompts_13b", op="rope", requests=12, heads=40, kv_heads=40, head_size=128, block=16, prefix=300,
             ctx_lo=0, ctx_hi=0, new_lo=40, new_hi=1100, pad=0, norms=False, fused=True, theta=10000.0),
        # one request alone, nothing shared: latency
        dict(name="attn_one_request", op="attention", requests=1, heads=32, kv_heads=32, head_size=128, block=16, prefix=0,
             ctx_lo=776, ctx_hi=776, new_lo=1, new_hi=1, pad=0),
        # 16 continuations of one prompt sampled in parallel, 7B
        dict(name="attn_samples_16", op="attention", requests=16, heads=32, kv_heads=32, head_size=128, block=16, prefix=2048,
             ctx_lo=1, ctx_hi=256, new_lo=1, new_hi=1, pad=0),
        # 64 conversations behind one system prompt, from just begun to nearly full, 7B; a captured step for up to 72
        dict(name="attn_chats_64", op="attention", requests=64, heads=32, kv_heads=32, head_size=128, block=16, prefix=1024,
             ctx_lo=1, ctx_hi=4000, new_lo=1, new_hi=1, pad=8),
        # 128 short conversations about one long document, 8 key/value heads
        dict(name="attn_document_128", op="attention", requests=128, heads=32, kv_heads=8, head_size=128, block=64, prefix=8192,
             ctx_lo=100, ctx_hi=2000, new_lo=1, new_hi=1, pad=0),
        # four long documents, 40 heads over 8 key/value heads, nothing shared
        dict(name="attn_long_4", op="attention", requests=4, heads=40, kv_heads=8, head_size=128, block=128, prefix=0,
             ctx_lo=20000, ctx_hi=131000, new_lo=1, new_hi=1, pad=0),
        # the first turns of 8 conversations behind a system prompt: whole prompts
        dict(name="attn_prompts_8", op="attention", requests=8, heads=32, kv_heads=32, head_size=128, block=16, prefix=512,
             ctx_lo=0, ctx_hi=0, new_lo=50, new_hi=1500, pad=0),
        # a small model with heads of 64: next turns of a few tokens, decoding requests among them
        dict(name="attn_turns_small", op="attention", requests=19, heads=8, kv_heads=8, head_size=64, block=8, prefix=333,
             ctx_lo=1, ctx_hi=700, new_lo=1, new_hi=40, pad=5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(32, 32), (32, 32), (40, 40), (32, 8), (40, 8), (4, 4), (8, 8), (16, 2), (8, 1)]


def draw(rng):
    op = rng.choice(["tables", "rope", "rope", "attention", "attention", "attention", "attention"])
    kind = rng.choice(["decode", "decode", "turns", "prompts"])
    c = dict(op=op, requests=_log_int(rng, 1, 64 if kind == "prompts" else 160), block=rng.choice([8, 16, 16, 32, 64, 128]),
             prefix=rng.choice([0, _log_int(rng, 1, 12000)]), ctx_lo=0, ctx_hi=0, new_lo=1, new_hi=1,
             pad=rng.choice([0, 0, rng.randint(1, 40)]))
    if kind != "prompts":
        c["ctx_hi"] = _log_int(rng, 1, 6000)
        c["ctx_lo"] = _log_int(rng, 1, c["ctx_hi"])
    if kind == "turns":
        c["new_hi"] = _log_int(rng, 2, 200)
    if kind == "prompts":
        c["new_hi"] = _log_int(rng, 2, 1500)
        c["new_lo"] = _log_int(rng, 1, c["new_hi"])
    if op == "tables":
        c["short"] = rng.choice([0, 0, rng.randint(1, 60)])
        return c
    c["heads"], c["kv_heads"] = rng.choice(_HEADS)
    c["head_size"] = rng.choice([128, 128, 64])
    if op == "rope":
        c.update(norms=rng.choice([True, False]), fused=rng.choice([True, False]), theta=rng.choice([10000.0, 500000.0]))
        limit, most = 4.0e8, work(listed()[4])["bytes"]
    else:
        limit, most = 6.0e9, max(work(x)["bytes"] for x in listed())
    while True:  # as large as the listed ones at most, and small enough for the padded plain form
        ctx, new = _lengths(c)
        w = work(c)
        padded = c["requests"] * (max(ctx) + max(new)) * c["kv_heads"] * c["head_size"] * 4
        scores = c["requests"] * max(new) * c["heads"] * (c["prefix"] + max(ctx) + max(new)) * 4 if op == "attention" else 0
        if w["bytes"] <= most and w["flops"] <= 4.0e10 and padded <= limit and scores <= limit:
            return c
        if c["requests"] > 2:
            c["requests"] = c["requests"] * 2 // 3
        else:
            c["prefix"] //= 2
            c["new_hi"] = max(1, c["new_hi"] // 2)
            c["new_lo"] = min(c["new_lo"], c["new_hi"])
            c["ctx_hi"] //= 2
            c["ctx_lo"] = min(c["ctx_lo"], c["ctx_hi"])


def _spread(lo, hi, n, turn):
    """n lengths from lo to hi, even steps of the logarithm, begun `turn` places on."""
    a, b = math.log(lo + 1), math.log(hi + 1)
    v = [round(math.exp(a + (b - a) * (i / (n - 1) if n > 1 else 1.0))) - 1 for i in range(n)]
    return v[turn:] + v[:turn]


def _lengths(case):
    """Rows that each request has cached, and the tokens that it brings."""
    n = case["requests"]
    return _spread(case["ctx_lo"], case["ctx_hi"], n, 0), _spread(case["new_lo"], case["new_hi"], n, n // 3)


def _blocks(rows, size):
    return -(-rows // size)


# ---------------------------------------------------------------- inputs

def _floats(gen, *shape, std=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(_HALF)


def _batch(case, seed, gen):
    """The requests of a step: lengths, tables of random blocks, the tokens' positions."""
    size, n = case["block"], case["requests"]
    ctx, new = _lengths(case)
    order = torch.randperm(n, generator=torch.Generator().manual_seed(int(seed))).tolist()
    ctx, new = [ctx[i] for i in order], [new[i] for i in order]
    before, after = [_blocks(c, size) for c in ctx], [_blocks(c + m, size) for c, m in zip(ctx, new)]
    stride = max(after) + 3  # room for later steps
    shared = _blocks(case["prefix"], size) if case["op"] == "attention" else 0
    total = sum(after) + shared + 5
    ids = torch.randperm(total, generator=gen, device="cuda").to(_INT)
    grid = torch.arange(stride, device="cuda")[None, :]

    def table(used):
        u = torch.tensor(used, device="cuda")
        first = torch.cumsum(u, 0) - u
        return torch.where(grid < u[:, None], ids[(first[:, None] + grid).clamp(max=total - 1)], -1).to(_INT)

    starts = torch.tensor([0] + new, device="cuda").cumsum(0)
    s = dict(requests=n, size=size, prefix=case["prefix"], stride=stride, n_blocks=total, tokens=sum(new) + case["pad"],
             cached=torch.tensor(ctx, device="cuda", dtype=_INT), counts=torch.tensor(new, device="cuda", dtype=_INT),
             before=table(before), tables=table(after), free=ids[sum(before):].contiguous(),
             prefix_table=ids[total - shared:] if shared else ids[:0],
             starts=starts.to(_INT), max_new=max(new), max_length=max(c + m for c, m in zip(ctx, new)),
             lengths=(ctx, new))
    t = torch.arange(s["tokens"], device="cuda")
    b = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp(max=n - 1)
    row = s["cached"].long()[b] + t - starts[b]
    live = t < starts[-1]
    s["positions"] = torch.where(live, row + case["prefix"], -1).to(_INT)
    page = s["tables"].long()[b, (row // size).clamp(max=stride - 1)]
    s["slots"] = torch.where(live, page * size + row % size, -1).to(_INT)
    return s


def _cache(case, s, gen):
    """Blocks of keys and values, one more than the pool has: where a plain store puts rows that have no slot."""
    s["kv_heads"], s["head_size"], s["heads"] = case["kv_heads"], case["head_size"], case["heads"]
    shape = (s["n_blocks"] + 1, s["size"], s["kv_heads"], s["head_size"])
    s["key"], s["value"] = _floats(gen, *shape), _floats(gen, *shape)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = _batch(case, seed, gen)
    s["op"] = case["op"]
    n, t = s["requests"], s["tokens"]
    ints = lambda k: torch.zeros(k, device="cuda", dtype=_INT)  # noqa: E731
    if case["op"] == "tables":
        need = sum(_blocks(a + b, s["size"]) - _blocks(a, s["size"]) for a, b in zip(*s["lengths"]))
        s["taken"] = torch.tensor([3], device="cuda", dtype=_INT)  # blocks that earlier steps took
        s["free"] = torch.cat([s["free"][:3], s["free"]])[:max(3, 3 + need - case["short"])].contiguous()
        s["tables"] = s["before"].clone()
        s["out"] = dict(lengths=ints(n), starts=ints(n + 1), positions=ints(t), slots=ints(t), taken=ints(1))
    else:
        _cache(case, s, gen)
        d, hq, hk = s["head_size"], s["heads"], s["kv_heads"]
    if case["op"] == "rope":
        if case["fused"]:  # the three products' results side by side
            qkv = _floats(gen, t, (hq + 2 * hk) * d)
            s["q"], s["k"], s["v"] = qkv[:, :hq * d], qkv[:, hq * d:(hq + hk) * d], qkv[:, (hq + hk) * d:]
        else:
            s["q"], s["k"], s["v"] = _floats(gen, t, hq * d), _floats(gen, t, hk * d), _floats(gen, t, hk * d)
        s["gammas"] = [(1.0 + _floats(gen, d, std=0.1).float()).to(_HALF) for _ in range(2)] if case["norms"] else None
        s["theta"], s["eps"] = case["theta"], 1e-5
        s["result"] = torch.zeros(t, hq * d, device="cuda", dtype=_HALF)
    elif case["op"] == "attention":
        s["q"] = _floats(gen, t, hq * d)
        s["scale"] = 1.0 / math.sqrt(d)
        s["result"] = torch.zeros(t, hq * d, device="cuda", dtype=_HALF)
    return s


# ---------------------------------------------------------------- the plain forms

def _plain_tables(s):
    size, prefix, tokens = s["size"], s["prefix"], s["tokens"]
    ctx, new = s["cached"].long(), s["counts"].long()
    ends = torch.cumsum(new, 0)
    begins = ends - new
    fits = (ctx + new <= s["stride"] * size) & (ends <= tokens)
    first = (ctx + size - 1) // size
    need = torch.where(fits, (ctx + new + size - 1) // size - first, 0)
    upto = torch.cumsum(need, 0)
    admitted = fits & ((need == 0) | (s["taken"] + upto <= s["free"].numel()))
    grid = torch.arange(s["stride"], device="cuda")[None, :]
    j = grid - first[:, None]
    at = (s["taken"] + (upto - need)[:, None] + j).clamp(0, s["free"].numel() - 1)
    tables = torch.where(admitted[:, None] & (j >= 0) & (j < need[:, None]), s["free"][at], s["tables"])
    t = torch.arange(tokens, device="cuda")
    b = torch.searchsorted(ends, t, right=True).clamp(max=s["requests"] - 1)
    row = ctx[b] + t - begins[b]
    live = (t < ends[-1]) & admitted[b]
    page = tables[b, (row // size).clamp(0, s["stride"] - 1)]
    starts = torch.cat([begins, ends[-1:]]).clamp(max=tokens)
    return [tables, torch.where(admitted, ctx + new, ctx).to(_INT), starts.to(_INT), torch.where(live, row + prefix, -1).to(_INT),
            torch.where(live, page * size + row % size, -1).to(_INT),
            (s["taken"] + torch.where(admitted, upto, 0).max()).to(_INT)]


def _plain_rope(s):
    d, t = s["head_size"], s["tokens"]
    half = d // 2
    rate = s["theta"] ** (-2.0 * torch.arange(half, device="cuda", dtype=torch.float64) / d)
    angle = s["positions"].double()[:, None, None] * rate
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    live = (s["positions"] >= 0)[:, None]

    def turned(x, gamma):
        y = x.float().view(t, -1, d)
        if gamma is not None:
            y = y * torch.rsqrt(torch.mean(y * y, -1, keepdim=True) + s["eps"]) * gamma.float()
        a, b = y[..., :half], y[..., half:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).view(t, -1).to(_HALF)

    gq, gk = s["gammas"] or (None, None)
    s["result"].copy_(torch.where(live, turned(s["q"], gq), s["result"]))
    rows = torch.where(s["slots"] >= 0, s["slots"].long(), s["n_blocks"] * s["size"])
    width = s["kv_heads"] * d
    s["key"].view(-1, width)[rows] = turned(s["k"], gk)
    s["value"].view(-1, width)[rows] = s["v"]
    return [s["result"], s["key"][:-1], s["value"][:-1]]


def _rows(s):
    """Cache row of every row of every request, up to the longest."""
    r = torch.arange(s["max_length"], device="cuda")
    page = s["tables"].long()[:, r // s["size"]].clamp(min=0)
    return page * s["size"] + r % s["size"]


def _plain_attention(s):
    d, hk, n, width = s["head_size"], s["kv_heads"], s["requests"], s["max_new"]
    g = s["heads"] // hk
    starts, t = s["starts"].long(), torch.arange(s["tokens"], device="cuda")
    at = (starts[:-1, None] + torch.arange(width, device="cuda")).clamp(max=s["tokens"] - 1)  # [request][its tokens]
    q = s["q"].view(s["tokens"], hk, g, d)[at].float().permute(0, 2, 1, 3, 4)  # [request][kv head][token][g][d]
    visible = (s["positions"].long()[at] - s["prefix"] + 1)[:, None, :, None, None]
    rows = _rows(s)
    k = s["key"].view(-1, hk, d)[rows].permute(0, 2, 3, 1).float()
    x = torch.matmul(q.reshape(n, hk, width * g, d), k).view(n, hk, width, g, -1) * s["scale"]
    del k
    x = torch.where(torch.arange(s["max_length"], device="cuda") < visible, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    if s["prefix"]:
        p = torch.arange(s["prefix"], device="cuda")
        shared = s["prefix_table"].long()[p // s["size"]] * s["size"] + p % s["size"]
        kp = s["key"].view(-1, hk, d)[shared].permute(1, 2, 0).float()
        y = torch.matmul(q.permute(1, 0, 2, 3, 4).reshape(hk, -1, d), kp).view(hk, n, width, g, -1) * s["scale"]
        y = y.permute(1, 0, 2, 3, 4)
        top = torch.maximum(top, y.amax(-1, keepdim=True))
    top = torch.where(top == -math.inf, 0.0, top)
    x = torch.exp(x - top)
    total = x.sum(-1, keepdim=True)
    v = s["value"].view(-1, hk, d)[rows].permute(0, 2, 1, 3).float()
    out = torch.matmul(x.reshape(n, hk, width * g, -1), v).view(n, hk, width, g, d)
    del v, x
    if s["prefix"]:
        y = torch.exp(y - top)
        total = total + y.sum(-1, keepdim=True)
        vp = s["value"].view(-1, hk, d)[shared].permute(1, 0, 2).float()
        z = torch.matmul(y.permute(1, 0, 2, 3, 4).reshape(hk, -1, s["prefix"]), vp)
        out = out + z.view(hk, n, width, g, d).permute(1, 0, 2, 3, 4)
    out = (out / total).permute(0, 2, 1, 3, 4).reshape(n * width, -1)
    b = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp(max=n - 1)
    mine = out[(b * width + t - starts[b]).clamp(max=n * width - 1)].to(_HALF)
    s["result"].copy_(torch.where((s["positions"] >= 0)[:, None], mine, s["result"]))
    return s["result"]


# ---------------------------------------------------------------- the framework's calls

_library = None


def _capi():
    global _library
    if _library is None:
        from managedllama2_amd import capi
        from managedllama2_amd.device import init
        init(0)
        _library = capi
    return _library


def _own_batch(capi, s, **other):
    """llama2_batch of the step: the pointers that a host keeps."""
    f = dict(block_tables=s["tables"], lengths=s["cached"], query_starts=s["starts"], positions=s["positions"], slots=s["slots"])
    f.update(other)
    return capi.Batch(prefix_table=s["prefix_table"].data_ptr() or None, n_requests=s["requests"], n_tokens=s["tokens"],
                      table_stride=s["stride"], prefix_length=s["prefix"], max_length=s["max_length"],
                      **{k: v.data_ptr() for k, v in f.items()})


def _own_cache(capi, s):
    return capi.PagedCache(key=s["key"].data_ptr(), value=s["value"].data_ptr(), block_stride=0, n_blocks=s["n_blocks"],
                           block_size=s["size"], n_kv_heads=s["kv_heads"], head_size=s["head_size"])


def _own(s):
    capi = _capi()
    if s["op"] == "tables":
        o = s["out"]
        batch = _own_batch(capi, s, lengths=o["lengths"], query_starts=o["starts"], positions=o["positions"], slots=o["slots"])
        capi.call("llama2_batch_tables", batch, s["cached"].data_ptr(), s["counts"].data_ptr(), s["free"].data_ptr(),
                  s["free"].numel(), s["taken"].data_ptr(), o["taken"].data_ptr(), s["size"])
        return [s["tables"], o["lengths"], o["starts"], o["positions"], o["slots"], o["taken"]]
    batch, cache = _own_batch(capi, s), _own_cache(capi, s)
    if s["op"] == "rope":
        gq, gk = [g.data_ptr() for g in s["gammas"]] if s["gammas"] else (None, None)
        capi.call("llama2_batch_qk_norm_rope", s["result"].data_ptr(), s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), gq,
                  gk, batch, cache, s["heads"], s["result"].stride(0), s["q"].stride(0), s["k"].stride(0), s["eps"], s["theta"])
        return [s["result"], s["key"][:-1], s["value"][:-1]]
    capi.call("llama2_batch_attention", s["result"].data_ptr(), s["q"].data_ptr(), batch, cache, s["heads"],
              s["result"].stride(0), s["q"].stride(0), s["scale"])
    return s["result"]


def run(state):
    if own:
        return _own(state)
    return {"tables": _plain_tables, "rope": _plain_rope, "attention": _plain_attention}[state["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    ctx, new = _lengths(case)
    n, t = case["requests"], sum(new)
    if case["op"] == "tables":
        size = case["block"]
        blocks = sum(_blocks(a + b, size) - _blocks(a, size) for a, b in zip(ctx, new))
        # lengths, counts, blocks taken, tables written; starts, lengths, positions, slots
        return dict(bytes=4 * (2 * n + 2 * blocks + 2 * n + 1 + 2 * (t + case["pad"])), flops=0)
    d, hq, hk = case["head_size"], case["heads"], case["kv_heads"]
    if case["op"] == "rope":  # q read and written, k and v read and written, position and slot
        return dict(bytes=t * (2 * (2 * hq + 4 * hk) * d + 8), flops=t * (hq + hk) * d * (7 if case["norms"] else 3))
    seen = sum(b * case["prefix"] + b * a + b * (b + 1) // 2 for a, b in zip(ctx, new))
    rows = case["prefix"] + sum(ctx) + t
    return dict(bytes=4 * rows * hk * d + 4 * t * hq * d, flops=4 * seen * hq * d)


# ---------------------------------------------------------------- 64 bits

def _exact_rope(s):
    d = s["head_size"]
    i = torch.arange(d // 2, device="cuda", dtype=torch.float64)
    angle = s["positions"].double().unsqueeze(1) / torch.pow(torch.tensor(s["theta"], device="cuda", dtype=torch.float64), 2.0 * i / d)
    wheel = torch.polar(torch.ones_like(angle), angle).unsqueeze(1)  # a pair of elements as one complex number
    live = torch.nonzero(s["positions"] >= 0).flatten()

    def head_by_head(x, gamma):
        y = x.double().unflatten(1, (-1, d))
        if gamma is not None:
            y = y / (y.square().sum(-1, keepdim=True) / d + s["eps"]).sqrt() * gamma.double()
        z = torch.view_as_real(torch.complex(y[..., :d // 2].contiguous(), y[..., d // 2:].contiguous()) * wheel)
        return torch.cat([z[..., 0], z[..., 1]], -1).flatten(1)

    gq, gk = s["gammas"] if s["gammas"] else (None, None)
    q, k = head_by_head(s["q"], gq), head_by_head(s["k"], gk)
    out, key, value = s["result"].double(), s["key"].double(), s["value"].double()
    out[live] = q[live]
    where = s["slots"].long()[live]
    key.flatten(2).flatten(0, 1)[where] = k[live]
    value.flatten(2).flatten(0, 1)[where] = s["v"].double()[live]
    return [out, key[:-1], value[:-1]]


def _exact_attention(s):
    d, g, size = s["head_size"], s["heads"] // s["kv_heads"], s["size"]
    out = s["result"].double()
    first = 0
    for b, (ctx, new) in enumerate(zip(*s["lengths"])):
        pages = s["tables"][b, :_blocks(ctx + new, size)].long()
        own_rows = lambda c: c[pages].flatten(0, 1)[:ctx + new]  # noqa: E731
        if s["prefix"]:
            shared = s["prefix_table"].long()
            both = lambda c: torch.cat([c[shared].flatten(0, 1)[:s["prefix"]], own_rows(c)])  # noqa: E731
        else:
            both = own_rows
        k, v = both(s["key"]), both(s["value"])
        seen = s["prefix"] + ctx + 1 + torch.arange(new, device="cuda")
        hidden = torch.arange(k.shape[0], device="cuda")[None, :] >= seen[:, None]
        for h in range(s["heads"]):
            q = s["q"][first:first + new, h * d:(h + 1) * d].double()
            x = (q @ k[:, h // g].double().t().contiguous() * s["scale"]).masked_fill(hidden, -math.inf)
            out[first:first + new, h * d:(h + 1) * d] = torch.softmax(x, 1) @ v[:, h // g].double()
        first += new
    return out


def exact(case, seed):
    if case["op"] == "tables":  # whole numbers
        return None
    s = prepare(case, seed)
    return _exact_rope(s) if case["op"] == "rope" else _exact_attention(s)
