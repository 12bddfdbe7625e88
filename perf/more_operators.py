"""The products, norms and answers of a step of several requests, as cases that can be timed and compared.

Around the rotation and the attention of such a step every layer has products of all tokens with int4 tensors, beside which
each request may have low-rank adapters of its own (several customers' fine-tunings of one model), and norms with the
residual in between; behind the last layer stand the probabilities that a server reports beside its tokens:

op "project"    llama2_batch_mat_mul_int4: up to four int4 tensors times the rows of all tokens, adapters and residual beside them.
op "swiglu"     llama2_batch_mat_mul_swiglu: gate and up projection, both with adapters, activation and product.
op "norm"       llama2_batch_residual_rmsnorm: a block's output normed (where the model does that), gated, scaled and added to the
                residual stream, and the norm in front of the next block.
op "log_probs"  llama2_batch_log_probs: log probabilities of given tokens, entropy and the most likely tokens of every row.

Sizes are those of synth.LLAMA2_7B (4096, 11008), synth.LLAMA2_13B (5120, 13824) and small models, with fewer key/value heads
too.  Activations, adapters and logits are fp16, weights int4 in groups of 128, as in the whole framework.
"""
import ctypes
import math

import torch

own = False

_HALF, _INT, _FLOAT = torch.float16, torch.int32, torch.float32
_GROUP = 128


def listed():
    return [
        # one request alone: latency of the output projection of 7B, with the residual and an adapter
        dict(name="project_one_token", op="project", tokens=1, pad=0, rows=4096, cols="4096", residual=True, adapters=8, max_rank=16,
             rank_lo=16, users=1, runs=1),
        # a decode step of 48 requests, captured for 56: q, k and v of 7B, most requests with one of 20 adapters
        dict(name="project_qkv_48", op="project", tokens=48, pad=8, rows=4096, cols="4096,4096,4096", residual=False, adapters=20,
             max_rank=32, rank_lo=8, users=40, runs=48),
        # a decode step of 13B without adapters: down projection onto the residual stream
        dict(name="project_down_13b_24", op="project", tokens=24, pad=0, rows=13824, cols="5120", residual=True, adapters=0, max_rank=0,
             rank_lo=0, users=0, runs=24),
        # nine prompts, q of 32 heads, k and v of 8, adapters of rank 64
        dict(name="project_prompts_1100", op="project", tokens=1100, pad=0, rows=4096, cols="4096,1024,1024", residual=False, adapters=6,
             max_rank=64, rank_lo=64, users=7, runs=9),
        # one request alone: the gated block's first half of 7B
        dict(name="swiglu_one_token", op="swiglu", tokens=1, pad=0, rows=4096, cols="11008", adapters=8, max_rank=16, rank_lo=16, users=1,
             runs=1),
        # 64 requests of 13B, each with an adapter of its own
        dict(name="swiglu_13b_64", op="swiglu", tokens=64, pad=0, rows=5120, cols="13824", adapters=64, max_rank=16, rank_lo=4, users=64,
             runs=64),
        # prompts of 7B
        dict(name="swiglu_prompts_700", op="swiglu", tokens=700, pad=0, rows=4096, cols="11008", adapters=4, max_rank=16, rank_lo=16,
             users=2, runs=5),
        # the norm behind a block of 7B: a decode step of 48, captured for 56
        dict(name="norm_48", op="norm", tokens=48, pad=8, size=4096, sandwich=False, gate=False, scale=1.0),
        # prompts of a model of 13B's width that norms before and after its blocks and gates them
        dict(name="norm_prompts_4000", op="norm", tokens=4000, pad=0, size=5120, sandwich=True, gate=True, scale=0.22),
        # the sampled tokens of one request, large vocabulary
        dict(name="log_probs_one", op="log_probs", tokens=1, pad=0, vocab=128000, given=1, top=5, temperature=0.8, masked=0.0),
        # a decode step of 48 requests that asked for five alternatives, vocabularies cut down by a grammar
        dict(name="log_probs_48", op="log_probs", tokens=48, pad=8, vocab=32000, given=1, top=5, temperature=1.0, masked=0.7),
        # scoring prompts: all rows, four candidates each and twenty alternatives
        dict(name="log_probs_prompts_2000", op="log_probs", tokens=2000, pad=0, vocab=32000, given=4, top=20, temperature=1.0, masked=0.0),
    ]


_MODELS = [(4096, 11008), (4096, 11008), (5120, 13824), (2048, 5632), (1024, 2816), (256, 640), (520, 1400)]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["project", "project", "project", "swiglu", "swiglu", "norm", "log_probs"])
    c = dict(op=op, tokens=_log_int(rng, 1, 1100), pad=rng.choice([0, 0, rng.randint(1, 20)]))
    dim, hidden = rng.choice(_MODELS)
    if op in ("project", "swiglu"):
        c["rows"] = dim
        c["residual"] = False
        if op == "swiglu":
            c["cols"] = str(hidden)
            c["tokens"] = min(c["tokens"], 700)
        else:
            kind = rng.choice(["qkv", "grouped", "out", "down"])
            c["rows"] = hidden if kind == "down" else dim
            c["cols"] = {"qkv": "%d,%d,%d" % (dim, dim, dim), "grouped": "%d,%d,%d" % (dim, dim // 4, dim // 4)}.get(kind, str(dim))
            c["residual"] = kind in ("out", "down")
        c["runs"] = rng.randint(1, min(c["tokens"], 64)) if c["tokens"] > 64 else c["tokens"]
        c["adapters"] = rng.choice([0, _log_int(rng, 1, 64)])
        c["max_rank"] = rng.choice([8, 16, 16, 32, 64]) if c["adapters"] else 0
        c["rank_lo"] = rng.randint(1, c["max_rank"]) if c["adapters"] else 0
        c["users"] = rng.randint(0, c["runs"]) if c["adapters"] else 0
    elif op == "norm":
        c.update(tokens=_log_int(rng, 1, 4000), size=rng.choice([dim, dim, hidden]), sandwich=rng.choice([True, False]),
                 gate=rng.choice([True, False]), scale=rng.choice([1.0, 0.22]))
        c["tokens"] = min(c["tokens"], 4000 * 5120 // c["size"])
    else:
        c.update(vocab=rng.choice([32000, 32000, 512, 1001, 50257, 128000]), given=rng.choice([0, 1, 1, 4, 9]), top=rng.choice([0, 1, 5, 20, 32]),
                 temperature=rng.choice([1.0, 1.0, 0.7, 1.5]), masked=rng.choice([0.0, 0.0, 0.5, 0.99]))
        c["tokens"] = min(_log_int(rng, 1, 2000), 2000 * 32000 // c["vocab"])
        if c["given"] + c["top"] == 0:
            c["given"] = 1
    return c


def _cols(case):
    return [int(v) for v in case["cols"].split(",")]


def _tensors(case):
    return _cols(case) * 2 if case["op"] == "swiglu" else _cols(case)


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, even steps of the logarithm."""
    return [round(math.exp(math.log(lo) + math.log(hi / lo) * (i / (n - 1) if n > 1 else 1.0))) for i in range(n)]


def _ranks(case):
    return _spread(case["rank_lo"], case["max_rank"], case["adapters"]) if case["adapters"] else []


def _runs(case):
    """Tokens of each request, and its adapter (-1: none): requests with adapters are spread among those without."""
    n = case["runs"]
    share = _spread(1, 40, n) if case["tokens"] > n else [1] * n
    total = sum(share)
    ends = [case["tokens"] * sum(share[:i + 1]) // total for i in range(n)]
    lengths = [b - a for a, b in zip([0] + ends, ends)]
    users = case["users"]
    adapter = [-1] * n
    for i in range(users):
        adapter[i * n // users] = i * 7 % case["adapters"]
    return lengths, adapter


# ---------------------------------------------------------------- inputs

def _floats(gen, *shape, std=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda", dtype=_FLOAT) * std).to(_HALF)


def _tensor(gen, k, n):
    """An int4 tensor: words of eight weights, zero points around 8, scales that give results of about 1 for inputs of 1."""
    groups, words = -(-k // _GROUP), -(-k // 32) * 4
    w = torch.randint(-2 ** 31, 2 ** 31 - 1, (n, words), generator=gen, device="cuda", dtype=torch.int64).to(_INT)
    z = torch.randint(6, 10, (n, -(-groups // 8) * 8), generator=gen, device="cuda", dtype=torch.int64)
    z = (z.view(n, -1, 8) << (4 * torch.arange(8, device="cuda"))).sum(-1)
    z = torch.where(z >= 2 ** 31, z - 2 ** 32, z).to(_INT)
    s = (0.5 + torch.rand(n, groups, generator=gen, device="cuda")) * (0.21 / math.sqrt(k))
    return dict(k=k, n=n, w=w, z=z.contiguous(), s=s.to(_HALF))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op, t = case["op"], case["tokens"] + case["pad"]
    s = dict(op=op, tokens=t)
    positions = torch.randint(0, 4000, (t,), generator=gen, device="cuda", dtype=torch.int64)
    s["positions"] = torch.where(torch.arange(t, device="cuda") < case["tokens"], positions, -1).to(_INT)
    if op in ("project", "swiglu"):
        k = case["rows"]
        s["x"], s["k"] = _floats(gen, t, k), k
        s["tensors"] = [_tensor(gen, k, n) for n in _tensors(case)]
        lengths, adapter = _runs(case)
        order = torch.randperm(len(lengths), generator=torch.Generator().manual_seed(int(seed))).tolist()
        ids = [a for i in order for a in [adapter[i]] * lengths[i]] + [-1] * case["pad"]
        s["ids"] = ids
        s["token_adapters"] = torch.tensor(ids, device="cuda", dtype=_INT)
        for x in s["tensors"]:
            x["adapters"] = None
            if case["adapters"]:
                a, r = case["adapters"], case["max_rank"]
                x["adapters"] = dict(down=_floats(gen, a, r, k, std=1 / math.sqrt(k)), up=_floats(gen, a, x["n"], r, std=0.05), rank=r,
                                     ranks=torch.tensor(_ranks(case), device="cuda", dtype=_INT),
                                     scales=torch.rand(a, generator=gen, device="cuda") + 1.0)
        outputs = _cols(case)
        s["residual"] = [_floats(gen, t, n, std=2.0) for n in outputs] if case.get("residual") else None
        s["result"] = [torch.zeros(t, n, device="cuda", dtype=_HALF) for n in outputs]
    elif op == "norm":
        n = case["size"]
        gamma = lambda: (1.0 + _floats(gen, n, std=0.1).float()).to(_HALF)  # noqa: E731
        s.update(size=n, residual=_floats(gen, t, n, std=3.0), input=_floats(gen, t, n), gamma=gamma(), scale=case["scale"], eps=1e-5,
                 input_gamma=gamma() if case["sandwich"] else None, gate=gamma() if case["gate"] else None)
        s["result"] = [torch.zeros(t, n, device="cuda", dtype=_HALF) for _ in range(2)]
    else:
        v = case["vocab"]
        x = _floats(gen, t, v, std=2.5)
        top = torch.randint(0, v, (t, 6), generator=gen, device="cuda", dtype=torch.int64)  # what the context makes likely
        x.scatter_add_(1, top, _floats(gen, t, 6, std=3.0).abs() + 5)
        if case["masked"]:
            x[torch.rand(t, v, generator=gen, device="cuda") < case["masked"]] = -math.inf
            x[:, :32] = _floats(gen, t, 32)
        s.update(x=x, vocab=v, given=case["given"], top=case["top"], temperature=case["temperature"])
        tokens = torch.randint(0, v, (t, case["given"]), generator=gen, device="cuda", dtype=torch.int64)
        if case["given"]:
            tokens[:, 0] = top[:, 0]
        s["given_tokens"] = tokens.to(_INT)
        s["result"] = [torch.zeros(t, case["given"], device="cuda"), torch.zeros(t, device="cuda"),
                       torch.zeros(t, case["top"], device="cuda", dtype=_INT), torch.zeros(t, case["top"], device="cuda")]
    return s


# ---------------------------------------------------------------- the plain forms

def _dequantised(x):
    """The tensor's values, [n][k]."""
    nibbles = 4 * torch.arange(8, device="cuda", dtype=_INT)
    w = ((x["w"][:, :, None] >> nibbles) & 15).view(x["n"], -1)[:, :x["k"]]
    groups = x["s"].shape[1]
    z = ((x["z"][:, :, None] >> nibbles) & 15).view(x["n"], -1)[:, :groups]
    group = torch.arange(x["k"], device="cuda") // _GROUP
    return (w - z[:, group]).float() * x["s"].float()[:, group]


def _plain_product(s, x):
    a = s["x"].float()
    y = torch.matmul(a, _dequantised(x).t())
    p = x["adapters"]
    if p:
        count, rank = p["ranks"].numel(), p["rank"]
        h = torch.matmul(a, p["down"].float().reshape(count * rank, -1).t()).view(-1, count, rank)
        mine = s["token_adapters"][:, None] == torch.arange(count, device="cuda")
        used = torch.arange(rank, device="cuda") < p["ranks"][:, None]
        h = torch.where(mine[:, :, None] & used, h * p["scales"][:, None], 0.0)  # own adapter and its ranks alone
        y = y + torch.matmul(h.view(-1, count * rank), p["up"].float().permute(0, 2, 1).reshape(count * rank, -1))
    return y


def _live(s):
    return (s["positions"] >= 0)[:, None]


def _plain_project(s):
    for i, x in enumerate(s["tensors"]):
        y = _plain_product(s, x)
        if s["residual"]:
            y = y + s["residual"][i].float()
        s["result"][i].copy_(torch.where(_live(s), y.to(_HALF), s["result"][i]))
    return s["result"]


def _plain_swiglu(s):
    g, u = _plain_product(s, s["tensors"][0]), _plain_product(s, s["tensors"][1])
    y = (g / (1.0 + torch.exp(-g)) * u).to(_HALF)
    s["result"][0].copy_(torch.where(_live(s), y, s["result"][0]))
    return s["result"]


def _plain_norm(s):
    y = s["input"].float()
    if s["input_gamma"] is not None:
        y = y * torch.rsqrt(torch.mean(y * y, -1, keepdim=True) + s["eps"]) * s["input_gamma"].float()
    if s["gate"] is not None:
        y = y * s["gate"].float()
    x = s["residual"].float() + y * s["scale"]
    n = x * torch.rsqrt(torch.mean(x * x, -1, keepdim=True) + s["eps"]) * s["gamma"].float()
    for out, v in zip(s["result"], (n, x)):
        out.copy_(torch.where(_live(s), v.to(_HALF), out))
    return s["result"]


def _plain_log_probs(s):
    live = s["positions"] >= 0
    x = s["x"].float() / s["temperature"]
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    lp = x - top - torch.log(total)
    p = e / total
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(1)
    order = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :s["top"]]  # equal ones: the lowest index first
    given = torch.gather(lp, 1, s["given_tokens"].long())
    new = [given, entropy, order.to(_INT), torch.gather(lp, 1, order)]
    for out, v in zip(s["result"], new):
        out.copy_(torch.where(live.view(-1, *[1] * (v.dim() - 1)), v, out))
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


def _pointer(t):
    return t.data_ptr() if t is not None and t.numel() else None


def _own_calls(capi, s):
    """Name and arguments of the call: what a host keeps from step to step."""
    batch = capi.Batch(positions=s["positions"].data_ptr(), n_requests=1, n_tokens=s["tokens"], max_length=1)
    if s["op"] == "norm":
        n, (out, residual_out) = s["size"], s["result"]
        return "llama2_batch_residual_rmsnorm", [out.data_ptr(), residual_out.data_ptr(), s["residual"].data_ptr(), s["input"].data_ptr(),
                                                 s["gamma"].data_ptr(), _pointer(s["input_gamma"]), _pointer(s["gate"]), batch, n, n, n, n, n,
                                                 s["scale"], s["eps"]]
    if s["op"] == "log_probs":
        given, entropy, tokens, top = s["result"]
        return "llama2_batch_log_probs", [_pointer(given), entropy.data_ptr(), _pointer(tokens), _pointer(top), s["x"].data_ptr(),
                                          _pointer(s["given_tokens"]), s["positions"].data_ptr(), s["tokens"], s["vocab"], s["vocab"],
                                          s["given"], s["top"], s["temperature"]]
    weights, adapters = [], []
    for x in s["tensors"]:
        weights.append(capi.QWeight(x["w"].data_ptr(), x["z"].data_ptr(), x["s"].data_ptr()))
        p = x["adapters"]
        adapters.append(ctypes.pointer(capi.Adapters(down=p["down"].data_ptr(), up=p["up"].data_ptr(), scales=p["scales"].data_ptr(),
                                                     ranks=p["ranks"].data_ptr(), n_adapters=p["ranks"].numel(), max_rank=p["rank"]))
                        if p else None)
    ids = s["token_adapters"].data_ptr()
    if s["op"] == "swiglu":
        n = s["tensors"][0]["n"]
        return "llama2_batch_mat_mul_swiglu", [s["result"][0].data_ptr(), s["x"].data_ptr(), *weights, s["k"], n, n, s["k"], *adapters, ids, batch]
    matrices = (capi.BatchMatrix * len(weights))()
    for i, x in enumerate(s["tensors"]):
        matrices[i] = capi.BatchMatrix(weight=weights[i], output=s["result"][i].data_ptr(), adapters=adapters[i], cols=x["n"],
                                       residual=s["residual"][i].data_ptr() if s["residual"] else None, output_stride=x["n"],
                                       residual_stride=x["n"])
    return "llama2_batch_mat_mul_int4", [matrices, len(weights), s["x"].data_ptr(), s["k"], s["k"], ids, batch]


def _own(s):
    capi = _capi()
    if "call" not in s:
        s["call"] = _own_calls(capi, s)
    name, args = s["call"]
    capi.call(name, *args)
    return s["result"]


def run(state):
    if own:
        return _own(state)
    return {"project": _plain_project, "swiglu": _plain_swiglu, "norm": _plain_norm, "log_probs": _plain_log_probs}[state["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    op, t = case["op"], case["tokens"]
    if op == "norm":  # input and residual stream read, residual stream and output written
        return dict(bytes=8 * t * case["size"], flops=t * case["size"] * (10 if case["sandwich"] else 6))
    if op == "log_probs":
        return dict(bytes=t * (2 * case["vocab"] + 4 + 8 * case["given"] + 8 * case["top"]), flops=6 * t * case["vocab"])
    k = case["rows"]
    lengths, adapter = _runs(case)
    ranks = _ranks(case)
    used = {a for a, n in zip(adapter, lengths) if a >= 0 and n}
    moved, flops = 2 * t * k + 8 * t, 0
    for n in _tensors(case):
        groups = -(-k // _GROUP)
        moved += n * (-(-k // 32) * 16 + 2 * groups + 4 * -(-groups // 8)) + sum(2 * ranks[a] * (k + n) for a in used)
        flops += 2 * t * k * n + sum(2 * m * ranks[a] * (k + n) for a, m in zip(adapter, lengths) if a >= 0)
    moved += sum(2 * t * n * (2 if case.get("residual") else 1) for n in _cols(case))
    return dict(bytes=moved, flops=flops)


# ---------------------------------------------------------------- 64 bits

def _exact_tensor(x):
    """[k][n], group by group."""
    words = x["w"].to(torch.int64) & 0xFFFFFFFF
    n = torch.stack([words >> 4 * i & 15 for i in range(8)], 2).flatten(1).double()
    zeros = x["z"].to(torch.int64) & 0xFFFFFFFF
    z = torch.stack([zeros >> 4 * i & 15 for i in range(8)], 2).flatten(1).double()
    for g in range(x["s"].shape[1]):
        part = n[:, g * _GROUP:(g + 1) * _GROUP]
        part -= z[:, g:g + 1]
        part *= x["s"][:, g:g + 1].double()
    return n[:, :x["k"]].t().contiguous()


def _exact_product(s, x):
    rows = s["x"].double()
    y = rows @ _exact_tensor(x)
    p = x["adapters"]
    if p is None:
        return y
    for a in sorted(set(s["ids"]) - {-1}):  # adapter by adapter
        at = torch.tensor([i for i, b in enumerate(s["ids"]) if b == a], device="cuda")
        r = int(p["ranks"][a])
        low = rows[at] @ p["down"][a, :r].double().t().contiguous()
        y[at] += (low @ p["up"][a, :, :r].double().t().contiguous()) * p["scales"][a].double()
    return y


def exact(case, seed):
    s = prepare(case, seed)
    live = torch.nonzero(s["positions"] >= 0).flatten()
    out = [r.double() for r in s["result"]]
    if case["op"] == "project":
        for i, x in enumerate(s["tensors"]):
            y = _exact_product(s, x)
            out[i][live] = (y + s["residual"][i].double() if s["residual"] else y)[live]
    elif case["op"] == "swiglu":
        g, u = (_exact_product(s, x) for x in s["tensors"])
        out[0][live] = (g * torch.sigmoid(g) * u)[live]
    elif case["op"] == "norm":
        def normed(v, gamma):
            return v / (v.square().sum(1, keepdim=True) / s["size"] + s["eps"]).sqrt() * gamma.double()
        y = s["input"].double()
        if s["input_gamma"] is not None:
            y = normed(y, s["input_gamma"])
        if s["gate"] is not None:
            y = y * s["gate"].double()
        x = s["residual"].double() + s["scale"] * y
        out[0][live], out[1][live] = normed(x, s["gamma"])[live], x[live]
    else:
        for row in live.tolist():
            x = s["x"][row].double() / s["temperature"]
            lp = torch.log_softmax(x, 0)
            out[0][row] = lp[s["given_tokens"][row].long()]
            seen = lp[lp > -math.inf]
            out[1][row] = -(seen.exp() * seen).sum()
            if s["top"]:
                out[3][row] = torch.topk(lp, s["top"])[0]
        out[2] = None
    return out
