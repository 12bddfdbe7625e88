"""Whole steps of several requests through the operators of such steps, from the embedding to the log probabilities: a small model,
prompts and then captured steps of single tokens, some requests with low-rank adapters; held to a forward pass in 64 bits and, without
adapters, to the framework's decoder of one sequence."""
import ctypes as C
import math

import numpy as np
import pytest

import product_util as pu
from managedllama2_amd import capi, hostlib, synth
from managedllama2_amd.device import Adapters, DeviceVariable, PagedCache, QWeight, RequestBatch, init
from managedllama2_amd.modules import (BatchAttention, BatchLogProbs, BatchMatMulInt4, BatchMatMulSwiGLU, BatchQKNormRoPE, BatchResidualRMSNorm,
                                       BatchTables, Embedding, MatVec)
from managedllama2_amd.transformer import Transformer

pytestmark = pytest.mark.gpu
CFG = dict(dim=256, hidden_dim=640, n_layers=2, n_heads=2, n_kv_heads=2, vocab_size=512, seq_len=64, rope_theta=10000.0)
DIM, HIDDEN, HEADS, D, VOCAB = 256, 640, 2, 128, 512
SHAPES = dict(q=(DIM, DIM), k=(DIM, DIM), v=(DIM, DIM), o=(DIM, DIM), gate=(DIM, HIDDEN), up=(DIM, HIDDEN), down=(HIDDEN, DIM))
RANKS, MAX_RANK = [4, 16, 9], 16
up = pu.up


def adapters_of(rng):
    """Host arrays per layer and tensor: (down, up, ranks, scales)."""
    pools = []
    for _ in range(CFG["n_layers"]):
        layer = {}
        for name, (K, N) in SHAPES.items():
            p = pu.Pool(rng, RANKS, MAX_RANK, K, N)
            layer[name] = (p.down.reshape(3, MAX_RANK, K), p.up.reshape(3, N, MAX_RANK), p.ranks, p.scales)
        pools.append(layer)
    return pools


class Model:
    def __init__(self, model, pools, requests, tokens):
        init(0)
        self.requests, self.tokens = requests, tokens
        self.layers = [{n: QWeight.from_host(*L[n]) for n in SHAPES} | {n: up(L[n]) for n in ("rms_att", "rms_ffn")} for L in model["layers"]]
        self.pools = [{n: Adapters.from_host(d, u, r, s) for n, (d, u, r, s) in P.items()} for P in pools]
        self.embedding, self.classifier, self.final = up(model["embedding"]), up(model["classifier"]), up(model["rms_final"])
        self.caches = [PagedCache(24, 8, HEADS, D) for _ in self.layers]
        self.batch = RequestBatch(requests, tokens, 6, 48)
        self.free, self.counts = up(np.arange(24, dtype=np.int32)[::-1].copy()), DeviceVariable.zeros(np.int32, requests)
        halfs = lambda n: DeviceVariable.zeros(np.float16, tokens * n)  # noqa: E731
        self.x, self.xb, self.q, self.k, self.v, self.att, self.y = (halfs(DIM) for _ in range(7))
        self.h, self.logits = halfs(HIDDEN), halfs(VOCAB)
        self.ids = DeviceVariable.from_host(np.full(tokens, -1, np.int32))
        self.input, self.given, self.top = (DeviceVariable.zeros(np.int32, n) for n in (tokens, tokens, tokens * 4))
        self.lp, self.entropy, self.top_lp = (DeviceVariable.zeros(np.float32, n) for n in (tokens, tokens, tokens * 4))
        self.mat, self.swiglu, self.norm, self.answers = BatchMatMulInt4(), BatchMatMulSwiGLU(), BatchResidualRMSNorm(), BatchLogProbs()
        self.row = [DeviceVariable.window(self.x, t * DIM * 2, np.float16, DIM) for t in range(tokens)]
        self.out = [(DeviceVariable.window(self.logits, t * VOCAB * 2, np.float16, VOCAB), DeviceVariable.window(self.xb, t * DIM * 2, np.float16, DIM))
                    for t in range(tokens)]

    def issue(self):
        b, ids = self.batch, self.ids
        BatchTables().Forward(b, self.counts, self.free, 8)
        for t in range(self.tokens):
            Embedding().Forward(self.row[t], self.embedding, DIM, self.input, t)
        self.norm.Forward(self.xb, self.x, None, self.layers[0]["rms_att"], DIM, b)
        for i, (L, P, cache) in enumerate(zip(self.layers, self.pools, self.caches)):
            self.mat.Forward([(o, L[n], DIM, None, P[n]) for o, n in ((self.q, "q"), (self.k, "k"), (self.v, "v"))], self.xb, DIM, b, ids)
            BatchQKNormRoPE().Forward(self.q, self.q, self.k, self.v, b, cache, HEADS, 10000.0)
            BatchAttention().Forward(self.att, self.q, b, cache, HEADS, D ** -0.5)
            self.mat.Forward([(self.x, L["o"], DIM, self.x, P["o"])], self.att, DIM, b, ids)
            self.norm.Forward(self.xb, self.x, None, L["rms_ffn"], DIM, b)
            self.swiglu.Forward(self.h, self.xb, L["gate"], L["up"], DIM, HIDDEN, b, ids, P["gate"], P["up"])
            self.mat.Forward([(self.y, L["down"], DIM, None, P["down"])], self.h, HIDDEN, b, ids)
            after = self.layers[i + 1]["rms_att"] if i + 1 < len(self.layers) else self.final
            self.norm.Forward(self.xb, self.x, self.y, after, DIM, b)
        for o, x in self.out:
            MatVec().Forward(o, x, self.classifier, DIM, VOCAB)
        self.answers.Forward(self.lp, self.entropy, self.top, self.top_lp, self.logits, self.tokens, VOCAB, self.given, 1, 4, 1.0, b.positions)


def forward(model, pools, tokens, adapter):
    """Logits of every token of one sequence, in 64 bits."""
    n = len(tokens)
    f = lambda a: a.astype(np.float64)  # noqa: E731
    x = f(model["embedding"]).reshape(VOCAB, DIM)[tokens]
    norm = lambda v, g: v / np.sqrt((v * v).mean(-1, keepdims=True) + 1e-5) * f(g)  # noqa: E731
    angle = np.arange(n)[:, None] * 10000.0 ** (-2 * np.arange(64) / D)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    turn = lambda v: np.concatenate([v[..., :64] * c - v[..., 64:] * s, v[..., :64] * s + v[..., 64:] * c], -1)  # noqa: E731
    for L, P in zip(model["layers"], pools):
        def mul(v, name):
            K, N = SHAPES[name]
            y = v @ pu.dequantised(L[name], K, N).T
            if adapter >= 0:
                d, u, r, scale = P[name]
                r = r[adapter]
                y = y + float(scale[adapter]) * (v @ f(d[adapter, :r]).T) @ f(u[adapter, :, :r]).T
            return y
        a = norm(x, L["rms_att"])
        q, k, v = (mul(a, name).reshape(n, HEADS, D) for name in "qkv")
        q, k = turn(q), turn(k)
        scores = np.einsum("thd,shd->hts", q, k) * D ** -0.5
        scores[:, np.triu(np.ones((n, n), bool), 1)] = -np.inf
        p = np.exp(scores - scores.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        x = x + mul(np.einsum("hts,shd->thd", p, v).reshape(n, DIM), "o")
        a = norm(x, L["rms_ffn"])
        g = mul(a, "gate")
        x = x + mul(g / (1 + np.exp(-g)) * mul(a, "up"), "down")
    return norm(x, model["rms_final"]) @ f(model["classifier"]).reshape(VOCAB, DIM).T


def small_model():
    """Results of the products of about the size of their inputs, so that neither block drowns the other."""
    model = synth.random_model(CFG, seed=41, rms_random=True)
    for L in model["layers"]:
        for name in SHAPES:
            L[name][2][:] = (L[name][2].astype(np.float32) * np.float32(0.08 * math.sqrt(DIM / SHAPES[name][0]))).astype(np.float16)
    model["embedding"] = (model["embedding"].astype(np.float32) * 50).astype(np.float16)
    model["classifier"] = (model["classifier"].astype(np.float32) * 8).astype(np.float16)
    return model


def check_answers(m, t, what):
    logits = m.logits.to_host().reshape(-1, VOCAB)[t]
    lp, entropy = pu.log_probs(logits, 1.0)
    given = int(m.given[t])
    assert abs(float(m.lp[t]) - lp[given]) < 1e-5 and abs(float(m.entropy[t]) - entropy) < 1e-5, what
    assert np.array_equal(m.top.to_host().reshape(-1, 4)[t], pu.top_tokens(logits, 4)), what


def test_prompts_then_captured_steps_with_adapters():
    rng = synth.rng_for(1801)
    model, pools = small_model(), adapters_of(rng)
    prompts, adapter, pad = [7, 1, 12, 3, 20], [0, -1, 2, 1, 0], 2
    requests = len(prompts)
    text = [rng.integers(3, VOCAB, 40).astype(np.int32) for _ in range(requests)]
    want = [forward(model, pools, t, a) for t, a in zip(text, adapter)]
    biggest = [np.abs(w).max(-1) for w in want]
    m = Model(model, pools, requests, sum(prompts) + pad)
    m.input.copy_to_device(np.concatenate([t[:n] for t, n in zip(text, prompts)] + [np.zeros(pad, np.int32)]))
    m.ids.copy_to_device(np.concatenate([np.full(n, a) for a, n in zip(adapter, prompts)] + [np.full(pad, 1)]).astype(np.int32))
    m.counts.copy_to_device(np.array(prompts, np.int32))
    m.given.copy_to_device(rng.integers(0, VOCAB, m.tokens).astype(np.int32))
    m.issue()
    got, at = m.logits.to_host().reshape(-1, VOCAB).astype(np.float64), 0
    # fp16 between the modules: 13 roundings of half a step, 2^-11 of a vector's size at most, each as large at the end as the rest of the
    # network makes it; the residual stream and the norms keep that near 1: 13 * 2^-11 = 6.3e-3 where all point one way
    for b, n in enumerate(prompts):
        err = np.abs(got[at:at + n] - want[b][:n]).max(-1) / biggest[b][:n]
        assert err.max() <= 1e-2, (b, err.max())
        at += n
    for t in range(0, sum(prompts), 5):
        check_answers(m, t, t)
    d = Model(model, pools, requests, requests + pad)  # steps of single tokens over the same caches
    d.caches, d.free, d.pools = m.caches, m.free, m.pools
    for name in ("blockTables", "lengths", "taken"):
        setattr(d.batch, name, getattr(m.batch, name))
    position, graph = list(prompts), C.c_void_p()
    for step in range(12):
        counts = (rng.random(requests) < 0.8).astype(np.int32)
        live = np.flatnonzero(counts)
        fill = lambda v, rest: np.concatenate([v, np.full(d.tokens - len(v), rest)]).astype(np.int32)  # noqa: E731
        d.counts.copy_to_device(counts)
        d.input.copy_to_device(fill([text[b][position[b]] for b in live], 5))
        d.ids.copy_to_device(fill([adapter[b] for b in live], 2))
        d.given.copy_to_device(rng.integers(0, VOCAB, d.tokens).astype(np.int32))
        if step == 1:
            capi.call("llama2_graph_begin_capture")
            try:
                d.issue()
            finally:
                capi.call("llama2_graph_end_capture", C.byref(graph))
        if step == 0 or step % 5 == 4:
            d.issue()
        else:
            capi.call("llama2_graph_launch", graph)
        got = d.logits.to_host().reshape(-1, VOCAB).astype(np.float64)
        for t, b in enumerate(live):
            err = np.abs(got[t] - want[b][position[b]]).max() / biggest[b][position[b]]
            assert err <= 1e-2, (step, b, err)
            check_answers(d, t, (step, b))
            position[b] += 1
    capi.call("llama2_graph_destroy", graph)


def test_without_adapters_the_same_as_the_decoder_of_one_sequence():
    rng = synth.rng_for(1802)
    model, pools = small_model(), adapters_of(rng)
    text = rng.integers(3, VOCAB, 18).astype(np.int32)
    m = Model(model, pools, 1, len(text))
    m.input.copy_to_device(text)
    m.counts.copy_to_device(np.array([len(text)], np.int32))
    m.issue()
    got = m.logits.to_host().reshape(-1, VOCAB).astype(np.float64)
    t = Transformer(dict(CFG), model, mode=capi.DECODE_MODULES)
    t.runstate.tokens.copy_to_device(text)
    for pos in range(len(text)):
        t.Forward(pos, pos + 1)
        one = t.runstate.logits.to_host().astype(np.float64)
        # both are within 1e-2 of 64 bits (above); this is what two such passes differ by
        assert np.abs(one - got[pos]).max() <= 2e-2 * np.abs(one).max(), pos
    t.close()


def test_cpp_module_classes_do_the_same():
    rng = synth.rng_for(1803)
    model, pools = small_model(), adapters_of(rng)
    m = Model(model, pools, 3, 30)
    m.counts.copy_to_device(np.array([9, 1, 17], np.int32))
    BatchTables().Forward(m.batch, m.counts, m.free, 8)
    L, P = m.layers[0], m.pools[0]["o"]
    att, x0 = (rng.standard_normal((30, DIM)).astype(np.float16) for _ in range(2))
    m.att.copy_to_device(att)
    m.ids.copy_to_device(rng.integers(-1, 3, 30).astype(np.int32))
    m.given.copy_to_device(rng.integers(0, VOCAB, 30).astype(np.int32))
    m.logits.copy_to_device(rng.standard_normal(30 * VOCAB).astype(np.float16))
    post, after = (up((1 + 0.1 * rng.standard_normal(DIM)).astype(np.float16)) for _ in range(2))
    written = (m.x, m.xb, m.h, m.y, m.lp, m.entropy, m.top)

    def fresh():
        m.x.copy_to_device(x0)
        for v in written[1:]:
            capi.call("llama2_memset", v.ptr, 0x33, v.nbytes)

    fresh()
    m.mat.Forward([(m.x, L["o"], DIM, m.x, P)], m.att, DIM, m.batch, m.ids)
    m.norm.Forward(m.xb, m.x, None, L["rms_ffn"], DIM, m.batch)
    m.swiglu.Forward(m.h, m.xb, L["gate"], L["up"], DIM, HIDDEN, m.batch)
    m.mat.Forward([(m.y, L["down"], DIM)], m.h, HIDDEN, m.batch)
    m.norm.Forward(m.xb, m.x, m.y, after, DIM, m.batch, inputGamma=post)
    m.answers.Forward(m.lp, m.entropy, m.top, None, m.logits, 30, VOCAB, m.given, 1, 4, 1.0, m.batch.positions)
    want = [v.to_host() for v in written]
    fresh()
    w = capi.LayerWeights(output=L["o"].struct(), gate=L["gate"].struct(), up=L["up"].struct(), down=L["down"].struct(),
                          rms_feed_forward=L["rms_ffn"].ptr)
    args = lambda hidden: (m.batch, w, m.att, m.x, m.xb, m.h, m.y, DIM, hidden, P, m.ids, post, after, m.logits, VOCAB, m.given, m.lp,  # noqa: E731
                           m.entropy, m.top, 4)
    hostlib.batch_block(*args(HIDDEN))
    for a, v in zip(want, written):
        assert np.array_equal(a.view(np.uint8), v.to_host().view(np.uint8))
    with pytest.raises(hostlib.HostError, match="cols"):
        hostlib.batch_block(*args(HIDDEN + 4))
