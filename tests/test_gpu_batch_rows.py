"""Residual with norms and log probabilities of many rows against 64-bit restatements (product_util.py)."""
import ctypes as C

import numpy as np
import pytest

import product_util as pu
from managedllama2_amd import capi, synth
from managedllama2_amd.device import init

pytestmark = pytest.mark.gpu
up = pu.up


@pytest.fixture(autouse=True, scope="module")
def ready():
    init(0)


def rng(*stream):
    return synth.rng_for(1750, *stream)


# ---------------------------------------------------------------- residual and norms
def norm_case(g, tokens, size, pad=0, extra=0, x=True, gamma=True, input_gamma=False, gate=False, scale=1.0, eps=1e-5, std=1.0):
    t = tokens + pad
    rows = lambda s: (g.standard_normal((t, size + extra)) * s).astype(np.float16)  # noqa: E731
    vec = lambda use: (1 + 0.2 * g.standard_normal(size)).astype(np.float16) if use else None  # noqa: E731
    c = dict(residual=rows(2 * std), x=rows(std) if x else None, gamma=vec(gamma), input_gamma=vec(input_gamma), gate=vec(gate), scale=scale,
             eps=eps, size=size, extra=extra, tokens=t)
    c["positions"] = np.where(np.arange(t) < tokens, np.arange(t), -1).astype(np.int32)
    for name in ("residual", "x"):
        if c[name] is not None:
            c[name][tokens:] = np.nan
    return c


def norm_run(c, output=True, residual_output=True, in_place=False):
    d = {k: up(c[k]) if c[k] is not None else None for k in ("residual", "x", "gamma", "input_gamma", "gate", "positions")}
    ptr = lambda v: v.ptr if v is not None else None  # noqa: E731
    stride = c["size"] + c["extra"]
    guard = lambda: up(np.full((c["tokens"], stride), pu.GUARD, np.float16))  # noqa: E731
    out = (d["x"] if in_place else guard()) if output and c["gamma"] is not None else None
    res = (d["residual"] if in_place else guard()) if residual_output else None
    batch = capi.Batch(positions=d["positions"].ptr, n_requests=1, n_tokens=c["tokens"], max_length=1)
    capi.call("llama2_batch_residual_rmsnorm", ptr(out), ptr(res), d["residual"].ptr, ptr(d["x"]), ptr(d["gamma"]), ptr(d["input_gamma"]),
              ptr(d["gate"]), batch, c["size"], stride, stride, stride, stride, c["scale"], c["eps"])
    return [v.to_host().reshape(c["tokens"], stride) if v is not None else None for v in (out, res)]


def norm_check(c, **how):
    got = norm_run(c, **how)
    live, n = c["positions"] >= 0, c["size"]
    want = pu.norm_rows(c["residual"][live, :n], None if c["x"] is None else c["x"][live, :n], c["gamma"], c["input_gamma"], c["gate"],
                        float(np.float32(c["scale"])), float(np.float32(c["eps"])))
    for g, w, before in zip(got, want, (c["x"], c["residual"])):
        if g is None:
            continue
        untouched = before if how.get("in_place") else np.full_like(g, pu.GUARD)
        assert np.array_equal(g[~live].view(np.uint16), untouched[~live].view(np.uint16))
        assert np.array_equal(g[:, n:].view(np.uint16), untouched[:, n:].view(np.uint16))
        err = np.abs(g[live, :n].astype(np.float64) - w[0])
        worst = np.unravel_index(np.argmax(err - w[1]), err.shape)
        assert (err <= w[1]).all(), (worst, g[live, :n][worst], w[0][worst], w[1][worst])
    return got


@pytest.mark.parametrize("size", [8, 64, 520, 2048, 2056, 4096, 5120, 8192, 8200, 13824, 16384, 16392, 32768, 65536])
def test_sizes(size):
    for i, kw in enumerate((dict(), dict(input_gamma=True, gate=True, scale=0.22, extra=16), dict(gate=True, scale=-1.5), dict(input_gamma=True),
                            dict(x=False), dict(gamma=False))):
        norm_check(norm_case(rng(1, size, i), 3, size, pad=i % 3, **kw), residual_output=i != 4)


@pytest.mark.parametrize("tokens", [1, 2, 63, 300, 1500])
def test_numbers_of_rows(tokens):
    norm_check(norm_case(rng(2, tokens), tokens, 512, pad=5, input_gamma=True))
    norm_check(norm_case(rng(3, tokens), tokens, 4096, pad=1))


def test_results_larger_than_the_caches():
    c = norm_case(rng(16), 2100, 4096, pad=3, input_gamma=True, gate=True, scale=0.5)
    apart, place = norm_check(c), norm_check(c, in_place=True)
    for a, b in zip(apart, place):
        assert np.array_equal(a[:2100].view(np.uint16), b[:2100].view(np.uint16))


def test_in_place():
    c = norm_case(rng(4), 40, 4096, pad=4, input_gamma=True, gate=True, extra=8)
    apart, place = norm_check(c), norm_check(c, in_place=True)
    for a, b in zip(apart, place):
        assert np.array_equal(a[:40, :4096].view(np.uint16), b[:40, :4096].view(np.uint16))


def test_values_at_the_ends():
    c = norm_case(rng(5), 6, 1024, input_gamma=True)
    c["x"][0] = 0  # eps keeps its norm finite
    c["residual"][1] = 0
    c["x"][1] = 0
    c["x"][2] = 60000  # squares beyond fp16
    c["x"][3] = 2.0 ** -24
    norm_check(c)
    c["x"][4, 7] = np.inf  # this row only
    c["x"][5, 9] = np.nan
    got = norm_run(c)
    clean = norm_run({**c, "x": np.where(np.isfinite(c["x"]), c["x"], 0).astype(np.float16)})
    for g, w in zip(got, clean):
        assert np.array_equal(g[:4].view(np.uint16), w[:4].view(np.uint16))
        assert np.isnan(g[4:]).any(1).all()


def test_the_same_as_the_module_of_one_row():
    """Without an input: llama2_rmsnorm of every row, which rounds the same number once."""
    c = norm_case(rng(6), 5, 4096, x=False)
    got, _ = norm_run(c, residual_output=False)
    for t in range(5):
        x, g, o = up(c["residual"][t]), up(c["gamma"]), up(np.zeros(4096, np.float16))
        capi.call("llama2_rmsnorm", o.ptr, x.ptr, g.ptr, 4096, 1e-5)
        (want, bound), _ = pu.norm_rows(c["residual"][t:t + 1], None, c["gamma"], None, None, 1.0, float(np.float32(1e-5)))
        assert (np.abs(o.to_host() - want) <= bound).all() and (np.abs(got[t] - want) <= bound).all()


# ---------------------------------------------------------------- log probabilities
def lp_run(x, tokens, n_top, temperature=1.0, positions=None, stride=None, offset=0, skip=()):
    rows, vocab = x.shape
    stride = stride or vocab
    buffer = np.full(offset + (rows - 1) * stride + vocab, np.nan, np.float16)  # NaN in front of the rows and between them
    for r in range(rows):
        buffer[offset + r * stride:offset + r * stride + vocab] = x[r]
    d, n = up(buffer), tokens.shape[1]
    outs = dict(lp=np.full((rows, n), 5.0, np.float32), h=np.full(rows, 5.0, np.float32), top=np.full((rows, n_top), -9, np.int32),
                tlp=np.full((rows, n_top), 5.0, np.float32))
    dev = {k: up(v) if v.size and k not in skip else None for k, v in outs.items()}
    ptr = lambda v: v.ptr if v is not None else None  # noqa: E731
    dt, dp = up(tokens) if n else None, up(positions) if positions is not None else None
    capi.call("llama2_batch_log_probs", ptr(dev["lp"]), ptr(dev["h"]), ptr(dev["top"]), ptr(dev["tlp"]), d.ptr + 2 * offset, ptr(dt), ptr(dp),
              rows, vocab, stride, n, n_top, temperature)
    return {k: dev[k].to_host().reshape(v.shape) if dev[k] is not None else None for k, v in outs.items()}


def lp_check(x, tokens, n_top, temperature=1.0, positions=None, **how):
    got = lp_run(x, tokens, n_top, temperature, positions, **how)
    for r in range(len(x)):
        if positions is not None and positions[r] < 0:
            for k, v in got.items():
                if v is not None:
                    assert (v[r] == (-9 if k == "top" else 5)).all()
            continue
        lp, h = pu.log_probs(x[r], temperature)
        # the difference to the largest logit is exact but for 2^-24 of it, so is its product with 1 / temperature (twice); the
        # exponentials: 2^-21 of each with the same in front of them (|d| e^d <= 0.37), their sum over v terms, the logarithm
        v = x.shape[1]
        finite = lambda a: np.where(np.isfinite(a), np.abs(a), 0)  # noqa: E731
        spread = finite((x[r].astype(np.float64) - np.max(finite(x[r]))) / temperature)
        share = (v / 16 + 32) * 2.0 ** -24 + 2.0 ** -20

        def close(g, w, what):
            w = np.asarray(w, np.float64)
            bound = 2.0 ** -22 * finite(w) + share + 2.0 ** -22 * spread.max()
            same = (np.isnan(g) & np.isnan(w)) | (g == w)
            with np.errstate(invalid="ignore"):
                ok = same | (np.abs(g - w) <= bound)
            assert ok.all(), (what, r, g, w)

        if got["lp"] is not None:
            close(got["lp"][r], [lp[t] if 0 <= t < v else -np.inf for t in tokens[r]], "log probability")
        if got["h"] is not None:
            close(got["h"][r], h, "entropy")
        if got["top"] is not None:
            want = pu.top_tokens(x[r], n_top)
            assert np.array_equal(got["top"][r], want), (r, got["top"][r], want)
            if got["tlp"] is not None:
                close(got["tlp"][r], np.where(want >= 0, lp[np.maximum(want, 0)], -np.inf), "of a top token")
    return got


def logits(g, rows, vocab, std=2.5):
    return (g.standard_normal((rows, vocab)) * std).astype(np.float16)


@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 64, 65, 512, 1000, 1001, 1024, 1025, 8191, 8192, 32000, 32768, 32769, 50257, 128000])
@pytest.mark.parametrize("rows", [1, 5])
def test_vocabularies(vocab, rows):
    g = rng(7, vocab, rows)
    x = logits(g, rows, vocab)
    lp_check(x, g.integers(0, vocab, (rows, 3)).astype(np.int32), 20, 0.8)
    lp_check(x, g.integers(-2, vocab + 2, (rows, 2)).astype(np.int32), 64, stride=vocab + 3, offset=5)


@pytest.mark.parametrize("n_top", [0, 1, 2, 5, 32, 63, 64])
@pytest.mark.parametrize("n_given", [0, 1, 9, 1024])
def test_numbers_of_answers(n_top, n_given):
    g = rng(8, n_top, n_given)
    x = logits(g, 3, 3000)
    lp_check(x, g.integers(0, 3000, (3, n_given)).astype(np.int32), n_top, positions=np.array([4, -1, 0], np.int32))
    for skip in (("h",), ("tlp",)):
        if n_top or n_given:
            lp_check(x, g.integers(0, 3000, (3, n_given)).astype(np.int32), n_top, skip=skip)


@pytest.mark.parametrize("vocab", [5, 100, 3000, 32000, 40000])
def test_equal_logits_come_by_index(vocab):
    g = rng(9, vocab)
    t = np.zeros((1, 1), np.int32)
    for levels in (1, 2, 3, 50):
        x = g.integers(0, levels, (4, vocab)).astype(np.float16)
        x[1] *= -1  # -0 beside 0
        x[2, ::2] = -0.0
        lp_check(x, np.repeat(t, 4, 0), 64)
    x = np.zeros((2, vocab), np.float16)  # few above many equal ones, the last ones
    x[0, -3:] = 1
    x[1, vocab // 2:] = -1
    lp_check(x, np.repeat(t, 2, 0), 40)


@pytest.mark.parametrize("vocab", [9, 1000, 32000, 60000])
def test_masked_logits(vocab):
    g = rng(10, vocab)
    x = logits(g, 9, vocab)
    x[0] = -np.inf  # nothing is left
    x[1, 1:] = -np.inf  # the first one
    x[2, :-1] = -np.inf  # the last one
    x[3, g.random(vocab) < 0.9] = -np.inf
    x[4] = -65504  # masked with the lowest number, one left
    x[4, vocab // 2] = 3
    x[5] = -65504  # all of them
    x[6, vocab // 3] = np.inf
    x[7, ::3] = np.nan
    x[8] = np.nan
    tokens = g.integers(0, vocab, (9, 4)).astype(np.int32)
    tokens[:, 0] = vocab // 2
    lp_check(x, tokens, 12)
    lp_check(x, tokens, 64, 0.1)


@pytest.mark.parametrize("vocab", [3, 64, 700, 4097, 32000, 45000])
def test_few_or_many_logits_beside_masked_and_nan(vocab):
    """Every number of logits that are left, with NaN among them: the likeliest tokens are found in other ways then."""
    g = rng(14, vocab)
    rows = 12
    x = np.full((rows, vocab), -np.inf, np.float16)
    for r in range(rows):
        left = [0, 1, 2, 5, 63, 64, 65, 200, 2047, 2049, 6000, vocab][r]
        at = g.permutation(vocab)[:left] if r % 2 else np.arange(min(left, vocab)) * 4 % vocab  # spread, or in few places
        x[r, at] = g.integers(-3, 3, len(at))
    tokens = g.integers(0, vocab, (rows, 2)).astype(np.int32)
    lp_check(x, tokens, 64)
    lp_check(x, tokens, 5)
    x[::2, g.random(vocab) < 0.5] = np.nan
    x[1::2, :-2] = np.where(g.random(vocab - 2) < 0.999, np.nan, x[1::2, :-2]) if vocab > 2 else np.nan
    lp_check(x, tokens, 64)


@pytest.mark.parametrize("rows", [1, 3, 30, 130, 300])
def test_segments_of_rows(rows):
    """Rows in as many segments as there are compute units for, or in those that they need."""
    g = rng(15, rows)
    for vocab in (4100, 32000, 70001):
        x = logits(g, rows, vocab)
        x[0, vocab // 2:] = -np.inf  # whole segments of nothing
        if rows > 2:
            x[1, -1] = np.nan
            x[2, 100] = np.inf
        pos = np.where(np.arange(rows) % 5 == 3, -1, 1).astype(np.int32)
        for n_top in (1, 64):
            lp_check(x, g.integers(0, vocab, (rows, 2)).astype(np.int32), n_top, 0.7, pos)


@pytest.mark.parametrize("vocab,n_top", [(270000, 1), (1 << 20, 0), (1 << 20, 2), (1000003, 64)])
def test_vocabularies_of_many_segments(vocab, n_top):
    g = rng(18, vocab, n_top)
    lp_check(logits(g, 1, vocab), g.integers(0, vocab, (1, 3)).astype(np.int32), n_top)


@pytest.mark.parametrize("temperature", [1e-3, 0.05, 1.0, 7.0, 1e4])
def test_temperatures(temperature):
    g = rng(11, int(temperature * 1000))
    x = logits(g, 4, 32000, 6.0)
    x[1] = g.uniform(-60000, 60000, 32000)
    x[2, 77] = 60000
    lp_check(x, g.integers(0, 32000, (4, 4)).astype(np.int32), 20, temperature)


def test_many_rows():
    g = rng(12)
    x = logits(g, 700, 1001)
    got = lp_check(x, g.integers(0, 1001, (700, 2)).astype(np.int32), 5, positions=np.where(np.arange(700) % 7, 3, -1).astype(np.int32))
    again = lp_run(x, np.zeros((700, 2), np.int32), 5, positions=np.where(np.arange(700) % 7, 3, -1).astype(np.int32))
    assert np.array_equal(got["h"].view(np.uint32), again["h"].view(np.uint32))


def test_two_graphs_that_share_a_workspace():
    """Rows in segments, whose parts lie in the library's scratch: two graphs and eager calls take turns."""
    g = rng(17)
    shapes, graphs = ((2, 32000, 20), (5, 70001, 7)), []
    for rows, vocab, n_top in shapes:
        lp_run(logits(g, rows, vocab), np.zeros((rows, 1), np.int32), n_top)
        x, h, top = up(logits(g, rows, vocab)), up(np.zeros(rows, np.float32)), up(np.zeros((rows, n_top), np.int32))
        graph = C.c_void_p()
        capi.call("llama2_graph_begin_capture")
        try:
            capi.call("llama2_batch_log_probs", None, h.ptr, top.ptr, None, x.ptr, None, None, rows, vocab, vocab, 0, n_top, 1.0)
        finally:
            capi.call("llama2_graph_end_capture", C.byref(graph))
        graphs.append((graph, x, h, top))
    for turn in range(4):
        new = [logits(g, rows, vocab) for rows, vocab, _ in shapes]
        for (graph, x, _, _), v in zip(graphs, new):
            x.copy_to_device(v)
        for graph, *_ in graphs[::1 - turn % 2 * 2]:
            capi.call("llama2_graph_launch", graph)
        lp_check(logits(g, 3, 40000), np.zeros((3, 1), np.int32), 5)
        for (graph, x, h, top), v, (rows, vocab, n_top) in zip(graphs, new, shapes):
            again = lp_run(v, np.zeros((rows, 1), np.int32), n_top)
            assert np.array_equal(h.to_host().view(np.uint32), again["h"].view(np.uint32)), turn
            assert np.array_equal(top.to_host().reshape(rows, n_top), [pu.top_tokens(r, n_top) for r in v]), turn
    for graph, *_ in graphs:
        capi.call("llama2_graph_destroy", graph)


def test_both_captured_and_replayed():
    g = rng(13)
    x, tokens = up(logits(g, 12, 4000)), up(g.integers(0, 4000, (12, 2)).astype(np.int32))
    lp, h, top = up(np.zeros((12, 2), np.float32)), up(np.zeros(12, np.float32)), up(np.zeros((12, 8), np.int32))
    c = norm_case(g, 12, 4000)
    r, y, gamma, pos, out = up(c["residual"]), up(c["x"]), up(c["gamma"]), up(c["positions"]), up(np.zeros((12, 4000), np.float16))
    batch = capi.Batch(positions=pos.ptr, n_requests=1, n_tokens=12, max_length=1)

    def issue():
        capi.call("llama2_batch_residual_rmsnorm", out.ptr, r.ptr, r.ptr, y.ptr, gamma.ptr, None, None, batch, 4000, 4000, 4000, 4000, 4000, 1.0,
                  1e-5)
        capi.call("llama2_batch_log_probs", lp.ptr, h.ptr, top.ptr, None, x.ptr, tokens.ptr, pos.ptr, 12, 4000, 4000, 2, 8, 1.0)

    graph = C.c_void_p()
    capi.call("llama2_graph_begin_capture")
    try:
        issue()
    finally:
        capi.call("llama2_graph_end_capture", C.byref(graph))
    res = c["residual"]
    for turn in range(4):
        new = logits(g, 12, 4000)
        positions = np.where(g.random(12) < 0.3, -1, 5).astype(np.int32)
        x.copy_to_device(new)
        pos.copy_to_device(positions)
        before = [v.to_host() for v in (lp, h, top, r, out)]
        capi.call("llama2_graph_launch", graph)
        got = [v.to_host() for v in (lp, h, top, r, out)]
        live = positions >= 0
        for b, a in zip(before, got):
            assert np.array_equal(a.reshape(12, -1)[~live].view(np.uint8), b.reshape(12, -1)[~live].view(np.uint8))
        (want, bound), (wr, br) = pu.norm_rows(res[live], c["x"][live], c["gamma"], None, None, 1.0, float(np.float32(1e-5)))
        assert (np.abs(got[4].reshape(12, -1)[live] - want) <= bound).all() and (np.abs(got[3].reshape(12, -1)[live] - wr) <= br).all()
        res = got[3].reshape(12, -1)
        for t in np.flatnonzero(live):
            assert np.array_equal(got[2].reshape(12, 8)[t], pu.top_tokens(new[t], 8)), turn
    capi.call("llama2_graph_destroy", graph)
