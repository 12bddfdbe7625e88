"""Log probabilities and entropies held to what the arithmetic of each value allows, NaN of both kinds, and more rows than a launch takes.

The bounds.  u = 2^-24 is half a step of fp32, relative.  With x the logits, T the temperature, delta = (max - x) / T, p the probabilities, L = log sum
exp(-delta), m = sum p delta, q = sum p delta^2:

  exponential   max - x is rounded once, 1 / T (with log2 e) once, their product once: 3 u delta of the exponent, so as much of e relative;
                the instruction itself 2 u.  A row in segments does so twice, from a logit to its segment's largest and from there to the row's: the
                deltas add up to one, and 2 u more, and 2 u for the two products that join them.  Below 2^-126 it is 0, which is less than any bound.
  sum           of positive terms: 32 in a row at most, two halves, 6 steps in a wavefront, 8 wavefronts, 6 steps of segments: 54 u
                E = (3 m + 60) u
  log           4 u of L (two steps of its own), and E of the sum
  log p         = -delta - L: 3 u of delta, log, and one rounding:  3 u delta + 4 u L + E + u |log p|
  entropy       = L + m, m the quotient of the sum of e (x - max), all of one sign, and the sum: each term as its exponential and 2 u for the
                difference and the product, added up as above, 2 u for where segments meet, product with 1 / T and division 5 u:
                (3 q + 71 m) u + E m, with log and one rounding of the result
"""
import numpy as np
import pytest

import product_util as pu
from managedllama2_amd import capi, synth
from managedllama2_amd.device import DeviceVariable, init

pytestmark = pytest.mark.gpu
up = pu.up
U = 2.0 ** -24


@pytest.fixture(autouse=True, scope="module")
def ready():
    init(0)


def rng(*stream):
    return synth.rng_for(1850, *stream)


def call(x, tokens, n_top, temperature=1.0):
    rows, vocab = x.shape
    lp, h = up(np.zeros((rows, tokens.shape[1]), np.float32)), up(np.zeros(rows, np.float32))
    top, tlp = up(np.zeros((rows, n_top), np.int32)), up(np.zeros((rows, n_top), np.float32))
    given, asked = up(x), up(tokens)
    capi.call("llama2_batch_log_probs", lp.ptr, h.ptr, top.ptr, tlp.ptr, given.ptr, asked.ptr, None, rows, vocab, vocab, tokens.shape[1], n_top,
              temperature)
    return lp.to_host().reshape(tokens.shape), h.to_host(), top.to_host().reshape(rows, n_top), tlp.to_host().reshape(rows, n_top)


def exact(x, temperature):
    """One row with something above -infinity -> (log p, bounds, entropy, its bound)."""
    d = (x.astype(np.float64).max() - x.astype(np.float64)) / float(np.float32(temperature))
    e = np.exp(-d)
    total = e.sum()
    p, L = e / total, np.log(total)
    seen = p > 0
    m, q = (p[seen] * d[seen]).sum(), (p[seen] * d[seen] ** 2).sum()
    E = (3 * m + 60) * U
    lp = -d - L
    with np.errstate(invalid="ignore"):
        bound = 3 * U * d + 4 * U * L + E + U * np.abs(lp)
    return lp, bound, L + m, (3 * q + 71 * m) * U + E * m + 4 * U * L + E + U * (L + m)


def check(x, tokens, n_top, temperature=1.0, tight=False):
    """tight: also of all together, where independent roundings leave far less: half a step of the result, one each of 1 / T and L, 2^-22 in all."""
    lp, h, top, tlp = call(x, tokens, n_top, temperature)
    off, size, h_off, h_size = 0.0, 0.0, 0.0, 0.0
    for r in range(len(x)):
        want, bound, entropy, h_bound = exact(x[r], temperature)
        order = pu.top_tokens(x[r], n_top)
        assert np.array_equal(top[r], order), r
        there = order >= 0
        assert np.isneginf(tlp[r][~there]).all()
        for got, at in ((lp[r], tokens[r]), (tlp[r][there], order[there])):
            masked = np.isneginf(want[at])
            assert np.array_equal(np.isneginf(got), masked), (r, got, want[at])
            err = np.abs(got.astype(np.float64)[~masked] - want[at][~masked])
            assert (err <= bound[at][~masked]).all(), (r, err.max(), (err / bound[at][~masked]).max())
            off, size = off + (err ** 2).sum(), size + (want[at][~masked] ** 2).sum()
        assert abs(h[r] - entropy) <= h_bound, (r, h[r], entropy, h_bound)
        h_off, h_size = h_off + (h[r] - entropy) ** 2, h_size + entropy ** 2
    if tight:
        assert off <= 2.0 ** -44 * size and h_off <= 2.0 ** -44 * h_size, (np.sqrt(off / size), np.sqrt(h_off / h_size))


def logits(g, rows, vocab, std=2.5):
    return (g.standard_normal((rows, vocab)) * std).astype(np.float16)


@pytest.mark.parametrize("vocab", [2, 65, 1001, 4096, 4097, 32000, 50257, 128000])
@pytest.mark.parametrize("rows", [1, 30, 300])
def test_rows_in_one_piece_and_in_segments(vocab, rows):
    g = rng(1, vocab, rows)
    if rows * vocab > 1 << 24:
        rows = 40
    x = logits(g, rows, vocab)
    check(x, g.integers(0, vocab, (rows, 40)).astype(np.int32), 8, 0.8, tight=vocab > 1000 and rows > 1)


@pytest.mark.parametrize("temperature", [1e-3, 0.05, 0.7, 1.0, 7.0, 1e4])
@pytest.mark.parametrize("vocab", [3000, 70001])
def test_temperatures_and_spreads(temperature, vocab):
    """Spreads from next to nothing to fp16's whole range, and numbers that stand for masked ones: what has no probability adds no error."""
    g = rng(2, int(temperature * 1000), vocab)
    x = logits(g, 8, vocab)
    x[1] *= 0.01
    x[2] *= 8
    x[3] = g.uniform(-60000, 60000, vocab)
    x[4, g.random(vocab) < 0.9] = -np.inf
    x[5, g.random(vocab) < 0.9] = -65504
    x[6] = -65504
    x[6, vocab // 2] = 65504
    x[7] = -65504  # all alike
    check(x, g.integers(0, vocab, (8, 20)).astype(np.int32), 20, temperature)


@pytest.mark.parametrize("temperature", [2e-30, 1e30])
@pytest.mark.parametrize("vocab", [3000, 70001])
def test_the_ends_of_the_temperatures(temperature, vocab):
    g = rng(5, vocab)
    x = logits(g, 3, vocab)
    x[1] = g.uniform(-65504, 65504, vocab)
    x[2, ::2] = -np.inf
    check(x, g.integers(0, vocab, (3, 20)).astype(np.int32), 5, temperature)


@pytest.mark.parametrize("vocab", [700, 32000, 70001])
def test_nan_that_signals(vocab):
    """The likeliest tokens beside NaN of both kinds, which say nothing about their neighbours in a word or in a lane."""
    g = rng(3, vocab)
    x = logits(g, 6, vocab)
    bits = x.view(np.uint16)
    for r, share in enumerate((0.0005, 0.01, 0.3, 0.9, 0.999)):
        at = g.random(vocab) < share
        at[g.integers(0, vocab)] = True
        bits[r, at] = g.choice(np.array([0x7C01, 0x7D00, 0xFC01, 0xFDFF, 0x7E00, 0xFE00], np.uint16), at.sum())
    best = np.argsort(-x[5].astype(np.float64))[:20]
    bits[5, best ^ 1 if vocab % 2 == 0 else np.minimum(best + 1, vocab - 1)] = 0x7C01  # next to the likeliest
    lp, h, top, tlp = call(x, np.zeros((6, 1), np.int32), 40)
    for r in range(6):
        assert np.array_equal(top[r], pu.top_tokens(x[r], 40)), r
    assert np.isnan(lp).all() and np.isnan(h).all() and np.isnan(tlp).all()


@pytest.mark.parametrize("vocab,n_top", [(24, 3), (32776, 2)])
def test_more_rows_than_a_launch_takes(vocab, n_top):
    """32768 rows; of long ones all but a few are without a position, and stay as they were."""
    rows = 2 * 32768 + 5
    g = rng(4, vocab)
    live = np.array([0, 1, 32767, 32768, 32769, 65535, 65536, rows - 1])
    positions = np.full(rows, -1, np.int32)
    positions[live] = 3
    x = logits(g, len(live), vocab)
    far = DeviceVariable(np.float16, rows * vocab)
    capi.call("llama2_memset", far.ptr, 0xFF, far.nbytes)
    for i, r in enumerate(live):
        far.copy_to_device(x[i], int(r) * vocab)
    tokens = g.integers(0, vocab, (rows, 2)).astype(np.int32)
    lp, h = up(np.full((rows, 2), 7, np.float32)), up(np.full(rows, 7, np.float32))
    top, tlp = up(np.full((rows, n_top), -7, np.int32)), up(np.full((rows, n_top), 7, np.float32))
    asked, at = up(tokens), up(positions)
    capi.call("llama2_batch_log_probs", lp.ptr, h.ptr, top.ptr, tlp.ptr, far.ptr, asked.ptr, at.ptr, rows, vocab, vocab, 2, n_top, 1.0)
    lp, h, top, tlp = lp.to_host().reshape(rows, 2), h.to_host(), top.to_host().reshape(rows, n_top), tlp.to_host().reshape(rows, n_top)
    for i, r in enumerate(live):
        want, bound, entropy, h_bound = exact(x[i], 1.0)
        assert (np.abs(lp[r] - want[tokens[r]]) <= bound[tokens[r]]).all() and abs(h[r] - entropy) <= h_bound, r
        order = pu.top_tokens(x[i], n_top)
        assert np.array_equal(top[r], order) and (np.abs(tlp[r] - want[order]) <= bound[order]).all(), r
    rest = positions < 0
    assert (lp[rest] == 7).all() and (h[rest] == 7).all() and (top[rest] == -7).all() and (tlp[rest] == 7).all()
