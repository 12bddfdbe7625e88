"""Attention of a step of several requests (llama2_batch_attention) where scores are far apart: sums of a great many small
weights, and scores so large that neighbouring fp32 numbers are whole powers of two of a weight apart."""
import numpy as np
import pytest

import batch_util as bu
from managedllama2_amd import synth

pytestmark = pytest.mark.gpu

LOG2E = float(np.float32(1.44269504088896340736))
# one token each (narrow tiles), prompts (wide tiles), few prompt tiles of many passes (two halves of a workgroup)
SHAPES = [([300, 90], [1, 1]), ([300, 90], [40, 30]), ([0, 256], [300, 64])]


def hull(s, got):
    """An average is finite and lies between the values it is an average of (2^-10: fp16 weights and results)."""
    rows = s.rows_of(s.value).astype(np.float32).reshape(-1, s.width)
    group = s.heads // s.kv_heads
    shared = s.row_numbers(s.prefix_table, s.prefix)
    for b in range(len(s.ctx)):
        own = s.row_numbers(s.table[b], s.lengths[b])
        for t in range(s.starts[b], s.starts[b + 1]):
            v = rows[np.concatenate([shared, own[:s.positions[t] - s.prefix + 1]])]
            for h in range(s.heads):
                at = slice(h // group * s.d, (h // group + 1) * s.d)
                g, lo, hi = got[t, h * s.d:(h + 1) * s.d].astype(np.float32), v[:, at].min(0), v[:, at].max(0)
                slack = 2.0 ** -10 * np.maximum(np.abs(lo), np.abs(hi)) + 2.0 ** -24
                assert np.isfinite(g).all() and (g >= lo - slack).all() and (g <= hi + slack).all(), (b, t, h)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ctx,new", SHAPES)
@pytest.mark.parametrize("prefix", [0, 80])
@pytest.mark.parametrize("scale", [300.0, 3e4, -1e9, 1e30])
def test_scores_of_any_size_leave_an_average(d, ctx, new, prefix, scale):
    """Scaled scores of 2^22 .. 2^114.  Where the best row leads by more than the scores' errors it is the output."""
    s = bu.Step(synth.rng_for(1421, d, len(ctx), prefix), ctx, new, 16, heads=2, kv_heads=1, d=d, prefix=prefix, fill=np.nan)
    s.key *= np.float16(1000)
    s.scale = scale
    s.upload()
    got = s.run()
    hull(s, got)
    keys, values = (s.rows_of(c).reshape(-1, s.width) for c in (s.key, s.value))
    shared, decided = s.row_numbers(s.prefix_table, s.prefix), 0
    for b in range(len(ctx)):
        own = s.row_numbers(s.table[b], s.lengths[b])
        for t in range(s.starts[b], s.starts[b + 1]):
            rows = np.concatenate([shared, own[:s.positions[t] - s.prefix + 1]])
            k = keys[rows].astype(np.float64)
            for h in range(s.heads):
                q = s.q[t, h * d:(h + 1) * d].astype(np.float64)
                x = k @ q * scale * LOG2E
                # d products and sums in fp32, the scale as fp32 and its product
                error = (d + 4) * 2.0 ** -24 * (np.abs(k) @ np.abs(q)).max() * abs(scale) * LOG2E
                order = np.argsort(x)
                if len(rows) > 1 and x[order[-1]] - x[order[-2]] < 2 * error + 40:
                    continue
                decided += 1
                want = values[rows[order[-1]]].astype(np.float64)  # times a weight, as fp16 or fp32, over that weight
                err = np.abs(got[t, h * d:(h + 1) * d] - want)
                assert (err <= 2.0 ** -10 * np.abs(want) + 2.0 ** -24).all(), (b, t, h, err.max())
    assert decided * 2 > sum(new) * s.heads


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ctx,new", SHAPES)
@pytest.mark.parametrize("power", [10, 23, 24, 25, 26, 27, 28])
def test_large_scores_that_grow_in_small_steps(d, ctx, new, power):
    """Scores of 1.5 * 2^power that grow by 8 from tile to tile: the reference of the exponents lags by as much as it may, and
    what it is rounded by comes on top."""
    s = bu.Step(synth.rng_for(1422, d, power), ctx, new, 16, heads=1, kv_heads=1, d=d)
    s.scale = 1.0 / LOG2E
    s.key[:], s.q[:] = 0, 0
    half = power // 2
    s.q[:, 0], s.q[:, 1] = 1.5 * 2.0 ** half, 8.0
    keys = s.rows_of(s.key)
    for b in range(len(ctx)):
        r = np.arange(s.lengths[b])
        keys[s.table[b, r // s.size], r % s.size, 0] = 2.0 ** (power - half)
        keys[s.table[b, r // s.size], r % s.size, 1] = r // 32
    s.upload()
    hull(s, s.run())
    if power == 10:
        s.check()


@pytest.mark.parametrize("power", [10, 24, 25, 26, 27, 28])
def test_large_scores_of_many_requests_that_grow_in_small_steps(power):
    """The same, by 8 every 128 rows, for as many narrow tiles that a wavefront goes over several tiles of rows."""
    s = bu.Step(synth.rng_for(1424, power), [290] * 26, [1] * 26, 16, heads=40, kv_heads=40, d=64)
    s.scale = 1.0 / LOG2E
    s.key[:], s.q[:] = 0, 0
    half = power // 2
    s.q[:, 0::64], s.q[:, 1::64] = 1.5 * 2.0 ** half, 8.0
    keys = s.rows_of(s.key)
    for b in range(len(s.ctx)):
        r = np.arange(s.lengths[b])
        at = s.table[b, r // s.size], r % s.size
        keys[at[0], at[1], 0::64] = 2.0 ** (power - half)
        keys[at[0], at[1], 1::64] = (r // 128)[:, None]
    s.upload()
    hull(s, s.run())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("lead", [18, 21, 25])
@pytest.mark.parametrize("best", [0, 59000])
def test_many_small_weights_count(d, new, lead, best):
    """60000 rows of 2^-lead of the best one's weight: those that fp16 holds with fewer bits than others are part of both sums."""
    s = bu.Step(synth.rng_for(1423, d), [60000 - new], [new], 128, heads=1, kv_heads=1, d=d)
    s.scale = 1.0 / LOG2E
    s.key[:], s.q[:], s.value[:] = 0, 0, 1
    s.q[:, 0] = lead
    at = s.table[0, best // 128], best % 128
    s.rows_of(s.key)[at][0] = 1
    s.rows_of(s.value)[at][:] = 0
    s.check()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (8, 2), (40, 40)])
@pytest.mark.parametrize("prefix,ctx", [(0, [2, 16, 59]), (0, [0, 1, 2, 30] * 8), (30, [1, 40, 100]), (70, [0, 3, 20, 9] * 6)])
def test_tiles_of_single_tokens_keep_the_weights_in_fp32(d, heads, kv_heads, prefix, ctx):
    """Scores are multiples of 1/4, exact in fp32, so that what is left of an element that nearly cancels is the weights' own error."""
    rng = synth.rng_for(1425, d, heads, kv_heads, prefix)
    s = bu.Step(rng, ctx, [1] * len(ctx), 16, heads=heads, kv_heads=kv_heads, d=d, prefix=prefix)
    s.scale = 0.25
    for x in (s.key.reshape(-1, kv_heads, d), s.q.reshape(-1, heads, d)):
        x[...] = 0
        x[..., :4] = rng.integers(-2, 3, x[..., :4].shape)
    s.upload()
    got = s.run().astype(np.float64)
    keys, values = (s.rows_of(c).reshape(-1, kv_heads, d).astype(np.float64) for c in (s.key, s.value))
    shared = s.row_numbers(s.prefix_table, prefix)
    # 24 requests of 40 heads behind 70 rows have these read once for all 24 of them, in wide tiles: weights as fp16, off by half a
    # step of it (2^-11) each in the one sum and so in the other
    wide = 2.0 ** -11 if prefix == 70 and kv_heads == 40 else 0.0
    for b in range(len(ctx)):
        rows = np.concatenate([shared, s.row_numbers(s.table[b], s.lengths[b])])
        for h in range(heads):
            k, v = keys[rows, h // (heads // kv_heads)], values[rows, h // (heads // kv_heads)]
            x = k @ s.q[b, h * d:(h + 1) * d].astype(np.float64) * 0.25
            w = np.exp(x - x.max())
            want, size = w @ v / w.sum(), w @ np.abs(v) / w.sum()
            # weights as two fp16 numbers (2^-22; what is left below fp16's smallest, 2^-31 of the largest weight), exponents up to 16 from the
            # constant log2(e), two products and a difference (4 times 2^-24 each), exp2 2^-22; both sums; the result as fp16
            eps = wide + 2.0 ** -22 + 2 * (4 * 2.0 ** -24 * 16 + 2.0 ** -22) + 2 * len(rows) * 2.0 ** -24
            bound = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + eps * size + len(rows) * 2.0 ** -31 * np.abs(v).max()
            err = np.abs(got[b, h * d:(h + 1) * d] - want)
            assert (err <= bound).all(), (b, h, (err / bound).max())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ctx,prefix", [([200, 50], 0), ([0, 31], 0), ([300, 90], 100), ([5, 20], 40)])
def test_infinite_values_reach_single_tokens(d, ctx, prefix):
    """A value that is not finite, in a row that every query of its tile attends: its element of the output is that, the others are
    what they were."""
    s = bu.Step(synth.rng_for(1426, d, len(ctx), prefix), ctx, [1, 1], 16, heads=4, kv_heads=2, d=d, prefix=prefix)
    clean = s.check().astype(np.float32)
    rows = s.rows_of(s.value)
    own = s.ctx[0] // 2
    rows[s.table[0, own // 16], own % 16, [0, d // 2, d + 5]] = np.inf, -np.inf, np.nan
    if prefix:
        rows[s.prefix_table[prefix // 32], 3, d - 1] = np.inf
    s.upload()
    got = s.run().astype(np.float32).reshape(2, 4, d)
    want = clean.reshape(2, 4, d).copy()
    want[0, :2, 0], want[0, :2, d // 2], want[0, 2:, 5] = np.inf, -np.inf, np.nan  # two heads of queries to one of keys
    if prefix:
        want[:, :2, d - 1] = np.inf
    same = np.isfinite(want)
    assert np.array_equal(got[~same], want[~same], equal_nan=True)
    assert np.array_equal(got[same], want[same])
