"""What a product's sums are made of, by the number of tokens: errors where inputs have a large offset in common, and numbers that are not finite."""
import numpy as np
import pytest

import product_util as pu
from managedllama2_amd import synth
from managedllama2_amd.device import init

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def ready():
    init(0)


def rng(*stream):
    return synth.rng_for(1900, *stream)


def sizes(q, K, N):
    """(w + z) s of every weight, in 64 bits."""
    W, Z, S = (a.reshape(N, -1) for a in q)
    nibbles = lambda a: ((a[:, :, None] >> (4 * np.arange(8, dtype=np.uint32))) & 15).reshape(N, -1).astype(np.float64)  # noqa: E731
    group = np.arange(K) // 128
    return (nibbles(W)[:, :K] + nibbles(Z)[:, group]) * np.abs(S.astype(np.float64))[:, group]


@pytest.mark.parametrize("offset", [0.0, 30.0, 3000.0])
@pytest.mark.parametrize("K,N,tensors", [(512, 264, 1), (4096, 520, 1), (4096, 264, 3), (11008, 264, 1), (4096, 520, 2)])
@pytest.mark.parametrize("tokens", [1, 2, 20, 70])
def test_inputs_with_a_large_offset_in_common(offset, K, N, tensors, tokens):
    """One token, where the kernels of a decode step take it: for every 32 inputs sum x w and z sum x apart in fp32, each of up to 32 terms and 2 more,
    then the scale and a sum of K / 32 terms, 64 lanes of which add up in 6 steps: off by at most (48 + K / 2048 + 8) 2^-24 of |x| (w + z) s, here twice
    that for the dot product's own rounding.  More tokens: of |x| |w - z| s (product_util.product)."""
    gated = tensors == 2
    p = pu.Product(rng(1, K, tensors, tokens), tokens, K, [N] * (1 if gated else tensors), gated)
    p.x[:] = (p.x.astype(np.float64) + offset).astype(np.float16)
    got = p.upload().run()
    x = np.abs(p.x.astype(np.float64))
    sums = []
    for q in p.q:
        y, bound = pu.product(p.x, q, K, N)
        if tokens == 1:
            bound = (56 + K // 2048) * 2.0 ** -23 * (x @ sizes(q, K, N).T)
        sums.append((y, bound))
    if gated:
        with np.errstate(over="ignore"):
            sums = [pu.swiglu(*sums[0], *sums[1])]
    for out, (y, bound) in zip(got, sums):
        with np.errstate(over="ignore"):
            inside = np.abs(y) + bound < 65000  # the others are rounded to infinity, or next to it
        err = np.abs(out.astype(np.float64) - y)
        assert inside.mean() > (0.3 if gated else 0.9) and (err <= pu.rounded(y, bound))[inside].all(), (err - pu.rounded(y, bound))[inside].max()


@pytest.mark.parametrize("tokens", [1, 2, 20, 50, 70, 300, 3001])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("wrong", [np.inf, -np.inf, np.nan])
def test_numbers_that_are_not_finite(tokens, gated, wrong):
    """An input, or a number of an adapter's: all results that it contributes to are not finite, whatever the kernel, and no others differ."""
    K, max_rank = 264, 64 if tokens == 3001 else 16
    p = pu.Product(rng(2, tokens, gated), tokens, K, [88], gated, [max_rank, 9, 5, max_rank - 1], max_rank, ids=np.arange(tokens) % 4).upload()
    want = p.run()[0]
    token, other = tokens // 2, np.arange(tokens)
    x, down, up = p.x.copy(), [q.down.copy() for q in p.pools], [q.up.copy() for q in p.pools]

    def restore():
        p.x[:] = x
        for q, d, u in zip(p.pools, down, up):
            q.down[:], q.up[:] = d, u

    def check(hit, columns, what):
        got = p.upload().run()[0]
        touched = np.zeros_like(got, bool)
        touched[np.ix_(hit, columns)] = True
        assert not np.isfinite(got[touched]).any(), what
        assert np.array_equal(got[~touched].view(np.uint16), want[~touched].view(np.uint16)), what
        restore()

    everywhere = np.ones(88, bool)
    p.x[token, 131] = wrong
    check(other == token, everywhere, "an input")
    for a in {0, int(p.ids[token])}:
        rank = int(p.pools[0].ranks[a])
        p.pools[0].down_of(a)[rank - 1, 77] = wrong
        check(p.ids[:tokens] == a, everywhere, "down %d" % a)
        p.pools[-1].up_of(a)[17, rank - 1] = wrong
        check(p.ids[:tokens] == a, np.arange(88) == 17, "up %d" % a)
