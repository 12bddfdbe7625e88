"""Adapters of many tokens, so many of them and so many in use that every way of finding, sharing and reading them is taken; inputs whose rows lie as far
apart as they may.  Against 64-bit restatements (product_util.py)."""
import numpy as np
import pytest

import product_util as pu
from managedllama2_amd import capi, synth
from managedllama2_amd.device import DeviceVariable, init

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def ready():
    init(0)


def rng(*stream):
    return synth.rng_for(1800, *stream)


def spread(g, tokens, pool):
    """Adapters of the tokens: blocks of 64 with (nearly) as many adapters as tokens, with about 24, with 3 among which one has more than 16 tokens,
    and with the pool's last ones, one after the other, some tokens without any."""
    ids = np.empty(tokens, np.int32)
    for t in range(0, tokens, 64):
        n = min(64, tokens - t)
        ids[t:t + n] = (g.integers(-1, pool, n), g.integers(0, 24, n) * (pool // 24) + t // 64 % 5, g.choice([7, pool - 1, pool // 2], n, p=[0.6, 0.2, 0.2]),
                        g.integers(max(pool - 40, 0), pool + 2, n))[t // 64 % 4]
    return ids


@pytest.mark.parametrize("tokens,K", [(1601, 1032), (403, 4104), (801, 5128)])
@pytest.mark.parametrize("gated", [False, True])
def test_blocks_of_tokens_with_dozens_of_adapters_of_hundreds(tokens, K, gated):
    """What the ranks receive in items of tokens that share an adapter: several items for a workgroup, adapters behind those whose ranks are in its
    table, rows of up to 4096 inputs, of up to 5120, and longer ones."""
    max_rank, pool = 32, 600
    assert 4 * tokens * K * max_rank > (2e8 if K <= 5120 else 5e8)  # above these bytes they are taken so
    g = rng(1, tokens, gated)
    ranks = np.resize([32, 5, 16, 0, 31, 17, 1, 8], pool)
    p = pu.Product(g, tokens, K, [40], gated, ranks, max_rank, residual=not gated, pad=3, pool_stride=8, ids=0)
    p.ids[:tokens] = spread(g, tokens, pool)
    assert (p.ids[:tokens] >= 512).any() and len(np.unique(p.ids[:64])) > 40
    p.upload().check()


@pytest.mark.parametrize("tokens", [300, 49100])
def test_a_pool_of_70000_adapters(tokens):
    """Numbers of 17 bits, told apart bit by bit: token by token, and in items."""
    pool, max_rank, K = 70000, 128, 8
    assert (4 * tokens * K * max_rank > 2e8) == (tokens > 300)
    g = rng(2, tokens)
    p = pu.Product(g, tokens, K, [8], False, np.resize([3, 128, 0, 17, 8], pool), max_rank, junk=np.inf, ids=0)
    p.ids[:] = spread(g, tokens, pool)
    for t in range(0, tokens - 64, 640):  # neighbours in one bit each
        p.ids[t:t + 17] = 65536 + 1234 ^ np.concatenate([1 << np.arange(13), [0, 1 << 16, 65536 + 1234, 1 << 12]])
    p.upload().check()


def test_rows_of_inputs_as_far_apart_as_they_may_be():
    """2^24 halfs: offsets within a block of tokens are ints.  NaN between the rows."""
    stride, K = 1 << 24, 520
    most = 760
    far = DeviceVariable(np.float16, (most - 1) * stride + K)
    capi.call("llama2_memset", far.ptr, 0xFF, far.nbytes)
    for tokens, cols, gated, max_rank, ids in ((1, [264], False, 16, None), (20, [264], False, 16, None), (33, [4400], False, 16, None),
                                               (50, [1000], True, 16, None), (193, [88], False, 16, None), (most, [40], False, 128, None),
                                               (100, [88], True, 0, None), (most, [40], True, 128, 1)):
        p = pu.Product(rng(3, tokens, gated), tokens, K, cols, gated, [max_rank, 3, 0, max_rank // 2] if max_rank else (), max_rank, ids=ids).upload()
        want = p.check(str(tokens))[0]
        for t in range(tokens):
            far.copy_to_device(p.x[t], t * stride)
        outs = p.outputs()
        name, *args = p.args(outs)
        args[1 if gated else 2] = far.ptr
        args[7 if gated else 4] = stride
        capi.call(name, *args)
        assert np.array_equal(outs[0].to_host().view(np.uint16), want.ravel().view(np.uint16)), (tokens, gated)
