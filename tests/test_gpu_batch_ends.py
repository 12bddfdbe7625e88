"""The most outputs of a tensor, the most tokens of a step, against 64-bit restatements (product_util.py)."""
import ctypes as C

import numpy as np
import pytest

import product_util as pu
from managedllama2_amd import capi, synth
from managedllama2_amd.device import DeviceVariable, init

pytestmark = pytest.mark.gpu
MOST = 1 << 20


@pytest.fixture(autouse=True, scope="module")
def ready():
    init(0)


def rng(*stream):
    return synth.rng_for(1950, *stream)


@pytest.mark.parametrize("tokens", [1, 16, 20, 50, 70, 200])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("adapters", [False, True])
def test_as_many_outputs_as_there_may_be(tokens, gated, adapters):
    """w - z is -1 and 1 in turn, and an adapter's rows are all alike, so that all outputs of a token are equal."""
    K, max_rank = 264, 8
    words, groups = 9 * 4, 3
    w, z, s = (DeviceVariable.zeros(t, MOST * n) for t, n in ((np.uint32, words), (np.uint32, 1), (np.float16, groups)))
    for v, byte in ((w, 0x53), (z, 0x44), (s, 0x2C)):
        capi.call("llama2_memset", v.ptr, byte, v.nbytes)
    scale = float(np.full(1, 0x2C2C, np.uint16).view(np.float16)[0])
    g = rng(1, tokens, gated)
    x = g.standard_normal((tokens, K)).astype(np.float16)
    down = (g.standard_normal((2, max_rank, K)) / np.sqrt(K)).astype(np.float16)
    up = DeviceVariable.zeros(np.float16, 2 * MOST * max_rank)
    capi.call("llama2_memset", up.ptr, 0x2E, up.nbytes)
    u = float(np.full(1, 0x2E2E, np.uint16).view(np.float16)[0])
    ids = np.arange(tokens) % 3 - 1
    dx, dd, di, dp = pu.up(x), pu.up(down), pu.up(ids.astype(np.int32)), pu.up(np.zeros(tokens, np.int32))
    ranks, scales = pu.up(np.array([8, 5], np.int32)), pu.up(np.array([1.5, 0.5], np.float32))
    pool = C.pointer(capi.Adapters(down=dd.ptr, up=up.ptr, scales=scales.ptr, ranks=ranks.ptr, n_adapters=2, max_rank=max_rank)) if adapters else None
    out = DeviceVariable.zeros(np.float16, tokens * MOST)
    batch = capi.Batch(positions=dp.ptr, n_requests=1, n_tokens=tokens, max_length=1)
    q = capi.QWeight(w.ptr, z.ptr, s.ptr)
    if gated:
        capi.call("llama2_batch_mat_mul_swiglu", out.ptr, dx.ptr, q, q, K, MOST, MOST, K, pool, pool, di.ptr, batch)
    else:
        m = (capi.BatchMatrix * 1)(capi.BatchMatrix(weight=q, output=out.ptr, adapters=pool, cols=MOST, output_stride=MOST))
        capi.call("llama2_batch_mat_mul_int4", m, 1, dx.ptr, K, K, di.ptr, batch)
    got = out.to_host().reshape(tokens, MOST)
    v, size = x.astype(np.float64), np.abs(x.astype(np.float64))
    y = scale * (v[:, 1::2].sum(1) - v[:, ::2].sum(1))
    bound = (56 + 128) * 2.0 ** -23 * scale * 9 * size.sum(1)  # w + z at most 9
    if adapters:
        for t, a in enumerate(ids):
            if a >= 0:
                r, f = (8, 5)[a], (1.5, 0.5)[a]
                h = down[a, :r].astype(np.float64) @ v[t]
                y[t] += f * u * h.sum()
                # as in product_util.Pool.add
                bound[t] += f * u * ((K + 8) * 2.0 ** -23 * (np.abs(down[a, :r].astype(np.float64)) @ size[t]) + 2.0 ** -22 * np.abs(h).max()
                                     + (2 * r + 8) * 2.0 ** -23 * np.abs(h)).sum()
    if gated:
        y, bound = pu.swiglu(y, bound, y, bound)
    for end in (got.min(1), got.max(1)):  # NaN if there is any
        assert (np.abs(end.astype(np.float64) - y) <= pu.rounded(y, bound)).all()


def test_as_many_tokens_as_there_may_be():
    p = pu.Product(rng(2), MOST, 8, [16], False, [8, 3], 8, residual=True, x_extra=8).upload()
    p.check()
    pu.Product(rng(3), MOST - 7, 16, [8], True, pad=7).upload().check()


def test_norms_of_as_many_rows():
    g = rng(4)
    rows = lambda: g.standard_normal((MOST, 8)).astype(np.float16)  # noqa: E731
    residual, x, gamma = rows(), rows(), np.linspace(0.5, 1.5, 8).astype(np.float16)
    dr, dx, dg, dp = pu.up(residual), pu.up(x), pu.up(gamma), pu.up(np.where(np.arange(MOST) % 5 == 3, -1, 1).astype(np.int32))
    out = DeviceVariable.from_host(np.full((MOST, 8), pu.GUARD, np.float16))
    batch = capi.Batch(positions=dp.ptr, n_requests=1, n_tokens=MOST, max_length=1)
    capi.call("llama2_batch_residual_rmsnorm", out.ptr, dr.ptr, dr.ptr, dx.ptr, dg.ptr, None, None, batch, 8, 8, 8, 8, 8, 0.5, 1e-5)
    live = np.arange(MOST) % 5 != 3
    for got, (want, bound), before in zip((out, dr), pu.norm_rows(residual, x, gamma, None, None, 0.5, float(np.float32(1e-5))),
                                          (np.full_like(residual, pu.GUARD), residual)):
        got = got.to_host().reshape(MOST, 8)
        assert (np.abs(got.astype(np.float64) - want) <= bound)[live].all() and np.array_equal(got[~live], before[~live])
