"""Products of the rows of many tokens with int4 tensors, low-rank adapters beside them, and the gated block's first half,
against 64-bit restatements (product_util.py)."""
import ctypes as C
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

import product_util as pu
from managedllama2_amd import capi, synth
from managedllama2_amd.device import init

pytestmark = pytest.mark.gpu

RANKS = [16, 0, 1, 5, 8, 13, 24, 32]


@pytest.fixture(autouse=True, scope="module")
def ready():
    init(0)


def rng(*stream):
    return synth.rng_for(1700, *stream)


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 31, 33, 48, 64, 65, 100, 130, 257])
@pytest.mark.parametrize("gated", [False, True])
def test_numbers_of_tokens(tokens, gated):
    pu.Product(rng(1, tokens, gated), tokens, 264, [88], gated, RANKS, 32, pad=tokens % 5, residual=not gated).upload().check()


@pytest.mark.parametrize("K", [8, 24, 120, 128, 136, 256, 1000, 1032, 4096, 11008])
@pytest.mark.parametrize("tokens", [3, 70, 140])
def test_lengths_of_a_row(K, tokens):
    pu.Product(rng(2, K, tokens), tokens, K, [40], False, [8, 3], 8, x_extra=16, extra=8).upload().check()
    pu.Product(rng(3, K, tokens), tokens, K, [24], True, [8, 3], 8, x_extra=8, extra=24).upload().check()


@pytest.mark.parametrize("cols", [[8], [16], [24, 8], [1000], [264, 40, 8, 520], [512, 512, 512], [1376]])
@pytest.mark.parametrize("tokens", [1, 20, 50, 200])
def test_widths(cols, tokens):
    pu.Product(rng(4, tokens, *cols), tokens, 384, cols, False, [4, 16, 7], 16, residual=len(cols) % 2 == 1, extra=16).upload().check()
    pu.Product(rng(5, tokens, *cols), tokens, 384, cols[:1], True).upload().check()


@pytest.mark.parametrize("K", [8, 120, 512, 1032, 2048, 4096, 5120, 8192, 10240, 11008, 13824, 14336, 14344])
@pytest.mark.parametrize("max_rank", [0, 16, 128])
def test_one_token(K, max_rank):
    """One tensor, three of one width, gate and up: on the kernels of a decode step where they take the shape."""
    for i, (cols, gated) in enumerate((([72], False), ([136] * 3, False), ([1000], True), ([520], False))):
        ranks = [max_rank, 0, 3, max_rank - 1] if max_rank else ()
        for id in (0, 2, 3, 1, -1) if max_rank else (-1,):
            p = pu.Product(rng(30, K, max_rank, i, id + 1), 1, K, cols, gated, ranks, max_rank, residual=not gated and i != 1, pool_stride=8 * i, extra=8,
                           x_extra=8, ids=id)
            if i == 1:
                p.pools[1] = None
                p.residual = [p.x[:, :8].repeat(18, 1)] * 3
            p.upload().check(str((i, id)))
    p.positions[:] = -1
    p.live = 0
    got = p.upload().run()[0]
    assert (got == pu.GUARD).all()


@pytest.mark.parametrize("tokens", [1, 20, 50, 70])
def test_scales_and_zero_points_at_odd_places(tokens):
    for gated in (False, True):
        p = pu.Product(rng(31, tokens, gated), tokens, 520, [88], gated).upload()
        want = p.run()[0]
        moved = []
        for (_, Z, S), w in zip(p.q, p.weights):
            s, z = pu.up(np.concatenate([np.full(1, np.nan, np.float16), S.ravel()])), pu.up(np.concatenate([np.full(1, 77, np.uint32), Z.ravel()]))
            moved.append((capi.QWeight(w.Weight.ptr, z.ptr + 4, s.ptr + 2), s, z))
        outs = p.outputs()
        name, *args = p.args(outs)
        if gated:
            args[2], args[3] = moved[0][0], moved[1][0]
        else:
            args[0][0].weight = moved[0][0]
        capi.call(name, *args)
        got = outs[0].to_host().reshape(want.shape).astype(np.float64)
        assert (np.abs(got[:tokens] - p.reference()[0][0]) <= p.reference()[0][1]).all()


@pytest.mark.parametrize("columns", [3000, 5000, 8000, 21000, 27000])
@pytest.mark.parametrize("tokens", [1, 16, 18, 32, 40, 64])
@pytest.mark.parametrize("adapters", [False, True])
def test_tiles_of_few_and_many_columns(columns, tokens, adapters):
    """Every tile that the numbers of columns and tokens choose, with rows and tokens left over at its end."""
    ranks, max_rank = ([8, 3, 0, 16], 16) if adapters else ([], 0)
    pu.Product(rng(20, columns, tokens, adapters), tokens, 392, [columns - 1000, 1000], False, ranks, max_rank, residual=True, pad=1).upload().check()
    pu.Product(rng(21, columns, tokens, adapters), tokens, 392, [columns // 16 * 8], True, ranks, max_rank, pad=1).upload().check()


@pytest.mark.parametrize("columns", [3000, 5000, 8000])
@pytest.mark.parametrize("tokens", [65, 130, 192, 193])
def test_several_blocks_of_tokens_with_many_adapters(columns, tokens):
    ranks = [8, 3, 0, 16, 7, 16, 1, 15, 4, 2]
    pu.Product(rng(32, columns, tokens), tokens, 392, [columns - 1000, 1000], False, ranks, 16, residual=True, pad=1).upload().check()
    pu.Product(rng(33, columns, tokens), tokens, 392, [columns // 16 * 8], True, ranks, 16, pad=1).upload().check()


@pytest.mark.parametrize("K,cols,tokens", [(16520, 104, 3), (16520, 24, 40), (16520, 6400, 40), (32768, 40, 1), (32768, 40, 50), (32776, 40, 1),
                                           (32776, 24, 40), (40000, 24, 100), (65536, 40, 2), (65536, 24, 20)])
def test_long_rows(K, cols, tokens):
    pu.Product(rng(22, K, cols, tokens), tokens, K, [cols], False, [16, 5], 16).upload().check()
    if K <= 32768 and cols < 1000:
        pu.Product(rng(23, K, cols, tokens), tokens, K, [cols], True, [16, 5], 16).upload().check()


def test_a_tensor_of_more_than_two_gibibytes():
    """65 and more tokens of it, in launches of up to 4096; w - z is -1 and 1 in turn, so that all outputs of a token are equal."""
    K, N, tokens = 32768, 131080, 4097
    w, z, s = pu.DeviceVariable.zeros(np.uint32, N * K // 8), pu.DeviceVariable.zeros(np.uint32, N * 32), pu.DeviceVariable.zeros(np.float16, N * 256)
    for v, byte in ((w, 0x53), (z, 0x44), (s, 0x1C)):
        capi.call("llama2_memset", v.ptr, byte, v.nbytes)
    base = rng(34).standard_normal((61, K)).astype(np.float16)
    x = pu.up(base[np.arange(tokens) % 61])
    out, positions = pu.DeviceVariable.zeros(np.float16, tokens * N), pu.up(np.zeros(tokens, np.int32))
    m = (capi.BatchMatrix * 1)(capi.BatchMatrix(weight=capi.QWeight(w.ptr, z.ptr, s.ptr), output=out.ptr, cols=N, output_stride=N))
    batch = capi.Batch(positions=positions.ptr, n_requests=1, n_tokens=tokens, max_length=1)
    capi.call("llama2_batch_mat_mul_int4", m, 1, x.ptr, K, K, None, batch)
    scale = float(np.full(1, 0x1C1C, np.uint16).view(np.float16)[0])
    for t in (0, 31, 63, 64, 1000, 4095, 4096):
        v = base[t % 61].astype(np.float64)
        want, size = scale * (v[1::2].sum() - v[::2].sum()), scale * np.abs(v).sum()
        got = pu.DeviceVariable.window(out, t * N * 2, np.float16, N).to_host().astype(np.float64)
        # as in product_util.product and rounded
        assert (np.abs(got - want) <= pu.rounded(np.float64(want), (128 + K // 128 + 16) * 2.0 ** -23 * size)).all(), (t, got, want)


def test_more_tokens_than_a_launch_takes():
    pu.Product(rng(24), 4133, 264, [40, 24], False, RANKS, 32, residual=True, pad=7).upload().check()
    pu.Product(rng(25), 4133, 264, [24], True, RANKS, 32, pad=7).upload().check()


@pytest.mark.parametrize("max_rank", [8, 16, 24, 64, 72, 128])
@pytest.mark.parametrize("tokens", [1, 16, 40, 150])
@pytest.mark.parametrize("gated", [False, True])
def test_ranks(max_rank, tokens, gated):
    """Adapters of every rank, infinities and NaN beyond each rank and between them, and every way that tokens can use them."""
    ranks = sorted({0, 1, 7, max_rank // 2, max_rank - 1, max_rank})
    for i, junk in enumerate((np.nan, -np.inf)):
        g = rng(6, max_rank, tokens, gated, i)
        pu.Product(g, tokens, 520, [72], gated, ranks + [max_rank + 50, -3], max_rank, pool_stride=(0, 24)[i], junk=junk).upload().check("any")
    one = pu.Product(rng(7, max_rank, tokens), tokens, 520, [72], gated, [max_rank] * 3, max_rank, ids=1).upload()
    one.check("one for all")
    each = pu.Product(rng(8, max_rank, tokens), tokens, 136, [72], gated, [max_rank] * tokens, max_rank, ids=np.arange(tokens)[::-1]).upload()
    each.check("one for each")


@pytest.mark.parametrize("tokens,K,max_rank", [(2000, 520, 72), (3001, 264, 64), (300, 5000, 64), (1100, 4096, 16), (150, 11008, 128)])
@pytest.mark.parametrize("gated", [False, True])
def test_adapters_of_many_tokens(tokens, K, max_rank, gated):
    """So many that tokens which share an adapter are taken together."""
    ranks = [max_rank, 0, 1, max_rank // 2, max_rank - 1, 7]
    for i, (ids, junk) in enumerate(((None, np.nan), (2, np.inf), (np.sort(rng(26, tokens).integers(-1, 7, tokens)), -np.inf))):
        p = pu.Product(rng(27, tokens, gated, i), tokens, K, [40], gated, ranks, max_rank, pool_stride=16 * i, junk=junk, ids=ids).upload()
        want = p.check(str(i))[0]
    for pool in p.pools:
        pool.up_of(2)[::3, :1] = np.nan
    p.x[4, 5] = np.inf
    got = p.upload().run()[0]
    hit = (p.ids == 2) | (np.arange(tokens) == 4)
    assert np.array_equal(got[~hit].view(np.uint16), want[~hit].view(np.uint16)) and not np.isfinite(got[hit]).all(1).any()


def test_only_some_matrices_have_adapters():
    p = pu.Product(rng(9), 37, 256, [64, 128, 64], False, [8, 16], 16)
    p.pools[1] = None
    p.upload().check()
    for keep in (0, 1):
        s = pu.Product(rng(10, keep), 37, 256, [64], True, [8, 16], 16)
        s.pools[1 - keep] = None
        s.upload().check()


@pytest.mark.parametrize("tokens", [1, 20, 50, 130, 1700])
def test_pools_of_different_sizes(tokens):
    """An adapter that one tensor has and another does not, and ranks of different widths."""
    for gated in (False, True):
        for ids in (np.arange(tokens) % 7 - 1, 2):
            p = pu.Product(rng(35, tokens, gated), tokens, 512, [64] if gated else [64, 64, 64], gated, [8, 24, 3, 31, 16], 32, ids=ids)
            p.pools[1] = pu.Pool(rng(36, tokens, gated), [40, 7], 64, 512, 64)
            p.upload().check(str(gated))


@pytest.mark.parametrize("tokens", [5, 60, 300])
def test_residual_in_place_and_outputs_side_by_side(tokens):
    p = pu.Product(rng(11, tokens), tokens, 640, [256], residual=True, in_place=True, pad=3).upload()
    p.check()
    q = pu.Product(rng(12, tokens), tokens, 256, [64, 32, 40], ranks=[8], max_rank=8, pad=2).upload()
    want = q.run()
    wide = pu.up(np.full((q.tokens, 64 + 32 + 40 + 8), pu.GUARD, np.float16))
    name, m, *rest = q.args([wide] * 3)
    at = 0
    for i, n in enumerate(q.cols):
        m[i].output, m[i].output_stride = wide.ptr + 2 * at, 144
        at += n
    capi.call(name, m, *rest)
    got = wide.to_host().reshape(q.tokens, -1)
    assert np.array_equal(got[:, :136].view(np.uint16), np.concatenate(want, 1).view(np.uint16)) and (got[:, 136:] == pu.GUARD).all()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("tokens", [6, 90, 200])
def test_what_one_token_or_adapter_holds_stays_with_it(gated, tokens):
    p = pu.Product(rng(13, tokens, gated), tokens, 264, [48], gated, [8, 12, 16], 16, ids=np.arange(tokens) % 4 - 1).upload()
    want = p.run()[0]
    for pool in p.pools:
        pool.down_of(1)[:12, ::7] = np.inf
        pool.up_of(1)[::3, :12] = np.nan
    p.x[4, 5] = np.inf
    p.upload()
    got = p.run()[0]
    hit = (p.ids == 1) | (np.arange(tokens) == 4)
    assert np.array_equal(got[~hit].view(np.uint16), want[~hit].view(np.uint16))
    assert not np.isfinite(got[hit]).all(1).any()


@pytest.mark.parametrize("tokens", [20, 200])
def test_sizes_of_what_the_ranks_receive(tokens):
    """Adapters whose inner values lie far outside fp16's range, or far below it, lose nothing."""
    for i, (d, u) in enumerate(((3.0e4, 1.0e-6), (2.0 ** -14, 200.0), (60000.0, 2.0 ** -20))):
        p = pu.Product(rng(14, tokens, i), tokens, 512, [64], False, [16, 5], 16, junk=0.0)
        for pool in p.pools:
            pool.down[:] = (pool.down.astype(np.float32) * d).clip(-65504, 65504).astype(np.float16)
            pool.up[:] = (pool.up.astype(np.float32) * u).astype(np.float16)
        p.upload().check()
    p.x[:, :512] = 0
    p.upload().check("zeros")


@pytest.mark.parametrize("tokens", [1, 48, 300])
@pytest.mark.parametrize("gated", [False, True])
def test_captured_steps_replayed(tokens, gated):
    """Inputs, adapters of the tokens and tokens without a position change between replays; eager calls of other sizes stand between."""
    p = pu.Product(rng(15, tokens, gated), tokens, 512, [96], gated, RANKS, 32).upload()
    other = pu.Product(rng(16, tokens, gated), tokens + 70, 640, [104], gated, RANKS, 32).upload()
    other.run()
    outs = p.outputs()
    capi.call(*p.args(outs))
    g = C.c_void_p()
    capi.call("llama2_graph_begin_capture")
    try:
        capi.call(*p.args(outs))
    finally:
        capi.call("llama2_graph_end_capture", C.byref(g))
    r = rng(17, tokens)
    for turn in range(4):
        p.x[:, :512] = r.standard_normal((p.tokens, 512))
        p.ids[:] = r.integers(-1, len(RANKS), p.tokens)
        p.positions[:] = np.where(r.random(p.tokens) < 0.3, -1, 7)
        for dev, host in ((p.dx, p.x), (p.di, p.ids), (p.dp, p.positions)):
            dev.copy_to_device(host)
        outs[0].copy_to_device(np.full((p.tokens, 96), pu.GUARD, np.float16))
        capi.call("llama2_graph_launch", g)
        other.run()
        got = outs[0].to_host().reshape(p.tokens, -1)
        eager = p.run()[0]
        assert np.array_equal(got.view(np.uint16), eager.view(np.uint16)), turn
        dead = p.positions < 0
        assert (got[dead] == pu.GUARD).all()
        want, bound = p.reference()[0]
        assert (np.abs(got.astype(np.float64) - want) <= bound)[~dead].all(), turn
    capi.call("llama2_graph_destroy", g)


def test_two_graphs_that_share_a_workspace():
    """Steps of different kernels, captured one after the other and replayed in turn, with their packed inputs and what the ranks receive in
    the library's scratch."""
    steps, graphs = [], []
    for i, (tokens, K, cols, gated) in enumerate(((1, 512, 96, False), (50, 392, 8000, False), (300, 640, 88, True))):
        steps.append(pu.Product(rng(28, i), tokens, K, [cols], gated, RANKS, 32).upload())
    want = [p.run()[0] for p in steps]
    for p in steps:
        outs, graph = p.outputs(), C.c_void_p()
        capi.call("llama2_graph_begin_capture")
        try:
            capi.call(*p.args(outs))
        finally:
            capi.call("llama2_graph_end_capture", C.byref(graph))
        graphs.append((graph, outs[0]))
    for order in ((0, 1, 2), (2, 0, 1), (1, 1, 0, 2)):
        for i in order:
            graphs[i][1].copy_to_device(np.zeros(want[i].shape, np.float16))
        for i in order:
            capi.call("llama2_graph_launch", graphs[i][0])
        for i in order:
            assert np.array_equal(graphs[i][1].to_host().view(np.uint16), want[i].ravel().view(np.uint16)), (order, i)
    for graph, _ in graphs:
        capi.call("llama2_graph_destroy", graph)


def test_threads_that_call_at_once():
    steps = [pu.Product(rng(29, i), tokens, 392, [cols], bool(i % 2), RANKS, 32).upload()
             for i, (tokens, cols) in enumerate(((1, 264), (20, 264), (50, 8000), (200, 88)))]
    want = [p.run()[0] for p in steps]
    wrong = []

    def work(p, w):
        for _ in range(20):
            if not np.array_equal(p.run()[0].view(np.uint16), w.view(np.uint16)):
                wrong.append(p.tokens)

    threads = [threading.Thread(target=work, args=a) for a in zip(steps, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


CAPTURE = """
import ctypes as C, sys
sys.path[:0] = [%r, %r]
import product_util as pu
from managedllama2_amd import capi, synth
from managedllama2_amd.device import init
init(0)
p = pu.Product(synth.rng_for(1718), 1000, 4096, [8], False, [128], 128, ids=0, junk=0.0).upload()
outs, g = p.outputs(), C.c_void_p()
capi.call("llama2_graph_begin_capture")
try:
    rc = capi.raw(*p.args(outs))
    said = capi.last_error()
finally:
    capi.call("llama2_graph_end_capture", C.byref(g))
assert rc == capi.ERR_INVALID_ARGUMENT and "capture" in said, (rc, said)
capi.call("llama2_graph_destroy", g)
p.check()
print("refused, then done")
"""


def test_a_call_that_would_need_scratch_in_a_capture_is_refused():
    """In a process of its own, whose library has no scratch yet from other calls."""
    here = os.path.dirname(os.path.abspath(__file__))
    out = subprocess.run([sys.executable, "-c", CAPTURE % (here, os.path.dirname(here))], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0 and "refused, then done" in out.stdout, out.stderr[-2000:]


def test_one_token_beside_the_module_of_one_token():
    """llama2_mat_vec_int4 and llama2_mat_vec_swiglu round the same sums, added in another order."""
    for gated, K, N in ((False, 4096, 512), (True, 2048, 352)):
        p = pu.Product(rng(19, gated), 1, K, [N], gated).upload()
        out = p.outputs()[0]
        ws, ss, zs = synth.qweight_sizes(K)
        w = [v for q in p.weights for v in (q.Weight.ptr, q.Zeros.ptr, q.Scales.ptr)]
        capi.call("llama2_mat_vec_swiglu" if gated else "llama2_mat_vec_int4", out.ptr, p.dx.ptr, *w, K, N, zs, ss, ws)
        one, (want, bound) = out.to_host().astype(np.float64), p.reference()[0]
        assert (np.abs(one - want[0]) <= bound[0]).all()
        p.check()
