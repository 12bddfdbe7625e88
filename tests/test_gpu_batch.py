"""GPU parity of the operators of a step of several requests (block tables and slots, norm + rotation + store into the
paged cache, attention behind a shared prefix) against 64-bit restatements (batch_util), one by one and as a step runs them."""
import ctypes as C
import math

import numpy as np
import pytest

import batch_util as bu
from managedllama2_amd import capi, synth
from managedllama2_amd.device import DeviceVariable
from gpu_util import up

pytestmark = pytest.mark.gpu


def zeros(n):
    return up(np.zeros(n, np.int32))


# ---------------------------------------------------------------- tables

class TablesCall:
    def __init__(self, table, cached, counts, free, taken, size, prefix, n_tokens):
        self.host = (table, cached, counts, free, taken, size, prefix, n_tokens)
        n = len(cached)
        self.table, self.cached, self.counts = up(table), up(cached), up(counts)
        self.free, self.n_free = up(free if len(free) else np.zeros(1, np.int32)), len(free)
        self.taken = up(np.array([taken], np.int32))
        self.lengths, self.starts, self.positions, self.slots, self.new_taken = zeros(n), zeros(n + 1), zeros(n_tokens), zeros(n_tokens), zeros(1)
        self.size = size
        self.batch = capi.Batch(block_tables=self.table.ptr, lengths=self.lengths.ptr, query_starts=self.starts.ptr,
                                positions=self.positions.ptr, slots=self.slots.ptr, n_requests=n, n_tokens=n_tokens,
                                table_stride=table.shape[1], prefix_length=prefix)

    def run(self):
        capi.call("llama2_batch_tables", self.batch, self.cached.ptr, self.counts.ptr, self.free.ptr, self.n_free, self.taken.ptr,
                  self.new_taken.ptr, self.size)

    def check(self, what):
        self.run()
        table, cached, counts, free, taken, size, prefix, n_tokens = self.host
        want = bu.tables(*self.host)
        got = (self.table.to_host().reshape(table.shape), self.lengths.to_host(), self.starts.to_host(), self.positions.to_host(),
               self.slots.to_host(), int(self.new_taken[0]))
        for name, g, w in zip(("tables", "lengths", "starts", "positions", "slots", "taken"), got, want):
            assert np.array_equal(g, w), "%s: %s differ at %s" % (what, name, np.argwhere(np.asarray(g) != np.asarray(w))[:4])


def tables_case(seed, n, size, ctx_hi, new_hi, pad=0, short=0, odd=False, prefix=0, stride=None, taken=2):
    rng = synth.rng_for(1201, seed)
    cached = rng.integers(0, ctx_hi + 1, n).astype(np.int32)
    counts = rng.integers(0, new_hi + 1, n).astype(np.int32)
    if odd:  # requests that must be refused, each for another reason
        counts[rng.integers(0, n, max(1, n // 9))] = -3
        cached[rng.integers(0, n, max(1, n // 9))] = -1
        cached[rng.integers(0, n, max(1, n // 9))] = 0x7FFFFFFF
        counts[rng.integers(0, n)] = 0x7FFFFFF0
    have = -(-np.clip(cached, 0, ctx_hi) // size)
    stride = stride or int(-(-(ctx_hi + new_hi) // size)) + 1
    need = int((-(-(np.clip(cached, 0, ctx_hi) + np.clip(counts, 0, new_hi)) // size) - have).sum())
    ids = rng.permutation(int(have.sum()) + need + taken + 10).astype(np.int32)
    table = np.full((n, stride), -5, np.int32)
    at = 0
    for b in range(n):
        k = min(int(have[b]), stride)
        table[b, :k] = ids[at:at + k]
        at += k
    free = ids[at:at + max(0, need + taken - short)].copy()
    total = int(np.clip(counts, 0, new_hi).sum())
    return TablesCall(table, cached, counts, free, min(taken, len(free)), size, prefix, max(1, total + pad))


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 200, 1023, 1024, 1025, 2500])
@pytest.mark.parametrize("size", [8, 16, 1024])
def test_tables_of_decode_steps(n, size):
    tables_case(n, n, size, 3000, 1, pad=n % 7, prefix=n * 3).check("decode %d %d" % (n, size))


@pytest.mark.parametrize("n,size,new_hi,pad,short", [(1, 8, 1, 0, 0), (1, 16, 5000, 3, 0), (7, 8, 700, 0, 0), (48, 16, 2000, 5, 100),
                                                     (300, 32, 90, 1, 17), (1100, 8, 40, 64, 400), (5, 128, 40000, 0, 3)])
def test_tables_of_prompts_and_a_pool_that_runs_dry(n, size, new_hi, pad, short):
    tables_case(50 + n, n, size, 0 if n == 48 else 200, new_hi, pad, short, prefix=11).check("prompts")


@pytest.mark.parametrize("n", [3, 70, 1500])
@pytest.mark.parametrize("short", [0, 5])
def test_tables_refuse_single_requests(n, short):
    tables_case(n, n, 16, 400, 20, 9, short, odd=True, prefix=5).check("odd")


def test_tables_too_narrow_and_too_few_tokens():
    tables_case(7, 90, 16, 400, 30, 0, 0, stride=20).check("table_stride")
    tables_case(8, 90, 16, 400, 30, -200).check("n_tokens")
    tables_case(9, 1300, 8, 400, 30, -9000, 50).check("n_tokens of 1300 requests")


@pytest.mark.parametrize("taken", [-1, 5, 0x7FFFFFFF])
def test_tables_with_a_count_of_taken_blocks_that_cannot_be(taken):
    c = tables_case(11, 20, 16, 100, 20)
    table, cached, counts, free, _, size, prefix, n_tokens = c.host
    TablesCall(table, cached, counts, free[:4], taken, size, prefix, n_tokens).check("taken %d" % taken)
    TablesCall(table, cached, counts, free[:0], 0, size, prefix, n_tokens).check("no free blocks")


def test_tables_of_a_request_that_goes_on_behind_a_refused_one():
    """One needs two blocks where one is left, the next none, the last one: the second goes on, and the count says that the list is
    exhausted; from then on nobody gets a block and the count stays."""
    size = 8
    table = np.array([[0, -5, -5], [1, -5, -5], [2, -5, -5]], np.int32)
    cached, counts, free = np.array([8, 3, 8], np.int32), np.array([9, 2, 1], np.int32), np.array([9, 7, 6, 5], np.int32)
    c = TablesCall(table, cached, counts, free, 3, size, 0, 12)
    c.check("dry")
    assert c.lengths.to_host().tolist() == [8, 5, 8] and int(c.new_taken[0]) == 3 + 2 > len(free)
    c = TablesCall(table, np.array([8, 5, 8], np.int32), counts, free, 5, size, 0, 12)
    c.check("still dry")
    assert c.lengths.to_host().tolist() == [8, 7, 8] and int(c.new_taken[0]) == 5


def test_tables_of_block_ids_that_have_no_slots():
    # 16 rows per block: 2^27 - 1 is the last id whose slots are ints; 2^28 would come out as block 0 again
    ids = [(1 << 27) - 1, 1 << 27, 1 << 28, (1 << 28) + 3, -1, -(1 << 31), 5]
    n = len(ids)
    table, cached, counts = up(np.zeros((n, 2), np.int32)), zeros(n), up(np.full(n, 2, np.int32))
    lengths, starts, positions, slots = zeros(n), zeros(n + 1), zeros(2 * n), zeros(2 * n)
    b = capi.Batch(table.ptr, lengths.ptr, starts.ptr, positions.ptr, slots.ptr, None, n, 2 * n, 2, 0, 0)
    free, taken = up(np.array(ids, np.int32)), zeros(1)
    capi.call("llama2_batch_tables", b, cached.ptr, counts.ptr, free.ptr, n, taken.ptr, taken.ptr, 16)
    first = [i * 16 if 0 <= i < 1 << 27 else -1 for i in ids]
    assert slots.to_host().tolist() == [v for s in first for v in (s, s + 1 if s >= 0 else -1)]
    assert positions.to_host().tolist() == [0, 1] * n and table.to_host().reshape(n, 2)[:, 0].tolist() == ids


def test_tables_in_place_and_replayed():
    """Lengths and the number of taken blocks updated in place: a captured step counts on by itself."""
    c = tables_case(12, 40, 8, 50, 1, pad=4, short=-200, stride=30)
    table, lengths, counts, free, taken, size, prefix, n_tokens = c.host
    c.batch.lengths = c.cached.ptr
    run = lambda: capi.call("llama2_batch_tables", c.batch, c.cached.ptr, c.counts.ptr, c.free.ptr, c.n_free, c.taken.ptr, c.taken.ptr, size)  # noqa: E731
    g = C.c_void_p()
    capi.call("llama2_graph_begin_capture")
    try:
        run()
    finally:
        capi.call("llama2_graph_end_capture", C.byref(g))
    for rep in range(30):
        if rep % 3 == 2:
            run()
        else:
            capi.call("llama2_graph_launch", g)
        table, lengths, starts, positions, slots, taken = bu.tables(table, lengths, counts, free, taken, size, prefix, n_tokens)
        assert np.array_equal(c.cached.to_host(), lengths) and int(c.taken[0]) == taken, rep
        assert np.array_equal(c.table.to_host().reshape(table.shape), table) and np.array_equal(c.slots.to_host(), slots), rep
        assert np.array_equal(c.positions.to_host(), positions) and np.array_equal(c.starts.to_host(), starts), rep
    capi.call("llama2_graph_destroy", g)


# ---------------------------------------------------------------- norm, rotation, store

class RopeCall:
    def __init__(self, rng, positions, slots, heads, kv_heads, d, size, n_blocks, norms="both", fused=False, stride_extra=0, eps=1e-5,
                 theta=10000.0, in_place=False, std=1.0):
        self.positions, self.slots = np.asarray(positions, np.int32), np.asarray(slots, np.int32)
        t = len(self.positions)
        self.heads, self.kv_heads, self.d, self.size, self.n_blocks, self.eps, self.theta = heads, kv_heads, d, size, n_blocks, eps, theta
        wq, wk = heads * d, kv_heads * d
        f16 = lambda *shape: (rng.standard_normal(shape, np.float32) * std).astype(np.float16)  # noqa: E731
        if fused:
            qkv = f16(t, wq + 2 * wk + 8)
            self.q, self.k, self.v = qkv[:, :wq], qkv[:, wq:wq + wk], qkv[:, wq + wk:wq + 2 * wk]
            self.dev = up(qkv)
            self.ptr = [self.dev.offset_pointer(x) for x in (0, wq, wq + wk)]
            self.stride = [qkv.shape[1]] * 2
        else:
            self.q, self.k, self.v = f16(t, wq), f16(t, wk), f16(t, wk)
            self.dev = [up(self.q), up(self.k), up(self.v)]
            self.ptr = [x.ptr for x in self.dev]
            self.stride = [wq, wk]
        gamma = lambda: (1 + 0.2 * rng.standard_normal(d, np.float32)).astype(np.float16)  # noqa: E731
        self.gq = gamma() if norms in ("both", "q") else None
        self.gk = gamma() if norms in ("both", "k") else None
        self.dg = [up(g) if g is not None else None for g in (self.gq, self.gk)]
        self.block = size * wk + stride_extra
        self.key, self.value = f16(n_blocks, self.block), f16(n_blocks, self.block)
        self.dk, self.dv, self.dp, self.ds = up(self.key), up(self.value), up(self.positions), up(self.slots)
        self.in_place = in_place
        self.out = None if in_place else up(np.full((t, wq + 16), 55.0, np.float16))
        self.batch = capi.Batch(positions=self.dp.ptr, slots=self.ds.ptr, n_requests=1, n_tokens=t)
        self.cache = capi.PagedCache(key=self.dk.ptr, value=self.dv.ptr, block_stride=self.block, n_blocks=n_blocks, block_size=size,
                                     n_kv_heads=kv_heads, head_size=d)

    def run(self):
        wq = self.heads * self.d
        out, stride = (self.ptr[0], self.stride[0]) if self.in_place else (self.out.ptr, wq + 16)
        capi.call("llama2_batch_qk_norm_rope", out, *self.ptr, *[g.ptr if g else None for g in self.dg], self.batch, self.cache,
                  self.heads, stride, *self.stride, self.eps, self.theta)
        if self.in_place:
            got = (self.dev if not isinstance(self.dev, list) else self.dev[0]).to_host().reshape(len(self.positions), -1)
            return got[:, :wq]
        got = self.out.to_host().reshape(-1, wq + 16)
        assert (got[:, wq:] == 55).all()
        return got[:, :wq]

    def check(self, what=""):
        got = self.run()
        keys, values = self.dk.to_host().reshape(self.key.shape), self.dv.to_host().reshape(self.value.shape)
        live, wk = self.positions >= 0, self.kv_heads * self.d
        before = self.q if self.in_place else np.full_like(self.q, 55)
        assert np.array_equal(got[~live], before[~live]), what
        pos = np.maximum(self.positions, 0)
        self.close(got[live], *[x[live] for x in bu.rope(self.q, pos, self.gq, self.eps, self.theta, self.d)], what + " q")
        k, size = bu.rope(self.k, pos, self.gk, self.eps, self.theta, self.d)
        stored = live & (self.slots >= 0) & (self.slots < self.n_blocks * self.size)
        at = self.slots[stored]
        rows = lambda c: c[:, :self.size * wk].reshape(-1, wk)  # noqa: E731
        want_k, want_v = self.key.copy(), self.value.copy()
        self.close(rows(keys)[at], k[stored], size[stored], what + " k")
        want_k[:, :self.size * wk] = want_k[:, :self.size * wk]
        rk, rv = want_k[:, :self.size * wk].reshape(-1, wk).copy(), want_v[:, :self.size * wk].reshape(-1, wk).copy()
        rk[at], rv[at] = rows(keys)[at], self.v[stored]
        want_k[:, :self.size * wk], want_v[:, :self.size * wk] = rk.reshape(self.n_blocks, -1), rv.reshape(self.n_blocks, -1)
        assert np.array_equal(keys.view(np.uint16), want_k.view(np.uint16)), what + ": other keys changed"
        assert np.array_equal(values.view(np.uint16), want_v.view(np.uint16)), what + ": values"

    def close(self, got, want, size, what):
        # result rounded to fp16; cosine and sine to 2^-21 (argument rounded at up to half a turn, 2 ulp of the function); the mean of
        # squares in fp32, at most d roundings, the root and two products: 2^-16 covers all of it for d <= 128
        bound = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + 2.0 ** -16 * size
        err = np.abs(got.astype(np.float64) - want)
        assert (err <= bound).all(), "%s: off by %.3e, %.3e allowed" % (what, (err - bound).max(), bound.flat[np.argmax(err - bound)])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(32, 32), (8, 2), (5, 1), (16, 16), (17, 17), (1, 1), (40, 8)])
@pytest.mark.parametrize("norms", ["both", None])
def test_rope_heads(d, heads, kv_heads, norms):
    rng = synth.rng_for(1301, d, heads, kv_heads)
    t = 13
    RopeCall(rng, rng.integers(0, 5000, t), rng.permutation(10 * 16)[:t], heads, kv_heads, d, 16, 10, norms).check()


@pytest.mark.parametrize("tokens", [1, 2, 3, 100, 1500])
@pytest.mark.parametrize("fused,in_place", [(False, False), (True, False), (True, True), (False, True)])
def test_rope_tokens_and_layouts(tokens, fused, in_place):
    rng = synth.rng_for(1302, tokens, fused, in_place)
    blocks = tokens // 8 + 2
    RopeCall(rng, rng.integers(0, 100000, tokens), rng.permutation(blocks * 8)[:tokens], 6, 2, 128, 8, blocks, "q" if fused else "k", fused,
             stride_extra=24, in_place=in_place).check()


@pytest.mark.parametrize("theta", [1.0, 10000.0, 1e6])
def test_rope_far_positions(theta):
    """Angles of positions that 24 bits do not hold, up to the last one there is."""
    rng = synth.rng_for(1303)
    p = np.array([0, 1, 2, 16777217, 33554431, 100000007, 1 << 30, (1 << 31) - 1, (1 << 31) - 2, 1234567890])
    RopeCall(rng, p, rng.permutation(32)[:len(p)], 4, 4, 128, 16, 2, None, theta=theta).check()
    RopeCall(rng, p, rng.permutation(32)[:len(p)], 4, 4, 64, 16, 2, "both", theta=theta).check()


def test_rope_skips_tokens_without_position_or_slot():
    rng = synth.rng_for(1304)
    p = np.array([5, -1, 7, 8, -1, 9, 10, 11, -2])
    s = np.array([3, 4, -1, 31, -1, 32, 0x7FFFFFFF, 0, 9])  # 32 and beyond: no slot of the cache
    for in_place in (False, True):
        RopeCall(rng, p, s, 4, 2, 128, 16, 2, "both", in_place=in_place).check()


def test_rope_extreme_values():
    rng = synth.rng_for(1305)
    c = RopeCall(rng, [3, 4000], [1, 9], 2, 2, 128, 16, 1, "both", std=1e-4)  # mean of squares far below eps' square root
    c.check("small")
    RopeCall(rng, [3, 4000], [1, 9], 2, 2, 128, 16, 1, "both", eps=0.0, std=400.0).check("large")
    RopeCall(rng, [3, 4000], [1, 9], 2, 2, 64, 16, 1, "both", eps=0.0, std=1e-6).check("subnormal")


def test_rope_agrees_with_the_module_of_one_token():
    """Without norms it is RoPERotation for every token, up to the roundings of the angle."""
    rng = synth.rng_for(1306)
    c = RopeCall(rng, [0, 1, 77, 511], [0, 1, 2, 3], 4, 4, 128, 16, 1, None)
    got, keys = c.run(), None
    keys = c.dk.to_host().reshape(16, -1)
    for t, p in enumerate(c.positions):
        dq, dk = up(c.q[t]), up(c.k[t])
        capi.call("llama2_rope", dq.ptr, dk.ptr, 4, 128, int(p), 10000.0, 4)
        for a, b in ((dq.to_host(), got[t]), (dk.to_host(), keys[t])):
            # the module's angle is off by up to p * 2^-23 of itself (an fp32 frequency times an fp32 position)
            assert np.abs(a.astype(np.float32) - b).max() <= 8 * (2.0 ** -11 + p * 2.0 ** -22), p


# ---------------------------------------------------------------- attention

def step(seed, ctx, new, size=16, **other):
    return bu.Step(synth.rng_for(1401, seed), ctx, new, size, **other)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 2), (5, 1), (16, 1), (17, 1), (40, 8), (130, 1)])
def test_attention_heads(d, heads, kv_heads):
    for prefix in (0, 100):
        step(heads, [0, 5, 130, 33], [1, 1, 1, 1], prefix=prefix, heads=heads, kv_heads=kv_heads, d=d, fill=np.nan).check("prefix %d" % prefix)


@pytest.mark.parametrize("rows", [1, 2, 3, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 777, 1024, 1025, 2049])
def test_attention_lengths_of_one_request(rows):
    step(rows, [rows - 1], [1], heads=2, kv_heads=2, fill=np.nan).check("decode")
    step(rows, [0], [rows], heads=1, kv_heads=1, d=64, fill=np.inf).check("prompt")


@pytest.mark.parametrize("prefix", [1, 8, 31, 63, 64, 65, 128, 200, 1000, 1025, 2300])
@pytest.mark.parametrize("new", [[1, 1, 1], [1, 3, 0, 7], [40, 1, 25], [200, 130, 71]])
def test_attention_prefix_lengths(prefix, new):
    ctx = [prefix % 7, 40, 0, 300][:len(new)]
    step(prefix, ctx, new, heads=2, kv_heads=1, prefix=prefix, fill=np.nan, pad=3).check("prefix")


@pytest.mark.parametrize("prefix", [13, 31, 32, 33, 63, 64, 65, 127, 128, 200, 1025])
@pytest.mark.parametrize("requests,heads,kv_heads", [(70, 40, 40), (16, 80, 40), (30, 32, 32), (300, 8, 8)])
def test_attention_shared_prefixes(prefix, requests, heads, kv_heads):
    """Enough requests and heads that the prefix is shared: in narrow tiles (bounds for long own rows) and in wide ones, with
    several tokens per request among them."""
    prefix = max(prefix, -(-(1 << 15) // ((requests - 1) * kv_heads)))
    rng = synth.rng_for(1405, prefix, requests)
    ctx, ones = rng.integers(0, 40, requests), np.ones(requests, int)
    step(prefix, ctx, ones, 8, heads=heads, kv_heads=kv_heads, d=64, prefix=prefix, pad=2, extra=5000, fill=np.nan).check("narrow")
    new = np.where(rng.random(requests) < 0.2, rng.integers(0, 6, requests), 1)
    step(prefix, ctx, new, 16, heads=heads, kv_heads=kv_heads, d=64, prefix=prefix, pad=2, fill=np.nan).check("turns")
    if prefix in (65, 200):
        step(prefix, ctx, ones, 8, heads=heads, kv_heads=kv_heads, d=128, prefix=prefix, fill=np.nan).check("d 128")


@pytest.mark.parametrize("requests", [2, 16, 17, 65, 130, 300])
def test_attention_many_requests(requests):
    """Columns of the shared rows: a narrow tile, several of them, wide tiles; requests without tokens among them."""
    rng = synth.rng_for(1402, requests)
    ctx = np.exp(rng.uniform(0, 6, requests)).astype(int)
    new = np.where(rng.random(requests) < 0.1, 0, 1)
    new[0] = 1
    for prefix in (0, 70, 700):
        step(requests, ctx, new, heads=2, kv_heads=2, prefix=prefix, pad=5, fill=np.nan).check("prefix %d" % prefix)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(40, 40), (80, 20), (40, 8)])
@pytest.mark.parametrize("prefix", [0, 10, 33])
def test_attention_many_short_requests(d, heads, kv_heads, prefix):
    """A wavefront per tile: more tiles than workgroups fit, a few rows each, some requests with several tokens or none."""
    rng = synth.rng_for(1406, d, heads, prefix)
    n = -(-800 // kv_heads)
    ctx, new = rng.integers(0, 64 - prefix - 4, n), rng.choice([0, 1, 1, 1, 1, 1, 1, 1, 3], n)
    new[0], ctx[1], new[1] = 1, 0, 1
    step(n, ctx, new, 8, heads=heads, kv_heads=kv_heads, d=d, prefix=prefix, pad=3, fill=np.nan).check("short")


@pytest.mark.parametrize("size", [8, 16, 32, 64, 128, 256, 1024])
def test_attention_block_sizes(size):
    for kv_heads in (1, 3):
        step(size, [700, 3, 90], [2, 20, 1], size, heads=3, kv_heads=kv_heads, prefix=90, stride_extra=40, fill=np.nan).check("size %d" % size)
        step(size, [700, 3, 90], [1, 1, 1], size, heads=3, kv_heads=kv_heads, prefix=90, stride_extra=40, fill=np.nan).check("size %d" % size)


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [5, 1, 16, 2], [17, 60, 1, 128], [129, 1, 300, 64], [1, 400, 1, 1]])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (4, 1), (10, 2)])
def test_attention_turns(new, heads, kv_heads):
    """Requests that bring different numbers of tokens; a single long prompt among decoding requests."""
    for prefix in (0, 77):
        for d in (64, 128):
            step(sum(new), [9, 260, 0, 64], new, heads=heads, kv_heads=kv_heads, d=d, prefix=prefix, pad=2, fill=np.nan).check("d %d" % d)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("prefix", [0, 1, 64, 65, 130, 300])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (4, 1)])
def test_attention_few_tiles_of_many_passes(d, prefix, heads, kv_heads):
    """Fewer tiles than compute units: the passes go to two halves of a workgroup by turns, odd and even numbers of them, shared
    rows and own ones; requests of few tokens and of none among them, blocks that are none, and pieces."""
    for ctx, new in (([0, 256], [300, 64]), ([190, 0, 3], [130, 1, 400]), ([255, 30, 900, 0], [129, 3, 150, 16]), ([0, 9], [700, 0]),
                     ([1800, 40], [200, 90])):
        s = step(prefix + len(ctx), ctx, new, heads=heads, kv_heads=kv_heads, d=d, prefix=prefix, pad=3, fill=np.nan)
        s.check("new %s" % new)
        for b, r in ((0, 0), (0, 16 * 7), (len(ctx) - 1, 16)):  # these rows' blocks
            if r < s.lengths[b]:
                s.table[b, r // s.size] = -1 - r
        s.check("new %s, blocks that are none" % new)


def test_attention_long_requests_in_many_pieces():
    step(1, [9000, 20, 3000], [1, 1, 1], 64, heads=4, kv_heads=1, fill=np.nan).check("decode")
    step(2, [9000, 20, 3000], [2, 30, 1], 64, heads=4, kv_heads=2, prefix=5000, fill=np.nan).check("turns")
    step(3, [70000], [1], 1024, heads=1, kv_heads=1, d=64, fill=np.nan).check("one")


def test_attention_bounds_larger_than_the_lengths():
    """A captured step: max_length and n_tokens of later steps."""
    for new in ([1, 1, 1], [30, 2, 1]):
        for prefix in (0, 50):
            step(4, [5, 200, 64], new, heads=2, kv_heads=2, prefix=prefix, extra=30000, pad=40, fill=np.nan).check("new %s" % new, out_extra=24)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 65504.0])
def test_attention_later_rows_have_no_influence(bad, d):
    """Keys and values of a request's later tokens: whatever they hold, tokens in front of them do not see it."""
    for new, watch in (([1, 6, 1], [(1, 3)]), ([90, 200, 30], [(0, 10), (1, 150), (2, 29)]), ([16, 12, 1], [(0, 15), (1, 1)])):
        for heads, kv_heads in ((2, 2), (4, 1)):
            s = step(int(sum(new)), [30, 64, 0], new, heads=heads, kv_heads=kv_heads, d=d, prefix=40)
            clean = s.check()
            for b, first in watch:  # rows of tokens first .. of request b
                r = np.arange(s.ctx[b] + first, s.lengths[b])
                for c in (s.key, s.value):
                    s.rows_of(c)[s.table[b, r // s.size], r % s.size] = bad
            s.upload()
            got = s.run()
            for b in range(3):
                first = min([f for w, f in watch if w == b], default=s.new[b])
                t = slice(s.starts[b], s.starts[b] + first)
                assert np.array_equal(got[t], clean[t]) or np.abs(got[t].astype(np.float32) - clean[t]).max() <= 2.0 ** -10 * np.abs(
                    clean[t]).max(), (new, heads, b)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [[6, 1], [100, 3], [200, 70]])
def test_attention_values_that_are_not_finite(new, d):
    """An infinite value reaches the tokens that attend its row, at its element; the others do not notice."""
    s = step(12, [20, 50], new, heads=2, kv_heads=1, d=d, prefix=30)
    clean = s.check()
    own = s.ctx[0] + new[0] // 2 # row of the token in the middle
    rows = s.rows_of(s.value)
    at = s.table[0, own // s.size], own % s.size
    for value, elements in ((np.inf, (0, 5)), (-np.inf, (d // 2,)), (np.nan, (d - 1,))):
        for e in elements:
            rows[at[0], at[1], e] = value
    s.upload()
    got = s.run().astype(np.float32)
    sees = np.zeros(len(got), bool)
    sees[new[0] // 2:new[0]] = True
    assert np.abs(got[~sees] - clean[~sees]).max() <= 2.0 ** -10 * np.abs(clean).max()
    for h in (0, d):
        g = got[sees][:, h:h + d]
        assert (g[:, [0, 5]] == np.inf).all() and (g[:, d // 2] == -np.inf).all() and np.isnan(g[:, d - 1]).all()
        others = np.setdiff1d(np.arange(d), [0, 5, d // 2, d - 1])
        assert np.abs(g[:, others] - clean[sees][:, h:h + d][:, others]).max() <= 2.0 ** -10 * np.abs(clean).max()


def test_attention_without_rows_and_without_blocks():
    """Blocks that are none are not attended; tokens whose blocks all are give zeros."""
    for new in ([1, 1, 1], [20, 30, 40], [3, 90, 1]):
        for prefix in (0, 100):
            s = step(6, [100, 200, 70], new, heads=2, kv_heads=1, prefix=prefix, fill=np.nan)
            s.table[0, :] = -1
            s.table[1, 1] = s.n_blocks
            s.table[1, 5] = -1 << 31
            s.table[2, 0] = 0x7FFFFFFF
            s.key[0] = s.value[0] = np.nan  # what a clamped id would read
            for b in range(3):
                s.table[b][s.table[b] == 0] = -1
            if prefix:
                s.prefix_table = np.where(s.prefix_table == 0, -1, s.prefix_table).astype(np.int32)
                s.prefix_table[2] = -9
            got = s.check("new %s prefix %d" % (new, prefix))
            if not prefix:
                assert not got[:new[0]].any()


def test_attention_positions_beyond_the_rows():
    """A position whose rows max_length (or the table) does not hold attends those that there are, up to the largest int."""
    for new in ([1, 1], [30, 2], [300, 1]):
        for prefix in (0, 70):
            s = step(8, [40, 300], new, heads=2, kv_heads=1, prefix=prefix)
            s.positions[s.starts[2] - 1] = s.positions[s.starts[1] - 1] = (1 << 31) - 1
            s.max_length = min(s.lengths)
            s.upload()
            got = s.run()
            for b in (0, 1):  # the others' positions are what they were; max_length cuts all of them
                t = slice(s.starts[b], s.starts[b + 1])
                last = np.minimum(s.positions[t], prefix + s.max_length - 1)
                flat = [np.ascontiguousarray(s.rows_of(c)).reshape(-1, s.width) for c in (s.key, s.value)]
                want, bound = bu.attention(s.q[t], *flat, s.row_numbers(s.prefix_table, prefix), s.row_numbers(s.table[b], s.lengths[b]),
                                           last, prefix, s.scale, s.kv_heads, s.d)
                assert (np.abs(got[t].astype(np.float64) - want) <= bound).all(), (new, prefix, b)


def test_attention_large_scores():
    """Scores of thousands, both signs, a negative scale, and keys at the end of the type."""
    for d in (64, 128):
        for new in ([1, 1], [40, 30]):
            s = step(8, [300, 90], new, heads=2, kv_heads=1, d=d, prefix=80)
            s.key *= np.float16(30)
            s.check("large")
            s.scale = -0.3
            s.check("negative")
            s.scale = 0.0
            s.check("all alike")
            s.scale = 1.0 / math.sqrt(d)
            s.key[:] = np.where(s.key > 0, 65504, -65504)
            s.q[:] = np.abs(s.q)
            s.upload()
            assert np.isfinite(s.run()).all()


def test_attention_is_the_same_every_time():
    s = step(9, [4000, 30, 700], [1, 25, 1], heads=8, kv_heads=2, prefix=900)
    s.upload()
    first = s.run()
    for _ in range(5):
        assert np.array_equal(first.view(np.uint16), s.run().view(np.uint16))


@pytest.mark.parametrize("d", [64, 128])
def test_operators_beyond_4_gb(d):
    """Blocks at the far end of a cache of more than 4 GB (and 2^31 elements)."""
    kv, size = 8, 128
    block = size * kv * d
    n_blocks = (5 << 30) // (2 * block)
    key, value = DeviceVariable(np.float16, n_blocks * block), DeviceVariable(np.float16, n_blocks * block)
    cache = capi.PagedCache(key=key.ptr, value=value.ptr, block_stride=0, n_blocks=n_blocks, block_size=size, n_kv_heads=kv, head_size=d)
    rng = synth.rng_for(1403, d)
    t = 2 * size + 5
    table = np.array([n_blocks - 1, 1, n_blocks // 2 + 3], np.int32)
    rows = np.arange(t)
    slots, positions = (table[rows // size] * size + rows % size).astype(np.int32), rows.astype(np.int32)
    q, k, v = (rng.standard_normal((t, kv * d), np.float32).astype(np.float16) for _ in range(3))
    dev = dict(block_tables=up(table), query_starts=up(np.array([0, t], np.int32)), positions=up(positions), slots=up(slots))
    batch = capi.Batch(n_requests=1, n_tokens=t, table_stride=3, prefix_length=0, max_length=t, **{n: x.ptr for n, x in dev.items()})
    dq, dk, dv, rq, out = up(q), up(k), up(v), up(np.zeros_like(q)), up(np.zeros_like(q))
    capi.call("llama2_batch_qk_norm_rope", rq.ptr, dq.ptr, dk.ptr, dv.ptr, None, None, batch, cache, kv, kv * d, kv * d, kv * d, 0.0, 10000.0)
    capi.call("llama2_batch_attention", out.ptr, rq.ptr, batch, cache, kv, kv * d, kv * d, d ** -0.5)
    for b, first in zip(table, (0, size, 2 * size)):
        n = min(size, t - first)
        got = value.to_host(n * kv * d, int(b) * block).reshape(n, -1)
        assert np.array_equal(got, v[first:first + n])
    rotated = np.concatenate([key.to_host(size * kv * d, int(b) * block).reshape(size, -1) for b in table])[:t]
    want, size_k = bu.rope(k, positions, None, 0.0, 10000.0, d)
    assert (np.abs(rotated - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -16 * size_k + 2.0 ** -25).all()
    want, bound = bu.attention(rq.to_host().reshape(t, -1), rotated, v, np.zeros(0, int), rows, positions, 0, d ** -0.5, kv, d)
    assert (np.abs(out.to_host().reshape(t, -1) - want) <= bound).all()


def test_refusals_reach_the_caller():
    s = step(10, [5], [1], heads=2, kv_heads=2)
    s.upload()
    out = up(np.zeros_like(s.q))
    call = lambda **o: capi.raw("llama2_batch_attention", out.ptr, s.dq.ptr, s.batch, s.cache, o.get("heads", 2), 256, 256, 0.1)  # noqa: E731
    assert call() == capi.OK
    assert call(heads=3) == capi.ERR_INVALID_ARGUMENT and "n_kv_heads" in capi.last_error()
    s.cache.head_size = 96
    assert call() == capi.ERR_UNSUPPORTED and "head_size" in capi.last_error()
    assert capi.raw("llama2_batch_tables", s.batch, None, None, None, 0, None, None, 16) == capi.ERR_INVALID_ARGUMENT
    assert capi.raw("llama2_batch_qk_norm_rope", None, None, None, None, None, None, s.batch, s.cache, 2, 256, 256, 256, 0.0,
                    1e4) == capi.ERR_UNSUPPORTED


def test_attention_agrees_with_the_module_of_one_sequence():
    """A contiguous cache is a paged one whose blocks follow each other: llama2_multi_head_attention up to the fp16 scores that
    the reference's arithmetic stores."""
    rng = synth.rng_for(1404)
    dim, heads, rows = 512, 4, 900
    q, k, v = synth.normal_f16(rng, dim), synth.normal_f16(rng, 1024 * dim), synth.normal_f16(rng, 1024 * dim)
    dq, dk, dv, out, want = up(q), up(k), up(v), up(np.zeros(dim, np.float16)), up(np.zeros(dim, np.float16))
    capi.call("llama2_multi_head_attention", want.ptr, dq.ptr, dk.ptr, dv.ptr, 128, dim, rows, 128 ** -0.5, heads)
    dev = dict(block_tables=up(np.arange(64, dtype=np.int32)), query_starts=up(np.array([0, 1], np.int32)),
               positions=up(np.array([rows - 1], np.int32)))
    batch = capi.Batch(n_requests=1, n_tokens=1, table_stride=64, prefix_length=0, max_length=1024, **{n: x.ptr for n, x in dev.items()})
    cache = capi.PagedCache(key=dk.ptr, value=dv.ptr, block_stride=0, n_blocks=64, block_size=16, n_kv_heads=heads, head_size=128)
    capi.call("llama2_batch_attention", out.ptr, dq.ptr, batch, cache, heads, dim, dim, 128 ** -0.5)
    a, b = out.to_host().astype(np.float64), want.to_host().astype(np.float64)
    # |score| < 8: stored as fp16 off by up to 2^-9, so every weight by 2^-8 at most
    assert np.abs(a - b).max() <= 2.0 ** -8 * np.abs(v).max() * 0.5
