"""The operators of a step of several requests as a server runs them: a prefix read once, prompts behind it, then steps of
one token each, captured once and replayed while lengths, tables and free blocks count on on the device.  Every step is
compared with a 64-bit restatement over the cache as it lies there, and the decode steps of every request with the
framework's modules of one sequence (llama2_rope, llama2_multi_head_attention) over a contiguous cache."""
import ctypes as C

import numpy as np
import pytest

import batch_util as bu
from managedllama2_amd import capi, hostlib, synth
from managedllama2_amd.device import DeviceVariable, PagedCache, RequestBatch, init
from managedllama2_amd.modules import BatchAttention, BatchQKNormRoPE, BatchTables
from gpu_util import up

pytestmark = pytest.mark.gpu

THETA, D = 10000.0, 128


class Server:
    """One layer: tables, rotation with the store, attention; q, k, v come from outside instead of from products."""

    def __init__(self, heads, kv_heads, block_size, n_blocks, requests, tokens, stride, max_length, prefix_rows=0, seed=1):
        init(0)
        self.heads, self.kv_heads, self.size, self.tokens, self.requests, self.prefix = heads, kv_heads, block_size, tokens, requests, prefix_rows
        self.cache = PagedCache(n_blocks, block_size, kv_heads, D)
        ids = synth.rng_for(1501, seed).permutation(n_blocks).astype(np.int32)
        n_prefix = -(-prefix_rows // block_size)
        self.prefix_ids, self.free_ids = ids[:n_prefix], ids[n_prefix:]
        self.free = up(self.free_ids)
        self.batch = RequestBatch(requests, tokens, stride, max_length, up(self.prefix_ids) if n_prefix else None, prefix_rows)
        self.counts = DeviceVariable.zeros(np.int32, requests)
        self.q, self.out = (DeviceVariable.zeros(np.float16, tokens * heads * D) for _ in range(2))
        self.k, self.v = (DeviceVariable.zeros(np.float16, tokens * kv_heads * D) for _ in range(2))
        self.norms = None
        self.tables, self.rope, self.attention = BatchTables(), BatchQKNormRoPE(), BatchAttention()

    def issue(self):
        self.tables.Forward(self.batch, self.counts, self.free, self.size)
        gq, gk = self.norms or (None, None)
        self.rope.Forward(self.q, self.q, self.k, self.v, self.batch, self.cache, self.heads, THETA, gq, gk)
        self.attention.Forward(self.out, self.q, self.batch, self.cache, self.heads, D ** -0.5)

    def put(self, counts, q, k, v):
        self.counts.copy_to_device(np.asarray(counts, np.int32))
        for dev, host in ((self.q, q), (self.k, k), (self.v, v)):
            dev.copy_to_device(host)

    def check(self, what):
        """The outputs of the step that just ran, from the rotated queries and the cache as they are now."""
        rows = lambda c: c.to_host().reshape(-1, self.kv_heads * D)  # noqa: E731
        key, value = rows(self.cache.key), rows(self.cache.value)
        table = self.batch.blockTables.to_host().reshape(self.requests, -1)
        starts, lengths, positions = self.batch.queryStarts.to_host(), self.batch.lengths.to_host(), self.batch.positions.to_host()
        q, out = self.q.to_host().reshape(self.tokens, -1), self.out.to_host().reshape(self.tokens, -1)
        r = np.arange(self.prefix)
        shared = self.prefix_ids[r // self.size].astype(np.int64) * self.size + r % self.size if self.prefix else r
        for b in range(self.requests):
            t = slice(starts[b], starts[b + 1])
            if t.start == t.stop or positions[t.start] < 0:
                continue
            r = np.arange(lengths[b])
            own = table[b, r // self.size].astype(np.int64) * self.size + r % self.size
            want, bound = bu.attention(q[t], key, value, shared, own, positions[t], self.prefix, D ** -0.5, self.kv_heads, D)
            err = np.abs(out[t].astype(np.float64) - want)
            assert (err <= bound).all(), "%s, request %d: off by %.2e, %.2e allowed" % (what, b, err.max(), bound.flat[np.argmax(err - bound)])


def normal(rng, *shape):
    return rng.standard_normal(shape, np.float32).astype(np.float16)


@pytest.mark.parametrize("heads,kv_heads,norms", [(4, 4, False), (8, 2, True)])
@pytest.mark.parametrize("prefix", [0, 75])
def test_prompts_then_captured_decode_steps(heads, kv_heads, norms, prefix):
    rng = synth.rng_for(1502, heads, prefix)
    size, requests, pad, steps = 16, 9, 3, 40
    wq, wk = heads * D, kv_heads * D
    prompts = [1, 20, 7, 33, 16, 0, 64, 2, 15]
    s = Server(heads, kv_heads, size, 120, requests, sum(prompts) + pad, 12, 190, prefix)
    if norms:
        s.norms = [up((1 + 0.1 * rng.standard_normal(D)).astype(np.float16)) for _ in range(2)]
    history = [[] for _ in range(requests)]  # per request: unrotated k and v of every own row
    if prefix:  # read as a request of its own, whose blocks are then the shared ones
        first = Server(heads, kv_heads, size, 120, 1, prefix, 12, prefix)
        first.cache, first.free, first.norms = s.cache, up(s.prefix_ids), s.norms
        shared_k, shared_v = normal(rng, prefix, wk), normal(rng, prefix, wk)
        first.put([prefix], normal(rng, prefix, wq), shared_k, shared_v)
        first.issue()
        first.check("prefix")
        assert np.array_equal(first.batch.blockTables.to_host()[:len(s.prefix_ids)], s.prefix_ids)
    # the prompts
    n = s.tokens
    q, k, v = normal(rng, n, wq), normal(rng, n, wk), normal(rng, n, wk)
    s.put(prompts, q, k, v)
    s.issue()
    s.check("prompts")
    at = 0
    for b, m in enumerate(prompts):
        history[b] += [(k[t], v[t]) for t in range(at, at + m)]
        at += m
    # decode, one token each, in buffers of the same size: a padded, captured step
    d = Server(heads, kv_heads, size, 120, requests, requests + pad, 12, 190, prefix)
    d.cache, d.free, d.norms, d.free_ids, d.prefix_ids = s.cache, s.free, s.norms, s.free_ids, s.prefix_ids
    for name in ("blockTables", "lengths", "taken"):
        setattr(d.batch, name, getattr(s.batch, name))
    d.batch.prefixTable = s.batch.prefixTable
    g = C.c_void_p()
    for step in range(steps):
        counts = (rng.random(requests) < 0.9).astype(np.int32)
        q, k, v = normal(rng, d.tokens, wq), normal(rng, d.tokens, wk), normal(rng, d.tokens, wk)
        d.put(counts, q, k, v)
        guard = np.full(d.tokens * wq, 9.0, np.float16)
        d.out.copy_to_device(guard)
        if step == 0:
            d.issue()  # eager: the scratch exists from here on
        elif step == 1:
            capi.call("llama2_graph_begin_capture")
            try:
                d.issue()
            finally:
                capi.call("llama2_graph_end_capture", C.byref(g))
            capi.call("llama2_graph_launch", g)
        elif step % 7 == 0:
            d.issue()  # the program's own work between replays
        else:
            capi.call("llama2_graph_launch", g)
        d.check("step %d" % step)
        total = int(counts.sum())
        out = d.out.to_host().reshape(d.tokens, wq)
        assert (out[total:] == 9).all()  # rows behind the last request
        for b, t in zip(np.flatnonzero(counts), range(total)):
            history[b].append((k[t], v[t]))
        assert d.batch.lengths.to_host().tolist() == [len(h) for h in history]
        if kv_heads == heads and not norms and step % 13 == 0:  # the framework's modules of one sequence
            for b, t in list(zip(np.flatnonzero(counts), range(total)))[::3]:
                rows = ([(shared_k[i], shared_v[i]) for i in range(prefix)] if prefix else []) + history[b]
                ks, vs = (np.stack([r[i] for r in rows]) for i in (0, 1))
                dk, dv, dq, o, dummy = up(ks), up(vs), up(q[t]), up(np.zeros(wq, np.float16)), up(np.zeros(wq, np.float16))
                for p in range(len(rows)):
                    capi.call("llama2_rope", dq.ptr if p == len(rows) - 1 else dummy.ptr, dk.offset_pointer(p * wk), heads, D, p, THETA, heads)
                capi.call("llama2_multi_head_attention", o.ptr, dq.ptr, dk.ptr, dv.ptr, D, wq, len(rows), D ** -0.5, heads)
                # that one stores scores as fp16: |score| < 8 off by 2^-9, a weight by 2^-8 of itself
                assert np.abs(o.to_host().astype(np.float32) - out[t]).max() <= 2.0 ** -8 * np.abs(vs).max(), (step, b)
    capi.call("llama2_graph_destroy", g)
    assert int(d.batch.taken[0]) == sum(-(-len(h) // size) for h in history)


@pytest.mark.parametrize("norms", [False, True])
def test_cpp_module_classes_do_the_same(norms):
    """BatchTables, BatchQKNormRoPE and BatchAttention of the C++ host beside those of this one: prompts, then single tokens."""
    rng = synth.rng_for(1505, int(norms))
    heads, kv_heads = 8, 2
    both = [Server(heads, kv_heads, 16, 40, 4, 60, 8, 100, 20) for _ in range(2)]
    gammas = [up((1 + 0.1 * rng.standard_normal(D)).astype(np.float16)) for _ in range(2)] if norms else None
    shared = normal(rng, 16 * 2 * kv_heads * D)
    for s in both:
        s.norms = gammas
        for c in (s.cache.key, s.cache.value):  # the prefix's rows
            for i, block in enumerate(s.prefix_ids):
                c.copy_to_device(shared[i * 16 * kv_heads * D:(i + 1) * 16 * kv_heads * D], int(block) * 16 * kv_heads * D)
    for counts in ([30, 1, 0, 17], [1, 1, 1, 1], [0, 2, 40, 1]):
        q, k, v = normal(rng, 60, heads * D), normal(rng, 60, kv_heads * D), normal(rng, 60, kv_heads * D)
        for s in both:
            s.put(counts, q, k, v)
            s.out.copy_to_device(np.full(60 * heads * D, 5.0, np.float16))
        both[0].issue()
        s = both[1]
        gq, gk = gammas or (None, None)
        hostlib.batch_step(s.batch, s.cache, s.counts, s.free, s.batch.taken, s.q, s.k, s.v, s.out, heads, THETA, D ** -0.5, gq, gk)
        for get in (lambda s: s.q, lambda s: s.out, lambda s: s.cache.key, lambda s: s.cache.value, lambda s: s.batch.blockTables,
                    lambda s: s.batch.lengths, lambda s: s.batch.slots, lambda s: s.batch.positions, lambda s: s.batch.taken):
            a, b = (get(s).to_host() for s in both)
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8)), counts
        both[0].check("%s" % counts)
    s.cache.headSize = 96
    with pytest.raises(hostlib.HostError, match="head_size"):
        hostlib.batch_step(s.batch, s.cache, s.counts, s.free, s.batch.taken, s.q, s.k, s.v, s.out, heads, THETA, D ** -0.5)


def test_a_pool_that_runs_dry_stops_requests_one_by_one():
    rng = synth.rng_for(1503)
    s = Server(2, 1, 8, 7, 5, 5, 6, 48, 0)  # 7 blocks for 5 requests
    lengths = np.zeros(5, np.int64)
    for step in range(30):
        s.put([1] * 5, normal(rng, 5, 256), normal(rng, 5, 128), normal(rng, 5, 128))
        before = s.cache.key.to_host()
        s.out.copy_to_device(np.full(5 * 256, 3.0, np.float16))
        s.issue()
        slots = s.batch.slots.to_host()
        now = s.batch.lengths.to_host()
        assert ((now - lengths == 1) == (slots >= 0)).all()
        assert (s.out.to_host().reshape(5, 256)[slots < 0] == 3).all()
        if (slots < 0).all():
            assert np.array_equal(before.view(np.uint16), s.cache.key.to_host().view(np.uint16))
        s.check("step %d" % step)
        lengths = now
    assert int(s.batch.taken[0]) == 7 and lengths.max() == 16 and lengths.min() == 8


def test_blocks_left_behind_a_refused_prompt_are_handed_out_once_taken_is_put_right():
    """A captured step, updated in place: a prompt that asks for more than is left stands in front of a request in the middle of a
    block, a resting one and padding, so that `taken` passes the list's end; the host sets it to the blocks that the lengths say were handed
    out, pauses the prompt, and the others get what is left, no block twice."""
    size, requests, free = 8, 6, np.array([20, 21, 22, 23, 24, 25], np.int32)
    b = RequestBatch(requests, 40, 6, 48)
    table = np.full((requests, 6), -5, np.int32)
    table[:, 0] = range(requests)
    lengths = np.array([8, 8, 3, 8, 0, 0], np.int32)
    b.blockTables.copy_to_device(table)
    b.lengths.copy_to_device(lengths)
    dfree, counts = up(free), up(np.zeros(requests, np.int32))
    BatchTables().Forward(b, counts, dfree, size)  # nobody brings anything
    assert np.array_equal(b.lengths.to_host(), lengths) and int(b.taken[0]) == 0
    g = C.c_void_p()
    capi.call("llama2_graph_begin_capture")
    try:
        BatchTables().Forward(b, counts, dfree, size)
    finally:
        capi.call("llama2_graph_end_capture", C.byref(g))
    blocks = lambda n: int((-(-n // size)).sum())  # noqa: E731
    taken, dry = 0, 0
    for step, new in enumerate(([9, 1, 1, 9, 0, 0], [1, 25, 1, 1, 0, 0], [0, 1, 1, 8, 0, 0], [30, 0, 8, 0, 0, 0], [0, 9, 1, 0, 1, 0])):
        counts.copy_to_device(np.array(new, np.int32))
        capi.call("llama2_graph_launch", g)
        want = bu.tables(table, lengths, np.array(new, np.int32), free, taken, size, 0, 40)
        got = b.blockTables.to_host().reshape(table.shape), b.lengths.to_host()
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]) and int(b.taken[0]) == want[5], step
        used = taken + blocks(got[1]) - blocks(lengths)
        assert used <= int(b.taken[0]) and used <= len(free)
        if int(b.taken[0]) > len(free):  # as the header says
            dry += 1
            b.taken.copy_to_device(np.array([used], np.int32))
        table, lengths, taken = got[0], got[1], used
        mine = np.concatenate([table[r, :blocks(lengths[r:r + 1])] for r in range(requests)])
        assert len(set(mine.tolist())) == len(mine)
    assert dry >= 2 and taken == len(free)
    capi.call("llama2_graph_destroy", g)


def test_large_tables_in_place():
    """More tokens than one workgroup takes, lengths and taken blocks updated in place, also when replayed."""
    import test_gpu_batch as tb
    for odd, n, new_hi in ((False, 60, 400), (True, 1500, 30)):
        c = tb.tables_case(21 + n, n, 16, 300, new_hi, 40, 30, odd=odd, prefix=9, stride=80)
        table, lengths, counts, free, taken, size, prefix, n_tokens = c.host
        assert n_tokens > 4096
        c.batch.lengths = c.cached.ptr
        run = lambda: capi.call("llama2_batch_tables", c.batch, c.cached.ptr, c.counts.ptr, c.free.ptr, c.n_free, c.taken.ptr, c.taken.ptr, size)  # noqa: E731
        run()
        g = C.c_void_p()
        capi.call("llama2_graph_begin_capture")
        try:
            run()
        finally:
            capi.call("llama2_graph_end_capture", C.byref(g))
        for rep in range(4):
            table, lengths, starts, positions, slots, taken = bu.tables(table, lengths, counts, free, taken, size, prefix, n_tokens)
            assert np.array_equal(c.cached.to_host(), lengths) and int(c.taken[0]) == taken, rep
            assert np.array_equal(c.table.to_host().reshape(table.shape), table) and np.array_equal(c.slots.to_host(), slots), rep
            assert np.array_equal(c.positions.to_host(), positions) and np.array_equal(c.starts.to_host(), starts), rep
            capi.call("llama2_graph_launch", g)
        capi.call("llama2_graph_destroy", g)


def test_captured_attentions_share_scratch_and_counters():
    """Steps of different shapes captured one by one (joined in the launch, by a second one, without pieces), replayed by turns
    with eager calls between, the last of which needs more scratch than there was at capture."""
    rng = lambda i: synth.rng_for(1501, i)  # noqa: E731
    steps = [bu.Step(rng(0), [900], [1], 16, heads=8, kv_heads=8, fill=np.nan),
             bu.Step(rng(1), [700, 30, 2100], [1, 1, 1], 16, heads=8, kv_heads=2, fill=np.nan, pad=2),
             bu.Step(rng(2), [300, 0, 64], [40, 130, 1], 32, heads=4, kv_heads=2, d=64, prefix=100, fill=np.nan),
             bu.Step(rng(3), list(range(40)), [1] * 40, 8, heads=8, kv_heads=8, d=64, prefix=300, fill=np.nan)]
    large = bu.Step(rng(4), [5000] * 30, [3] * 30, 64, heads=16, kv_heads=16, d=64)
    graphs, outs, want = [], [], []
    for s in steps:
        want.append(s.check())  # also allocates what a capture must not
    for s in steps:
        out, g = DeviceVariable.from_host(np.full((s.tokens, s.heads * s.d), 77.0, np.float16)), C.c_void_p()
        args = (out.ptr, s.dq.ptr, s.batch, s.cache, s.heads, s.heads * s.d, s.heads * s.d, s.scale)
        capi.call("llama2_graph_begin_capture")
        try:
            capi.call("llama2_batch_attention", *args)
        finally:
            capi.call("llama2_graph_end_capture", C.byref(g))
        graphs.append(g)
        outs.append(out)
    for turn in range(4):
        order = synth.rng_for(1502, turn).permutation(len(steps))
        for i in order:
            capi.call("llama2_memset", outs[i].ptr, 0x55, outs[i].size * 2)
            capi.call("llama2_graph_launch", graphs[i])
        for i in order:
            live = steps[i].positions >= 0
            got = outs[i].to_host().reshape(want[i].shape)
            assert np.array_equal(got[live].view(np.uint16), want[i][live].view(np.uint16)), (turn, i)
            assert (got[~live].view(np.uint16) == 0x5555).all(), (turn, i)
        if turn == 1:
            large.upload()
            first = large.run()
            assert np.array_equal(first.view(np.uint16), large.run().view(np.uint16))
        steps[turn].run()
    for g in graphs:
        capi.call("llama2_graph_destroy", g)
