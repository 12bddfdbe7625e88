"""Plain restatements, in 64 bits, of the operators of a step of several requests, and inputs for them."""
import math

import numpy as np

from managedllama2_amd import capi
from managedllama2_amd.device import DeviceVariable


def tables(block_tables, cached, counts, free, taken, size, prefix, n_tokens):
    """llama2_batch_tables on host arrays, request by request: (tables, lengths, starts, positions, slots, taken)."""
    table, stride = block_tables.copy(), block_tables.shape[1]
    lengths, starts = cached.copy(), np.zeros(len(cached) + 1, np.int64)
    positions, slots = np.full(n_tokens, -1, np.int32), np.full(n_tokens, -1, np.int32)
    left = len(free) - taken if 0 <= taken <= len(free) else 0
    used, begin, blocked = 0, 0, 0  # blocked: what the requests so far asked for; used: up to the last one that goes on
    for b, (c, n) in enumerate(zip(cached.tolist(), counts.tolist())):
        end = begin + max(n, 0)
        fits = c >= 0 and n >= 0 and c + n <= stride * size and end <= n_tokens
        if fits:
            first = -(-c // size)
            need = -(-(c + n) // size) - first
            blocked += need
            if need == 0 or blocked <= left:
                table[b, first:first + need] = free[taken + blocked - need:taken + blocked] if need else []
                used = blocked
                lengths[b] = c + n
                rows = np.arange(c, c + n)
                positions[begin:end] = prefix + rows
                slots[begin:end] = table[b, rows // size] * size + rows % size
        starts[b + 1] = end
        begin = end
    return table, lengths, np.minimum(starts, n_tokens).astype(np.int32), positions, slots, taken + used if 0 <= taken <= len(free) else taken


def rope(x, positions, gamma, eps, theta, d):
    """x: [tokens][heads * d] -> (rotated, |a| + |b| of each pair, for the tolerance), in 64 bits."""
    y = x.astype(np.float64).reshape(len(x), -1, d)
    if gamma is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * gamma.astype(np.float64)
    i = np.arange(d // 2)
    # the angle in extended precision: a position of 2^31 leaves 64 - 31 bits behind the point
    angle = positions.astype(np.longdouble)[:, None] * np.longdouble(theta) ** (-2 * i.astype(np.longdouble) / d)
    turns = angle / (2 * np.longdouble("3.14159265358979323846264338327950288"))
    angle = ((turns - np.floor(turns)) * 2 * np.longdouble("3.14159265358979323846264338327950288")).astype(np.float64)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = y[..., :d // 2], y[..., d // 2:]
    size = np.abs(a) + np.abs(b)
    return np.concatenate([a * c - b * s, a * s + b * c], -1).reshape(x.shape), np.concatenate([size, size], -1).reshape(x.shape)


def attention(q, key, value, prefix_rows, own_rows, positions, prefix, scale, kv_heads, d):
    """One request's tokens.  q: [n][heads * d]; key, value: [rows][kv_heads * d] of the whole cache; prefix_rows, own_rows: cache
    rows, -1: not in the cache.  Returns (out, bound of the error) in 64 bits."""
    n, heads = len(q), q.shape[1] // d
    rows = np.concatenate([prefix_rows, own_rows]).astype(np.int64)
    at = np.concatenate([np.full(len(prefix_rows), -1), np.arange(len(own_rows))])
    seen = (rows >= 0)[None, :] & (at[None, :] <= (positions - prefix)[:, None])
    k = key[np.maximum(rows, 0)].astype(np.float64).reshape(len(rows), kv_heads, d)
    v = value[np.maximum(rows, 0)].astype(np.float64).reshape(len(rows), kv_heads, d)
    out, bound = np.zeros((n, heads * d)), np.zeros((n, heads * d))
    for h in range(heads):
        x = q[:, h * d:(h + 1) * d].astype(np.float64)
        kh, vh = k[:, h // (heads // kv_heads)], v[:, h // (heads // kv_heads)]
        for t in range(n):
            use = seen[t]
            if not use.any():
                continue
            s = kh[use] @ x[t] * scale
            reach = (np.abs(kh[use]) @ np.abs(x[t])).max() * abs(scale)  # of the terms of a score
            p = np.exp(s - s.max())
            y, size = p @ vh[use] / p.sum(), p @ np.abs(vh[use]) / p.sum()
            m = use.sum()
            # fp16 result; probabilities as fp16 (half a step each), their exponents: d terms in fp32, the scale and the base
            # (|s| 2^-24 each), exp2 itself 2^-22; sums over m rows in fp32 in any order; below fp16's normal numbers half a step is
            # 2^-25, of probabilities that enter times 2^6: 2^-31 of the largest
            eps = 2.0 ** -11 + 2 * ((d + 4) * 2.0 ** -24 * reach + 4 * 2.0 ** -24 * np.abs(s).max() + 2.0 ** -22) + 2 * m * 2.0 ** -24
            out[t, h * d:(h + 1) * d] = y
            bound[t, h * d:(h + 1) * d] = 2.0 ** -11 * np.abs(y) + 2.0 ** -25 + eps * size + m * 2.0 ** -31 * np.abs(vh[use]).max()
    return out, bound


class Step:
    """Requests with `ctx` cached rows that bring `new` tokens, over a cache of random blocks, and everything on the device."""

    def __init__(self, rng, ctx, new, size, prefix=0, heads=4, kv_heads=4, d=128, pad=0, extra=0, stride_extra=0, fill=None):
        self.ctx, self.new, self.size, self.prefix = list(ctx), list(new), size, prefix
        self.heads, self.kv_heads, self.d, self.pad = heads, kv_heads, d, pad
        self.lengths = [c + n for c, n in zip(ctx, new)]
        blocks = [-(-v // size) for v in self.lengths]
        shared = -(-prefix // size)
        self.n_blocks = sum(blocks) + shared + 3
        ids = rng.permutation(self.n_blocks).astype(np.int32)
        self.table_stride = max(blocks) + 2
        self.table = np.full((len(ctx), self.table_stride), -7, np.int32)  # -7: must not be read, or not followed
        at = 0
        for b, k in enumerate(blocks):
            self.table[b, :k] = ids[at:at + k]
            at += k
        self.prefix_table = ids[at:at + shared]
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.tokens = int(self.starts[-1]) + pad
        self.positions = np.full(self.tokens, -1, np.int32)
        for b, (c, n) in enumerate(zip(ctx, new)):
            self.positions[self.starts[b]:self.starts[b] + n] = prefix + c + np.arange(n)
        self.max_length = max(self.lengths) + extra
        self.width = kv_heads * d
        self.block_halfs = size * self.width + stride_extra
        shape = (self.n_blocks, self.block_halfs)
        self.key = rng.standard_normal(shape, np.float32).astype(np.float16)
        self.value = rng.standard_normal(shape, np.float32).astype(np.float16)
        self.q = rng.standard_normal((self.tokens, heads * d), np.float32).astype(np.float16)
        self.scale = 1.0 / math.sqrt(d)
        if fill is not None:  # everything that no token may see
            keep = np.zeros((self.n_blocks, size), bool)
            for b in range(len(ctx)):
                r = np.arange(self.lengths[b])
                keep[self.table[b, r // size], r % size] = True
            r = np.arange(prefix)
            keep[self.prefix_table[r // size], r % size] = True
            for c in (self.key, self.value):
                self.rows_of(c)[~keep] = fill
                c[:, size * self.width:] = fill

    def rows_of(self, cache):
        return cache[:, :self.size * self.width].reshape(self.n_blocks, self.size, self.width)

    def row_numbers(self, table, n):
        r = np.arange(n)
        block = table[r // self.size]
        return np.where((block >= 0) & (block < self.n_blocks), block.astype(np.int64) * self.size + r % self.size, -1)

    def reference(self):
        flat = [np.ascontiguousarray(self.rows_of(c)).reshape(-1, self.width) for c in (self.key, self.value)]
        out, bound = np.zeros((self.tokens, self.heads * self.d)), np.zeros((self.tokens, self.heads * self.d))
        shared = self.row_numbers(self.prefix_table, self.prefix)
        for b in range(len(self.ctx)):
            t = slice(self.starts[b], self.starts[b + 1])
            out[t], bound[t] = attention(self.q[t], *flat, shared, self.row_numbers(self.table[b], self.lengths[b]), self.positions[t],
                                         self.prefix, self.scale, self.kv_heads, self.d)
        return out, bound

    def upload(self):
        up = DeviceVariable.from_host
        self.dev = dict(block_tables=up(self.table), query_starts=up(self.starts), positions=up(self.positions))
        self.dk, self.dv, self.dq = up(self.key), up(self.value), up(self.q)
        self.dp = up(self.prefix_table) if self.prefix else None
        self.batch = capi.Batch(prefix_table=self.dp.ptr if self.dp else None, n_requests=len(self.ctx), n_tokens=self.tokens,
                                table_stride=self.table_stride, prefix_length=self.prefix, max_length=self.max_length,
                                **{k: v.ptr for k, v in self.dev.items()})
        self.cache = capi.PagedCache(key=self.dk.ptr, value=self.dv.ptr, block_stride=self.block_halfs, n_blocks=self.n_blocks,
                                     block_size=self.size, n_kv_heads=self.kv_heads, head_size=self.d)

    def run(self, out_extra=0):
        """The output, a guard value wherever nothing was written."""
        width = self.heads * self.d
        out = DeviceVariable.from_host(np.full((self.tokens, width + out_extra), 77.0, np.float16))
        capi.call("llama2_batch_attention", out.ptr, self.dq.ptr, self.batch, self.cache, self.heads, width + out_extra, width,
                  self.scale)
        got = out.to_host().reshape(self.tokens, width + out_extra)
        assert (got[:, width:] == 77).all()
        return got[:, :width]

    def check(self, what="", **other):
        self.upload()
        got = self.run(**other)
        want, bound = self.reference()
        dead = self.positions < 0
        assert (got[dead] == 77).all(), "%s: rows without a token were written" % what
        live = ~dead
        err = np.abs(got[live].astype(np.float64) - want[live])
        assert np.isfinite(got[live]).all(), (what, np.argwhere(~np.isfinite(got[live]))[:3])
        worst = np.unravel_index(np.argmax(err - bound[live]), err.shape)
        assert (err <= bound[live]).all(), "%s: at %s got %r want %r bound %.2e" % (what, worst, got[live][worst], want[live][worst],
                                                                                   bound[live][worst])
        return got
