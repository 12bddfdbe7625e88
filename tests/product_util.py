"""Plain restatements, in 64 bits, of the products, norms and log probabilities of a step of several requests, bounds of the
error that their arithmetic allows, and inputs for them."""
import ctypes as C

import numpy as np

from managedllama2_amd import capi, synth
from managedllama2_amd.device import DeviceVariable, QWeight

up = DeviceVariable.from_host
GUARD = np.float16(77.0)


def dequantised(q, K, N):
    """(W, Z, S) of synth.random_qweight -> [N][K] in 64 bits."""
    W, Z, S = (a.reshape(N, -1) for a in q)
    nibbles = lambda a: ((a[:, :, None] >> (4 * np.arange(8, dtype=np.uint32))) & 15).reshape(N, -1).astype(np.float64)  # noqa: E731
    group = np.arange(K) // 128
    return (nibbles(W)[:, :K] - nibbles(Z)[:, group]) * S.astype(np.float64)[:, group]


class Pool:
    """Adapters of one tensor; `junk` fills everything beyond an adapter's rank and between the adapters."""

    def __init__(self, rng, ranks, max_rank, K, N, stride=0, junk=np.nan):
        self.ranks, self.max_rank, self.K, self.N, self.stride = np.asarray(ranks, np.int32), max_rank, K, N, stride
        n = len(ranks)
        self.down = np.full((n, max_rank * K + stride), junk, np.float16)
        self.up = np.full((n, N * max_rank + stride), junk, np.float16)
        self.scales = rng.uniform(0.5, 2.0, n).astype(np.float32)
        for a, r in enumerate(np.clip(self.ranks, 0, max_rank)):
            self.down_of(a)[:r] = rng.standard_normal((r, K)) / np.sqrt(K)
            self.up_of(a)[:, :r] = rng.standard_normal((N, r)) * 0.2

    def down_of(self, a):
        return self.down[a, :self.max_rank * self.K].reshape(self.max_rank, self.K)

    def up_of(self, a):
        return self.up[a, :self.N * self.max_rank].reshape(self.N, self.max_rank)

    def upload(self):
        self.dev = [up(self.down), up(self.up), up(self.scales), up(self.ranks)]
        d, u, s, r = (v.ptr for v in self.dev)
        return capi.Adapters(down=d, up=u, scales=s, ranks=r, down_stride=self.down.shape[1] if self.stride else 0,
                             up_stride=self.up.shape[1] if self.stride else 0, n_adapters=len(self.ranks), max_rank=self.max_rank)

    def add(self, y, bound, x, ids):
        """The adapters' part of every token, onto y and its error onto bound."""
        for t, a in enumerate(ids):
            if not 0 <= a < len(self.ranks):
                continue
            r = int(np.clip(self.ranks[a], 0, self.max_rank))
            if r == 0:
                continue
            d, u, f = self.down_of(a)[:r].astype(np.float64), self.up_of(a)[:, :r].astype(np.float64), float(self.scales[a])
            h = d @ x[t]
            # fp32 sums over K terms, in any order: (K + 8) 2^-24 of their sizes, twice for the matrix cores' own rounding; two fp16
            # numbers: 2^-22 of the largest; then r terms
            off = (self.K + 8) * 2.0 ** -23 * (np.abs(d) @ np.abs(x[t])) + 2.0 ** -22 * np.abs(h).max()
            y[t] += f * (u @ h)
            bound[t] += abs(f) * (np.abs(u) @ (off + (2 * r + 8) * 2.0 ** -23 * np.abs(h)))


def product(x, q, K, N, pool=None, ids=None):
    """x: [tokens][K] -> (sums, bound of the error of sums in fp32), in 64 bits."""
    w, x = dequantised(q, K, N), x.astype(np.float64)
    y = x @ w.T
    # the products are exact; 128 of a group, the scale, the groups: in any order, twice for the matrix cores' own rounding
    bound = (128 + K // 128 + 16) * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T)
    if pool is not None:
        pool.add(y, bound, x, ids)
    return y, bound


def rounded(y, bound):
    """The bound with the rounding to fp16 behind it (below its normal numbers a step is 2^-24)."""
    return bound + 2.0 ** -11 * (np.abs(y) + bound) + 2.0 ** -25


def swiglu(g, gb, u, ub):
    s = 1.0 / (1.0 + np.exp(-g))
    # d(g s)/dg <= 1.1; exp of |g| <= 100 in fp32: (|g| + 2) 2^-24, a division and products
    bound = np.abs(u) * (1.1 * gb + np.abs(g * s) * (np.abs(g) + 8) * 2.0 ** -23) + (np.abs(g * s) + 1.1 * gb) * ub
    return g * s * u, bound


class Product:
    """A call of either product on random tensors."""

    def __init__(self, rng, tokens, K, cols, gated=False, ranks=(), max_rank=16, residual=False, pad=0, extra=0, x_extra=0, pool_stride=0,
                 junk=np.nan, ids=None, in_place=False):
        self.K, self.cols, self.gated, self.tokens, self.live = K, cols, gated, tokens + pad, tokens
        self.extra, self.x_extra, self.in_place = extra, x_extra, in_place
        tensors = cols * 2 if gated else cols
        self.q = [synth.random_qweight(rng, K, n) for n in tensors]
        for W, Z, S in self.q:  # results of about 1
            S[:] = (S.astype(np.float32) * np.float32(8 / np.sqrt(K))).astype(np.float16)
        self.pools = [Pool(rng, ranks, max_rank, K, n, pool_stride, junk) if len(ranks) else None for n in tensors]
        self.x = np.full((self.tokens, K + x_extra), np.nan, np.float16)  # NaN behind the rows, and in rows without a token
        self.x[:tokens, :K] = rng.standard_normal((tokens, K))
        self.ids = np.full(self.tokens, -1, np.int32)
        if len(ranks):
            self.ids[:] = rng.integers(-1, len(ranks) + 1, self.tokens) if ids is None else ids  # one too many: none
        self.positions = np.full(self.tokens, -1, np.int32)
        self.positions[:tokens] = rng.integers(0, 5000, tokens)
        self.residual = [rng.standard_normal((self.tokens, n + extra)).astype(np.float16) for n in cols] if residual else None

    def upload(self):
        self.weights = [QWeight.from_host(*q) for q in self.q]
        self.adapters = [p.upload() if p else None for p in self.pools]
        self.dx, self.di, self.dp = up(self.x), up(self.ids), up(self.positions)
        self.dr = [up(r) for r in self.residual] if self.residual else None
        self.batch = capi.Batch(positions=self.dp.ptr, n_requests=1, n_tokens=self.tokens, max_length=1)
        return self

    def outputs(self):
        if self.in_place:
            return [up(r) for r in self.residual]
        return [up(np.full((self.tokens, n + self.extra), GUARD, np.float16)) for n in self.cols]

    def args(self, outs):
        any_pool = any(p is not None for p in self.pools)
        ids = self.di.ptr if any_pool else None
        refs = [C.pointer(a) if a is not None else None for a in self.adapters]
        if self.gated:
            n = self.cols[0]
            return ("llama2_batch_mat_mul_swiglu", outs[0].ptr, self.dx.ptr, self.weights[0].struct(), self.weights[1].struct(), self.K, n,
                    n + self.extra, self.K + self.x_extra, refs[0], refs[1], ids, self.batch)
        m = (capi.BatchMatrix * len(self.cols))()
        for i, n in enumerate(self.cols):
            res = outs[i] if self.in_place else self.dr[i] if self.dr else None
            m[i] = capi.BatchMatrix(weight=self.weights[i].struct(), output=outs[i].ptr, residual=res.ptr if res else None, adapters=refs[i],
                                    cols=n, output_stride=n + self.extra, residual_stride=n + self.extra)
        return ("llama2_batch_mat_mul_int4", m, len(self.cols), self.dx.ptr, self.K, self.K + self.x_extra, ids, self.batch)

    def run(self):
        outs = self.outputs()
        capi.call(*self.args(outs))
        return [o.to_host().reshape(self.tokens, -1) for o in outs]

    def reference(self):
        x, ids = self.x[:self.live, :self.K], self.ids[:self.live]
        tensors = self.cols * 2 if self.gated else self.cols
        got = [product(x, q, self.K, n, p, ids) for q, n, p in zip(self.q, tensors, self.pools)]
        if self.gated:
            got = [swiglu(*got[0], *got[1])]
        if self.residual:
            got = [(y + r[:self.live, :n].astype(np.float64), b + 2.0 ** -23 * (np.abs(y) + np.abs(r[:self.live, :n])))
                   for (y, b), r, n in zip(got, self.residual, self.cols)]
        return [(y, rounded(y, b)) for y, b in got]

    def check(self, what=""):
        outs = self.run()
        before = self.residual if self.in_place else None
        for i, (out, (want, bound)) in enumerate(zip(outs, self.reference())):
            n = self.cols[i]
            untouched = before[i] if before else np.full_like(out, GUARD)
            assert np.array_equal(out[self.live:].view(np.uint16), untouched[self.live:].view(np.uint16)), "%s: rows without a token were written" % what
            assert np.array_equal(out[:, n:].view(np.uint16), untouched[:, n:].view(np.uint16)), "%s: written behind a row" % what
            got = out[:self.live, :n].astype(np.float64)
            assert np.isfinite(got).all(), (what, np.argwhere(~np.isfinite(got))[:4])
            err = np.abs(got - want)
            worst = np.unravel_index(np.argmax(err - bound), err.shape)
            assert (err <= bound).all(), "%s: tensor %d at %s got %r want %r bound %.2e" % (what, i, worst, got[worst], want[worst], bound[worst])
            # half a step at most for each result, and of the sums what K random roundings leave
            norm = np.linalg.norm
            assert norm(err) <= 2.0 ** -11 * norm(want) + 0.05 * norm(bound) + 2.0 ** -25 * np.sqrt(err.size), (what, norm(err) / norm(want))
        return outs


def rms(v, eps):
    return v / np.sqrt((v * v).mean(-1, keepdims=True) + eps)


def norm_rows(residual, x, gamma, input_gamma, gate, scale, eps):
    """((output, bound), (residual output, bound)) in 64 bits."""
    r = residual.astype(np.float64)
    b = np.zeros_like(r)
    n = residual.shape[1]
    slack = (n + 16) * 2.0 ** -24  # of a mean of squares of n fp32 terms, half of it in its root
    if x is not None:
        y = x.astype(np.float64)
        if input_gamma is not None:
            y = rms(y, eps) * input_gamma.astype(np.float64)
        if gate is not None:
            y = y * gate.astype(np.float64)
        r = r + scale * y
        b = np.abs(scale * y) * (slack + 2.0 ** -22) + 2.0 ** -23 * np.abs(r)
    out = None
    if gamma is not None:
        m = np.sqrt((r * r).mean(-1, keepdims=True) + eps)
        o = r / m * gamma.astype(np.float64)
        ob = np.abs(gamma.astype(np.float64)) / m * (b + np.abs(r) * (slack + 2.0 ** -22 + np.sqrt((b * b).mean(-1, keepdims=True)) / m))
        out = o, rounded(o, ob)
    return out, (r, rounded(r, b))


def log_probs(x, temperature):
    """One row -> (log probabilities, entropy) in 64 bits."""
    x = x.astype(np.float64) / float(np.float32(temperature))
    if np.isnan(x).any() or (x == np.inf).any():
        return np.full(len(x), np.nan), np.nan
    if (x == -np.inf).all():
        return np.full(len(x), -np.inf), 0.0
    d = x - x.max()
    lp = d - np.log(np.exp(d).sum())
    seen = lp[lp > -np.inf]
    return lp, -(np.exp(seen) * seen).sum()


def top_tokens(x, n):
    """In the order of the logits, NaN last, equal ones by index; -1 where there are no more."""
    v = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    order = np.lexsort((np.arange(len(x)), -v, np.isnan(x)))[:n]
    return np.concatenate([order, np.full(n - len(order), -1)]).astype(np.int32)
