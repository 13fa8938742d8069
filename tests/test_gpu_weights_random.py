"""Random calls on caches that track weights: appends, writes, decode steps of both
forms, prompt pieces, their queries observed, evictions, truncations and new
beginnings of several sequences and two layers, mixed.  Outputs, sums, own positions
and rows are held to a plain copy of the cache, in 64 bits."""
import numpy as np
import pytest
from test_gpu_weights import DECODE, OBSERVE, TYPES, U, chosen, stored, weights_of
from typed_rows import attend

pytestmark = pytest.mark.gpu

LAYERS = (3, 7)
N_SEQ, LIMIT = 3, 208


class _Run:
    def __init__(self, pkg, ctx, ty, seed):
        self.pkg, self.ctx, self.ty, self.rng = pkg, ctx, ty, np.random.default_rng(seed)
        self.kv = pkg.KVCache(ctx, n_slots=2, max_pages=N_SEQ * LIMIT // 16, max_seqs=N_SEQ, max_tokens_per_seq=LIMIT, ggml_type=TYPES[ty])
        self.kv.track_weights(True)
        self.ids = [self.kv.seq_create() for _ in range(N_SEQ)]
        # rows and sums by layer and sequence; a kv head's tokens have an order of their own
        self.k = np.zeros((2, N_SEQ, LIMIT, 1024), np.float32)
        self.v = self.k.copy()
        self.w = np.zeros((2, N_SEQ, LIMIT, 4))
        self.off = np.zeros((2, N_SEQ, LIMIT, 4))  # what the sums may be off
        self.own = np.zeros((2, N_SEQ, LIMIT, 4), int)
        self.n, self.gone, self.kept = np.zeros((2, N_SEQ), int), np.zeros(N_SEQ, int), np.zeros(N_SEQ, int)
        self.d_one = ctx.array(np.ones(256, np.float32))
        self.bufs = {k: ctx.empty((LIMIT, n)) for k, n in (("qg", 12288), ("q", 6144), ("g", 6144), ("k", 1024))}
        self.checked = 0

    def rows(self, n, width=1024):
        return self.rng.standard_normal((n, width)).astype(np.float32)

    def put(self, x, s, p, k, v):
        n = len(k)
        self.k[x, s, p:p + n], self.v[x, s, p:p + n] = stored(k, self.ty), stored(v, self.ty)
        self.w[x, s, p:p + n] = self.off[x, s, p:p + n] = 0
        self.own[x, s, p:p + n] = (self.gone[s] + p + np.arange(n))[:, None]
        self.n[x, s] = max(self.n[x, s], p + n)

    def add(self, x, s, q, end, query=DECODE):
        w, e = weights_of(q, self.k[x, s, :end], query)
        self.off[x, s, :end] += e + 8 * U * (self.w[x, s, :end] + w)
        self.w[x, s, :end] += w

    def turned(self, s, p, qg, key):
        """Query, gate and key rows as the framework turns them, at the token's own position."""
        self.bufs["qg"].zero()
        c = self.ctx
        c.attn_pre(1, p + int(self.gone[s]), self.d_one, self.d_one, c.array(qg), c.array(key), self.bufs["q"], self.bufs["g"], self.bufs["k"])
        return self.bufs["q"].download(1)[0], self.bufs["g"].download(1)[0], self.bufs["k"].download(1)

    def sums(self, x, s, n):
        w, t = self.ctx.empty((max(1, n), 4)), self.ctx.empty((max(1, n), 4), np.int32)
        self.kv.weights_get(LAYERS[x], [self.ids[s]], [0], [n], w, t)
        return w.download(n), t.download(n)

    def check(self, x, s):
        n = int(self.n[x, s])
        w, t = self.sums(x, s, n)
        assert np.all(np.abs(w - self.w[x, s, :n]) <= self.off[x, s, :n] * 1.01 + 1e-30) and np.array_equal(t, self.own[x, s, :n])
        k, v = self.ctx.empty((max(1, n), 1024)), self.ctx.empty((max(1, n), 1024))
        self.kv.read(LAYERS[x], self.ids[s], 0, n, k, v)
        assert np.array_equal(k.download(n), self.k[x, s, :n]) and np.array_equal(v.download(n), self.v[x, s, :n])
        self.checked += 1

    # ---- calls

    def write(self, x, s):
        p = int(self.rng.integers(self.kept[s], self.n[x, s] + 1))
        n = int(min(self.rng.integers(1, 40), LIMIT - p))
        if n < 1:
            return
        k, v = self.rows(n), self.rows(n)
        if self.rng.random() < 0.5:
            self.kv.write(LAYERS[x], self.ids[s], p, n, self.ctx.array(k), self.ctx.array(v))
        else:
            q, out = self.rows(n, 6144), self.ctx.empty((n, 24, 256))
            self.kv.attn_prefill(LAYERS[x], self.ids[s], p, n, self.ctx.array(q), self.ctx.array(k), self.ctx.array(v), out)
        self.put(x, s, p, k, v)

    def decode(self, x, _):
        some = [int(s) for s in self.rng.permutation(N_SEQ) if self.n[x, s] < LIMIT][:int(self.rng.integers(1, N_SEQ + 1))]
        if not some:
            return
        n = len(some)
        # at the end, or over an earlier position past the last eviction
        pos = [int(self.n[x, s]) if self.rng.random() < 0.7 else int(self.rng.integers(self.kept[s], self.n[x, s] + 1)) for s in some]
        key, val, out = self.rows(n), self.rows(n), self.ctx.empty((n, 24, 256))
        ids = [self.ids[s] for s in some]
        if self.rng.random() < 0.5:
            q, g, ks = self.rows(n, 6144), self.rows(n, 6144), key
            self.kv.attn_decode(LAYERS[x], ids, pos, self.ctx.array(q), out, k_new=self.ctx.array(key), v_new=self.ctx.array(val), gate=self.ctx.array(g))
        else:
            qg = self.rows(n, 12288)
            self.kv.full_core(LAYERS[x], ids, pos, self.d_one, self.d_one, self.ctx.array(qg), self.ctx.array(key), self.ctx.array(val), out)
            q, g, ks = np.empty((n, 6144), np.float32), np.empty((n, 6144), np.float32), np.empty_like(key)
            for b, (s, p) in enumerate(zip(some, pos)):
                q[b], g[b], k = self.turned(s, p, qg[b], key[b])
                ks[b] = k[0]
        got = out.download()
        for b, (s, p) in enumerate(zip(some, pos)):
            self.put(x, s, p, ks[b:b + 1], val[b:b + 1])
            self.add(x, s, q[b], p + 1)
            want, bound = attend(q[b], self.k[x, s, :p + 1], self.v[x, s, :p + 1], g[b])
            assert np.all(np.abs(got[b] - want) <= bound)
            self.checked += 1

    def observe(self, x, s):
        n = int(self.n[x, s])
        if n < 1:
            return
        end = int(self.rng.integers(1, n + 1))
        m = int(min(self.rng.integers(1, 40), end))
        q = self.rows(m, 6144)
        self.kv.attn_observe(LAYERS[x], self.ids[s], end - m, m, self.ctx.array(q))
        for u in range(m):
            self.add(x, s, q[u], end - m + u + 1, OBSERVE[self.ty])

    def evict(self, _, s):
        n = int(min(self.n[0, s], self.n[1, s]))  # a sequence's layers hold as many as each other
        if n < self.kept[s] or self.n[0, s] != self.n[1, s]:
            return
        keep = int(self.rng.integers(0, n + 1))
        recent = int(self.rng.integers(0, keep + 1))
        before = [self.sums(x, s, n) for x in range(2)]
        self.kv.evict([self.ids[s]], [n], [keep], [recent])
        for x in range(2):
            w, t = before[x]
            for j in range(4):
                at = chosen(w[:, j], t[:, j], n, keep, n + int(self.gone[s]) - recent)
                dims = slice(256 * j, 256 * j + 256)
                for a in (self.k, self.v):
                    a[x, s, :keep, dims] = a[x, s, at, dims]
                for a in (self.w, self.off, self.own):
                    a[x, s, :keep, j] = a[x, s, at, j]
            self.n[x, s] = keep
        if keep < n:
            self.gone[s] += n - keep
            self.kept[s] = keep
        assert self.kv.seq_evicted(self.ids[s]) == self.gone[s]

    def level(self, _, s):
        """Both layers as long as each other, as after a whole step."""
        x = int(self.n[0, s] > self.n[1, s])
        n, p = int(abs(self.n[0, s] - self.n[1, s])), int(self.n[:, s].min())
        if n:
            k, v = self.rows(n), self.rows(n)
            self.kv.write(LAYERS[x], self.ids[s], p, n, self.ctx.array(k), self.ctx.array(v))
            self.put(x, s, p, k, v)
        self.evict(0, s)

    def truncate(self, _, s):
        n = int(self.rng.integers(self.kept[s], self.n[:, s].max() + 1))
        self.kv.seq_truncate(self.ids[s], n)
        self.n[:, s] = np.minimum(self.n[:, s], n)
        if n == 0:
            self.gone[s] = self.kept[s] = 0

    def reset(self, _, s):
        if self.rng.random() < 0.5:
            self.kv.seq_reset(self.ids[s])
        else:
            self.kv.seq_truncate(self.ids[s], 0)
        self.n[:, s] = self.gone[s] = self.kept[s] = 0


@pytest.mark.parametrize("ty", sorted(TYPES))
@pytest.mark.parametrize("seed", range(3))
def test_random_calls(pkg, ctx, ty, seed):
    r = _Run(pkg, ctx, ty, 100 * seed + 7)
    try:
        ops = [r.write] * 4 + [r.decode] * 6 + [r.observe] * 3 + [r.level] * 4 + [r.truncate, r.reset]
        for _ in range(70):
            op = ops[int(r.rng.integers(len(ops)))]
            x, s = int(r.rng.integers(2)), int(r.rng.integers(N_SEQ))
            print(op.__name__, x, s, r.n.tolist(), r.kept.tolist(), flush=True)
            op(x, s)
            if r.rng.random() < 0.3:
                r.check(x, s)
        for x in range(2):
            for s in range(N_SEQ):
                r.check(x, s)
        assert r.checked >= 20
    finally:
        r.kv.close()
