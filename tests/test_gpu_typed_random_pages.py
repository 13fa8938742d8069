"""Random calls on typed caches whose sequences lie on pages that the caller
places (q38_seq_set_pages), some of them grown by the pool afterwards: appends,
decode steps of both forms, prompt pieces over the block images, truncations and
replacements mixed, each output against 64-bit arithmetic on a plain copy, each
held as a whole to its roundings' 2-norm too, and a refused placement changes nothing."""
import numpy as np
import pytest
from typed_prefill import PREFILL_TOL
from typed_rows import NORMAL_TOL, TYPES, attend, off_by, stored

pytestmark = pytest.mark.gpu

LAYERS = (3, 7)
LIMIT, N_SEQ, POOL = 288, 4, 60


class _Run:
    def __init__(self, pkg, ctx, ty, seed):
        self.pkg, self.ctx, self.ty, self.rng = pkg, ctx, TYPES[ty], np.random.default_rng(seed)
        self.kv = pkg.KVCache(ctx, n_slots=2, max_pages=POOL, max_seqs=N_SEQ, max_tokens_per_seq=LIMIT, ggml_type=self.ty)
        self.ids = [self.kv.seq_create() for _ in range(N_SEQ)]
        self.k = np.zeros((2, N_SEQ, LIMIT, 1024), np.float32)
        self.v = self.k.copy()
        self.length = np.zeros((2, N_SEQ), int)
        self.placed = [[] for _ in range(N_SEQ)]  # known pages
        self.w = ctx.array((1 + 0.2 * self.rng.standard_normal(256)).astype(np.float32))
        self.qg, self.q, self.g, self.kn = (ctx.empty((LIMIT, n)) for n in (12288, 6144, 6144, 1024))
        self.qg.zero()
        self.refused = self.checked = 0

    def rows(self, n, width=1024):
        return self.rng.standard_normal((n, width)).astype(np.float32)

    def put(self, x, s, p, k, v):
        n = len(k)
        self.k[x, s, p:p + n], self.v[x, s, p:p + n] = stored(k, self.ty), stored(v, self.ty)
        self.length[x, s] = max(self.length[x, s], p + n)

    def keys(self, p, key):
        self.ctx.attn_pre(len(key), p, self.w, self.w, self.qg, self.ctx.array(key), self.q, self.g, self.kn)
        return self.kn.download(len(key))

    def fits(self, s, end):
        """Whether positions below `end` have pages or find them."""
        return end <= LIMIT and (end + 15) // 16 - self.kv.seq_capacity(self.ids[s]) // 16 <= self.kv.free_pages()

    def place(self, s):
        """The sequence starts anew on pages in a random order, of the pages that no other is known to hold."""
        held = {p for o in range(N_SEQ) if o != s for p in self.placed[o]}
        free = [p for p in range(POOL) if p not in held]
        want = [int(p) for p in self.rng.permutation(free)[:self.rng.integers(1, 12)]]
        before = (self.kv.free_pages(), [self.kv.seq_capacity(i) for i in self.ids])
        try:
            self.kv.seq_set_pages(self.ids[s], want)
        except self.pkg.Q38Error as e:  # one that the pool gave to a sequence
            assert "not free" in str(e)
            assert before == (self.kv.free_pages(), [self.kv.seq_capacity(i) for i in self.ids])
            self.refused += 1
            return
        self.placed[s], self.length[:, s] = want, 0

    def truncate(self, s, n):
        self.kv.seq_truncate(self.ids[s], n)
        self.length[:, s] = np.minimum(self.length[:, s], n)
        self.placed[s] = self.placed[s][:(n + 15) // 16]

    def check(self, got, q, x, s, end, g, tol, wider=1.0):
        want, bound = attend(q, self.k[x, s, :end], self.v[x, s, :end], g)
        assert np.all(np.abs(got - want) <= bound * wider) and off_by(got, want) <= tol, (x, s, end)
        self.checked += 1

    def append(self, x):
        some = [int(s) for s in self.rng.permutation(N_SEQ)[:self.rng.integers(1, N_SEQ + 1)]]
        pos = [int(self.rng.integers(0, self.length[x, s] + 1)) for s in some]
        cnt = [int(self.rng.integers(0, 70)) for _ in some]
        cnt = [c if self.fits(s, p + c) else 0 for s, p, c in zip(some, pos, cnt)]
        need = sum(max(0, (p + c + 15) // 16 - self.kv.seq_capacity(self.ids[s]) // 16) for s, p, c in zip(some, pos, cnt) if c)
        if need > self.kv.free_pages() or not sum(cnt):
            return
        key, val = self.rows(sum(cnt)), self.rows(sum(cnt))
        self.kv.append(LAYERS[x], [self.ids[s] for s in some], pos, cnt, self.w, self.ctx.array(key), self.ctx.array(val))
        at = 0
        for s, p, n in zip(some, pos, cnt):
            if n:
                self.put(x, s, p, self.keys(p, key[at:at + n]), val[at:at + n])
            at += n

    def decode(self, x, core):
        some = [int(s) for s in self.rng.permutation(N_SEQ)[:self.rng.integers(1, N_SEQ + 1)]]
        pos = [int(self.length[x, s]) if self.rng.random() < 0.7 else int(self.rng.integers(0, self.length[x, s] + 1)) for s in some]
        keep = [i for i, (s, p) in enumerate(zip(some, pos)) if self.fits(s, p + 1)]
        some, pos = [some[i] for i in keep], [pos[i] for i in keep]
        n = len(some)
        if not n or sum(self.kv.seq_capacity(self.ids[s]) <= p for s, p in zip(some, pos)) > self.kv.free_pages():
            return
        key, val, out, ctx = self.rows(n), self.rows(n), self.ctx.empty((n, 24, 256)), self.ctx
        ids = [self.ids[s] for s in some]
        if core:
            qg = self.rows(n, 12288)
            self.kv.full_core(LAYERS[x], ids, pos, self.w, self.w, ctx.array(qg), ctx.array(key), ctx.array(val), out)
            q, g, ks = np.empty((n, 6144), np.float32), np.empty((n, 6144), np.float32), key.copy()
            for b, p in enumerate(pos):
                ctx.attn_pre(1, p, self.w, self.w, ctx.array(qg[b]), ctx.array(key[b]), self.q, self.g, self.kn)
                q[b], g[b], ks[b] = self.q.download(1), self.g.download(1), self.kn.download(1)
        else:
            q, g, ks = self.rows(n, 6144), self.rows(n, 6144), key
            self.kv.attn_decode(LAYERS[x], ids, pos, ctx.array(q), out, k_new=ctx.array(key), v_new=ctx.array(val), gate=ctx.array(g))
        got = out.download()
        for b, (s, p) in enumerate(zip(some, pos)):
            self.put(x, s, p, ks[b:b + 1], val[b:b + 1])
            self.check(got[b], q[b], x, s, p + 1, g[b], 3 * NORMAL_TOL)

    def prefill(self, x):
        s = int(self.rng.integers(N_SEQ))
        p = int(self.rng.integers(0, self.length[x, s] + 1)) if self.rng.random() < 0.4 else int(self.length[x, s])
        n = int(self.rng.integers(1, 70))
        if not self.fits(s, p + n):
            return
        q, k, v, out = self.rows(n, 6144), self.rows(n), self.rows(n), self.ctx.empty((n, 24, 256))
        given = self.rng.random() < 0.5
        if not given:
            self.kv.write(LAYERS[x], self.ids[s], p, n, self.ctx.array(k), self.ctx.array(v))
        self.kv.attn_prefill(LAYERS[x], self.ids[s], p, n, self.ctx.array(q), self.ctx.array(k) if given else None,
                             self.ctx.array(v) if given else None, out)
        self.put(x, s, p, k, v)
        got = out.download()
        for t in {0, n // 2, n - 1}:
            self.check(got[t], q[t], x, s, p + t + 1, None, 3 * PREFILL_TOL, 2.0 ** 7)

    def gather(self, x):
        some = [int(s) for s in self.rng.integers(0, N_SEQ, self.rng.integers(1, 7))]
        spans = [sorted(int(v) for v in self.rng.integers(0, self.length[x, s] + 1, 2)) for s in some]
        n = sum(b - a for a, b in spans)
        k, v = self.ctx.empty((max(n, 1), 1024)), self.ctx.empty((max(n, 1), 1024))
        self.kv.gather(LAYERS[x], [self.ids[s] for s in some], [a for a, _ in spans], [b - a for a, b in spans], k, v)
        for got, have in ((k, self.k), (v, self.v)):
            assert np.array_equal(got.download(n), np.concatenate([have[x, s, a:b] for s, (a, b) in zip(some, spans)]))
        self.checked += 1


@pytest.mark.parametrize("ty", sorted(TYPES))
@pytest.mark.parametrize("seed", range(5))
def test_random_pages(pkg, ctx, ty, seed):
    r = _Run(pkg, ctx, ty, 7000 + seed)
    try:
        for s in range(N_SEQ):
            r.place(s)
        for _ in range(90):
            x = int(r.rng.integers(2))
            op = r.rng.choice(["append", "decode", "core", "prefill", "truncate", "place", "gather"], p=[.2, .18, .17, .18, .07, .12, .08])
            if op in ("append", "prefill", "gather"):
                getattr(r, op)(x)
            elif op == "truncate":
                s = int(r.rng.integers(N_SEQ))
                r.truncate(s, int(r.rng.integers(0, r.length[:, s].max() + 1)))
            elif op == "place":
                r.place(int(r.rng.integers(N_SEQ)))
            else:
                r.decode(x, op == "core")
        for x in range(2):
            for s in range(N_SEQ):
                n = int(r.length[x, s])
                k, v = ctx.empty((max(n, 1), 1024)), ctx.empty((max(n, 1), 1024))
                r.kv.read(LAYERS[x], r.ids[s], 0, n, k, v)
                assert np.array_equal(k.download(n), r.k[x, s, :n]) and np.array_equal(v.download(n), r.v[x, s, :n])
        assert r.checked >= 30
    finally:
        r.kv.close()
