"""Random calls on typed caches of several sequences and two layers: appends,
writes, decode steps of both forms, prompt pieces, truncations, resets, gathers
and pages placed by the caller, mixed, each output against 64-bit arithmetic on
a plain copy of what the cache should hold, and the whole cache against that
copy at the end."""
import numpy as np
import pytest
from typed_rows import F32, NORMAL_TOL, TYPES, attend, off_by, stored

pytestmark = pytest.mark.gpu

LAYERS = (3, 7)


class Model:
    """The rows that each sequence holds, per layer, as the type stores them (NaN where nothing was stored yet)."""

    def __init__(self, ty, n_seq, limit):
        self.ty = ty
        self.k = np.full((2, n_seq, limit, 1024), np.nan, np.float32)
        self.v = self.k.copy()

    def put(self, layer, s, p, k, v):
        n = k.shape[0]
        self.k[layer, s, p:p + n], self.v[layer, s, p:p + n] = stored(k, self.ty), stored(v, self.ty)


def _keys(ctx, bufs, w, p, key):
    """The key rows that the framework's norm and rotation give."""
    n = key.shape[0]
    ctx.attn_pre(n, p, w, w, bufs["qg"], ctx.array(key), bufs["q"], bufs["g"], bufs["k"])
    return bufs["k"].download(n)


@pytest.mark.parametrize("ty", sorted(TYPES))
@pytest.mark.parametrize("seed", range(6))
def test_random_calls(pkg, ctx, ty, seed):
    rng = np.random.default_rng(1000 * seed + 1)
    n_seq, limit = 4, 320
    kv = pkg.KVCache(ctx, n_slots=2, max_pages=n_seq * limit // 16, max_seqs=n_seq, max_tokens_per_seq=limit,
                     ggml_type=TYPES[ty])
    m = Model(TYPES[ty], n_seq, limit)
    ids = [kv.seq_create() for _ in range(n_seq)]
    w = ctx.array((1 + 0.2 * rng.standard_normal(256)).astype(np.float32))
    bufs = {k: ctx.empty((limit, n)) for k, n in (("qg", 12288), ("q", 6144), ("g", 6144), ("k", 1024))}
    bufs["qg"].zero()
    length = [[0] * n_seq, [0] * n_seq]  # positions stored so far, per layer
    rows = lambda n: rng.standard_normal((n, 1024)).astype(np.float32)  # noqa: E731
    checked = 0
    try:
        for step in range(70):
            layer = int(rng.integers(2))
            L = LAYERS[layer]
            op = rng.choice(["append", "write", "decode", "core", "prefill", "truncate", "reset", "gather", "pages"],
                            p=[.2, .1, .2, .15, .15, .06, .03, .08, .03])
            if op == "append":
                some = [int(s) for s in rng.permutation(n_seq)[:rng.integers(1, n_seq + 1)]]
                pos = [int(rng.integers(0, length[layer][s] + 1)) for s in some]
                cnt = [int(min(rng.integers(0, 60), limit - p)) for p in pos]
                key, val = rows(max(1, sum(cnt))), rows(max(1, sum(cnt)))
                kv.append(L, [ids[s] for s in some], pos, cnt, w, ctx.array(key), ctx.array(val))
                at = 0
                for s, p, n in zip(some, pos, cnt):
                    if n:
                        m.put(layer, s, p, _keys(ctx, bufs, w, p, key[at:at + n]), val[at:at + n])
                    length[layer][s] = max(length[layer][s], p + n)
                    at += n
            elif op == "write":
                s = int(rng.integers(n_seq))
                p = int(rng.integers(0, length[layer][s] + 1))
                n = int(min(rng.integers(1, 40), limit - p))
                if n < 1:
                    continue
                k, v = rows(n), rows(n)
                kv.write(L, ids[s], p, n, ctx.array(k), ctx.array(v))
                m.put(layer, s, p, k, v)
                length[layer][s] = max(length[layer][s], p + n)
            elif op in ("decode", "core"):
                some = [int(s) for s in rng.permutation(n_seq) if length[layer][s] < limit][:int(rng.integers(1, n_seq + 1))]
                if not some:
                    continue
                # at the end, or over an earlier position
                pos = [length[layer][s] if rng.random() < 0.7 else int(rng.integers(0, length[layer][s] + 1)) for s in some]
                n = len(some)
                key, val = rows(n), rows(n)
                out = ctx.empty((n, 24, 256))
                if op == "decode":
                    q = rng.standard_normal((n, 6144)).astype(np.float32)
                    g = rng.standard_normal((n, 6144)).astype(np.float32)
                    kv.attn_decode(L, [ids[s] for s in some], pos, ctx.array(q), out, k_new=ctx.array(key),
                                   v_new=ctx.array(val), gate=ctx.array(g))
                    ks = key
                else:
                    qg = rng.standard_normal((n, 12288)).astype(np.float32)
                    kv.full_core(L, [ids[s] for s in some], pos, w, w, ctx.array(qg), ctx.array(key), ctx.array(val), out)
                    q, g, ks = np.empty((n, 6144), np.float32), np.empty((n, 6144), np.float32), np.empty_like(key)
                    for b, p in enumerate(pos):
                        ctx.attn_pre(1, p, w, w, ctx.array(qg[b]), ctx.array(key[b]), bufs["q"], bufs["g"], bufs["k"])
                        q[b], g[b], ks[b] = bufs["q"].download(1), bufs["g"].download(1), bufs["k"].download(1)
                got = out.download()
                for b, (s, p) in enumerate(zip(some, pos)):
                    m.put(layer, s, p, ks[b:b + 1], val[b:b + 1])
                    length[layer][s] = max(length[layer][s], p + 1)
                    want, bound = attend(q[b], m.k[layer, s, :p + 1], m.v[layer, s, :p + 1], g[b])
                    assert np.all(np.abs(got[b] - want) <= bound), (step, op, s, p)
                    # normed heads times weights of up to 1.6 make scores some 3 times a plain N(0, 1)'s
                    assert off_by(got[b], want) <= 3 * NORMAL_TOL
                    checked += 1
            elif op == "prefill":
                s = int(rng.integers(n_seq))
                p = int(rng.integers(0, length[layer][s] + 1)) if rng.random() < 0.4 else length[layer][s]
                n = int(min(rng.integers(1, 70), limit - p))
                if n < 1:
                    continue
                q, k, v = rng.standard_normal((n, 6144)).astype(np.float32), rows(n), rows(n)
                out = ctx.empty((n, 24, 256))
                given = rng.random() < 0.5
                if not given:
                    kv.write(L, ids[s], p, n, ctx.array(k), ctx.array(v))
                kv.attn_prefill(L, ids[s], p, n, ctx.array(q), ctx.array(k) if given else None,
                                ctx.array(v) if given else None, out)
                m.put(layer, s, p, k, v)
                length[layer][s] = max(length[layer][s], p + n)
                got = out.download()
                for t in {0, n // 2, n - 1}:
                    want, bound = attend(q[t], m.k[layer, s, :p + t + 1], m.v[layer, s, :p + t + 1])
                    assert np.all(np.abs(got[t] - want) <= bound * 2.0 ** 7), (step, op, s, p, t)
                    checked += 1
            elif op == "truncate":
                s = int(rng.integers(n_seq))
                n = int(rng.integers(0, max(length[0][s], length[1][s]) + 1))
                kv.seq_truncate(ids[s], n)
                for x in range(2):
                    length[x][s] = min(length[x][s], n)
            elif op == "reset":
                s = int(rng.integers(n_seq))
                kv.seq_reset(ids[s])
                length[0][s] = length[1][s] = 0
            elif op == "pages":
                # an empty sequence's pages placed by the caller, out of what is free
                s = int(rng.integers(n_seq))
                kv.seq_reset(ids[s])
                length[0][s] = length[1][s] = 0
                kv.seq_reserve(ids[s], int(rng.integers(1, limit + 1)))
            else:
                some = [int(s) for s in rng.integers(0, n_seq, rng.integers(1, 6))]
                spans = []
                for s in some:
                    a, b = sorted(int(v) for v in rng.integers(0, length[layer][s] + 1, 2))
                    spans.append((a, b - a))
                n = sum(c for _, c in spans)
                k, v = ctx.empty((max(n, 1), 1024)), ctx.empty((max(n, 1), 1024))
                kv.gather(L, [ids[s] for s in some], [a for a, _ in spans], [c for _, c in spans], k, v, ggml_type=F32)
                want_k = np.concatenate([m.k[layer, s, a:a + c] for s, (a, c) in zip(some, spans)])
                want_v = np.concatenate([m.v[layer, s, a:a + c] for s, (a, c) in zip(some, spans)])
                assert np.array_equal(k.download(n), want_k) and np.array_equal(v.download(n), want_v), (step, op)
                checked += 1
        for x in range(2):
            for s in range(n_seq):
                n = length[x][s]
                k, v = ctx.empty((max(n, 1), 1024)), ctx.empty((max(n, 1), 1024))
                kv.read(LAYERS[x], ids[s], 0, n, k, v)
                assert np.array_equal(k.download(n), m.k[x, s, :n]) and np.array_equal(v.download(n), m.v[x, s, :n])
        assert checked >= 20
    finally:
        kv.close()
