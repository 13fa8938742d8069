"""Prompt pieces and full_core over typed caches, each token's output held as a
whole to what the arithmetic's roundings add up to for N(0, 1) inputs, besides
the bound of every value (tests/typed_prefill.py; tests/test_typed_prefill.py plants
mistakes in the same assertions)."""
from types import SimpleNamespace

import numpy as np
import pytest
from typed_prefill import PREFILL_TOL
from typed_rows import NORMAL_TOL, TYPES, attend, off_by, stored

# normed heads times weights of up to 1.6 make scores some 3 times a plain N(0, 1)'s
CORE_TOL = 3 * NORMAL_TOL


def piece(base, n, ident):
    """A piece of n tokens after `base` others, with one row more than it covers."""
    rng = np.random.default_rng(1000 * base + n)
    K, V = (rng.standard_normal((base + n + 1, 1024)).astype(np.float32) for _ in range(2))
    q, g = (rng.standard_normal((n, 24, 256)).astype(np.float32) for _ in range(2))
    return SimpleNamespace(base=base, n=n, q=q, g=g, K=K, V=V, k=stored(K, ident), v=stored(V, ident))


def check_prefill(got, x, t):
    """Token t of the piece: each value off by 2^7 of what 32-bit products allow at most, all of them by PREFILL_TOL."""
    end = x.base + t + 1
    want, bound = attend(x.q[t], x.k[:end], x.v[:end], x.g[t])
    off = np.abs(got.astype(np.float64) - want)
    print(f"[bound] {float((off / bound).max()) / 2 ** 7:.4f} of the bound, 2-norm {off_by(got, want):.2e}", flush=True)
    assert np.all(np.isfinite(got)) and np.all(off <= bound * 2.0 ** 7) and off_by(got, want) <= PREFILL_TOL


def check_core(got, want, bound):
    off = np.abs(got.astype(np.float64) - want)
    print(f"[bound] {float((off / bound).max()):.4f} of the bound, 2-norm {off_by(got, want):.2e}", flush=True)
    assert np.all(np.isfinite(got)) and np.all(off <= bound) and off_by(got, want) <= CORE_TOL


def core_inputs(ref, P, ident):
    """A query as full_core forms it, and P rows of which the last is a formed key."""
    rng = np.random.default_rng(P)
    wq, wk = ((1 + 0.2 * rng.standard_normal(256)).astype(np.float32) for _ in range(2))
    q = np.concatenate([ref.rmsnorm(r, wq) for r in rng.standard_normal((24, 256)).astype(np.float32)])
    q = ref.rope(q.astype(np.float32), 24, P - 1).reshape(24, 256)
    k, v = (rng.standard_normal((P, 1024)).astype(np.float32) for _ in range(2))
    last = np.concatenate([ref.rmsnorm(r, wk) for r in k[P - 1].reshape(4, 256)])
    k[P - 1] = ref.rope(last.astype(np.float32), 4, P - 1).reshape(1024)
    return q.astype(np.float32), stored(k, ident), stored(v, ident), rng.standard_normal((24, 256)).astype(np.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("ty", sorted(TYPES))
@pytest.mark.parametrize("base,n", [(0, 1), (0, 33), (0, 200), (5, 40), (33, 7), (300, 65), (999, 130)])
def test_prefill(pkg, ctx, ty, base, n):
    x = piece(base, n, TYPES[ty])
    total = base + n
    kv = pkg.KVCache(ctx, n_slots=1, max_pages=(total + 15) // 16, max_seqs=1, max_tokens_per_seq=total, ggml_type=TYPES[ty])
    s, out = kv.seq_create(), ctx.empty((n, 24, 256))
    try:
        if base:
            kv.write(3, s, 0, base, ctx.array(x.K[:base]), ctx.array(x.V[:base]))
        kv.attn_prefill(3, s, base, n, ctx.array(x.q), ctx.array(x.K[base:total]), ctx.array(x.V[base:total]), out,
                        gate=ctx.array(x.g))
        got = out.download()
        for t in sorted({0, 1, 15, 16, 31, 32, n // 3, n // 2, n - 2, n - 1} & set(range(n))):
            check_prefill(got[t], x, t)
    finally:
        kv.close()


@pytest.mark.gpu
@pytest.mark.parametrize("ty", sorted(TYPES))
def test_full_core(pkg, ctx, ty):
    """At the first position, within a page, at a page's ends and far on, one call for all and one each."""
    lengths = [1, 2, 16, 17, 40, 1500]
    rng = np.random.default_rng(8)
    n = len(lengths)
    kv = pkg.KVCache(ctx, n_slots=1, max_pages=110, max_seqs=n, max_tokens_per_seq=1504, ggml_type=TYPES[ty])
    ids = [kv.seq_create() for _ in lengths]
    for s, m in zip(ids, lengths):
        K, V = (rng.standard_normal((m, 1024)).astype(np.float32) for _ in range(2))
        kv.write(3, s, 0, m, ctx.array(K), ctx.array(V))
    wq, wk = (ctx.array((1 + 0.2 * rng.standard_normal(256)).astype(np.float32)) for _ in range(2))
    qg, key, val = (ctx.array(rng.standard_normal((n, m)).astype(np.float32)) for m in (12288, 1024, 1024))
    out, q, g, k = ctx.empty((n, 24, 256)), ctx.empty((1, 6144)), ctx.empty((1, 6144)), ctx.empty((1, 1024))
    pos = [m - 1 for m in lengths]
    try:
        kv.full_core(3, ids, pos, wq, wk, qg, key, val, out)
        got = out.download()
        for b, (s, m) in enumerate(zip(ids, lengths)):
            rows = ctx.empty((m, 1024)), ctx.empty((m, 1024))
            kv.read(3, s, 0, m, *rows)
            ctx.attn_pre(1, m - 1, wq, wk, qg.offset(b * 12288), key.offset(b * 1024), q, g, k)
            want, bound = attend(q.download(1), rows[0].download(), rows[1].download(), g.download(1))
            check_core(got[b], want, bound)
            kv.full_core(3, [s], [m - 1], wq, wk, qg.offset(b * 12288), key.offset(b * 1024), val.offset(b * 1024), out)
            check_core(out.download(1)[0], want, bound)
    finally:
        kv.close()
