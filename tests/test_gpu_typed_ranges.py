"""One token's attention over 16- and 8-bit rows whose values differ by many
orders (tests/typed_ranges.py has the inputs and the limits)."""
import numpy as np
import pytest
from parity import decode_split
from typed_ranges import CASES, IDENT, IDS, attend_by_weight, case, check, heads_of
from typed_rows import attend, stored

pytestmark = pytest.mark.gpu


def _cache(pkg, ctx, ty, rows, seqs=1):
    P = rows[0][0].shape[0]
    kv = pkg.KVCache(ctx, n_slots=1, max_pages=seqs * ((P + 15) // 16), max_seqs=seqs, max_tokens_per_seq=P, ggml_type=IDENT[ty])
    ids = [kv.seq_create() for _ in range(seqs)]
    for s, (K, V) in zip(ids, rows):
        kv.write(3, s, 0, P, ctx.array(K), ctx.array(V))
    return kv, ids


@pytest.mark.parametrize("ty,name,args", CASES, ids=IDS)
def test_values_of_many_sizes(pkg, ctx, ty, name, args):
    """Whole contexts in one split (eight chains of pages) and in the automatic one."""
    Q, K, V, k, v, tol = case(ty, name, args)
    want, bound = attend_by_weight(Q, k, v, IDENT[ty])
    kv, ids = _cache(pkg, ctx, ty, [(K, V)])
    out = ctx.empty((24, 256))
    try:
        for split in (4096, None):
            with decode_split(ctx, split):
                kv.attn_decode(3, ids, [K.shape[0] - 1], ctx.array(Q), out)
            check(out.download(), want, bound, tol, heads_of(name))
    finally:
        kv.close()


@pytest.mark.parametrize("ty", sorted(IDENT))
def test_a_batch_of_them(pkg, ctx, ty):
    """Several sequences in one call, and the new token's own row the large one."""
    some = [c for c in CASES if c[0] == ty and c[1] in ("no_weight", "little_weight")][:3]
    made = [case(*c) for c in some]
    P = made[0][1].shape[0]
    kv, ids = _cache(pkg, ctx, ty, [(m[1], m[2]) for m in made], len(made))
    n = len(made)
    out = ctx.empty((n, 24, 256))
    try:
        kv.attn_decode(3, ids, [P - 1] * n, ctx.array(np.stack([m[0] for m in made])), out)
        got = out.download()
        for m, g in zip(made, got):
            check(g, *attend_by_weight(m[0], m[3], m[4], IDENT[ty]), m[5])
        # token P - 1 given again, large and without weight
        key, val = (np.stack([m[i][P - 1] for m in made]) for i in (1, 2))
        key[:, ::256] = -300.0
        val = (val * np.float32(1e3 if ty == "f16" else 1e9)).astype(np.float32)
        kv.attn_decode(3, ids, [P - 1] * n, ctx.array(np.stack([m[0] for m in made])), out, k_new=ctx.array(key),
                       v_new=ctx.array(val))
        got = out.download()
        for b, (m, g) in enumerate(zip(made, got)):
            k, v = m[3].copy(), m[4].copy()
            k[P - 1], v[P - 1] = stored(key[b:b + 1], IDENT[ty])[0], stored(val[b:b + 1], IDENT[ty])[0]
            check(g, *attend_by_weight(m[0], k, v, IDENT[ty]), m[5])
    finally:
        kv.close()


def test_values_near_the_ends_of_f32(pkg, ctx):
    """8-bit rows of 1e-34 and of 1e37 values, alone and mixed."""
    P = 300
    for seed, sizes in enumerate(([1e-34], [1e37], [1e-34, 1e37], [1e37, 1e-30, 1.0])):
        rng = np.random.default_rng(seed)
        Q = rng.standard_normal((24, 256)).astype(np.float32)
        K, V = rng.standard_normal((P, 1024)).astype(np.float32), rng.uniform(-1, 1, (P, 1024)).astype(np.float32)
        V *= np.resize(np.array(sizes, np.float32), P)[:, None]
        kv, ids = _cache(pkg, ctx, "q8_k", [(K, V)])
        out = ctx.empty((24, 256))
        try:
            for split in (4096, None):
                with decode_split(ctx, split):
                    kv.attn_decode(3, ids, [P - 1], ctx.array(Q), out)
                k, v = stored(K, IDENT["q8_k"]), stored(V, IDENT["q8_k"])
                want, bound = attend_by_weight(Q, k, v, IDENT["q8_k"])
                off = np.abs(out.download().astype(np.float64) - want)
                assert np.all(off <= bound), (sizes, float((off / bound).max()))
                assert np.all(off <= attend(Q, k, v)[1])
        finally:
            kv.close()
