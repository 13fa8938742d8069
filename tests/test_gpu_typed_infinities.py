"""Stored infinities and NaN in rows that count: what they may spoil, and that
they spoil nothing else."""
import numpy as np
import pytest
from parity import decode_split
from typed_rows import TYPES

pytestmark = pytest.mark.gpu

P, AT, HEAD, DIM = 200, 70, 2, 37


def _bits(a):
    return np.ascontiguousarray(a, np.float32).view(np.uint32)


def _spoiled(ty, which):
    """[24][256]: the outputs that a bad element at dim DIM of kv head HEAD reaches."""
    s = np.zeros((24, 256), bool)
    s[6 * HEAD:6 * HEAD + 6, slice(None) if which == "key" or ty == "q8_k" else DIM] = True
    return s


@pytest.mark.parametrize("ty", sorted(TYPES))
@pytest.mark.parametrize("which", ["key", "value"])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan, 1e5])
def test_they_stay_where_they_are(pkg, ctx, ty, which, bad):
    """Two sequences, one with a bad element; 1e5 is one in an F16 cache alone."""
    rng = np.random.default_rng(3)
    K, V = (rng.standard_normal((2, P, 1024)).astype(np.float32) for _ in range(2))
    Q, G = (rng.standard_normal((2, 24, 256)).astype(np.float32) for _ in range(2))
    k, v = K.copy(), V.copy()
    (k if which == "key" else v)[0, AT, 256 * HEAD + DIM] = bad
    kv = pkg.KVCache(ctx, n_slots=1, max_pages=2 * 13, max_seqs=2, max_tokens_per_seq=208, ggml_type=TYPES[ty])
    ids = [kv.seq_create(), kv.seq_create()]
    d_q, d_g, out = ctx.array(Q), ctx.array(G), ctx.empty((2, 24, 256))
    try:
        for split in (None, 4096):
            got = []
            for keys, values in ((K, V), (k, v)):
                for b, s in enumerate(ids):
                    kv.write(3, s, 0, P, ctx.array(keys[b]), ctx.array(values[b]))
                with decode_split(ctx, split):
                    kv.attn_decode(3, ids, [P - 1] * 2, d_q, out, gate=d_g)
                got.append(out.download())
            clean, dirty = got
            other = ~_spoiled(ty, which)
            if which == "value" or not np.isfinite(bad):
                assert np.array_equal(_bits(dirty[1]), _bits(clean[1]))
                assert np.array_equal(_bits(dirty[0][other]), _bits(clean[0][other]))
            if which == "value" and ty != "q8_k" and not (np.isfinite(bad) and ty == "bf16"):
                assert not np.isfinite(dirty[0][~other]).any()
            # the new token's own row the bad one
            kv.write(3, ids[0], 0, P, ctx.array(K[0]), ctx.array(V[0]))
            key, val = K[:, P - 1].copy(), V[:, P - 1].copy()
            (key if which == "key" else val)[0, 256 * HEAD + DIM] = bad
            with decode_split(ctx, split):
                kv.attn_decode(3, ids, [P - 1] * 2, d_q, out, k_new=ctx.array(key), v_new=ctx.array(val), gate=d_g)
            dirty = out.download()
            assert np.array_equal(_bits(dirty[1]), _bits(clean[1]))
            assert np.array_equal(_bits(dirty[0][other]), _bits(clean[0][other]))
            # and calls that end before it
            kv.write(3, ids[0], 0, P, ctx.array(k[0]), ctx.array(v[0]))
            kv.attn_decode(3, ids, [AT - 1] * 2, d_q, out, gate=d_g)
            assert np.isfinite(out.download()).all()
    finally:
        kv.close()


@pytest.mark.parametrize("ty", sorted(TYPES))
@pytest.mark.parametrize("which", ["key", "value"])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_prefill(pkg, ctx, ty, which, bad):
    """In a prompt piece: a key's spoils the tokens from it on, a value's its dim; the next call over other positions nothing."""
    rng = np.random.default_rng(4)
    K, V = (rng.standard_normal((P, 1024)).astype(np.float32) for _ in range(2))
    Q = rng.standard_normal((P, 24, 256)).astype(np.float32)
    k, v = K.copy(), V.copy()
    (k if which == "key" else v)[AT, 256 * HEAD + DIM] = bad
    kv = pkg.KVCache(ctx, n_slots=1, max_pages=13, max_seqs=1, max_tokens_per_seq=208, ggml_type=TYPES[ty])
    s, d_q, out = kv.seq_create(), ctx.array(Q), ctx.empty((P, 24, 256))
    try:
        kv.attn_prefill(3, s, 0, P, d_q, ctx.array(K), ctx.array(V), out)
        clean = out.download()
        kv.attn_prefill(3, s, 0, P, d_q, ctx.array(k), ctx.array(v), out)
        dirty = out.download()
        other = ~_spoiled(ty, which)
        assert np.array_equal(_bits(dirty[:, other]), _bits(clean[:, other]))
        # the prompt again in pieces: what comes before the bad row's piece is as it was
        kv.attn_prefill(3, s, 0, AT, d_q, ctx.array(k[:AT]), ctx.array(v[:AT]), out)
        first = out.download(AT)
        kv.seq_truncate(s, 0)
        kv.attn_prefill(3, s, 0, AT, d_q, ctx.array(K[:AT]), ctx.array(V[:AT]), out)
        assert np.array_equal(_bits(first), _bits(out.download(AT)))
    finally:
        kv.close()
