"""Key rows whose f64 sum of squares lies next to a rounding border of its f32
mean, where the order of the additions decides: the append, full_core's new row
and q38_attn_pre's give the same row."""
import numpy as np
import pytest
from typed_rows import F32, TYPES, stored


def _four_squares(n):
    a = int(np.sqrt(n))
    while a >= 0:
        b = int(np.sqrt(n - a * a))
        for y in range(b, max(b - 40, -1), -1):
            r = n - a * a - y * y
            for z in range(int(np.sqrt(r)), -1, -1):
                t = int(round(np.sqrt(r - z * z)))
                if z * z + t * t == r:
                    return a, y, z, t
        a -= 1
    raise AssertionError(n)


def _scale(mean):
    mean = np.float32(mean)
    return np.float32(1.0) / np.sqrt(mean + np.float32(1e-6))


def _border_rows(n_rows):
    """Heads of one size N = 2^24 + 1 + 4i, an odd sum of four squares halfway between
    two f32 numbers, and two lumps of 2^-29 -- half of N's last place in f64 -- elsewhere:
    added to each other first they tip the mean over the border, one by one they
    are lost.  Only sizes whose scales differ are taken."""
    rows, n = [], 2 ** 24 + 1
    rng = np.random.default_rng(4)
    while len(rows) < 4 * n_rows:
        n += 4
        if _scale((n - 1) / 256) == _scale((n + 1) / 256):
            continue
        x = np.zeros(256, np.float32)
        # lanes of four dims, in rows of 16 lanes: the lumps in two other quads of the row, or other rows
        lane, other = rng.choice(64, 2, replace=False) if rng.random() < 0.3 else (8, 12)
        at = 0 if 0 not in (lane, other) else 63
        x[4 * at:4 * at + 4] = _four_squares(n)
        x[4 * lane:4 * lane + 2] = 2.0 ** -15
        x[4 * other:4 * other + 2] = 2.0 ** -15
        rows.append(x)
    return np.stack(rows).reshape(n_rows, 1024)


def test_the_rows_tell_orders_apart():
    x = _border_rows(4).reshape(16, 256).astype(np.float64)
    for r in x:
        one = 0.0
        for v in r:
            one += v * v
        both = float(np.sort(r * r).cumsum()[-1])  # the small ones first
        assert np.float32(one / 256) != np.float32(both / 256) and _scale(one / 256) != _scale(both / 256)


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32"] + sorted(TYPES))
def test_same_rows_whichever_kernel(pkg, ctx, ty):
    n = 24
    ident = F32 if ty == "f32" else TYPES[ty]
    key = _border_rows(n)
    val = np.random.default_rng(5).standard_normal((n, 1024)).astype(np.float32)
    w = ctx.array(np.ones(256, np.float32))
    d_k, d_v = ctx.array(key), ctx.array(val)
    qg, q, g, k = (ctx.empty((n, m)) for m in (12288, 6144, 6144, 1024))
    qg.zero()
    kv = pkg.KVCache(ctx, n_slots=1, max_pages=16, max_seqs=2, max_tokens_per_seq=64, ggml_type=ident)
    got_k, got_v = ctx.empty((n, 1024)), ctx.empty((n, 1024))
    try:
        a, b = kv.seq_create(), kv.seq_create()
        for pos in (0, 5):
            ctx.attn_pre(n, pos, w, w, qg, d_k, q, g, k)
            want = stored(k.download(), ident)
            kv.append(3, [a], [pos], [n], w, d_k, d_v)
            kv.read(3, a, pos, n, got_k, got_v)
            assert np.array_equal(got_k.download(), want)
            if ty == "f32":  # its full_core sums a head by half-waves
                continue
            out = ctx.empty((1, 24, 256))
            kv.write(3, b, 0, n, d_v, d_v)
            for t in range(n):
                kv.full_core(3, [b], [pos + t], w, w, qg, d_k.offset(1024 * t), d_v.offset(1024 * t), out)
            kv.read(3, b, pos, n, got_k, got_v)
            assert np.array_equal(got_k.download(), want)
    finally:
        kv.close()
