"""KV caches of 4-bit (MXFP4) rows: every check of the typed caches
(test_gpu_kv_types.py), with the rows as 4-bit blocks stand for them, and what is
particular to those."""
import importlib.util
import os

import numpy as np
import pytest
import typed_rows
from mxfp4_rows import MXFP4, stored4
from typed_rows import attend, rms64, rope64

pytestmark = pytest.mark.gpu


def _typed_checks():
    """The typed caches' checks with one type more."""
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "test_gpu_kv_types.py")
    spec = importlib.util.spec_from_file_location("kv_checks_mxfp4", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.TYPES = {"mxfp4": MXFP4}
    m.stored = lambda x, ty: stored4(x) if ty == MXFP4 else typed_rows.stored(x, ty)
    return m


K = _typed_checks()
TY = "mxfp4"


@pytest.mark.parametrize("pos0,n", [(0, 1), (0, 16), (5, 1), (15, 2), (3, 13), (16, 16), (7, 50), (31, 1), (0, 163), (33, 95)])
def test_write_and_read(pkg, ctx, pos0, n):
    K.test_write_and_read(pkg, ctx, TY, pos0, n)


def test_rows_of_every_size(pkg, ctx):
    """Zeros of either sign, ties, the ends of the scale's range, subnormal values, sizes a hair on either side of 7 units."""
    rng = np.random.default_rng(5)
    x = K._rows(rng, 48)
    x[0] = 0.0
    x[1, :256] = -0.0
    x[2] *= 1e-30
    x[3] *= 1e30
    x[4, :] = 2.0 * np.sign(x[4])
    x[5, :32] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 6.5] * 2
    x[6, :32] = x[5, :32]
    x[6, 7] = np.nextafter(np.float32(7), np.float32(8))
    x[7] = np.finfo(np.float32).max * np.sign(x[7])
    x[8] *= np.float32(2.0 ** -126)
    x[9] = np.float32(2.0 ** -126) * rng.integers(0, 9, 1024)
    x[10] = np.float32(2.0 ** -149) * rng.integers(-2 ** 23, 2 ** 23, 1024)  # subnormal
    x[11] *= (2.0 ** rng.integers(-126, 126, 1024).astype(np.float64)).astype(np.float32)
    for r in range(12, 48):  # halfway cases at every scale
        x[r] = (rng.choice([-1, 1], 1024) * rng.integers(0, 33, 1024) * 0.25 * 2.0 ** (7 * (r - 30))).astype(np.float32)
    v = x[::-1].copy()
    with K.Cache(pkg, ctx, TY, [48]) as c:
        c.kv.write(3, c.seqs[0], 0, 48, ctx.array(x), ctx.array(v))
        k, got_v = c.read(c.seqs[0], 0, 48)
        for got, src in ((k, x), (got_v, v)):
            want = stored4(src)
            bad = np.argwhere(got != want)
            assert bad.size == 0, (bad[:5], got[tuple(bad[0])], want[tuple(bad[0])], src[tuple(bad[0])])
        # as the call of one token stores them
        for t in range(48):
            c.kv.attn_decode(3, [c.seqs[0]], [t], ctx.array(np.zeros(6144, np.float32)), ctx.empty((6144,)),
                             k_new=ctx.array(v[t]), v_new=ctx.array(x[t]))
        k, got_v = c.read(c.seqs[0], 0, 48)
        assert np.array_equal(k, stored4(v)) and np.array_equal(got_v, stored4(x))


@pytest.mark.parametrize("n_seq", [1, 5, 67])
def test_append_equals_pre_then_write(pkg, ctx, n_seq):
    K.test_append_equals_pre_then_write(pkg, ctx, TY, n_seq)


def test_infinities_spoil_their_block_alone(pkg, ctx):
    """A block with an infinity or NaN reads back NaN or infinite, those beside it as they were stored."""
    rng = np.random.default_rng(3)
    x = K._rows(rng, 16)
    spoilt = np.zeros((16, 1024), bool)
    for t, bad in enumerate((np.inf, -np.inf, np.nan)):
        x[t, 100 * t + 5] = bad
        spoilt[t, (100 * t + 5) // 32 * 32:][:32] = True
    with K.Cache(pkg, ctx, TY, [16]) as c:
        c.kv.write(3, c.seqs[0], 0, 16, ctx.array(x), ctx.array(x[::-1].copy()))
        k, v = c.read(c.seqs[0], 0, 16)
        for got, src, bad in ((k, x, spoilt), (v, x[::-1], spoilt[::-1])):
            assert not np.isfinite(got[bad]).any()
            assert np.array_equal(got[~bad], stored4(src)[~bad])


def test_far_positions(pkg, ctx):
    """Rows past 2^16 positions, in a pool whose offsets pass 2^32 bytes."""
    n_pages, limit = 500000, 16 * 80000
    kv = pkg.KVCache(ctx, n_slots=2, max_pages=n_pages, max_seqs=1, max_tokens_per_seq=limit, ggml_type=MXFP4)
    try:
        s = kv.seq_create()
        kv.seq_set_pages(s, list(range(0, 66000)) + [n_pages - 1, n_pages - 2, n_pages - 3])
        rng = np.random.default_rng(2)
        pos = 16 * 66000 + 5
        key, val = K._rows(rng, 30), K._rows(rng, 30)
        w = np.ones(256, np.float32)
        kv.append(7, [s], [pos], [30], ctx.array(w), ctx.array(key), ctx.array(val))
        k, v = ctx.empty((30, 1024)), ctx.empty((30, 1024))
        kv.read(7, s, pos, 30, k, v)
        assert np.array_equal(v.download(), stored4(val))
        want = rope64(rms64(key.reshape(30, 4, 256), w), np.arange(pos, pos + 30)).reshape(-1, 32)
        # a value is off by half a step at most: 1 of the scale's units, of which the largest has 3.5 or more
        assert np.all(np.abs(k.download().reshape(-1, 32) - want) <= np.abs(want).max(1, keepdims=True) / 3.5 * 1.01)
        q = (8 * rng.standard_normal((24, 256))).astype(np.float32)
        d_o = ctx.empty((24, 256))
        kv.attn_decode(7, [s], [pos + 29], ctx.array(q), d_o)
        got, k, v = d_o.download(), k.download().astype(np.float64), v.download().astype(np.float64)
        for h in range(24):
            kk, vv = (x[:, 256 * (h // 6):256 * (h // 6) + 256] for x in (k, v))
            sc = kk @ q[h] / 16
            top = max(sc.max(), 0.0)
            p = np.exp(sc - top) / (np.exp(sc - top).sum() + pos * np.exp(-top))
            # the bound of the typed caches' check of far positions
            big = (np.abs(kk) @ np.abs(q[h])).max() / 16
            e = 2 * (264 * big + 4 + np.abs(sc).max()) * 2.0 ** -24 + 256 * 2.0 ** -24 + 2.0 ** -21
            bound = 1.01 * e * (p @ np.abs(vv)) + 30 * 2.0 ** -31 * np.abs(vv).max()
            assert np.all(np.abs(got[h] - p @ vv) <= bound), h
    finally:
        kv.close()


@pytest.mark.parametrize("P", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 200, 400, 600, 1000])
def test_decode_lengths(pkg, ctx, P):
    K.test_decode_lengths(pkg, ctx, TY, P)


@pytest.mark.parametrize("split", [16, 32, 48, 80, 512, 1024, 4096])
def test_decode_splits(pkg, ctx, split):
    K.test_decode_splits(pkg, ctx, TY, split)


@pytest.mark.parametrize("size", [2.0 ** 90, 2.0 ** 104, 2.0 ** 112])
def test_decode_queries_near_the_end_of_f32(pkg, ctx, size):
    K.test_decode_queries_near_the_end_of_f32(pkg, ctx, TY, size)


@pytest.mark.parametrize("case", ["rising", "falling", "peaked", "large", "tiny", "flat", "huge_q", "huge_v", "mixed_heads"])
def test_decode_score_ranges(pkg, ctx, case):
    K.test_decode_score_ranges(pkg, ctx, TY, case)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_rows_past_the_end_do_not_count(pkg, ctx, bad):
    K.test_rows_past_the_end_do_not_count(pkg, ctx, TY, bad)


def test_nan_in_one_head_stays_there(pkg, ctx):
    K.test_nan_in_one_head_stays_there(pkg, ctx)


def test_decode_batch(pkg, ctx):
    K.test_decode_batch(pkg, ctx, TY)


def test_full_core(pkg, ctx):
    K.test_full_core(pkg, ctx, TY)


@pytest.mark.parametrize("n_seq", [1, 3])
def test_decode_graph(pkg, ctx, n_seq):
    K.test_decode_graph(pkg, ctx, TY, n_seq)


@pytest.mark.parametrize("base,n", [(0, 1), (0, 33), (0, 200), (5, 40), (33, 7), (300, 65)])
def test_prefill(pkg, ctx, base, n):
    K.test_prefill(pkg, ctx, TY, base, n)


def test_prefill_after_decode_and_truncate(pkg, ctx):
    K.test_prefill_after_decode_and_truncate(pkg, ctx, TY)


def test_gather_comes_as_f32_alone(pkg, ctx):
    with K.Cache(pkg, ctx, TY, [16]) as c:
        o = ctx.empty((2, 1024))
        with pytest.raises(pkg.Q38Error, match="not as type 39"):
            c.kv.gather(3, c.seqs, [0], [2], o, o, ggml_type=MXFP4)


def test_values_of_many_sizes_in_a_row(pkg, ctx):
    """Blocks of one row whose scales differ by many orders: each dim keeps its own."""
    P = 333
    rng = np.random.default_rng(12)
    k, v = K._rows(rng, P), K._rows(rng, P)
    size = np.repeat(2.0 ** rng.integers(-20, 20, (P, 32)), 32, 1)
    q = rng.standard_normal((24, 256)).astype(np.float32)
    v = (v * size).astype(np.float32)
    with K.Cache(pkg, ctx, TY, [P]) as c:
        for split in (None, 4096):
            got = K._decode(ctx, c, k, v, q, None, P, split=split).reshape(24, 256).astype(np.float64)
            want, bound = attend(q, stored4(k), stored4(v))
            # attend()'s last term takes the largest value of a row's; of the weights' bf16 parts none is lost
            assert np.all(np.abs(got - want) <= bound)
            vv = stored4(v).astype(np.float64)
            for h in range(24):
                kk = stored4(k)[:, 256 * (h // 6):256 * (h // 6) + 256].astype(np.float64)
                s = kk @ q[h].astype(np.float64) / 16
                p = np.exp(s - s.max())
                p /= p.sum()
                big = (np.abs(kk) @ np.abs(q[h])).max() / 16
                e = 2.0 * ((264 * big + 4 + np.abs(s).max()) * 2.0 ** -24) + (P + 16) * 2.0 ** -24 + 2.0 ** -21
                each = e * (p @ np.abs(vv[:, 256 * (h // 6):256 * (h // 6) + 256])) * 1.01
                assert np.all(np.abs(got[h] - want[h]) <= each)
