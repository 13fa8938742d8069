"""KV caches of F16, BF16 and Q8_K rows: the rows in and out of their pages,
and every call that reads them, against plain 64-bit arithmetic on the values
that the stored rows stand for (tests/typed_rows.py has the references and the
derivation of the bounds)."""
import ctypes
import os

import numpy as np
import pytest
from parity import decode_split
from typed_rows import F32, NORMAL_TOL, Q8_K, TYPES, attend, off_by, rms64, rope64, stored

pytestmark = pytest.mark.gpu

typed = pytest.mark.parametrize("ty", sorted(TYPES))
all_types = pytest.mark.parametrize("ty", ["f32"] + sorted(TYPES))


def _id(ty):
    return F32 if ty == "f32" else TYPES[ty]


class Cache:
    """A cache with a randomly permuted page table, and the rows it should hold."""

    def __init__(self, pkg, ctx, ty, lengths, seed=1, spare=4, slots=1, limit=None):
        self.ctx, self.ty = ctx, _id(ty)
        pages = [(n + 15) // 16 + spare for n in lengths]
        self.kv = pkg.KVCache(ctx, n_slots=slots, max_pages=sum(pages) + 3, max_seqs=len(lengths),
                              max_tokens_per_seq=limit or 16 * max(pages), ggml_type=self.ty)
        order = np.random.default_rng(seed).permutation(sum(pages))
        self.seqs, at = [], 0
        for n in pages:
            s = self.kv.seq_create()
            self.kv.seq_set_pages(s, order[at:at + n].tolist())
            self.seqs.append(s)
            at += n

    def read(self, seq, pos0, n, layer=3):
        k, v = self.ctx.empty((max(n, 1), 1024)), self.ctx.empty((max(n, 1), 1024))
        self.kv.read(layer, seq, pos0, n, k, v)
        out = k.download(n), v.download(n)
        k.free(), v.free()
        return out

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.kv.close()


def _rows(rng, n, sigma=1.0):
    return (sigma * rng.standard_normal((n, 1024))).astype(np.float32)


def _bits(a):
    return np.ascontiguousarray(a, np.float32).view(np.uint32)


# ------------------------------------------------------------------ rows


@typed
@pytest.mark.parametrize("pos0,n", [(0, 1), (0, 16), (5, 1), (15, 2), (3, 13), (16, 16), (7, 50), (31, 1), (0, 163), (33, 95)])
def test_write_and_read(pkg, ctx, ty, pos0, n):
    """Every row comes back as its type rounds it, and the rows around it stay as they were."""
    rng = np.random.default_rng(100 * pos0 + n)
    old, new = _rows(rng, 176), _rows(rng, n, 3.0)
    old_v, new_v = _rows(rng, 176), _rows(rng, n, 0.1)
    with Cache(pkg, ctx, ty, [176]) as c:
        c.kv.write(3, c.seqs[0], 0, 176, ctx.array(old), ctx.array(old_v))
        c.kv.write(3, c.seqs[0], pos0, n, ctx.array(new), ctx.array(new_v))
        k, v = c.read(c.seqs[0], 0, 176)
        for got, a, b in ((k, old, new), (v, old_v, new_v)):
            want = stored(a, c.ty)
            want[pos0:pos0 + n] = stored(b, c.ty)
            assert np.array_equal(_bits(got), _bits(want))


@typed
def test_rows_of_every_size(pkg, ctx, ref, ty):
    """Zero rows, tiny and large values, ties of the largest size with either
    sign first, values at and past the ends of the type's range; the 8-bit
    rows as the engine's quantiser rounds them."""
    rng = np.random.default_rng(5)
    x = _rows(rng, 32)
    x[0] = 0.0
    x[1, :256] = 0.0
    x[2] *= 1e-30
    x[3] *= 1e30 if ty != "f16" else 1e4
    x[4, :] = 2.0 * np.sign(x[4])            # all of one size
    x[5, 10], x[5, 20] = 9.0, -9.0
    x[6, 300], x[6, 290] = 9.0, -9.0
    x[7, :256] = np.linspace(-1, 1, 256, dtype=np.float32)
    x[8] = np.float32(1.0) + np.arange(1024, dtype=np.float32) * np.float32(2.0 ** -9)  # halfway cases in 16 bits
    if ty == "f16":
        x[9, :4] = [65504.0, 65519.0, 65520.0, -1e6]
        x[10] *= 1e-7                        # subnormal halves
    if ty == "q8_k":
        x[11, :512] *= 1e-38                 # no finite inverse scale
    v = x[::-1].copy()
    with Cache(pkg, ctx, ty, [32]) as c:
        c.kv.write(3, c.seqs[0], 0, 32, ctx.array(x), ctx.array(v))
        k, got_v = c.read(c.seqs[0], 0, 32)
        zero = np.abs(x) < 3e-37 if ty == "q8_k" else np.zeros(x.shape, bool)  # zeros of either sign there
        assert np.array_equal(np.where(zero, 0, _bits(k)), np.where(zero, 0, _bits(stored(x, c.ty))))
        zero = zero[::-1]
        assert np.array_equal(np.where(zero, 0, _bits(got_v)), np.where(zero, 0, _bits(stored(v, c.ty))))
        assert not k[np.abs(x) < 3e-37].any() or ty != "q8_k"
        if ty == "q8_k":
            q, _, s = ref.q8k_split(ref.quantize_q8_k(x), 32, 1024)
            want = (q.reshape(32, 4, 256) * s[:, :, None]).astype(np.float32).reshape(32, 1024)
            assert np.array_equal(k, want)


@all_types
@pytest.mark.parametrize("n_seq", [1, 5, 67])
def test_append_equals_pre_then_write(pkg, ctx, ty, n_seq):
    """A ragged batch (pieces of 0 to 90 tokens at any position, more
    sequences than one launch takes) against q38_attn_pre's key rows stored
    with q38_kv_write, bit for bit, with the rows around them untouched; and
    the keys against the formula in 64 bits."""
    rng = np.random.default_rng(n_seq)
    pos = rng.integers(0, 400, n_seq)
    cnt = np.where(rng.random(n_seq) < 0.2, 0, rng.integers(1, 91, n_seq))
    cnt[-1] = 37
    total = int(cnt.sum())
    key, val = _rows(rng, total), _rows(rng, total)
    w = (1 + 0.2 * rng.standard_normal(256)).astype(np.float32)
    d_w, d_k, d_v = ctx.array(w), ctx.array(key), ctx.array(val)
    qg, q_out, gate_out, k_out = (ctx.empty((max(1, total), n)) for n in (12288, 6144, 6144, 1024))
    qg.zero()
    lengths = [512] * n_seq
    fill = _rows(rng, 512)
    d_fill = ctx.array(fill)
    with Cache(pkg, ctx, ty, lengths, seed=3) as c, Cache(pkg, ctx, ty, lengths, seed=4) as e:
        for x in (c, e):
            for s in x.seqs:
                x.kv.write(3, s, 0, 512, d_fill, d_fill)
        order = rng.permutation(n_seq)
        c.kv.append(3, [c.seqs[i] for i in order], pos[order].tolist(), cnt[order].tolist(), d_w, d_k, d_v)
        at = 0
        for i in order:
            n, p = int(cnt[i]), int(pos[i])
            if n:
                ctx.attn_pre(n, p, d_w, d_w, qg, d_k.offset(at * 1024), q_out, gate_out, k_out)
                e.kv.write(3, e.seqs[i], p, n, k_out, d_v.offset(at * 1024))
                got = k_out.download(n).reshape(n, 4, 256)
                want = rope64(rms64(key[at:at + n].reshape(n, 4, 256), w), np.arange(p, p + n))
                # norm: 4 roundings; each turned value a sum of two products of rounded factors
                size = np.abs(rms64(key[at:at + n].reshape(n, 4, 256), w)).max()
                assert np.abs(got - want).max() <= 12 * 2.0 ** -24 * size
            a, b = c.read(c.seqs[i], 0, 512), e.read(e.seqs[i], 0, 512)
            assert np.array_equal(_bits(a[0]), _bits(b[0])) and np.array_equal(_bits(a[1]), _bits(b[1]))
            at += n
        # the same rows gathered, in another order and more than once
        some = [int(i) for i in order[:3]] * 2
        n_rows = int(sum(cnt[i] for i in some))
        g_k, g_v = ctx.empty((n_rows + 1, 1024)), ctx.empty((n_rows + 1, 1024))
        mark = np.full((n_rows + 1, 1024), 7.5, np.float32)
        g_k.upload(mark), g_v.upload(mark)
        c.kv.gather(3, [c.seqs[i] for i in some], [int(pos[i]) for i in some], [int(cnt[i]) for i in some], g_k, g_v)
        got_k, got_v = g_k.download(), g_v.download()
        at = 0
        for i in some:
            n = int(cnt[i])
            k, v = c.read(c.seqs[i], int(pos[i]), n)
            assert np.array_equal(_bits(got_k[at:at + n]), _bits(k)) and np.array_equal(_bits(got_v[at:at + n]), _bits(v))
            at += n
        assert np.all(got_k[n_rows:] == 7.5) and np.all(got_v[n_rows:] == 7.5)


@pytest.mark.parametrize("ty,dtype", [("f16", np.float16), ("bf16", np.uint16)])
def test_gather_as_stored(pkg, ctx, ty, dtype):
    rng = np.random.default_rng(8)
    x, v = _rows(rng, 100), _rows(rng, 100)
    with Cache(pkg, ctx, ty, [100, 100]) as c:
        for s in c.seqs:
            c.kv.write(3, s, 0, 100, ctx.array(x), ctx.array(v))
        k16, v16 = ctx.empty((62, 1024), np.uint16), ctx.empty((62, 1024), np.uint16)
        k16.zero(), v16.zero()
        c.kv.gather(3, c.seqs, [3, 90], [51, 10], k16, v16, ggml_type=c.ty)
        for got, src in ((k16.download(), x), (v16.download(), v)):
            rows = np.concatenate((src[3:54], src[90:100]))
            have = got[:61].view(np.float16).astype(np.float32) if dtype == np.float16 else \
                (got[:61].astype(np.uint32) << 16).view(np.float32)
            assert np.array_equal(have, stored(rows, c.ty)) and not got[61:].any()


@typed
def test_far_positions(pkg, ctx, ty):
    """Rows past 2^16 positions, in a pool whose offsets pass 2^32 bytes."""
    n_pages = {"f16": 140000, "bf16": 140000, "q8_k": 260000}[ty]
    limit = 16 * 80000
    kv = pkg.KVCache(ctx, n_slots=2, max_pages=n_pages, max_seqs=1, max_tokens_per_seq=limit, ggml_type=_id(ty))
    try:
        s = kv.seq_create()
        # the sequence's last pages are the pool's last ones
        kv.seq_set_pages(s, list(range(0, 66000)) + [n_pages - 1, n_pages - 2, n_pages - 3])
        rng = np.random.default_rng(2)
        pos = 16 * 66000 + 5
        key, val = _rows(rng, 30), _rows(rng, 30)
        w = np.ones(256, np.float32)
        kv.append(7, [s], [pos], [30], ctx.array(w), ctx.array(key), ctx.array(val))
        k, v = ctx.empty((30, 1024)), ctx.empty((30, 1024))
        kv.read(7, s, pos, 30, k, v)
        assert np.array_equal(_bits(v.download()), _bits(stored(val, _id(ty))))
        want = rope64(rms64(key.reshape(30, 4, 256), w), np.arange(pos, pos + 30)).reshape(30, 1024)
        step = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "q8_k": 0.5 / 127}[ty] * 1.01
        size = np.abs(want).max() if ty == "q8_k" else np.abs(want)
        assert np.all(np.abs(k.download() - want) <= step * size + 1e-5)
        # one token's attention over all of them: the positions before are zero
        # rows, whose weight is exp(0) each
        q = (8 * rng.standard_normal((24, 256))).astype(np.float32)
        d_o = ctx.empty((24, 256))
        kv.attn_decode(7, [s], [pos + 29], ctx.array(q), d_o)
        got, k, v = d_o.download(), k.download().astype(np.float64), v.download().astype(np.float64)
        for h in range(24):
            kk, vv = (x[:, 256 * (h // 6):256 * (h // 6) + 256] for x in (k, v))
            sc = kk @ q[h] / 16
            top = max(sc.max(), 0.0)
            p = np.exp(sc - top) / (np.exp(sc - top).sum() + pos * np.exp(-top))
            want = p @ vv
            # typed_rows.attend's bound; a sum's longest chain is no n terms: a
            # lane adds 4 weights a page, 128 at most of a split's 4096 / 8 tokens,
            # the joins of lanes, waves and splits add fewer than 100
            big = (np.abs(kk) @ np.abs(q[h])).max() / 16
            e = 2 * (264 * big + 4 + np.abs(sc).max()) * 2.0 ** -24 + 256 * 2.0 ** -24 + 2.0 ** -21
            bound = 1.01 * e * (p @ np.abs(vv)) + 30 * 2.0 ** -31 * np.abs(vv).max()
            assert np.all(np.abs(got[h] - want) <= bound), h
        kv.read(3, s, pos, 30, k_rest := ctx.empty((30, 1024)), ctx.empty((30, 1024)))
        assert not k_rest.download().any()
    finally:
        kv.close()


# ------------------------------------------------------------------ decode


def _check(got, want, bound, normal=False):
    """normal: the inputs are N(0, 1), and the error of the whole output is held to what random roundings add up to."""
    off = np.abs(got.reshape(24, 256).astype(np.float64) - want)
    worst = float((off / bound).max())
    print(f"[bound] {worst:.3f} of the bound, 2-norm {off_by(got, want):.2e}", flush=True)
    assert np.all(np.isfinite(got)) and worst <= 1.0
    assert not normal or off_by(got, want) <= NORMAL_TOL


def test_nan_in_one_head_stays_there(pkg, ctx):
    """A query head of NaN, and a cached key of NaN or infinity in one kv head, leave the other heads as they are."""
    P = 300
    rng = np.random.default_rng(19)
    K, V = _rows(rng, P), _rows(rng, P)
    Q = rng.standard_normal((24, 256)).astype(np.float32)
    for ty in sorted(TYPES):
        with Cache(pkg, ctx, ty, [P]) as c:
            for split in (None, 4096):
                clean = _decode(ctx, c, K, V, Q, None, P, split=split).reshape(24, 256)
                q = Q.copy()
                q[8, 3] = np.nan
                got = _decode(ctx, c, K, V, q, None, P, split=split).reshape(24, 256)
                other = np.arange(24) != 8
                assert np.isnan(got[8]).all() and np.array_equal(_bits(got[other]), _bits(clean[other]))
                k = K.copy()
                k[100, 256 * 2 + 7] = np.nan
                got = _decode(ctx, c, k, V, Q, None, P, split=split).reshape(24, 256)
                other = np.arange(24) // 6 != 2
                assert np.array_equal(_bits(got[other]), _bits(clean[other]))
                if ty != "q8_k":  # (a quantised row's NaN is a zero)
                    assert np.isnan(got[~other]).all()


def _decode(ctx, c, K, V, Q, G, P, split=None, appends=True, layer=3):
    """The last token appended by the call or beforehand; returns the output."""
    s = c.seqs[0]
    d_k, d_v, d_q, d_o = ctx.array(K), ctx.array(V), ctx.array(Q), ctx.empty((24, 256))
    d_g = ctx.array(G) if G is not None else None
    n = P - 1 if appends else P
    if n:
        c.kv.write(layer, s, 0, n, d_k, d_v)
    d_o.upload(np.full((24, 256), np.nan, np.float32))
    with decode_split(ctx, split):
        if appends:
            c.kv.attn_decode(layer, [s], [P - 1], d_q, d_o, k_new=d_k.offset((P - 1) * 1024),
                             v_new=d_v.offset((P - 1) * 1024), gate=d_g)
        else:
            c.kv.attn_decode(layer, [s], [P - 1], d_q, d_o, gate=d_g)
    got = d_o.download()
    for d in (d_k, d_v, d_q, d_o) + ((d_g,) if d_g is not None else ()):
        d.free()
    return got


@typed
@pytest.mark.parametrize("P", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 200, 1000])
def test_decode_lengths(pkg, ctx, ty, P):
    """One position, whole and partial pages, one split and many; the new
    token appended by the call (and stored as the type rounds it) or before."""
    rng = np.random.default_rng(P)
    K, V = _rows(rng, P), _rows(rng, P)
    Q, G = rng.standard_normal((24, 256)).astype(np.float32), rng.standard_normal((24, 256)).astype(np.float32)
    with Cache(pkg, ctx, ty, [P]) as c:
        got = _decode(ctx, c, K, V, Q, G, P)
        k, v = c.read(c.seqs[0], 0, P)
        assert np.array_equal(_bits(k), _bits(stored(K, c.ty))) and np.array_equal(_bits(v), _bits(stored(V, c.ty)))
        want, bound = attend(Q, k, v, G)
        _check(got, want, bound, normal=True)
        again = _decode(ctx, c, K, V, Q, G, P, appends=False)
        assert np.array_equal(_bits(got), _bits(again))


@typed
@pytest.mark.parametrize("split", [16, 32, 48, 80, 512, 1024, 4096])
def test_decode_splits(pkg, ctx, ty, split):
    """3003 tokens in splits from one page (188 of them) to the whole context."""
    rng = np.random.default_rng(split)
    K, V = _rows(rng, 3003), _rows(rng, 3003)
    Q = rng.standard_normal((24, 256)).astype(np.float32)
    with Cache(pkg, ctx, ty, [3003]) as c:
        got = _decode(ctx, c, K, V, Q, None, 3003, split=split)
        want, bound = attend(Q, stored(K, c.ty), stored(V, c.ty))
        _check(got, want, bound, normal=True)


@typed
@pytest.mark.parametrize("size", [2.0 ** 90, 2.0 ** 104, 2.0 ** 112])
def test_decode_queries_near_the_end_of_f32(pkg, ctx, ty, size):
    """Scores so large that each head's best token takes all: the output is
    that token's value.  Scores lie at most some 2^7 from the query's size, far
    from 2^128, and each is off by 264 u S at most (typed_rows.attend), S = sum
    |q k| / 16: a head whose first two are further apart than twice that has
    every other weight underflow.  Its value then passes through a sum over
    one weight's two or three parts, the joins' products and a division: 2^-21
    of it at most."""
    P = 300
    rng = np.random.default_rng(int(np.log2(size)))
    K, V = _rows(rng, P), _rows(rng, P)
    Q = (size * rng.standard_normal((24, 256))).astype(np.float32)
    with Cache(pkg, ctx, ty, [P]) as c:
        k, v = (stored(x, c.ty).reshape(P, 4, 256).astype(np.float64) for x in (K, V))
        for split in (None, 4096):
            got = _decode(ctx, c, K, V, Q, None, P, split=split).reshape(24, 256)
            checked = 0
            for h in range(24):
                s = k[:, h // 6] @ Q[h].astype(np.float64) / 16
                first, second = np.sort(s)[::-1][:2]
                if first - second < 4 * 264 * 2.0 ** -24 * (np.abs(k[:, h // 6]) @ np.abs(Q[h].astype(np.float64)) / 16).max():
                    continue
                want = v[s.argmax(), h // 6]
                assert np.all(np.abs(got[h] - want) <= 2.0 ** -21 * np.abs(want)), h
                checked += 1
            assert checked >= 20


@typed
@pytest.mark.parametrize("case", ["rising", "falling", "peaked", "large", "tiny", "flat", "huge_q", "huge_v", "mixed_heads"])
def test_decode_score_ranges(pkg, ctx, ty, case):
    """Running maxima that rise at every page or never, one weight that takes
    all, scores of hundreds, values that vanish, queries near the ends of the
    f32 range of sizes and heads of very different ones."""
    P = 700
    rng = np.random.default_rng(len(case))
    K, V = _rows(rng, P), _rows(rng, P)
    Q = rng.standard_normal((24, 256)).astype(np.float32)
    unit = np.zeros(1024, np.float32)
    unit[::256] = 4.0
    if case in ("rising", "falling"):
        Q[:, 0] = 4.0
        ramp = np.arange(P, dtype=np.float32)[:, None] * 0.25
        K += (ramp if case == "rising" else ramp[::-1]) * unit[None, :]
    elif case == "peaked":
        Q[:, 0] = 10.0
        K[351] += 20 * unit
    elif case == "large":
        Q *= 30
    elif case == "tiny":
        Q *= 1e-12
        V *= 1e-12 if ty != "f16" else 1e-2
    elif case == "flat":
        K[:] = K[0]
    elif case == "huge_q":
        Q *= 1e18
        K *= 1e-18 if ty != "f16" else 1.0
        Q *= 1.0 if ty != "f16" else 1e-18
    elif case == "huge_v":
        V *= 1e32 if ty != "f16" else 1e4
        Q *= 4
    elif case == "mixed_heads":
        Q *= (10.0 ** rng.uniform(-6, 1, (24, 1))).astype(np.float32)
    with Cache(pkg, ctx, ty, [P]) as c:
        for split in (None, 4096):
            got = _decode(ctx, c, K, V, Q, None, P, split=split)
            want, bound = attend(Q, stored(K, c.ty), stored(V, c.ty))
            _check(got, want, bound)


def test_decode_8bit_scales_far_apart(pkg, ctx):
    """Value rows whose scales differ by many orders: small ones first, a large
    one late, rows of zeros between."""
    P = 400
    rng = np.random.default_rng(77)
    for k in range(3):
        K, V = _rows(rng, P), _rows(rng, P)
        Q = rng.standard_normal((24, 256)).astype(np.float32)
        V *= (10.0 ** (rng.uniform(-20, 6, (P, 1)) if k == 0 else np.linspace(-12, 3, P)[:, None] if k == 1 else
                       np.linspace(3, -30, P)[:, None])).astype(np.float32)
        V[50:70] = 0.0
        if k == 2:
            V[:40] = 0.0
        with Cache(pkg, ctx, "q8_k", [P]) as c:
            for split in (None, 4096):
                got = _decode(ctx, c, K, V, Q, None, P, split=split)
                want, bound = attend(Q, stored(K, Q8_K), stored(V, Q8_K))
                _check(got, want, bound)


@typed
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_rows_past_the_end_do_not_count(pkg, ctx, ty, bad):
    """A page's rows past the sequence's last position hold NaN or infinities
    (a longer sequence's old rows): outputs are the same bit for bit."""
    P = 37
    rng = np.random.default_rng(6)
    K, V = _rows(rng, P), _rows(rng, P)
    Q, G = rng.standard_normal((24, 256)).astype(np.float32), rng.standard_normal((24, 256)).astype(np.float32)
    with Cache(pkg, ctx, ty, [64]) as c:
        clean = _decode(ctx, c, K, V, Q, G, P)
        junk = np.full((64, 1024), bad, np.float32)
        c.kv.write(3, c.seqs[0], 0, 64, ctx.array(junk), ctx.array(junk))
        assert np.array_equal(_bits(_decode(ctx, c, K, V, Q, G, P)), _bits(clean))
        assert np.array_equal(_bits(_decode(ctx, c, K, V, Q, G, P, appends=False)), _bits(clean))
        # a prefill's key blocks too
        d_o = ctx.empty((P, 24, 256))
        q = rng.standard_normal((P, 24, 256)).astype(np.float32)
        c.kv.attn_prefill(3, c.seqs[0], 0, P, ctx.array(q), ctx.array(K), ctx.array(V), d_o)
        assert np.all(np.isfinite(d_o.download()))


def _batch(pkg, ctx, ty, lengths, seed, slots=1):
    rng = np.random.default_rng(seed)
    c = Cache(pkg, ctx, ty, lengths, seed=seed, slots=slots)
    rows = []
    for s, n in zip(c.seqs, lengths):
        K, V = _rows(rng, n), _rows(rng, n)
        for slot in range(slots):
            c.kv.write(4 * slot + 3, s, 0, n, ctx.array(K), ctx.array(V))
        rows.append((stored(K, c.ty), stored(V, c.ty)))
    return c, rows, rng


@typed
def test_decode_batch(pkg, ctx, ty):
    """70 sequences of 1 to 2000 tokens on permuted pages, more than a launch
    takes; one given twice in a call that appends nothing."""
    lengths = [int(n) for n in np.random.default_rng(1).integers(1, 300, 70)]
    lengths[3], lengths[66], lengths[10] = 2000, 1777, 1
    c, rows, rng = _batch(pkg, ctx, ty, lengths, 31)
    with c:
        ids = list(range(70)) + [3]
        Q = rng.standard_normal((71, 24, 256)).astype(np.float32)
        d_o = ctx.empty((71, 24, 256))
        c.kv.attn_decode(3, [c.seqs[i] for i in ids], [lengths[i] - 1 for i in ids], ctx.array(Q), d_o)
        got = d_o.download()
        for b, i in enumerate(ids):
            want, bound = attend(Q[b], *rows[i])
            _check(got[b], want, bound, normal=True)


def _core_inputs(ctx, rng, n):
    x = {k: rng.standard_normal((n, w)).astype(np.float32) for k, w in (("qg", 12288), ("key", 1024), ("value", 1024))}
    x["qn"], x["kn"] = ((1 + 0.2 * rng.standard_normal(256)).astype(np.float32) for _ in range(2))
    return x, {k: ctx.array(v) for k, v in x.items()}


@typed
def test_full_core(pkg, ctx, ty):
    """full_core on sequences at 0, within a page, at a page's first and last
    position and far on, against its parts (attn_pre, append, attn_decode) bit
    for bit, and against the formula; and the form that allocates nothing."""
    lengths = [1, 40, 49, 64, 1500]
    c, _, rng = _batch(pkg, ctx, ty, lengths, 41)
    e, _, _ = _batch(pkg, ctx, ty, lengths, 41)
    with c, e:
        pos = [n - 1 for n in lengths]
        x, d = _core_inputs(ctx, rng, 5)
        out, out2, parts = (ctx.empty((5, 24, 256)) for _ in range(3))
        c.kv.full_core(3, c.seqs, pos, d["qn"], d["kn"], d["qg"], d["key"], d["value"], out)
        q, g, k = ctx.empty((5, 6144)), ctx.empty((5, 6144)), ctx.empty((5, 1024))
        for b, p in enumerate(pos):
            ctx.attn_pre(1, p, d["qn"], d["kn"], d["qg"].offset(b * 12288), d["key"].offset(b * 1024),
                         q.offset(b * 6144), g.offset(b * 6144), k.offset(b * 1024))
        e.kv.append(3, e.seqs, pos, [1] * 5, d["kn"], d["key"], d["value"])
        e.kv.attn_decode(3, e.seqs, pos, q, parts, gate=g)
        assert np.array_equal(_bits(out.download()), _bits(parts.download()))
        for s, t, n in zip(c.seqs, e.seqs, lengths):
            a, b = c.read(s, 0, n), e.read(t, 0, n)
            assert np.array_equal(_bits(a[0]), _bits(b[0])) and np.array_equal(_bits(a[1]), _bits(b[1]))
        c.kv.full_core_noalloc(3, c.seqs, pos, d["qn"], d["kn"], d["qg"], d["key"], d["value"], out2)
        assert np.array_equal(_bits(out.download()), _bits(out2.download()))
        got, qs, gs = out.download(), q.download(), g.download()
        for b, (s, n) in enumerate(zip(c.seqs, lengths)):
            want, bound = attend(qs[b], *c.read(s, 0, n), gs[b])
            _check(got[b], want, bound)


@typed
@pytest.mark.parametrize("n_seq", [1, 3])
def test_decode_graph(pkg, ctx, ty, n_seq):
    """Two layers' calls replayed as a graph, over page boundaries and split
    counts, with eager work between the replays: every replay equals the plain
    calls on a second cache bit for bit."""
    lengths = [200] * n_seq
    c, _, rng = _batch(pkg, ctx, ty, lengths, 51, slots=2)
    e, _, _ = _batch(pkg, ctx, ty, lengths, 51, slots=2)
    with c, e:
        x, d = _core_inputs(ctx, rng, n_seq)
        q = ctx.array(rng.standard_normal((n_seq, 6144)).astype(np.float32))
        o1, o2, p1, p2 = (ctx.empty((n_seq, 24, 256)) for _ in range(4))
        graph = c.kv.decode_graph(c.seqs, [150] * n_seq, [
            {"layer": 3, "q": d["qg"], "k_new": d["key"], "v_new": d["value"], "q_norm": d["qn"], "k_norm": d["kn"], "out": o1},
            {"layer": 7, "q": q, "k_new": d["key"], "v_new": d["value"], "out": o2}])
        other = c.kv.decode_graph(c.seqs, [100] * n_seq, [{"layer": 3, "q": q, "out": p2}])
        with graph, other:
            for p in (150, 159, 160, 15, 199, 207):
                pos = [p - 7 * i for i in range(n_seq)]
                graph.set_positions(pos)
                graph.launch()
                a1, a2 = o1.download(), o2.download()
                e.kv.full_core(3, e.seqs, pos, d["qn"], d["kn"], d["qg"], d["key"], d["value"], p1)
                e.kv.attn_decode(7, e.seqs, pos, q, p2, k_new=d["key"], v_new=d["value"])
                assert np.array_equal(_bits(a1), _bits(p1.download())) and np.array_equal(_bits(a2), _bits(p2.download()))
                # a second graph on the same cache between the replays
                other.set_positions([50] * n_seq)
                other.launch()
                e.kv.attn_decode(3, e.seqs, [50] * n_seq, q, p1)
                assert np.array_equal(_bits(p2.download()), _bits(p1.download()))
                graph.launch()
                assert np.array_equal(_bits(a1), _bits(o1.download())) and np.array_equal(_bits(a2), _bits(o2.download()))


# ------------------------------------------------------------------ prefill


@typed
@pytest.mark.parametrize("base,n", [(0, 1), (0, 33), (0, 200), (5, 40), (33, 7), (300, 65)])
def test_prefill(pkg, ctx, ty, base, n):
    """Causal attention of a prompt piece over a typed cache, the rows given
    with the call or stored beforehand, against 64 bits: the kernel's products
    of bf16 pairs carry 2^-16 of each operand."""
    rng = np.random.default_rng(base + n)
    K, V = _rows(rng, base + n), _rows(rng, base + n)
    Q, G = (rng.standard_normal((n, 24, 256)).astype(np.float32) for _ in range(2))
    with Cache(pkg, ctx, ty, [base + n]) as c, Cache(pkg, ctx, ty, [base + n]) as e:
        outs = []
        for x, given in ((c, True), (e, False)):
            if base:
                x.kv.write(3, x.seqs[0], 0, base, ctx.array(K[:base]), ctx.array(V[:base]))
            d_k, d_v, d_o = ctx.array(K[base:]), ctx.array(V[base:]), ctx.empty((n, 24, 256))
            if not given:
                x.kv.write(3, x.seqs[0], base, n, d_k, d_v)
            x.kv.attn_prefill(3, x.seqs[0], base, n, ctx.array(Q), d_k if given else None, d_v if given else None, d_o,
                              gate=ctx.array(G))
            outs.append(d_o.download())
        assert np.array_equal(_bits(outs[0]), _bits(outs[1]))
        k, v = stored(K, c.ty), stored(V, c.ty)
        for t in range(0, n, max(1, n // 7)):
            want, bound = attend(Q[t], k[:base + t + 1], v[:base + t + 1], G[t])
            # each product off by 2^-15 of its size instead of 2^-22: the bound's score term grows by 2^7
            _check(outs[0][t], want, bound * 2.0 ** 7)


@typed
def test_prefill_after_decode_and_truncate(pkg, ctx, ty):
    """Block images follow the rows: a piece, a decode step's append, a
    truncate, an append of other rows, and prefills over them."""
    rng = np.random.default_rng(9)
    P = 100
    K, V = _rows(rng, P), _rows(rng, P)
    w = np.ones(256, np.float32)
    with Cache(pkg, ctx, ty, [160]) as c:
        s = c.seqs[0]
        q = rng.standard_normal((64, 24, 256)).astype(np.float32)
        d_q, d_o, d_o2 = ctx.array(q), ctx.empty((64, 24, 256)), ctx.empty((64, 24, 256))
        c.kv.attn_prefill(3, s, 0, 64, d_q, ctx.array(K[:64]), ctx.array(V[:64]), d_o)
        c.kv.attn_decode(3, [s], [64], d_q, d_o2, k_new=ctx.array(K[64]), v_new=ctx.array(V[64]))
        c.kv.seq_truncate(s, 48)
        c.kv.append(3, [s], [40], [30], ctx.array(w), ctx.array(K[:30]), ctx.array(V[:30]))
        c.kv.attn_prefill(3, s, 60, 10, d_q, None, None, d_o)
        got = d_o.download(10)
        c.kv.set_prefill_cache(False)
        c.kv.attn_prefill(3, s, 60, 10, d_q, None, None, d_o2)
        assert np.array_equal(_bits(got), _bits(d_o2.download(10)))
        k, v = c.read(s, 0, 70)
        for t in range(10):
            want, bound = attend(q[t], k[:61 + t], v[:61 + t])
            _check(got[t], want, bound * 2.0 ** 7)


# ------------------------------------------------------------------ refusals, and a run of them together


def test_refused_calls_change_nothing(pkg, ctx):
    rng = np.random.default_rng(3)
    with Cache(pkg, ctx, "bf16", [40, 40], spare=0) as c:
        K = _rows(rng, 40)
        for s in c.seqs:
            c.kv.write(3, s, 0, 40, ctx.array(K), ctx.array(K))
        w, k, o = ctx.array(np.ones(256, np.float32)), ctx.array(_rows(rng, 64)), ctx.empty((64, 1024))
        state = lambda: (c.kv.free_pages(), [c.kv.seq_capacity(s) for s in c.seqs])  # noqa: E731
        before = state()
        a, b = c.seqs
        for call, why in (
                (lambda: c.kv.append(3, [a, a], [0, 1], [1, 1], w, k, k), "appears twice"),
                (lambda: c.kv.append(3, [a, b], [0, 47], [1, 2], w, k, k), "past the context limit"),
                (lambda: c.kv.append(4, [a], [0], [1], w, k, k), "not a full-attention layer"),
                (lambda: c.kv.append(3, [a], [0], [1], w, k, None), "NULL argument"),
                (lambda: c.kv.append(3, [a], [0], [1], w, k.ptr + 4, k), "16-byte aligned"),
                (lambda: c.kv.append(3, [a], [0, 0], [1], w, k, k), "differ in number"),
                (lambda: c.kv.gather(3, [a], [0], [2], o, o, ggml_type=1), "not as type 1"),
                (lambda: c.kv.gather(3, [a], [47], [2], o, o), "past the context limit"),
                (lambda: c.kv.attn_decode(3, [a], [48], o, o), "past the context limit"),
                (lambda: pkg.KVCache(ctx, 1, 4, 1, 16, ggml_type=12), "a KV cache holds")):
            with pytest.raises(pkg.Q38Error, match=why):
                call()
        assert state() == before
        for s in c.seqs:
            assert np.array_equal(c.read(s, 0, 40)[0], stored(K, c.ty))


@typed
def test_two_contexts_at_once(pkg, ctx, ty):
    """Calls of two contexts in turn, neither waited for: each has its stream
    and workspace, and gives what it gives alone."""
    rng = np.random.default_rng(23)
    other = pkg.Context(0)
    try:
        lengths, sides = [1500, 900, 40], []
        for c in (ctx, other):
            cache = Cache(pkg, c, ty, lengths, seed=len(sides))
            key, val = _rows(rng, sum(lengths)), _rows(rng, sum(lengths))
            w = c.array((1 + 0.2 * rng.standard_normal(256)).astype(np.float32))
            qg, k, v = (c.array(rng.standard_normal((3, n)).astype(np.float32)) for n in (12288, 1024, 1024))
            sides.append((c, cache, c.array(key), c.array(val), w, qg, k, v, [c.empty((3, 6144)) for _ in range(6)]))

        def step(i, side):
            c, cache, key, val, w, qg, k, v, out = side
            if i == 0:
                cache.kv.append(3, cache.seqs, [0, 0, 0], lengths, w, key, val)
            cache.kv.full_core(3, cache.seqs, [n + i for n in lengths], w, w, qg, k, v, out[i])
            c.add_rms_norm(3, 6144, out[i], qg, residual=qg, y=out[i])

        for side in sides:  # alone
            for i in range(6):
                step(i, side)
            side[0].sync()
        alone = [[o.download() for o in side[-1]] for side in sides]
        for side in sides:
            for s in side[1].seqs:
                side[1].kv.seq_truncate(s, 0)
            for o in side[-1]:
                o.zero()
            side[0].sync()
        for i in range(6):  # and in turn
            for side in sides:
                step(i, side)
        for side, want in zip(sides, alone):
            for o, x in zip(side[-1], want):
                assert np.isfinite(x).all() and np.array_equal(_bits(o.download()), _bits(x))
        for side in sides:
            side[1].kv.close()
    finally:
        other.close()


def test_append_is_not_captured(pkg, ctx):
    """Refused while the context's stream captures (a replay would leave stale
    prefill images), with the capture and the cache as they were."""
    hip = ctypes.CDLL(os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "lib", "libamdhip64.so"))
    rng = np.random.default_rng(17)
    stream, graph = ctypes.c_void_p(ctx.stream()), ctypes.c_void_p()
    with Cache(pkg, ctx, "f16", [40]) as c:
        w, k = ctx.array(np.ones(256, np.float32)), ctx.array(_rows(rng, 40))
        c.kv.write(3, c.seqs[0], 0, 40, k, k)
        before = c.read(c.seqs[0], 0, 40)
        ctx.sync()
        assert hip.hipStreamBeginCapture(stream, 2) == 0
        try:
            with pytest.raises(pkg.Q38Error, match="captured"):
                c.kv.append(3, c.seqs, [0], [4], w, k, k)
        finally:
            assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        hip.hipGraphDestroy(graph)
        assert all(np.array_equal(a, b) for a, b in zip(before, c.read(c.seqs[0], 0, 40)))
        c.kv.append(3, c.seqs, [0], [4], w, k, k)
        assert not np.array_equal(before[0], c.read(c.seqs[0], 0, 40)[0])


@typed
def test_prompts_then_tokens(pkg, ctx, ty):
    """As a server uses them: two prompts' rows appended raw in one call, each
    prompt's attention over the stored rows, then token after token of both
    through the layer norm, an 8-bit projection and full_core, a rejected
    token rolled back; the last token against 64 bits."""
    rng = np.random.default_rng(12)
    lens = [50, 23]
    width = 512
    with Cache(pkg, ctx, ty, lens) as c:
        total = sum(lens)
        x, d = _core_inputs(ctx, rng, total)
        q, g, k = ctx.empty((total, 6144)), ctx.empty((total, 6144)), ctx.empty((total, 1024))
        o = ctx.empty((total, 24, 256))
        c.kv.append(3, c.seqs, [0, 0], lens, d["kn"], d["key"], d["value"])
        at = 0
        for s, n in zip(c.seqs, lens):
            ctx.attn_pre(n, 0, d["qn"], d["kn"], d["qg"].offset(at * 12288), d["key"].offset(at * 1024),
                         q.offset(at * 6144), g.offset(at * 6144), k.offset(at * 1024))
            c.kv.attn_prefill(3, s, 0, n, q.offset(at * 6144), None, None, o.offset(at * 6144), gate=g.offset(at * 6144))
            at += n
        w = ctx.array((1 + 0.1 * rng.standard_normal(width)).astype(np.float32))
        mats = [ctx.array((0.02 * rng.standard_normal((rows, width))).astype(np.float32)) for rows in (12288, 1024, 1024)]
        h = ctx.array(rng.standard_normal((2, width)).astype(np.float32))
        y, q8 = ctx.empty((2, width)), ctx.empty((ctx.q8k_bytes(2, width),), np.uint8)
        qg, key, val, out = ctx.empty((2, 12288)), ctx.empty((2, 1024)), ctx.empty((2, 1024)), ctx.empty((2, 24, 256))
        pos = list(lens)
        for step in range(20):
            delta = ctx.array(rng.standard_normal((2, width)).astype(np.float32))
            ctx.add_rms_norm(2, width, delta, w, residual=h, sum_out=h, y=y, q8k=q8)
            ctx.dequantize_q8_k(2, width, q8, y)
            for m, dst, rows in zip(mats, (qg, key, val), (12288, 1024, 1024)):
                ctx.gemv_f32(0, rows, width, m, y, 2, dst)
            c.kv.full_core(3, c.seqs, pos, d["qn"], d["kn"], qg, key, val, out)
            if step == 9:  # the token of the first sequence is not kept
                c.kv.seq_truncate(c.seqs[0], pos[0])
            else:
                pos[0] += 1
            pos[1] += 1
        last = [pos[0] - 1, pos[1] - 1]
        got = out.download()
        for b, s in enumerate(c.seqs):
            ctx.attn_pre(1, last[b], d["qn"], d["kn"], qg.offset(b * 12288), key.offset(b * 1024), q, g, k)
            kk, vv = c.read(s, 0, last[b] + 1)
            want, bound = attend(q.download(1), kk, vv, g.download(1))
            _check(got[b], want, bound)
