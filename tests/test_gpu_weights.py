"""Sums of attention weights and eviction, over caches of every type that tracks
them, against plain 64-bit arithmetic on the values that the stored rows stand for."""
import numpy as np
import pytest
import typed_rows
from mxfp4_rows import MXFP4, stored4
from parity import decode_split
from typed_rows import attend, rms64, rope64

pytestmark = pytest.mark.gpu

TYPES = dict(typed_rows.TYPES, mxfp4=MXFP4)
typed = pytest.mark.parametrize("ty", sorted(TYPES))
U = 2.0 ** -24


def stored(x, ty):
    return stored4(x) if ty == "mxfp4" else typed_rows.stored(x, TYPES[ty])


#: What a query's parts leave of it: 22 bits in a decode; where a prompt's queries are observed over bf16 operands, two parts
#: rounded to nearest, each off by 2^-8 of what it stands for.
DECODE = 2.0 ** -22
OBSERVE = {"f16": 2.0 ** -22, "q8_k": 2.0 ** -22, "bf16": 2.0 ** -16, "mxfp4": 2.0 ** -16}


def weights_of(q, k, query=DECODE):
    """One token's softmax weights in 64 bits per kv head, [n][4], and a bound on what a kernel may be off.

    A score is off by (264 S + |s|) u at most (typed_rows.attend), S = sum |q k| / 16 over its row; a weight by that much
    of itself, by the denominator's own error (the largest score's, and (n + 16) u for the sum's order), 4 u for the exponential
    and its argument and 4 u for the division and the sum over heads; what a query's parts leave, `query` of S, in both."""
    n = k.shape[0]
    out, bound = np.zeros((n, 4)), np.zeros((n, 4))
    q, k = q.reshape(24, 256).astype(np.float64), k.astype(np.float64)
    for h in range(24):
        kk = k[:, 256 * (h // 6):256 * (h // 6) + 256]
        s = kk @ q[h] / 16.0
        size = np.abs(kk) @ np.abs(q[h]) / 16.0
        p = np.exp(s - s.max())
        p /= p.sum()
        e = (264 * size + np.abs(s) + 264 * size.max() + np.abs(s).max() + n + 24) * U + query * (size + size.max())
        out[:, h // 6] += p
        bound[:, h // 6] += 1.01 * e * p + 1e-37
    return out, bound


class Cache:
    def __init__(self, pkg, ctx, ty, lengths, seed=1, spare=4, slots=1):
        self.pkg, self.ctx, self.ty = pkg, ctx, ty
        pages = [(n + 15) // 16 + spare for n in lengths]
        self.kv = pkg.KVCache(ctx, n_slots=slots, max_pages=sum(pages) + 3, max_seqs=len(lengths), max_tokens_per_seq=16 * max(pages),
                              ggml_type=TYPES[ty])
        self.kv.track_weights(True)
        order = np.random.default_rng(seed).permutation(sum(pages))
        self.seqs, at = [], 0
        for n in pages:
            s = self.kv.seq_create()
            self.kv.seq_set_pages(s, order[at:at + n].tolist())
            self.seqs.append(s)
            at += n

    def weights(self, seq, n, layer=3, pos0=0):
        w, t = self.ctx.empty((max(1, n), 4)), self.ctx.empty((max(1, n), 4), np.int32)
        self.kv.weights_get(layer, [seq], [pos0], [n], w, t)
        return w.download(n), t.download(n)

    def rows(self, seq, n, layer=3):
        k, v = self.ctx.empty((max(1, n), 1024)), self.ctx.empty((max(1, n), 1024))
        self.kv.read(layer, seq, 0, n, k, v)
        return k.download(n), v.download(n)

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.kv.close()


def _rows(rng, n, sigma=1.0):
    return (sigma * rng.standard_normal((n, 1024))).astype(np.float32)


def _q(rng, n=1):
    return rng.standard_normal((n, 24, 256)).astype(np.float32)


def _bits(a):
    return np.ascontiguousarray(a, np.float32).view(np.uint32)


def _held(got, want, bound):
    off = np.abs(got.astype(np.float64) - want)
    print(f"[bound] {float((off / bound).max()):.3f} of the bound", flush=True)
    assert np.all(np.isfinite(got)) and np.all(off <= bound)


# ------------------------------------------------------------------ decode


@typed
@pytest.mark.parametrize("P", [1, 2, 15, 16, 17, 33, 63, 64, 255, 257, 1000])
def test_decode_adds_its_weights(pkg, ctx, ty, P):
    """Outputs equal those of a cache that tracks nothing, bit for bit; each call adds its weights to the positions it reads
    and touches none behind; an appended row starts its sum."""
    rng = np.random.default_rng(P)
    K, V, Q, G = _rows(rng, P + 20), _rows(rng, P + 20), _q(rng, 3), _q(rng, 3)
    d_q, d_g, d_k, d_v = ctx.array(Q), ctx.array(G), ctx.array(K), ctx.array(V)
    with Cache(pkg, ctx, ty, [P + 20]) as c:
        plain = pkg.KVCache(ctx, 1, P // 16 + 8, 1, 16 * (P // 16 + 8), ggml_type=TYPES[ty])
        s, t = c.seqs[0], plain.seq_create()
        c.kv.write(3, s, 0, P + 20, d_k, d_v)
        plain.write(3, t, 0, P + 20, d_k, d_v)
        mark = rng.standard_normal((P + 20, 4)).astype(np.float32)
        c.kv.weights_put(3, [s], [0], [P + 20], ctx.array(mark))
        o, o2 = ctx.empty((24, 256)), ctx.empty((24, 256))
        k = stored(K, ty)
        want, bound = mark[:P].astype(np.float64), np.zeros((P, 4))
        for i, split in enumerate((None, 16, 4096)):
            # the second call appends its row
            new = dict(k_new=d_k.offset((P - 1) * 1024), v_new=d_v.offset((P - 1) * 1024)) if i == 1 else {}
            with decode_split(ctx, split):
                c.kv.attn_decode(3, [s], [P - 1], d_q.offset(i * 6144), o, gate=d_g.offset(i * 6144), **new)
                plain.attn_decode(3, [t], [P - 1], d_q.offset(i * 6144), o2, gate=d_g.offset(i * 6144), **new)
            assert np.array_equal(_bits(o.download()), _bits(o2.download()))
            w, e = weights_of(Q[i], k[:P])
            if i == 1:
                want[-1], bound[-1] = 0, 0
            bound += e + U * (np.abs(want) + w)
            want += w
        got, tokens = c.weights(s, P + 20)
        _held(got[:P], want, bound)
        assert np.array_equal(_bits(got[P:]), _bits(mark[P:]))
        assert np.array_equal(tokens, np.arange(P + 20)[:, None].repeat(4, 1))
        plain.close()


@typed
def test_decode_batch_and_far_splits(pkg, ctx, ty):
    """70 sequences, more than a launch takes, some with many splits."""
    rng = np.random.default_rng(7)
    lengths = [int(n) for n in rng.integers(1, 200, 70)]
    lengths[3], lengths[66], lengths[10] = 5000, 1777, 1
    with Cache(pkg, ctx, ty, lengths, spare=1) as c:
        rows = [(_rows(rng, n), _rows(rng, n)) for n in lengths]
        for s, (K, V) in zip(c.seqs, rows):
            c.kv.write(3, s, 0, len(K), ctx.array(K), ctx.array(V))
        Q, o = _q(rng, 70), ctx.empty((70, 24, 256))
        d_q = ctx.array(Q)
        for _ in range(2):
            c.kv.attn_decode(3, c.seqs, [n - 1 for n in lengths], d_q, o)
        got = o.download()
        for b, (s, (K, V)) in enumerate(zip(c.seqs, rows)):
            k = stored(K, ty)
            out, bound = attend(Q[b], k, stored(V, ty))
            assert np.all(np.abs(got[b] - out) <= bound)
            w, e = weights_of(Q[b], k)
            _held(c.weights(s, len(K))[0], 2 * w, 2 * e + 4 * U * w)


@typed
def test_full_core_and_its_forms(pkg, ctx, ty):
    """full_core, the form that allocates nothing and a graph of it leave the same rows, outputs and sums, bit for bit."""
    lengths = [1, 40, 49, 64, 700]
    rng = np.random.default_rng(41)
    pos = [n - 1 for n in lengths]
    x = {k: rng.standard_normal((5, w)).astype(np.float32) for k, w in (("qg", 12288), ("key", 1024), ("value", 1024))}
    x["qn"], x["kn"] = ((1 + 0.2 * rng.standard_normal(256)).astype(np.float32) for _ in range(2))
    d = {k: ctx.array(v) for k, v in x.items()}
    K = [_rows(rng, n) for n in lengths]
    results = []
    for form in ("core", "noalloc", "graph"):
        with Cache(pkg, ctx, ty, lengths, slots=2) as c:
            for s, k in zip(c.seqs, K):
                c.kv.write(7, s, 0, len(k), ctx.array(k), ctx.array(k))
            out, got = ctx.empty((5, 24, 256)), []
            args = (d["qn"], d["kn"], d["qg"], d["key"], d["value"], out)
            graph = None
            if form == "graph":
                graph = c.kv.decode_graph(c.seqs, [max(0, p - 1) for p in pos], [
                    {"layer": 7, "q": d["qg"], "k_new": d["key"], "v_new": d["value"], "q_norm": d["qn"], "k_norm": d["kn"], "out": out}])
            for _ in range(3):
                if graph:
                    graph.set_positions(pos)
                    graph.launch()
                elif form == "core":
                    c.kv.full_core(7, c.seqs, pos, *args)
                else:
                    c.kv.full_core_noalloc(7, c.seqs, pos, *args)
                got.append(out.download())
                ctx.sync()
            for s, n in zip(c.seqs, lengths):
                got += [*c.rows(s, n, 7), c.weights(s, n, 7)[0]]
                # the other layer has none
                assert not c.weights(s, n, 3)[0].any()
            if graph:
                graph.close()
            results.append(got)
    for other in results[1:]:
        assert all(np.array_equal(_bits(a), _bits(b)) for a, b in zip(results[0], other))
    # the last token's own weight is this call's alone: each call stored it anew
    with Cache(pkg, ctx, ty, [1]) as c:
        o = ctx.empty((24, 256))
        for _ in range(3):
            c.kv.full_core(3, c.seqs, [0], d["qn"], d["kn"], d["qg"], d["key"], d["value"], o)
        # 1 for each of six heads: two exponentials of one score to different references (4 u, and 6 u each for
        # arguments of up to 8 in size), a reciprocal (2 u), six additions
        assert np.abs(c.weights(c.seqs[0], 1)[0].astype(np.float64) - 6).max() <= 6 * 24 * U


def test_a_stored_row_starts_at_zero(pkg, ctx):
    """Whichever call stores it; rows beside it keep their sums."""
    rng = np.random.default_rng(3)
    with Cache(pkg, ctx, "bf16", [100, 50]) as c:
        mark = (1 + rng.random((100, 4))).astype(np.float32)
        K = _rows(rng, 100)
        d_k = ctx.array(K)

        def reset():
            for s, n in zip(c.seqs, (100, 50)):
                c.kv.weights_put(3, [s], [0], [n], ctx.array(mark))

        def check(spans):
            for i, (s, n) in enumerate(zip(c.seqs, (100, 50))):
                want = mark[:n].copy()
                lo, hi = spans[i]
                want[lo:hi] = 0
                got, tokens = c.weights(s, n)
                assert np.array_equal(got, want) and np.array_equal(tokens, np.arange(n)[:, None].repeat(4, 1))

        reset()
        c.kv.write(3, c.seqs[0], 5, 23, d_k, d_k)
        check([(5, 28), (0, 0)])
        reset()
        c.kv.append(3, c.seqs, [17, 48], [33, 2], ctx.array(np.ones(256, np.float32)), d_k, d_k)
        check([(17, 50), (48, 50)])
        reset()
        c.kv.attn_prefill(3, c.seqs[1], 10, 30, ctx.array(_q(rng, 30)), d_k, d_k, ctx.empty((30, 24, 256)))
        check([(0, 0), (10, 40)])
        reset()
        c.kv.attn_prefill(3, c.seqs[1], 10, 30, ctx.array(_q(rng, 30)), None, None, ctx.empty((30, 24, 256)))
        check([(0, 0), (0, 0)])
        # many sequences' worth in one call, in another order
        c.kv.weights_put(3, c.seqs[::-1], [3, 90], [7, 10], None, ctx.array(np.arange(68).reshape(17, 4), np.int32))
        w, t = c.weights(c.seqs[1], 50)
        assert not w[3:10].any() and np.array_equal(w[10:], mark[10:50]) and np.array_equal(t[3:10].reshape(-1), np.arange(28))
        w, t = c.weights(c.seqs[0], 100)
        assert not w[90:].any() and np.array_equal(t[90:].reshape(-1), np.arange(28, 68)) and np.array_equal(w[:90], mark[:90])


@typed
@pytest.mark.parametrize("P", [2049, 4096])
def test_decode_of_one_long_split(pkg, ctx, ty, P):
    """A split of more tokens than its workgroup's threads take at once adds its sums in the decode launch."""
    rng = np.random.default_rng(P)
    K, Q = _rows(rng, P), _q(rng)
    with Cache(pkg, ctx, ty, [P]) as c, decode_split(ctx, 4096):
        s, o = c.seqs[0], ctx.empty((24, 256))
        c.kv.write(3, s, 0, P - 1, ctx.array(K), ctx.array(K))
        last = ctx.array(K[-1:])
        c.kv.attn_decode(3, [s], [P - 1], ctx.array(Q), o, k_new=last, v_new=last)
        got, t = c.weights(s, P)
        want, bound = weights_of(Q[0], stored(K, ty))
        _held(got, want, bound)
        assert np.array_equal(t, np.repeat(np.arange(P)[:, None], 4, 1))


def test_two_caches_of_one_context(pkg, ctx):
    """Calls on two tracking caches in turn, with one workspace between them, give what each gives by itself, bit for bit."""
    rng = np.random.default_rng(3)
    lengths, n = {"mxfp4": 700, "bf16": 300}, 20
    K = {ty: _rows(rng, P) for ty, P in lengths.items()}
    Q = {ty: _q(rng, n) for ty in lengths}

    def steps(c, ty, out):
        """One call of the run after the other."""
        s, P, q = c.seqs[0], lengths[ty], ctx.array(Q[ty])
        c.kv.write(3, s, 0, P, ctx.array(K[ty]), ctx.array(K[ty]))
        yield
        c.kv.attn_observe(3, s, P - n, n, q)
        yield
        o = ctx.empty((24, 256))
        held = P
        for u in range(6):
            new = ctx.array(K[ty][u:u + 1])
            c.kv.attn_decode(3, [s], [held], q.offset(u * 6144), o, k_new=new, v_new=new)
            yield
            out.append(_bits(o.download()))
            held += 1
            if u == 2:
                c.kv.evict([s], [held], [200], [16])
                held = 200
                yield
        out.extend([_bits(c.weights(s, held)[0]), c.weights(s, held)[1]] + [_bits(x) for x in c.rows(s, held)])

    alone, together = {}, {}
    for ty in lengths:
        with Cache(pkg, ctx, ty, [lengths[ty]]) as c:
            for _ in steps(c, ty, alone.setdefault(ty, [])):
                pass
    with Cache(pkg, ctx, "mxfp4", [700]) as c, Cache(pkg, ctx, "bf16", [300]) as d:
        runs = [steps(c, "mxfp4", together.setdefault("mxfp4", [])), steps(d, "bf16", together.setdefault("bf16", []))]
        while runs:
            runs = [r for r in runs if next(r, "done") != "done"]
    for ty in lengths:
        assert len(alone[ty]) == len(together[ty]) == 10
        for x, y in zip(alone[ty], together[ty]):
            assert np.array_equal(x, y)


# ------------------------------------------------------------------ a prompt's queries


@typed
@pytest.mark.parametrize("base,n", [(0, 1), (0, 2), (0, 16), (0, 17), (15, 2), (0, 70), (31, 33), (999, 1), (990, 20), (300, 48), (2000, 7)])
def test_observe(pkg, ctx, ty, base, n):
    """Every query's causal weights added to what is there, none behind the last one."""
    rng = np.random.default_rng(1000 * base + n)
    P = base + n
    K, Q = _rows(rng, P + 5), _q(rng, n)
    mark = rng.random((P + 5, 4)).astype(np.float32)
    with Cache(pkg, ctx, ty, [P + 5]) as c:
        s = c.seqs[0]
        c.kv.write(3, s, 0, P + 5, ctx.array(K), ctx.array(K))
        c.kv.weights_put(3, [s], [0], [P + 5], ctx.array(mark))
        c.kv.attn_observe(3, s, base, n, ctx.array(Q))
        got, _ = c.weights(s, P + 5)
        k = stored(K, ty)
        want, bound = mark[:P].astype(np.float64), np.zeros((P, 4))
        for u in range(n):
            w, e = weights_of(Q[u], k[:base + u + 1], OBSERVE[ty])
            want[:base + u + 1] += w
            bound[:base + u + 1] += e
        bound += (n + 6 * n) * U * want  # its own sum's order
        _held(got[:P], want, bound)
        assert np.array_equal(_bits(got[P:]), _bits(mark[P:]))
        # the same again, bit for bit
        c.kv.weights_put(3, [s], [0], [P + 5], ctx.array(mark))
        c.kv.attn_observe(3, s, base, n, ctx.array(Q))
        assert np.array_equal(_bits(c.weights(s, P + 5)[0]), _bits(got))


@pytest.mark.parametrize("ty,P,n", [(ty, P, n) for ty in sorted(TYPES) for P, n in ((24576, 2), (24577, 1), (24600, 19))] +
                         [("bf16", 4800, 300), ("q8_k", 4800, 300)])
def test_observe_long_and_many(pkg, ctx, ty, P, n):
    """Contexts on both sides of the one from which scores are formed twice, and more groups of queries than are kept at once."""
    rng = np.random.default_rng(P + n)
    K, Q = _rows(rng, P), _q(rng, n)
    with Cache(pkg, ctx, ty, [P]) as c:
        s = c.seqs[0]
        c.kv.write(3, s, 0, P, ctx.array(K), ctx.array(K))
        c.kv.attn_observe(3, s, P - n, n, ctx.array(Q))
        got, _ = c.weights(s, P)
        k = stored(K, ty)
        want, bound = np.zeros((P, 4)), np.zeros((P, 4))
        for u in range(n):
            w, e = weights_of(Q[u], k[:P - n + u + 1], OBSERVE[ty])
            want[:P - n + u + 1] += w
            bound[:P - n + u + 1] += e
        _held(got, want, bound + 7 * n * U * want)
        c.kv.weights_put(3, [s], [0], [P])
        c.kv.attn_observe(3, s, P - n, n, ctx.array(Q))
        assert np.array_equal(_bits(c.weights(s, P)[0]), _bits(got))


@typed
def test_observe_equals_decode_steps(pkg, ctx, ty):
    """A long context with large and small queries: the sums of one call against those of decode steps."""
    rng = np.random.default_rng(5)
    P, n = 5003, 21
    K, Q = _rows(rng, P), _q(rng, n)
    Q *= (10.0 ** rng.uniform(-3, 0.7, (n, 24, 1))).astype(np.float32)
    with Cache(pkg, ctx, ty, [P]) as c:
        s = c.seqs[0]
        c.kv.write(3, s, 0, P, ctx.array(K), ctx.array(K))
        d_q, o = ctx.array(Q), ctx.empty((24, 256))
        c.kv.attn_observe(3, s, P - n, n, d_q)
        got, _ = c.weights(s, P)
        c.kv.weights_put(3, [s], [0], [P])
        for u in range(n):
            c.kv.attn_decode(3, [s], [P - n + u], d_q.offset(u * 6144), o)
        steps, _ = c.weights(s, P)
        k, bound = stored(K, ty), np.zeros((P, 4))
        for u in range(n):
            bound[:P - n + u + 1] += weights_of(Q[u], k[:P - n + u + 1], OBSERVE[ty])[1]
        _held(got, steps.astype(np.float64), 2 * bound + 14 * n * U * np.maximum(got, steps))
        assert abs(float(got.astype(np.float64).sum()) - 24 * n) < 1e-2


# ------------------------------------------------------------------ eviction


def chosen(w, tokens, n, keep, first_recent):
    """Where the token that ends at each of the first `keep` positions was (one kv head)."""
    rank = [(0 if tokens[p] >= first_recent else 1, 1 if np.isnan(w[p]) else 0, 0 if np.isnan(w[p]) else -float(w[p]), p) for p in range(n)]
    stays = set(r[-1] for r in sorted(rank)[:keep])
    late = iter(sorted(p for p in stays if p >= keep))
    return [p if p in stays else next(late) for p in range(keep)]


def _evict_and_check(c, seqs, n, keep, recent, layers, before):
    """before: (k, v, weights, tokens, evicted) of each sequence and layer."""
    c.kv.evict(seqs, n, keep, recent)
    for s, m, kp, r in zip(seqs, n, keep, recent):
        for layer in layers:
            k0, v0, w0, t0, gone = before[s, layer]
            k1, v1 = c.rows(s, kp, layer)
            w1, t1 = c.weights(s, kp, layer)
            for j in range(4):
                at = chosen(w0[:, j], t0[:, j], m, kp, m + gone - r)
                dims = slice(256 * j, 256 * j + 256)
                assert np.array_equal(_bits(k1[:, dims]), _bits(k0[at][:, dims]))
                assert np.array_equal(_bits(v1[:, dims]), _bits(v0[at][:, dims]))
                assert np.array_equal(_bits(w1[:, j]), _bits(w0[at, j])) and np.array_equal(t1[:, j], t0[at, j])
        assert c.kv.seq_evicted(s) == before[s, layers[0]][4] + m - kp
        assert c.kv.seq_capacity(s) == (kp + 15) // 16 * 16


def _state(c, seqs, n, layers):
    return {(s, layer): (*c.rows(s, m, layer), *c.weights(s, m, layer), c.kv.seq_evicted(s)) for s, m in zip(seqs, n) for layer in layers}


@typed
def test_evict(pkg, ctx, ty):
    """Ragged sequences over two layers: none, one, some and all evicted; ties, zeros of either sign, infinities, NaN; recent tokens that
    weigh nothing; a second eviction of what is left and has come since."""
    rng = np.random.default_rng(17)
    n = [1, 16, 17, 100, 333, 1200, 40, 64]
    keep = [1, 1, 16, 33, 250, 77, 0, 64]
    recent = [0, 1, 3, 33, 10, 16, 0, 64]
    with Cache(pkg, ctx, ty, n, slots=2) as c:
        for s, m in zip(c.seqs, n):
            for layer in (3, 7):
                c.kv.write(layer, s, 0, m, ctx.array(_rows(rng, m)), ctx.array(_rows(rng, m)))
                w = np.round(np.exp(rng.normal(-2, 2, (m, 4))), 2).astype(np.float32)  # many ties
                w[rng.random((m, 4)) < 0.1] = 0.0
                w[rng.random((m, 4)) < 0.05] = -0.0
                w[rng.random((m, 4)) < 0.03] = np.nan
                w[rng.random((m, 4)) < 0.03] = -1.0
                w[rng.random((m, 4)) < 0.02] = np.inf
                c.kv.weights_put(layer, [s], [0], [m], ctx.array(w))
        free = c.kv.free_pages()
        held = sum(c.kv.seq_capacity(s) for s in c.seqs) // 16
        _evict_and_check(c, c.seqs, n, keep, recent, (3, 7), _state(c, c.seqs, n, (3, 7)))
        assert c.kv.free_pages() == free + held - sum((k + 15) // 16 for k in keep)
        # more tokens, and again, in another order of sequences
        more = [m + 9 for m in keep]
        for s, kp in zip(c.seqs, keep):
            for layer in (3, 7):
                c.kv.write(layer, s, kp, 9, ctx.array(_rows(rng, 9)), ctx.array(_rows(rng, 9)))
        for s, kp in zip(c.seqs, keep):
            assert np.array_equal(c.weights(s, 9, 7, kp)[1], (kp + c.kv.seq_evicted(s) + np.arange(9))[:, None].repeat(4, 1))
        order = rng.permutation(8)
        seqs, more, less = [c.seqs[i] for i in order], [more[i] for i in order], [max(4, keep[i] // 2) for i in order]
        _evict_and_check(c, seqs, more, less, [min(12, x) for x in less], (3, 7), _state(c, seqs, more, (3, 7)))


@typed
def test_evict_long(pkg, ctx, ty):
    """More pages than the choice's workgroup has threads."""
    rng = np.random.default_rng(23)
    P = 40001
    with Cache(pkg, ctx, ty, [P]) as c:
        s = c.seqs[0]
        c.kv.write(3, s, 0, P, ctx.array(_rows(rng, P)), ctx.array(_rows(rng, P)))
        c.kv.weights_put(3, [s], [0], [P], ctx.array(np.round(rng.random((P, 4)) * 500).astype(np.float32)))
        _evict_and_check(c, [s], [P], [P // 2], [100], (3,), _state(c, [s], [P], (3,)))


def test_evict_many_sequences(pkg, ctx):
    """More than a launch takes."""
    rng = np.random.default_rng(29)
    n = [int(x) for x in rng.integers(1, 60, 67)]
    with Cache(pkg, ctx, "mxfp4", n, spare=0) as c:
        for s, m in zip(c.seqs, n):
            c.kv.write(3, s, 0, m, ctx.array(_rows(rng, m)), ctx.array(_rows(rng, m)))
            c.kv.weights_put(3, [s], [0], [m], ctx.array(rng.random((m, 4)).astype(np.float32)))
        keep = [int(rng.integers(0, m + 1)) for m in n]
        _evict_and_check(c, c.seqs, n, keep, [k // 3 for k in keep], (3,), _state(c, c.seqs, n, (3,)))


# ------------------------------------------------------------------ a run of them together


@typed
@pytest.mark.parametrize("form", ["core", "graph"])
def test_generation_in_a_bounded_cache(pkg, ctx, ty, form):
    """A prompt, its last queries observed, an eviction, decode steps with an eviction whenever the cache is full, over one layer:
    each step's output is the attention over the tokens that a plain model of the cache holds, turned at their own positions."""
    rng = np.random.default_rng(11)
    P, keep, recent, limit, steps = 120, 50, 8, 64, 45
    w = (1 + 0.2 * rng.standard_normal(256)).astype(np.float32)
    d_w = ctx.array(w)
    total = P + steps
    qg, key, val = (rng.standard_normal((total, n)).astype(np.float32) for n in (12288, 1024, 1024))
    turned_k = rope64(rms64(key.reshape(-1, 4, 256), w), np.arange(total)).reshape(-1, 1024)
    with Cache(pkg, ctx, ty, [P], spare=2) as c:
        s = c.seqs[0]
        d_qg, d_key, d_val = ctx.array(qg), ctx.array(key), ctx.array(val)
        q, g, k = ctx.empty((P, 6144)), ctx.empty((P, 6144)), ctx.empty((P, 1024))
        ctx.attn_pre(P, 0, d_w, d_w, d_qg, d_key, q, g, k)
        c.kv.attn_prefill(3, s, 0, P, q, k, d_val, ctx.empty((P, 6144)), gate=g)
        c.kv.attn_observe(3, s, P - 16, 16, q.offset((P - 16) * 6144))
        # the plain model: per kv head the own positions of the tokens held, in the cache's order
        order = [list(range(P)) for _ in range(4)]

        def evict(n):
            w0, t0 = c.weights(s, n)
            for j in range(4):
                assert t0[:, j].tolist() == order[j]
                at = chosen(w0[:, j], t0[:, j], n, keep, n + c.kv.seq_evicted(s) - recent)
                order[j] = [order[j][p] for p in at]
            c.kv.evict([s], [n], [keep], [recent])
            for j in range(4):
                assert c.weights(s, keep)[1][:, j].tolist() == order[j]
                last = P if n == P else P + step + 1
                assert set(range(last - recent, last)) <= set(order[j])

        step = 0
        evict(P)
        out, n = ctx.empty((24, 256)), keep
        graph = None
        slots = [ctx.empty((m,)) for m in (12288, 1024, 1024)]
        for step in range(steps):
            t = P + step
            for buf, x in zip(slots, (qg, key, val)):
                buf.upload(x[t])
            if form == "core":
                c.kv.full_core(3, [s], [n], d_w, d_w, *slots, out)
            else:
                if graph is None:
                    graph = c.kv.decode_graph([s], [n], [{"layer": 3, "q": slots[0], "k_new": slots[1], "v_new": slots[2],
                                                         "q_norm": d_w, "k_norm": d_w, "out": out}])
                graph.set_positions([n])
                graph.launch()
            for j in range(4):
                order[j].append(t)
            n += 1
            got = out.download().reshape(24, 256)
            ks, vs = c.rows(s, n)
            qn = qg[t].reshape(24, 2, 256)
            q64 = rope64(rms64(qn[None, :, 0], w), [t])[0].astype(np.float32)
            # what the cache holds: the tokens of the model, turned at their own positions, in the type's rounding
            for j in range(4):
                dims = slice(256 * j, 256 * j + 256)
                assert np.array_equal(_bits(vs[:, dims]), _bits(stored(val, ty)[order[j]][:, dims]))
                far = np.abs(ks[:, dims] - stored(turned_k.astype(np.float32), ty)[order[j]][:, dims])
                # one step of the type where a rounding fell the other way
                assert far.max() <= {"f16": 2.0 ** -8, "bf16": 2.0 ** -5, "q8_k": 0.1, "mxfp4": 2.01}[ty]
                assert np.mean(far > 1e-4) < 0.01
            want, bound = attend(q64, ks, vs, qn[:, 1])
            # the query's own norm and turn: some 8 roundings of it besides
            assert np.all(np.abs(got - want) <= 4 * bound)
            if n == limit:
                evict(n)
                n = keep
                if graph is not None:
                    with pytest.raises(pkg.Q38Error, match="evicted tokens since"):
                        graph.launch()
        assert c.kv.seq_evicted(s) == P + steps - n
        if graph is not None:
            graph.close()


def test_begun_anew(pkg, ctx):
    """What an eviction leaves, and what takes it back; refusals that need a device."""
    rng = np.random.default_rng(2)
    with Cache(pkg, ctx, "mxfp4", [100, 100]) as c:
        K = ctx.array(_rows(rng, 100))
        for s in c.seqs:
            c.kv.write(3, s, 0, 100, K, K)
        a, b = c.seqs
        c.kv.evict([a], [100], [40], [10])
        w = ctx.array(np.ones(256, np.float32))
        for call, why in ((lambda: c.kv.append(3, [a], [40], [2], w, K, K), "has evicted tokens"),
                          (lambda: c.kv.seq_truncate(a, 39), "in no order"),
                          (lambda: c.kv.track_weights(False), "has evicted tokens"),
                          (lambda: c.kv.evict([a], [39], [3], [1]), "since its last eviction"),
                          (lambda: c.kv.evict([a], [100], [3], [1]), "not reserved"),
                          (lambda: c.kv.attn_decode(3, [b, b], [99, 99], K, K), "appears twice")):
            with pytest.raises(pkg.Q38Error, match=why):
                call()
        assert c.kv.seq_evicted(a) == 60 and c.kv.seq_evicted(b) == 0
        c.kv.append(3, [b, a], [98, 40], [2, 0], w, K, K)
        c.kv.seq_truncate(a, 40)
        for anew in (lambda: c.kv.seq_truncate(a, 0), lambda: c.kv.seq_reset(a)):
            anew()
            assert c.kv.seq_evicted(a) == 0
            c.kv.append(3, [a], [0], [100], w, K, K)
            assert np.array_equal(c.weights(a, 100)[1][:, 0], np.arange(100))
            c.kv.evict([a], [100], [40], [10])
        c.kv.seq_free(a)
        c.kv.track_weights(False)
        with pytest.raises(pkg.Q38Error, match="does not track"):
            c.kv.weights_get(3, [b], [0], [1], K)
        o = ctx.empty((24, 256))
        c.kv.attn_decode(3, [b], [99], K, o)
        c.kv.track_weights(True)
        assert np.array_equal(c.weights(b, 100)[1][:, 3], np.arange(100)) and not c.weights(b, 100)[0].any()
    kv = pkg.KVCache(ctx, 1, 4, 1, 64)
    with pytest.raises(pkg.Q38Error, match="F32 rows"):
        kv.track_weights(True)
    kv.close()


def test_graph_recorded_before_tracking_is_refused(pkg, ctx):
    kv = pkg.KVCache(ctx, 1, 4, 1, 64, ggml_type=MXFP4)
    s = kv.seq_create()
    kv.seq_reserve(s, 32)
    q, o = ctx.array(np.zeros(6144, np.float32)), ctx.empty((24, 256))
    with kv.decode_graph([s], [20], [{"layer": 3, "q": q, "out": o}]) as graph:
        kv.track_weights(True)
        for call in (graph.launch, lambda: graph.set_positions([21])):
            with pytest.raises(pkg.Q38Error, match="tracking of weights has changed"):
                call()
        kv.track_weights(False)
        graph.set_positions([21])
        graph.launch()
        ctx.sync()
    # tracking off and on again under a graph: its arguments still name the sums
    kv.track_weights(True)
    with kv.decode_graph([s], [20], [{"layer": 3, "q": q, "out": o}]) as graph:
        graph.launch()
        kv.track_weights(False)
        kv.track_weights(True)
        graph.launch()
        w = ctx.empty((21, 4))
        kv.weights_get(3, [s], [0], [21], w)
        assert np.abs(w.download().sum(0) - 6).max() <= 6 * 40 * U
    kv.close()


def test_prefill_and_images_follow_an_eviction(pkg, ctx):
    """Prompt pieces before and after an eviction: the block images of what moved are formed anew."""
    rng = np.random.default_rng(31)
    for ty in sorted(TYPES):
        with Cache(pkg, ctx, ty, [200]) as c:
            s = c.seqs[0]
            K, V, Q = _rows(rng, 230), _rows(rng, 230), _q(rng, 200)
            out, out2 = ctx.empty((200, 24, 256)), ctx.empty((200, 24, 256))
            c.kv.attn_prefill(3, s, 0, 200, ctx.array(Q), ctx.array(K[:200]), ctx.array(V[:200]), out)
            c.kv.attn_observe(3, s, 180, 20, ctx.array(Q[180:]))
            c.kv.evict([s], [200], [77], [9])
            c.kv.attn_prefill(3, s, 77, 30, ctx.array(Q), ctx.array(K[200:]), ctx.array(V[200:]), out)
            got = out.download(30)
            c.kv.set_prefill_cache(False)
            c.kv.attn_prefill(3, s, 77, 30, ctx.array(Q), None, None, out2)
            assert np.array_equal(_bits(got), _bits(out2.download(30)))
            k, v = c.rows(s, 107)
            assert np.array_equal(_bits(v[77:]), _bits(stored(V[200:], ty)))
            for t in (0, 13, 29):
                want, bound = attend(Q[t], k[:78 + t], v[:78 + t])
                assert np.all(np.abs(got[t] - want) <= bound * 2.0 ** 7)


def test_two_graphs_two_layers(pkg, ctx):
    """Two recorded graphs of two layers each on one tracking cache, replayed in turn with eager steps between: outputs and
    sums equal those of plain calls on another cache, bit for bit."""
    rng = np.random.default_rng(37)
    lengths = [90, 300]
    with Cache(pkg, ctx, "mxfp4", lengths, slots=2) as c, Cache(pkg, ctx, "mxfp4", lengths, slots=2, seed=8) as e:
        for n, a, b in zip(lengths, c.seqs, e.seqs):
            K = ctx.array(_rows(rng, n))
            for layer in (3, 7):
                c.kv.write(layer, a, 0, n, K, K)
                e.kv.write(layer, b, 0, n, K, K)
        q1, q2 = ctx.array(_q(rng, 2)), ctx.array(_q(rng, 2))
        k = ctx.array(_rows(rng, 2))
        o = [ctx.empty((2, 24, 256)) for _ in range(6)]
        calls = lambda a, b: [{"layer": 3, "q": q1, "out": a}, {"layer": 7, "q": q2, "k_new": k, "v_new": k, "out": b}]  # noqa: E731
        with c.kv.decode_graph(c.seqs, [80, 250], calls(o[0], o[1])) as g, c.kv.decode_graph(c.seqs, [40, 290], calls(o[2], o[3])) as h:
            for pos in ([80, 250], [89, 299], [15, 16]):
                for graph, x, at in ((g, o[0:2], pos), (h, o[2:4], [p // 2 for p in pos])):
                    graph.set_positions(at)
                    for _ in range(2):
                        graph.launch()
                        e.kv.attn_decode(3, e.seqs, at, q1, o[4])
                        e.kv.attn_decode(7, e.seqs, at, q2, o[5], k_new=k, v_new=k)
                        assert np.array_equal(_bits(x[0].download()), _bits(o[4].download()))
                        assert np.array_equal(_bits(x[1].download()), _bits(o[5].download()))
                c.kv.attn_decode(3, c.seqs, pos, q2, o[4])
                e.kv.attn_decode(3, e.seqs, pos, q2, o[5])
            for n, a, b in zip(lengths, c.seqs, e.seqs):
                for layer in (3, 7):
                    assert np.array_equal(_bits(c.weights(a, n, layer)[0]), _bits(e.weights(b, n, layer)[0]))


def test_sums_of_large_contexts_past_2_32_bytes(pkg, ctx):
    """Pages at the end of a pool whose sums' and rows' offsets pass 2^32 bytes: decode, observe and eviction there."""
    n_pages = 4300000 // 2
    kv = pkg.KVCache(ctx, 2, n_pages, 1, 16 * 200, ggml_type=MXFP4)
    try:
        kv.track_weights(True)
        s = kv.seq_create()
        kv.seq_set_pages(s, [n_pages - 1 - i for i in range(20)])
        rng = np.random.default_rng(4)
        P = 315
        K, V, Q = _rows(rng, P), _rows(rng, P), _q(rng, 5)
        kv.write(7, s, 0, P, ctx.array(K), ctx.array(V))
        o = ctx.empty((24, 256))
        kv.attn_decode(7, [s], [P - 1], ctx.array(Q[0]), o)
        kv.attn_observe(7, s, P - 4, 4, ctx.array(Q[1:]))
        w, t = ctx.empty((P, 4)), ctx.empty((P, 4), np.int32)
        kv.weights_get(7, [s], [0], [P], w, t)
        k = stored(K, "mxfp4")
        want, off = weights_of(Q[0], k)
        for u in range(4):
            a, e = weights_of(Q[1 + u], k[:P - 3 + u], OBSERVE["mxfp4"])
            want[:P - 3 + u] += a
            off[:P - 3 + u] += e + 40 * U * want[:P - 3 + u]
        w0, t0 = w.download(), t.download()
        _held(w0, want, off)
        kv.evict([s], [P], [100], [10])
        k1, v1 = ctx.empty((100, 1024)), ctx.empty((100, 1024))
        kv.read(7, s, 0, 100, k1, v1)
        for j in range(4):
            at = chosen(w0[:, j], t0[:, j], P, 100, P - 10)
            dims = slice(256 * j, 256 * j + 256)
            assert np.array_equal(k1.download()[:, dims], k[at][:, dims])
            assert np.array_equal(v1.download()[:, dims], stored(V, "mxfp4")[at][:, dims])
    finally:
        kv.close()
