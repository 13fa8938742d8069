"""A sequence that has evicted tokens, handed on to another cache."""
import numpy as np
import pytest
from test_gpu_weights import Cache, _bits, _q, _rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ty", ["f16", "bf16", "mxfp4"])
@pytest.mark.parametrize("form", ["core", "graph"])
def test_goes_on_bit_for_bit(pkg, ctx, ty, form):
    """Rows, sums, own positions and the evicted count carried over: decode steps, a prompt's piece and a second eviction give
    what they give where the sequence was.  (Rows of these types stand for values that they store again as they are.)"""
    rng = np.random.default_rng(5)
    P, keep, more, layers = 150, 60, 9, (3, 7)
    w = ctx.array((1 + 0.2 * rng.standard_normal(256)).astype(np.float32))
    steps = 20
    qg, key, val = (rng.standard_normal((more + steps, n)).astype(np.float32) for n in (12288, 1024, 1024))
    with Cache(pkg, ctx, ty, [P], slots=2) as a, Cache(pkg, ctx, ty, [P, P], slots=2, seed=9) as b:
        s, t = a.seqs[0], b.seqs[1]
        out = ctx.empty((24, 256))
        for layer in layers:
            d_k, d_v = ctx.array(_rows(rng, P)), ctx.array(_rows(rng, P))
            a.kv.write(layer, s, 0, P, d_k, d_v)
            a.kv.attn_observe(layer, s, P - 30, 30, ctx.array(_q(rng, 30)))
        a.kv.evict([s], [P], [keep], [10])
        for i in range(more):
            for layer in layers:
                a.kv.full_core(layer, [s], [keep + i], w, w, *(ctx.array(x[i]) for x in (qg, key, val)), out)
        n = keep + more
        b.kv.seq_reserve(t, n)
        for layer in layers:
            k, v, sums, own = ctx.empty((n, 1024)), ctx.empty((n, 1024)), ctx.empty((n, 4)), ctx.empty((n, 4), np.int32)
            a.kv.gather(layer, [s], [0], [n], k, v)
            a.kv.weights_get(layer, [s], [0], [n], sums, own)
            b.kv.write(layer, t, 0, n, k, v)
            b.kv.weights_put(layer, [t], [0], [n], sums, own)
        b.kv.seq_set_evicted(t, a.kv.seq_evicted(s), keep)
        assert b.kv.seq_evicted(t) == P - keep

        def same():
            assert b.kv.seq_evicted(t) == a.kv.seq_evicted(s)
            for layer in layers:
                for x, y in zip(a.rows(s, n, layer) + a.weights(s, n, layer), b.rows(t, n, layer) + b.weights(t, n, layer)):
                    assert np.array_equal(np.ascontiguousarray(x).view(np.uint32), np.ascontiguousarray(y).view(np.uint32))

        same()
        slots = [ctx.empty((m,)) for m in (12288, 1024, 1024)]
        outs = [ctx.empty((24, 256)) for _ in range(4)]
        graphs = {}
        for i in range(more, more + steps):
            for buf, x in zip(slots, (qg, key, val)):
                buf.upload(x[i])
            for c, q, o in ((a, s, outs[:2]), (b, t, outs[2:])):
                if form == "core":
                    for layer, to in zip(layers, o):
                        c.kv.full_core(layer, [q], [n], w, w, *slots, to)
                    continue
                if c not in graphs:
                    graphs[c] = c.kv.decode_graph([q], [n], [{"layer": layer, "q": slots[0], "k_new": slots[1], "v_new": slots[2],
                                                             "q_norm": w, "k_norm": w, "out": to} for layer, to in zip(layers, o)])
                graphs[c].set_positions([n])
                graphs[c].launch()
            for x, y in zip(outs[:2], outs[2:]):
                assert np.array_equal(_bits(x.download()), _bits(y.download()))
            n += 1
            if i == more + 8:
                for c, q in ((a, s), (b, t)):
                    c.kv.evict([q], [n], [50], [20])
                n = 50
                same()
        # a prompt's piece behind it
        Q, K, V = ctx.array(_q(rng, 7)), ctx.array(_rows(rng, 7)), ctx.array(_rows(rng, 7))
        o = [ctx.empty((7, 24, 256)) for _ in range(2)]
        for (c, q), to in zip(((a, s), (b, t)), o):
            c.kv.attn_prefill(3, q, n, 7, Q, K, V, to)
            c.kv.attn_observe(3, q, n, 7, Q)
            c.kv.write(7, q, n, 7, K, V)
        n += 7
        assert np.array_equal(_bits(o[0].download()), _bits(o[1].download()))
        same()
        for g in graphs.values():
            g.close()
