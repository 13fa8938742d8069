"""One token's attention where a head's scores come from its small query elements,
on large key elements, beside large ones on small keys: each product counts by its
own size."""
import numpy as np
import pytest
from parity import decode_split
from typed_rows import NORMAL_TOL, TYPES, attend, off_by, stored

P = 500


def _inputs(ratio, seed):
    """Queries of N(0, 1) / ratio on keys of N(0, 1) ratio, and in dim 1 a query of ratio on keys of N(0, 1) / (16
    ratio): scores of standard deviation 1, whose sums and roundings are as for N(0, 1) inputs."""
    rng = np.random.default_rng(seed)
    r = np.float32(ratio)
    Q = rng.standard_normal((24, 256)).astype(np.float32) / r
    K, V = (rng.standard_normal((P, 1024)).astype(np.float32) for _ in range(2))
    K *= r
    Q[:, 1] = r
    K[:, 1::256] /= np.float32(16.0) * r * r
    return Q, K, V


def _tol(ty, ratio):
    """A bf16 query has f32's exponents.  In f16 parts, the lower one 2^11 times as large and the largest element
    2^9 units at least, an element is off by 2^-36 units, 2^-45 of the largest, however small it is: 1/sqrt(3) of that in
    the root mean square, times 254 keys of size `ratio` over 16, in a score; held to twice that besides N(0, 1)'s."""
    return NORMAL_TOL + (0.0 if ty == "bf16" else 2 * 2.0 ** -45 * ratio * ratio * np.sqrt(254) / 16 / np.sqrt(3))


CASES = [("f16", 30.0), ("f16", 1000.0), ("f16", 8000.0)] + [(ty, r) for ty in ("bf16", "q8_k") for r in (30.0, 1000.0, 1e5)]


@pytest.mark.gpu
@pytest.mark.parametrize("ty,ratio", CASES)
def test_small_queries_on_large_keys(pkg, ctx, ty, ratio):
    Q, K, V = _inputs(ratio, int(ratio))
    kv = pkg.KVCache(ctx, n_slots=1, max_pages=32, max_seqs=1, max_tokens_per_seq=512, ggml_type=TYPES[ty])
    s, out = kv.seq_create(), ctx.empty((24, 256))
    k, v = stored(K, TYPES[ty]), stored(V, TYPES[ty])
    want, bound = attend(Q, k, v)
    try:
        kv.write(3, s, 0, P, ctx.array(K), ctx.array(V))
        for split in (4096, None):
            with decode_split(ctx, split):
                kv.attn_decode(3, [s], [P - 1], ctx.array(Q), out)
            got = out.download()
            worst = max(off_by(g, w) for g, w in zip(got, want))
            print(f"[bound] {float((np.abs(got - want) / bound).max()):.4f} of the bound, 2-norm {worst:.2e}", flush=True)
            assert np.all(np.abs(got - want) <= bound) and worst <= _tol(ty, ratio)
    finally:
        kv.close()


@pytest.mark.parametrize("ty,ratio", CASES)
def test_the_limits_on_the_cpu(ty, ratio):
    """Plain 32-bit products hold them; two f16 parts of one scale do not from a ratio of 1000 on."""
    Q, K, V = _inputs(ratio, int(ratio))
    k, v = stored(K, TYPES[ty]), stored(V, TYPES[ty])
    want, _ = attend(Q, k, v)

    def off(q):
        return max(off_by(attend(q, k, v)[0][h], want[h]) for h in range(24))

    f = np.float32
    s = np.stack([(k[:, 256 * (h // 6):256 * (h // 6) + 256] @ Q[h]) * f(0.0625) for h in range(24)])
    w = np.exp(s - s.max(1, keepdims=True))
    got = np.stack([w[h] @ v[:, 256 * (h // 6):256 * (h // 6) + 256] / w[h].sum(dtype=f) for h in range(24)])
    assert max(off_by(g, x) for g, x in zip(got, want)) <= NORMAL_TOL
    unit = np.exp2(10 - np.ceil(np.log2(np.abs(Q).max(1, keepdims=True)))).astype(f)
    x = Q * unit
    hi = x.astype(np.float16).astype(f)
    plain = (hi + (x - hi).astype(np.float16).astype(f)) / unit
    larger = (hi + ((x - hi) * f(2048)).astype(np.float16).astype(f) / f(2048)) / unit
    if ty != "bf16":
        assert off(larger) <= _tol(ty, ratio)
    if ratio >= 1000:
        assert off(plain) > _tol(ty, ratio)
