"""The residual's addition, the layer norm and its Q8_K rows (add_rms_norm),
and dequantize_q8_k, against the formula step by step."""
import ctypes
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _formula(x, r, w):
    """h and y with the operator's roundings: h and every product once, the mean and 1 / sqrt in f32, the sum of squares in 64 bits."""
    h = x if r is None else (x + r).astype(np.float32)
    mean = ((h.astype(np.float64) ** 2).sum(-1, keepdims=True) / h.shape[-1]).astype(np.float32)
    scale = np.float32(1.0) / np.sqrt(mean + np.float32(1e-6), dtype=np.float32)
    return h, ((h * scale).astype(np.float32) * w).astype(np.float32)


def _inputs(rng, t, n, size=1.0):
    return ((size * rng.standard_normal((t, n))).astype(np.float32), (size * rng.standard_normal((t, n))).astype(np.float32),
            (1 + 0.2 * rng.standard_normal(n)).astype(np.float32))


@pytest.mark.parametrize("width", [1, 2, 3, 4, 5, 63, 255, 256, 257, 260, 1000, 1024, 1028, 4100, 5120, 6144, 8191, 17408, 20480,
                                   20484, 20736, 49152, 50001])
@pytest.mark.parametrize("tokens", [1, 3, 8])
def test_norm(ctx, width, tokens):
    rng = np.random.default_rng(width + tokens)
    x, r, w = _inputs(rng, tokens, width)
    h, y = _formula(x, r, w)
    d_x, d_r, d_w = ctx.array(x), ctx.array(r), ctx.array(w)
    d_h, d_y = ctx.empty((tokens, width)), ctx.empty((tokens, width))
    ctx.add_rms_norm(tokens, width, d_x, d_w, residual=d_r, sum_out=d_h, y=d_y)
    got = d_y.download()
    assert np.array_equal(d_h.download(), h)
    # the 64-bit sums, in any order, round to the same f32 mean; each later step is the formula's
    assert np.array_equal(got, y)
    exact = h.astype(np.float64) / np.sqrt((h.astype(np.float64) ** 2).mean(-1, keepdims=True) + 1e-6) * w
    # roundings: mean (halved by the root), + eps (halved), root, reciprocal, two products
    assert np.all(np.abs(got - exact) <= 5.5 * 2.0 ** -24 * np.abs(exact) + 1e-45)


@pytest.mark.parametrize("width", [256, 512, 768, 5120, 17408, 20480, 20736, 49152])
@pytest.mark.parametrize("tokens", [1, 2, 9])
def test_q8k_rows(ctx, ref, width, tokens):
    """The Q8_K rows are the quantiser's of y, sums and scales included."""
    rng = np.random.default_rng(width * tokens)
    x, r, w = _inputs(rng, tokens, width, 5.0)
    x[0, :256], r[0, :256] = 0.0, 0.0                 # a block of zeros
    if width > 256:
        w[256:512] = np.sign(w[256:512])              # values of one size where h has them
        x[0, 256:512], r[0, 256:512] = 2.0 * np.sign(x[0, 256:512]), 0.0
    _, y = _formula(x, r, w)
    d = [ctx.array(v) for v in (x, r, w)]
    q8 = ctx.empty((ctx.q8k_bytes(tokens, width) + 64,), np.uint8)
    q8.upload(np.full(q8.shape, 0x5A, np.uint8))
    ctx.add_rms_norm(tokens, width, d[0], d[2], residual=d[1], q8k=q8)
    got = q8.download()
    want = ref.quantize_q8_k(y)
    assert np.array_equal(got[:-64], want) and np.all(got[-64:] == 0x5A)
    other, values = ctx.empty((ctx.q8k_bytes(tokens, width),), np.uint8), ctx.empty((tokens, width))
    ctx.quantize_q8_k(tokens, width, ctx.array(y), other)
    assert np.array_equal(other.download(), got[:-64])
    ctx.dequantize_q8_k(tokens, width, q8, values)
    q, _, s = ref.q8k_split(want, tokens, width)
    assert np.array_equal(values.download(), (q.reshape(tokens, -1, 256) * s[:, :, None]).astype(np.float32).reshape(tokens, width))


@pytest.mark.parametrize("width", [5, 256, 5120, 20736])
@pytest.mark.parametrize("form", ["sum=x", "sum=residual", "y=x", "y=residual", "both", "same input", "no residual"])
def test_in_place(ctx, width, form):
    rng = np.random.default_rng(width)
    x, r, w = _inputs(rng, 7, width)
    d_x, d_r, d_w = ctx.array(x), ctx.array(r), ctx.array(w)
    h, y = _formula(x, r, w)
    other = ctx.empty((7, width))
    if form == "sum=x":
        ctx.add_rms_norm(7, width, d_x, d_w, residual=d_r, sum_out=d_x, y=other)
        got = d_x, other
    elif form == "sum=residual":
        ctx.add_rms_norm(7, width, d_x, d_w, residual=d_r, sum_out=d_r, y=other)
        got = d_r, other
    elif form == "y=x":
        ctx.add_rms_norm(7, width, d_x, d_w, residual=d_r, sum_out=other, y=d_x)
        got = other, d_x
    elif form == "y=residual":
        ctx.add_rms_norm(7, width, d_x, d_w, residual=d_r, sum_out=other, y=d_r)
        got = other, d_r
    elif form == "both":
        ctx.add_rms_norm(7, width, d_x, d_w, residual=d_r, sum_out=d_r, y=d_x)
        got = d_r, d_x
    elif form == "same input":
        h, y = _formula(x, x, w)
        ctx.add_rms_norm(7, width, d_x, d_w, residual=d_x, sum_out=d_x, y=other)
        got = d_x, other
    else:
        h, y = _formula(x, None, w)
        ctx.add_rms_norm(7, width, d_x, d_w, sum_out=other, y=d_x)
        got = other, d_x
    assert np.array_equal(got[0].download(), h) and np.array_equal(got[1].download(), y)


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_rows_off_16_bytes(ctx, shift):
    """f32 rows need only their own alignment."""
    rng = np.random.default_rng(shift)
    x, r, w = _inputs(rng, 3, 1000)
    bufs = [ctx.empty((4, 1024)) for _ in range(5)]
    for b, v in zip(bufs, (x, r, w)):
        flat = np.zeros(4096, np.float32)
        flat[shift:shift + v.size] = v.reshape(-1)
        b.upload(flat.reshape(4, 1024))
    for b in bufs[3:]:
        b.zero()
    p = [b.offset(shift) for b in bufs]
    ctx.add_rms_norm(3, 1000, p[0], p[2], residual=p[1], sum_out=p[3], y=p[4])
    for b, want in zip(bufs[3:], _formula(x, r, w)):
        got = b.download().reshape(-1)
        assert np.array_equal(got[shift:shift + want.size], want.reshape(-1))
        assert not got[:shift].any() and not got[shift + want.size:].any()


def test_extremes(ctx):
    """Rows of zeros, sizes whose squares leave the f32 range, and NaN and
    infinities, which stay in their own row."""
    rng = np.random.default_rng(4)
    x, r, w = _inputs(rng, 8, 5120)
    x[0], r[0] = 0.0, 0.0
    x[1] *= 1e-25
    r[1] = 0.0
    x[2] *= 1e15
    x[4, 77] = np.nan
    x[6, 5] = np.inf
    d_h, d_y = ctx.empty((8, 5120)), ctx.empty((8, 5120))
    ctx.add_rms_norm(8, 5120, ctx.array(x), ctx.array(w), residual=ctx.array(r), sum_out=d_h, y=d_y)
    with np.errstate(all="ignore"):
        h, y = _formula(x, r, w)
    got_h, got_y = d_h.download(), d_y.download()
    for t in (0, 1, 2, 3, 5, 7):
        assert np.array_equal(got_h[t], h[t]) and np.array_equal(got_y[t], y[t]), t
    assert np.isnan(got_y[4]).all() and np.array_equal(got_y[6], y[6], equal_nan=True)


def test_many_rows(ctx):
    """More rows than the chip holds at once, an odd number."""
    rng = np.random.default_rng(10)
    t = 4099
    x, r, w = _inputs(rng, t, 768)
    d_h, d_y = ctx.empty((t, 768)), ctx.empty((t, 768))
    q8 = ctx.empty((ctx.q8k_bytes(t, 768),), np.uint8)
    ctx.add_rms_norm(t, 768, ctx.array(x), ctx.array(w), residual=ctx.array(r), sum_out=d_h, y=d_y, q8k=q8)
    h, y = _formula(x, r, w)
    assert np.array_equal(d_h.download(), h) and np.array_equal(d_y.download(), y)
    other = ctx.empty((ctx.q8k_bytes(t, 768),), np.uint8)
    ctx.quantize_q8_k(t, 768, d_y, other)
    assert np.array_equal(other.download(), q8.download())


@pytest.mark.parametrize("width,rows", [(4, (1 << 24) - 1), (1, (1 << 22) - 1)])
def test_most_rows_of_a_call(pkg, ctx, width, rows):
    """The most rows that one launch holds, in registers and value by value; one more is refused."""
    rng = np.random.default_rng(12)
    x = rng.standard_normal((rows, width), np.float32)
    w = (1 + 0.2 * rng.standard_normal(width)).astype(np.float32)
    d_x, d_w, d_y = ctx.array(x), ctx.array(w), ctx.empty((rows + 1, width))
    d_y.upload(np.full((rows + 1, width), -7.0, np.float32))
    ctx.add_rms_norm(rows, width, d_x, d_w, y=d_y)
    got = d_y.download()
    assert np.all(got[rows] == -7.0)
    for at in (slice(0, 5000), slice(rows // 2, rows // 2 + 5000), slice(rows - 5000, rows)):
        assert np.array_equal(got[at], _formula(x[at], None, w)[1])
    assert not np.any(got[:rows] == -7.0)
    d_more = ctx.empty((rows + 1, width))
    with pytest.raises(pkg.Q38Error, match="too large"):
        ctx.add_rms_norm(rows + 1, width, d_more, d_w, y=d_y)
    for d in (d_x, d_w, d_y, d_more):
        d.free()


def test_captured_and_replayed(pkg, ctx):
    """Captured from the context's stream and replayed: every replay equals the
    eager call, with eager work between the replays."""
    hip = ctypes.CDLL(os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "lib", "libamdhip64.so"))
    rng = np.random.default_rng(11)
    x, r, w = _inputs(rng, 5, 5120)
    d_x, d_r, d_w = ctx.array(x), ctx.array(r), ctx.array(w)
    d_h, d_y, e_h, e_y = (ctx.empty((5, 5120)) for _ in range(4))
    q8, e_q8 = (ctx.empty((ctx.q8k_bytes(5, 5120),), np.uint8) for _ in range(2))
    stream, graph, execu = ctypes.c_void_p(ctx.stream()), ctypes.c_void_p(), ctypes.c_void_p()
    ctx.sync()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    ctx.add_rms_norm(5, 5120, d_x, d_w, residual=d_r, sum_out=d_h, y=d_y, q8k=q8)
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(execu), graph, None, None, ctypes.c_size_t(0)) == 0
    try:
        for i in range(5):
            d_x.upload((x * (i + 1)).astype(np.float32))
            d_h.zero(), d_y.zero(), q8.zero()
            assert hip.hipGraphLaunch(execu, stream) == 0
            got = d_h.download(), d_y.download(), q8.download()
            ctx.add_rms_norm(5, 5120, d_x, d_w, residual=d_r, sum_out=e_h, y=e_y, q8k=e_q8)
            for a, b in zip(got, (e_h, e_y, e_q8)):
                assert np.array_equal(a, b.download())
            h, y = _formula((x * (i + 1)).astype(np.float32), r, w)
            assert np.array_equal(got[0], h) and np.array_equal(got[1], y)
    finally:
        hip.hipGraphExecDestroy(execu)
        hip.hipGraphDestroy(graph)
