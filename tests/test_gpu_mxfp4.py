"""MXFP4 conversion, products, packed products and the MLP through the C ABI
against the 64-bit oracle (tests/mx_oracle.py).

Conversions are exact: codes, scales and padding are compared bit by bit.
fp32 products may be off by mx_oracle.product_bound; bf16 results by half a
unit in the last place more (2^-9 of the value; 2^-8 allowed).  Packed products
take operands whose scales are near each other, so that every partial sum is a
whole number of units below 2^24 and fp32 is exact: bit by bit again."""
import numpy as np
import pytest

import aiehlc_amd as mi
import mx_oracle as mx

pytestmark = pytest.mark.gpu

DT = {"f32": mi.F32, "bf16": mi.BF16}


def _say(*a):
    print("[case]", *a, flush=True)


def _up(ctx, x, dtype):
    return ctx.upload(mx.bf16_bits(x) if dtype == "bf16" else np.asarray(x, np.float32))


def _down(ctx, buf, dtype, shape):
    if dtype == "bf16":
        return mx.from_bf16_bits(ctx.download(buf, np.uint16, shape))
    return ctx.download(buf, np.float32, shape)


def _packed(ctx, rows, cols, fill=0xA5):
    """Buffers of a packed matrix, full of a pattern that a kernel has to overwrite."""
    q, s = mi.mxfp4_shapes(rows, cols)
    return ctx.upload(np.full(q, fill, np.uint8)), ctx.upload(np.full(s, fill, np.uint8))


def _values(rng, R, C, dtype, spread=20):
    """Values of many sizes, with whole blocks of zeros, single large values, ties between codes and tiny ones."""
    x = rng.standard_normal((R, C)) * np.exp2(rng.integers(-spread, spread + 1, (R, (C + 31) // 32)).repeat(32, 1)[:, :C])
    ties = rng.random((R, C)) < 0.2
    x = np.where(ties, rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 7, -0.25, -5, 0, -0.0], (R, C)), x)
    x[rng.random((R, C)) < 0.05] = 0
    x[:, :C // 3:7] *= 1e-30
    return mx.bf16(x).astype(np.float64) if dtype == "bf16" else np.float32(x).astype(np.float64)


SHAPES = [(1, 1), (1, 32), (3, 33), (2, 255), (5, 257), (1, 4096), (33, 512), (64, 513), (100, 1000), (257, 1025),
          (513, 70), (1500, 31), (1023, 300)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_quant_equals_the_oracle_bit_by_bit(ctx, shape, dtype):
    R, C = shape
    _say("quant", R, C, dtype)
    x = _values(np.random.default_rng(R * 7919 + C), R, C, dtype)
    dx = _up(ctx, x, dtype)
    q, t = _packed(ctx, R, C), _packed(ctx, C, R)
    q1, t1 = _packed(ctx, R, C), _packed(ctx, C, R)
    ctx.quant_mxfp4(dx, R, C, *q, *t, dtype=DT[dtype])       # both axes in one call
    ctx.quant_mxfp4(dx, R, C, *q1, dtype=DT[dtype])          # each alone
    ctx.quant_mxfp4(dx, R, C, None, None, *t1, dtype=DT[dtype])
    ctx.wait(60_000)
    for bufs, want in ((q, mx.pack(x)), (q1, mx.pack(x)), (t, mx.pack(x.T)), (t1, mx.pack(x.T))):
        for b, w in zip(bufs, want):
            got = ctx.download(b)
            assert np.array_equal(got, w), int(np.count_nonzero(got != w))
    for out in ("f32", "bf16"):
        dy = ctx.empty((R, C), np.float32 if out == "f32" else np.uint16)
        ctx.dequant_mxfp4(*q, dy, R, C, dtype=DT[out])
        ctx.wait(60_000)
        assert np.array_equal(_down(ctx, dy, out, (R, C)), mx.values(*mx.pack(x), C))
        dy.free()
    for b in (dx, *q, *t, *q1, *t1):
        b.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quant_strides_and_element_alignment(ctx, dtype):
    R, C, ld, off = 70, 301, 333, 1
    _say("quant strided", dtype)
    rng = np.random.default_rng(5)
    flat = _values(rng, 1, off + R * ld, dtype)[0]
    x = np.stack([flat[off + r * ld: off + r * ld + C] for r in range(R)])
    buf = _up(ctx, flat, dtype)
    esize = 2 if dtype == "bf16" else 4
    q, t = _packed(ctx, R, C), _packed(ctx, C, R)
    ctx.quant_mxfp4(buf.ptr + off * esize, R, C, *q, *t, dtype=DT[dtype], ldx=ld)
    out = _up(ctx, np.full(off + R * ld, 7.0), dtype)
    ctx.dequant_mxfp4(*q, out.ptr + off * esize, R, C, dtype=DT[dtype], ldy=ld)
    ctx.wait(60_000)
    for bufs, want in ((q, mx.pack(x)), (t, mx.pack(x.T))):
        for b, w in zip(bufs, want):
            assert np.array_equal(ctx.download(b), w)
    got = _down(ctx, out, dtype, (off + R * ld,))
    want = np.full(off + R * ld, 7.0)
    for r in range(R):
        want[off + r * ld: off + r * ld + C] = mx.values(*mx.pack(x), C)[r]
    assert np.array_equal(got, want)  # nothing between the rows was written
    for b in (buf, out, *q, *t):
        b.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quant_extremes(ctx, dtype):
    """Infinities, NaN, the largest and the smallest values, along both axes."""
    _say("quant extremes", dtype)
    x = np.zeros((64, 128))
    big, tiny = (3.38953139e38, 2.0**-133) if dtype == "bf16" else (3.4028234e38, 2.0**-149)
    x[0, :4] = [big, -big, big / 2, 1]
    x[1, 5], x[2, 40], x[3, 70] = np.inf, -np.inf, np.nan
    x[4, :3] = [tiny, -tiny, 3 * tiny]
    x[5, 64:67] = [2.0**-126, 2.0**-127, -2.0**-125]
    x[6, 32:35] = [2.0**-124, 2.0**-125, 2.0**-123]
    x = np.float32(x).astype(np.float64)
    dx = _up(ctx, x, dtype)
    q, t = _packed(ctx, 64, 128), _packed(ctx, 128, 64)
    ctx.quant_mxfp4(dx, 64, 128, *q, *t, dtype=DT[dtype])
    dy = ctx.empty((64, 128), np.float32)
    ctx.dequant_mxfp4(*q, dy, 64, 128, dtype=mi.F32)
    ctx.wait(60_000)
    for bufs, src in ((q, x), (t, x.T)):
        Q, S = mx.pack(src)
        gq, gs = ctx.download(bufs[0]), ctx.download(bufs[1])
        assert np.array_equal(gs, S)
        rows, cols = src.shape
        assert np.array_equal(mx.values(gq, gs, cols), mx.values(Q, S, cols), equal_nan=True)
    assert np.array_equal(ctx.download(dy), np.float32(mx.values(*mx.pack(x), 128)), equal_nan=True)
    for b in (dx, dy, *q, *t):
        b.free()


def _operand(rng, R, K, spread=1, step=None):
    """A random packed matrix: every code, scale bytes around 127."""
    x = rng.standard_normal((R, K)) * np.exp2(rng.integers(-spread, spread + 1, (R, (K + 31) // 32)).repeat(32, 1)[:, :K])
    return mx.pack(x)


def _smallest_scale(P, K):
    """Per row, of the blocks that hold anything."""
    s = mx.block_scales(P[1])[:, :(K + 31) // 32].astype(np.float64)
    return np.exp2(np.where(s > 0, s, 254).min(1) - 127)


# products of one row to many, of a few k to many, of one column to many, even and odd
GEMMS = [(1, 1, 1), (1, 16, 32), (1, 4096, 512), (1, 333, 11008), (3, 17, 255), (8, 4096, 1024), (16, 48, 257),
         (17, 65, 513), (33, 100, 768), (64, 512, 2048), (65, 31, 4096), (100, 1000, 300), (128, 128, 256),
         (129, 257, 1025), (256, 256, 512), (257, 300, 1280), (300, 513, 2304), (512, 640, 256), (700, 1100, 1111),
         (1024, 1024, 1024)]


@pytest.fixture()
def cus(ctx, request):
    """Products planned for that many CUs: few tiles are then many."""
    was = ctx.plan_set_cus(request.param)
    yield request.param
    ctx.plan_set_cus(was)


# k of 1 to 9 groups of 512 columns and a half, in whole and odd numbers of pairs of k-tiles, on every tile
GEMMS += [(260, 130, 256 * i) for i in (3, 4, 5, 6, 7, 8, 9, 11, 18)]


@pytest.mark.parametrize("cus", [256, 8, 1], indirect=True)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", GEMMS)
def test_gemm(ctx, shape, dtype, cus):
    M, N, K = shape
    _say("gemm", M, N, K, dtype, "cus", cus)
    rng = np.random.default_rng(M * 31 + N * 7 + K)
    A, B = _operand(rng, M, K, 12), _operand(rng, N, K, 12)
    a, b = mx.values(*A, K), mx.values(*B, K)
    want, bound = a @ b.T, mx.product_bound(a, b)
    if dtype == "bf16":
        bound = bound + 2.0**-8 * np.abs(want)
    dA, dB = [ctx.upload(v) for v in A], [ctx.upload(v) for v in B]
    ldc = N + 3
    C = _up(ctx, np.full((M, ldc), -7.0), dtype)
    for ld in (ldc, N):
        ctx.gemm_mxfp4(*dA, *dB, C, M, N, K, dtype=DT[dtype], ldc=ld)
        ctx.wait(60_000)
        flat = _down(ctx, C, dtype, (M * ldc,)).astype(np.float64)
        got = flat[:M * ld].reshape(M, ld)
        assert (np.abs(got[:, :N] - want) <= bound).all(), float((np.abs(got[:, :N] - want) / (bound + 1e-300)).max())
        if ld == ldc:
            assert (got[:, N:] == -7).all()  # nothing between the rows was written
    for x in (*dA, *dB, C):
        x.free()


@pytest.mark.parametrize("cus", [256, 8, 1], indirect=True)
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 96, 300), (3, 33, 64), (16, 255, 512), (17, 257, 1024), (40, 11008, 256),
                                   (70, 513, 2048), (129, 1000, 257), (256, 512, 768), (300, 800, 513), (513, 1025, 1024)])
def test_packed_product_bit_by_bit(ctx, shape, relu, cus):
    M, N, K = shape
    _say("gemm_rq", M, N, K, relu, "cus", cus)
    rng = np.random.default_rng(M + N + K)
    A, B = _operand(rng, M, K), _operand(rng, N, K)
    a, b = mx.values(*A, K), mx.values(*B, K)
    c = a @ b.T
    want = mx.pack(np.maximum(c, 0) if relu else c)
    # columns whose partial sums fp32 holds exactly: multiples of a quarter of the smallest scales' product, below
    # 2^24 of them (not so where the last block is one small value); the others may round to the code beside
    unit = 0.25 * np.outer(_smallest_scale(A, K), _smallest_scale(B, K))
    holds = np.abs(a) @ np.abs(b).T < 2.0**24 * unit
    held = np.pad(holds, ((0, 0), (0, -N % 512)), constant_values=True).reshape(M, -1, 32).all(-1)
    assert held.mean() > 0.5
    dA, dB = [ctx.upload(v) for v in A], [ctx.upload(v) for v in B]
    y = _packed(ctx, M, N)
    ctx.gemm_mxfp4_rq(*dA, *dB, *y, M, N, K, relu=relu)
    ctx.wait(60_000)
    gs, gq = ctx.download(y[1]), ctx.download(y[0])
    s, t = mx.block_scales(gs), mx.block_scales(want[1])
    assert np.array_equal(s[held], t[held]) and (np.abs(s.astype(int) - t) <= 1).all()
    # (a sum that is zero may carry either sign: compared as values, and the padding as bytes)
    off = np.abs(mx.values(gq, gs, N) - mx.values(*want, N))
    step = np.where(held, 0, 2.0 * np.exp2(np.maximum(s, t).astype(np.float64) - 127)).repeat(32, 1)[:, :N]
    assert (off <= step).all()
    assert not gq[:, (N + 1) // 2:].any()
    for x in (*dA, *dB, *y):
        x.free()


def test_nan_scales_and_overflow_stay_in_their_rows(ctx):
    M, N, K = 40, 70, 600
    _say("gemm nan")
    rng = np.random.default_rng(3)
    xa, xb = rng.standard_normal((M, K)), rng.standard_normal((N, K))
    xa[7, 100], xb[65, 599], xa[9, :] = np.nan, np.inf, 0
    A, B = mx.pack(xa), mx.pack(xb)
    a, b = mx.values(*A, K), mx.values(*B, K)
    dA, dB = [ctx.upload(v) for v in A], [ctx.upload(v) for v in B]
    C, y = ctx.empty((M, N), np.float32), _packed(ctx, M, N)
    ctx.gemm_mxfp4(*dA, *dB, C, M, N, K)
    ctx.gemm_mxfp4_rq(*dA, *dB, *y, M, N, K, relu=True)
    ctx.wait(60_000)
    got = ctx.download(C)
    want_nan = np.zeros((M, N), bool)
    want_nan[7, :] = want_nan[:, 65] = True
    assert np.array_equal(np.isnan(got), want_nan)
    rows, cols = np.delete(np.arange(M), 7), np.delete(np.arange(N), 65)
    i = np.ix_(rows, cols)
    assert (np.abs(got[i] - a[rows] @ b[cols].T) <= mx.product_bound(a[rows], b[cols])).all()
    assert (got[9, cols] == 0).all()
    # packed: the NaN row and, elsewhere, the block of columns that holds column 65
    s = mx.block_scales(ctx.download(y[1]))
    nan = np.zeros((M, 16), bool)
    nan[7, :3] = nan[:, 2] = True
    assert np.array_equal(s == 255, nan)
    for x in (*dA, *dB, C, *y):
        x.free()


@pytest.mark.parametrize("shape", [(1, 64, 96, 32), (5, 300, 513, 77), (40, 256, 1100, 128), (300, 512, 768, 300)])
def test_mlp_is_its_two_products(ctx, shape):
    M, K, F, N = shape
    _say("mlp", shape)
    rng = np.random.default_rng(M)
    X, W1, W2 = _operand(rng, M, K), _operand(rng, F, K), _operand(rng, N, F)
    h = mx.pack(np.maximum(mx.values(*X, K) @ mx.values(*W1, K).T, 0))
    hv, w2 = mx.values(*h, F), mx.values(*W2, F)
    bufs = [ctx.upload(v) for m in (X, W1, W2) for v in m]
    H, Y = _packed(ctx, M, F), ctx.empty((M, N), np.float32)
    ctx.mlp_mxfp4(*bufs, *H, Y, M, K, F, N, dtype=mi.F32)
    ctx.wait(60_000)
    assert np.array_equal(mx.values(ctx.download(H[0]), ctx.download(H[1]), F), hv)
    assert (np.abs(ctx.download(Y) - hv @ w2.T) <= mx.product_bound(hv, w2)).all()
    for x in (*bufs, *H, Y):
        x.free()


def test_gradients_of_a_linear_layer(ctx):
    """Y = X W^T with each operand rounded along the axis its product contracts: dX = dY W and dW = dY^T X
    from packed transposes, against the formulas and against differences of the (rounded) products."""
    M, N, K = 70, 90, 130
    _say("linear gradients")
    rng = np.random.default_rng(9)
    X, W, dY = (np.float32(rng.standard_normal(s)).astype(np.float64) for s in ((M, K), (N, K), (M, N)))
    dx, dw, dy = (ctx.upload(np.float32(v)) for v in (X, W, dY))
    xt, wt, yq, yt = _packed(ctx, K, M), _packed(ctx, K, N), _packed(ctx, M, N), _packed(ctx, N, M)
    ctx.quant_mxfp4(dx, M, K, None, None, *xt, dtype=mi.F32)
    ctx.quant_mxfp4(dw, N, K, None, None, *wt, dtype=mi.F32)
    ctx.quant_mxfp4(dy, M, N, *yq, *yt, dtype=mi.F32)
    gX, gW = ctx.empty((M, K), np.float32), ctx.empty((N, K), np.float32)
    ctx.gemm_mxfp4(*yq, *wt, gX, M, K, N)
    ctx.gemm_mxfp4(*yt, *xt, gW, N, K, M)
    ctx.wait(60_000)
    r = {n: mx.values(*mx.pack(v), v.shape[1]) for n, v in (("yq", dY), ("yt", dY.T), ("xt", X.T), ("wt", W.T))}
    for got, a, b in ((gX, r["yq"], r["wt"]), (gW, r["yt"], r["xt"])):
        assert (np.abs(ctx.download(got) - a @ b.T) <= mx.product_bound(a, b)).all()
    # differences: L = sum(dY . (X W^T)) with the rounded dY and W is linear in X, so a unit step has no error
    for i, k in ((0, 0), (69, 129), (33, 64)):
        step = np.zeros((M, K))
        step[i, k] = 1
        d = (r["yq"] * ((X + step) @ r["wt"])).sum() - (r["yq"] * (X @ r["wt"])).sum()
        assert abs(ctx.download(gX)[i, k] - d) <= mx.product_bound(r["yq"], r["wt"])[i, k] + 1e-9
    for x in (dx, dw, dy, *xt, *wt, *yq, *yt, gX, gW):
        x.free()


def test_graph_replays(ctx):
    """Quantise + product recorded once, replayed on new contents, with eager work in between."""
    M, K, N = 5, 700, 300
    _say("graph")
    rng = np.random.default_rng(4)
    W = _operand(rng, N, K)
    dW = [ctx.upload(v) for v in W]
    dX, q, C = ctx.empty((M, K), np.float32), _packed(ctx, M, K), ctx.empty((M, N), np.float32)
    ctx.wait(60_000)
    with ctx.record() as g:
        ctx.quant_mxfp4(dX, M, K, *q, dtype=mi.F32)
        ctx.gemm_mxfp4(*q, *dW, C, M, N, K)
    for i in range(4):
        x = np.float32(rng.standard_normal((M, K)))
        ctx.copy_h2d(dX, x)
        g.launch()
        ctx.wait(60_000)
        got = ctx.download(C)
        ctx.quant_mxfp4(dX, M, K, *q, dtype=mi.F32)
        ctx.gemm_mxfp4(*q, *dW, C, M, N, K)
        ctx.wait(60_000)
        assert np.array_equal(got, ctx.download(C))
        a, b = mx.values(*mx.pack(x), K), mx.values(*W, K)
        assert (np.abs(got - a @ b.T) <= mx.product_bound(a, b)).all()
    g.destroy()
    for x in (*dW, dX, *q, C):
        x.free()


def test_refusals(ctx):
    d = ctx.empty((1 << 16,), np.uint8)
    p = d.ptr

    def refused(name, *args, text):
        assert ctx.call_status(name, *args) == mi.MIAIE_EINVAL, (name, args)
        assert text in ctx.last_error(), ctx.last_error()

    q = "miaie_quant_mxfp4"
    refused(q, None, 0, 4, 4, 4, p, p, None, None, text="X is NULL")
    refused(q, p, 2, 4, 4, 4, p, p, None, None, text="dtype=2")
    refused(q, p, 0, 0, 4, 4, p, p, None, None, text="R=0")
    refused(q, p, 0, 4, -1, 4, p, p, None, None, text="C=-1")
    refused(q, p, 0, 4, 4, 3, p, p, None, None, text="ldx=3")
    refused(q, p + 2, 0, 4, 4, 4, p, p, None, None, text="misaligned")
    refused(q, p + 1, 1, 4, 4, 4, p, p, None, None, text="misaligned")
    refused(q, p, 0, 4, 4, 4, None, None, None, None, text="all NULL")
    refused(q, p, 0, 4, 4, 4, p, None, None, None, text="Xs is NULL")
    refused(q, p, 0, 4, 4, 4, None, None, None, p, text="Xtq is NULL")
    refused(q, p, 0, 4, 4, 4, p + 8, p, None, None, text="16-byte aligned")
    refused(q, p, 0, 1 << 30, 4, 4, p, p, None, None, text="too large")
    refused(q, p, 0, 4, 1 << 30, 1 << 30, None, None, p, p, text="too large")
    dq = "miaie_dequant_mxfp4"
    refused(dq, p, p, None, 0, 4, 4, 4, text="Y is NULL")
    refused(dq, p, p, p, 3, 4, 4, 4, text="dtype=3")
    refused(dq, p, None, p, 0, 4, 4, 4, text="Xs is NULL")
    refused(dq, p, p, p, 0, 4, 4, 2, text="ldy=2")
    g = "miaie_gemm_mxfp4"
    refused(g, p, p, p, p, None, 0, 4, 4, 4, 4, text="C is NULL")
    refused(g, p, p, p, p, p, 0, 4, 4, 0, 4, text="K=0")
    refused(g, p, p, p, p, p, 0, 4, 4, 4, 3, text="ldc=3")
    refused(g, p, p, None, p, p, 0, 4, 4, 4, 4, text="Bq is NULL")
    refused(g, p, p + 4, p, p, p, 0, 4, 4, 4, 4, text="16-byte aligned")
    refused(g, p, p, p, p, p + 2, 0, 4, 4, 4, 4, text="misaligned")
    r = "miaie_gemm_mxfp4_rq"
    refused(r, p, p, p, p, p, None, 4, 4, 4, 0, text="Ys is NULL")
    refused(r, p, p, p, p, p, p, 4, 4, 4, 2, text="relu=2")
    m = "miaie_mlp_mxfp4"
    refused(m, *[p] * 6, None, p, p, 0, 4, 4, 4, 4, 4, text="Hq is NULL")
    refused(m, *[p] * 9, 0, 4, 4, 0, 4, 4, text="F=0")
    refused(m, *[p] * 9, 5, 4, 4, 4, 4, 4, text="dtype=5")
    ctx.wait(10_000)
    d.free()


def test_two_streams_share_nothing(ctx):
    """Contexts on two streams, their calls interleaved without waiting: no call uses memory of the library's."""
    M, K, N = 16, 2048, 512
    _say("two streams")
    rng = np.random.default_rng(6)
    ctxs = [ctx, mi.Context(0)]
    try:
        work = []
        for c in ctxs:
            A, B = _operand(rng, M, K), _operand(rng, N, K)
            bufs = [c.upload(v) for v in (*A, *B)]
            outs = [c.empty((M, N), np.float32) for _ in range(4)]
            c.wait(60_000)
            work.append((c, mx.values(*A, K), mx.values(*B, K), bufs, outs))
        for i in range(4):
            for c, _, _, bufs, outs in work:
                c.gemm_mxfp4(*bufs, outs[i], M, N, K)
        for c, a, b, bufs, outs in work:
            c.wait(60_000)
            for o in outs:
                assert (np.abs(c.download(o) - a @ b.T) <= mx.product_bound(a, b)).all()
            for x in (*bufs, *outs):
                x.free()
    finally:
        ctxs[1].close()


def test_captured_by_the_caller():
    """A caller's own HIP graph of a block's calls, replayed on another stream beside eager calls of the context,
    every replay against the eager result."""
    from hip_capture import Capture

    _say("caller's capture")
    cap = Capture()
    try:
        c = cap.ctx
        M, K, F = 12, 300, 700
        rng = np.random.default_rng(11)
        W1, W2 = _operand(rng, F, K), _operand(rng, K, F)
        w = [c.upload(v) for v in (*W1, *W2)]
        X, wn = c.empty((M, K), np.float32), c.upload(np.float32(1 + 0.1 * rng.standard_normal(K)))
        q, h = _packed(c, M, K), _packed(c, M, F)
        b, out, y, rstd = (c.empty(s, np.float32) for s in ((M, K), (M, K), (M, K), (2, M)))
        dw, work = [c.empty((K,), np.float32) for _ in range(2)], c.empty((1024 * K,), np.float32)
        dx, db = c.empty((M, K), np.float32), c.empty((M, K), np.float32)
        kw = {"stream_dtype": mi.F32, "branch_dtype": mi.F32}

        def block():
            c.quant_mxfp4(X, M, K, *q, dtype=mi.F32)
            c.mlp_mxfp4(*q, *w, *h, b, M, K, F, K, dtype=mi.F32)
            c.norm_block(X, b, None, wn, wn, out, y, rstd, M, K, **kw)
            c.norm_block_grad(out, b, None, wn, wn, rstd, X, b, dx, db, None, *dw, work, mi.norm_work_bytes(K), M, K, **kw)

        results = (out, y, dx, db, *dw)
        exe, grids = cap.record(block)
        assert len(grids) == 6  # conversion, two products, norms, their gradient and the sums of its parts
        for i in range(4):
            x = np.float32(rng.standard_normal((M, K)))
            c.copy_h2d(X, x)
            cap.sync()
            cap.replay(exe)
            cap.sync()
            got = [c.download(r) for r in results]
            block()
            cap.sync()
            for g, r in zip(got, results):
                assert np.array_equal(g, c.download(r)), i
            v = mx.values(*mx.pack(x), K)
            hv = mx.values(*mx.pack(np.maximum(v @ mx.values(*W1, K).T, 0)), F)
            want = hv @ mx.values(*W2, F).T
            assert np.abs(c.download(b) - want).max() <= 0.02 * np.abs(want).max()  # (a code of h may round the other way)
        cap.ok(cap.hip.hipGraphExecDestroy(exe))
        for t in (*w, X, wn, *q, *h, b, out, y, rstd, *dw, work, dx, db):
            t.free()
    finally:
        cap.close()
