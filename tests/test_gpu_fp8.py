"""8-bit floating point conversion and products through the C ABI against the
64-bit oracle (tests/fp8_oracle.py).

Conversions are exact: codes, scales and padding are compared bit by bit.  Products
of operands whose sums fp32 holds exactly are, too; others may be off by
fp8_oracle.product_bound, bf16 results by half a unit in the last place more (2^-8
of the value)."""
import numpy as np
import pytest

import aiehlc_amd as mi
import fp8_oracle as fp8

pytestmark = pytest.mark.gpu

DT = {"f32": mi.F32, "bf16": mi.BF16}


def _say(*a):
    print("[case]", *a, flush=True)


def _up(ctx, x, dtype):
    return ctx.upload(fp8.bf16_bits(x) if dtype == "bf16" else np.asarray(x, np.float32))


def _down(ctx, buf, dtype, shape):
    if dtype == "bf16":
        return fp8.from_bf16_bits(ctx.download(buf, np.uint16, shape))
    return ctx.download(buf, np.float32, shape)


def _packed(ctx, rows, cols, block=1):
    """Buffers of a packed matrix, full of a pattern that a kernel has to overwrite."""
    q, s = mi.fp8_shapes(rows, cols, block)
    return ctx.upload(np.full(q, 0xA5, np.uint8)), ctx.upload(np.full(s, -7.0, np.float32))


def _values(rng, R, C, dtype, spread=20):
    """Values of many sizes, with blocks of zeros, single large values, ties between codes and tiny ones."""
    x = rng.standard_normal((R, C)) * np.exp2(rng.integers(-spread, spread + 1, (R, (C + 63) // 64)).repeat(64, 1)[:, :C])
    ties = rng.random((R, C)) < 0.2
    x = np.where(ties, rng.choice([17, 19, 21, 27, 34, 38, 2.125, -2.125, 448, 449, 464, -432, 0, -0.0], (R, C)), x)
    x[rng.random((R, C)) < 0.05] = 0
    x[:, :C // 3:7] *= 1e-30
    if R > 2:
        x[R // 2] = 0
    return fp8.bf16(x).astype(np.float64) if dtype == "bf16" else np.float32(x).astype(np.float64)


def _same(ctx, bufs, want):
    for b, w in zip(bufs, want):
        got = ctx.download(b)
        assert np.array_equal(got, w, equal_nan=got.dtype.kind == "f"), int(np.count_nonzero(got != w))


SHAPES = [(1, 1), (1, 128), (3, 33), (2, 255), (5, 257), (1, 4096), (33, 512), (127, 129), (128, 128), (129, 1000),
          (513, 70), (1500, 31), (1023, 300)]


@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_quant_equals_the_oracle_bit_by_bit(ctx, shape, dtype, block):
    R, C = shape
    _say("quant", R, C, dtype, block)
    x = _values(np.random.default_rng(R * 7919 + C), R, C, dtype)
    dx = _up(ctx, x, dtype)
    q, t, q1, t1 = (_packed(ctx, *s, block) for s in ((R, C), (C, R), (R, C), (C, R)))
    kw = {"block": block, "dtype": DT[dtype]}
    ctx.quant_fp8(dx, R, C, *q, *t, **kw)  # both axes in one call
    ctx.quant_fp8(dx, R, C, *q1, **kw)     # each alone
    ctx.quant_fp8(dx, R, C, None, None, *t1, **kw)
    ctx.wait(60_000)
    rows, cols = fp8.pack(x, block), fp8.pack(x.T, block)
    for bufs, want in ((q, rows), (q1, rows), (t, cols), (t1, cols)):
        _same(ctx, bufs, want)
    for out in ("f32", "bf16"):
        dy = ctx.empty((R, C), np.float32 if out == "f32" else np.uint16)
        ctx.dequant_fp8(*q, dy, R, C, block=block, dtype=DT[out])
        ctx.wait(60_000)
        want = fp8.values(*rows, R, C, block)
        assert np.array_equal(_down(ctx, dy, out, (R, C)), fp8.bf16(want) if out == "bf16" else want.astype(np.float32))
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
    ctx.quant_fp8(buf.ptr + off * esize, R, C, *q, *t, dtype=DT[dtype], ldx=ld)
    out = _up(ctx, np.full(off + R * ld, 7.0), dtype)
    ctx.dequant_fp8(*q, out.ptr + off * esize, R, C, dtype=DT[dtype], ldy=ld)
    ctx.wait(60_000)
    _same(ctx, q, fp8.pack(x))
    _same(ctx, t, fp8.pack(x.T))
    got = _down(ctx, out, dtype, (off + R * ld,))
    want, v = np.full(off + R * ld, 7.0), fp8.rounded(x)
    for r in range(R):
        want[off + r * ld: off + r * ld + C] = fp8.bf16(v[r]) if dtype == "bf16" else v[r]
    assert np.array_equal(got, want.astype(np.float32))  # nothing between the rows was written
    for b in (buf, out, *q, *t):
        b.free()


@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quant_extremes(ctx, dtype, block):
    """Infinities, NaN, the largest and the smallest values, along both axes."""
    _say("quant extremes", dtype, block)
    R, C = 260, 600
    x = np.zeros((R, C))
    big, tiny = (3.38953139e38, 2.0**-133) if dtype == "bf16" else (3.4028234e38, 2.0**-149)
    x[0, :4] = [big, -big, big / 2, 1]
    x[1, 130], x[2, 260], x[130, 400] = np.inf, -np.inf, np.nan
    x[4, 129:132] = [tiny, -tiny, 3 * tiny]
    x[200, 513:516] = [2.0**-126, 2.0**-127, -2.0**-125]
    x[201, 512:515] = [448 * 2.0**-126, 2.0**-126, 449 * 2.0**-126]
    x = np.float32(x).astype(np.float64)
    dx = _up(ctx, x, dtype)
    q, t = _packed(ctx, R, C, block), _packed(ctx, C, R, block)
    ctx.quant_fp8(dx, R, C, *q, *t, block=block, dtype=DT[dtype])
    y = ctx.empty((R, C), np.float32)
    ctx.dequant_fp8(*q, y, R, C, block=block, dtype=mi.F32)
    ctx.wait(60_000)
    stored = fp8.bf16(x).astype(np.float64) if dtype == "bf16" else x
    for bufs, m in ((q, stored), (t, stored.T)):
        Q, S = fp8.pack(m, block)
        assert np.array_equal(ctx.download(bufs[1]), S, equal_nan=True)
        finite = np.isfinite(fp8.spread(S, *Q.shape, block))  # (codes of a block of NaN are not specified)
        assert np.array_equal(ctx.download(bufs[0])[finite], Q[finite])
    assert np.array_equal(ctx.download(y), fp8.values(*fp8.pack(stored, block), R, C, block).astype(np.float32), equal_nan=True)
    for b in (dx, y, *q, *t):
        b.free()


def _operands(rng, M, N, K, b_block, exact=False):
    """A packed by the library's rule; B too, or weights with any scales.  exact: elements 0 to 3 in halves, scales
    that are powers of two near each other: every sum is a multiple of 2^-6 below 9 K 2^4 <= 2^18 (K <= 1820); beyond
    that sums of random signs stay below it."""
    if exact:
        pA, pB = ((fp8.encode(rng.integers(-6, 7, (n, fp8.up(K))) / 2 * (np.arange(fp8.up(K)) < K)),
                   np.exp2(rng.integers(-2, 3, (fp8.up(K) // 128, -(-n // b)))).astype(np.float32))
                  for n, b in ((M, 1), (N, b_block)))
        return pA, pB
    A, B = rng.standard_normal((M, K)), rng.standard_normal((N, K))
    A *= np.exp2(rng.integers(-3, 4, (M, (K + 127) // 128)).repeat(128, 1)[:, :K])
    pA, pB = fp8.pack(A), fp8.pack(B, b_block)
    if b_block == 128:
        pB = pB[0], (pB[1] * rng.uniform(0.4, 1.9, pB[1].shape)).astype(np.float32)
    return pA, pB


GEMMS = [(1, 1, 1), (1, 33, 300), (4, 16, 128), (16, 48, 256), (17, 40, 129), (7, 777, 1000), (15, 64, 4100), (64, 64, 512),
         (33, 129, 640), (130, 260, 384), (333, 777, 1000), (256, 256, 128), (129, 385, 1), (100, 100, 2049)]


@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("b_block", [1, 128])
@pytest.mark.parametrize("shape", GEMMS)
def test_gemm(ctx, shape, b_block, exact):
    M, N, K = shape
    _say("gemm", M, N, K, b_block, "exact" if exact else "")
    rng = np.random.default_rng(M * 31 + N * 7 + K + b_block)
    pA, pB = _operands(rng, M, N, K, b_block, exact)
    a, b = fp8.values(*pA, M, K), fp8.values(*pB, N, K, b_block)
    want, bound = a @ b.T, 0 if exact else fp8.product_bound(a, b)
    dA, dB = [ctx.upload(v) for v in pA], [ctx.upload(v) for v in pB]
    for dtype, ldc in (("f32", N), ("bf16", N), ("f32", N + 3), ("bf16", N + 5)):
        C = _up(ctx, np.full(M * ldc + 1, 7.0), dtype)
        esize = 2 if dtype == "bf16" else 4
        ctx.gemm_fp8(*dA, *dB, C.ptr + esize, M, N, K, b_block=b_block, dtype=DT[dtype], ldc=ldc)
        ctx.wait(60_000)
        flat = _down(ctx, C, dtype, (M * ldc + 1,))
        got = flat[1:].reshape(M, ldc)
        off = np.abs(got[:, :N] - want) - bound - (2.0**-8 * np.abs(want) if dtype == "bf16" else 0)
        assert (off <= 0).all(), (dtype, ldc, off.max())
        assert flat[0] == 7 and (got[:, N:] == 7).all()
        C.free()
    for b_ in (*dA, *dB):
        b_.free()


# large enough for 256 x 256 tiles, with each number of steps around the stages of LDS
LARGE = [(2049, 4100, 300, 128), (2048, 4096, 128, 128), (4096, 2048, 256, 1), (2560, 3333, 385, 1), (1999, 4096, 1100, 128)]


@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("M, N, K, b_block", LARGE)
def test_gemm_of_many_tiles(ctx, M, N, K, b_block, exact):
    _say("gemm", M, N, K, b_block, "exact" if exact else "")
    rng = np.random.default_rng(K)
    pA, pB = _operands(rng, M, N, K, b_block, exact)
    a, b = fp8.values(*pA, M, K), fp8.values(*pB, N, K, b_block)
    want, bound = a @ b.T, 0 if exact else fp8.product_bound(a, b)
    dA, dB = [ctx.upload(v) for v in pA], [ctx.upload(v) for v in pB]
    for dtype in ("f32", "bf16"):
        C = ctx.upload(np.full((M, N), 7, np.float32 if dtype == "f32" else np.uint16))
        ctx.gemm_fp8(*dA, *dB, C, M, N, K, b_block=b_block, dtype=DT[dtype])
        ctx.wait(60_000)
        off = np.abs(_down(ctx, C, dtype, (M, N)) - want) - bound - (2.0**-8 * np.abs(want) if dtype == "bf16" else 0)
        assert (off <= 0).all(), (dtype, off.max())
        C.free()
    for b_ in (*dA, *dB):
        b_.free()


@pytest.mark.parametrize("b_block", [1, 128])
@pytest.mark.parametrize("shape", [(5, 40, 600), (200, 300, 600)])
def test_gemm_nan_scales(ctx, shape, b_block):
    """A block of NaN in A makes its rows NaN, one in B its columns, and nothing else."""
    M, N, K = shape
    _say("gemm NaN", shape, b_block)
    pA, pB = _operands(np.random.default_rng(3), M, N, K, b_block)
    pA[1][2, 3] = np.nan
    pB[1][1, N // 2 // b_block] = np.nan
    rows, cols = np.zeros(M, bool), np.zeros(N, bool)
    rows[3] = True
    at = N // 2 // b_block * b_block
    cols[at:at + b_block] = True
    dA, dB, C = [ctx.upload(v) for v in pA], [ctx.upload(v) for v in pB], ctx.empty((M, N), np.float32)
    ctx.gemm_fp8(*dA, *dB, C, M, N, K, b_block=b_block)
    ctx.wait(60_000)
    assert np.array_equal(np.isnan(ctx.download(C)), rows[:, None] | cols[None])
    for b_ in (*dA, *dB, C):
        b_.free()


def test_linear_layer_and_its_gradients(ctx):
    """Forward, dX and dW of Y = X . W^T, every operand packed by the library, through one chain."""
    M, N, K = 200, 300, 520
    _say("linear layer")
    rng = np.random.default_rng(11)
    X, W, dY = (fp8.bf16(rng.standard_normal(s)).astype(np.float64) for s in ((M, K), (N, K), (M, N)))
    d = [_up(ctx, v, "bf16") for v in (X, W, dY)]
    xq, xt, wq, wt, yq, yt = (_packed(ctx, *s) for s in
                              ((M, K, 1), (K, M, 1), (N, K, 128), (K, N, 128), (M, N, 1), (N, M, 1)))
    Y, dX, dW = ctx.empty((M, N), np.float32), ctx.empty((M, K), np.float32), ctx.empty((N, K), np.float32)
    ctx.quant_fp8(d[0], M, K, *xq, *xt)
    ctx.quant_fp8(d[1], N, K, *wq, *wt, block=128)
    ctx.quant_fp8(d[2], M, N, *yq, *yt)
    ctx.gemm_fp8(*xq, *wq, Y, M, N, K)
    ctx.gemm_fp8(*yq, *wt, dX, M, K, N)
    ctx.gemm_fp8(*yt, *xt, dW, N, K, M, b_block=1)
    ctx.wait(60_000)
    for got, a, b in ((Y, fp8.rounded(X), fp8.rounded(W, 128)), (dX, fp8.rounded(dY), fp8.rounded(W.T, 128)),
                      (dW, fp8.rounded(dY.T), fp8.rounded(X.T))):
        assert (np.abs(ctx.download(got) - a @ b.T) <= fp8.product_bound(a, b)).all()
    for b_ in (*d, *xq, *xt, *wq, *wt, *yq, *yt, Y, dX, dW):
        b_.free()
