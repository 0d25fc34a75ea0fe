"""The MXFP4 products' tiles (aiehlc_amd/csrc/gemm_mxfp4.hip) that the shapes of
tests/test_gpu_mxfp4.py do not reach; tests/test_mx_plan.py checks that the two
lists together reach every kernel.  Tolerances and comparisons are that file's."""
import numpy as np
import pytest

import aiehlc_amd as mi
import mx_oracle as mx
from test_gpu_mxfp4 import _down, _operand, _packed, _say, _smallest_scale, _up

pytestmark = pytest.mark.gpu


def test_mlp_refuses_both_products_before_the_first(ctx):
    """The second product of this MLP has 2^24 tiles of 256 x 256, more than a launch takes: nothing is queued."""
    d = ctx.empty((1 << 16,), np.uint8)
    p = d.ptr
    for dtype in (mi.F32, mi.BF16):
        rc = ctx.call_status("miaie_mlp_mxfp4", *[p] * 9, dtype, 1 << 20, 1, 1, 1 << 20, 1 << 20)
        assert rc == mi.MIAIE_EINVAL and "too large" in ctx.last_error(), ctx.last_error()
    ctx.wait(10_000)
    d.free()


# (out, M, N, K, CUs planned for): ragged rows and columns, k in whole and odd numbers of pairs of k-tiles before
# and after the steady loop, one tile and several, more than four rows of tiles
ROWS_16x32 = [("f32", 6, 641, 98, 4), ("f32", 8, 653, 1197, 3), ("f32", 6, 442, 1387, 8), ("bf16", 8, 603, 723, 3),
              ("bf16", 5, 620, 1066, 12), ("mx", 7, 465, 681, 16), ("mx", 8, 428, 1192, 256)]
ROWS_16x64 = [("f32", 7, 444, 1001, 4), ("f32", 11, 859, 948, 4), ("f32", 74, 168, 2172, 16), ("bf16", 7, 343, 3618, 6),
              ("bf16", 14, 251, 1093, 1), ("bf16", 10, 565, 3304, 12), ("mx", 8, 672, 904, 4), ("mx", 6, 474, 3897, 8)]
ROWS_32x16 = [("f32", 84, 73, 162, 4), ("f32", 21, 45, 1174, 3), ("f32", 112, 37, 3680, 6), ("bf16", 99, 47, 956, 12),
              ("bf16", 126, 47, 3728, 12)]
ROWS_64x32 = [("f32", 101, 95, 939, 6), ("f32", 55, 95, 3483, 3), ("f32", 128, 87, 2155, 6), ("bf16", 60, 82, 712, 3),
              ("bf16", 111, 82, 1172, 6)]
TILE_256x256 = [("f32", 132, 256, 1501, 1), ("f32", 131, 256, 1558, 1), ("f32", 130, 256, 1878, 1), ("f32", 136, 256, 2118, 1),
                ("f32", 132, 256, 2317, 1), ("f32", 132, 256, 2627, 1), ("f32", 129, 145, 1458, 1), ("f32", 132, 132, 1792, 1),
                ("f32", 140, 131, 1845, 1), ("f32", 138, 130, 2304, 1), ("f32", 135, 130, 2560, 1), ("f32", 133, 146, 2655, 1),
                ("f32", 134, 151, 3840, 1), ("f32", 1300, 1700, 2200, 6), ("bf16", 138, 130, 669, 1), ("bf16", 1157, 1281, 520, 16),
                ("mx", 151, 131, 867, 1), ("mx", 135, 138, 1280, 1), ("mx", 1411, 2177, 1100, 20)]
TILE_256x128 = [("f32", 133, 128, 4360, 1), ("f32", 134, 128, 4633, 1), ("f32", 135, 128, 4888, 1), ("f32", 129, 128, 5627, 1),
                ("f32", 130, 128, 5888, 1), ("f32", 252, 5, 4608, 1), ("f32", 673, 2, 4818, 1), ("f32", 455, 4, 5022, 2),
                ("f32", 683, 1, 5461, 3), ("f32", 606, 1, 5737, 3), ("f32", 1290, 900, 4700, 16), ("bf16", 137, 128, 1362, 1),
                ("bf16", 133, 128, 1699, 1), ("bf16", 138, 128, 1921, 1), ("bf16", 135, 128, 2154, 1), ("bf16", 132, 128, 2410, 1),
                ("bf16", 134, 128, 2726, 1), ("bf16", 239, 33, 1536, 1), ("bf16", 248, 4, 1792, 1), ("bf16", 140, 34, 1860, 1),
                ("bf16", 485, 2, 2304, 2), ("bf16", 454, 3, 2560, 2), ("bf16", 390, 2, 2816, 2), ("bf16", 1290, 900, 4700, 16),
                ("mx", 164, 1, 2048, 1), ("mx", 129, 1, 2073, 1), ("mx", 405, 1, 2456, 3), ("mx", 132, 1, 2816, 1),
                ("mx", 264, 1, 3840, 2), ("mx", 142, 1, 3891, 1), ("mx", 1290, 900, 4700, 16)]
MIXED = [("f32", 134, 896, 1026, 3), ("f32", 129, 640, 1816, 2), ("f32", 129, 640, 2090, 2), ("f32", 131, 640, 4382, 2),
         ("f32", 134, 640, 4748, 2), ("f32", 129, 640, 5120, 2), ("f32", 133, 791, 1030, 3), ("f32", 136, 775, 1296, 3),
         ("f32", 143, 804, 1606, 3), ("f32", 141, 530, 1863, 2), ("f32", 129, 543, 2204, 2), ("f32", 138, 518, 2354, 2),
         ("f32", 132, 525, 2816, 2), ("f32", 133, 563, 3776, 2), ("f32", 1300, 1700, 2200, 12), ("f32", 1290, 900, 4700, 20),
         ("bf16", 211, 1152, 1, 2), ("bf16", 131, 768, 313, 2), ("bf16", 133, 640, 522, 2), ("bf16", 142, 640, 772, 2),
         ("bf16", 137, 640, 1065, 2), ("bf16", 134, 640, 1292, 2), ("bf16", 140, 640, 1545, 2), ("bf16", 182, 1148, 1, 4),
         ("bf16", 142, 681, 260, 2), ("bf16", 130, 538, 514, 2), ("bf16", 131, 513, 1024, 2), ("bf16", 130, 575, 1062, 2),
         ("bf16", 137, 542, 1396, 2), ("bf16", 131, 520, 1792, 2), ("bf16", 136, 524, 2048, 2), ("bf16", 2500, 1100, 600, 20),
         ("bf16", 1411, 2177, 1100, 12), ("bf16", 1311, 2304, 1700, 12), ("mx", 255, 896, 1, 3), ("mx", 137, 521, 288, 2),
         ("mx", 146, 513, 517, 2), ("mx", 131, 538, 830, 2), ("mx", 132, 582, 1069, 2), ("mx", 149, 530, 1337, 2),
         ("mx", 132, 527, 1596, 2), ("mx", 129, 515, 2048, 2), ("mx", 2500, 1100, 600, 20), ("mx", 1311, 2304, 1700, 12)]
KERNELS = {(mi.KERNEL_ROWS, 16, 32): ROWS_16x32, (mi.KERNEL_ROWS, 16, 64): ROWS_16x64, (mi.KERNEL_ROWS, 32, 16): ROWS_32x16,
           (mi.KERNEL_ROWS, 64, 32): ROWS_64x32, (mi.KERNEL_PIPE, 256, 256): TILE_256x256,
           (mi.KERNEL_PIPE, 256, 128): TILE_256x128, (mi.KERNEL_PIPE_MIXED, 256, 256): MIXED}
CASES = [(k, c) for k, cases in KERNELS.items() for c in cases]
OUT = {"f32": mi.F32, "bf16": mi.BF16, "mx": mi.MXFP4}


def planned(case):
    out, M, N, K, cus = case
    p = mi.plan_gemm_mxfp4(M, N, K, OUT[out], cus)
    return p["kernel"], p["tile_m"], p["tile_n"]


@pytest.fixture()
def cus(ctx):
    """Sets the CUs that products are planned for; the device's own again afterwards."""
    was = []
    yield lambda n: was.append(ctx.plan_set_cus(n))
    if was:
        ctx.plan_set_cus(was[0])


@pytest.mark.parametrize("kernel, case", [c for c in CASES if c[1][0] != "mx"])
def test_product(ctx, cus, kernel, case):
    out, M, N, K, n = case
    _say("gemm", case)
    assert planned(case) == kernel
    cus(n)
    rng = np.random.default_rng(M * 31 + N * 7 + K)
    A, B = _operand(rng, M, K, 12), _operand(rng, N, K, 12)
    a, b = mx.values(*A, K), mx.values(*B, K)
    want, bound = a @ b.T, mx.product_bound(a, b)
    if out == "bf16":
        bound = bound + 2.0**-8 * np.abs(want)
    dA, dB = [ctx.upload(v) for v in A], [ctx.upload(v) for v in B]
    ldc = N + 3
    C = _up(ctx, np.full((M, ldc), -7.0), out)
    ctx.gemm_mxfp4(*dA, *dB, C, M, N, K, dtype=OUT[out], ldc=ldc)
    ctx.wait(60_000)
    got = _down(ctx, C, out, (M, ldc)).astype(np.float64)
    assert (np.abs(got[:, :N] - want) <= bound).all(), float((np.abs(got[:, :N] - want) / (bound + 1e-300)).max())
    assert (got[:, N:] == -7).all()  # nothing between the rows was written
    for x in (*dA, *dB, C):
        x.free()


def _packed_expectation(A, B, K, relu):
    """The packed product, and which of its blocks of 32 hold sums that fp32 holds exactly (as in
    test_gpu_mxfp4.test_packed_product_bit_by_bit)."""
    a, b = mx.values(*A, K), mx.values(*B, K)
    c = a @ b.T
    unit = 0.25 * np.outer(_smallest_scale(A, K), _smallest_scale(B, K))
    holds = np.abs(a) @ np.abs(b).T < 2.0**24 * unit
    M, N = c.shape
    held = np.pad(holds, ((0, 0), (0, -N % 512)), constant_values=True).reshape(M, -1, 32).all(-1)
    return mx.pack(np.maximum(c, 0) if relu else c), held


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("kernel, case", [c for c in CASES if c[1][0] == "mx"])
def test_packed_product(ctx, cus, kernel, case, relu):
    _, M, N, K, n = case
    _say("gemm_rq", case, relu)
    assert planned(case) == kernel
    cus(n)
    rng = np.random.default_rng(M + N + K)
    A, B = _operand(rng, M, K, 0), _operand(rng, N, K, 0)
    want, held = _packed_expectation(A, B, K, relu)
    assert held[:, :(N + 31) // 32].mean() > 0.5
    dA, dB = [ctx.upload(v) for v in A], [ctx.upload(v) for v in B]
    y = _packed(ctx, M, N)
    ctx.gemm_mxfp4_rq(*dA, *dB, *y, M, N, K, relu=relu)
    ctx.wait(60_000)
    gq, gs = ctx.download(y[0]), ctx.download(y[1])
    s, t = mx.block_scales(gs), mx.block_scales(want[1])
    assert np.array_equal(s[held], t[held]) and (np.abs(s.astype(int) - t) <= 1).all()
    # (a sum that is zero may carry either sign: compared as values, and the padding as bytes; a block whose sums
    # fp32 rounds may take the code beside)
    off = np.abs(mx.values(gq, gs, N) - mx.values(*want, N))
    step = np.where(held, 0, 2.0 * np.exp2(np.maximum(s, t).astype(np.float64) - 127)).repeat(32, 1)[:, :N]
    assert (off <= step).all()
    assert not gq[:, (N + 1) // 2:].any()
    for x in (*dA, *dB, *y):
        x.free()


SPECIAL = [("f32", 138, 130, 2304, 1), ("f32", 143, 804, 1606, 3), ("f32", 134, 128, 4633, 1), ("f32", 300, 200, 513, 8),
           ("bf16", 138, 130, 669, 1), ("bf16", 142, 681, 260, 2), ("bf16", 140, 34, 1860, 1), ("bf16", 300, 200, 513, 8),
           ("mx", 151, 131, 867, 1), ("mx", 149, 530, 1337, 2), ("mx", 1290, 900, 4700, 16), ("mx", 300, 200, 513, 16)]


@pytest.mark.parametrize("case", SPECIAL)
def test_nan_and_overflow_stay_in_their_rows_and_columns_of_a_tile(ctx, cus, case):
    out, M, N, K, n = case
    _say("special values", case)
    assert planned(case)[0] != mi.KERNEL_ROWS
    cus(n)
    rng = np.random.default_rng(M + K)
    xa, xb = rng.standard_normal((M, K)), rng.standard_normal((N, K))
    xa[9], xb[3] = np.abs(xa[9]) * 2.0**100, np.abs(xb[3]) * 2.0**100  # their product is beyond fp32
    xa[M - 2, K // 2], xb[N - 1, K - 1] = np.nan, -np.inf
    A, B = mx.pack(xa), mx.pack(xb)
    a, b = mx.values(*A, K), mx.values(*B, K)
    dA, dB = [ctx.upload(v) for v in A], [ctx.upload(v) for v in B]
    want = a @ b.T
    want[9, 3] = np.inf
    nan = np.isnan(want)
    assert nan[M - 2].all() and nan[:, N - 1].all() and nan.sum() == M + N - 1
    if out == "mx":
        y = _packed(ctx, M, N)
        ctx.gemm_mxfp4_rq(*dA, *dB, *y, M, N, K, relu=True)
        ctx.wait(60_000)
        bad = np.pad(nan | np.isinf(want), ((0, 0), (0, -N % 512))).reshape(M, -1, 32).any(-1)
        s = mx.block_scales(ctx.download(y[1]))
        assert np.array_equal(s == 255, bad)
        t = mx.block_scales(mx.pack(np.maximum(want, 0))[1])
        assert (np.abs(s.astype(int) - t) <= 1).all()
        bufs = y
    else:
        C = _up(ctx, np.full((M, N), -7.0), out)
        ctx.gemm_mxfp4(*dA, *dB, C, M, N, K, dtype=OUT[out])
        ctx.wait(60_000)
        got = _down(ctx, C, out, (M, N)).astype(np.float64)
        assert np.array_equal(np.isnan(got), nan) and got[9, 3] == np.inf
        fine = ~nan
        fine[9, 3] = False
        bound = mx.product_bound(np.nan_to_num(a), np.nan_to_num(b)) + (2.0**-8 * np.abs(want) if out == "bf16" else 0)
        assert (np.abs(got - want)[fine] <= bound[fine]).all()
        bufs = [C]
    for x in (*dA, *dB, *bufs):
        x.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_nan_stays_in_its_token_through_the_mlp(ctx, cus, dtype):
    """Both products on tiles: a token with a NaN gives a row of NaN, the others what they give without it."""
    M, K, F, N, n = 300, 512, 768, 300, 2
    _say("mlp nan", dtype)
    for out, cols, k in (("mx", F, K), (dtype, N, F)):
        assert planned((out, M, cols, k, n))[0] != mi.KERNEL_ROWS
    cus(n)
    rng = np.random.default_rng(M)
    x, W1, W2 = rng.standard_normal((M, K)), _operand(rng, F, K), _operand(rng, N, F)
    Y, results = _up(ctx, np.zeros((M, N)), dtype), []
    w, H = [ctx.upload(v) for v in (*W1, *W2)], _packed(ctx, M, F)
    for bad in (False, True):
        if bad:
            x[257, 31] = np.nan
        X = [ctx.upload(v) for v in mx.pack(x)]
        ctx.mlp_mxfp4(*X, *w, *H, Y, M, K, F, N, dtype=OUT[dtype])
        ctx.wait(60_000)
        results.append(_down(ctx, Y, dtype, (M, N)))
        for v in X:
            v.free()
    others = np.arange(M) != 257
    assert np.isnan(results[1][257]).all() and np.isfinite(results[0]).all()
    assert np.array_equal(results[0][others], results[1][others])
    for v in (*w, *H, Y):
        v.free()
