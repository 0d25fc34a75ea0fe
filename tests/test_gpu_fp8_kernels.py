"""Every kernel of the 8-bit products at small sizes: planned for fewer compute
units than there are (miaie_plan_set_cus), small products take the tiles that large
ones take (tests/test_fp8_plan.py checks which).  The tests themselves, their
oracles and tolerances are those of tests/test_gpu_fp8.py and
tests/test_gpu_experts.py."""
import numpy as np
import pytest

import aiehlc_amd as mi
import fp8_oracle as fp8
import test_gpu_experts as experts
import test_gpu_fp8 as basic

pytestmark = pytest.mark.gpu

# M, N, K, compute units; steps of 128 k around the stages of LDS (2 or 3)
DENSE = [(3, 70, 2500, 256), (2, 50, 4500, 256), (4, 130, 1000, 256), (6, 21, 1108, 8), (3, 65, 300, 4), (12, 201, 1, 1),
         (12, 195, 129, 1), (70, 193, 333, 1), (61, 193, 461, 1), (12, 201, 699, 1), (196, 70, 128, 1), (195, 12, 205, 1),
         (133, 65, 333, 1), (132, 65, 385, 1), (67, 131, 589, 1), (67, 150, 615, 1), (65, 131, 845, 1), (75, 137, 2872, 1),
         (127, 255, 2945, 1), (194, 129, 512, 1), (130, 195, 589, 1), (131, 210, 616, 1), (131, 194, 896, 1),
         (300, 513, 1500, 2)]
# tokens, choices, experts, their choice, N, K, compute units
SLOTS = [(107, 2, 2, "even", 31, 77, 1), (204, 1, 2, "holes", 40, 205, 1), (301, 1, 1, "even", 22, 257, 1), (248, 1, 4, "even", 71, 462, 1),
         (97, 1, 1, "one", 79, 769, 1), (278, 1, 1, "even", 131, 128, 1), (195, 1, 1, "even", 129, 205, 1), (199, 1, 1, "even", 129, 257, 1),
         (170, 3, 3, "twice", 159, 406, 3), (257, 3, 3, "even", 300, 513, 1), (385, 1, 1, "even", 270, 845, 1), (500, 2, 4, "holes", 259, 640, 1),
         (19, 1, 4, "even", 22, 462, 1), (13, 1, 1, "even", 70, 129, 2), (31, 2, 5, "even", 65, 384, 256), (66, 1, 1, "one", 30, 896, 8),
         (1, 1, 6, "even", 99, 402, 2), (2, 1, 1, "even", 17, 513, 1), (9, 3, 8, "one", 130, 2048, 256), (5, 2, 3, "twice", 33, 8200, 256),
         (4, 2, 2, "even", 70, 16500, 256)]
# tokens, choices, experts, their choice, D, F, Nout, compute units
MLPS = [(96, 1, 1, "even", 1, 128, 40, 1), (130, 1, 1, "even", 205, 256, 33, 1), (160, 1, 3, "even", 505, 128, 70, 3),
        (97, 1, 1, "even", 845, 128, 64, 1), (192, 1, 1, "even", 77, 128, 33, 1), (200, 1, 1, "even", 256, 128, 40, 1),
        (127, 3, 3, "twice", 402, 128, 70, 3), (400, 2, 3, "holes", 640, 256, 130, 1), (5, 1, 1, "even", 128, 128, 33, 8),
        (18, 1, 3, "even", 406, 128, 64, 8), (70, 1, 1, "one", 769, 128, 70, 1), (1, 1, 4, "even", 493, 128, 64, 1),
        (3, 4, 4, "even", 128, 256, 70, 256), (9, 2, 5, "one", 900, 128, 33, 256)]


@pytest.fixture
def planned(ctx):
    yield lambda cus: ctx.plan_set_cus(cus)
    ctx.plan_set_cus(256)


@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("b_block", [1, 128])
@pytest.mark.parametrize("M, N, K, cus", DENSE)
def test_gemm_on_every_kernel(ctx, planned, M, N, K, cus, b_block, exact):
    planned(cus)
    print("[case]", mi.plan_gemm_fp8(M, N, K, b_block, cus), flush=True)
    basic.test_gemm(ctx, (M, N, K), b_block, exact)


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("T, k, E, kind, N, K, cus", SLOTS)
def test_products_over_slots_on_every_kernel(ctx, planned, T, k, E, kind, N, K, cus, gather):
    planned(cus)
    print("[case]", mi.plan_experts_fp8(T, k, E, N, K, False, cus), flush=True)
    experts.test_products_over_slots(ctx, T, k, E, kind, N, K, gather)


@pytest.mark.parametrize("T, k, E, kind, D, F, N, cus", MLPS)
def test_mlp_on_every_kernel(ctx, planned, T, k, E, kind, D, F, N, cus):
    planned(cus)
    print("[case]", mi.plan_experts_fp8(T, k, E, F, D, True, cus), flush=True)
    experts.test_mlp(ctx, T, k, E, kind, D, F, N)


@pytest.mark.parametrize("M", [1, 2, 3, 4])
@pytest.mark.parametrize("N, K", [(1, 8193), (37, 20000), (129, 8192)])
def test_few_rows_of_long_weights(ctx, M, N, K):
    """More blocks of k than a workgroup keeps of A at a time."""
    basic._say("few rows", M, N, K)
    rng = np.random.default_rng(M + K)
    pA, pB = basic._operands(rng, M, N, K, 128)
    a, b = fp8.values(*pA, M, K), fp8.values(*pB, N, K, 128)
    want, bound = a @ b.T, fp8.product_bound(a, b)
    d, C = [ctx.upload(v) for v in (*pA, *pB)], ctx.empty((M, N), np.float32)
    ctx.gemm_fp8(*d, C, M, N, K)
    ctx.wait(60_000)
    assert (np.abs(ctx.download(C) - want) <= bound).all()
    for buf in (*d, C):
        buf.free()


def test_short_products_have_exact_sums(ctx):
    """Up to 1024 CUs and one: the same bits from every kernel, where every sum is exact."""
    basic._say("one result on every kernel")
    M, N, K = 260, 390, 600
    rng = np.random.default_rng(8)
    pA, pB = basic._operands(rng, M, N, K, 128, exact=True)
    want = (fp8.values(*pA, M, K) @ fp8.values(*pB, N, K, 128).T).astype(np.float32)
    d, C = [ctx.upload(v) for v in (*pA, *pB)], ctx.empty((M, N), np.float32)
    try:
        for cus in (1, 2, 3, 5, 8, 13, 20, 64, 1024):
            ctx.plan_set_cus(cus)
            ctx.gemm_fp8(*d, C, M, N, K)
            ctx.wait(60_000)
            assert np.array_equal(ctx.download(C), want), (cus, mi.plan_gemm_fp8(M, N, K, 128, cus))
    finally:
        ctx.plan_set_cus(256)
        for buf in (*d, C):
            buf.free()
