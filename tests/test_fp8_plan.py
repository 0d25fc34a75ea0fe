"""The choice of kernel of the 8-bit products (miaie_plan_gemm_fp8,
miaie_plan_experts_fp8): host functions, so these run without a GPU."""
import random

import pytest

import aiehlc_amd as mi

DENSE_TILES = [(256, 256), (128, 256), (128, 128), (64, 128), (64, 64)]
MOST = (1 << 32) - 1


def test_plans():
    assert mi.plan_gemm_fp8(8192, 8192, 8192) == {"kernel": mi.KERNEL_PIPE, "tile_m": 256, "tile_n": 256,
                                                  "workgroups": 1024, "threads": 512}
    # one token: four waves share out the 32 blocks of k of 16 columns
    assert mi.plan_gemm_fp8(1, 11008, 4096) == {"kernel": mi.KERNEL_ROWS, "tile_m": 4, "tile_n": 16, "workgroups": 688,
                                                "threads": 256}
    assert mi.plan_gemm_fp8(1, 11008, 4096, b_block=1)["kernel"] == mi.KERNEL_PIPE  # (no weights)
    # few slots an expert read its matrices once for four rows
    assert mi.plan_experts_fp8(8, 8, 64, 2048, 4096, swiglu=True)["kernel"] == mi.KERNEL_ROWS
    assert mi.plan_experts_fp8(2048, 8, 64, 2048, 4096, swiglu=True)["tile_m"] == 256


@pytest.mark.parametrize("b_block", [1, 128])
def test_every_documented_product_has_a_kernel(b_block):
    rng = random.Random(b_block)
    sizes = [(1 << 25, 128, 1), (128, 1 << 25, 1 << 23), (1, 1 << 25, 1 << 23), (4, 1 << 25, 1), (5, 1 << 25, 1),
             ((1 << 19) - 1, 1 << 12, 1 << 23), ((1 << 12) - 1, 1 << 19, 1), (256 * 2047, 256 * 4096, 128), (1, 1, 1)]
    for i in range(20000):
        M, N, K = sizes[i] if i < len(sizes) else (int(2 ** rng.uniform(0, most)) for most in (25, 25, 23))
        if -(-M // 256) * -(-N // 256) >= 1 << 23:
            continue
        p = mi.plan_gemm_fp8(M, N, K, b_block, rng.choice([1, 7, 256, 1 << 20]))
        assert 0 < p["workgroups"] * p["threads"] <= MOST, (M, N, K)
        if p["kernel"] == mi.KERNEL_ROWS:
            assert M <= 4 and b_block == 128 and p["workgroups"] == -(-N // p["tile_n"])
        else:
            assert (p["tile_m"], p["tile_n"]) in DENSE_TILES
            assert p["workgroups"] == -(-M // p["tile_m"]) * -(-N // p["tile_n"])


def test_every_documented_product_over_slots_has_a_kernel():
    rng = random.Random(3)
    for i in range(20000):
        E, k = int(2 ** rng.uniform(0, 10)), int(2 ** rng.uniform(0, 6))
        T = int(2 ** rng.uniform(0, 23)) // k or 1
        N, K = int(2 ** rng.uniform(0, 20)), int(2 ** rng.uniform(0, 20))
        for swiglu in (False, True):
            if swiglu:
                N = -(-N // 128) * 128
            n = 2 * N if swiglu else N
            if mi.experts_rows(T, k, E) // 128 * -(-n // 128) > 1 << 22:
                continue
            p = mi.plan_experts_fp8(T, k, E, N, K, swiglu, rng.choice([1, 7, 256, 1 << 20]))
            used = min(E, T * k)
            tiles = lambda rows: used + (T * k - used) // rows  # noqa: E731 (what the header's slots can fill)
            assert 0 < (p["workgroups"] + 8) * p["threads"] <= MOST + 1, (T, k, E, N, K)
            rows = 128 if p["kernel"] == mi.KERNEL_ROWS else p["tile_m"]
            assert p["workgroups"] == tiles(rows) * -(-N // p["tile_n"])


def _kernel(p):
    return p["kernel"], p["tile_m"], p["tile_n"], p["threads"]


def test_the_gpu_tests_reach_every_kernel():
    import test_gpu_fp8 as basic
    import test_gpu_fp8_kernels as kernels

    for b_block in (1, 128):
        seen = {_kernel(mi.plan_gemm_fp8(*shape, b_block, cus)) for *shape, cus in kernels.DENSE}
        seen |= {_kernel(mi.plan_gemm_fp8(*shape, b_block)) for shape in basic.GEMMS}
        rng = random.Random(1)
        for _ in range(20000):
            M, N, K = (int(2 ** rng.uniform(0, most)) for most in (15, 15, 14))
            assert _kernel(mi.plan_gemm_fp8(M, N, K, b_block, rng.choice([1, 8, 256]))) in seen, (M, N, K)
    slots = {_kernel(mi.plan_experts_fp8(T, k, E, N, K, False, cus)) for T, k, E, _, N, K, cus in kernels.SLOTS}
    glu = {_kernel(mi.plan_experts_fp8(T, k, E, F, D, True, cus)) for T, k, E, _, D, F, _, cus in kernels.MLPS}
    for _ in range(20000):
        E, k = int(2 ** rng.uniform(0, 8)), rng.randint(1, 8)
        T, N, K = (int(2 ** rng.uniform(0, most)) for most in (13, 12, 13))
        cus = rng.choice([1, 8, 256])
        assert _kernel(mi.plan_experts_fp8(T, k, E, N, K, False, cus)) in slots
        assert _kernel(mi.plan_experts_fp8(T, k, E, -(-N // 128) * 128, K, True, cus)) in glu


@pytest.mark.parametrize("args", [(0, 1, 1), (1, 0, 1), (1, 1, 0), ((1 << 25) + 1, 1, 1), (1, (1 << 25) + 1, 1),
                                  (1, 1, (1 << 23) + 1), (256 << 12, 256 << 11, 1), (1, 1, 1, 2), (1, 1, 1, 1, 0)])
def test_refused_products(args):
    with pytest.raises(mi.MiaieError):
        mi.plan_gemm_fp8(*args)


@pytest.mark.parametrize("args", [(0, 1, 1, 1, 1), (1, 0, 1, 1, 1), (1, 65, 1, 1, 1), (1, 1, 0, 1, 1), (1, 1, 1025, 1, 1),
                                  (1 << 22, 3, 1, 1, 1), (1, 1, 1, 0, 1), (1, 1, 1, (1 << 20) + 1, 1), (1, 1, 1, 1, 0),
                                  (1, 1, 1, 1, (1 << 20) + 1), (1, 1, 1, 64, 1, True), (1, 1, 1, 128, 1, 2),
                                  (1 << 20, 8, 64, 1 << 20, 1), (1, 1, 1, 1, 1, False, 0)])
def test_refused_products_over_slots(args):
    with pytest.raises(mi.MiaieError):
        mi.plan_experts_fp8(*args)
    T, k, E = args[:3]
    sizes = 1 <= k <= 64 and 1 <= E <= 1024 and 1 <= T * k <= 1 << 23
    assert bool(mi.experts_rows(T, k, E)) == bool(mi.experts_order_bytes(T, k, E)) == sizes
