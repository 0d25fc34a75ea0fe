"""Few slots an expert on average, and one expert with many of them: the kernels for
few rows take four of its rows at a time, shared out over the launch's workgroups.
Results as tests/test_gpu_experts.py has them, and a time that does not grow with the
largest expert."""
import time

import numpy as np
import pytest

import aiehlc_amd as mi
import test_gpu_experts as experts

pytestmark = pytest.mark.gpu


# tokens, choices, experts, their choice: one expert takes several fours of rows, the last of them not full
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("T, k, E, kind, N, K", [(32, 1, 8, "one", 33, 4100), (23, 1, 8, "one", 130, 2050), (150, 1, 100, "one", 70, 2048),
                                                 (130, 1, 64, "one", 17, 4096), (50, 2, 70, "twice", 40, 9000), (7, 2, 4, "one", 513, 8200)])
def test_products(ctx, T, k, E, kind, N, K, gather):
    assert mi.plan_experts_fp8(T, k, E, N, K)["kernel"] == mi.KERNEL_ROWS
    experts.test_products_over_slots(ctx, T, k, E, kind, N, K, gather)


@pytest.mark.parametrize("T, k, E, kind, D, F, N", [(16, 1, 8, "one", 300, 256, 70), (200, 1, 64, "one", 129, 128, 40),
                                                    (130, 1, 70, "one", 128, 384, 33), (7, 2, 8, "twice", 513, 128, 64)])
def test_mlp(ctx, T, k, E, kind, D, F, N):
    assert mi.plan_experts_fp8(T, k, E, F, D, True)["kernel"] == mi.KERNEL_ROWS
    experts.test_mlp(ctx, T, k, E, kind, D, F, N)


@pytest.mark.parametrize("k, pairs", [(1, 128), (8, 256)])
def test_time_of_a_popular_expert(ctx, k, pairs):
    """As many slots of one expert read one expert's matrices, and take no longer than those of all 64."""
    E, D, F, N, T = 64, 2048, 512, 2048, pairs // k
    R = mi.experts_rows(T, k, E)

    def packed(rows, cols, block, count=1):
        (r, c), (b, n) = mi.fp8_shapes(rows, cols, block)
        return ctx.upload(np.zeros((count, r, c), np.uint8)), ctx.upload(np.ones((count, b, n), np.float32))

    X, W1, W2, H = packed(T, D, 1), packed(2 * F, D, 128, E), packed(N, F, 128, E), packed(R, F, 1)
    w, Y, out = ctx.upload(np.ones((T, k), np.float32)), ctx.empty((R, N), np.float32), ctx.empty((T, N), np.float32)
    us = {}
    for kind, idx in (("all", np.arange(T * k) % E), ("one", np.full(T * k, 5))):
        order = experts._order(ctx, idx.reshape(T, k).astype(np.int32), E)
        times = []
        for _ in range(5):
            start = time.perf_counter()
            for _ in range(20):
                ctx.experts_mlp_fp8(order, w, *X, *W1, *W2, *H, Y, out, T, k, E, D, F, N, dtype=mi.F32)
            ctx.wait(60_000)
            times.append((time.perf_counter() - start) / 20 * 1e6)
        us[kind] = min(times)
        order.free()
    print("[case]", k, pairs, us, flush=True)
    experts._free(*X, *W1, *W2, *H, w, Y, out)
    assert us["one"] <= 1.25 * us["all"], us
