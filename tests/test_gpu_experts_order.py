"""The order of many pairs: more than 64 workgroups of 1024 take at once, so that a
wave places several rows of 64 in turn, up to the most that are documented."""
import numpy as np
import pytest

import aiehlc_amd as mi
import fp8_oracle as fp8
import test_gpu_experts as experts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["random", "one", "runs", "holes", "none"])
@pytest.mark.parametrize("T, k, E", [(65537, 1, 1), (9001, 8, 64), (131071, 1, 1024), (70000, 3, 5), (1 << 20, 8, 7)])
def test_order_of_many(ctx, T, k, E, kind):
    print("[case] order", T, k, E, kind, flush=True)
    rng = np.random.default_rng(T + E)
    idx = rng.integers(0, E, (T, k), dtype=np.int32)
    if kind == "one":
        idx[:] = E - 1
    if kind == "runs":  # of one expert, longer and shorter than a row of 64
        idx = np.repeat(rng.integers(0, E, T * k, dtype=np.int32), rng.integers(1, 200, T * k))[:T * k].reshape(T, k)
    if kind == "holes":
        idx[rng.random((T, k)) < 0.4] = -1
        idx[rng.random((T, k)) < 0.1] = E
    if kind == "none":
        idx[:] = -3
    o = fp8.order(np.ascontiguousarray(idx), E)
    order = experts._order(ctx, np.ascontiguousarray(idx), E)
    got = ctx.download(order)
    assert 4 * len(got) == mi.experts_order_bytes(T, k, E)
    assert np.array_equal(got, o["all"]), np.flatnonzero(got != o["all"])[:10]
    order.free()
