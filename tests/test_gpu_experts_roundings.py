"""Where miaie_experts_mlp_fp8 rounds (include/miaie.h): behind H, whose codes are read
back here, once to bf16 in Y and once in out with dtype MIAIE_BF16, and nowhere with
MIAIE_F32."""
import numpy as np
import pytest

import aiehlc_amd as mi
import fp8_oracle as fp8
import test_gpu_experts as experts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T, k, E, kind, D, F, N", [(3, 2, 4, "even", 200, 256, 130), (5, 1, 8, "even", 128, 4224, 40),
                                                    (333, 2, 7, "holes", 300, 384, 200), (600, 2, 2, "even", 129, 256, 300)])
def test_roundings_behind_h(ctx, T, k, E, kind, D, F, N, dtype):
    print("[case]", T, k, E, kind, D, F, N, dtype, flush=True)
    rng = np.random.default_rng(T + D)
    idx, w, X, (Q1, S1, _), (Q2, S2, V2) = experts._mlp_case(rng, T, k, E, kind, D, F, N)
    o, order = fp8.order(idx, E), experts._order(ctx, idx, E)
    R = o["rows"]
    xq, W = [ctx.upload(v) for v in fp8.pack(X)], [ctx.upload(v) for v in (Q1, S1, Q2, S2)]
    dw, hq = ctx.upload(w), experts._packed(ctx, R, F)
    dY, dout = (experts._up(ctx, np.full((n, N), 7.0), dtype) for n in (R, T))
    ctx.experts_mlp_fp8(order, dw, *xq, *W, *hq, dY, dout, T, k, E, D, F, N, dtype=experts.DT[dtype])
    ctx.wait(60_000)
    h = fp8.values(ctx.download(hq[0]), ctx.download(hq[1]), R, F)
    Y, out = experts._down(ctx, dY, dtype, (R, N)), experts._down(ctx, dout, dtype, (T, N))
    half = 2.0**-8 if dtype == "bf16" else 0.0  # of a rounding to bf16
    y, bound = np.zeros((R, N)), np.zeros((R, N))
    for e, slots in fp8.used_slots(o):
        y[slots], bound[slots] = h[slots] @ V2[e].T, fp8.product_bound(h[slots], V2[e])
    live = o["pair"] >= 0
    assert (np.abs(Y - y)[live] <= (bound + half * (np.abs(y) + bound))[live]).all()
    # the sum of what Y holds: a rounding of 2^-24 for each product and each addition
    Y = np.where(live[:, None], Y, 0.0)
    want, size = fp8.combine(o, Y, w), fp8.combine(o, np.abs(Y), np.abs(w))
    sums = 2.0**-23 * k * size
    assert (np.abs(out - want) <= sums + half * (np.abs(want) + sums)).all()
    if dtype == "f32":  # nothing between H and out is rounded to fewer bits
        assert (np.abs(out - fp8.combine(o, y, w)) <= fp8.combine(o, bound, np.abs(w)) + sums).all()
    experts._free(order, *xq, *W, dw, *hq, dY, dout)
