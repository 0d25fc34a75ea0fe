"""Where miaie_experts_mlp_fp8 and the sums over slots round (include/miaie.h): behind H,
whose codes are read back here, to bf16 in Y and in out with dtype MIAIE_BF16, in out
alone with MIAIE_F32_SLOTS, and nowhere with MIAIE_F32."""
import numpy as np
import pytest

import aiehlc_amd as mi
import fp8_oracle as fp8
import test_gpu_experts as experts

pytestmark = pytest.mark.gpu


TYPES = [("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32")]  # of Y and out


@pytest.mark.parametrize("ty, dtype", TYPES)
@pytest.mark.parametrize("T, k, E, kind, D, F, N", [(3, 2, 4, "even", 200, 256, 130), (5, 1, 8, "even", 128, 4224, 40),
                                                    (333, 2, 7, "holes", 300, 384, 200), (600, 2, 2, "even", 129, 256, 300)])
def test_roundings_behind_h(ctx, T, k, E, kind, D, F, N, ty, dtype):
    print("[case]", T, k, E, kind, D, F, N, ty, dtype, flush=True)
    rng = np.random.default_rng(T + D)
    idx, w, X, (Q1, S1, _), (Q2, S2, V2) = experts._mlp_case(rng, T, k, E, kind, D, F, N)
    o, order = fp8.order(idx, E), experts._order(ctx, idx, E)
    R = o["rows"]
    xq, W = [ctx.upload(v) for v in fp8.pack(X)], [ctx.upload(v) for v in (Q1, S1, Q2, S2)]
    dw, hq = ctx.upload(w), experts._packed(ctx, R, F)
    dY, dout = experts._up(ctx, np.full((R, N), 7.0), ty), experts._up(ctx, np.full((T, N), 7.0), dtype)
    ctx.experts_mlp_fp8(order, dw, *xq, *W, *hq, dY, dout, T, k, E, D, F, N, dtype=experts.DT[dtype], y_dtype=experts.DT[ty])
    ctx.wait(60_000)
    h = fp8.values(ctx.download(hq[0]), ctx.download(hq[1]), R, F)
    Y, out = experts._down(ctx, dY, ty, (R, N)), experts._down(ctx, dout, dtype, (T, N))
    y_half, half = (2.0**-8 if t == "bf16" else 0.0 for t in (ty, dtype))  # of a rounding to bf16
    y, bound = np.zeros((R, N)), np.zeros((R, N))
    for e, slots in fp8.used_slots(o):
        y[slots], bound[slots] = h[slots] @ V2[e].T, fp8.product_bound(h[slots], V2[e])
    live = o["pair"] >= 0
    assert (np.abs(Y - y)[live] <= (bound + y_half * (np.abs(y) + bound))[live]).all()
    assert (Y[~live] == 7).all()
    # the sum of what Y holds: a rounding of 2^-24 for each product and each addition
    Y = np.where(live[:, None], Y, 0.0)
    want, size = fp8.combine(o, Y, w), fp8.combine(o, np.abs(Y), np.abs(w))
    sums = 2.0**-23 * k * size
    assert (np.abs(out - want) <= sums + half * (np.abs(want) + sums)).all()
    if ty == "f32":  # of what is between H and out, nothing is rounded to fewer bits
        want = fp8.combine(o, y, w)
        all_of = fp8.combine(o, bound, np.abs(w)) + sums
        assert (np.abs(out - want) <= all_of + half * (np.abs(want) + all_of)).all()
    experts._free(order, *xq, *W, dw, *hq, dY, dout)


@pytest.mark.parametrize("T, k, E, kind", experts.SLOTS)
def test_fp32_rows_beside_bf16(ctx, T, k, E, kind):
    """The sum over slots and its gradient; the gradient's tolerance is that of experts.test_combine_and_its_gradient."""
    rng = np.random.default_rng(T + k)
    idx = experts._choices(rng, T, k, E, kind)
    o, order = fp8.order(idx, E), experts._order(ctx, idx, E)
    R, live = o["rows"], o["pair"] >= 0
    for C, ldy, ldo in ((1, 1, 1), (7, 8, 9), (300, 307, 303), (2500, 2500, 2500)):
        print("[case] combine", T, k, E, kind, C, flush=True)
        Y, dout = np.float32(rng.standard_normal((R, ldy))), experts._stored(rng.standard_normal((T, ldo)), "bf16")
        Y[~live] = np.nan
        w = np.float32(rng.standard_normal((T, k)))
        dY, dw, dd = ctx.upload(Y), ctx.upload(w), experts._up(ctx, dout, "bf16")
        y = np.where(live[:, None], Y[:, :C], 0).astype(np.float64)
        for ww, buf in ((w, dw), (None, None)):
            out = experts._up(ctx, np.full((T, ldo), 7.0), "bf16")
            ctx.experts_combine(order, dY, buf, out, T, k, E, C, y_dtype=mi.F32, ldy=ldy, ldo=ldo)
            ctx.wait(60_000)
            got, want = experts._down(ctx, out, "bf16", (T, ldo)), fp8.combine(o, y, ww)
            sums = 2.0**-23 * k * fp8.combine(o, np.abs(y), None if ww is None else np.abs(ww))
            assert (np.abs(got[:, :C] - want) <= sums + 2.0**-8 * (np.abs(want) + sums)).all()
            assert (got[:, C:] == 7).all()
            out.free()
        g = ctx.upload(np.full((T, k), -9, np.float32))
        ctx.experts_combine_grad(order, dY, dd, g, T, k, E, C, y_dtype=mi.F32, ldy=ldy, ldo=ldo)
        ctx.wait(60_000)
        want, size = np.zeros((T, k)), np.zeros((T, k))
        for t, j in zip(*np.nonzero(o["slot"] >= 0)):
            p = y[o["slot"][t, j]] * dout[t, :C]
            want[t, j], size[t, j] = p.sum(), np.abs(p).sum()
        assert (np.abs(ctx.download(g) - want) <= 2.0**-24 * (C / 64 + 16) * size).all()
        experts._free(dY, dw, dd, g)
    order.free()


def test_refused_types(ctx):
    d = ctx.upload(np.full(1 << 16, 0x5A, np.uint8))
    p, wide = d.ptr, mi.BF16 | mi.F32_SLOTS
    calls = {"experts_mlp_fp8": lambda y, t: (*[p] * 10, y, p, t, 4, 2, 8, 16, 128, 16, 16),
             "experts_combine": lambda y, t: (p, y, p, p, t, 4, 2, 8, 16, 16, 16),
             "experts_combine_grad": lambda y, t: (p, y, p, p, t, 4, 2, 8, 16, 16, 16)}
    for name, args in calls.items():
        for dtype in (mi.F32 | mi.F32_SLOTS, 2 | mi.F32_SLOTS, -1):
            assert ctx.call_status("miaie_" + name, *args(p, dtype)) == mi.MIAIE_EINVAL and f"dtype={dtype}" in ctx.last_error()
        assert ctx.call_status("miaie_" + name, *args(p + 2, wide)) == mi.MIAIE_EINVAL and "Y is misaligned" in ctx.last_error()
    # products and conversions have one type
    assert ctx.call_status("miaie_experts_gemm_fp8", *[p] * 6, wide, 4, 2, 8, 16, 16, 16, 0) == mi.MIAIE_EINVAL
    assert ctx.call_status("miaie_experts_quant_fp8", p, p, wide, p, p, p, p, p, 4, 2, 8, 16, 16) == mi.MIAIE_EINVAL
    ctx.wait(10_000)
    assert (ctx.download(d) == 0x5A).all()
    d.free()
