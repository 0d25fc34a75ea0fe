"""Routing of tokens to experts and the experts' products through the C ABI
against the 64-bit oracle (tests/fp8_oracle.py).

Choices, orders and conversions are compared value by value, fp32 weights and
their gradients to a few units in the last place, products by
fp8_oracle.product_bound."""
import numpy as np
import pytest

import aiehlc_amd as mi
import fp8_oracle as fp8

pytestmark = pytest.mark.gpu

DT = {"f32": mi.F32, "bf16": mi.BF16}
SCORING = {"softmax": mi.SOFTMAX, "sigmoid": mi.SIGMOID}


def _say(*a):
    print("[case]", *a, flush=True)


def _up(ctx, x, dtype):
    return ctx.upload(fp8.bf16_bits(x) if dtype == "bf16" else np.asarray(x, np.float32))


def _down(ctx, buf, dtype, shape):
    if dtype == "bf16":
        return fp8.from_bf16_bits(ctx.download(buf, np.uint16, shape)).astype(np.float64)
    return ctx.download(buf, np.float32, shape).astype(np.float64)


def _packed(ctx, rows, cols, block=1):
    q, s = mi.fp8_shapes(rows, cols, block)
    return ctx.upload(np.full(q, 0xA5, np.uint8)), ctx.upload(np.full(s, -7.0, np.float32))


def _free(*bufs):
    for b in bufs:
        if b is not None:
            b.free()


def _stored(x, dtype):
    return fp8.bf16(x).astype(np.float64) if dtype == "bf16" else np.float32(x).astype(np.float64)


# ---------------------------------------------------------------- routing
# tokens, experts, top_k, groups, kept, group_top, bias
ROUTES = [(1, 1, 1, 1, 1, 1, False), (1, 256, 8, 8, 4, 2, True), (8, 256, 8, 8, 4, 2, True), (33, 64, 6, 1, 1, 1, False),
          (70, 128, 4, 1, 1, 1, True), (19, 7, 2, 1, 1, 1, False), (21, 7, 7, 7, 7, 1, True), (40, 160, 6, 8, 3, 1, False),
          (17, 512, 32, 64, 8, 2, False), (9, 1024, 64, 1, 1, 1, False), (9, 1000, 33, 10, 2, 2, True),
          (30, 65, 64, 1, 1, 1, False), (12, 24, 5, 4, 2, 2, False)]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("case", ROUTES)
def test_route(ctx, case, scoring):
    T, E, k, groups, kept, top, biased = case
    rng = np.random.default_rng(T * 1000 + E)
    for dtype in ("f32", "bf16"):
        _say("route", case, scoring, dtype)
        ld = E + 3
        l = _stored(rng.standard_normal((T, ld)) * 2, dtype)
        if dtype == "bf16":
            l = np.round(l * 4) / 4  # many equal logits
        if T > 2 and E > 2:
            l[1, 1:E] = -np.inf                # one expert to choose
            l[2, :] = -np.inf                  # none
            l[3 % T, rng.random(ld) < 0.5] = -np.inf
        bias = np.float32(rng.standard_normal(E) * 0.1) if biased else None
        if biased and E > 4:
            bias[4] = -np.inf
        for renorm in (True, False):
            want_i, want_w = fp8.route(l[:, :E], bias, k, scoring, groups, kept, top, renorm, 2.5)
            dl, db = _up(ctx, l, dtype), None if bias is None else ctx.upload(bias)
            di, dw = ctx.upload(np.full((T, k), -9, np.int32)), ctx.upload(np.full((T, k), -9, np.float32))
            ctx.route_experts(dl, db, di, dw, T, k, E, scoring=SCORING[scoring], groups=groups, groups_kept=kept,
                              group_top=top, renormalize=renorm, scale=2.5, dtype=DT[dtype], ld=ld)
            ctx.wait(60_000)
            assert np.array_equal(ctx.download(di), want_i)
            # one rounding of a value of 64 bits (exp to a few units of those)
            assert (np.abs(ctx.download(dw) - want_w) <= 2.0**-23 * np.abs(want_w) + 1e-44).all()
            # the gradient, also where an expert is there twice and where there is none
            idx, d = want_i.copy(), np.float32(rng.standard_normal((T, k)))
            if k > 1 and T > 3:
                idx[0, 1] = idx[0, 0]
                idx[3, k - 1] = E
            g, ldd = ctx.upload(np.full((T, E + 1), -9, np.float32)), E + 1
            dd, dx = ctx.upload(d), ctx.upload(idx)
            ctx.route_experts_grad(dl, dx, dd, g, T, k, E, scoring=SCORING[scoring], renormalize=renorm, scale=2.5,
                                   dtype=DT[dtype], ld=ld, ldd=ldd)
            ctx.wait(60_000)
            got, want = ctx.download(g), fp8.route_grad(l[:, :E], idx, d, scoring, renorm, 2.5)
            # p comes from an exponential, a sum in a tree and a quotient in fp32: 14 half units at most (2^-20) of each
            # term, of which a gradient is the difference
            size = fp8.route_grad_terms(l[:, :E], idx, d, scoring, renorm, 2.5)
            assert (np.abs(got[:, :E] - want) <= 2.0**-20 * size + 1e-30).all()
            assert (got[:, E:] == -9).all()
            _free(dl, db, di, dw, g, dd, dx)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_route_nan_and_infinity(ctx, scoring, biased):
    _say("route NaN", scoring, biased)
    T, E, k = 6, 40, 3
    l = np.random.default_rng(4).standard_normal((T, E)).astype(np.float32)
    l[1, 7] = np.nan
    l[2, 9] = np.inf
    l[3, :] = -np.inf
    l[4, 2] = -np.inf
    bias = np.zeros(E, np.float32)
    bias[2] = np.nan  # of an expert that only token 4 cannot choose
    dl, db = ctx.upload(l), ctx.upload(bias) if biased else None
    di, dw = ctx.empty((T, k), np.int32), ctx.empty((T, k), np.float32)
    ctx.route_experts(dl, db, di, dw, T, k, E, scoring=SCORING[scoring])
    ctx.wait(60_000)
    idx, w = ctx.download(di), ctx.download(dw)
    for t in range(T):
        nan = t == 1 or (t == 2 and scoring == "softmax") or (biased and t not in (3, 4))
        assert np.isnan(w[t]).all() == nan and np.isnan(w[t]).any() == nan, (t, w[t])
    assert (idx[3] == -1).all() and (w[3] == 0).all()
    assert 7 not in idx[1] and (not biased or 2 not in idx)
    _free(dl, db, di, dw)


# ---------------------------------------------------------------- slots
def _choices(rng, T, k, E, kind):
    """idx of a routing: even, of one expert, with pairs that have none, with one expert twice."""
    if kind == "one":
        return np.full((T, k), E - 1, np.int32)
    idx = np.stack([rng.permutation(E)[:k] if k <= E else rng.integers(0, E, k) for _ in range(T)]).astype(np.int32)
    if kind == "holes":
        idx[rng.random((T, k)) < 0.3] = -1
        idx[rng.random((T, k)) < 0.05] = E
        idx[T // 2:] = np.where(rng.random((T - T // 2, 1)) < 0.5, -1, idx[T // 2:])
    if kind == "none":
        idx[:] = -1
    if kind == "twice" and k > 1:
        idx[:, 1] = idx[:, 0]
    return idx


def _order(ctx, idx, E):
    T, k = idx.shape
    n = mi.experts_order_bytes(T, k, E) // 4
    order, d = ctx.upload(np.full(n, -7, np.int32)), ctx.upload(idx)
    ctx.experts_order(d, order, T, k, E)
    ctx.wait(60_000)
    d.free()
    return order


@pytest.mark.parametrize("kind", ["even", "one", "holes", "none", "twice"])
@pytest.mark.parametrize("T, k, E", [(1, 1, 1), (1, 8, 256), (8, 8, 64), (333, 2, 7), (130, 1, 1), (1023, 3, 100), (2048, 8, 64),
                                     (65, 64, 1024), (5000, 6, 1000)])
def test_order(ctx, T, k, E, kind):
    _say("order", T, k, E, kind)
    idx = _choices(np.random.default_rng(T + E), T, k, E, kind)
    o = fp8.order(idx, E)
    assert mi.experts_rows(T, k, E) == o["rows"] and mi.experts_order_bytes(T, k, E) == 4 * len(o["all"])
    order = _order(ctx, idx, E)
    got = ctx.download(order)
    assert np.array_equal(got, o["all"]), np.flatnonzero(got != o["all"])[:10]
    order.free()


def _experts(rng, E, rows, cols):
    """Packed weights of E experts, scales that are no powers of two; and their values."""
    Q, S, V = [], [], []
    for _ in range(E):
        q, s = fp8.pack(rng.standard_normal((rows, cols)) * cols**-0.5, 128)
        s = (s * rng.uniform(0.5, 1.0, s.shape)).astype(np.float32)
        Q.append(q), S.append(s), V.append(fp8.values(q, s, rows, cols, 128))
    return np.stack(Q), np.stack(S), V


def _conversion(ctx, o, call, want, C):
    """Both forms of a conversion over slots, together and alone, against the values that `want` has in the slots."""
    R, used = o["rows"], o["used"]
    forms = [(_packed(ctx, R, C), _packed(ctx, C, R)), (_packed(ctx, R, C), (None, None)), ((None, None), _packed(ctx, C, R))]
    for q, t in forms:
        call(q, t)
    ctx.wait(60_000)
    for q, t in forms:
        if q[0]:
            Q, S = fp8.pack(want[:used]) if used else (np.zeros((0, fp8.up(C)), np.uint8), np.zeros((fp8.up(C) // 128, 0)))
            gq, gs = ctx.download(q[0]), ctx.download(q[1])
            yield gq[:used], Q, gs[:, :used], S
            assert (gq[used:] == 0xA5).all() and (gs[:, used:] == -7).all()  # behind the slots in use
        if t[0]:
            Q, S = fp8.pack(want[:used].T) if used else (np.zeros((C, 0), np.uint8), np.zeros((0, C)))
            gq, gs = ctx.download(t[0]), ctx.download(t[1])
            yield gq[:, :used], Q, gs[:used // 128], S
            assert (gq[:, used:] == 0xA5).all() and (gs[used // 128:] == -7).all()
        _free(*q, *t)


SLOTS = [(1, 1, 1, "even"), (8, 8, 64, "even"), (5, 2, 3, "none"), (333, 2, 7, "holes"), (200, 3, 4, "twice"), (300, 2, 3, "one")]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T, k, E, kind", SLOTS)
def test_conversion_of_tokens(ctx, T, k, E, kind, dtype):
    rng = np.random.default_rng(T + k)
    idx = _choices(rng, T, k, E, kind)
    o, order = fp8.order(idx, E), _order(ctx, idx, E)
    for C, ld in ((128, 128), (301, 311)):
        for weighted in (False, True):
            _say("slots", T, k, E, kind, dtype, C, weighted)
            X = _stored(rng.standard_normal((T, ld)), dtype)
            w = np.float32(rng.standard_normal((T, k))) if weighted else None
            dx, dw = _up(ctx, X, dtype), None if w is None else ctx.upload(w)
            want = fp8.over_slots(o, X[:, :C])
            if weighted:  # (the product is rounded to fp32)
                want = np.float32(want) * np.float32(fp8.over_slots(o, np.ones((T, 1)), w))
            for gq, Q, gs, S in _conversion(ctx, o, lambda q, t: ctx.experts_quant_fp8(order, dx, dw, *q, *t, T, k, E, C,
                                                                                     dtype=DT[dtype], ldx=ld), want, C):
                assert np.array_equal(gq, Q) and np.array_equal(gs, S)
            _free(dx, dw)
    order.free()


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("T, k, E, kind", SLOTS)
def test_swiglu(ctx, T, k, E, kind, grad):
    """Codes are the oracle's but where fp32 falls on the other side of a border: a step of the format then, and few."""
    rng = np.random.default_rng(T + k)
    idx = _choices(rng, T, k, E, kind)
    o, order = fp8.order(idx, E), _order(ctx, idx, E)
    R, F = o["rows"], 256
    for dtype, ld in (("f32", 2 * F), ("bf16", 2 * F + 9)):
        _say("swiglu", T, k, E, kind, dtype, "gradient" if grad else "")
        GU, dH = _stored(rng.standard_normal((R, ld)) * 3, dtype), np.float32(rng.standard_normal((R, F + 1)))
        live = o["pair"] >= 0
        GU[~live], dH[~live] = np.nan, np.nan  # rows of padding are not read
        if live.any():
            r = np.flatnonzero(live)[0]
            GU[r, :4] = [-100, 100, -90, 0]
        d, dd = _up(ctx, GU, dtype), ctx.upload(dH)
        v = np.where(live[:, None], GU[:, :2 * F], 0.0)
        want = fp8.swiglu_grad(v, np.where(live[:, None], dH[:, :F], 0.0)) if grad else fp8.swiglu(v)
        if grad:
            call = lambda q, t: ctx.experts_swiglu_grad_fp8(order, d, dd, *q, *t, T, k, E, F, dtype=DT[dtype], ldgu=ld, ldh=F + 1)
        else:
            call = lambda q, t: ctx.experts_swiglu_fp8(order, d, *q, *t, T, k, E, F, dtype=DT[dtype], ldgu=ld)
        C = 2 * F if grad else F
        for gq, Q, gs, S in _conversion(ctx, o, call, want, C):
            assert np.array_equal(gs, S)
            a, b = fp8.decode(gq), fp8.decode(Q)
            # about 2^-21 of the values (an exponential, a quotient, four products) stand next to one of 2^-4 borders
            assert (np.abs(a - b) <= np.maximum(2.0**-3 * np.abs(b), 2.0**-9)).all() and (a != b).sum() <= 1e-3 * a.size
        _free(d, dd)
    order.free()


PRODUCTS = [(1, 1, 1, "even", 33, 300), (8, 8, 64, "even", 128, 512), (8, 2, 3, "none", 70, 128), (333, 2, 7, "holes", 200, 129),
            (40, 3, 4, "twice", 260, 1100), (300, 2, 3, "one", 48, 640), (700, 2, 3, "even", 513, 385), (20, 1, 2, "one", 30, 2000)]


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("T, k, E, kind, N, K", PRODUCTS)
def test_products_over_slots(ctx, T, k, E, kind, N, K, gather):
    rng = np.random.default_rng(T + N)
    idx = _choices(rng, T, k, E, kind)
    o, order = fp8.order(idx, E), _order(ctx, idx, E)
    R = o["rows"]
    A = fp8.pack(rng.standard_normal((T if gather else R, K)))
    A[0][:, :K][rng.random((len(A[0]), K)) < 0.1] = 0
    a = fp8.values(*A, *((T if gather else R), K))
    if not gather:  # rows of padding are not read
        A[1][:, o["pair"] < 0] = np.nan
    Q, S, V = _experts(rng, E, N, K)
    dA, dB = [ctx.upload(v) for v in A], [ctx.upload(Q), ctx.upload(S)]
    for dtype, ldc in (("f32", N), ("bf16", N + 5)):
        _say("products", T, k, E, kind, N, K, dtype, gather)
        C = _up(ctx, np.full((R, ldc), 7.0), dtype)
        ctx.experts_gemm_fp8(order, *dA, *dB, C, T, k, E, N, K, gather=gather, dtype=DT[dtype], ldc=ldc)
        ctx.wait(60_000)
        got, seen = _down(ctx, C, dtype, (R, ldc)), np.zeros(R, bool)
        for e, slots in fp8.used_slots(o):
            rows = a[o["pair"][slots] // k] if gather else a[slots]
            want = rows @ V[e].T
            bound = fp8.product_bound(rows, V[e]) + (2.0**-8 * np.abs(want) if dtype == "bf16" else 0)
            assert (np.abs(got[slots, :N] - want) <= bound).all(), e
            seen[slots] = True
        assert (got[~seen] == 7).all() and (got[:, N:] == 7).all()  # padding and what is behind stay as they were
        C.free()
    _free(order, *dA, *dB)


@pytest.mark.parametrize("T, k, E, kind, M, N", [(1, 1, 1, "even", 33, 40), (333, 2, 7, "holes", 200, 129), (8, 2, 3, "none", 70, 128),
                                                 (700, 2, 3, "even", 257, 300), (600, 2, 4, "one", 128, 513)])
def test_weight_gradients(ctx, T, k, E, kind, M, N):
    rng = np.random.default_rng(T + N)
    idx = _choices(rng, T, k, E, kind)
    o, order = fp8.order(idx, E), _order(ctx, idx, E)
    R = o["rows"]
    live = o["pair"] >= 0
    ab = [np.where(live[:, None], rng.standard_normal((R, n)), 0.0).T for n in (M, N)]
    packs = [fp8.pack(m) for m in ab]
    for Q, S in packs:  # behind the slots in use nothing is read
        Q[:, o["used"]:], S[o["used"] // 128:] = 0x7f, np.nan
    v = [np.nan_to_num(fp8.values(*p, len(m), R)) for p, m in zip(packs, ab)]
    d = [ctx.upload(x) for p in packs for x in p]
    for dtype, ldc in (("f32", N), ("bf16", N + 3)):
        _say("weight gradients", T, k, E, kind, M, N, dtype)
        C = _up(ctx, np.full((E, M, ldc), 7.0), dtype)
        ctx.experts_wgrad_fp8(order, *d, C, T, k, E, M, N, dtype=DT[dtype], ldc=ldc)
        ctx.wait(60_000)
        got = _down(ctx, C, dtype, (E, M, ldc))
        assert (got[..., N:] == 7).all()
        for e in range(E):
            s = slice(o["start"][e], o["start"][e + 1])
            a, b = v[0][:, s], v[1][:, s]
            want = a @ b.T
            bound = fp8.product_bound(a, b) + (2.0**-8 * np.abs(want) if dtype == "bf16" else 0)
            assert (np.abs(got[e, :, :N] - want) <= bound).all(), e
        C.free()
    _free(order, *d)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T, k, E, kind", SLOTS)
def test_combine_and_its_gradient(ctx, T, k, E, kind, dtype):
    rng = np.random.default_rng(T + k)
    idx = _choices(rng, T, k, E, kind)
    o, order = fp8.order(idx, E), _order(ctx, idx, E)
    R = o["rows"]
    for C, ldy, ldo in ((1, 1, 1), (300, 307, 303), (2500, 2500, 2500)):
        _say("combine", T, k, E, kind, dtype, C)
        Y, dout = _stored(rng.standard_normal((R, ldy)), dtype), _stored(rng.standard_normal((T, ldo)), dtype)
        live = o["pair"] >= 0
        Y[~live] = np.nan
        w = np.float32(rng.standard_normal((T, k)))
        dY, dw, dd = _up(ctx, Y, dtype), ctx.upload(w), _up(ctx, dout, dtype)
        y = np.where(live[:, None], Y[:, :C], 0.0)
        for ww, buf in ((w, dw), (None, None)):
            out = _up(ctx, np.full((T, ldo), 7.0), dtype)
            ctx.experts_combine(order, dY, buf, out, T, k, E, C, dtype=DT[dtype], ldy=ldy, ldo=ldo)
            ctx.wait(60_000)
            got, want = _down(ctx, out, dtype, (T, ldo)), fp8.combine(o, y, ww)
            # a rounding a term, and half a unit of bf16
            size = fp8.combine(o, np.abs(y), None if ww is None else np.abs(ww))
            assert (np.abs(got[:, :C] - want) <= 2.0**-23 * k * size + (2.0**-8 * np.abs(want) if dtype == "bf16" else 0)).all()
            assert (got[:, C:] == 7).all()
            out.free()
        g = ctx.upload(np.full((T, k), -9, np.float32))
        ctx.experts_combine_grad(order, dY, dd, g, T, k, E, C, dtype=DT[dtype], ldy=ldy, ldo=ldo)
        ctx.wait(60_000)
        want, size = np.zeros((T, k)), np.zeros((T, k))
        for t, j in zip(*np.nonzero(o["slot"] >= 0)):
            p = y[o["slot"][t, j]] * dout[t, :C]
            want[t, j], size[t, j] = p.sum(), np.abs(p).sum()
        # a lane adds C / 64 products one by one, and seven steps join the lanes
        assert (np.abs(ctx.download(g) - want) <= 2.0**-24 * (C / 64 + 16) * size).all()
        _free(dY, dw, dd, g)
    order.free()


# ---------------------------------------------------------------- the MLP
def _mlp_case(rng, T, k, E, kind, D, F, N):
    idx = _choices(rng, T, k, E, kind)
    w = np.where((idx >= 0) & (idx < E), rng.random((T, k)), 0).astype(np.float32)
    X = fp8.bf16(rng.standard_normal((T, D))).astype(np.float64)
    return idx, w, X, _experts(rng, E, 2 * F, D), _experts(rng, E, N, F)


def _mlp(o, w, X, V1, V2, F):
    """(out, size): the MLP in 64 bits, and the size that an error of one code of H has in it."""
    T, k = w.shape
    Y, size = np.zeros((o["rows"], V2[0].shape[0])), np.zeros((o["rows"], V2[0].shape[0]))
    x = fp8.rounded(X)
    for e, slots in fp8.used_slots(o):
        h = fp8.rounded(fp8.swiglu(x[o["pair"][slots] // k] @ V1[e].T))
        Y[slots] = h @ V2[e].T
        size[slots] = np.sqrt((h * h) @ (V2[e] * V2[e]).T)
    return fp8.combine(o, Y, w), np.sqrt(fp8.combine(o, size**2, w.astype(np.float64)**2))


MLPS = [(1, 1, 1, "even", 64, 128, 70), (8, 8, 64, "even", 512, 256, 512), (5, 2, 3, "none", 70, 128, 33),
        (333, 2, 7, "holes", 1000, 384, 1000), (300, 2, 3, "one", 200, 256, 130), (90, 3, 4, "twice", 129, 128, 257)]


@pytest.mark.parametrize("T, k, E, kind, D, F, N", MLPS)
def test_mlp(ctx, T, k, E, kind, D, F, N):
    rng = np.random.default_rng(T + D)
    idx, w, X, (Q1, S1, V1), (Q2, S2, V2) = _mlp_case(rng, T, k, E, kind, D, F, N)
    o, order = fp8.order(idx, E), _order(ctx, idx, E)
    want, size = _mlp(o, w, X, V1, V2, F)
    xq = [ctx.upload(v) for v in fp8.pack(X)]
    W = [ctx.upload(v) for v in (Q1, S1, Q2, S2)]
    dw, hq = ctx.upload(w), _packed(ctx, o["rows"], F)
    for dtype, ldo in (("bf16", N), ("f32", N + 3)):
        _say("mlp", T, k, E, kind, D, F, N, dtype)
        Y, out = _up(ctx, np.full((o["rows"], N), 7.0), dtype), _up(ctx, np.full((T, ldo), 7.0), dtype)
        ctx.experts_mlp_fp8(order, dw, *xq, *W, *hq, Y, out, T, k, E, D, F, N, dtype=DT[dtype], ldo=ldo)
        ctx.wait(60_000)
        got = _down(ctx, out, dtype, (T, ldo))
        # Fused sums differ from the 64-bit ones by 2^-13 of a product at most, 2^-16 of a sum as a rule: one code of H
        # in some hundred is its neighbour, 2^-3 of its value off.  All of them at random: 2^-3 / sqrt(100) of the
        # size, of which eight times are allowed; and the roundings of Y and out.
        bound = 0.1 * size + (2.0**-7 * (np.abs(want) + size) if dtype == "bf16" else 0)
        assert (np.abs(got[:, :N] - want) <= bound).all()
        if want.any():
            assert np.linalg.norm(got[:, :N] - want) <= (2.0**-6 if dtype == "bf16" else 2.0**-7) * np.linalg.norm(size)
        assert (got[:, N:] == 7).all()
        h = np.zeros((o["rows"], 1), bool)  # H of padding is not written
        h[o["pair"] >= 0] = True
        assert (ctx.download(hq[0])[~h[:, 0]] == 0xA5).all()
        _free(Y, out)
    _free(order, dw, *xq, *W, *hq)
