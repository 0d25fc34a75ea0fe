"""The 8-bit operators, the routing and the experts' products as they are used
together: a served step and a training step, recorded, captured by a caller, on
several streams, on tensors past 2^32 bytes; and what the entry points refuse."""
import numpy as np
import pytest

import aiehlc_amd as mi
import fp8_oracle as fp8
from hip_capture import Capture
from test_gpu_experts import SCORING, _down, _experts, _free, _mlp, _packed, _say, _up

pytestmark = pytest.mark.gpu


def _transposed(Q, S, rows, cols):
    """Packed weights of experts, block 128, packed along the other axis: the same codes and scales."""
    qt = np.zeros((len(Q), cols, fp8.up(rows)), np.uint8)
    qt[:, :, :rows] = Q[:, :, :cols].transpose(0, 2, 1)
    return qt, np.ascontiguousarray(S.transpose(0, 2, 1))


class Step:
    """A layer of experts in bf16: forward, and all of its gradients."""

    def __init__(self, ctx, T, k, E, D, F, N, seed, scoring="softmax"):
        rng = np.random.default_rng(seed)
        self.ctx, self.sizes, self.scoring = ctx, (T, k, E, D, F, N), scoring
        self.X, self.dout = (fp8.bf16(rng.standard_normal((T, n))).astype(np.float64) for n in (D, N))
        self.logits = np.float32(rng.standard_normal((T, E)))
        self.logits[T - T // 10:] = -np.inf  # the padding of a batch
        self.W1, self.W2 = _experts(rng, E, 2 * F, D), _experts(rng, E, N, F)
        R = self.R = mi.experts_rows(T, k, E)
        up = ctx.upload
        self.x, self.g, self.l = _up(ctx, self.X, "bf16"), _up(ctx, self.dout, "bf16"), up(self.logits)
        self.w1, self.w2 = [up(v) for v in self.W1[:2]], [up(v) for v in self.W2[:2]]
        self.w1t, self.w2t = [up(v) for v in _transposed(*self.W1[:2], 2 * F, D)], [up(v) for v in _transposed(*self.W2[:2], N, F)]
        self.xq, self.h, self.hs, self.gq, self.dgu = (_packed(ctx, *s) for s in ((T, D), (R, F), (R, F), (R, N), (R, 2 * F)))
        self.xt, self.ht, self.gt, self.dgut = (_packed(ctx, n, R) for n in (D, F, N, 2 * F))
        e16, e32 = (lambda *s: ctx.upload(np.zeros(s, np.uint16))), (lambda *s: ctx.upload(np.zeros(s, np.float32)))
        self.order = up(np.zeros(mi.experts_order_bytes(T, k, E) // 4, np.int32))
        self.served, self.out, self.dx = e16(T, N), e16(T, N), e16(T, D)
        self.y, self.ys, self.gu, self.dxs = e16(R, N), e16(R, N), e16(R, 2 * F), e16(R, D)
        self.idx, self.w, self.dw = up(np.zeros((T, k), np.int32)), e32(T, k), e32(T, k)
        self.dh, self.dl, self.dw1, self.dw2 = e32(R, F), e32(T, E), e32(E, 2 * F, D), e32(E, N, F)

    def serve(self, ctx=None):
        c, (T, k, E, D, F, N) = ctx or self.ctx, self.sizes
        c.route_experts(self.l, None, self.idx, self.w, T, k, E, scoring=SCORING[self.scoring])
        c.experts_order(self.idx, self.order, T, k, E)
        c.quant_fp8(self.x, T, D, *self.xq)
        c.experts_mlp_fp8(self.order, self.w, *self.xq, *self.w1, *self.w2, *self.hs, self.ys, self.served, T, k, E, D, F, N)

    def train(self, ctx=None):
        c, (T, k, E, D, F, N) = ctx or self.ctx, self.sizes
        o, s = self.order, (T, k, E)
        c.route_experts(self.l, None, self.idx, self.w, *s, scoring=SCORING[self.scoring])
        c.experts_order(self.idx, o, *s)
        c.quant_fp8(self.x, T, D, *self.xq)
        c.experts_gemm_fp8(o, *self.xq, *self.w1, self.gu, *s, 2 * F, D, gather=True)
        c.experts_swiglu_fp8(o, self.gu, *self.h, *self.ht, *s, F)
        c.experts_gemm_fp8(o, *self.h, *self.w2, self.y, *s, N, F)
        c.experts_combine(o, self.y, self.w, self.out, *s, N)
        c.experts_combine_grad(o, self.y, self.g, self.dw, *s, N)
        c.route_experts_grad(self.l, self.idx, self.dw, self.dl, *s, scoring=SCORING[self.scoring])
        c.experts_quant_fp8(o, self.g, self.w, *self.gq, *self.gt, *s, N)
        c.experts_quant_fp8(o, self.x, None, None, None, *self.xt, *s, D)
        c.experts_gemm_fp8(o, *self.gq, *self.w2t, self.dh, *s, F, N, dtype=mi.F32)
        c.experts_swiglu_grad_fp8(o, self.gu, self.dh, *self.dgu, *self.dgut, *s, F)
        c.experts_gemm_fp8(o, *self.dgu, *self.w1t, self.dxs, *s, D, 2 * F)
        c.experts_combine(o, self.dxs, None, self.dx, *s, D)
        c.experts_wgrad_fp8(o, *self.gt, *self.ht, self.dw2, *s, N, F)
        c.experts_wgrad_fp8(o, *self.dgut, *self.xt, self.dw1, *s, 2 * F, D)

    RESULTS = ["idx", "w", "served", "out", "dw", "dl", "dx", "dw1", "dw2"]

    def results(self):
        return {n: self.ctx.download(getattr(self, n)) for n in self.RESULTS}

    def clear(self):
        for n in self.RESULTS:
            b = getattr(self, n)
            self.ctx.copy_h2d(b, np.full(b.shape, 9, b.dtype))

    def free(self):
        for v in vars(self).values():
            for b in v if isinstance(v, (list, tuple)) else (v,):
                if isinstance(b, mi.DeviceBuffer):
                    b.free()


def _same(got, want):
    for n in want:
        assert np.array_equal(got[n], want[n]), n


STEPS = [(1, 1, 1, 128, 128, 64), (120, 2, 4, 256, 256, 200), (40, 3, 16, 300, 128, 257), (700, 2, 3, 129, 128, 130)]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("sizes", STEPS)
def test_a_layer_and_its_gradients(ctx, sizes, scoring):
    T, k, E, D, F, N = sizes
    _say("layer", sizes, scoring)
    st = Step(ctx, *sizes, seed=T + E, scoring=scoring)
    st.serve()
    st.train()
    ctx.wait(60_000)
    r = st.results()
    want_i, want_w = fp8.route(st.logits, None, k, scoring)
    assert np.array_equal(r["idx"], want_i)
    assert (np.abs(r["w"] - want_w) <= 2.0**-23 * want_w).all()
    w, o = r["w"].astype(np.float64), fp8.order(want_i, E)
    V1, V2 = st.W1[2], st.W2[2]
    served, size = _mlp(o, w, st.X, V1, V2, F)
    got = _down(ctx, st.served, "bf16", (T, N))
    # (as tests/test_gpu_experts.py derives them)
    assert np.linalg.norm(got - served) <= 2.0**-6 * np.linalg.norm(size)
    # The gradients in 64 bits of the layer without 8-bit roundings, W apart.  A packed element is off by 2^-4 of itself
    # at most, spread over the step: 2^-4 / sqrt(3) of a matrix in the 2-norm, which products of independent terms
    # keep.  Of X, H, dout w and d(gate, up) at most four are in a result; a derivative of silu is at most 1.1 and
    # moves with its argument, so X counts twice: sqrt(5) 2^-4 / sqrt(3) = 0.081 of a result whose terms are
    # independent.  bf16 adds 2^-9 / sqrt(3) for each of GU, Y and the result.
    dX, dW1, dW2, dw = np.zeros((T, D)), np.zeros((E, 2 * F, D)), np.zeros((E, N, F)), np.zeros((T, k))
    sizes_dw = np.zeros((T, k))
    for e, slots in fp8.used_slots(o):
        pair = o["pair"][slots]
        t, j = pair // k, pair % k
        gu = st.X[t] @ V1[e].T
        h, g = fp8.swiglu(gu), st.dout[t] * w[t, j][:, None]
        d = fp8.swiglu_grad(gu, g @ V2[e])
        y = h @ V2[e].T
        dw[t, j] = (y * st.dout[t]).sum(1)
        sizes_dw[t, j] = np.linalg.norm(y, axis=1) * np.linalg.norm(st.dout[t], axis=1) / np.sqrt(N)
        np.add.at(dX, t, d @ V1[e])
        dW1[e], dW2[e] = d.T @ st.X[t], g.T @ h
    out = {"dx": _down(ctx, st.dx, "bf16", (T, D)), "dw1": r["dw1"].astype(np.float64), "dw2": r["dw2"].astype(np.float64)}
    for n, want in (("dx", dX), ("dw1", dW1), ("dw2", dW2)):
        assert np.linalg.norm(out[n] - want) <= 0.1 * np.linalg.norm(want), (n, np.linalg.norm(out[n] - want) / np.linalg.norm(want))
    # dw = <dout, Y>: a sum of N terms of random signs, off by as much of its size (single sums of three such sizes)
    assert np.linalg.norm(r["dw"] - dw) <= 0.1 * (1 + 3 / np.sqrt(T * k)) * np.linalg.norm(sizes_dw), "dw"
    dl = fp8.route_grad(st.logits, want_i, r["dw"].astype(np.float64), scoring, True, 1.0)
    terms = fp8.route_grad_terms(st.logits, want_i, r["dw"].astype(np.float64), scoring, True, 1.0)
    assert (np.abs(r["dl"] - dl) <= 2.0**-20 * terms + 1e-30).all()
    pad = st.logits[:, 0] == -np.inf if T >= 10 else np.zeros(T, bool)
    for n in ("out", "served", "dx", "dw", "dl"):  # tokens of padding
        assert not r[n][pad].any(), n
    st.clear()  # again: the same bits
    st.serve()
    st.train()
    ctx.wait(60_000)
    _same(st.results(), r)
    st.free()


def test_recorded_steps(ctx):
    _say("recorded")
    st = Step(ctx, 120, 2, 4, 256, 256, 200, seed=5)
    st.serve()
    st.train()
    ctx.wait(60_000)
    want = st.results()
    with ctx.record() as chain:
        st.serve()
        st.train()
    for rep in range(4):
        st.clear()
        chain.launch()
        ctx.wait(60_000)
        _same(st.results(), want)
        st.train()  # eager work of the program's own between the replays
        ctx.wait(60_000)
        _same(st.results(), want)
    st.free()


def test_captured_steps_replay_on_another_stream():
    """Two graphs of one caller, replayed together with eager steps of the context: nothing is shared."""
    _say("captured")
    cap = Capture()
    try:
        steps = [Step(cap.ctx, 120, 2, 4, 256, 256, 200, seed=5), Step(cap.ctx, 33, 3, 8, 256, 128, 130, seed=6),
                 Step(cap.ctx, 2, 2, 8, 300, 128, 70, seed=7)]
        for st in steps:
            st.serve()
            st.train()
        cap.sync()
        want = [st.results() for st in steps]

        def both(st):
            st.serve()
            st.train()

        graphs = [cap.record(lambda st=st: both(st)) for st in steps[:2]]
        for rep in range(4):
            for st in steps:
                st.clear()
            cap.sync()
            for exe, grids in graphs:
                assert len(grids) >= 20  # kernels alone
                cap.replay(exe)
            both(steps[2])
            cap.sync()
            for st, w in zip(steps, want):
                _same(st.results(), w)
        for st in steps:
            st.free()
        for exe, _ in graphs:
            cap.ok(cap.hip.hipGraphExecDestroy(exe))
    finally:
        cap.close()


def test_two_streams_at_once(ctx):
    """Steps of two contexts, their calls interleaved without waiting; weights of the other's stream."""
    _say("two streams")
    other = mi.Context(0)
    try:
        a, b = Step(ctx, 120, 2, 4, 256, 256, 200, seed=5), Step(other, 90, 2, 8, 256, 256, 130, seed=9)
        for st in (a, b):
            st.serve()
            st.train()
            st.ctx.wait(60_000)
        want = a.results(), b.results()
        for st in (a, b):
            st.clear()
        for _ in range(3):
            a.serve()
            b.train()
            a.train()
            b.serve()
        ctx.wait(60_000)
        other.wait(60_000)
        _same(a.results(), want[0])
        _same(b.results(), want[1])
        b.train(ctx)  # the same buffers on the other context, which has nothing of its own in them
        ctx.wait(60_000)
        _same(b.results(), want[1])
        a.free()
        b.free()
    finally:
        other.close()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_scores_that_round_to_the_same(ctx, scoring):
    """Without a bias the larger logit comes first, with one (of zeros) the lower index of equal scores."""
    _say("equal scores", scoring)
    if scoring == "sigmoid":
        row = [40.0, 60.0, -3.0, 50.0, 60.0, 1e30, 2.0]      # 1 in 64 bits above 37
    else:
        row = [0.0, 1e-20, -1000.0, -900.0, 1e-30, -800.0, -1e-25]  # e^x is 1, or 0 next to the others
    E, k = len(row), 6
    by_logit = sorted(range(E), key=lambda e: (-row[e], e))[:k]
    s = fp8.scores(np.float64([row]), scoring)[0]
    by_score = sorted(range(E), key=lambda e: (-s[e], e))[:k]
    assert by_logit != by_score
    l, zero = ctx.upload(np.float32([row])), ctx.upload(np.zeros(E, np.float32))
    idx, w = ctx.empty((1, k), np.int32), ctx.empty((1, k), np.float32)
    for bias, want in ((None, by_logit), (zero, by_score)):
        ctx.route_experts(l, bias, idx, w, 1, k, E, scoring=SCORING[scoring], renormalize=False)
        ctx.wait(60_000)
        assert ctx.download(idx)[0].tolist() == want
        assert (np.abs(ctx.download(w)[0] - s[want]) <= 2.0**-23 * s[want]).all()
    _free(l, zero, idx, w)


@pytest.mark.parametrize("R, C", [(40, 70), (384, 300), (128, 128)])
def test_matrices_of_experts_packed_one_after_another(ctx, R, C):
    """Along both axes; an expert's scales start wherever the one's before end."""
    _say("experts' weights", R, C)
    E = 3
    W = fp8.bf16(np.random.default_rng(R).standard_normal((E, R, C))).astype(np.float64)
    (sq, ss), (tq, ts) = mi.fp8_shapes(R, C, 128), mi.fp8_shapes(C, R, 128)
    d = [_up(ctx, w, "bf16") for w in W]
    q, s, t, u = (ctx.empty((E, *n), dt) for n, dt in ((sq, np.uint8), (ss, np.float32), (tq, np.uint8), (ts, np.float32)))
    for e in range(E):
        ctx.quant_fp8(d[e], R, C, q.ptr + e * np.prod(sq), s.ptr + 4 * e * np.prod(ss), t.ptr + e * np.prod(tq),
                      u.ptr + 4 * e * np.prod(ts), block=128)
    ctx.wait(60_000)
    for e in range(E):
        for got_q, got_s, x in ((q, s, W[e]), (t, u, W[e].T)):
            Q, S = fp8.pack(x, 128)
            assert np.array_equal(ctx.download(got_q)[e], Q) and np.array_equal(ctx.download(got_s)[e], S)
    _free(*d, q, s, t, u)


# ---------------------------------------------------------------- beyond 2^32 bytes
def _at(ctx, buf, offset, arr):
    """Writes arr at a byte offset of a buffer."""
    arr = np.ascontiguousarray(arr)
    ctx.copy_h2d(mi.DeviceBuffer(ctx, buf.ptr + offset, arr.nbytes), arr)


def _part(ctx, buf, offset, dtype, shape):
    return ctx.download(mi.DeviceBuffer(ctx, buf.ptr + offset, 0), dtype, shape)


@pytest.mark.parametrize("M", [2, 70])
def test_weights_past_32_bits(ctx, M):
    """B of 4.9e9 bytes, of which the first and last rows are looked at (an element 0x7f in memory as it comes is a NaN
    of its own column)."""
    N, K = 600_000, 8192
    _say("long weights", M)
    rng = np.random.default_rng(M)
    qA, sA = fp8.pack(rng.standard_normal((M, K)))
    rows = 128
    Q, S = fp8.pack(rng.standard_normal((2 * rows, K)), 128)
    ends = slice(0, rows), slice(N - N % 128, N)
    B, C = ctx.empty((N, K), np.uint8), ctx.empty((M, N), np.float32)
    scales = np.ones((K // 128, -(-N // 128)), np.float32)
    scales[:, 0], scales[:, -1] = S[:, 0], S[:, 1]
    _at(ctx, B, 0, Q[:rows])
    _at(ctx, B, ends[1].start * K, Q[rows:rows + N % 128])
    d = [ctx.upload(v) for v in (qA, sA, scales)]
    ctx.gemm_fp8(d[0], d[1], B, d[2], C, M, N, K)
    ctx.wait(60_000)
    got, a, b = ctx.download(C), fp8.values(qA, sA, M, K), fp8.values(Q, S, 2 * rows, K, 128)
    for at, part in ((ends[0], b[:rows]), (ends[1], b[rows:rows + N % 128])):
        assert (np.abs(got[:, at] - a @ part.T) <= fp8.product_bound(a, part)).all()
    _free(B, C, *d)


def test_a_result_past_32_bits(ctx):
    M, N, K = 70_000, 20_000, 128
    _say("large result")
    rng = np.random.default_rng(4)
    A, (qB, sB) = rng.standard_normal((256, K)), fp8.pack(rng.standard_normal((N, K)), 128)
    qa, sa = fp8.pack(A)
    qA, sA = np.zeros((M, K), np.uint8), np.ones((1, M), np.float32)
    qA[-256:], sA[:, -256:] = qa, sa
    d, C = [ctx.upload(v) for v in (qA, sA, qB, sB)], ctx.empty((M, N), np.float32)
    ctx.gemm_fp8(*d, C, M, N, K)
    ctx.wait(60_000)
    got = _part(ctx, C, 4 * (M - 256) * N, np.float32, (256, N))
    a, b = fp8.values(qa, sa, 256, K), fp8.values(qB, sB, N, K, 128)
    assert (np.abs(got - a @ b.T) <= fp8.product_bound(a, b)).all()
    assert not _part(ctx, C, 4 * (M - 257) * N, np.float32, (N,)).any()
    _free(C, *d)


def test_a_conversion_past_32_bits(ctx):
    R, C = 300_000, 8192
    _say("large conversion")
    X, tail = ctx.empty((R, C), np.uint16), 200
    x = fp8.bf16(np.random.default_rng(1).standard_normal((tail, C))).astype(np.float64)
    _at(ctx, X, 2 * (R - tail) * C, fp8.bf16_bits(x))
    q, t = [ctx.empty(s, dt) for s, dt in zip(mi.fp8_shapes(R, C), (np.uint8, np.float32))], [
        ctx.empty(s, dt) for s, dt in zip(mi.fp8_shapes(C, R), (np.uint8, np.float32))]
    ctx.quant_fp8(X, R, C, *q, *t)
    Y = ctx.empty((R, C), np.float32)
    ctx.dequant_fp8(*q, Y, R, C, dtype=mi.F32)
    ctx.wait(60_000)
    Q, S = fp8.pack(x)
    assert np.array_equal(_part(ctx, q[0], (R - tail) * C, np.uint8, (tail, C)), Q)
    assert np.array_equal(ctx.download(q[1])[:, R - tail:], S)
    assert np.array_equal(_part(ctx, Y, 4 * (R - tail) * C, np.float32, (tail, C)), fp8.values(Q, S, tail, C))
    last = R // 128 * 128  # the last block along the columns: rows 299904 on
    Qt, St = fp8.pack(x[last - R:].T)
    assert np.array_equal(_part(ctx, t[0], (C - 1) * fp8.up(R) + last, np.uint8, (128,)), Qt[-1])
    assert np.array_equal(ctx.download(t[1])[-1], St[0])
    _free(X, Y, *q, *t)


def test_slots_past_32_bits(ctx):
    """330000 slots of 16384 columns (5.4e9 bytes) of one expert."""
    T, E, N, K = 330_000, 1, 40, 16384
    _say("many slots")
    rng = np.random.default_rng(2)
    idx, order = ctx.upload(np.zeros((T, 1), np.int32)), ctx.empty((mi.experts_order_bytes(T, 1, E) // 4,), np.int32)
    R, tail = mi.experts_rows(T, 1, E), 300
    (sq, ss), A = mi.fp8_shapes(R, K), rng.standard_normal((tail, K))
    q, s = ctx.empty(sq, np.uint8), np.ones(ss, np.float32)
    Q, S = fp8.pack(A)
    s[:, T - tail:T] = S
    _at(ctx, q, (T - tail) * K, Q)
    W = _experts(rng, E, N, K)
    d, C = [ctx.upload(v) for v in (s, *W[:2])], ctx.empty((R, N), np.float32)
    ctx.experts_order(idx, order, T, 1, E)
    ctx.experts_gemm_fp8(order, q, d[0], d[1], d[2], C, T, 1, E, N, K, dtype=mi.F32)
    ctx.wait(60_000)
    a = fp8.values(Q, S, tail, K)
    got = _part(ctx, C, 4 * (T - tail) * N, np.float32, (tail, N))
    assert (np.abs(got - a @ W[2][0].T) <= fp8.product_bound(a, W[2][0])).all()
    _free(idx, order, q, C, *d)


# ---------------------------------------------------------------- refusals
def test_refusals(ctx):
    d = ctx.upload(np.full(1 << 16, 0x5A, np.uint8))
    p, F32, BF16 = d.ptr, mi.F32, mi.BF16

    def refused(name, *args, text):
        assert ctx.call_status("miaie_" + name, *args) == mi.MIAIE_EINVAL, (name, args)
        assert text in ctx.last_error(), ctx.last_error()

    def one_by_one(name, good, bad):
        """Each argument (position, value, text) in place of a good one."""
        for at, value, text in bad:
            args = list(good)
            args[at] = value
            refused(name, *args, text=text)

    one_by_one("quant_fp8", (p, F32, 4, 4, 4, 1, p, p, p, p),
               [(0, None, "X is NULL"), (0, p + 2, "misaligned"), (1, 2, "dtype=2"), (2, 0, "R=0"), (3, (1 << 30) + 1, "C="),
                (4, 3, "ldx=3"), (5, 64, "block=64"), (6, None, "Xq is NULL"), (7, None, "Xs is NULL"), (8, p + 8, "16-byte"),
                (9, None, "Xts is NULL")])
    refused("quant_fp8", p, F32, 4, 4, 4, 1, None, None, None, None, text="all NULL")
    refused("quant_fp8", p, F32, 1 << 30, 128, 128, 1, p, p, None, None, text="too large")
    one_by_one("dequant_fp8", (p, p, 1, p, F32, 4, 4, 4),
               [(0, p + 1, "16-byte"), (1, None, "Xs is NULL"), (2, 0, "block=0"), (3, None, "Y is NULL"), (3, p + 1, "misaligned"),
                (4, 7, "dtype=7"), (5, -1, "R=-1"), (6, 0, "C=0"), (7, 3, "ldy=3")])
    one_by_one("gemm_fp8", (p, p, p, p, 128, p, BF16, 4, 4, 4, 4),
               [(0, None, "Aq is NULL"), (1, p + 2, "4-byte"), (2, None, "Bq is NULL"), (3, None, "Bs is NULL"), (4, 2, "b_block=2"),
                (5, None, "C is NULL"), (5, p + 1, "misaligned"), (6, 4, "dtype=4"), (7, 0, "M=0"), (8, (1 << 25) + 1, "N="),
                (9, (1 << 23) + 1, "K="), (10, 3, "ldc=3")])
    refused("gemm_fp8", p, p, p, p, 128, p, BF16, 1 << 25, 1 << 25, 4, 1 << 25, text="too large")
    #                         logits, dtype, bias, idx, w, tokens, top_k, experts, ld, scoring, groups, kept, top, renorm, scale
    one_by_one("route_experts", (p, F32, p, p, p, 4, 2, 8, 8, 0, 4, 2, 1, 1, 1.0),
               [(0, None, "logits is NULL"), (1, 5, "dtype=5"), (2, p + 2, "bias"), (3, None, "idx is NULL"), (4, None, "w is NULL"),
                (5, 0, "tokens=0"), (6, 0, "top_k=0"), (6, 65, "top_k=65"), (6, 5, "top_k=5 of 4"), (7, 1025, "experts=1025"),
                (8, 7, "ld=7"), (9, 2, "scoring=2"), (10, 3, "does not divide"), (10, 0, "groups=0"), (11, 5, "groups_kept=5"),
                (12, 3, "group_top=3"), (13, 2, "renormalize=2"), (14, float("nan"), "scale"), (14, float("inf"), "scale")])
    one_by_one("route_experts_grad", (p, F32, p, p, p, 4, 2, 8, 8, 8, 0, 1, 1.0),
               [(0, p + 1, "misaligned"), (2, None, "idx is NULL"), (3, None, "dw is NULL"), (4, None, "dlogits is NULL"),
                (5, (1 << 25) + 1, "tokens"), (8, 7, "ld=7"), (9, 7, "ldd=7"), (10, -1, "scoring=-1"), (11, -1, "renormalize=-1")])
    one_by_one("experts_order", (p, p, 4, 2, 8),
               [(0, None, "idx is NULL"), (1, None, "order is NULL"), (1, p + 2, "order"), (2, 0, "tokens=0"),
                (2, 1 << 23, "tokens=8388608"), (3, 65, "top_k=65"), (4, 0, "experts=0")])
    #            order w  X       W1      W2      H      Y  out dtype T  k  E   D   F  N  ldo
    mlp = (p, p, p, p, p, p, p, p, p, p, p, p, BF16, 4, 2, 8, 16, 128, 16, 16)
    one_by_one("experts_mlp_fp8", mlp,
               [(0, None, "order is NULL"), (1, None, "w is NULL"), (2, None, "Xq is NULL"), (4, p + 8, "16-byte"), (7, None, "W2s is NULL"),
                (8, None, "Hq is NULL"), (10, p + 1, "Y"), (11, None, "out is NULL"), (12, 3, "dtype=3"), (13, 0, "tokens=0"),
                (16, 0, "D=0"), (17, 64, "F=64"), (17, 0, "F=0"), (18, (1 << 20) + 1, "Nout="), (19, 15, "ldo=15")])
    refused("experts_mlp_fp8", *mlp[:13], 1 << 20, 2, 8, 4096, 128, 16, 16, text="2^32 bytes")
    refused("experts_mlp_fp8", *mlp[:13], 4, 2, 8, 1 << 20, 4096, 16, 16, text="2^32 bytes")
    one_by_one("experts_gemm_fp8", (p, p, p, p, p, p, F32, 4, 2, 8, 16, 16, 16, 0),
               [(0, p + 1, "order"), (1, None, "Aq is NULL"), (4, None, "Bs is NULL"), (5, None, "C is NULL"), (6, 9, "dtype=9"),
                (8, 0, "top_k=0"), (10, 0, "N=0"), (11, (1 << 20) + 1, "K="), (12, 15, "ldc=15"), (13, 2, "gather=2")])
    refused("experts_gemm_fp8", p, p, p, p, p, p, F32, 1 << 20, 8, 64, 1 << 20, 16, 1 << 20, 0, text="too large")
    refused("experts_gemm_fp8", p, p, p, p, p, p, F32, 1 << 20, 2, 8, 16, 4096, 16, 1, text="2^32 bytes")
    one_by_one("experts_quant_fp8", (p, p, BF16, p, p, p, p, p, 4, 2, 8, 16, 16),
               [(1, None, "X is NULL"), (2, 2, "dtype=2"), (3, p + 2, "w"), (4, None, "Xq is NULL"), (7, None, "Xts is NULL"),
                (10, 0, "experts=0"), (11, 0, "C=0"), (12, 15, "ldx=15")])
    refused("experts_quant_fp8", p, p, BF16, None, None, None, None, None, 4, 2, 8, 16, 16, text="all NULL")
    one_by_one("experts_swiglu_fp8", (p, p, BF16, p, p, p, p, 4, 2, 8, 128, 256),
               [(1, None, "GU is NULL"), (3, None, "Xq is NULL"), (10, 130, "F=130"), (11, 255, "ldgu=255")])
    one_by_one("experts_swiglu_grad_fp8", (p, p, BF16, p, p, p, p, p, 4, 2, 8, 128, 256, 128),
               [(1, p + 1, "GU"), (3, None, "dH is NULL"), (4, None, "Xq is NULL"), (11, 100, "F=100"), (12, 255, "ldgu=255"),
                (13, 127, "ldh=127")])
    one_by_one("experts_wgrad_fp8", (p, p, p, p, p, p, F32, 4, 2, 8, 16, 16, 16),
               [(1, None, "Atq is NULL"), (4, p + 2, "4-byte"), (5, None, "C is NULL"), (10, 0, "M=0"), (11, 0, "N=0"), (12, 15, "ldc=15")])
    refused("experts_wgrad_fp8", p, p, p, p, p, p, F32, 4, 2, 8, 1 << 20, 1 << 20, 1 << 20, text="too large")
    one_by_one("experts_combine", (p, p, p, p, F32, 4, 2, 8, 16, 16, 16),
               [(1, None, "Y is NULL"), (2, p + 2, "w"), (3, None, "out is NULL"), (8, 0, "C=0"), (9, 15, "ldy=15"), (10, 15, "ldo=15")])
    one_by_one("experts_combine_grad", (p, p, p, p, F32, 4, 2, 8, 16, 16, 16),
               [(1, None, "Y is NULL"), (2, None, "dout is NULL"), (3, None, "dw is NULL"), (9, 15, "ldy=15"), (10, 0, "ldo=0")])
    ctx.wait(10_000)
    assert (ctx.download(d) == 0x5A).all()
    d.free()
