"""The norms around a block and their gradients through the C ABI against the
64-bit oracle (tests/mx_oracle.py).

Tolerances: every fp32 operation is off by at most 2^-24 of its result; a value
of out or y takes fewer than 16 of them, the mean under a root sums squares in
chains of at most 16 + 10 additions (half of their error reaches the root), so
2^-19 of the terms' magnitudes covers both; a result stored in bf16 is off by
2^-9 more (2^-8 allowed).  A gradient is a sum of terms that may cancel: its
bound is 2^-19 of the sum of their magnitudes; a sum over rows adds up to
rows / 256 + 256 values in chains: (rows / 256 + 256) 2^-24 of the magnitudes' sum
more.  The second norm and the gradients are compared from the stored stream."""
import numpy as np
import pytest

import aiehlc_amd as mi
import mx_oracle as mx

pytestmark = pytest.mark.gpu

DT = {"f32": mi.F32, "bf16": mi.BF16}
REL = 2.0**-19


def _q(x, dtype):
    return (mx.bf16(x) if dtype == "bf16" else np.float32(x)).astype(np.float64)


def _up(ctx, x, dtype, ld=None):
    x = np.asarray(x)
    if ld is not None and ld != x.shape[1]:
        w = np.full((x.shape[0], ld), 9.0)
        w[:, :x.shape[1]] = x
        x = w
    return ctx.upload(mx.bf16_bits(x) if dtype == "bf16" else np.float32(x))


def _down(ctx, buf, dtype, shape):
    if dtype == "bf16":
        return mx.from_bf16_bits(ctx.download(buf, np.uint16, shape)).astype(np.float64)
    return ctx.download(buf, np.float32, shape).astype(np.float64)


def _close(got, want, bound, dtype="f32", what=""):
    bound = bound + (2.0**-8 if dtype == "bf16" else 2.0**-23) * np.abs(want) + 1e-37
    far = np.abs(got - want) / bound
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert not (far > 1).any(), (what, float(np.nanmax(far)))


CASES = [  # rows, cols, stream, branch, gate_rows (None: no gate), parts
    (1, 4096, "bf16", "bf16", None, "ab"), (1, 1, "f32", "f32", 1, "ab"), (3, 7, "f32", "bf16", 2, "ab"),
    (5, 64, "bf16", "f32", 5, "ab"), (7, 511, "bf16", "bf16", 1, "ab"), (33, 513, "f32", "f32", 10, "ab"),
    (9, 1024, "f32", "bf16", 4, "ab"), (300, 1025, "bf16", "bf16", 300, "ab"), (130, 2048, "f32", "bf16", 1, "ab"),
    (64, 4095, "bf16", "bf16", 16, "ab"), (17, 5000, "f32", "f32", 17, "ab"), (12, 8192, "bf16", "bf16", 5, "ab"),
    (4, 16384, "f32", "bf16", 4, "ab"), (3, 16383, "bf16", "f32", 1, "ab"), (1000, 96, "bf16", "bf16", 3, "ab"),
    (2000, 33, "f32", "f32", 2000, "ab"), (50, 1000, "bf16", "bf16", None, "b"), (50, 1000, "f32", "bf16", None, "a"),
    (20, 4096, "bf16", "bf16", 7, "a"),
    # several turns of a gradient's workgroups: over gates, and over the rows of one gate
    (600, 4100, "f32", "bf16", 1, "ab"), (1100, 2100, "bf16", "bf16", 2, "ab"), (300, 8200, "bf16", "f32", 1, "ab"),
    (9000, 33, "f32", "f32", None, "ab"), (1300, 2500, "f32", "f32", 1300, "ab"), (700, 8300, "bf16", "bf16", 350, "ab"),
]


def _make(rng, rows, cols, st, bt, gate_rows, parts):
    t = {"x": _q(rng.standard_normal((rows, cols)) * np.exp2(3 * rng.random(cols)), st)}
    if "a" in parts:
        t["b"] = _q(rng.standard_normal((rows, cols)) * 0.5, bt)
        t["w_after"] = _q(1 + 0.1 * rng.standard_normal(cols), "f32")
        if gate_rows:
            t["gate"] = _q(rng.standard_normal((-(-rows // gate_rows), cols)), bt)
    if "b" in parts:
        t["w_before"] = _q(1 + 0.1 * rng.standard_normal(cols), "f32")
    return t


@pytest.mark.parametrize("pad", [0, 5])
@pytest.mark.parametrize("case", CASES)
def test_norm_block_and_its_gradient(ctx, case, pad):
    rows, cols, st, bt, gate_rows, parts = case
    print("[case] norm", case, pad, flush=True)
    rng = np.random.default_rng(rows * 131 + cols)
    t = _make(rng, *case)
    alpha, eps, ldx, ldb, k = 0.75, 1e-3, cols + pad, cols + 2 * pad, gate_rows or rows
    after, before = "a" in parts, "b" in parts
    bufs = []

    def up(x, dtype, ld=None):
        bufs.append(_up(ctx, x, dtype, ld))
        return bufs[-1]

    dx, dwa, dwb = up(t["x"], st, ldx), None, None
    db = up(t["b"], bt, ldb) if after else None
    dgate = up(t["gate"], bt) if "gate" in t else None
    if after:
        dwa = up(t["w_after"], "f32")
    if before:
        dwb = up(t["w_before"], "f32")
    out = up(np.full((rows, ldx), 9.0), st) if after else None
    y = up(np.full((rows, ldb), 9.0), bt) if before else None
    rstd = up(np.full((2, rows), 9.0), "f32")
    kw = {"ldx": ldx, "ldb": ldb, "gate_rows": gate_rows, "stream_dtype": DT[st], "branch_dtype": DT[bt], "alpha": alpha}
    ctx.norm_block(dx, db, dgate, dwa, dwb, out, y, rstd, rows, cols, eps=eps, **kw)
    ctx.wait(60_000)
    r, _, ra, _ = mx.norm_block(t["x"], t.get("b"), t.get("gate"), t.get("w_after"), None, k, alpha, eps)
    if after:
        got = _down(ctx, out, st, (rows, ldx))
        _close(got[:, :cols], r, REL * (np.abs(alpha * t["x"]) + np.abs(r - alpha * t["x"])), st, "out")
        assert (got[:, cols:] == 9).all()
        r = got[:, :cols]  # the stored stream
    _, want_y, _, rb = mx.norm_block(r, None, None, None, t.get("w_before"), k, alpha, eps)
    if before:
        got = _down(ctx, y, bt, (rows, ldb))
        _close(got[:, :cols], want_y, REL * np.abs(want_y), bt, "y")
        assert (got[:, cols:] == 9).all()
    kept = _down(ctx, rstd, "f32", (2, rows))
    if after:
        _close(kept[0], ra, REL * ra, what="rstd")
    if before:
        _close(kept[1], rb, REL * rb, what="rstd")

    # ---- gradient, all results, then each alone and in place
    dout, dy = _q(rng.standard_normal((rows, cols)), st), _q(rng.standard_normal((rows, cols)), bt)
    want = mx.norm_block_grad(r, t.get("b"), t.get("gate"), t.get("w_after"), t.get("w_before"), kept[0], kept[1], dout,
                              dy if before else None, k, alpha)
    rr = up(r, st, ldx)
    ddout, ddy = up(dout, st, ldx), (up(dy, bt, ldb) if before else None)
    shapes = {"dx": (rows, ldx), "db": (rows, ldb), "dgate": t["gate"].shape if "gate" in t else None, "dw_after": (cols,),
              "dw_before": (cols,)}
    types = {"dx": st, "db": bt, "dgate": "f32", "dw_after": "f32", "dw_before": "f32"}
    g = {n: up(np.full(shapes[n], 9.0), types[n]) for n in want}
    nbytes = mi.norm_work_bytes(cols)
    work = ctx.empty((nbytes // 4,), np.float32)
    bufs.append(work)

    def grad(res, d_out=ddout, d_y=ddy, wk=work):
        ctx.norm_block_grad(rr, db, dgate, dwa, dwb, rstd, d_out, d_y, res.get("dx"), res.get("db"), res.get("dgate"),
                            res.get("dw_after"), res.get("dw_before"), wk, nbytes, rows, cols, **kw)
        ctx.wait(60_000)

    grad(g)
    # magnitudes of the terms of each gradient
    mag = _magnitudes(t, r, kept, dout, dy if before else None, k, alpha)
    first = {n: _down(ctx, g[n], types[n], shapes[n]) for n in g}
    chain = (rows / 256 + 256) * 2.0**-24
    for n, w in want.items():
        got = first[n][:, :cols] if first[n].ndim == 2 else first[n]
        _close(got, w, (REL + (chain if n[1] in "gw" else 0)) * mag[n], types[n], n)
        if n in ("dx", "db"):
            assert (first[n][:, cols:] == 9).all()
    grad(g)  # the same call, the same bits
    for n in g:
        assert np.array_equal(first[n], _down(ctx, g[n], types[n], shapes[n])), n
    for n in g:  # one at a time
        one = {n: up(np.full(shapes[n], 9.0), types[n])}
        grad(one, wk=work if types[n] == "f32" and n not in ("dx", "db") else None)
        assert np.array_equal(first[n], _down(ctx, one[n], types[n], shapes[n])), n
    # dx over dout, db over dy
    inplace = {**g, "dx": ddout, **({"db": ddy} if before and after else {})}
    grad(inplace)
    for n in ("dx", "db"):
        if n in inplace:
            assert np.array_equal(first[n], _down(ctx, inplace[n], types[n], shapes[n])), n
    for b in bufs:
        b.free()


def _magnitudes(t, r, kept, dout, dy, k, alpha):
    """Sums of the magnitudes of each gradient's terms."""
    ra, rb = kept[0][:, None], kept[1][:, None]
    dr, m = np.abs(dout), {}
    if dy is not None:
        n, tt = np.abs(r) * rb, np.abs(dy) * np.abs(t["w_before"])
        m["dw_before"] = (np.abs(dy) * n).sum(0)
        dr = dr + rb * (tt + n * (tt * n).mean(1, keepdims=True))
    m["dx"] = dr * abs(alpha)
    if "b" in t:
        n, g = np.abs(t["b"]) * ra, 1.0
        if "gate" in t:
            g = np.abs(t["gate"])[np.arange(len(r)) // k]
            p = dr * np.abs(t["w_after"]) * n
            m["dgate"] = np.stack([p[i:i + k].sum(0) for i in range(0, len(r), k)])
        m["dw_after"] = (dr * g * n).sum(0)
        u = dr * g * np.abs(t["w_after"])
        m["db"] = ra * (u + n * (u * n).mean(1, keepdims=True))
    else:
        m["dx"] = dr
    return m


def test_gradient_equals_differences(ctx):
    """Central differences of the 64-bit forward pass (step 1e-4: off by less than 1e-7 of the terms) against
    the device's fp32 gradients."""
    rows, cols, k, alpha, eps = 5, 40, 2, 0.75, 1e-3
    print("[case] norm differences", flush=True)
    rng = np.random.default_rng(8)
    t = _make(rng, rows, cols, "f32", "f32", k, "ab")
    t["x"] = _q(rng.standard_normal((rows, cols)), "f32")
    dout, dy = (_q(rng.standard_normal((rows, cols)), "f32") for _ in range(2))
    d = {n: _up(ctx, v, "f32") for n, v in t.items()}
    out, y, rstd = (ctx.empty(s, np.float32) for s in ((rows, cols), (rows, cols), (2, rows)))
    kw = {"gate_rows": k, "stream_dtype": mi.F32, "branch_dtype": mi.F32, "alpha": alpha}
    ctx.norm_block(d["x"], d["b"], d["gate"], d["w_after"], d["w_before"], out, y, rstd, rows, cols, eps=eps, **kw)
    g = {n: ctx.empty(t[n].shape, np.float32) for n in t}
    ddout, ddy, work = _up(ctx, dout, "f32"), _up(ctx, dy, "f32"), ctx.empty((1024 * cols,), np.float32)
    ctx.norm_block_grad(out, d["b"], d["gate"], d["w_after"], d["w_before"], rstd, ddout, ddy, g["x"], g["b"], g["gate"],
                        g["w_after"], g["w_before"], work, 4096 * cols, rows, cols, **kw)
    ctx.wait(60_000)

    def loss(v):
        o, yy, _, _ = mx.norm_block(v["x"], v["b"], v["gate"], v["w_after"], v["w_before"], k, alpha, eps)
        return (o * dout).sum() + (yy * dy).sum()

    for n, v in t.items():
        got = ctx.download(g[n])
        for i in list(np.ndindex(v.shape))[::7]:
            up, down = {**t, n: v.copy()}, {**t, n: v.copy()}
            up[n][i] += 1e-4
            down[n][i] -= 1e-4
            want = (loss(up) - loss(down)) / 2e-4
            # gradients here are sums of terms up to about 10: 2^-19 of those, and the differences' own error
            assert abs(got[i] - want) <= 3e-5 * max(1, abs(want)), (n, i, got[i], want)
    for b in (*d.values(), out, y, rstd, *g.values(), ddout, ddy, work):
        b.free()


def test_rows_of_zeros_infinities_and_nan(ctx):
    """A row of zeros norms to zeros (eps > 0); an infinity or NaN stays in its row."""
    rows, cols = 6, 600
    print("[case] norm special rows", flush=True)
    rng = np.random.default_rng(2)
    t = _make(rng, rows, cols, "f32", "bf16", None, "ab")
    t["x"][1], t["b"][1] = 0, 0
    t["b"][2, 5], t["x"][3, 7] = np.inf, np.nan
    d = {n: _up(ctx, v, "bf16" if n == "b" else "f32") for n, v in t.items()}
    out, y = ctx.empty((rows, cols), np.float32), ctx.empty((rows, cols), np.uint16)
    ctx.norm_block(d["x"], d["b"], None, d["w_after"], d["w_before"], out, y, None, rows, cols, stream_dtype=mi.F32)
    ctx.wait(60_000)
    o, yy = ctx.download(out), _down(ctx, y, "bf16", (rows, cols))
    assert (o[1] == 0).all() and (yy[1] == 0).all()
    assert np.isnan(o[2]).any() and np.isnan(yy[2]).all() and np.isnan(yy[3]).all()
    fine = [0, 1, 4, 5]
    assert np.isfinite(o[fine]).all() and np.isfinite(yy[fine]).all()
    for b in (*d.values(), out, y):
        b.free()


def test_refusals(ctx):
    d = ctx.empty((1 << 16,), np.uint8)
    p = d.ptr

    def refused(name, *args, text):
        assert ctx.call_status(name, *args) == mi.MIAIE_EINVAL, (name, args)
        assert text in ctx.last_error(), ctx.last_error()

    f, n = "miaie_norm_block", (4, 8, 8, 8, 4, 0, 0, mi._f(1), mi._f(0))
    refused(f, None, p, p, p, p, p, p, p, *n, text="x is NULL")
    refused(f, p, None, None, None, None, None, None, p, *n, text="nothing to do")
    refused(f, p, p, p, None, p, p, p, p, *n, text="w_after")
    refused(f, p, p, p, p, p, None, p, p, *n, text="out")
    refused(f, p, None, p, None, p, None, p, p, *n, text="without b")
    refused(f, p, p, p, p, None, p, p, p, *n, text="come together")
    refused(f, p, p, p, p, p, p, p, p, 0, *n[1:], text="rows=0")
    refused(f, p, p, p, p, p, p, p, p, 4, 16385, *n[2:], text="cols=16385")
    refused(f, p, p, p, p, p, p, p, p, 4, 8, 7, *n[3:], text="ldx=7")
    refused(f, p, p, p, p, p, p, p, p, 4, 8, 8, 7, *n[4:], text="ldb=7")
    refused(f, p, p, p, p, p, p, p, p, 4, 8, 8, 8, 0, *n[5:], text="gate_rows=0")
    refused(f, p, p, p, p, p, p, p, p, 4, 8, 8, 8, 4, 2, 0, *n[7:], text="stream_dtype=2")
    refused(f, p, p, p, p, p, p, p, p, 4, 8, 8, 8, 4, 0, -1, *n[7:], text="branch_dtype=-1")
    refused(f, p, p, p, p, p, p, p, p, *n[:8], mi._f(-1), text="eps")
    refused(f, p, p, p, p, p, p, p, p, *n[:8], mi._f(float("nan")), text="eps")
    refused(f, p + 2, p, p, p, p, p, p, p, *n, text="x is misaligned")
    refused(f, p, p, p, p + 2, p, p, p, p, *n, text="w_after is misaligned")
    h, m = "miaie_norm_block_grad", (mi._sz(4096 * 8), 4, 8, 8, 8, 4, 0, 0, mi._f(1))
    refused(h, p, p, p, p, p, p, None, None, p, p, p, p, p, p, *m, text="neither dout nor dy")
    refused(h, p, p, p, p, p, p, p, p, None, None, None, None, None, p, *m, text="no gradient wanted")
    refused(h, p, None, None, None, None, p, p, None, p, None, None, None, None, p, *m, text="no norm ran")
    refused(h, None, p, p, p, p, p, p, p, p, p, p, p, p, p, *m, text="dy takes r")
    refused(h, p, p, p, p, p, p, p, None, p, p, p, p, None, p, *m, text="w_before")
    refused(h, p, None, None, None, p, p, p, p, p, p, None, None, None, p, *m, text="b takes w_after")
    refused(h, p, p, None, p, p, p, p, p, p, p, p, p, p, p, *m, text="dgate without gate")
    refused(h, p, p, p, p, p, None, p, p, p, p, p, p, p, p, *m, text="rstd is NULL")
    refused(h, p, p, p, p, p, p, p, p, p, p, p, p, p, None, *m, text="work is NULL")
    refused(h, p, p, p, p, p, p, p, p, p, p, p, p, p, p, mi._sz(4096 * 8 - 1), *m[1:], text="work_bytes")
    ctx.wait(10_000)
    d.free()


def test_example_of_a_whole_block():
    """aiehlc_amd/harness/miaie_examples block: norm, conversion, 4-bit MLP, norm with gate and residual, through the
    C++ host surface, against its own golden."""
    import os
    import subprocess

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    for args in ((), ("5", "200", "333"), ("300", "512", "1000")):
        print("[case] miaie_examples block", *args, flush=True)
        r = subprocess.run([os.path.join(root, "aiehlc_amd", "harness", "miaie_examples"), "block", *args], capture_output=True,
                           text=True, timeout=100)
        assert r.returncode == 0 and "CPU result matches" in r.stdout, (r.returncode, r.stdout, r.stderr)
