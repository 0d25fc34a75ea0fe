"""Forms of the norms around a block and of the MXFP4 conversion that
include/miaie.h documents and the other files do not run: a gradient without
dout, results over their inputs, and every scale and code back to fp32 and
bf16.  Against the 64-bit oracle (tests/mx_oracle.py) with the tolerances of
tests/test_gpu_norm_block.py."""
import numpy as np
import pytest

import aiehlc_amd as mi
import mx_oracle as mx
from test_gpu_norm_block import DT, REL, _close, _down, _magnitudes, _make, _q, _up

pytestmark = pytest.mark.gpu


def _say(*a):
    print("[case]", *a, flush=True)


FORMS = [(1, 64, "f32", "f32", 1), (5, 700, "bf16", "bf16", 2), (70, 4096, "f32", "bf16", 70), (300, 1111, "bf16", "f32", 1),
         (20, 8192, "f32", "f32", 7), (6, 9001, "bf16", "bf16", 6), (3, 16384, "f32", "bf16", 1)]


@pytest.mark.parametrize("case", FORMS)
def test_stream_and_branch_in_place(ctx, case):
    """out over x gives the bits of a separate out; so does db over b, in every type and at every row width."""
    rows, cols, st, bt, k = case
    _say("in place", case)
    rng = np.random.default_rng(rows * 3 + cols)
    t = _make(rng, rows, cols, st, bt, k, "ab")
    dout, dy = _q(rng.standard_normal((rows, cols)), st), _q(rng.standard_normal((rows, cols)), bt)
    x, b, gate = _up(ctx, t["x"], st), _up(ctx, t["b"], bt), _up(ctx, t["gate"], bt)
    wa, wb = _up(ctx, t["w_after"], "f32"), _up(ctx, t["w_before"], "f32")
    ddout, ddy = _up(ctx, dout, st), _up(ctx, dy, bt)
    out, y, y2, db = _up(ctx, t["x"] * 0, st), _up(ctx, dy * 0, bt), _up(ctx, dy * 0, bt), _up(ctx, dy * 0, bt)
    rstd = ctx.empty((2, rows), np.float32)
    kw = {"gate_rows": k, "stream_dtype": DT[st], "branch_dtype": DT[bt], "alpha": 0.75}
    ctx.norm_block(x, b, gate, wa, wb, out, y, rstd, rows, cols, **kw)
    ctx.norm_block_grad(out, b, gate, wa, wb, rstd, ddout, ddy, None, db, None, None, None, None, 0, rows, cols, **kw)
    ctx.norm_block(x, b, gate, wa, wb, x, y2, rstd, rows, cols, **kw)
    ctx.norm_block_grad(out, b, gate, wa, wb, rstd, ddout, ddy, None, b, None, None, None, None, 0, rows, cols, **kw)
    ctx.wait(60_000)
    for one, other, dt in ((out, x, st), (y, y2, bt), (db, b, bt)):
        assert np.array_equal(_down(ctx, one, dt, (rows, cols)), _down(ctx, other, dt, (rows, cols)))
    for buf in (x, b, gate, wa, wb, ddout, ddy, out, y, y2, db, rstd):
        buf.free()


@pytest.mark.parametrize("parts", ["ab", "b"])
@pytest.mark.parametrize("case", FORMS)
def test_gradient_without_dout(ctx, case, parts):
    """dout NULL is a dout of zeros: the same bits as with one, and the formula's values."""
    rows, cols, st, bt, k = case
    _say("no dout", case, parts)
    rng = np.random.default_rng(rows * 5 + cols)
    t = _make(rng, rows, cols, st, bt, k if parts == "ab" else None, parts)
    dy = _q(rng.standard_normal((rows, cols)), bt)
    ra = _q(1 / np.sqrt((t["b"] * t["b"]).mean(1)), "f32") if "b" in t else np.ones(rows)
    rb = _q(1 / np.sqrt((t["x"] * t["x"]).mean(1)), "f32")
    types = {"x": st, "b": bt, "gate": bt, "w_after": "f32", "w_before": "f32"}
    d = {n: _up(ctx, v, types[n]) for n, v in t.items()}
    rstd, ddy, zero = _up(ctx, np.stack((ra, rb)), "f32"), _up(ctx, dy, bt), _up(ctx, np.zeros((rows, cols)), st)
    want = mx.norm_block_grad(t["x"], t.get("b"), t.get("gate"), t.get("w_after"), t["w_before"], ra, rb, None, dy, k, 0.75)
    out = {"dx": st, "db": bt, "dgate": "f32", "dw_after": "f32", "dw_before": "f32"}
    work = ctx.empty((1024 * cols,), np.float32)
    results = []
    for dout in (None, zero):
        g = {n: _up(ctx, np.full(want[n].shape, 9.0), out[n]) for n in want}
        ctx.norm_block_grad(d["x"], d.get("b"), d.get("gate"), d.get("w_after"), d["w_before"], rstd, dout, ddy,
                            *(g.get(n) for n in out), work, mi.norm_work_bytes(cols), rows, cols, gate_rows=k,
                            stream_dtype=DT[st], branch_dtype=DT[bt], alpha=0.75)
        ctx.wait(60_000)
        results.append({n: _down(ctx, g[n], out[n], want[n].shape) for n in want})
        for buf in g.values():
            buf.free()
    mag = _magnitudes(t, t["x"], np.stack((ra, rb)), np.zeros((rows, cols)), dy, k, 0.75)
    chain = (rows / 256 + 256) * 2.0**-24
    for n, w in want.items():
        assert np.array_equal(results[0][n], results[1][n]), n
        _close(results[0][n], w, (REL + (chain if n[1] in "gw" else 0)) * mag[n], out[n], n)
    for buf in (*d.values(), rstd, ddy, zero, work):
        buf.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_every_scale_and_code_back(ctx, dtype):
    """Scale bytes 0 to 252 with every code, exactly (subnormal results too); 255 is NaN."""
    _say("every scale", dtype)
    R, C = 256, 32
    Q = np.zeros((R, 128), np.uint8)
    Q[:, :16] = np.arange(16) | (15 - np.arange(16)) << 4  # every code, in both halves of a byte
    S = np.zeros((1, R, 4, 4), np.uint8)
    S[0, :, 0, 0] = np.arange(R)
    q, s = ctx.upload(Q), ctx.upload(S)
    y = ctx.empty((R, C), np.float32 if dtype == "f32" else np.uint16)
    ctx.dequant_mxfp4(q, s, y, R, C, dtype=DT[dtype])
    ctx.wait(60_000)
    got, want = _down(ctx, y, dtype, (R, C)), mx.values(Q, S, C)
    assert np.array_equal(got[:253], want[:253])
    assert np.isnan(got[255]).all() and np.isnan(want[255]).all()
    for b in (q, s, y):
        b.free()
