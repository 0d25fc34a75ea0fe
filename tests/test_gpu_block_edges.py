"""Edges of the norms around a block: row lanes without a row in their gradients,
and infinities there, against the 64-bit oracle (tests/mx_oracle.py); the grid
planned for very many compute units."""
import numpy as np
import pytest

import aiehlc_amd as mi
import mx_oracle as mx
from test_gpu_norm_block import _make, _q, _up

pytestmark = pytest.mark.gpu


def _say(*a):
    print("[case]", *a, flush=True)


def _same_where_not_finite(got, want, what):
    """NaN where the oracle has NaN, and its infinities with their signs."""
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    inf = np.isinf(want)
    assert np.array_equal(np.isinf(got), inf) and np.array_equal(got[inf], want[inf]), what


# rows that leave row lanes of a gradient's workgroup idle: one row, gates of fewer rows than lanes, a gate's
# rows split unevenly, more gates than 128 with a last turn of fewer, and a last gate of fewer rows
IDLE = [(1, 64, 1), (5, 600, 3), (37, 100, 37), (300, 96, 1), (257, 1000, 2), (259, 8200, 2)]


@pytest.mark.parametrize("where", ["w_after", "w_before", "gate"])
@pytest.mark.parametrize("rows, cols, k", IDLE)
def test_infinite_weights_reach_only_the_sums_of_real_rows(ctx, rows, cols, k, where):
    """A lane without a row adds nothing to the sums over rows, not even 0 x infinity."""
    _say("idle lanes", rows, cols, k, where)
    rng = np.random.default_rng(rows + cols)
    t = _make(rng, rows, cols, "f32", "f32", k, "ab")
    t[where][..., 5] = np.inf
    dout, dy = (_q(rng.standard_normal((rows, cols)), "f32") for _ in range(2))
    r, ra, rb = t["x"], *(_q(1 / np.sqrt((v * v).mean(1)), "f32") for v in (t["b"], t["x"]))
    with np.errstate(invalid="ignore"):
        want = mx.norm_block_grad(r, t["b"], t["gate"], t["w_after"], t["w_before"], ra, rb, dout, dy, k, 0.75)
    bufs = [_up(ctx, v, "f32") for v in (r, t["b"], t["gate"], t["w_after"], t["w_before"], np.stack((ra, rb)), dout, dy)]
    names = ("dx", "db", "dgate", "dw_after", "dw_before")
    g = [ctx.empty(want[n].shape, np.float32) for n in names]
    work = ctx.empty((1024 * cols,), np.float32)
    ctx.norm_block_grad(*bufs, *g, work, mi.norm_work_bytes(cols), rows, cols, gate_rows=k, stream_dtype=mi.F32,
                        branch_dtype=mi.F32, alpha=0.75)
    ctx.wait(60_000)
    for n, buf in zip(names, g):
        _same_where_not_finite(ctx.download(buf).astype(np.float64), want[n], n)
    for b in (*bufs, *g, work):
        b.free()


def test_norm_grid_planned_for_very_many_cus():
    """miaie_plan_set_cus takes any count: 16 workgroups a CU stay within an int."""
    from hip_capture import Capture

    _say("norm grid")
    rows, cols = 100, 64
    cap = Capture()
    try:
        c = cap.ctx
        x, w, y = (c.upload(np.ones(s, np.float32)) for s in ((rows, cols), (cols,), (rows, cols)))
        grids = []
        for cus in (256, 1 << 28):
            c.plan_set_cus(cus)
            exe, g = cap.record(lambda: c.norm_block(x, None, None, None, w, None, y, None, rows, cols,
                                                     stream_dtype=mi.F32, branch_dtype=mi.F32))
            cap.ok(cap.hip.hipGraphExecDestroy(exe))
            grids.append(g)
        assert grids[0] == grids[1] == [(25, 1, 1)]  # four rows of 64 threads a workgroup
        for b in (x, w, y):
            b.free()
    finally:
        cap.close()
