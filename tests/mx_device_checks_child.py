"""Run by tests/test_gpu_mx_device_checks.py in a process of its own, with
MIAIE_LIB_DIR pointing at the device-checked build (aiehlc_amd/lib_dbg): the
MXFP4 and norm kernels on buffers exactly as long as the header says, results
against the oracle and no access outside a known buffer; then buffers declared
shorter than they are, whose accesses past the declared end miaie_wait names.

Prints one JSON object and exits 0 when every check passed."""
import json
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "tests")]

import aiehlc_amd as mi  # noqa: E402
import mx_oracle as mx  # noqa: E402


def main() -> int:
    assert os.path.abspath(mi.LIB_DIR).endswith("lib_dbg"), mi.LIB_DIR
    ctx = mi.Context(0)
    assert ctx.device_checks(), "the library at MIAIE_LIB_DIR is not the device-checked build"
    rng = np.random.default_rng(7)
    cases, planted = [], []

    def say(*a):
        print("[step]", *a, file=sys.stderr, flush=True)

    def packed(rows, cols):
        return [ctx.empty(s, np.uint8) for s in mi.mxfp4_shapes(rows, cols)]

    def free(*bufs):
        for b in bufs:
            b.free()

    for R, C in ((1, 1), (3, 257), (70, 1025), (513, 70), (600, 33)):
        for bf in (False, True):
            say("quant", R, C, bf)
            x = rng.standard_normal((R, C))
            x = (mx.bf16(x) if bf else np.float32(x)).astype(np.float64)
            # (offset by one element: as unaligned as the header allows)
            flat = np.concatenate(([0.0], x.ravel()))
            d = ctx.upload(mx.bf16_bits(flat) if bf else np.float32(flat))
            q, t, q1, t1 = packed(R, C), packed(C, R), packed(R, C), packed(C, R)
            at, dt = d.ptr + (2 if bf else 4), mi.BF16 if bf else mi.F32
            ctx.quant_mxfp4(at, R, C, *q, *t, dtype=dt)
            ctx.quant_mxfp4(at, R, C, *q1, dtype=dt)
            ctx.quant_mxfp4(at, R, C, None, None, *t1, dtype=dt)
            y = ctx.empty((R, C), np.uint16 if bf else np.float32)
            ctx.dequant_mxfp4(*q, y, R, C, dtype=dt)
            ctx.wait(120_000)
            for got, want in ((q, mx.pack(x)), (q1, mx.pack(x)), (t, mx.pack(x.T)), (t1, mx.pack(x.T))):
                assert all(np.array_equal(ctx.download(g), w) for g, w in zip(got, want)), (R, C)
            free(d, y, *q, *t, *q1, *t1)
            cases.append(f"quant {R}x{C} {'bf16' if bf else 'f32'}")

    # every tile and row kernel: planned for few CUs, small products take the large tiles
    shapes = [(1, 33, 300, 256), (3, 40, 1100, 256), (7, 70, 600, 256), (8, 600, 512, 4), (16, 90, 257, 256), (15, 700, 1024, 4),
              (30, 33, 512, 256), (31, 300, 768, 16), (31, 300, 768, 2), (60, 70, 2048, 256), (64, 200, 1024, 4), (130, 140, 512, 4),
              (300, 260, 1300, 2), (257, 300, 256, 1), (513, 770, 768, 2), (520, 900, 2304, 3)]
    for M, N, K, cus in shapes:
        say("gemm", M, N, K, "cus", cus)
        ctx.plan_set_cus(cus)
        A, B = (mx.pack(rng.standard_normal((r, K))) for r in (M, N))
        a, b = mx.values(*A, K), mx.values(*B, K)
        dA, dB = [ctx.upload(v) for v in A], [ctx.upload(v) for v in B]
        C, y = ctx.empty((M, N), np.float32), packed(M, N)
        c16 = ctx.empty((M, N), np.uint16)
        ctx.gemm_mxfp4(*dA, *dB, C, M, N, K)
        ctx.gemm_mxfp4(*dA, *dB, c16, M, N, K, dtype=mi.BF16)
        ctx.gemm_mxfp4_rq(*dA, *dB, *y, M, N, K, relu=True)
        ctx.wait(120_000)
        want, bound = a @ b.T, mx.product_bound(a, b)
        assert (np.abs(ctx.download(C) - want) <= bound).all(), (M, N, K)
        assert (np.abs(mx.from_bf16_bits(ctx.download(c16)) - want) <= bound + 2.0**-8 * np.abs(want)).all(), (M, N, K)
        s, t = mx.block_scales(ctx.download(y[1])), mx.block_scales(mx.pack(np.maximum(want, 0))[1])
        assert (np.abs(s.astype(int) - t) <= 1).all() and not ctx.download(y[0])[:, (N + 1) // 2:].any(), (M, N, K)
        free(*dA, *dB, C, c16, *y)
        cases.append(f"gemm {M}x{N}x{K} on {cus} CUs")
    ctx.plan_set_cus(256)

    for rows, cols, k in ((1, 4096, 1), (5, 33, 2), (70, 1000, 70), (300, 1111, 1), (9, 8192, 4), (3, 16383, 3)):
        say("norm", rows, cols, k)
        x, b = (np.float32(rng.standard_normal((rows, cols))).astype(np.float64) for _ in range(2))
        gate = np.float32(rng.standard_normal((-(-rows // k), cols))).astype(np.float64)
        wa, wb = (np.float32(1 + 0.1 * rng.standard_normal(cols)).astype(np.float64) for _ in range(2))
        d = [ctx.upload(np.float32(v)) for v in (x, b, gate, wa, wb)]
        out, y = ctx.empty((rows, cols), np.float32), ctx.empty((rows, cols), np.float32)
        rstd, work = ctx.empty((2, rows), np.float32), ctx.empty((1024 * cols,), np.float32)
        kw = {"gate_rows": k, "stream_dtype": mi.F32, "branch_dtype": mi.F32, "alpha": 0.5}
        ctx.norm_block(*d, out, y, rstd, rows, cols, **kw)
        g = [ctx.empty(s, np.float32) for s in ((rows, cols), (rows, cols), gate.shape, (cols,), (cols,))]
        ctx.norm_block_grad(out, *d[1:], rstd, d[0], d[1], *g, work, 4096 * cols, rows, cols, **kw)
        ctx.wait(120_000)
        r, yy, ra, rb = mx.norm_block(x, b, gate, wa, wb, k, 0.5, 1e-5)
        assert np.allclose(ctx.download(out), r, rtol=1e-5, atol=1e-5) and np.allclose(ctx.download(y), yy, rtol=1e-4, atol=1e-4)
        want = mx.norm_block_grad(r, b, gate, wa, wb, ra, rb, x, b, k, 0.5)
        for got, n in zip(g, ("dx", "db", "dgate", "dw_after", "dw_before")):
            scale = np.abs(want[n]).max()
            assert np.abs(ctx.download(got) - want[n]).max() <= 1e-4 * scale, (n, rows, cols)
        free(*d, *g, out, y, rstd, work)
        cases.append(f"norm {rows}x{cols}")

    def expect_fault(kind, source):
        rc = ctx.call_status("miaie_wait", 120_000)
        msg = ctx.last_error()
        assert rc == mi.MIAIE_EFAULT, (rc, msg)
        assert kind in msg and f"({source}, line " in msg, msg
        planted.append(msg)

    say("planted: B declared short in a tile product and in a product of one row")
    M, N, K = 300, 256, 512
    A, B = mx.pack(rng.standard_normal((M, K))), mx.pack(rng.standard_normal((N, K)))
    dA, dB, C = [ctx.upload(v) for v in A], [ctx.upload(v) for v in B], ctx.upload(np.full((M, N), 7.0, np.float32))
    ctx.debug_register(dB[0], B[0].nbytes // 2)
    ctx.gemm_mxfp4(*dA, *dB, C, M, N, K)
    expect_fault("global->LDS copy", "gemm_mxfp4.hip")
    ctx.gemm_mxfp4(*dA, *dB, C, 1, N, K)
    expect_fault("global->LDS copy", "gemm_mxfp4.hip")
    ctx.debug_register(dB[0], B[0].nbytes)
    say("planted: C declared short")
    ctx.copy_h2d(C, np.full((M, N), 7.0, np.float32))
    ctx.debug_register(C, 4 * N * (M // 2))
    ctx.gemm_mxfp4(*dA, *dB, C, M, N, K)
    expect_fault("store", "gemm_mxfp4.hip")
    assert (ctx.download(C)[M // 2:] == 7).all(), "a store past the declared extent reached memory"
    ctx.debug_register(C, 4 * N * M)
    say("planted: X declared short in a conversion")
    x = ctx.upload(np.zeros((64, 512), np.float32))
    q = packed(64, 512)
    ctx.debug_register(x, 4 * 512 * 32)
    ctx.quant_mxfp4(x, 64, 512, *q, dtype=mi.F32)
    expect_fault("load", "mxfp4.hpp")
    free(*dA, *dB, C, x, *q)
    ctx.close()
    print(json.dumps({"cases": cases, "planted": planted}), flush=True)
    return 0


if __name__ == "__main__":
    sys.exit(main())
