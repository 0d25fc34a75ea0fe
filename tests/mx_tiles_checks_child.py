"""Run by tests/test_gpu_mx_tiles_checked.py in a process of its own, with
MIAIE_LIB_DIR pointing at the device-checked build (aiehlc_amd/lib_dbg): a
product on every tile of tests/test_gpu_mx_tiles.py, on buffers exactly as long
as the header says, against the oracle.

Prints one JSON object and exits 0 when every check passed."""
import json
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "tests")]

import aiehlc_amd as mi  # noqa: E402
import mx_oracle as mx  # noqa: E402
import test_gpu_mx_tiles as tiles  # noqa: E402


def main() -> int:
    assert os.path.abspath(mi.LIB_DIR).endswith("lib_dbg"), mi.LIB_DIR
    ctx = mi.Context(0)
    assert ctx.device_checks(), "the library at MIAIE_LIB_DIR is not the device-checked build"
    rng = np.random.default_rng(17)
    done = []
    for kernel, case in tiles.CASES:
        out, M, N, K, cus = case
        if M * N * K > 1e9:
            continue
        print("[step]", *case, file=sys.stderr, flush=True)
        assert tiles.planned(case) == kernel
        ctx.plan_set_cus(cus)
        A, B = (mx.pack(rng.standard_normal((r, K))) for r in (M, N))
        a, b = mx.values(*A, K), mx.values(*B, K)
        dev = [ctx.upload(v) for v in (*A, *B)]
        want, bound = a @ b.T, mx.product_bound(a, b)
        if out == "mx":
            y = [ctx.empty(s, np.uint8) for s in mi.mxfp4_shapes(M, N)]
            ctx.gemm_mxfp4_rq(*dev, *y, M, N, K, relu=True)
            ctx.wait(110_000)
            s, t = mx.block_scales(ctx.download(y[1])), mx.block_scales(mx.pack(np.maximum(want, 0))[1])
            assert (np.abs(s.astype(int) - t) <= 1).all() and not ctx.download(y[0])[:, (N + 1) // 2:].any(), case
        else:
            y = [ctx.empty((M, N), np.float32 if out == "f32" else np.uint16)]
            ctx.gemm_mxfp4(*dev, *y, M, N, K, dtype=tiles.OUT[out])
            ctx.wait(110_000)
            got = ctx.download(y[0])
            if out == "bf16":
                got, bound = mx.from_bf16_bits(got), bound + 2.0**-8 * np.abs(want)
            assert (np.abs(got - want) <= bound).all(), case
        for v in (*dev, *y):
            v.free()
        done.append(case)
    ctx.close()
    print(json.dumps({"cases": done}), flush=True)
    return 0


if __name__ == "__main__":
    sys.exit(main())
