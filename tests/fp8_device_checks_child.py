"""Run by tests/test_gpu_fp8_device_checks.py in a process of its own, with
MIAIE_LIB_DIR pointing at the device-checked build (aiehlc_amd/lib_dbg): the 8-bit
operators, the routing and the experts' products on buffers exactly as long as the
header says, results against the oracle and no access outside a known buffer; then
buffers declared shorter than they are, whose accesses past the declared end
miaie_wait names.

Prints one JSON object and exits 0 when every check passed."""
import json
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "tests")]

import aiehlc_amd as mi  # noqa: E402
import fp8_oracle as fp8  # noqa: E402
import test_gpu_experts as experts  # noqa: E402
import test_gpu_experts_forms as forms  # noqa: E402
import test_gpu_fp8 as basic  # noqa: E402
import test_gpu_fp8_kernels as kernels  # noqa: E402


def main() -> int:
    assert os.path.abspath(mi.LIB_DIR).endswith("lib_dbg"), mi.LIB_DIR
    sys.stdout, out = sys.stderr, sys.stdout  # (the tests print their cases)
    ctx = mi.Context(0)
    assert ctx.device_checks(), "the library at MIAIE_LIB_DIR is not the device-checked build"
    cases, planted = [], []

    def run(f, *args):
        f(ctx, *args)
        ctx.wait(60_000)
        cases.append(f"{f.__name__} {args}")

    for shape in basic.SHAPES[::3]:
        for dtype in ("f32", "bf16"):
            run(basic.test_quant_equals_the_oracle_bit_by_bit, shape, dtype, 1)
            run(basic.test_quant_equals_the_oracle_bit_by_bit, shape, dtype, 128)
    for *shape, cus in kernels.DENSE:
        ctx.plan_set_cus(cus)
        for b_block in (1, 128):
            run(basic.test_gemm, shape, b_block, False)
    for *case, cus in kernels.SLOTS:
        ctx.plan_set_cus(cus)
        run(experts.test_products_over_slots, *case, cus % 2 == 1)
    for *case, cus in kernels.MLPS:
        ctx.plan_set_cus(cus)
        run(experts.test_mlp, *case)
    ctx.plan_set_cus(256)
    for case in experts.ROUTES[::2]:
        run(experts.test_route, case, "softmax")
    for T, k, E in ((1, 1, 1), (333, 2, 7), (65, 64, 1024)):
        run(experts.test_order, T, k, E, "holes")
    for sizes in forms.STEPS:
        run(forms.test_a_layer_and_its_gradients, sizes, "sigmoid")

    def expect_fault(kind, source):
        rc = ctx.call_status("miaie_wait", 60_000)
        msg = ctx.last_error()
        assert rc == mi.MIAIE_EFAULT, (rc, msg)
        assert kind in msg and f"({source}, line " in msg, msg
        planted.append(msg)

    M, N, K = 300, 256, 512
    rng = np.random.default_rng(1)
    A, B = fp8.pack(rng.standard_normal((M, K))), fp8.pack(rng.standard_normal((N, K)), 128)
    dA, dB, C = [ctx.upload(v) for v in A], [ctx.upload(v) for v in B], ctx.upload(np.full((M, N), 7.0, np.float32))
    print("[step] planted: B declared short in a tile product and in a product of one row", flush=True)
    ctx.debug_register(dB[0], B[0].nbytes // 2)
    ctx.gemm_fp8(*dA, *dB, C, M, N, K)
    expect_fault("global->LDS copy", "gemm_fp8.hip")
    a1 = [ctx.upload(A[0][:1]), ctx.upload(np.ascontiguousarray(A[1][:, :1]))]
    ctx.gemm_fp8(*a1, *dB, C, 1, N, K)
    expect_fault("load", "gemm_fp8.hip")
    ctx.debug_register(dB[0], B[0].nbytes)
    print("[step] planted: C declared short", flush=True)
    ctx.copy_h2d(C, np.full((M, N), 7.0, np.float32))
    ctx.debug_register(C, 4 * N * (M // 2))
    ctx.gemm_fp8(*dA, *dB, C, M, N, K)
    expect_fault("store", "gemm_fp8.hip")
    assert (ctx.download(C)[M // 2:] == 7).all(), "a store past the declared extent reached memory"
    ctx.debug_register(C, 4 * N * M)
    print("[step] planted: X declared short in a conversion", flush=True)
    x, q = ctx.upload(np.zeros((64, 512), np.float32)), [ctx.empty(s, t) for s, t in zip(mi.fp8_shapes(64, 512), (np.uint8, np.float32))]
    ctx.debug_register(x, 4 * 512 * 32)
    ctx.quant_fp8(x, 64, 512, *q, dtype=mi.F32)
    expect_fault("load", "quant_fp8.hip")
    print("[step] planted: logits declared short in a routing", flush=True)
    idx, w = ctx.empty((64, 2), np.int32), ctx.empty((64, 2), np.float32)
    ctx.route_experts(x, None, idx, w, 64, 2, 512)
    expect_fault("load", "route_experts.hip")
    ctx.close()
    sys.stdout = out
    print(json.dumps({"cases": cases, "planted": planted}), flush=True)
    return 0


if __name__ == "__main__":
    sys.exit(main())
