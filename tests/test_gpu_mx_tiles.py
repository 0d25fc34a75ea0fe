"""The MXFP4 products' tiles (aiehlc_amd/csrc/gemm_mxfp4.hip) that the shapes of
tests/test_gpu_mxfp4.py do not reach; tests/test_mx_plan.py checks that the two
lists together reach every kernel.  Tolerances and comparisons are that file's."""
import numpy as np
import pytest

import aiehlc_amd as mi

pytestmark = pytest.mark.gpu


def test_mlp_refuses_both_products_before_the_first(ctx):
    """The second product of this MLP has 2^24 tiles of 256 x 256, more than a launch takes: nothing is queued."""
    d = ctx.empty((1 << 16,), np.uint8)
    p = d.ptr
    for dtype in (mi.F32, mi.BF16):
        rc = ctx.call_status("miaie_mlp_mxfp4", *[p] * 9, dtype, 1 << 20, 1, 1, 1 << 20, 1 << 20)
        assert rc == mi.MIAIE_EINVAL and "too large" in ctx.last_error(), ctx.last_error()
    ctx.wait(10_000)
    d.free()
