"""What the Python binding's compute methods take for a device operand (CPU
only: the entry points are callbacks that record what reaches them)."""
import ctypes as C

import numpy as np
import pytest

import aiehlc_amd as mi

BLOCK = [  # method, entry point, the context's function, arguments of a call
    ("quant_mxfp4", "miaie_quant_mxfp4", "_f_quant", lambda a: (a, 4, 32, a, a)),
    ("dequant_mxfp4", "miaie_dequant_mxfp4", "_f_dequant", lambda a: (a, a, a, 4, 32)),
    ("gemm_mxfp4", "miaie_gemm_mxfp4", "_f_mx", lambda a: (a, a, a, a, a, 4, 4, 32)),
    ("gemm_mxfp4_rq", "miaie_gemm_mxfp4_rq", "_f_mx_rq", lambda a: (a, a, a, a, a, a, 4, 4, 32)),
    ("mlp_mxfp4", "miaie_mlp_mxfp4", "_f_mlp_mx", lambda a: (*[a] * 9, 4, 32, 32, 4)),
    ("norm_block", "miaie_norm_block", "_f_norm", lambda a: (*[a] * 8, 4, 32)),
    ("norm_block_grad", "miaie_norm_block_grad", "_f_norm_grad", lambda a: (*[a] * 14, 1 << 20, 4, 32)),
]
OLDER = [("gemm_bf16_f32", "miaie_gemm_bf16_f32", "_f_bf16", lambda a: (a, a, a, 4, 4, 32)),
         ("mlp_i8", "miaie_mlp_i8", "_f_mlp", lambda a: (a, a, a, a, a, 4, 4, 4, 4, 1, 1))]


class Whole:
    """Anything that int() takes."""

    def __int__(self):
        return 1 << 40


@pytest.mark.parametrize("method, name, attr, call", BLOCK + OLDER)
def test_addresses_of_every_kind_reach_the_entry_point(method, name, attr, call):
    res, args = mi._SIGS[name]
    seen = []
    ctx = object.__new__(mi.Context)
    ctx.handle = None
    setattr(ctx, attr, C.CFUNCTYPE(res, *args)(lambda *a: seen.append(a) or 0))
    pointers = [i for i, t in enumerate(args) if t is C.c_void_p and i > 0]
    for operand in (1 << 40, np.int64(1 << 40), np.uint64(1 << 40), Whole(), mi.DeviceBuffer(None, 1 << 40, 64)):
        getattr(ctx, method)(*call(operand))
        got = [seen[-1][i] for i in pointers]
        assert 1 << 40 in got and set(got) <= {1 << 40, None}, (type(operand), got)
    with pytest.raises((TypeError, ValueError, C.ArgumentError)):  # a host array is no device operand
        getattr(ctx, method)(*call(np.zeros(4)))
    assert len(seen) == 5
