"""What the Python binding's 8-bit, routing and experts' methods take for a device
operand (CPU only: the entry points are callbacks that record what reaches them)."""
import ctypes as C

import numpy as np
import pytest

import aiehlc_amd as mi
from test_binding_operands import Whole

METHODS = [  # method, entry point, the context's function, arguments of a call
    ("quant_fp8", "miaie_quant_fp8", "_f_quant8", lambda a: (a, 4, 32, a, a, a, a)),
    ("dequant_fp8", "miaie_dequant_fp8", "_f_dequant8", lambda a: (a, a, a, 4, 32)),
    ("gemm_fp8", "miaie_gemm_fp8", "_f_gemm8", lambda a: (a, a, a, a, a, 4, 4, 32)),
    ("route_experts", "miaie_route_experts", "_f_route", lambda a: (a, a, a, a, 4, 2, 8)),
    ("route_experts_grad", "miaie_route_experts_grad", "_f_route_grad", lambda a: (a, a, a, a, 4, 2, 8)),
    ("experts_order", "miaie_experts_order", "_f_order", lambda a: (a, a, 4, 2, 8)),
    ("experts_mlp_fp8", "miaie_experts_mlp_fp8", "_f_x_mlp", lambda a: (*[a] * 12, 4, 2, 8, 32, 128, 32)),
    ("experts_gemm_fp8", "miaie_experts_gemm_fp8", "_f_x_gemm", lambda a: (*[a] * 6, 4, 2, 8, 32, 128)),
    ("experts_quant_fp8", "miaie_experts_quant_fp8", "_f_x_quant", lambda a: (*[a] * 7, 4, 2, 8, 32)),
    ("experts_swiglu_fp8", "miaie_experts_swiglu_fp8", "_f_x_glu", lambda a: (*[a] * 6, 4, 2, 8, 128)),
    ("experts_swiglu_grad_fp8", "miaie_experts_swiglu_grad_fp8", "_f_x_glu_grad", lambda a: (*[a] * 7, 4, 2, 8, 128)),
    ("experts_wgrad_fp8", "miaie_experts_wgrad_fp8", "_f_x_wgrad", lambda a: (*[a] * 6, 4, 2, 8, 32, 32)),
    ("experts_combine", "miaie_experts_combine", "_f_x_sum", lambda a: (*[a] * 4, 4, 2, 8, 32)),
    ("experts_combine_grad", "miaie_experts_combine_grad", "_f_x_sum_grad", lambda a: (*[a] * 4, 4, 2, 8, 32)),
]


@pytest.mark.parametrize("method, name, attr, call", METHODS)
def test_addresses_of_every_kind_reach_the_entry_point(method, name, attr, call):
    (res, args), seen = mi._SIGS[name], []
    ctx = object.__new__(mi.Context)
    ctx.handle = None
    setattr(ctx, attr, C.CFUNCTYPE(res, *args)(lambda *a: seen.append(a) or 0))
    pointers = [i for i, t in enumerate(args) if t is C.c_void_p and i > 0]
    for operand in (1 << 40, np.int64(1 << 40), np.uint64(1 << 40), Whole(), mi.DeviceBuffer(None, 1 << 40, 64)):
        getattr(ctx, method)(*call(operand))
        assert {seen[-1][i] for i in pointers} == {1 << 40}, type(operand)
    with pytest.raises((TypeError, ValueError, C.ArgumentError)):  # a host array is no device operand
        getattr(ctx, method)(*call(np.zeros(4)))
    assert len(seen) == 5


def test_sizes_on_the_host():
    assert mi.fp8_shapes(5, 300) == ((5, 384), (3, 5)) and mi.fp8_shapes(130, 128, 128) == ((130, 128), (1, 2))
    lib = mi.load_library()
    for R, K, block in ((1, 1, 1), (130, 300, 1), (130, 300, 128), (1 << 20, 129, 128)):
        q, s = mi.fp8_shapes(R, K, block)
        assert lib.miaie_fp8_q_pitch(K) == q[1] and lib.miaie_fp8_q_bytes(R, K) == q[0] * q[1]
        assert lib.miaie_fp8_s_bytes(R, K, block) == 4 * s[0] * s[1]
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 2), ((1 << 30) + 1, 1, 1)):
        assert lib.miaie_fp8_s_bytes(*bad) == 0
