"""Ends of the documented ranges of the 8-bit operators, on the host."""
import os
import subprocess

import pytest

import aiehlc_amd as mi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("R, K", [(1 << 30, 1), (1, 1 << 30), (1 << 15, (1 << 22) - 128), ((1 << 22) - 128, 1 << 15), (1 << 20, 130944),
                                  ((1 << 23) - 1, 16256)])
def test_sizes_of_the_largest_matrices(R, K):
    lib = mi.load_library()
    blocks = lambda n: -(-n // 128)  # noqa: E731
    fits = blocks(R) * blocks(K) < 1 << 23
    assert lib.miaie_fp8_q_bytes(R, K) == (R * 128 * blocks(K) if fits else 0)
    assert lib.miaie_fp8_s_bytes(R, K, 1) == (4 * R * blocks(K) if fits else 0)
    assert lib.miaie_fp8_s_bytes(R, K, 128) == (4 * blocks(R) * blocks(K) if fits else 0)


@pytest.mark.parametrize("R, K", [(1 << 30, 128), (128, 1 << 30), (1 << 30, 1 << 30), (1 << 15, 1 << 22), (1 << 22, 1 << 15), (1 << 20, 1 << 17)])
def test_no_sizes_of_larger_ones(R, K):
    """128 x 128 blocks of 2^23 and more are no packed matrix: no bytes."""
    lib = mi.load_library()
    assert lib.miaie_fp8_q_bytes(R, K) == lib.miaie_fp8_s_bytes(R, K, 1) == lib.miaie_fp8_s_bytes(R, K, 128) == 0


def test_the_largest_products_over_slots():
    """2^22 blocks of 128 x 128: 8192 of slots by 512 of columns, gate and up counted both; not one more."""
    assert mi.experts_rows(1 << 20, 1, 1) == 128 * 8192
    for swiglu, N, unit in ((False, 65536, 1), (True, 32768, 128)):
        assert mi.plan_experts_fp8(1 << 20, 1, 1, N, 128, swiglu)["workgroups"] > 0
        with pytest.raises(mi.MiaieError, match="too large"):
            mi.plan_experts_fp8(1 << 20, 1, 1, N + unit, 128, swiglu)


def test_types_of_slots_rows():
    """What reaches the entry point as its dtype for the types of a result and of the slots' rows."""
    assert [mi._slots_dtype(*t) for t in ((mi.F32, None), (mi.BF16, None), (mi.F32, mi.F32), (mi.BF16, mi.BF16), (mi.BF16, mi.F32))] \
        == [mi.F32, mi.BF16, mi.F32, mi.BF16, mi.BF16 | mi.F32_SLOTS]
    for bad in ((mi.F32, mi.BF16), (mi.BF16, 2), (2, mi.F32)):
        with pytest.raises(ValueError):
            mi._slots_dtype(*bad)


def test_sizes_of_the_wrappers(tmp_path):
    """Undefined arithmetic ends the program."""
    exe = str(tmp_path / "host_experts_sizes_check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    f"-I{os.path.join(ROOT, 'include')}", os.path.join(ROOT, "tests", "host_experts_sizes_check.cpp"), "-o", exe],
                   check=True, timeout=300)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
