"""The choice of kernel of the MXFP4 products (miaie_plan_gemm_mxfp4): a host
function, so these run without a GPU."""
import random

import pytest

import aiehlc_amd as mi

OUTS = [mi.F32, mi.BF16, mi.MXFP4]
MOST = 1 << 30


def _groups(k):
    return (k + 511) // 512


def _documented(M, N, K, out):
    """What include/miaie.h says that a product takes."""
    return (max(M, N) * _groups(K) < MOST and (out != mi.MXFP4 or M * _groups(N) < MOST)
            and -(-M // 256) * -(-N // 256) < 1 << 24)


def test_plans():
    assert mi.plan_gemm_mxfp4(8192, 8192, 8192) == {"kernel": mi.KERNEL_PIPE, "tile_m": 256, "tile_n": 256,
                                                    "workgroups": 1024, "threads": 256}
    # the up-projection of 2048 tokens: 256 wide tiles fill one round, 176 narrow ones the next
    up = mi.plan_gemm_mxfp4(2048, 11008, 4096, mi.MXFP4)
    assert (up["kernel"], up["workgroups"]) == (mi.KERNEL_PIPE_MIXED, 256 + 176)
    one = mi.plan_gemm_mxfp4(1, 11008, 4096)
    assert (one["kernel"], one["tile_m"], one["tile_n"], one["workgroups"], one["threads"]) == (mi.KERNEL_ROWS, 16, 16, 688, 512)


@pytest.mark.parametrize("out", OUTS)
def test_every_documented_size_has_a_kernel(out):
    """A launch takes fewer than 2^32 threads; where one kernel's would be more, another's are not."""
    for M, N, K in ((1, MOST - 1, 512), (4, MOST - 1, 1), (MOST - 1, 1, 512), (1 << 18, 1 << 19, 1024),
                    (1 << 16, (1 << 24) - 1, 512), (5, (1 << 26) - 1, 8192), (1, 16383, 1 << 26), (16383, 16383, 1 << 26)):
        if _documented(M, N, K, out):
            p = mi.plan_gemm_mxfp4(M, N, K, out)
            assert 0 < p["workgroups"] * p["threads"] < 1 << 32, (M, N, K)
    rng = random.Random(out)
    for _ in range(20000):
        M, N, K = (int(2 ** rng.uniform(0, most)) for most in (30, 30, 26))
        cus = rng.choice([1, 7, 256, 1 << 20])
        if _documented(M, N, K, out):
            p = mi.plan_gemm_mxfp4(M, N, K, out, cus)
            assert p["workgroups"] * p["threads"] < 1 << 32 and p["workgroups"] > 0, (M, N, K, cus)
            rows, cols = -(-M // p["tile_m"]), -(-N // p["tile_n"])
            if p["kernel"] != mi.KERNEL_PIPE_MIXED and out != mi.MXFP4:
                assert p["workgroups"] == rows * cols


def test_refusals():
    for args, text in (((0, 4, 4), "M=0"), ((4, -1, 4), "N=-1"), ((4, 4, (1 << 26) + 1), "K="), ((MOST, 4, 4), "too large"),
                       ((4, 4, 4, 3), "out=3"), ((4, 4, 4, 0, 0), "cus=0"), ((1 << 20, 1 << 20, 1), "too large"),
                       ((1 << 29, 1024, 4, mi.MXFP4), "too large")):
        with pytest.raises(mi.MiaieError, match=text):
            mi.plan_gemm_mxfp4(*args)
