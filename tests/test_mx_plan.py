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


def _kernel(M, N, K, out, cus):
    """The kernel's template arguments: row kernels differ in the rows of A that they stage, tiles that write C in
    whether some of its columns end inside one."""
    p = mi.plan_gemm_mxfp4(M, N, K, out, cus)
    tile = p["kernel"], p["tile_m"], p["tile_n"]
    if p["kernel"] == mi.KERNEL_ROWS:
        return out, tile, (4 if M <= 4 else 8 if M <= 8 else 16) if p["tile_m"] == 16 else p["tile_m"]
    return out, tile, out != mi.MXFP4 and N % (128 if p["kernel"] == mi.KERNEL_PIPE_MIXED else p["tile_n"]) != 0


def test_the_gpu_tests_reach_every_kernel():
    """Everything that a product of any size takes on an MI355X is in the shapes of the GPU tests."""
    import test_gpu_mx_tiles as tiles
    import test_gpu_mxfp4 as basic

    tested = {_kernel(M, N, K, out, cus) for M, N, K in basic.GEMMS for out in (mi.F32, mi.BF16) for cus in (256, 8, 1)}
    packed = next(m.args[1] for m in basic.test_packed_product_bit_by_bit.pytestmark if m.args[0] == "shape")
    tested |= {_kernel(M, N, K, mi.MXFP4, cus) for M, N, K in packed for cus in (256, 8, 1)}
    tested |= {_kernel(M, N, K, tiles.OUT[out], cus) for _, (out, M, N, K, cus) in tiles.CASES}
    rng = random.Random(3)
    taken = {}
    for _ in range(150000):
        M, N, K = (int(2 ** rng.uniform(0, most)) for most in (13, 14.5, 15))
        if rng.random() < 0.4:
            N = max(256, N // 256 * 256)
        out = rng.choice(OUTS)
        taken.setdefault(_kernel(M, N, K, out, 256), (M, N, K))
    assert len(taken) >= 50
    assert not {k: v for k, v in taken.items() if k not in tested}


def test_refusals():
    for args, text in (((0, 4, 4), "M=0"), ((4, -1, 4), "N=-1"), ((4, 4, (1 << 26) + 1), "K="), ((MOST, 4, 4), "too large"),
                       ((4, 4, 4, 3), "out=3"), ((4, 4, 4, 0, 0), "cus=0"), ((1 << 20, 1 << 20, 1), "too large"),
                       ((1 << 29, 1024, 4, mi.MXFP4), "too large")):
        with pytest.raises(mi.MiaieError, match=text):
            mi.plan_gemm_mxfp4(*args)
