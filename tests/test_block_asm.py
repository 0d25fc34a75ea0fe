"""The generated gfx950 assembly (this build's, CPU only) of what
tests/test_mx_asm.py leaves out: the mixed tiles of the MXFP4 products, whose
matrix instructions are the pipelined kernel's inline assembly in a register
allocation of their own, that every instantiation of either is there and checked,
and the scratch memory of the norms' kernels."""
import os
import re
import subprocess

import pytest

import test_gemm16_asm as g
from test_mx_asm import MFMA, asm, step  # noqa: F401  (fixtures)

TILES = r"\S*gemm_mx_(?:pipe|mixed)\S*"
# three tiles, and mixed ones: fp32 and bf16 results each with and without columns that end inside a tile, packed
# results with and without the ReLU
N_PIPE, N_MIXED = 18, 6


def _metadata(s):
    """(name, bytes of scratch a thread, spilled registers) of every kernel."""
    for blk in s[s.index("amdhsa.kernels:"):].split("\n  - ")[1:]:
        m = re.search(r"\.name:\s+(\S+)", blk)
        if m:
            yield (m.group(1), *(int(re.search(rf"\.{key}:\s+(\d+)", blk).group(1))
                                 for key in ("private_segment_fixed_size", "vgpr_spill_count")))


def test_every_tile_is_there(asm):  # noqa: F811
    names = [n for n, _ in g._functions(asm, TILES)]
    assert sum("gemm_mx_pipe" in n for n in names) == N_PIPE and sum("gemm_mx_mixed" in n for n in names) == N_MIXED, names


def test_every_tile_is_free_of_scratch_and_hazards(asm, step):  # noqa: F811
    g._check_no_scratch(asm, "gemm_mx_pipe")
    g._check_no_scratch(asm, "gemm_mx_mixed")
    for name, body in g._functions(asm, TILES):
        # one kernel at a time: each has matrix instructions, all of them checked
        issued = sum(line.split()[0] == MFMA for line in body.split("\n") if line.split())
        checked = g._check_hazards(f"{name}:\n{body}.Lfunc_end0:\n", re.escape(name), MFMA)
        # twelve k-tiles in the text (four steady, two between, six at the end) of one instruction a 16 x 16 block
        blocks = 64 + 32 if "mixed" in name else 64 if "Li256ELi256E" in name else 32 if "Li256ELi128E" in name else 16
        assert checked == issued == 12 * blocks, (name, checked, issued)


def test_row_products_are_free_of_scratch(asm):  # noqa: F811
    g._check_no_scratch(asm, "gemm_mx_rows")


def test_scratch_of_the_norms(tmp_path):
    """What norm_block.hip says of its kernels: only the gradients of rows over 8192 columns, and of fp32 rows of 513
    to 4096, have registers in scratch memory, 60 bytes a thread at most."""
    if not g._have_hipcc():
        pytest.skip("hipcc not available")
    out = tmp_path / "norm_block.s"
    subprocess.run([g.HIPCC, *g.FLAGS, os.path.join(g.ROOT, "aiehlc_amd", "csrc", "norm_block.hip"), "-o", str(out)],
                   check=True, capture_output=True)
    kernels = list(_metadata(out.read_text()))
    assert sum("norm_fwd" in n for n, *_ in kernels) == 24 and sum("norm_bwd" in n for n, *_ in kernels) == 24
    for name, scratch, spilled in kernels:
        wide = "norm_bwd" in name and "Li1024ELi2E" in name
        fp32 = "norm_bwdIffLi" in name and any(f"Li{t}ELi1E" in name for t in (128, 256, 512))
        most = 60 if wide else 12 if fp32 else 0
        assert scratch <= most and (spilled == 0 or most), (name, scratch, spilled)
